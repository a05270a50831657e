// Attention of large trees of drafted tokens on the matrix cores (bfloat16): many rows share every key.
//
// A workgroup of W waves takes 32 W rows (nodes x the query heads of one key/value head) and a stretch of the request's slots; keys and
// values go through LDS in tiles of 64 slots, the next tile on its way into registers while the waves multiply the current one, each 32
// rows of its own:
//   S^T[key][row] = K[key][:] . Q[row][:]          O^T[d][row] += V^T[d][key] P^T[key][row]          (v_mfma_f32_32x32x16_bf16)
// Lane (q, h) of a product holds row q and of every 32 slots 16 s + 8 h + 0 .. 7 (s = 0, 1), which is the operand that the second product
// wants: the keys lie in LDS in the order that makes it so (bits 2 and 3 of a slot's number swapped).
// Masks, what is not finite, and parts that several workgroups make of a tile's slots: as in tree_attention_mfma.hip.
//
// Two requests of 64 nodes at 32,768 tokens, 64 heads of 128 on 8: 178 us, 0.56 PFLOP/s, 1.4 TB/s of keys and values in whatever cache they
// lie (all of them in one page: 161).  Matrix cores, vector instructions and LDS are busy a third of that each, and a wave waits for the one
// before the other; with two waves a SIMD little of it overlaps.  Two or four tiles on their way instead of one: the same (179, and for four
// no registers).  Eight waves of 256 rows: 169, and 49 instead of 36 us for one request of 32 nodes at 8,000.  Two blocks of 32 rows a wave,
// the products of one beside the weights of the other, need more registers than a wave has (279).
#include "draft_api.h"
#include "tree_attention.h"

namespace {

template <int D, int PSH, int W>
__global__ void __launch_bounds__(W * kWave) __attribute__((amdgpu_waves_per_eu(2, 2)))
tree_wide_kernel(TreeArgs p, TreeSplit sp) {
    constexpr int THREADS = W * kWave, ROWS = 32 * W, KT = 64, PS = 1 << PSH, PAGES = KT / PS;
    constexpr int KP = D + 8, VP = KT + 8;           // pitches of a key (D values) and of a lane of the values (KT slots) in LDS
    constexpr int DS = D / 16, DB = D / 32, CH = KT * D / 8 / THREADS;      // 16-byte chunks a thread and tile, keys and values each
    constexpr int LD = D == 64 ? 6 : 7, LPC = LD + PSH - 3;      // log2 of D and of a page's chunks
    static_assert(CH >= 1 && LPC >= 6, "a wave's chunks lie in one page");
    typedef const __attribute__((address_space(4))) int32_t *constant_t;
    __shared__ __attribute__((aligned(16))) bf16_t Ks[KT * KP];
    __shared__ __attribute__((aligned(16))) bf16_t Vs[D * VP];
    __shared__ int s_odd, s_seen;

    // the tiles of one (request, part, key/value head) lie on one die, one after the other
    const int G = p.heads / p.kv_heads, TQ = ROWS / G, nkv = p.kv_heads;
    const int unit = (int)(blockIdx.x / 8 / sp.tiles) * 8 + (int)(blockIdx.x % 8), tile = (int)(blockIdx.x / 8) % sp.tiles;
    if (unit >= p.num_segs * sp.splits * nkv) return;
    const int kvh = unit % nkv, split = unit / nkv % sp.splits, seg = unit / nkv / sp.splits;
    const int row0 = max(((constant_t)(uintptr_t)p.seg_start)[seg], 0);
    const int nodes = min(((constant_t)(uintptr_t)p.seg_start)[seg + 1], p.rows) - row0;
    const int kept0 = max(((constant_t)(uintptr_t)p.kept)[seg], 0);
    const int first_node = tile * TQ, ntok = min(min(TQ, nodes - first_node), p.max_nodes - first_node);
    if (ntok <= 0) return;
    const int n = (int)min((long)kept0 + nodes, min((long)p.table_stride << PSH, (long)INT_MAX - 4096));
    const int kept = min(kept0, n);
    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int q = lane & 31, h = lane >> 5;
    const int rr = wave * 32 + q, tq = rr / G, head = kvh * G + (rr - tq * G);
    const int row = tq < ntok ? row0 + first_node + tq : -1;
    const int lo_row = p.window > 0 && row >= 0 ? p.row_pos[row] - p.window + 1 : INT_MIN;
    int lo_min = INT_MIN, lo_max = INT_MIN;      // the first position that a row sees, the lowest and highest over the tile
    if (p.window > 0) {
        lo_min = INT_MAX;
        for (int i = lane; i < ntok; i += kWave) {
            const int lo = p.row_pos[row0 + first_node + i] - p.window + 1;
            lo_min = min(lo_min, lo);
            lo_max = max(lo_max, lo);
        }
#pragma unroll
        for (int step = 32; step > 0; step >>= 1) {
            lo_min = min(lo_min, __shfl_xor(lo_min, step));
            lo_max = max(lo_max, __shfl_xor(lo_max, step));
        }
        lo_min = __builtin_amdgcn_readfirstlane(lo_min);
        lo_max = __builtin_amdgcn_readfirstlane(lo_max);
    }
    const int first = max(0, min(lo_min, kept)) / KT * KT;
    const int live = max(1, (int)min((long)sp.splits, ((long)n - first + sp.per - 1) / sp.per));      // parts that hold slots
    if (split >= live) return;
    const int begin = first + split * sp.per, end = split == sp.splits - 1 ? n : min(n, begin + sp.per);

    bf16x8_t qf[DS];
#pragma unroll
    for (int ds = 0; ds < DS; ds++) {
#pragma unroll
        for (int e = 0; e < 8; e++) qf[ds][e] = (bf16_t)0.0f;
        if (row >= 0) qf[ds] = *(const bf16x8_t *)((const bf16_t *)p.q + (size_t)row * p.q_stride + (size_t)head * D + ds * 16 + h * 8);
        if (sp.negate) {
#pragma unroll
            for (int e = 0; e < 8; e++) qf[ds][e] = -qf[ds][e];
        }
    }

    // What of a chunk's place does not change from tile to tile.  The chunks of a page follow each other: keys with the token fastest.
    int page_of[CH], k_in_page[CH], v_in_page[CH], k_lds[CH], v_lds[CH], v_slot[CH];
#pragma unroll
    for (int c = 0; c < CH; c++) {
        const int ch = threadIdx.x + c * THREADS, in = ch & ((1 << LPC) - 1);
        page_of[c] = __builtin_amdgcn_readfirstlane(ch >> LPC);
        const int key = (page_of[c] << PSH) + (in & (PS - 1)), dc = in >> PSH;
        k_in_page[c] = in * 8;
        // (rows of a 32-slot block are read in the order that swaps bits 2 and 3 of a slot's number)
        k_lds[c] = ((key & ~12) | ((key & 4) << 1) | ((key & 8) >> 1)) * KP + dc * 8;
        const int d = in >> (PSH - 3), hc = in & ((1 << (PSH - 3)) - 1);
        v_in_page[c] = in * 8;
        v_slot[c] = (page_of[c] << PSH) + hc * 8;
        v_lds[c] = d * VP + v_slot[c];
    }
    const size_t page_elems = (size_t)nkv * D * PS, head_at = (size_t)kvh * D * PS;
    const int32_t *tbl = p.tables + (size_t)seg * p.table_stride;
    auto pages = [&](int k0) {      // a tile's pages, one a lane; 0 behind the end
        const int at = k0 + lane * PS;
        return lane < PAGES && at < end ? tbl[at >> PSH] : 0;
    };
    bf16x8_t kreg[CH], vreg[CH];
    auto fetch = [&](int page_lanes) {
#pragma unroll
        for (int c = 0; c < CH; c++) {
            int page = __builtin_amdgcn_readlane(page_lanes, page_of[c]);
            if ((unsigned)page >= (unsigned)p.num_pages) page = 0;      // masked and cleared
            const size_t base = (size_t)page * page_elems + head_at;
            kreg[c] = *(const bf16x8_t *)((const bf16_t *)p.kp + base + (unsigned)k_in_page[c]);
            vreg[c] = *(const bf16x8_t *)((const bf16_t *)p.vp + base + (unsigned)v_in_page[c]);
        }
    };

    f32x16_t o[DB];
#pragma unroll
    for (int db = 0; db < DB; db++)
#pragma unroll
        for (int i = 0; i < 16; i++) o[db][i] = 0.f;
    const float sc = sp.scale, tau = 8.0f / sc, nothing = kNothing / fmaxf(sc, 1.0f);
    float m_run = nothing, l_run = 0.f;       // the reference point in raw units; the sum over the lane's own slots
    if (threadIdx.x == 0) s_odd = 0;
    const int whole_end = min(kept, end) - KT;

    int here = pages(begin);       // the tile's page numbers, one a lane: asked for a tile ahead of its keys and values
    if (begin < end) fetch(here);
    int then = pages(begin + KT);
    for (int k0 = begin; k0 < end; k0 += KT) {
        const unsigned bad = (unsigned)__ballot((unsigned)here >= (unsigned)p.num_pages);
        const bool whole = k0 >= lo_max && k0 <= whole_end && bad == 0;
        const bool nodes_here = k0 + KT > kept;
        // a tile with nodes: the row's bits and the nodes' positions come while the tile is stored and the scores are made
        unsigned long long word_low = 0, word_high = 0;
        int at = INT_MIN;
        if (!whole && nodes_here) {
            const int w = max(k0 - kept, 0) >> 6, j = k0 - kept + lane;
            const int64_t *mine = p.seen + (size_t)max(row, 0) * p.words;
            word_low = (unsigned long long)mine[min(w, p.words - 1)];
            word_high = (unsigned long long)mine[min(w + 1, p.words - 1)];
            if (p.window > 0 && j >= 0 && j < nodes) at = p.row_pos[row0 + j];
        }
        __syncthreads();   // the previous tile has been read
        if (!whole) {
            // Slots that no row sees may hold anything, and weights of zero do not keep a NaN or an infinity out: they are cleared, and so is
            // what is not finite; the rows that see it are given it at the end.
            unsigned odd = 0;
#pragma unroll
            for (int c = 0; c < CH; c++) {
                u32x4_t v = __builtin_bit_cast(u32x4_t, vreg[c]);
                const int from = lo_min <= k0 + v_slot[c] ? 0 : lo_min - (k0 + v_slot[c]), to = (bad >> page_of[c] & 1) ? 0 : n - (k0 + v_slot[c]);
#pragma unroll
                for (int w = 0; w < 4; w++) {
                    v[w] &= (2 * w >= from && 2 * w < to ? 0x0000ffffu : 0u) | (2 * w + 1 >= from && 2 * w + 1 < to ? 0xffff0000u : 0u);
                    const unsigned full = ((v[w] & 0x7f807f80u) + 0x00800080u) & 0x80008000u;      // a full exponent carries into the sign's place
                    odd |= full;
                    v[w] &= ~((full >> 15) * 0xffffu);
                }
                vreg[c] = __builtin_bit_cast(bf16x8_t, v);
            }
            if (__any(odd != 0) && lane == 0) s_odd = 1;
        }
#pragma unroll
        for (int c = 0; c < CH; c++) {
            *(bf16x8_t *)(Ks + k_lds[c]) = kreg[c];
            *(bf16x8_t *)(Vs + v_lds[c]) = vreg[c];
        }
        __syncthreads();
        here = then;
        if (k0 + KT < end) {      // on its way while this tile is multiplied
            fetch(here);
            then = pages(k0 + 2 * KT);
        }

        f32x16_t s[2];
#pragma unroll
        for (int rb = 0; rb < 2; rb++) {
#pragma unroll
            for (int i = 0; i < 16; i++) s[rb][i] = 0.f;
            const bf16_t *krow = Ks + (rb * 32 + q) * KP + h * 8;
#pragma unroll
            for (int ds = 0; ds < DS; ds++)
                s[rb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*(const bf16x8_t *)(krow + ds * 16), qf[ds], s[rb], 0, 0, 0);
        }
        if (!whole) {
            const int to_kept = kept - k0;
            unsigned long long bits = low_bits(to_kept);
            if (p.window > 0) bits &= ~low_bits(lo_row <= k0 ? 0 : min(lo_row - k0, 64));
            if (nodes_here) {
                const int j0 = -to_kept;       // the node at the tile's first slot
                unsigned long long tree;
                if (j0 <= 0) {
                    tree = word_low << -j0;       // -j0 < KT
                } else {
                    const int w = j0 >> 6, sh = j0 & 63;
                    tree = w < p.words ? word_low >> sh : 0ull;
                    if (sh > 0 && w + 1 < p.words) tree |= word_high << (64 - sh);
                }
                if (p.window > 0) {      // a node's position, one a lane, against every row's edge
                    unsigned long long near = 0;
                    for (int r = 0; r < 32; r++) {
                        const unsigned long long one = __ballot(at >= __builtin_amdgcn_readlane(lo_row, r));
                        near = q == r ? one : near;
                    }
                    tree &= near;
                }
                bits |= tree & ~low_bits(to_kept) & low_bits(n - k0);
            }
#pragma unroll
            for (int i = 0; i < PAGES; i++)
                if (bad >> i & 1) bits &= ~(low_bits(PS) << (i * PS));
            if (row < 0) bits = 0;
            bits >>= 8 * h;
#pragma unroll
            for (int rb = 0; rb < 2; rb++)
#pragma unroll
                for (int i = 0; i < 16; i++)
                    if (!(bits >> (rb * 32 + 16 * (i >> 3) + (i & 7)) & 1)) s[rb][i] = -INFINITY;
        }
        float top = -INFINITY;
#pragma unroll
        for (int rb = 0; rb < 2; rb++)
#pragma unroll
            for (int i = 0; i < 16; i++) top = fmaxf(top, s[rb][i]);
        if (__any(top > m_run + tau)) {      // the reference point follows the maximum in steps of 2^8
            top = max_32_apart(top);
            const float m_new = top > m_run + tau ? top : m_run, alpha = exp2_fast((m_run - m_new) * sc);
            l_run *= alpha;
#pragma unroll
            for (int db = 0; db < DB; db++)
#pragma unroll
                for (int i = 0; i < 16; i++) o[db][i] *= alpha;
            m_run = m_new;
        }
        const float mc = m_run * sc;      // finite for a row that has seen nothing
        float sum = 0.f;
#pragma unroll
        for (int rb = 0; rb < 2; rb++)
#pragma unroll
            for (int i = 0; i < 16; i++) {
                s[rb][i] = exp2_fast(fmaf(s[rb][i], sc, -mc));
                sum += s[rb][i];
            }
        l_run += sum;
#pragma unroll
        for (int rb = 0; rb < 2; rb++)
#pragma unroll
            for (int s2 = 0; s2 < 2; s2++) {
                bf16x8_t pf;      // a weight is rounded to bfloat16 where it meets the values
#pragma unroll
                for (int e = 0; e < 8; e++) pf[e] = (bf16_t)s[rb][8 * s2 + e];
#pragma unroll
                for (int db = 0; db < DB; db++) {
                    const bf16x8_t a = *(const bf16x8_t *)(Vs + (db * 32 + q) * VP + rb * 32 + 16 * s2 + 8 * h);
                    o[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, pf, o[db], 0, 0, 0);
                }
            }
    }
    __syncthreads();
    if (s_odd && row >= 0) {      // values that are not finite reach the rows that see them here, slot by slot
        for (int slot = begin; slot < end; slot++) {
            if (!sees_slot<PSH>(p, seg, row0, kept, row, lo_row, slot)) continue;
            const int page = tbl[slot >> PSH];
#pragma unroll
            for (int db = 0; db < DB; db++)
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const float v = (float)((const bf16_t *)p.vp)[(size_t)page * page_elems + head_at + (size_t)(db * 32 + 8 * (i >> 2) + 4 * h + (i & 3)) * PS + (slot & (PS - 1))];
                    if (!(fabsf(v) < INFINITY)) o[db][i] += v;
                }
        }
    }
    float l = sum_32_apart(l_run), m = m_run == nothing ? -INFINITY : m_run * sc;      // in the exponent's units from here on
    if (live > 1) {
        // A part leaves its outputs, maximum and sum, each lane its own; the part that arrives last adds them up in their order.
        const size_t group = ((size_t)seg * nkv + kvh) * sp.tiles + tile;
        const __amdgpu_buffer_rsrc_t meet = workspace_buffer(sp.parts);
        constexpr unsigned kPart = (4 * DB + 1) * THREADS * 16;
        const unsigned base = (unsigned)(group * sp.splits) * kPart + threadIdx.x * 16, mine = base + split * kPart;
#pragma unroll
        for (int db = 0; db < DB; db++)
#pragma unroll
            for (int j = 0; j < 4; j++)
                hand_over(meet, mine + (db * 4 + j) * THREADS * 16, (f32x4_t){o[db][4 * j], o[db][4 * j + 1], o[db][4 * j + 2], o[db][4 * j + 3]});
        hand_over(meet, mine + 4 * DB * THREADS * 16, (f32x4_t){m, l, 0.f, 0.f});
        parts_published();
        __syncthreads();
        int *counter = sp.counters + group;
        if (threadIdx.x == 0) s_seen = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
        if (s_seen != live - 1) return;
        parts_visible();
        if (threadIdx.x == 0) __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);   // for the next launch
        m = -INFINITY;
        l = 0.f;
#pragma unroll
        for (int db = 0; db < DB; db++)
#pragma unroll
            for (int i = 0; i < 16; i++) o[db][i] = 0.f;
        for (int part = 0; part < live; part++) {
            const unsigned from = base + part * kPart;
            f32x4_t got[4 * DB];
            const f32x4_t ml = take_over(meet, from + 4 * DB * THREADS * 16);
#pragma unroll
            for (int i = 0; i < 4 * DB; i++) got[i] = take_over(meet, from + i * THREADS * 16);
            const float m_new = fmaxf(m, ml[0]);
            const float f0 = m == -INFINITY ? 0.f : exp2_fast(m - m_new), f1 = ml[0] == -INFINITY ? 0.f : exp2_fast(ml[0] - m_new);
            m = m_new;
            l = l * f0 + ml[1] * f1;
#pragma unroll
            for (int db = 0; db < DB; db++)
#pragma unroll
                for (int i = 0; i < 16; i++) o[db][i] = o[db][i] * f0 + got[db * 4 + (i >> 2)][i & 3] * f1;
        }
    }
    if (row < 0) return;
    if (p.sinks != nullptr) l += m == -INFINITY ? 1.0f : exp2_fast(p.sinks[head] * kLog2e - m);      // nothing seen: zero either way
    const float inv = l == 0.f ? 0.f : 1.0f / l;
    bf16_t *dst = (bf16_t *)p.out + ((size_t)row * p.heads + head) * D + 4 * h;
#pragma unroll
    for (int db = 0; db < DB; db++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            bf16x4_t v;
#pragma unroll
            for (int i = 0; i < 4; i++) v[i] = (bf16_t)(o[db][4 * j + i] * inv);
            *(bf16x4_t *)(dst + db * 32 + 8 * j) = v;
        }
}

template <int D, int PSH, int W>
int launch(const TreeArgs &a, int max_context, hipStream_t stream) {
    const int G = a.heads / a.kv_heads, TQ = 32 * W / G;
    TreeSplit sp;
    sp.tiles = (a.max_nodes + TQ - 1) / TQ;
    constexpr size_t part_bytes = (size_t)(4 * (D / 32) + 1) * W * kWave * 16;
    plan_tree(a, sp.tiles, 8 / W * compute_units(), 64, 8, max_context, part_bytes, &sp);
    const long units = (long)a.num_segs * sp.splits * a.kv_heads, blocks = (units + 7) / 8 * 8 * sp.tiles;
    FLLM_REQUIRE(blocks <= 0x7fffffffL, "tree_attention: grid too large");
    hipLaunchKernelGGL((tree_wide_kernel<D, PSH, W>), dim3((unsigned)blocks), dim3(W * kWave), 0, stream, a, sp);
    return fllm_check_launch("tree_attention");
}

}  // namespace

// heads of 128, at most 64 query heads a key/value head, pages of 8 to 64 (tree_attention_mfma.hip has checked the rest)
int fllm_tree_attention_wide(const TreeArgs &a, int max_context, hipStream_t stream) {
    if (a.page_size == 8) return launch<128, 3, 4>(a, max_context, stream);
    if (a.page_size == 16) return launch<128, 4, 4>(a, max_context, stream);
    if (a.page_size == 32) return launch<128, 5, 4>(a, max_context, stream);
    return launch<128, 6, 4>(a, max_context, stream);
}
