// Attention of large trees of drafted tokens on the matrix cores (bfloat16): many rows share every key.
//
// A workgroup of four waves takes 128 rows (nodes x the query heads of one key/value head) and a stretch of the request's slots; keys and
// values go through LDS in tiles of 64 slots, the next tile on its way into registers while the waves multiply the current one, each 32
// rows of its own:
//   S^T[key][row] = K[key][:] . Q[row][:]          O^T[d][row] += V^T[d][key] P^T[key][row]          (v_mfma_f32_32x32x16_bf16)
// Lane (q, h) of a product holds row q and of every 32 slots 16 s + 8 h + 0 .. 7 (s = 0, 1), which is the operand that the second product
// wants: the keys lie in LDS in the order that makes it so (bits 2 and 3 of a slot's number swapped).
// Masks, what is not finite, and parts that several workgroups make of a tile's slots: as in tree_attention_mfma.hip.
//
// Two requests of 64 and 34 nodes at 32,768 and 28,593 tokens, 64 heads of 128 on 8: 142 us, 0.71 PFLOP/s (from memory 145).  Bound by the matrix
// cores' rate on real numbers, 1.7 to 1.95 PFLOP/s (zeros: 2.5), and by what does not fit beside the products: with parts of the loop left out in
// turn the weights took 28 us, LDS reads 12, stores to LDS 15.  One product behind the other on one sum takes 52 cycles instead of 32: the
// scores take turns on two.  Operands are read from LDS six products ahead (written as a plain loop each is waited for: 178 us -> 164), the requests' slots are
// cut by what their lengths are (164 -> 155), the weights of a tile's second half are made between the products of the first, and a wave
// that multiplies goes ahead of the one that makes weights (153 -> 146; either alone 150 to 153).
// The same: 4 or 8 products ahead; two teams of waves that take turns at products and weights between barriers (152 to 158); four tiles on
// their way instead of one has no registers; 64 rows a wave with one wave a SIMD spills (275).

#include "draft_api.h"
#include "tree_attention.h"

namespace {

struct Place {
    int seg, unit, tile;      // request (-1: no work), part x key/value head, row tile
    int parts, per, tiles;    // of the request: parts of its slots, slots a part, tiles
    int start, turn;          // the request's first place on a die, and the die that its first unit lies on
    // the workgroup that has a unit of the request, of this tile
    __device__ __forceinline__ unsigned block_of(int u) const { return (unsigned)((start + u / 8 * tiles + tile) * 8 + (u + turn) % 8); }
};

// Where a workgroup works.  The requests' lengths are known here and not to the host: all of them are looked over (64 at a time, one a lane) and
// cut so that the workgroups that the device holds at a time (sp.places on each of 8 dies) have about as much each: parts of at most `per`
// rounds of KT slots.  The tiles of one (request, part, key/value head) lie on one die, one after the other.  Without places (at least as many
// requests and key/value heads as workgroups) every request stays whole and nothing is looked over.
template <int PSH, int KT>
__device__ __forceinline__ Place find_place(const TreeArgs &p, const TreeSplit &sp, int TQ) {
    const int lane = threadIdx.x & (kWave - 1), mine = blockIdx.x / 8, die = blockIdx.x % 8;
    Place at = {-1, 0, 0, 1, 1 << 28, 1, 0, 0};
    if (sp.places == 0) {
        const int unit = mine / sp.tiles * 8 + die;
        at.tile = mine % sp.tiles;
        at.unit = unit % p.kv_heads;
        if (unit < p.num_segs * p.kv_heads) at.seg = unit / p.kv_heads;
        return at;
    }
    auto request = [&](int s, int &tiles, int &rounds) {
        tiles = rounds = 0;
        if (s >= p.num_segs) return;
        const int row0 = max(p.seg_start[s], 0), nodes = min(p.seg_start[s + 1], p.rows) - row0;
        if (nodes <= 0) return;
        tiles = (min(nodes, p.max_nodes) + TQ - 1) / TQ;
        long n = min((long)max(p.kept[s], 0) + nodes, min((long)p.table_stride << PSH, (long)INT_MAX - 4096));
        if (p.window > 0) n = min(n, (long)p.window + nodes + KT);
        rounds = (int)((n + KT - 1) / KT);
    };
    auto over_lanes = [&](auto v) {
#pragma unroll
        for (int step = 32; step > 0; step >>= 1) v += __shfl_xor(v, step);
        return v;
    };
    float work = 0.f;
    int most = 0;
    for (int s0 = 0; s0 < p.num_segs; s0 += kWave) {
        int tiles, rounds;
        request(s0 + lane, tiles, rounds);
        work += (float)tiles * (float)rounds;
        most = max(most, rounds);
    }
    work = over_lanes(work);
#pragma unroll
    for (int step = 32; step > 0; step >>= 1) most = max(most, __shfl_xor(most, step));
    auto parts_of = [&](int rounds, int per) { return min((rounds + per - 1) / per, kMostSplits); };
    int per = max(sp.per, (int)fminf(work * (float)p.kv_heads / (float)(sp.places * 8), 1e8f));
    while (per < most) {
        int sum = 0;
        for (int s0 = 0; s0 < p.num_segs; s0 += kWave) {
            int tiles, rounds;
            request(s0 + lane, tiles, rounds);
            sum += parts_of(rounds, per) * p.kv_heads * tiles;
        }
        if (over_lanes(sum) <= sp.places * 8) break;
        per += 1 + per / 32;
    }
    int before = 0;
    for (int s0 = 0; s0 < p.num_segs; s0 += kWave) {
        int tiles, rounds;
        request(s0 + lane, tiles, rounds);
        const int parts = parts_of(rounds, per), places = (parts * p.kv_heads + 7) / 8 * tiles;
        int upto = places;
#pragma unroll
        for (int step = 1; step < kWave; step <<= 1) {
            const int low = __shfl_up(upto, step);
            upto += lane >= step ? low : 0;
        }
        const unsigned long long here = __ballot(mine < before + upto);
        if (here != 0) {
            const int from = __builtin_ctzll(here);
            at.parts = __builtin_amdgcn_readlane(parts, from);
            at.tiles = __builtin_amdgcn_readlane(tiles, from);
            rounds = __builtin_amdgcn_readlane(rounds, from);
            at.start = before + __builtin_amdgcn_readlane(upto, from) - __builtin_amdgcn_readlane(places, from);
            at.per = (rounds + at.parts - 1) / at.parts * KT;
            at.tile = (mine - at.start) % at.tiles;
            at.turn = (s0 + from) * p.kv_heads % 8;      // so that few key/value heads use all dies
            at.unit = (mine - at.start) / at.tiles * 8 + (die + 8 - at.turn) % 8;
            if (at.unit < at.parts * p.kv_heads) at.seg = s0 + from;
            break;
        }
        before += __builtin_amdgcn_readlane(upto, kWave - 1);
    }
    return at;
}

// The host's side: `slots` workgroups at a time, where the parts that they leave have room in the device workspace; parts of `least` rounds at
// least.  Returns the places that the grid has on each die.
long plan_places(const TreeArgs &a, int slots, int least, size_t part_bytes, TreeSplit *sp) {
    sp->negate = a.scale < 0.f;
    sp->scale = (a.scale < 0.f ? -a.scale : a.scale) * kLog2e;
    sp->counters = nullptr;
    sp->parts = nullptr;
    sp->splits = 1;
    sp->per = least;
    sp->places = 0;
    const long units = (long)a.num_segs * a.kv_heads, rounded = a.kv_heads % 8 ? (long)a.num_segs * sp->tiles : 0;
    void *ws = nullptr;
    size_t ws_bytes = 0;
    if (units < slots && units * sp->tiles * (long)sizeof(int) <= (long)kWorkspaceCounterBytes && fllm_device_workspace(&ws, &ws_bytes) &&
        ws_bytes > kWorkspaceCounterBytes) {
        const long room = (long)(std::min(ws_bytes - kWorkspaceCounterBytes, (size_t)0x7fffffff) / (8 * part_bytes)) - rounded;
        sp->places = (int)std::max(0l, std::min((long)slots / 8, room));
        sp->counters = (int *)ws;
        sp->parts = (float *)((unsigned char *)ws + kWorkspaceCounterBytes);
    }
    if (sp->places == 0) return (units + 7) / 8 * sp->tiles;
    return std::max((long)a.num_segs * ((a.kv_heads + 7) / 8) * sp->tiles, sp->places + rounded);
}

constexpr int D = 128, W = 4, THREADS = W * kWave, ROWS = 32 * W;       // lanes of a head, waves, rows of a tile

// PSH: pages of 1 << PSH tokens
template <int PSH>
__global__ void __launch_bounds__(THREADS) __attribute__((amdgpu_waves_per_eu(2, 2)))
tree_wide_kernel(TreeArgs p, TreeSplit sp) {
    constexpr int KT = 64, PS = 1 << PSH, PAGES = KT / PS;
    constexpr int KP = D + 8, VP = KT + 8;           // pitches of a key (D values) and of a lane of the values (KT slots) in LDS
    constexpr int DS = D / 16, DB = D / 32, CH = KT * D / 8 / THREADS;      // 16-byte chunks a thread and tile, keys and values each
    constexpr int LPC = 7 + PSH - 3;                 // log2 of a page's chunks
    static_assert((1 << LPC) == D * PS / 8 && LPC >= 6, "a wave's chunks lie in one page");
    typedef const __attribute__((address_space(4))) int32_t *constant_t;
    __shared__ __attribute__((aligned(16))) bf16_t Ks[KT * KP];
    __shared__ __attribute__((aligned(16))) bf16_t Vs[D * VP];
    __shared__ int s_odd, s_seen;

    const int G = p.heads / p.kv_heads, TQ = ROWS / G, nkv = p.kv_heads;
    const Place place = find_place<PSH, KT>(p, sp, TQ);
    if (place.seg < 0) return;
    const int kvh = place.unit % nkv, split = place.unit / nkv, seg = place.seg, tile = place.tile;
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
    const int live = max(1, (int)min((long)place.parts, ((long)n - first + place.per - 1) / place.per));      // parts that hold slots
    if (split >= live) return;
    const int begin = first + split * place.per, end = split == place.parts - 1 ? n : min(n, begin + place.per);

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

    int here = pages(begin), k0 = begin;       // the tile's page numbers, one a lane: asked for a tile ahead of its keys and values
    fetch(here);
    int then = pages(begin + KT);
    constexpr int kAhead = 6;        // operands on their way from LDS: a read takes as long as four products
    auto step = [&](auto whole_tile) __attribute__((always_inline)) {
        constexpr bool WHOLE = decltype(whole_tile)::value;
        const unsigned bad = WHOLE ? 0u : (unsigned)__ballot((unsigned)here >= (unsigned)p.num_pages);
        const bool nodes_here = !WHOLE && k0 + KT > kept;
        // a tile with nodes: the row's bits and the nodes' positions come while the tile is stored and the scores are made
        unsigned long long word_low = 0, word_high = 0;
        int at = INT_MIN;
        if (nodes_here) {
            const int w = max(k0 - kept, 0) >> 6, j = k0 - kept + lane;
            const int64_t *mine = p.seen + (size_t)max(row, 0) * p.words;
            word_low = (unsigned long long)mine[min(w, p.words - 1)];
            word_high = (unsigned long long)mine[min(w + 1, p.words - 1)];
            if (p.window > 0 && j >= 0 && j < nodes) at = p.row_pos[row0 + j];
        }
        __syncthreads();   // the previous tile has been read
        if constexpr (!WHOLE) {
            // Slots that no row sees may hold anything, and weights of zero do not keep a NaN or an infinity out: they are cleared, and so is
            // what is not finite; the rows that see it are given it at the end.  A kept slot is at the position of its number; a node is not, and
            // the window's edge clears none of them.
            const int low = min(lo_min, kept);
            unsigned odd = 0;
#pragma unroll
            for (int c = 0; c < CH; c++) {
                u32x4_t v = __builtin_bit_cast(u32x4_t, vreg[c]);
                const int from = low <= k0 + v_slot[c] ? 0 : low - (k0 + v_slot[c]), to = (bad >> page_of[c] & 1) ? 0 : n - (k0 + v_slot[c]);
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
        fetch(here);      // on its way while this tile is multiplied; behind the last: page 0, for nobody
        then = pages(k0 + 2 * KT);

        f32x16_t s[2];
#pragma unroll
        for (int rb = 0; rb < 2; rb++)
#pragma unroll
            for (int i = 0; i < 16; i++) s[rb][i] = 0.f;
        bf16x8_t ring[kAhead];
        auto key = [&](int i) { return *(const bf16x8_t *)(Ks + (i % 2 * 32 + q) * KP + h * 8 + i / 2 * 16); };
        auto value = [&](int i) { return *(const bf16x8_t *)(Vs + (i % DB * 32 + q) * VP + i / DB * 16 + 8 * h); };
#pragma unroll
        for (int i = 0; i < kAhead; i++) ring[i] = key(i);
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int i = 0; i < 2 * DS; i++) {
            __builtin_amdgcn_sched_barrier(0);
            s[i % 2] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ring[i % kAhead], qf[i / 2], s[i % 2], 0, 0, 0);
            if (i + kAhead < 2 * DS) ring[i % kAhead] = key(i + kAhead);
        }
        if constexpr (!WHOLE) {
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
        __builtin_amdgcn_s_setprio(0);
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
#pragma unroll
        for (int i = 0; i < kAhead; i++) ring[i] = value(i);
        __builtin_amdgcn_sched_barrier(0);
        const float mc = m_run * sc;      // finite for a row that has seen nothing
        bf16x8_t pf[4];
        auto weight = [&](int i) {
            const float w = exp2_fast(fmaf(s[i >> 4][i & 15], sc, -mc));
            l_run += w;
            pf[i >> 3][i & 7] = (bf16_t)w;      // a weight is rounded to bfloat16 where it meets the values
        };
#pragma unroll
        for (int i = 0; i < 16; i++) weight(i);      // those of the second 32 slots beside the products of the first
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int i = 0; i < 4 * DB; i++) {
            __builtin_amdgcn_sched_barrier(0);
            o[i % DB] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ring[i % kAhead], pf[i / DB], o[i % DB], 0, 0, 0);
            if (i + kAhead < 4 * DB) ring[i % kAhead] = value(i + kAhead);
            if (i < 2 * DB) {
#pragma unroll
                for (int e = 0; e < 8 / DB; e++) weight(16 + i * (8 / DB) + e);
            }
        }
        __builtin_amdgcn_s_setprio(0);
        k0 += KT;
    };
    do {
        while (k0 >= lo_max && k0 <= whole_end && __ballot((unsigned)here >= (unsigned)p.num_pages) == 0) step(std::true_type());      // every row sees all of it
        if (k0 >= end) break;
        step(std::false_type());
    } while (k0 < end);
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
        const unsigned mine = blockIdx.x * kPart + threadIdx.x * 16;
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
        for (int part = 0; part < live; part += 2) {      // two in one trip
            f32x4_t got[2][4 * DB], ml[2];
#pragma unroll
            for (int a = 0; a < 2; a++) {
                const unsigned from = place.block_of(min(part + a, live - 1) * nkv + kvh) * kPart + threadIdx.x * 16;
                ml[a] = take_over(meet, from + 4 * DB * THREADS * 16);
#pragma unroll
                for (int i = 0; i < 4 * DB; i++) got[a][i] = take_over(meet, from + i * THREADS * 16);
            }
#pragma unroll
            for (int a = 0; a < 2; a++) {
                if (part + a >= live) break;
                const float m_new = fmaxf(m, ml[a][0]);
                const float f0 = m == -INFINITY ? 0.f : exp2_fast(m - m_new), f1 = ml[a][0] == -INFINITY ? 0.f : exp2_fast(ml[a][0] - m_new);
                m = m_new;
                l = l * f0 + ml[a][1] * f1;
#pragma unroll
                for (int db = 0; db < DB; db++)
#pragma unroll
                    for (int i = 0; i < 16; i++) o[db][i] = o[db][i] * f0 + got[a][db * 4 + (i >> 2)][i & 3] * f1;
            }
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

template <int PSH>
int launch(const TreeArgs &a, hipStream_t stream) {
    const int G = a.heads / a.kv_heads, TQ = ROWS / G;
    TreeSplit sp;
    sp.tiles = (a.max_nodes + TQ - 1) / TQ;
    constexpr size_t part_bytes = (size_t)(4 * (D / 32) + 1) * THREADS * 16;
    const long places = plan_places(a, 8 / W * compute_units(), 8, part_bytes, &sp);
    FLLM_REQUIRE(places <= 0x7fffffffL / 8, "tree_attention: grid too large");
    const long blocks = places * 8;
    hipLaunchKernelGGL(tree_wide_kernel<PSH>, dim3((unsigned)blocks), dim3(THREADS), 0, stream, a, sp);
    return fllm_check_launch("tree_attention");
}

}  // namespace

// heads of 128, at most 64 query heads a key/value head, pages of 8 to 64 (tree_attention_mfma.hip has checked the rest)
int fllm_tree_attention_wide(const TreeArgs &a, hipStream_t stream) {
    if (a.page_size == 8) return launch<3>(a, stream);
    if (a.page_size == 16) return launch<4>(a, stream);
    if (a.page_size == 32) return launch<5>(a, stream);
    return launch<6>(a, stream);
}
