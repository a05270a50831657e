// Attention of trees of drafted tokens on the matrix cores, bfloat16 and float32: scores, softmax statistics and outputs accumulate in
// float32.
//
// A workgroup of eight waves takes a tile of 16 to 64 rows (nodes x the query heads of one key/value head) and a stretch of the request's
// slots; the waves (or pairs of them, where each has half of the rows) take blocks of neighbouring slots in turn, each with a running
// maximum and sum a row, and meet in LDS at the end.  Keys and values go from the pages straight into matrix operands, the next block's
// on their way while a block is multiplied:
//   S^T[key][row] = K[key][:] . Q[row][:]          O^T[d][row] += V^T[d][key] P^T[key][row]
// so that a lane keeps one row (of every 16) throughout and probabilities never leave its registers.
//   bfloat16  v_mfma_f32_16x16x32: blocks of 32 slots; a lane (c, g) has the scores of row c and wants those of slots 8 g .. 8 g + 7, so that a
//             value load is 16 bytes, 8 neighbouring tokens.
//   float32   v_mfma_f32_16x16x4: blocks of 16 slots; product e of four takes lane d = 16 j + 4 g + e of keys and queries, product i of four
//             the slots 4 g + i: the operands are the elements of 16-byte loads, and the scores are the second product's operand as they are.
// What bounds it, with keys and values in memory: few tiles, the trips to memory that follow each other (a request of 8 nodes at 1,000
// tokens of the 8B sizes 10.2 us, of which an empty launch is 2 and the parts' meeting 3); tiles as many as compute units, what a unit
// gets from L2 (8 requests of up to 26 nodes at 2,048: four tiles read every key, 27 us, 8.5 TB/s of them); full tiles of heads of 64, the
// exponentials and the other vector instructions (32 requests of up to 64 nodes at 6,144 127 us; with every key in L1 112); float32,
// trips to memory (4 requests of up to 13 nodes at 1,500 16.5 us: a wave has six blocks, and waits for 43 % of its time).  Blocks of twice the slots, or keys asked for two blocks ahead, need registers that two waves a SIMD do not have.
// Slots that every row of the tile sees need no mask; a block that holds nodes, the end, the window's edge or a page that is none gets a
// 64-bit mask a row.
#include "common.h"
#include "draft_api.h"
#include "tree_attention.h"

int fllm_tree_attention_wide(const TreeArgs &a, hipStream_t stream);      // tree_attention_wide.hip

namespace {

template <typename T> struct Operand;
template <> struct Operand<bf16_t> {
    typedef bf16x8_t vec;
    static constexpr int kStep = 32;      // slots that a value load of all lanes covers
    static constexpr int kPer = 8;        // elements of a 16-byte load
};
template <> struct Operand<float> {
    typedef f32x4_t vec;
    static constexpr int kStep = 16;
    static constexpr int kPer = 4;
};

// from slots 16 j + 4 g + i of two tiles j to slots 8 g .. 8 g + 7
__device__ __forceinline__ bf16x8_t neighbours(bf16x8_t p) {
    u32x4_t w = __builtin_bit_cast(u32x4_t, p);
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const auto h = __builtin_amdgcn_permlane32_swap(w[i], w[2 + i], false, false);
        const auto q = __builtin_amdgcn_permlane16_swap(h[0], h[1], false, false);
        w[i] = q[0];
        w[2 + i] = q[1];
    }
    return __builtin_bit_cast(bf16x8_t, w);
}

constexpr int q_pitch(int D, bool wide) { return D + (wide ? 4 : 8); }      // elements of a query row in LDS

template <typename T, int D, int ROWS, int KW>
constexpr size_t lds_area() {      // the queries while there are slots, the waves' outputs afterwards
    const size_t queries = (size_t)ROWS * q_pitch(D, sizeof(T) == 4) * sizeof(T), outputs = (size_t)KW * ROWS * (D + 4) * sizeof(float);
    return queries > outputs ? queries : outputs;
}
template <typename T, int D, int ROWS, int KW>
constexpr size_t lds_bytes() {
    return lds_area<T, D, ROWS, KW>() + (size_t)KW * ROWS * 2 * sizeof(float);
}

// The waves are RG groups of rows (16 NT each) times KW groups of slots.  PSH: pages of 1 << PSH tokens; of 8, two a score tile, otherwise of
// 16, 32 or 64.
// ALONE: no other tile reads the same keys.
template <typename T, int D, int NT, int PSH, int RG, int KW, bool ALONE>
__global__ void __launch_bounds__(RG * KW * kWave) __attribute__((amdgpu_waves_per_eu(2, 2)))
tree_attention_kernel(TreeArgs p, TreeSplit sp) {
    typedef typename Operand<T>::vec vec;
    constexpr bool kHalf = sizeof(T) == 2;
    constexpr int PER = Operand<T>::kPer, KB = Operand<T>::kStep, TILES = KB / 16, THREADS = RG * KW * kWave;
    constexpr int KD = D / (4 * PER);       // 16-byte loads of a key a lane
    constexpr bool P8 = PSH == 3;
    constexpr int PS = 1 << PSH, PMASK = PS - 1;
    constexpr int DT = D / 16, NP = P8 ? 2 * TILES : TILES, ROWS = 16 * NT * RG, QP = q_pitch(D, !kHalf), OP = D + 4;
    typedef const __attribute__((address_space(4))) int32_t *constant_t;      // the same for every lane: a scalar load
    // what a full exponent adds up to, in the halves of a word or in all of it
    constexpr unsigned kExponents = kHalf ? 0x7f807f80u : 0x7f800000u, kExponentStep = kHalf ? 0x00800080u : 0x00800000u,
                       kSigns = kHalf ? 0x80008000u : 0x80000000u;
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
    __shared__ int s_row[ROWS], s_lo[ROWS];      // a row's number (-1: none) and the first position it sees
    __shared__ int s_odd;      // a block held values that are not finite and had to be cleared
    T *qs = (T *)lds;                                                     // [ROWS][QP]
    float *sm_o = (float *)lds;                                           // [KW][ROWS][OP], when the queries have served
    float *sm_m = (float *)(lds + lds_area<T, D, ROWS, KW>()), *sm_l = sm_m + KW * ROWS;

    // One grid dimension: the tiles of one (request, part, key/value head) lie on one die, one after the other, so that what the first
    // reads from memory the others find in its L2.
    const int G = p.heads / p.kv_heads, TQ = ROWS / G;
    const int unit = (int)(blockIdx.x / 8 / sp.tiles) * 8 + (int)(blockIdx.x % 8), tile = (int)(blockIdx.x / 8) % sp.tiles;
    if (unit >= p.num_segs * sp.splits * p.kv_heads) return;
    const int kvh = unit % p.kv_heads, split = unit / p.kv_heads % sp.splits;
    int seg = unit / p.kv_heads / sp.splits;
    if (sp.sorted) {      // the longest request first
        const int l = threadIdx.x & (kWave - 1), length = l < p.num_segs ? p.kept[l] : INT_MIN;
        int rank = 0;
        for (int r = 0; r < p.num_segs; r++) {
            const int other = __builtin_amdgcn_readlane(length, r);
            rank += other > length || (other == length && r < l);
        }
        seg = __builtin_ctzll(__ballot(rank == seg));
    }
    const int row0 = max(((constant_t)(uintptr_t)p.seg_start)[seg], 0);
    const int nodes = min(((constant_t)(uintptr_t)p.seg_start)[seg + 1], p.rows) - row0;
    const int kept0 = max(((constant_t)(uintptr_t)p.kept)[seg], 0);
    const int first_node = tile * TQ, ntok = min(min(TQ, nodes - first_node), p.max_nodes - first_node);
    if (ntok <= 0) return;
    const int nkv = p.kv_heads;
    const int n = (int)min((long)kept0 + nodes, min((long)p.table_stride << PSH, (long)INT_MAX - 4096));
    const int kept = min(kept0, n);
    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int c = lane & 15, g = lane >> 4;
    const int kw = wave / RG, at_row = wave % RG * (16 * NT) + c;      // the wave's slots, and the lane's row of its first tile

    // the first position that a row sees, the lowest and highest over the tile (a node a lane)
    int lo_min = INT_MIN, lo_max = INT_MIN;
    if (p.window > 0) {
        lo_min = lo_max = p.row_pos[row0 + first_node + min(lane, ntok - 1)] - p.window + 1;
#pragma unroll
        for (int step = 32; step > 0; step >>= 1) {
            lo_min = min(lo_min, __shfl_xor(lo_min, step));
            lo_max = max(lo_max, __shfl_xor(lo_max, step));
        }
        lo_min = __builtin_amdgcn_readfirstlane(lo_min);
        lo_max = __builtin_amdgcn_readfirstlane(lo_max);
    }
    const int first = max(0, min(lo_min, kept)) / KB * KB;
    const int live = max(1, (int)min((long)sp.splits, ((long)n - first + sp.per - 1) / sp.per));      // parts that hold slots
    if (split >= live) return;
    const int begin = first + split * sp.per, end = split == sp.splits - 1 ? n : min(n, begin + sp.per);

    const constant_t tbl = (constant_t)(uintptr_t)(p.tables + (size_t)seg * p.table_stride);
    struct Pages {
        int page[NP];
        unsigned bad;       // a bit an entry that names no page (it reads page 0 and is masked)
    };
    auto block_pages = [&](int kb) {      // kb may lie behind the end: nothing is asked for there
        Pages pg;
        pg.bad = 0;
#pragma unroll
        for (int i = 0; i < NP; i++) {
            const int at = kb + i * (P8 ? 8 : 16);
            const int page = at < end ? tbl[at >> PSH] : 0;
            const bool good = (unsigned)page < (unsigned)p.num_pages;
            pg.page[i] = good ? page : 0;
            pg.bad |= good ? 0u : 1u << i;
        }
        return pg;
    };
    vec kf[TILES][KD], vf[DT];
    // A lane's place in a page is the same in every block; the rest of an address is a scalar wherever one page serves all lanes.
    constexpr size_t kHeadBytes = (size_t)D * PS * sizeof(T);
    // Rows of the score tiles.  A tile alone reads a key once, from memory: row c of score tile k is slot 16 k + c, a load is whole lines, carries
    // the non-temporal hint, and probabilities change lanes for it.  Where several tiles read the same keys most come from L2, and what
    // counts is the instructions: row c of score tile k is slot 8 (c / 4) + 4 (k % 2) + c % 4, so that a lane's
    // scores are of the neighbouring slots that its values are of.  Microseconds with one order and the hint / with the other: 8 requests
    // of 8 nodes at 16,000 kept tokens 62 / 75; of 26 nodes at 2,000 (4 tiles a key/value head) 23.6 / 19.8.
    constexpr bool kSwap = kHalf && ALONE, kNear = kHalf && !ALONE;
    const int k_token = kNear ? (P8 ? c & 3 : PSH == 4 ? (c & 3) + 8 * (c >> 2 & 1) : (c & 3) + 8 * (c >> 2)) : P8 ? c & 7 : c;
    const unsigned k_lane = kHalf ? (unsigned)(g * PS + k_token) * 16 : (unsigned)((g >> 1) * PS + k_token) * 32 + (g & 1) * 16;
    // piece j of a block's keys
    auto load_keys = [&](int kb, const Pages &pg, int j) __attribute__((always_inline)) {
        const size_t page_bytes = (size_t)nkv * kHeadBytes;
#pragma unroll
        for (int t = 0; t < TILES; t++) {
            const char *base = (const char *)p.kp + (size_t)kvh * kHeadBytes;
            if constexpr (kNear) {
                if constexpr (P8) base += (size_t)(c < 8 ? (c < 4 ? pg.page[0] : pg.page[1]) : (c < 12 ? pg.page[2] : pg.page[3])) * page_bytes;
                else if constexpr (PSH == 4) base += (size_t)(c < 8 ? pg.page[0] : pg.page[1]) * page_bytes;
                else base += (size_t)pg.page[0] * page_bytes + (size_t)(kb & PMASK) * 16;
                base += (t & 1) * 64;
            } else {
                if constexpr (P8) base += (size_t)(c < 8 ? pg.page[2 * t] : pg.page[2 * t + 1]) * page_bytes;
                else base += (size_t)pg.page[t] * page_bytes + (size_t)((kb + 16 * t) & PMASK) * (8 * sizeof(T));
            }
            const vec *from = (const vec *)(base + j * 64 * PS + k_lane);
            if constexpr (ALONE) kf[t][j] = __builtin_nontemporal_load(from);
            else kf[t][j] = *from;
        }
    };
    // values: bfloat16 the slots 8 g .. + 7 of a block, float32 4 g .. + 3
    const unsigned v_lane = (unsigned)(c * PS + (kHalf ? (P8 ? 0 : PSH == 4 ? 8 * (g & 1) : 8 * g) : (P8 ? 4 * (g & 1) : 4 * g))) * (unsigned)sizeof(T);
    // lanes 16 dt .. 16 dt + 15 of a block's values
    auto load_values = [&](int kb, const Pages &pg, int dt) __attribute__((always_inline)) {
        const char *base = (const char *)p.vp + (size_t)kvh * kHeadBytes;
        const size_t page_bytes = (size_t)nkv * kHeadBytes;
        if constexpr (kHalf && P8) base += (size_t)(g < 2 ? (g == 0 ? pg.page[0] : pg.page[1]) : (g == 2 ? pg.page[2] : pg.page[3])) * page_bytes;
        else if constexpr (kHalf ? PSH == 4 : P8) base += (size_t)(g < 2 ? pg.page[0] : pg.page[1]) * page_bytes;
        else base += (size_t)pg.page[0] * page_bytes + (size_t)(kb & PMASK) * sizeof(T);
        vf[dt] = *(const vec *)(base + dt * 16 * PS * (int)sizeof(T) + v_lane);
    };
    // The words of a block's nodes for the lane's row of tile t: the one that holds the first (bit j0 % 64) and the one behind it.
    struct Words {
        unsigned long long low, high;
    };
    auto words_of = [&](int t, int kb) {
        const int w = max(kb - kept, 0) >> 6;
        const int64_t *mine = p.seen + (size_t)max(s_row[at_row + t * 16], 0) * p.words;
        return Words{(unsigned long long)mine[min(w, p.words - 1)], (unsigned long long)mine[min(w + 1, p.words - 1)]};
    };
    // Which of the block's slots the lane's row of tile t sees, a bit a slot; `at` is the position of node kb - kept + lane.
    auto sight = [&](int t, int kb, unsigned bad, const Words &words, int at) -> unsigned long long {
        const int to_kept = kept - kb, lo = s_lo[at_row + t * 16];
        unsigned long long bits = low_bits(to_kept);
        if (p.window > 0) bits &= ~low_bits(lo <= kb ? 0 : min(lo - kb, 64));
        if (kb + KB > kept) {
            const int j0 = kb - kept;       // the node at the block's first slot
            unsigned long long tree;
            if (j0 <= 0) {
                tree = words.low << -j0;       // -j0 < KB
            } else {
                const int w = j0 >> 6, s = j0 & 63;
                tree = w < p.words ? words.low >> s : 0ull;
                if (s > 0 && w + 1 < p.words) tree |= words.high << (64 - s);
            }
            if (p.window > 0) {      // a node's position, one a lane, against every row's edge
                unsigned long long near = 0;
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    const unsigned long long one = __ballot(at >= __builtin_amdgcn_readlane(lo, r));
                    near = c == r ? one : near;
                }
                tree &= near;
            }
            bits |= tree & ~low_bits(to_kept) & low_bits(n - kb);
        }
        if (bad != 0) {
#pragma unroll
            for (int i = 0; i < NP; i++)
                if (bad >> i & 1) bits &= ~(low_bits(P8 ? 8 : 16) << (i * (P8 ? 8 : 16)));
        }
        return s_row[at_row + t * 16] < 0 ? 0ull : bits;
    };

    const float sc = sp.scale, tau = 8.0f / sc, nothing = kNothing / fmaxf(sc, 1.0f);
    f32x4_t o[NT][DT];
    float m_run[NT], l_run[NT];      // the reference point in raw units; the sum over the lane's own slots
#pragma unroll
    for (int t = 0; t < NT; t++) {
        m_run[t] = nothing;
        l_run[t] = 0.f;
#pragma unroll
        for (int dt = 0; dt < DT; dt++) o[t][dt] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
    }

    int kb = begin + kw * KB;
    Pages pg = block_pages(kb);
#pragma unroll
    for (int j = 0; j < KD; j++) load_keys(kb, pg, j);      // behind the end: page 0, for nobody
    if (threadIdx.x == 0) s_odd = 0;
    if ((int)threadIdx.x < ROWS) {
        const int tq = (int)threadIdx.x / G, row = row0 + first_node + tq;
        s_row[threadIdx.x] = tq < ntok ? row : -1;
        s_lo[threadIdx.x] = p.window > 0 && tq < ntok ? p.row_pos[row] - p.window + 1 : INT_MIN;
    }
    // the queries, while the first keys are on their way
    for (int i = threadIdx.x; i < ROWS * (D / PER); i += THREADS) {
        const int r = i / (D / PER), d = (i - r * (D / PER)) * PER;
        const int tq = r / G, hg = r - tq * G;
        vec v;
#pragma unroll
        for (int e = 0; e < PER; e++) v[e] = (T)0.0f;
        if (tq < ntok) v = *(const vec *)((const T *)p.q + (size_t)(row0 + first_node + tq) * p.q_stride + (size_t)(kvh * G + hg) * D + d);
        if (sp.negate) {
#pragma unroll
            for (int e = 0; e < PER; e++) v[e] = -v[e];
        }
        *(vec *)(qs + r * QP + d) = v;
    }
    __builtin_amdgcn_sched_barrier(0);       // loads come back in order: the scores do not wait for the values
    // (without a condition of their own: where it could have been skipped, keys would be waited for as if no values came after them)
#pragma unroll
    for (int dt = 0; dt < DT; dt++) load_values(kb, pg, dt);
    __syncthreads();
    // heads of 64 leave registers for the queries (32 requests of up to 64 nodes at 6,144: 134 -> 128 us); of 128 they stay in LDS
    constexpr bool kHeld = D == 64;
    vec qf[kHeld ? NT : 1][KD];
    if constexpr (kHeld) {
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int j = 0; j < KD; j++) qf[t][j] = *(const vec *)(qs + (at_row + t * 16) * QP + (4 * j + g) * PER);
    }
    unsigned bad = pg.bad;
    // a block's scores, weights and products; the next block's keys and values are asked for as soon as this one's are used
    auto block = [&](auto whole_block) __attribute__((always_inline)) {
        constexpr bool WHOLE = decltype(whole_block)::value;
        const int next = kb + KW * KB;
        f32x4_t s[NT][TILES];
        unsigned long long any = 0;      // the slots that a row sees
        bool grown = false;
        // a block with nodes: their bits and positions come while the scores are made
        Words words[NT];
        int at = INT_MIN;
        if constexpr (!WHOLE) {
            if (kb + KB > kept) {
#pragma unroll
                for (int t = 0; t < NT; t++) words[t] = words_of(t, kb);
                const int j = kb - kept + lane;
                if (p.window > 0 && lane < KB && j >= 0 && j < nodes) at = p.row_pos[row0 + j];
            }
        }
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int k = 0; k < TILES; k++) s[t][k] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
        constexpr int kQueries = kHeld || !kHalf ? 1 : KD * NT;
        vec ring[kQueries];
        if constexpr (!kHeld && kHalf) {      // all on their way at once (16 requests of up to 24 nodes in a window of 1,024 22.7 -> 22.2 us)
#pragma unroll
            for (int i = 0; i < kQueries; i++) ring[i] = *(const vec *)(qs + (at_row + i % NT * 16) * QP + (4 * (i / NT) + g) * PER);
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int j = 0; j < KD; j++) {
#pragma unroll
            for (int t = 0; t < NT; t++) {
                vec qv;
                if constexpr (kHeld) qv = qf[t][j];
                else if constexpr (kHalf) qv = ring[j * NT + t];
                else qv = *(const vec *)(qs + (at_row + t * 16) * QP + (4 * j + g) * PER);
#pragma unroll
                for (int k = 0; k < TILES; k++) {
                    if constexpr (kHalf) {
                        s[t][k] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[k][j], qv, s[t][k], 0, 0, 0);
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; e++) s[t][k] = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[k][j][e], qv[e], s[t][k], 0, 0, 0);
                    }
                }
            }
            load_keys(next, pg, j);      // behind the last block: page 0, for nobody
        }
#pragma unroll
        for (int t = 0; t < NT; t++) {
            if constexpr (!WHOLE) {
                unsigned long long bits = sight(t, kb, bad, words[t], at);
                any |= bits;
                bits >>= kNear ? 8 * g : 4 * g;
#pragma unroll
                for (int k = 0; k < TILES; k++)
#pragma unroll
                    for (int i = 0; i < 4; i++) s[t][k][i] = bits >> (kNear ? 32 * (k >> 1) + 4 * (k & 1) + i : 16 * k + i) & 1 ? s[t][k][i] : -INFINITY;
            }
            float top = -INFINITY;
#pragma unroll
            for (int k = 0; k < TILES; k++)
#pragma unroll
                for (int i = 0; i < 4; i++) top = fmaxf(top, s[t][k][i]);
            grown |= top > m_run[t] + tau;
        }
        // The reference point follows the maximum only when that has grown by more than 2^8 in the exponent's units: until then weights are
        // at most 256 times their final size, which sums and operands hold as well, nothing is rescaled and no lane asks another.
        if (__any(grown)) {
#pragma unroll
            for (int t = 0; t < NT; t++) {
                float top = -INFINITY;
#pragma unroll
                for (int k = 0; k < TILES; k++)
#pragma unroll
                    for (int i = 0; i < 4; i++) top = fmaxf(top, s[t][k][i]);
                top = max_32_apart(max_16_apart(top));
                const float m_new = top > m_run[t] + tau ? top : m_run[t];
                const float alpha = exp2_fast((m_run[t] - m_new) * sc);
                l_run[t] *= alpha;
#pragma unroll
                for (int dt = 0; dt < DT; dt++) o[t][dt] *= alpha;
                m_run[t] = m_new;
            }
        }
        vec pv[NT];        // the weights as the second product takes them
#pragma unroll
        for (int t = 0; t < NT; t++) {
            const float mc = m_run[t] * sc;      // finite for a row that has seen nothing
            float sum = 0.f;
#pragma unroll
            for (int k = 0; k < TILES; k++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    s[t][k][i] = exp2_fast(fmaf(s[t][k][i], sc, -mc));
                    sum += s[t][k][i];
                }
            l_run[t] += sum;
            // rounded to bfloat16 where they meet the values, which the matrix instruction takes in one type; sums stay in float32
            if constexpr (kSwap) pv[t] = neighbours(pack8(s[t][0], s[t][1]));
            else if constexpr (kHalf) pv[t] = pack8(s[t][0], s[t][1]);
            else pv[t] = s[t][0];
        }
        if constexpr (!WHOLE) {
            // Slots that nobody sees may hold anything, and weights of zero do not keep a NaN or an infinity out: they are cleared.
            // So is what is not finite and only some rows see; those rows are given it at the end.
#pragma unroll
            for (int step = 8; step > 0; step >>= 1) any |= __shfl_xor(any, step);
            unsigned odd = 0;
            const unsigned mine = (unsigned)(any >> (PER * g));
            u32x4_t keep;
#pragma unroll
            for (int w = 0; w < 4; w++) {
                if constexpr (kHalf) keep[w] = (mine >> (2 * w) & 1 ? 0x0000ffffu : 0u) | (mine >> (2 * w + 1) & 1 ? 0xffff0000u : 0u);
                else keep[w] = mine >> w & 1 ? ~0u : 0u;
            }
#pragma unroll
            for (int dt = 0; dt < DT; dt++) {
                const u32x4_t v = __builtin_bit_cast(u32x4_t, vf[dt]) & keep;
                vf[dt] = __builtin_bit_cast(vec, v);
#pragma unroll
                for (int w = 0; w < 4; w++) odd |= (v[w] & kExponents) + kExponentStep;       // a full exponent carries into the sign's place
            }
            if (__any((odd & kSigns) != 0)) {
                if (lane == 0) s_odd = 1;
#pragma unroll
                for (int dt = 0; dt < DT; dt++) {
                    u32x4_t v = __builtin_bit_cast(u32x4_t, vf[dt]);
#pragma unroll
                    for (int w = 0; w < 4; w++) {
                        const unsigned full = ((v[w] & kExponents) + kExponentStep) & kSigns;      // the sign bits of what is not finite
                        v[w] &= ~(kHalf ? ((full >> 15) * 0xffffu) : ((full >> 31) * 0xffffffffu));
                    }
                    vf[dt] = __builtin_bit_cast(vec, v);
                }
            }
        }
#pragma unroll
        for (int dt = 0; dt < DT; dt++) {
#pragma unroll
            for (int t = 0; t < NT; t++) {
                if constexpr (kHalf) {
                    o[t][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf[dt], pv[t], o[t][dt], 0, 0, 0);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; e++) o[t][dt] = __builtin_amdgcn_mfma_f32_16x16x4f32(vf[dt][e], pv[t][e], o[t][dt], 0, 0, 0);
                }
            }
            load_values(next, pg, dt);
        }
        kb = next;
        bad = pg.bad;
        pg = block_pages(kb + KW * KB);
    };
    if (kb < end) {
        pg = block_pages(kb + KW * KB);
        const int whole_end = min(kept, end) - KB;
        do {
            while (kb >= lo_max && kb <= whole_end && bad == 0) block(std::true_type());      // slots that every row sees
            if (kb >= end) break;
            block(std::false_type());
        } while (kb < end);
    }

    // The groups saw different slots: their statistics and outputs meet, four neighbouring outputs a thread.
    __syncthreads();      // the queries have been read
    const int met = max(1, min(KW, (end - begin + KB - 1) / KB));        // groups that had slots
    auto put_outputs = [&]() {
#pragma unroll
        for (int t = 0; t < NT; t++) {
            if (g == 0) {
                sm_m[kw * ROWS + at_row + t * 16] = m_run[t];
                sm_l[kw * ROWS + at_row + t * 16] = l_run[t];
            }
#pragma unroll
            for (int dt = 0; dt < DT; dt++) *(f32x4_t *)(sm_o + (kw * ROWS + at_row + t * 16) * OP + dt * 16 + 4 * g) = o[t][dt];
        }
    };
#pragma unroll
    for (int t = 0; t < NT; t++) {
        l_run[t] = sum_32_apart(sum_16_apart(l_run[t]));
        m_run[t] = m_run[t] == nothing ? -INFINITY : m_run[t] * sc;      // in the exponent's units from here on
    }
    if (kw < met) put_outputs();
    __syncthreads();
    const int live_rows = ntok * G;
    const size_t group = ((size_t)seg * p.kv_heads + kvh) * sp.tiles + tile;
    constexpr int PART = ROWS * (D + 4);      // floats of a part: outputs, then a maximum and a sum a row (four words a row)
    const __amdgpu_buffer_rsrc_t meet = workspace_buffer(sp.parts);
    auto finish = [&](int r, int d, f32x4_t acc, float m, float l) {
        const int tq = r / G, head = kvh * G + (r - tq * G);
        if (p.sinks != nullptr) l += m == -INFINITY ? 1.0f : exp2_fast(p.sinks[head] * kLog2e - m);      // nothing seen: zero either way
        const float inv = l == 0.f ? 0.f : 1.0f / l;
        T *dst = (T *)p.out + ((size_t)(row0 + first_node + tq) * p.heads + head) * D + d;
        T v[4];
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = (T)(acc[i] * inv);
        if constexpr (kHalf) *(bf16x4_t *)dst = (bf16x4_t){v[0], v[1], v[2], v[3]};
        else *(f32x4_t *)dst = (f32x4_t){v[0], v[1], v[2], v[3]};
    };
    for (int idx = threadIdx.x; idx < live_rows * (D / 4); idx += THREADS) {
        const int r = idx / (D / 4), d = (idx - r * (D / 4)) * 4;
        float m = -INFINITY;
        for (int w = 0; w < met; w++) m = fmaxf(m, sm_m[w * ROWS + r]);
        float l = 0.f;
        f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
        for (int w = 0; w < met; w++) {
            const float mw = sm_m[w * ROWS + r], f = mw == -INFINITY ? 0.f : exp2_fast(mw - m);
            l += sm_l[w * ROWS + r] * f;
            acc += *(const f32x4_t *)(sm_o + (w * ROWS + r) * OP + d) * f;
        }
        if (s_odd) {
            // Values that are not finite reach the rows that see them here: slot by slot, as the plain kernel would.
            const int row = row0 + first_node + r / G, lo = p.window > 0 ? p.row_pos[row] - p.window + 1 : INT_MIN;
            for (int slot = begin; slot < end; slot++) {
                if (!sees_slot<PSH>(p, seg, row0, kept, row, lo, slot)) continue;
                const int page = p.tables[(size_t)seg * p.table_stride + (slot >> PSH)];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float v = (float)((const T *)p.vp)[(((size_t)page * nkv + kvh) * D + d + i) * PS + (slot & PMASK)];
                    if (!(fabsf(v) < INFINITY)) acc[i] += v;
                }
            }
        }
        if (live == 1) {
            finish(r, d, acc, m, l);
        } else {
            const unsigned at = (unsigned)((group * sp.splits + split) * PART * sizeof(float));
            hand_over(meet, at + (unsigned)(r * D + d) * 4, acc);
            if (d == 0) hand_over(meet, at + (unsigned)(ROWS * D + r * 4) * 4, (f32x4_t){m, l, 0.f, 0.f});
        }
    }
    if (live == 1) return;
    // The part that arrives last adds them up, in their order: the result does not depend on which one that is.
    __shared__ int s_seen;
    parts_published();
    __syncthreads();
    int *counter = sp.counters + group;
    if (threadIdx.x == 0) s_seen = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    if (s_seen != live - 1) return;
    parts_visible();
    if (threadIdx.x == 0) __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);   // for the next launch
    const unsigned base = (unsigned)(group * sp.splits * PART * sizeof(float));
    constexpr unsigned kStep = PART * sizeof(float);
    // Eight parts at a time, their statistics and two pieces of their outputs in one trip; later ones move the maximum as slots do.
    for (int idx = threadIdx.x; idx < live_rows * (D / 8); idx += THREADS) {
        const int r = idx / (D / 8), d = (idx - r * (D / 8)) * 4;
        float m = -INFINITY, l = 0.f;
        f32x4_t acc[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
        for (int s0 = 0; s0 < live; s0 += 8) {
            f32x4_t ml[8], part[2][8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const unsigned from = base + min(s0 + i, live - 1) * kStep;
                ml[i] = take_over(meet, from + (unsigned)(ROWS * D + r * 4) * 4);
                part[0][i] = take_over(meet, from + (unsigned)(r * D + d) * 4);
                part[1][i] = take_over(meet, from + (unsigned)(r * D + d + D / 2) * 4);
            }
            float m_new = m;
#pragma unroll
            for (int i = 0; i < 8; i++) m_new = fmaxf(m_new, ml[i][0]);
            const float f = m == -INFINITY ? 0.f : exp2_fast(m - m_new);
            l *= f;
            acc[0] *= f;
            acc[1] *= f;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                if (s0 + i >= live) break;
                const float w = ml[i][0] == -INFINITY ? 0.f : exp2_fast(ml[i][0] - m_new);
                l += ml[i][1] * w;
                acc[0] += part[0][i] * w;
                acc[1] += part[1][i] * w;
            }
            m = m_new;
        }
        finish(r, d, acc[0], m, l);
        finish(r, d + D / 2, acc[1], m, l);
    }
}

template <typename T, int D, int NT, int PSH, int RG, int KW, bool ALONE>
int launch(const TreeArgs &a, int max_context, hipStream_t stream) {
    constexpr int ROWS = 16 * NT * RG;
    constexpr size_t smem = lds_bytes<T, D, ROWS, KW>();
    static_assert(smem + 8 * ROWS + 16 <= 160 * 1024, "more than a compute unit's LDS");
    const int G = a.heads / a.kv_heads, TQ = ROWS / G;
    TreeSplit sp;
    sp.tiles = (a.max_nodes + TQ - 1) / TQ;
    constexpr int round = KW * Operand<T>::kStep;
    constexpr size_t part_bytes = (size_t)ROWS * (D + 4) * sizeof(float);
    plan_tree(a, sp.tiles, compute_units(), round, sizeof(T) == 4 ? 1 : 2, max_context, part_bytes, &sp);
    // Where workgroups wait for each other's compute units the longest requests go first, so that no long one is left for the end: 32 requests of
    // up to 64 nodes at 3,100 to 6,144 tokens (1,024 tiles) 124 -> 120 us, of up to 26 at 6,000 81 -> 78; at 1,000, where looking at the lengths
    // takes longer, 27.5 -> 28.8.
    sp.sorted = a.num_segs > 1 && a.num_segs <= kWave && sp.splits == 1 && (long)a.num_segs * a.kv_heads * sp.tiles > compute_units() && reach_of(a, max_context) >= 4096;
    const long units = (long)a.num_segs * sp.splits * a.kv_heads, blocks = (units + 7) / 8 * 8 * sp.tiles;
    FLLM_REQUIRE(blocks <= 0x7fffffffL, "tree_attention: grid too large");
    static bool raised = false;      // more than the default 64 KiB of dynamic LDS has to be asked for once
    if (!raised) {
        const hipError_t e = hipFuncSetAttribute((const void *)tree_attention_kernel<T, D, NT, PSH, RG, KW, ALONE>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        FLLM_REQUIRE(e == hipSuccess, "tree_attention: cannot raise the LDS limit: %s", hipGetErrorString(e));
        raised = true;
    }
    hipLaunchKernelGGL((tree_attention_kernel<T, D, NT, PSH, RG, KW, ALONE>), dim3((unsigned)blocks), dim3(RG * KW * kWave), smem, stream, a, sp);
    return fllm_check_launch("tree_attention");
}

template <typename T, int D>
int launch_rows(const TreeArgs &a, int max_context, hipStream_t stream) {
    const int G = a.heads / a.kv_heads;
    const long rows = (long)a.max_nodes * G;
    auto go = [&](auto nt, auto rg, auto kw) {
        constexpr int NT = decltype(nt)::value, RG = decltype(rg)::value, KW = decltype(kw)::value;
        const bool alone = a.max_nodes <= 16 * NT * RG / G;
        auto of_page = [&](auto psh) {
            constexpr int PSH = decltype(psh)::value;
            if constexpr (RG == 1 && NT < 4) {
                if (alone) return launch<T, D, NT, PSH, RG, KW, true>(a, max_context, stream);
            }
            return launch<T, D, NT, PSH, RG, KW, false>(a, max_context, stream);
        };
        if (a.page_size == 8) return of_page(std::integral_constant<int, 3>());
        if (a.page_size == 16) return of_page(std::integral_constant<int, 4>());
        if (a.page_size == 32) return of_page(std::integral_constant<int, 5>());
        return of_page(std::integral_constant<int, 6>());
    };
    using one = std::integral_constant<int, 1>;
    using two = std::integral_constant<int, 2>;
    using four = std::integral_constant<int, 4>;
    using eight = std::integral_constant<int, 8>;
    // Which tiles.  All figures in microseconds, with keys and values in memory and in no cache, as a step's layers find them.
    // Of 16 rows while every tile has a compute unit and the keys that the tiles read again are few: a tile's fixed cost (its waves meet in LDS)
    // goes with its rows.  Tiles of 16 / of 32 at 32 heads on 8: a request of 8 nodes at 250, 1,000, 8,000 kept tokens 7.3 / 9.7, 10.8 / 16.2,
    // 19.3 / 20.5, of 26 nodes at 2,000 and 4,000 11.9 / 13.7 and 18.2 / 17.5; 8 requests of 8 at 1,000 and 2,000 15.5 / 17.8 and 21.0 / 18.8.
    const long pairs = (long)a.num_segs * a.kv_heads;
    const auto tiles_of = [&](int height) { return height < G ? LONG_MAX / 4 : pairs * ((a.max_nodes + height / G - 1) / (height / G)); };
    const long reach = reach_of(a, max_context);
    const int asked = fllm_option_tree_rows();
    const long tiles16 = tiles_of(16);
    if (G <= 16 && (asked ? asked == 16 : rows <= 16 || (tiles16 <= compute_units() && (sizeof(T) == 4 || tiles16 * reach <= 200000))))
        return go(one(), one(), eight());
    if constexpr (sizeof(T) == 4) {
        return go(two(), one(), eight());
    } else {
        // Of 32 rows while they fit the device side by side, of 64 where there are more of them.  Heads of 128 go to the kernel whose rows share
        // every key through LDS where there are more tiles than that, or where much is read again.  Tiles of 32 / of 64 / shared: 8 requests
        // of up to 26 nodes (256 tiles of 32) at 1,000, 4,000, 8,000 kept tokens 17.9 / 22.5 / 25.3, 44.1 / 49.4 / 44.7, 78.7 / 83.7 / 65.6; of up
        // to 64 nodes (512) 29.8 / 24.0 / 30.0, 68.6 / 65.0 / 59.5, 115 / 120 / 92; 32 of up to 26 (1,024) at 1,000 61.7 / 48.1 / 41.4.
        // Heads of 64, tiles of 32 / of 64: 8 of up to 26 nodes at 1,000, 4,000, 8,000 11.7 / 14.9, 25.6 / 24.7, 43.2 / 38.1; 32 of up to 26 at
        // 1,000 39.3 / 29.3.
        const long tiles32 = tiles_of(32);
        const bool much = tiles32 * (double)reach > (D == 128 ? 1500000 : 900000);
        if (G <= 32 && (asked ? asked <= 32 : rows <= 32 || (tiles32 <= compute_units() && !much))) return go(two(), one(), eight());
        if constexpr (D == 64) return go(four(), one(), eight());
        else if (asked ? asked == 128 : much || tiles_of(64) >= 2 * compute_units()) return fllm_tree_attention_wide(a, stream);
        else return go(two(), two(), four());
    }
}

}  // namespace

// 0: launched, negative: error, 1: shape declined (the caller uses the plain kernel)
int fllm_tree_attention_fast(const TreeArgs &a, int head_dim, int v_dim, int key_chunk, int dtype, int max_context, hipStream_t stream) {
    if (!fllm_fast_kernels_enabled()) return 1;
    if (v_dim != head_dim || key_chunk != 8 || (head_dim != 64 && head_dim != 128)) return 1;
    if (a.page_size != 8 && a.page_size != 16 && a.page_size != 32 && a.page_size != 64) return 1;
    const int G = a.heads / a.kv_heads, size = dtype == FLLM_F32 ? 4 : 2;
    if (G > (dtype == FLLM_F32 ? 32 : 64)) return 1;                   // a tile holds whole nodes
    const float size_of_scale = a.scale < 0.f ? -a.scale : a.scale;
    if (!(size_of_scale > 1e-30f && size_of_scale < 1e30f)) return 1;      // the reference point's step is a quotient of it
    if ((long)a.q_stride * size % 16 != 0 || (((uintptr_t)a.q | (uintptr_t)a.kp | (uintptr_t)a.vp | (uintptr_t)a.out) & 15) != 0) return 1;      // 16-byte loads
    if (dtype == FLLM_F32) return head_dim == 64 ? launch_rows<float, 64>(a, max_context, stream) : launch_rows<float, 128>(a, max_context, stream);
    return head_dim == 64 ? launch_rows<bf16_t, 64>(a, max_context, stream) : launch_rows<bf16_t, 128>(a, max_context, stream);
}
