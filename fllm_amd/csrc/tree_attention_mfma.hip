// Attention of trees of drafted tokens on the matrix cores, bfloat16 and float32: scores, softmax statistics and outputs accumulate in
// float32.
//
// A workgroup of four waves takes a tile of 16 NT rows (nodes x the query heads of one key/value head) and a stretch of the request's slots;
// the waves take blocks of neighbouring slots in turn, each with a running maximum and sum a row, and meet in LDS at the end.  Keys and
// values go from the pages straight into matrix operands, the next block's on their way while a block is multiplied:
//   S^T[key][row] = K[key][:] . Q[row][:]          O^T[d][row] += V^T[d][key] P^T[key][row]
// so that a lane keeps one row (of every 16) throughout and probabilities never leave its registers.
//   bfloat16  v_mfma_f32_16x16x32: blocks of 64 slots; a lane (c, g) of a score tile has the slots 4 g + i of row c and wants 8 g .. 8 g + 7,
//             so rows of 16 lanes change places between two tiles and a value load is 16 bytes, 8 neighbouring tokens.
//   float32   v_mfma_f32_16x16x4: blocks of 32 slots; product e of four takes lane d = 16 j + 4 g + e of keys and queries, product i of four
//             the slots 4 g + i: the operands are the elements of 16-byte loads, and the scores are the second product's operand as they are.
// Slots that every row of the tile sees need no mask; a block that holds nodes, the end, the window's edge or a page that is none gets a
// 64-bit mask a row.
#include <algorithm>
#include "common.h"
#include "draft_api.h"
#include "tree_attention.h"

namespace {

constexpr int kWaves = 4;
constexpr int kThreads = kWaves * kWave;
constexpr float kLog2e = 1.4426950408889634f;
typedef __attribute__((ext_vector_type(2))) float f32x2_t;

// What a launch adds to TreeArgs: how the slots are split and where the parts of a tile meet.
struct TreeSplit {
    int tiles;            // row tiles a request at most
    int splits, per;      // parts of the slots, slots a part (the last takes what is left)
    int *counters;        // one per (request, key/value head, tile), zero between launches
    float *parts;         // [request, key/value head, tile][split][16 NT rows of D outputs, then of a maximum and a sum]
    float scale;          // >= 0: the sign has gone into the queries
    int negate;
};

template <typename T> struct Operand;
template <> struct Operand<bf16_t> {
    typedef bf16x8_t vec;
    static constexpr int kTiles = 4;      // score tiles of 16 slots a block
    static constexpr int kPer = 8;        // elements of a 16-byte load
};
template <> struct Operand<float> {
    typedef f32x4_t vec;
    static constexpr int kTiles = 2;
    static constexpr int kPer = 4;
};

__device__ __forceinline__ bf16x8_t pack8(const f32x4_t &lo, const f32x4_t &hi) {
    bf16x8_t p;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        p[i] = (bf16_t)lo[i];
        p[4 + i] = (bf16_t)hi[i];
    }
    return p;
}

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

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// the `count` lowest bits
__device__ __forceinline__ unsigned long long low_bits(int count) {
    return count <= 0 ? 0ull : count >= 64 ? ~0ull : (1ull << count) - 1;
}

constexpr int q_pitch(int D, bool wide) { return D + (wide ? 4 : 8); }      // elements of a query row in LDS

template <typename T, int D, int NT>
constexpr size_t lds_bytes() {
    return (size_t)16 * NT * q_pitch(D, sizeof(T) == 4) * sizeof(T) + (size_t)kWaves * 16 * NT * (D + 4 + 2) * sizeof(float);
}

// PSH: pages of 1 << PSH tokens; of 8, two a score tile, otherwise of 16, 32 or 64.
template <typename T, int D, int NT, int PSH, int EU>
__global__ void __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(EU, EU)))
tree_attention_kernel(TreeArgs p, TreeSplit sp) {
    typedef typename Operand<T>::vec vec;
    constexpr bool kHalf = sizeof(T) == 2;
    constexpr int TILES = Operand<T>::kTiles, PER = Operand<T>::kPer, KB = 16 * TILES;
    constexpr int KD = D / (4 * PER);       // 16-byte loads of a key a lane
    constexpr bool P8 = PSH == 3;
    constexpr int PS = 1 << PSH, PMASK = PS - 1;
    constexpr int DT = D / 16, NP = P8 ? 2 * TILES : TILES, ROWS = 16 * NT, QP = q_pitch(D, !kHalf), OP = D + 4;
    typedef const __attribute__((address_space(4))) int32_t *constant_t;      // the same for every lane: a scalar load
    // what a full exponent adds up to, in the halves of a word or in all of it
    constexpr unsigned kExponents = kHalf ? 0x7f807f80u : 0x7f800000u, kExponentStep = kHalf ? 0x00800080u : 0x00800000u,
                       kSigns = kHalf ? 0x80008000u : 0x80000000u;
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
    __shared__ int s_odd;      // a block held values that are not finite and had to be cleared
    T *qs = (T *)lds;                                                     // [ROWS][QP]
    float *sm_o = (float *)(lds + (size_t)ROWS * QP * sizeof(T));         // [kWaves][ROWS][OP]
    float *sm_m = sm_o + kWaves * ROWS * OP, *sm_l = sm_m + kWaves * ROWS;

    // One grid dimension: the tiles of one (request, part, key/value head) lie on one die, one after the other, so that what the first
    // reads from memory the others find in its L2.
    const int G = p.heads / p.kv_heads, TQ = ROWS / G;
    const int unit = (int)(blockIdx.x / 8 / sp.tiles) * 8 + (int)(blockIdx.x % 8), tile = (int)(blockIdx.x / 8) % sp.tiles;
    if (unit >= p.num_segs * sp.splits * p.kv_heads) return;
    const int kvh = unit % p.kv_heads, split = unit / p.kv_heads % sp.splits, seg = unit / p.kv_heads / sp.splits;
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

    // the first position that a row sees, the lowest and highest over the tile
    int lo_row[NT], lo_min = INT_MIN, lo_max = INT_MIN;
    if (p.window > 0) {
        lo_min = INT_MAX;
#pragma unroll
        for (int t = 0; t < NT; t++) {
            const int tq = (t * 16 + c) / G;
            lo_row[t] = p.row_pos[row0 + first_node + min(tq, ntok - 1)] - p.window + 1;
            lo_min = min(lo_min, lo_row[t]);
            lo_max = max(lo_max, lo_row[t]);
        }
#pragma unroll
        for (int step = 8; step > 0; step >>= 1) {
            lo_min = min(lo_min, __shfl_xor(lo_min, step));
            lo_max = max(lo_max, __shfl_xor(lo_max, step));
        }
        lo_min = __builtin_amdgcn_readfirstlane(lo_min);
        lo_max = __builtin_amdgcn_readfirstlane(lo_max);
    } else {
#pragma unroll
        for (int t = 0; t < NT; t++) lo_row[t] = INT_MIN;
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
    vec kf[TILES][KD], vf[2][DT];
    // A lane's place in a page is the same in every block; the rest of an address is a scalar wherever one page serves all lanes.
    constexpr size_t kHeadBytes = (size_t)D * PS * sizeof(T);
    const unsigned k_lane = kHalf ? (unsigned)(g * PS + (P8 ? c & 7 : c)) * 16 : (unsigned)((g >> 1) * PS + (P8 ? c & 7 : c)) * 32 + (g & 1) * 16;
    auto load_keys = [&](int kb, const Pages &pg) {
#pragma unroll
        for (int t = 0; t < TILES; t++) {
            const char *base = (const char *)p.kp + (size_t)kvh * kHeadBytes + (P8 ? 0 : (size_t)((kb + 16 * t) & PMASK) * (8 * sizeof(T)));
            if (P8) base += (size_t)(c < 8 ? pg.page[P8 ? 2 * t : t] : pg.page[P8 ? 2 * t + 1 : t]) * nkv * kHeadBytes;
            else base += (size_t)pg.page[t] * nkv * kHeadBytes;
#pragma unroll
            for (int j = 0; j < KD; j++) kf[t][j] = __builtin_nontemporal_load((const vec *)(base + j * 64 * PS + k_lane));
        }
    };
    // values: bfloat16 the slots 32 h + 8 g .. + 7, float32 16 h + 4 g .. + 3
    const unsigned v_lane = (unsigned)(c * PS + (kHalf ? (P8 ? 0 : PSH == 4 ? 8 * (g & 1) : 8 * g) : (P8 ? 4 * (g & 1) : 4 * g))) * (unsigned)sizeof(T);
    auto load_values = [&](int kb, const Pages &pg) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const char *base = (const char *)p.vp + (size_t)kvh * kHeadBytes;
            const size_t page_bytes = (size_t)nkv * kHeadBytes;
            if constexpr (kHalf) {
                if constexpr (P8) base += (size_t)(g < 2 ? (g == 0 ? pg.page[4 * h] : pg.page[4 * h + 1]) : (g == 2 ? pg.page[4 * h + 2] : pg.page[4 * h + 3])) * page_bytes;
                else if constexpr (PSH == 4) base += (size_t)(g < 2 ? pg.page[2 * h] : pg.page[2 * h + 1]) * page_bytes;
                else base += (size_t)pg.page[2 * h] * page_bytes + (size_t)((kb + 32 * h) & PMASK) * sizeof(T);
            } else {
                if constexpr (P8) base += (size_t)(g < 2 ? pg.page[2 * h] : pg.page[2 * h + 1]) * page_bytes;
                else base += (size_t)pg.page[h] * page_bytes + (size_t)((kb + 16 * h) & PMASK) * sizeof(T);
            }
#pragma unroll
            for (int dt = 0; dt < DT; dt++) vf[h][dt] = *(const vec *)(base + dt * 16 * PS * (int)sizeof(T) + v_lane);
        }
    };
    // Which of the block's slots the lane's row of tile t sees, a bit a slot.
    auto sight = [&](int t, int kb, unsigned bad) -> unsigned long long {
        const int tq = (t * 16 + c) / G;
        const int to_kept = kept - kb;
        unsigned long long bits = low_bits(to_kept);
        if (p.window > 0) bits &= ~low_bits(lo_row[t] <= kb ? 0 : min(lo_row[t] - kb, 64));
        if (kb + KB > kept) {
            const int j0 = kb - kept;       // the node at the block's first slot
            const int64_t *mine = p.seen + (size_t)(row0 + first_node + min(tq, ntok - 1)) * p.words;
            unsigned long long tree;
            if (j0 <= 0) {
                tree = (unsigned long long)mine[0] << -j0;       // -j0 < KB
            } else {
                const int w = j0 >> 6, s = j0 & 63;
                tree = w < p.words ? (unsigned long long)mine[w] >> s : 0ull;
                if (s > 0 && w + 1 < p.words) tree |= (unsigned long long)mine[w + 1] << (64 - s);
            }
            if (p.window > 0) {      // a node's position, one a lane, against every row's edge
                const int j = j0 + lane;
                const int at = j >= 0 && j < nodes && lane < KB ? p.row_pos[row0 + j] : INT_MIN;
                unsigned long long near = 0;
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    const unsigned long long one = __ballot(at >= __builtin_amdgcn_readlane(lo_row[t], r));
                    near = c == r ? one : near;
                }
                tree &= near;
            }
            bits |= tree & ~low_bits(to_kept) & low_bits(n - kb);
        }
#pragma unroll
        for (int i = 0; i < NP; i++)
            if (bad >> i & 1) bits &= ~(low_bits(P8 ? 8 : 16) << (i * (P8 ? 8 : 16)));
        return tq < ntok ? bits : 0ull;
    };

    f32x4_t o[NT][DT];
    float m_run[NT], l_run[NT];      // the reference point in raw units; the sum over the lane's own slots
#pragma unroll
    for (int t = 0; t < NT; t++) {
        m_run[t] = -INFINITY;
        l_run[t] = 0.f;
#pragma unroll
        for (int dt = 0; dt < DT; dt++) o[t][dt] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
    }
    const float sc = sp.scale, tau = 8.0f / sc;

    int kb = begin + wave * KB;
    Pages pg = block_pages(kb);
    if (kb < end) load_keys(kb, pg);
    if (threadIdx.x == 0) s_odd = 0;
    // the queries, while the first keys are on their way
    for (int i = threadIdx.x; i < ROWS * (D / PER); i += kThreads) {
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
    if (kb < end) load_values(kb, pg);
    __syncthreads();
    unsigned bad = pg.bad;
    // a block's scores, weights and products; the next block's keys and values are asked for as soon as this one's are used
    auto block = [&](auto whole_block) __attribute__((always_inline)) {
        constexpr bool WHOLE = decltype(whole_block)::value;
        const int next = kb + kWaves * KB;
        bf16x8_t pb[NT][2];
        f32x4_t pf[NT][TILES];
        unsigned long long any = 0;      // the slots that a row sees
#pragma unroll
        for (int t = 0; t < NT; t++) {
            f32x4_t s[TILES];
#pragma unroll
            for (int k = 0; k < TILES; k++) s[k] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int j = 0; j < KD; j++) {
                const vec qv = *(const vec *)(qs + (t * 16 + c) * QP + (4 * j + g) * PER);
#pragma unroll
                for (int k = 0; k < TILES; k++) {
                    if constexpr (kHalf) {
                        s[k] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[k][j], qv, s[k], 0, 0, 0);
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; e++) s[k] = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[k][j][e], qv[e], s[k], 0, 0, 0);
                    }
                }
            }
            if constexpr (!WHOLE) {
                unsigned long long bits = sight(t, kb, bad);
                any |= bits;
                bits >>= 4 * g;
#pragma unroll
                for (int k = 0; k < TILES; k++)
#pragma unroll
                    for (int i = 0; i < 4; i++) s[k][i] = bits >> (16 * k + i) & 1 ? s[k][i] : -INFINITY;
            }
            float top = -INFINITY;
#pragma unroll
            for (int k = 0; k < TILES; k++)
#pragma unroll
                for (int i = 0; i < 4; i++) top = fmaxf(top, s[k][i]);
            top = max_32_apart(max_16_apart(top));
            // The reference point follows the maximum only when that has grown by more than 2^8 in the exponent's units: until then
            // weights are at most 256 times their final size, which sums and operands hold as well, and nothing is rescaled.
            const float m_new = top > m_run[t] + tau ? top : m_run[t];
            const float mc = m_new == -INFINITY ? 0.f : m_new * sc;       // nothing seen yet: exp2(-inf) = 0
            if (__any(m_new != m_run[t])) {
                const float alpha = exp2_fast(m_run[t] * sc - mc);
                l_run[t] *= alpha;
#pragma unroll
                for (int dt = 0; dt < DT; dt++) o[t][dt] *= alpha;
                m_run[t] = m_new;
            }
            float sum = 0.f;
#pragma unroll
            for (int k = 0; k < TILES; k++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    s[k][i] = exp2_fast(fmaf(s[k][i], sc, -mc));
                    sum += s[k][i];
                }
            l_run[t] += sum;
            if constexpr (kHalf) {
                pb[t][0] = neighbours(pack8(s[0], s[1]));       // a weight is rounded to bfloat16 where it meets the value
                pb[t][1] = neighbours(pack8(s[2], s[3]));
            } else {
#pragma unroll
                for (int k = 0; k < TILES; k++) pf[t][k] = s[k];
            }
        }
        if (next < end) load_keys(next, pg);
        if constexpr (!WHOLE) {
            // Slots that nobody sees may hold anything, and weights of zero do not keep a NaN or an infinity out: they are cleared.
            // So is what is not finite and only some rows see; those rows are given it at the end.
#pragma unroll
            for (int step = 8; step > 0; step >>= 1) any |= __shfl_xor(any, step);
            unsigned odd = 0;
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const unsigned mine = (unsigned)(any >> (4 * PER * h + PER * g));
                u32x4_t keep;
#pragma unroll
                for (int w = 0; w < 4; w++) {
                    if constexpr (kHalf) keep[w] = (mine >> (2 * w) & 1 ? 0x0000ffffu : 0u) | (mine >> (2 * w + 1) & 1 ? 0xffff0000u : 0u);
                    else keep[w] = mine >> w & 1 ? ~0u : 0u;
                }
#pragma unroll
                for (int dt = 0; dt < DT; dt++) {
                    const u32x4_t v = __builtin_bit_cast(u32x4_t, vf[h][dt]) & keep;
                    vf[h][dt] = __builtin_bit_cast(vec, v);
#pragma unroll
                    for (int w = 0; w < 4; w++) odd |= (v[w] & kExponents) + kExponentStep;       // a full exponent carries into the sign's place
                }
            }
            if (__any((odd & kSigns) != 0)) {
                if (lane == 0) s_odd = 1;
#pragma unroll
                for (int h = 0; h < 2; h++)
#pragma unroll
                    for (int dt = 0; dt < DT; dt++) {
                        u32x4_t v = __builtin_bit_cast(u32x4_t, vf[h][dt]);
#pragma unroll
                        for (int w = 0; w < 4; w++) {
                            const unsigned full = ((v[w] & kExponents) + kExponentStep) & kSigns;      // the sign bits of what is not finite
                            v[w] &= ~(kHalf ? ((full >> 15) * 0xffffu) : ((full >> 31) * 0xffffffffu));
                        }
                        vf[h][dt] = __builtin_bit_cast(vec, v);
                    }
            }
        }
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int dt = 0; dt < DT; dt++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    if constexpr (kHalf) {
                        o[t][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf[h][dt], pb[t][h], o[t][dt], 0, 0, 0);
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; e++) o[t][dt] = __builtin_amdgcn_mfma_f32_16x16x4f32(vf[h][dt][e], pf[t][h][e], o[t][dt], 0, 0, 0);
                    }
                }
        if (next < end) load_values(next, pg);
        kb = next;
        bad = pg.bad;
        pg = block_pages(kb + kWaves * KB);
    };
    if (kb < end) {
        pg = block_pages(kb + kWaves * KB);
        const int whole_end = min(kept, end) - KB;
        do {
        while (kb >= lo_max && kb <= whole_end && bad == 0) block(std::true_type());      // slots that every row sees
        if (kb >= end) break;
        block(std::false_type());
        } while (kb < end);
    }

    // The waves saw different slots: their statistics and outputs meet, four neighbouring outputs a thread.
#pragma unroll
    for (int t = 0; t < NT; t++) {
        const float l = sum_32_apart(sum_16_apart(l_run[t]));
        if (g == 0) {
            sm_m[wave * ROWS + t * 16 + c] = m_run[t] == -INFINITY ? -INFINITY : m_run[t] * sc;      // in the exponent's units from here on
            sm_l[wave * ROWS + t * 16 + c] = l;
        }
#pragma unroll
        for (int dt = 0; dt < DT; dt++) *(f32x4_t *)(sm_o + (wave * ROWS + t * 16 + c) * OP + dt * 16 + 4 * g) = o[t][dt];
    }
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
    for (int idx = threadIdx.x; idx < live_rows * (D / 4); idx += kThreads) {
        const int r = idx / (D / 4), d = (idx - r * (D / 4)) * 4;
        float m = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWaves; w++) m = fmaxf(m, sm_m[w * ROWS + r]);
        float l = 0.f;
        f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < kWaves; w++) {
            const float mw = sm_m[w * ROWS + r], f = mw == -INFINITY ? 0.f : exp2_fast(mw - m);
            l += sm_l[w * ROWS + r] * f;
            acc += *(const f32x4_t *)(sm_o + (w * ROWS + r) * OP + d) * f;
        }
        if (s_odd) {
            // Values that are not finite reach the rows that see them here: slot by slot, as the plain kernel would.
            const int row = row0 + first_node + r / G, lo = p.window > 0 ? p.row_pos[row] - p.window + 1 : INT_MIN;
            for (int slot = begin; slot < end; slot++) {
                const int j = slot - kept, page = p.tables[(size_t)seg * p.table_stride + (slot >> PSH)];
                const bool sees = (unsigned)page < (unsigned)p.num_pages &&
                                  (j < 0 ? slot >= lo : (j >> 6) < p.words && (p.seen[(size_t)row * p.words + (j >> 6)] >> (j & 63) & 1) && p.row_pos[row0 + j] >= lo);
                if (!sees) continue;
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
    float *factor = sm_o;                          // [live][ROWS]; the parts' shares of a row
    for (int i = threadIdx.x; i < live * live_rows; i += kThreads) {
        const int s = i / live_rows, r = i - s * live_rows;
        const f32x4_t ml = take_over(meet, base + s * kStep + (unsigned)(ROWS * D + r * 4) * 4);
        factor[s * ROWS + r] = ml[0];
        factor[(live + s) * ROWS + r] = ml[1];
    }
    __syncthreads();
    for (int r = threadIdx.x; r < live_rows; r += kThreads) {
        float m = -INFINITY, l = 0.f;
        for (int s = 0; s < live; s++) m = fmaxf(m, factor[s * ROWS + r]);
        for (int s = 0; s < live; s++) {
            const float ms = factor[s * ROWS + r], f = ms == -INFINITY ? 0.f : exp2_fast(ms - m);
            factor[s * ROWS + r] = f;
            l += factor[(live + s) * ROWS + r] * f;
        }
        sm_m[r] = m;
        sm_l[r] = l;
    }
    __syncthreads();
    for (int idx = threadIdx.x; idx < live_rows * (D / 4); idx += kThreads) {
        const int r = idx / (D / 4), d = (idx - r * (D / 4)) * 4;
        f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
        for (int s0 = 0; s0 < live; s0 += 8) {       // eight loads on their way at a time
            f32x4_t part[8];
#pragma unroll
            for (int i = 0; i < 8; i++) part[i] = take_over(meet, base + min(s0 + i, live - 1) * kStep + (unsigned)(r * D + d) * 4);
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (s0 + i < live) acc += part[i] * factor[(s0 + i) * ROWS + r];
        }
        finish(r, d, acc, sm_m[r], sm_l[r]);
    }
}

constexpr int kMostSplits = 64;

// Parts of the slots: as many as fill the device, and a round of the waves each at least.
void plan_splits(long groups, int slots_of_device, int round, int max_context, size_t part_bytes, size_t room, TreeSplit *sp) {
    const long span = (long)max_context + round;      // the first part starts on a block, at or below the first slot
    long want = groups > 0 ? slots_of_device / groups : 1;
    want = std::max(1l, std::min(want, (long)kMostSplits));
    want = std::min(want, (span + round - 1) / round);
    if (part_bytes * (size_t)groups > 0) want = std::min(want, (long)(room / (part_bytes * (size_t)groups)));
    want = std::max(want, 1l);
    sp->per = (int)(((span + want - 1) / want + round - 1) / round * round);
    sp->splits = (int)((span + sp->per - 1) / sp->per);
}

int compute_units() {
    static int cus = 0;
    if (cus == 0) {
        int dev = 0, n = 0;
        if (hipGetDevice(&dev) == hipSuccess) (void)hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev);
        cus = n > 0 ? n : 256;
    }
    return cus;
}

template <typename T, int D, int NT, int PSH, int EU>
int launch(const TreeArgs &a, int max_context, hipStream_t stream) {
    constexpr size_t smem = lds_bytes<T, D, NT>();
    static_assert(smem + 16 <= 160 * 1024, "more than a compute unit's LDS");
    // the parts' shares of the rows lie where the outputs of the waves were
    static_assert((size_t)2 * kMostSplits * 16 * NT <= (size_t)kWaves * 16 * NT * (D + 4), "the shares of all parts do not fit");
    const int G = a.heads / a.kv_heads, TQ = 16 * NT / G;
    TreeSplit sp;
    sp.tiles = (a.max_nodes + TQ - 1) / TQ;
    sp.negate = a.scale < 0.f;
    sp.scale = (a.scale < 0.f ? -a.scale : a.scale) * kLog2e;
    sp.counters = nullptr;
    sp.parts = nullptr;
    const long groups = (long)a.num_segs * a.kv_heads * sp.tiles;
    void *ws = nullptr;
    size_t ws_bytes = 0;
    const int round = kWaves * 16 * Operand<T>::kTiles;
    constexpr size_t part_bytes = (size_t)16 * NT * (D + 4) * sizeof(float);
    sp.splits = 1;
    sp.per = 1 << 28;
    const int context = (int)std::min({(long)max_context, (long)a.table_stride * a.page_size, 1l << 28});      // the last part takes what is left
    if (groups * (long)sizeof(int) <= (long)kWorkspaceCounterBytes && fllm_device_workspace(&ws, &ws_bytes) && ws_bytes > kWorkspaceCounterBytes) {
        plan_splits(groups, compute_units() * (int)std::min((size_t)EU, (160 * 1024) / smem), round, context, part_bytes,
                    std::min(ws_bytes - kWorkspaceCounterBytes, (size_t)0x7fffffff), &sp);
        sp.counters = (int *)ws;
        sp.parts = (float *)((unsigned char *)ws + kWorkspaceCounterBytes);
    }
    const long units = (long)a.num_segs * sp.splits * a.kv_heads, blocks = (units + 7) / 8 * 8 * sp.tiles;
    FLLM_REQUIRE(blocks <= 0x7fffffffL, "tree_attention: grid too large");
    static bool raised = false;      // more than the default 64 KiB of dynamic LDS has to be asked for once
    if (!raised) {
        const hipError_t e = hipFuncSetAttribute((const void *)tree_attention_kernel<T, D, NT, PSH, EU>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        FLLM_REQUIRE(e == hipSuccess, "tree_attention: cannot raise the LDS limit: %s", hipGetErrorString(e));
        raised = true;
    }
    hipLaunchKernelGGL((tree_attention_kernel<T, D, NT, PSH, EU>), dim3((unsigned)blocks), dim3(kThreads), smem, stream, a, sp);
    return fllm_check_launch("tree_attention");
}

template <typename T, int D>
int launch_rows(const TreeArgs &a, int max_context, hipStream_t stream) {
    const int G = a.heads / a.kv_heads;
    const long rows = (long)a.max_nodes * G;
    auto go = [&](auto nt, auto eu) {
        constexpr int NT = decltype(nt)::value, EU = decltype(eu)::value;
        if (a.page_size == 8) return launch<T, D, NT, 3, EU>(a, max_context, stream);
        if (a.page_size == 16) return launch<T, D, NT, 4, EU>(a, max_context, stream);
        if (a.page_size == 32) return launch<T, D, NT, 5, EU>(a, max_context, stream);
        return launch<T, D, NT, 6, EU>(a, max_context, stream);
    };
    using std::integral_constant;
    if (rows <= 16 && G <= 16) return go(integral_constant<int, 1>(), integral_constant<int, 2>());
    if constexpr (sizeof(T) == 4) {
        return go(integral_constant<int, 2>(), integral_constant<int, D == 128 ? 1 : 2>());
    } else {
        if (rows <= 32 && G <= 32) return go(integral_constant<int, 2>(), integral_constant<int, D == 128 ? 1 : 2>());
        return go(integral_constant<int, 4>(), integral_constant<int, D == 128 ? 1 : 2>());
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
