// What the kernels of tree attention share (draft_api.h says what the arguments mean).
#pragma once
#include <limits.h>
#include <stdint.h>
#include <algorithm>
#include "common.h"

struct TreeArgs {
    const void *q, *kp, *vp;
    void *out;
    const int32_t *tables, *row_pos, *seg_start, *kept;
    const int64_t *seen;
    const float *sinks;
    int q_stride, table_stride, num_segs, words, rows, heads, kv_heads, page_size, num_pages, window, max_nodes;
    float scale;
};

namespace {

constexpr float kLog2e = 1.4426950408889634f;

// What a launch adds to TreeArgs: how the slots are split and where the parts of a tile meet.
struct TreeSplit {
    int tiles;            // row tiles a request at most
    int splits, per;      // parts of the slots, slots a part (the last takes what is left)
    int places;           // where the kernel cuts the slots itself: places a die (per: rounds a part at least)
    int *counters;        // one per (request, key/value head, tile), zero between launches
    float *parts;         // [request, key/value head, tile][split][16 NT rows of D outputs, then of a maximum and a sum]
    float scale;          // >= 0: the sign has gone into the queries
    int negate;
    int sorted;           // requests in the order of their lengths (at most a wave's lanes of them, whole)
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

// The reference point of a row that has seen nothing: below every score, and still finite, in the exponent's units (of scales above 1) too.
constexpr float kNothing = -3e38f;
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// the `count` lowest bits
__device__ __forceinline__ unsigned long long low_bits(int count) {
    return count <= 0 ? 0ull : count >= 64 ? ~0ull : (1ull << count) - 1;
}

// Whether a row sees a slot, asked slot by slot.
template <int PSH>
__device__ __forceinline__ bool sees_slot(const TreeArgs &p, int seg, int row0, int kept, int row, int lo, int slot) {
    const int j = slot - kept, page = p.tables[(size_t)seg * p.table_stride + (slot >> PSH)];
    if ((unsigned)page >= (unsigned)p.num_pages) return false;
    if (j < 0) return slot >= lo;
    return (j >> 6) < p.words && (p.seen[(size_t)row * p.words + (j >> 6)] >> (j & 63) & 1) && p.row_pos[row0 + j] >= lo;
}

constexpr int kMostSplits = 32;

inline int compute_units() {
    static int cus = 0;
    if (cus == 0) {
        int dev = 0, n = 0;
        if (hipGetDevice(&dev) == hipSuccess) (void)hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev);
        cus = n > 0 ? n : 256;
    }
    return cus;
}

// The slots that a request's rows can see, at most.
inline long reach_of(const TreeArgs &a, int max_context) {
    long reach = std::min((long)max_context, (long)a.table_stride * a.page_size);
    if (a.window > 0) reach = std::min(reach, (long)a.window + a.max_nodes);
    return reach;
}

// How the slots of every tile are split, where the device workspace has room for what the parts leave: as many parts as give every one of
// `slots` workgroups one, of whole rounds (`round` slots, what a workgroup takes at a time); contexts of `whole` rounds at most stay whole.
inline void plan_tree(const TreeArgs &a, int tiles, int slots, int round, int whole, int max_context, size_t part_bytes, TreeSplit *sp) {
    sp->negate = a.scale < 0.f;
    sp->scale = (a.scale < 0.f ? -a.scale : a.scale) * kLog2e;
    sp->counters = nullptr;
    sp->parts = nullptr;
    sp->splits = 1;
    sp->per = 1 << 28;
    const long groups = (long)a.num_segs * a.kv_heads * tiles;
    if (groups <= 0 || groups * (long)sizeof(int) > (long)kWorkspaceCounterBytes) return;
    void *ws = nullptr;
    size_t ws_bytes = 0;
    if (!fllm_device_workspace(&ws, &ws_bytes) || ws_bytes <= kWorkspaceCounterBytes) return;
    const long span = std::min(reach_of(a, max_context), 1l << 28) + round;      // the first part starts on a round's edge; the last takes what is left
    const long rounds = (span + round - 1) / round;
    if (rounds - 1 <= whole) return;
    long want = std::min({slots / groups, (long)kMostSplits, rounds});
    want = std::min(want, (long)(std::min(ws_bytes - kWorkspaceCounterBytes, (size_t)0x7fffffff) / (part_bytes * (size_t)groups)));
    want = std::max(want, 1l);
    sp->per = (int)((rounds + want - 1) / want * round);
    sp->splits = (int)((span + sp->per - 1) / sp->per);
    sp->counters = (int *)ws;
    sp->parts = (float *)((unsigned char *)ws + kWorkspaceCounterBytes);
}

}  // namespace
