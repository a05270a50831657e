// What the kernels of tree attention are given (draft_api.h says what it means).
#pragma once
#include <limits.h>
#include <stdint.h>

struct TreeArgs {
    const void *q, *kp, *vp;
    void *out;
    const int32_t *tables, *row_pos, *seg_start, *kept;
    const int64_t *seen;
    const float *sinks;
    int q_stride, table_stride, num_segs, words, rows, heads, kv_heads, page_size, num_pages, window, max_nodes;
    float scale;
};
