// C ABI of the entry points that work on trees of drafted tokens; the conventions are those of api.h (launches on `stream`, 0 or a
// negative value and a message, no device memory allocated, element types 0 = float32 and 1 = bfloat16).
//
// A request has `kept` tokens in its pages.  A draft adds candidate continuations: the rows seg_start[s] .. seg_start[s + 1] - 1 of
// request s are its nodes 0, 1, ..; node i lies in the slot kept[s] + i of the request's cache, node 0 is the request's newest token,
// every other node's parent has a lower number.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

// goes up with these declarations
int fllm_draft_abi_version(void);

// Softmax attention of the nodes over pages.  Row r of request s (tables [num_segs, table_stride], kept [num_segs]) sees
//   the slots t < kept[s], and of the nodes those whose bit is set in seen[r, words] (bit j % 64 of word j / 64: node j),
//   with window > 0 only those at positions > row_pos[r] - window (a slot t < kept[s] is at position t, a node at its row_pos),
// and none in a page outside [0, num_pages).  sinks (float32 [heads] or null): the denominator also holds exp(sinks[head]).
// A row that sees nothing gives zeros; rows outside seg_start[0] .. seg_start[num_segs] are left as they were.  max_nodes and
// max_context: no request has more nodes, and no more kept tokens and nodes together (rows of nodes beyond are left as they were).
// keys [page][kv_head][head_dim / key_chunk][token][key_chunk], values [page][kv_head][v_dim][token]
int fllm_tree_attention(const void *q, int q_stride, const void *k_pages, const void *v_pages, const int32_t *tables, int table_stride,
                        const int32_t *row_pos, const int32_t *seg_start, int num_segs, const int32_t *kept, const int64_t *seen, int words,
                        void *out, int rows, int heads, int kv_heads, int head_dim, int v_dim, int page_size, int num_pages, float scale,
                        int window, int key_chunk, const float *sinks, int dtype, int max_nodes, int max_context, hipStream_t stream);

// The nodes that the model chose itself: path[s] = 0, then as long as there is one the lowest child c of the node reached (c beyond it,
// parents[c] == it) with drafted[c] == chosen[it]; at most max_path nodes, -1 behind them.  length[s]: their number; newest[s]: chosen of
// the last one.  A request without nodes: length 0, newest -1.
int fllm_follow_tree(const int32_t *drafted, const int32_t *parents, const int32_t *seg_start, int num_segs, const int32_t *chosen, int rows,
                     int32_t *path, int max_path, int32_t *length, int32_t *newest, hipStream_t stream);

// Slot kept[s] + path[s, i] of request s is copied to slot kept[s] + i, i < length[s], keys and values, in every layer.  path[s] rises: it
// ends ahead of an entry that does not (or is negative), and then nothing is overwritten before it is read.  A slot without a page is left out.
// k_store [layers][num_pages][kv_heads][k_dim / key_chunk][page_size][key_chunk], v_store [layers][num_pages][kv_heads][v_dim][page_size]
// (v_dim 0: none), elements of elem_bytes (2 or 4)
int fllm_move_tokens(void *k_store, void *v_store, int layers, int num_pages, int kv_heads, int k_dim, int v_dim, int page_size, int key_chunk,
                     int elem_bytes, const int32_t *tables, int table_stride, int num_segs, const int32_t *kept, const int32_t *path,
                     int max_path, const int32_t *length, hipStream_t stream);

// Page source[i] is copied to page target[i] (host arrays) in every layer of every store: stores[n] is [layers[n]][pages[n]] pages of
// page_bytes[n] bytes.  The targets differ from each other and from every source.
int fllm_copy_pages(void *const *stores, const int64_t *layers, const int64_t *pages, const int64_t *page_bytes, int num_stores,
                    const int32_t *source, const int32_t *target, int count, hipStream_t stream);

// fllm_rope_kv_store of api.h with the slot of every row given beside its position: rotated by row_pos, stored at row_slot.
int fllm_rope_kv_store_at(void *qkv, const int32_t *row_pos, const int32_t *row_slot, const int32_t *row_seg, const int32_t *tables,
                          int table_stride, const float *cos_table, const float *sin_table, void *k_pages, void *v_pages, int num_pages,
                          int rows, int heads, int kv_heads, int head_dim, int v_dim, int rope_dims, int pairing, int page_size,
                          int key_chunk, int dtype, int store_kv, hipStream_t stream);

#ifdef __cplusplus
}
#endif
