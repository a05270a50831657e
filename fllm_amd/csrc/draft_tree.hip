// A draft's way through the cache: which drafted tokens the model chose itself, their keys and values moved up behind the kept tokens, and
// pages copied for a request that goes on in two ways.
#include "common.h"
#include "draft_api.h"

namespace {

// One wave a request.  64 nodes at a time lie one in a lane; a step of the walk compares them with the node reached and takes the lowest
// that fits.  A child has a higher number than its parent, so the walk goes through the nodes once and ends.
__global__ void __launch_bounds__(kWave)
follow_tree_kernel(const int32_t *__restrict__ drafted, const int32_t *__restrict__ parents, const int32_t *__restrict__ seg_start,
                   const int32_t *__restrict__ chosen, int rows, int32_t *__restrict__ path, int max_path, int32_t *__restrict__ length,
                   int32_t *__restrict__ newest) {
    const int s = blockIdx.x, lane = threadIdx.x;
    const int row0 = max(seg_start[s], 0), nodes = min(seg_start[s + 1], rows) - row0;
    int32_t *mine = path + (size_t)s * max_path;
    int count = 0, at = -1, pick = -1;
    if (nodes > 0) {
        count = 1;
        at = 0;
        pick = chosen[row0];
        if (lane == 0) mine[0] = 0;
        for (int n0 = 0; n0 < nodes && count < max_path; n0 += kWave) {
            const int node = n0 + lane;
            const bool here = node < nodes;
            const int parent = here ? parents[row0 + node] : -1, token = here ? drafted[row0 + node] : 0, next = here ? chosen[row0 + node] : 0;
            while (count < max_path) {
                const unsigned long long fits = __ballot(here && node > at && parent == at && token == pick);
                if (fits == 0) break;       // the node reached has no such child here; it may have one further on
                const int first = __builtin_ctzll(fits);
                at = n0 + first;
                pick = __builtin_amdgcn_readlane(next, first);
                if (lane == 0) mine[count] = at;
                count++;
            }
        }
    }
    for (int i = count + lane; i < max_path; i += kWave) mine[i] = -1;
    if (lane == 0) {
        length[s] = count;
        newest[s] = pick;
    }
}

// A thread owns a chunk of a key (key_chunk values) or a lane of the values of one key/value head in one layer and moves it for all tokens
// of the path: no other thread reads or writes what it moves, and along a rising path no source lies ahead of a target written before.
template <typename E>
__global__ void __launch_bounds__(256)
move_tokens_kernel(E *__restrict__ k_store, E *__restrict__ v_store, int num_pages, int kv_heads, int k_dim, int v_dim, int page_size,
                   int key_chunk, const int32_t *__restrict__ tables, int table_stride, const int32_t *__restrict__ kept_of,
                   const int32_t *__restrict__ path, int max_path, const int32_t *__restrict__ length) {
    const int s = blockIdx.x, kvh = blockIdx.y, layer = blockIdx.z;
    const int count = min(length[s], max_path), kept = max(kept_of[s], 0);
    const int32_t *tbl = tables + (size_t)s * table_stride, *mine = path + (size_t)s * max_path;
    const long slots = (long)table_stride * page_size;
    const size_t k_layer = (size_t)num_pages * kv_heads * k_dim * page_size, v_layer = (size_t)num_pages * kv_heads * v_dim * page_size;
    int before = -1;
    for (int i = 0; i < count; i++) {
        const int node = mine[i];
        if (node <= before) break;
        before = node;
        const long from = (long)kept + node, to = (long)kept + i;
        if (node == i || from >= slots) continue;
        const int from_page = tbl[from / page_size], to_page = tbl[to / page_size];
        if ((unsigned)from_page >= (unsigned)num_pages || (unsigned)to_page >= (unsigned)num_pages) continue;
        const int from_at = (int)(from % page_size), to_at = (int)(to % page_size);
        for (int d = threadIdx.x; d < k_dim; d += blockDim.x)
            k_store[layer * k_layer + key_offset_chunked(to_page, kv_heads, kvh, page_size, k_dim, to_at, d, key_chunk)] =
                k_store[layer * k_layer + key_offset_chunked(from_page, kv_heads, kvh, page_size, k_dim, from_at, d, key_chunk)];
        for (int d = threadIdx.x; d < v_dim; d += blockDim.x)
            v_store[layer * v_layer + (((size_t)to_page * kv_heads + kvh) * v_dim + d) * page_size + to_at] =
                v_store[layer * v_layer + (((size_t)from_page * kv_heads + kvh) * v_dim + d) * page_size + from_at];
    }
}

constexpr int kPairs = 128;        // a launch carries that many pairs of pages in its arguments
constexpr int kStores = 8;
struct CopyArgs {
    char *base[kStores];
    int64_t page_bytes[kStores], layer_bytes[kStores];
    int32_t source[kPairs], target[kPairs];
};

// blockIdx: (piece of a page, layer, pair and store)
template <typename E>
__global__ void __launch_bounds__(256)
copy_pages_kernel(CopyArgs a, int store0, int count) {
    const int store = store0 + blockIdx.z / count, pair = blockIdx.z % count;
    char *layer = a.base[store] + (size_t)blockIdx.y * a.layer_bytes[store];
    const int64_t bytes = a.page_bytes[store];
    const E *from = (const E *)(layer + a.source[pair] * bytes);
    E *to = (E *)(layer + a.target[pair] * bytes);
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < bytes / (int64_t)sizeof(E); i += (int64_t)gridDim.x * 256) to[i] = from[i];
}

}  // namespace

extern "C" int fllm_follow_tree(const int32_t *drafted, const int32_t *parents, const int32_t *seg_start, int num_segs, const int32_t *chosen,
                                int rows, int32_t *path, int max_path, int32_t *length, int32_t *newest, hipStream_t stream) {
    FLLM_REQUIRE(rows >= 0 && num_segs >= 0 && max_path > 0, "follow_tree: bad sizes");
    if (num_segs == 0) return 0;
    hipLaunchKernelGGL(follow_tree_kernel, dim3(num_segs), dim3(kWave), 0, stream, drafted, parents, seg_start, chosen, rows, path, max_path,
                       length, newest);
    return fllm_check_launch("follow_tree");
}

extern "C" int fllm_move_tokens(void *k_store, void *v_store, int layers, int num_pages, int kv_heads, int k_dim, int v_dim, int page_size,
                                int key_chunk, int elem_bytes, const int32_t *tables, int table_stride, int num_segs, const int32_t *kept,
                                const int32_t *path, int max_path, const int32_t *length, hipStream_t stream) {
    FLLM_REQUIRE(layers >= 0 && num_pages > 0 && kv_heads > 0 && k_dim > 0 && v_dim >= 0 && page_size > 0 && table_stride > 0 && num_segs >= 0 &&
                     max_path > 0, "move_tokens: bad sizes");
    FLLM_REQUIRE(key_chunk > 0 && k_dim % key_chunk == 0, "move_tokens: keys of %d lanes cannot lie in chunks of %d", k_dim, key_chunk);
    FLLM_REQUIRE(elem_bytes == 2 || elem_bytes == 4, "move_tokens: elements of %d bytes", elem_bytes);
    FLLM_REQUIRE(v_dim == 0 || v_store != nullptr, "move_tokens: values are missing");
    FLLM_REQUIRE(kv_heads <= 65535 && layers <= 65535, "move_tokens: grid too large");
    if (layers == 0 || num_segs == 0) return 0;
    const dim3 grid(num_segs, kv_heads, layers);
    if (elem_bytes == 2)
        hipLaunchKernelGGL(move_tokens_kernel<uint16_t>, grid, dim3(256), 0, stream, (uint16_t *)k_store, (uint16_t *)v_store, num_pages, kv_heads,
                           k_dim, v_dim, page_size, key_chunk, tables, table_stride, kept, path, max_path, length);
    else
        hipLaunchKernelGGL(move_tokens_kernel<uint32_t>, grid, dim3(256), 0, stream, (uint32_t *)k_store, (uint32_t *)v_store, num_pages, kv_heads,
                           k_dim, v_dim, page_size, key_chunk, tables, table_stride, kept, path, max_path, length);
    return fllm_check_launch("move_tokens");
}

extern "C" int fllm_copy_pages(void *const *stores, const int64_t *layers, const int64_t *pages, const int64_t *page_bytes, int num_stores,
                               const int32_t *source, const int32_t *target, int count, hipStream_t stream) {
    FLLM_REQUIRE(num_stores >= 0 && num_stores <= kStores && count >= 0, "copy_pages: %d stores and %d pairs", num_stores, count);
    for (int n = 0; n < num_stores; n++) {
        FLLM_REQUIRE(layers[n] >= 0 && layers[n] <= 65535 && pages[n] >= 0 && page_bytes[n] >= 0, "copy_pages: bad sizes of store %d", n);
        for (int i = 0; i < count; i++)
            FLLM_REQUIRE(source[i] >= 0 && source[i] < pages[n] && target[i] >= 0 && target[i] < pages[n] && source[i] != target[i],
                         "copy_pages: page %d to page %d of %lld", source[i], target[i], (long long)pages[n]);
    }
    for (int i0 = 0; i0 < count; i0 += kPairs) {
        CopyArgs a;
        const int some = count - i0 < kPairs ? count - i0 : kPairs;
        for (int i = 0; i < some; i++) {
            a.source[i] = source[i0 + i];
            a.target[i] = target[i0 + i];
        }
        for (int n = 0; n < num_stores; n++) {
            a.base[n] = (char *)stores[n];
            a.page_bytes[n] = page_bytes[n];
            a.layer_bytes[n] = page_bytes[n] * pages[n];
            if (layers[n] == 0 || page_bytes[n] == 0) continue;
            const bool wide = (((uintptr_t)stores[n] | (uintptr_t)page_bytes[n]) & 15) == 0;
            const int64_t pieces = (page_bytes[n] / (wide ? 16 : 1) + 256 * 4 - 1) / (256 * 4);
            const dim3 grid((unsigned)(pieces < 65535 ? pieces : 65535), (unsigned)layers[n], (unsigned)some);
            if (wide)
                hipLaunchKernelGGL(copy_pages_kernel<u32x4_t>, grid, dim3(256), 0, stream, a, n, some);
            else
                hipLaunchKernelGGL(copy_pages_kernel<char>, grid, dim3(256), 0, stream, a, n, some);
            const int rc = fllm_check_launch("copy_pages");
            if (rc != 0) return rc;
        }
    }
    return 0;
}
