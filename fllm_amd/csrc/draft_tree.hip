// A draft's way through the cache: which drafted tokens the model chose itself, their keys and values moved up behind the kept tokens, and
// pages copied for a request that goes on in two ways.
#include "common.h"
#include "draft_api.h"

namespace {

// One wave a request.  64 nodes at a time lie one in a lane; a step of the walk compares them with the node reached and takes the lowest
// that fits.  A child has a higher number than its parent, so the walk goes through the nodes once and ends.  Bound by the launch and
// two trips to memory: 1.4 us for a request of 16 nodes, 3.1 us for 256 of up to 64.
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

// Moving.  A workgroup takes one key/value head of one request in a few layers: it lists the path's moves (64 entries of the path at a time),
// then moves eight tokens at a time, all reads ahead of all writes.  Along a rising path that is enough: what a move overwrites (slot i of
// the new order) can only be the source of a move of a lower number, never of one in a later eight.
constexpr int kMoves = 8;
struct MoveArgs {
    char *k, *v;
    const int32_t *tables, *kept, *path, *length;
    int num_pages, kv_heads, k_dim, v_dim, page_size, key_chunk, table_stride, max_path, layers, layers_each;
};

// E: an element.  U: what a key is moved in (16 bytes where its chunks are whole ones of those, else an element).
// Bound by the lines it touches: values lie transposed, a token's are 2 bytes of every row of a page, and the lines around them come along.
// Eight lanes take the eight tokens of a row of values, so that what goes to neighbouring slots goes out together.  48 requests, up to 9 of 64
// nodes kept, 16 layers of 8 heads of 64: 25 MB of keys and values in about 110 MB of lines, 18 us from the last cache, 29 us from memory; one
// request, 5 kept, 32 layers of 8 heads of 128: 4.5 us.
template <typename E, typename U>
__global__ void __launch_bounds__(256)
move_tokens_kernel(MoveArgs a) {
    __shared__ int s_from[kWave], s_to[kWave], s_from_page[kWave], s_to_page[kWave], s_moves, s_more;
    const int s = blockIdx.x, kvh = blockIdx.y, layer0 = blockIdx.z * a.layers_each, layer1 = min(layer0 + a.layers_each, a.layers);
    const int ps = a.page_size, chunk_bytes = a.key_chunk * (int)sizeof(E);
    const int k_units = a.k_dim * (int)sizeof(E) / (int)sizeof(U);            // of a token's key
    const size_t k_head = (size_t)a.k_dim * ps * sizeof(E), v_head = (size_t)a.v_dim * ps * sizeof(E);
    const size_t k_page = k_head * a.kv_heads, v_page = v_head * a.kv_heads;
    for (int i0 = 0; i0 < a.max_path; i0 += kWave) {
        if (threadIdx.x < kWave) {
            const int lane = threadIdx.x, i = i0 + lane;
            const int count = min(a.length[s], a.max_path), kept = max(a.kept[s], 0);
            const int32_t *mine = a.path + (size_t)s * a.max_path;
            const int node = i < count ? mine[i] : -1, before = i == 0 ? -1 : i < count ? mine[i - 1] : -1;
            const unsigned long long ends = __ballot(i >= count || node <= before);
            const int rising = ends ? __builtin_ctzll(ends) : kWave;          // entries of these 64 that the path has
            const long from = (long)kept + node, to = (long)kept + i, slots = (long)a.table_stride * ps;
            bool moves = lane < rising && node != i && from < slots;
            int from_page = 0, to_page = 0;
            if (moves) {
                const int32_t *tbl = a.tables + (size_t)s * a.table_stride;
                from_page = tbl[from / ps];
                to_page = tbl[to / ps];
                moves = (unsigned)from_page < (unsigned)a.num_pages && (unsigned)to_page < (unsigned)a.num_pages;
            }
            const unsigned long long all = __ballot(moves);
            if (moves) {
                const int n = __builtin_popcountll(all & ((1ull << lane) - 1));
                s_from[n] = (int)(from % ps);
                s_to[n] = (int)(to % ps);
                s_from_page[n] = from_page;
                s_to_page[n] = to_page;
            }
            if (lane == 0) {
                s_moves = __builtin_popcountll(all);
                s_more = rising == kWave;
            }
        }
        __syncthreads();
        const int moves = s_moves;
        const bool more = s_more != 0;
        for (int m0 = 0; m0 < moves; m0 += kMoves) {
            const int some = min(kMoves, moves - m0);
            for (int layer = layer0; layer < layer1; layer++) {
                char *k = a.k + (size_t)layer * a.num_pages * k_page + (size_t)kvh * k_head;
                char *v = a.v + (size_t)layer * a.num_pages * v_page + (size_t)kvh * v_head;
                // 128 pieces of keys and 128 lanes of values at a time, four of each a thread; wider heads take several rounds,
                // each with every token of its own lanes
                for (int u0 = 0; u0 < max(k_units, a.v_dim); u0 += 128) {
                    U kr[4];
                    E vr[4];
#pragma unroll
                    for (int n = 0; n < 4; n++) {
                        const int it = threadIdx.x + 256 * n, m = it % kMoves, u = u0 + it / kMoves;
                        if (m >= some) continue;
                        if (u < k_units) {
                            const int at = u * (int)sizeof(U);
                            kr[n] = *(const U *)(k + s_from_page[m0 + m] * k_page + ((size_t)(at / chunk_bytes) * ps + s_from[m0 + m]) * chunk_bytes + at % chunk_bytes);
                        }
                        if (u < a.v_dim) vr[n] = *(const E *)(v + s_from_page[m0 + m] * v_page + ((size_t)u * ps + s_from[m0 + m]) * sizeof(E));
                    }
                    __syncthreads();
#pragma unroll
                    for (int n = 0; n < 4; n++) {
                        const int it = threadIdx.x + 256 * n, m = it % kMoves, u = u0 + it / kMoves;
                        if (m >= some) continue;
                        if (u < k_units) {
                            const int at = u * (int)sizeof(U);
                            *(U *)(k + s_to_page[m0 + m] * k_page + ((size_t)(at / chunk_bytes) * ps + s_to[m0 + m]) * chunk_bytes + at % chunk_bytes) = kr[n];
                        }
                        if (u < a.v_dim) *(E *)(v + s_to_page[m0 + m] * v_page + ((size_t)u * ps + s_to[m0 + m]) * sizeof(E)) = vr[n];
                    }
                }
            }
        }
        if (!more) return;
        __syncthreads();      // the list has been read
    }
}

// A launch carries the pairs of pages in its arguments, which take 4 KiB at most with the 256 bytes that the compiler adds to them: as many as
// that has room for, in steps of 64.  A launch costs the host about 4 us.
constexpr int kPairs = 448;
constexpr int kStores = 8;
struct CopyArgs {
    char *base[kStores];
    int64_t page_bytes[kStores], layer_bytes[kStores];
    int32_t layers[kStores];
    int32_t source[kPairs], target[kPairs];
};
static_assert(sizeof(CopyArgs) + 8 + 256 <= 4096 && sizeof(CopyArgs) + 8 + 256 + 64 * 8 > 4096, "the arguments of a launch");

// blockIdx: (piece of a page, pair, layer and store).  A thread has four 16-byte pieces on their way.  Bound by memory: 400 pages of 16 layers
// (419 MB in and out) 84 us, 5.0 TB/s, where one copy of 4 GiB gets 5.4; a page of 32 layers to seven others 6.9 us, the first read by one of
// the seven and the others' from L2.
template <typename E>
__global__ void __launch_bounds__(256)
copy_pages_kernel(CopyArgs a, int most_layers) {
    const int store = blockIdx.z / most_layers, layer = blockIdx.z - store * most_layers;
    if (layer >= a.layers[store]) return;
    const int64_t bytes = a.page_bytes[store], count = bytes / (int64_t)sizeof(E);
    char *at = a.base[store] + (size_t)layer * a.layer_bytes[store];
    const E *from = (const E *)(at + a.source[blockIdx.y] * bytes);
    E *to = (E *)(at + a.target[blockIdx.y] * bytes);
    for (int64_t i = (int64_t)blockIdx.x * 1024 + threadIdx.x; i < count; i += (int64_t)gridDim.x * 1024) {
        E piece[4];
#pragma unroll
        for (int n = 0; n < 4; n++)
            if (i + 256 * n < count) piece[n] = from[i + 256 * n];
#pragma unroll
        for (int n = 0; n < 4; n++)
            if (i + 256 * n < count) to[i + 256 * n] = piece[n];
    }
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
    MoveArgs a = {(char *)k_store, (char *)v_store, tables, kept, path, length, num_pages, kv_heads, k_dim, v_dim, page_size, key_chunk, table_stride,
                  max_path, layers, 1};
    // a workgroup takes so many layers that 2,048 of them are on the device at a time: what it looks up serves all of them.  Microseconds with
    // 1,024 / 2,048 / 4,096 / a layer each: the 48 requests above 18.7 / 18.1 / 18.3 / 19.8, with up to 3 nodes kept 14.7 / 13.0 / 13.9 / 15.9.
    const long groups = (long)num_segs * kv_heads * layers;
    a.layers_each = (int)(groups > 2048 ? (groups + 2047) / 2048 : 1);
    if (a.layers_each > layers) a.layers_each = layers;
    const dim3 grid(num_segs, kv_heads, (layers + a.layers_each - 1) / a.layers_each);
    const bool wide = key_chunk * elem_bytes % 16 == 0 && ((uintptr_t)k_store & 15) == 0;
    if (elem_bytes == 2 && wide) hipLaunchKernelGGL((move_tokens_kernel<uint16_t, u32x4_t>), grid, dim3(256), 0, stream, a);
    else if (elem_bytes == 2) hipLaunchKernelGGL((move_tokens_kernel<uint16_t, uint16_t>), grid, dim3(256), 0, stream, a);
    else if (wide) hipLaunchKernelGGL((move_tokens_kernel<uint32_t, u32x4_t>), grid, dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((move_tokens_kernel<uint32_t, uint32_t>), grid, dim3(256), 0, stream, a);
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
    CopyArgs a;
    int64_t most = 0, most_layers = 0;
    bool wide = true;
    for (int n = 0; n < num_stores; n++) {
        a.base[n] = (char *)stores[n];
        a.page_bytes[n] = page_bytes[n];
        a.layer_bytes[n] = page_bytes[n] * pages[n];
        a.layers[n] = page_bytes[n] > 0 ? (int32_t)layers[n] : 0;
        if (a.layers[n] == 0) continue;
        most = page_bytes[n] > most ? page_bytes[n] : most;
        most_layers = layers[n] > most_layers ? layers[n] : most_layers;
        wide = wide && (((uintptr_t)stores[n] | (uintptr_t)page_bytes[n]) & 15) == 0;
    }
    FLLM_REQUIRE(most_layers * num_stores <= 65535, "copy_pages: %lld layers of %d stores", (long long)most_layers, num_stores);
    if (most == 0) return 0;
    const int64_t pieces = (most / (wide ? 16 : 1) + 1023) / 1024;
    for (int i0 = 0; i0 < count; i0 += kPairs) {
        const int some = count - i0 < kPairs ? count - i0 : kPairs;
        for (int i = 0; i < some; i++) {
            a.source[i] = source[i0 + i];
            a.target[i] = target[i0 + i];
        }
        const dim3 grid((unsigned)(pieces < 0x7fffff ? pieces : 0x7fffff), (unsigned)some, (unsigned)(most_layers * num_stores));
        if (wide) hipLaunchKernelGGL(copy_pages_kernel<u32x4_t>, grid, dim3(256), 0, stream, a, (int)most_layers);
        else hipLaunchKernelGGL(copy_pages_kernel<char>, grid, dim3(256), 0, stream, a, (int)most_layers);
        const int rc = fllm_check_launch("copy_pages");
        if (rc != 0) return rc;
    }
    return 0;
}
