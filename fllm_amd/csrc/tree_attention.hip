// Attention of trees of drafted tokens over the paged cache, plain form: one workgroup per (row, head), float32 arithmetic, softmax over
// runs of 256 keys with a running maximum and sum.  Any head size, page size and element type; the matrix-core kernels of
// tree_attention_mfma.hip take the shapes they are made for.  A key that the row does not see is neither multiplied nor added, whatever
// its slot holds.
#include "common.h"
#include "draft_api.h"
#include "tree_attention.h"

int fllm_tree_attention_fast(const TreeArgs &a, int head_dim, int v_dim, int key_chunk, int dtype, int max_context,
                             hipStream_t stream);      // tree_attention_mfma.hip; 1: shape declined

namespace {

constexpr int kBlock = 256;
constexpr int kWaves = kBlock / kWave;
constexpr int kMaxDimPerThread = 2;   // values of up to 512 lanes a head

template <typename T>
__global__ void __launch_bounds__(kBlock)
tree_attention_generic_kernel(TreeArgs p, int head_dim, int v_dim, int key_chunk) {
    extern __shared__ float smem[];
    float *qs = smem;                   // head_dim
    float *sc = smem + head_dim;        // kBlock: a key's weight, -1 for one that the row does not see
    float *scratch = sc + kBlock;       // kWaves
    __shared__ int s_seg;
    const int r = blockIdx.x, h = blockIdx.y;
    if (threadIdx.x == 0) s_seg = -1;
    __syncthreads();
    for (int s = threadIdx.x; s < p.num_segs; s += kBlock)
        if (p.seg_start[s] <= r && r < p.seg_start[s + 1]) s_seg = s;       // one of them at most
    __syncthreads();
    const int seg = s_seg;
    if (seg < 0) return;
    const int row0 = max(p.seg_start[seg], 0), nodes = min(p.seg_start[seg + 1], p.rows) - row0;
    if (r - row0 >= p.max_nodes) return;
    const int kept = max(p.kept[seg], 0);
    const long slots = (long)p.table_stride * p.page_size;
    const int n = (int)min((long)kept + nodes, min(slots, (long)INT_MAX - 4096));
    const int pos = p.row_pos[r];
    const int lo = p.window > 0 ? pos - p.window + 1 : INT_MIN;      // the first position that the row sees
    const int kvh = h / (p.heads / p.kv_heads);
    const int32_t *tbl = p.tables + (size_t)seg * p.table_stride;
    const T *qrow = (const T *)p.q + (size_t)r * p.q_stride + (size_t)h * head_dim;
    for (int c = threadIdx.x; c < head_dim; c += kBlock) qs[c] = to_f32<T>(qrow[c]);
    __syncthreads();

    float m = -INFINITY, l = 0.f;
    float acc[kMaxDimPerThread] = {0.f, 0.f};
    const int begin = lo > 0 ? min(lo, kept) : 0;
    for (int c0 = begin; c0 < n; c0 += kBlock) {
        const int key = c0 + threadIdx.x;
        bool sees = key < n;
        int page = -1;
        if (sees) {
            if (key < kept) {
                sees = key >= lo;
            } else {
                const int j = key - kept;
                sees = (j >> 6) < p.words && ((p.seen[(size_t)r * p.words + (j >> 6)] >> (j & 63)) & 1) && p.row_pos[row0 + j] >= lo;
            }
            if (sees) page = tbl[key / p.page_size];
            sees = sees && (unsigned)page < (unsigned)p.num_pages;
        }
        float s = -INFINITY;
        if (sees) {
            const T *kr = (const T *)p.kp + key_offset_chunked(page, p.kv_heads, kvh, p.page_size, head_dim, key % p.page_size, 0, key_chunk);
            const size_t chunk_step = (size_t)p.page_size * key_chunk;
            float dot = 0.f;
            for (int c = 0; c < head_dim; c++) dot = fmaf(qs[c], to_f32<T>(kr[(size_t)(c / key_chunk) * chunk_step + c % key_chunk]), dot);
            s = dot * p.scale;
        }
        const float m_new = fmaxf(m, block_max<kWaves>(s, scratch));
        const float alpha = m == -INFINITY ? 0.f : expf(m - m_new);
        const float w = !sees ? -1.f : s == -INFINITY ? 0.f : expf(s - m_new);
        sc[threadIdx.x] = w;
        l = l * alpha + block_sum<kWaves>(sees ? w : 0.f, scratch);   // the barriers inside also publish sc[]
        const int count = n - c0 < kBlock ? n - c0 : kBlock;
#pragma unroll
        for (int t = 0; t < kMaxDimPerThread; t++) {
            const int c = threadIdx.x + t * kBlock;
            if (c >= v_dim) break;
            float a = acc[t] * alpha;
            for (int j = 0; j < count; j++) {
                if (sc[j] < 0.f) continue;
                const int kj = c0 + j;
                a = fmaf(sc[j], to_f32<T>(((const T *)p.vp)[(((size_t)tbl[kj / p.page_size] * p.kv_heads + kvh) * v_dim + c) * p.page_size + kj % p.page_size]), a);
            }
            acc[t] = a;
        }
        m = m_new;
        __syncthreads();   // sc[] is rewritten by the next run
    }
    float keep = 1.0f;
    if (p.sinks != nullptr) {   // one more term exp(sink) in the denominator, with no key and no value
        const float sink = p.sinks[h];
        const float m_all = fmaxf(m, sink);
        keep = m == -INFINITY ? 0.f : expf(m - m_all);
        l = l * keep + (sink == m_all ? 1.f : expf(sink - m_all));
    }
    const float inv = l == 0.f ? 0.f : keep / l;      // a NaN stays one
#pragma unroll
    for (int t = 0; t < kMaxDimPerThread; t++) {
        const int c = threadIdx.x + t * kBlock;
        if (c < v_dim) ((T *)p.out)[((size_t)r * p.heads + h) * v_dim + c] = from_f32<T>(acc[t] * inv);
    }
}

}  // namespace

extern "C" int fllm_draft_abi_version(void) { return 1; }

extern "C" int fllm_tree_attention(const void *q, int q_stride, const void *k_pages, const void *v_pages, const int32_t *tables, int table_stride,
                                   const int32_t *row_pos, const int32_t *seg_start, int num_segs, const int32_t *kept, const int64_t *seen,
                                   int words, void *out, int rows, int heads, int kv_heads, int head_dim, int v_dim, int page_size,
                                   int num_pages, float scale, int window, int key_chunk, const float *sinks, int dtype, int max_nodes,
                                   int max_context, hipStream_t stream) {
    FLLM_REQUIRE(rows >= 0 && heads > 0 && kv_heads > 0 && head_dim > 0 && v_dim > 0 && page_size > 0 && table_stride > 0 && num_pages > 0,
                 "tree_attention: bad sizes");
    FLLM_REQUIRE(num_segs >= 0 && words > 0 && window >= 0 && max_nodes >= 0 && max_context >= 0,
                 "tree_attention: bad segments, words, window or bounds");
    FLLM_REQUIRE(heads % kv_heads == 0, "tree_attention: %d heads are not a multiple of %d key/value heads", heads, kv_heads);
    FLLM_REQUIRE(key_chunk > 0 && head_dim % key_chunk == 0, "tree_attention: keys of %d lanes cannot lie in chunks of %d", head_dim, key_chunk);
    FLLM_REQUIRE(q_stride >= heads * head_dim, "tree_attention: q_stride %d is shorter than heads * head_dim", q_stride);
    FLLM_REQUIRE(dtype == FLLM_F32 || dtype == FLLM_BF16, "tree_attention: unknown dtype %d", dtype);
    FLLM_REQUIRE(v_dim <= kBlock * kMaxDimPerThread && head_dim <= 8192, "tree_attention: heads of %d and %d lanes are too wide", head_dim, v_dim);
    FLLM_REQUIRE(heads <= 65535, "tree_attention: too many heads");
    if (rows == 0 || num_segs == 0 || max_nodes == 0) return 0;
    TreeArgs a;
    a.q = q;
    a.kp = k_pages;
    a.vp = v_pages;
    a.out = out;
    a.tables = tables;
    a.row_pos = row_pos;
    a.seg_start = seg_start;
    a.kept = kept;
    a.seen = seen;
    a.sinks = sinks;
    a.q_stride = q_stride;
    a.table_stride = table_stride;
    a.num_segs = num_segs;
    a.words = words;
    a.rows = rows;
    a.heads = heads;
    a.kv_heads = kv_heads;
    a.page_size = page_size;
    a.num_pages = num_pages;
    a.window = window;
    a.max_nodes = max_nodes;
    a.scale = scale;
    const int fast = fllm_tree_attention_fast(a, head_dim, v_dim, key_chunk, dtype, max_context, stream);
    if (fast <= 0) return fast;
    const dim3 grid(rows, heads);
    const size_t smem = (size_t)(head_dim + kBlock + kWaves) * sizeof(float);
    if (dtype == FLLM_F32)
        hipLaunchKernelGGL(tree_attention_generic_kernel<float>, grid, dim3(kBlock), smem, stream, a, head_dim, v_dim, key_chunk);
    else
        hipLaunchKernelGGL(tree_attention_generic_kernel<bf16_t>, grid, dim3(kBlock), smem, stream, a, head_dim, v_dim, key_chunk);
    return fllm_check_launch("tree_attention");
}
