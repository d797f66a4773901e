// Attention of a batch whose requests share a prefix: every query row sees the shared rows, which lie in one contiguous
// cache, and the rows of its own request, which lie in pages (ml2_prefix_attention).
//
//   o = sum_j p_j v_j,  p_j = exp(scale q.k_j - lse),  lse = log sum_j exp(scale q.k_j),  j over the prefix and own rows 0..last
//
// with last = length - queries + i for query i of a request that has `queries` rows in this call.
#include "../../include/ml2b200.h"

#include "batch_common.cuh"
#include "host_common.hpp"

#include <cmath>

namespace ml2 {

struct AttnBatch {
    void* out;
    float* lse;
    const void *q, *pk, *pv, *k, *v;
    const int *table, *lengths, *query_start;
    DeviceStatus* status;
    long long out_stride, q_stride, prefix_stride, cache_stride;
    int n_requests, n_rows, prefix, max_length, n_slots, table_stride, page_shift, n_heads, n_kv;
    float scale;
};

// One warp per (row, head): four dims per lane (head 128) or two (64), one key at a time.
template <typename T, int kHead>
__global__ void __launch_bounds__(128) prefix_attention_kernel(const AttnBatch p)
{
    constexpr int kPer = kHead / 32;
    const long long id = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    const int t = (int)(id / p.n_heads), h = (int)(id % p.n_heads), hk = h / (p.n_heads / p.n_kv);
    if (t >= p.n_rows || t >= p.query_start[p.n_requests]) return;
    int r = 0;
    while (r < p.n_requests - 1 && p.query_start[r + 1] <= t) ++r;
    const int queries = p.query_start[r + 1] - p.query_start[r];
    int length = p.lengths[r];
    if (lane == 0 && (length < 0 || length > p.max_length || p.query_start[r] < 0 || queries < 0 || queries > p.n_rows))
        report_input_error(p.status, kInputLength, r);
    length = min(length, p.max_length);
    const int seen = max(0, min(length, length - queries + (t - p.query_start[r]) + 1));
    const T* q = static_cast<const T*>(p.q) + t * p.q_stride + (long long)h * kHead + lane * kPer;
    float qf[kPer], acc[kPer] = {};
#pragma unroll
    for (int e = 0; e < kPer; ++e) qf[e] = (float)q[e] * p.scale;
    float m = -INFINITY, l = 0.f;
    for (long long j = -(long long)p.prefix; j < seen; ++j) {
        const T *k, *v;
        if (j < 0) {
            const long long at = (j + p.prefix) * p.prefix_stride + (long long)hk * kHead + lane * kPer;
            k = static_cast<const T*>(p.pk) + at;
            v = static_cast<const T*>(p.pv) + at;
        } else {
            const int page = p.table[(long long)r * p.table_stride + (j >> p.page_shift)];
            if (page < 0 || page >= (p.n_slots >> p.page_shift)) {
                if (lane == 0) report_input_error(p.status, kInputPage, r);
                continue;
            }
            const long long slot = ((long long)page << p.page_shift) + (j & ((1 << p.page_shift) - 1));
            const long long at = slot * p.cache_stride + (long long)hk * kHead + lane * kPer;
            k = static_cast<const T*>(p.k) + at;
            v = static_cast<const T*>(p.v) + at;
        }
        float s = 0.f;
#pragma unroll
        for (int e = 0; e < kPer; ++e) s += qf[e] * (float)k[e];
        s = warp_sum(s);
        const float mn = fmaxf(m, s), base = mn == -INFINITY ? 0.f : mn;
        const float c = expf(m - base), w = expf(s - base);
        l = l * c + w;
#pragma unroll
        for (int e = 0; e < kPer; ++e) acc[e] = acc[e] * c + (w == 0.f ? 0.f : w * (float)v[e]);
        m = mn;
    }
    T* o = static_cast<T*>(p.out) + t * p.out_stride + (long long)h * kHead + lane * kPer;
#pragma unroll
    for (int e = 0; e < kPer; ++e) o[e] = (T)(l == 0.f ? 0.f : acc[e] / l);
    if (p.lse && lane == 0) p.lse[(long long)t * p.n_heads + h] = l == 0.f ? -INFINITY : m + logf(l);
}

static int check_sizes(const char* what, int n_rows, int n_requests, int prefix, int max_length, int n_heads, int n_kv, int head_size)
{
    if (n_rows < 0 || n_requests < 1 || n_requests > kMaxRequests)
        return fail(ML2_E_INVALID, "%s: n_rows=%d n_requests=%d (1..%d)", what, n_rows, n_requests, kMaxRequests);
    if (prefix < 0 || max_length < 0) return fail(ML2_E_INVALID, "%s: prefix of %d rows, max_length=%d", what, prefix, max_length);
    if (n_heads < 1 || n_kv < 1 || n_heads % n_kv || n_heads > 65536)
        return fail(ML2_E_INVALID, "%s: n_heads=%d must be a multiple of n_kv_heads=%d", what, n_heads, n_kv);
    if (head_size != 64 && head_size != 128) return fail(ML2_E_INVALID, "%s: head_size=%d must be 64 or 128", what, head_size);
    return ML2_OK;
}

}  // namespace ml2

using namespace ml2;

extern "C" {

int ml2_prefix_attention_workspace(ml2_ctx* h, int n_rows, int n_requests, int prefix_length, int max_length, int n_heads, int n_kv_heads,
                                   int head_size, size_t* bytes)
{
    if (!h || !bytes) return fail(ML2_E_INVALID, "prefix_attention_workspace: null argument");
    if (int rc = check_sizes("prefix_attention_workspace", n_rows, n_requests, prefix_length, max_length, n_heads, n_kv_heads, head_size)) return rc;
    *bytes = 0;
    return ML2_OK;
}

int ml2_prefix_attention(ml2_ctx* h, int dtype, void* out, long long out_stride, float* lse, const void* query, long long query_stride,
                         int n_rows, const ml2_kv* prefix, const ml2_kv* cache, int page_size, const int* table, int table_stride,
                         const int* lengths, const int* query_start, int n_requests, int max_length, int n_heads, int n_kv_heads,
                         int head_size, float scale, void* workspace, size_t workspace_bytes)
{
    Ctx* ctx = reinterpret_cast<Ctx*>(h);
    if (!ctx || !prefix || !cache) return fail(ML2_E_INVALID, "prefix_attention: null argument");
    if (dtype != ML2_F16 && dtype != ML2_BF16) return fail(ML2_E_INVALID, "prefix_attention: dtype=%d is neither ML2_F16 nor ML2_BF16", dtype);
    if (prefix->rows < 0 || prefix->rows > INT32_MAX || cache->rows < 1 || cache->rows > INT32_MAX)
        return fail(ML2_E_INVALID, "prefix_attention: the prefix has %lld rows and the cache %lld", prefix->rows, cache->rows);
    if (int rc = check_sizes("prefix_attention", n_rows, n_requests, (int)prefix->rows, max_length, n_heads, n_kv_heads, head_size)) return rc;
    const int shift = page_shift(page_size);
    if (shift < 0) return fail(ML2_E_INVALID, "prefix_attention: page_size=%d must be a power of two, at most %d", page_size, kMaxPageSize);
    if (table_stride < 1 || (long long)table_stride * page_size > INT32_MAX)
        return fail(ML2_E_INVALID, "prefix_attention: table_stride=%d with page_size=%d", table_stride, page_size);
    if (max_length > table_stride * page_size)
        return fail(ML2_E_INVALID, "prefix_attention: max_length=%d passes the table's %d pages of %d", max_length, table_stride, page_size);
    if (!std::isfinite(scale)) return fail(ML2_E_INVALID, "prefix_attention: scale=%g", (double)scale);
    if (n_rows == 0) return ML2_OK;
    if (!out || !query || !table || !lengths || !query_start || !cache->key || !cache->value || (prefix->rows && (!prefix->key || !prefix->value)))
        return fail(ML2_E_INVALID, "prefix_attention: null argument");
    const long long q_width = (long long)n_heads * head_size, kv_width = (long long)n_kv_heads * head_size;
    if (out_stride < q_width || query_stride < q_width || cache->row_stride < kv_width || (prefix->rows && prefix->row_stride < kv_width))
        return fail(ML2_E_INVALID, "prefix_attention: a row stride is shorter than the row");
    if ((out_stride | query_stride | cache->row_stride | prefix->row_stride) % 8 || !aligned_to(16, out, query, cache->key, cache->value) ||
        !aligned_to(16, prefix->key, prefix->value, workspace))
        return fail(ML2_E_INVALID, "prefix_attention: pointers must be 16-byte aligned and row strides multiples of 8 elements");
    if (out == query) return fail(ML2_E_INVALID, "prefix_attention: out must not overlap the queries");
    if (int rc = use_device(ctx)) return rc;
    AttnBatch p{};
    p.out = out; p.lse = lse; p.q = query; p.pk = prefix->key; p.pv = prefix->value; p.k = cache->key; p.v = cache->value;
    p.table = table; p.lengths = lengths; p.query_start = query_start; p.status = input_status(ctx);
    p.out_stride = out_stride; p.q_stride = query_stride; p.prefix_stride = prefix->row_stride; p.cache_stride = cache->row_stride;
    p.n_requests = n_requests; p.n_rows = n_rows; p.prefix = (int)prefix->rows; p.max_length = max_length; p.n_slots = (int)cache->rows;
    p.table_stride = table_stride; p.page_shift = shift; p.n_heads = n_heads; p.n_kv = n_kv_heads; p.scale = scale;
    const unsigned grid = (unsigned)(((long long)n_rows * n_heads + 3) / 4);
    if (dtype == ML2_F16 && head_size == 128) prefix_attention_kernel<__half, 128><<<grid, 128, 0, ctx->stream>>>(p);
    if (dtype == ML2_F16 && head_size == 64) prefix_attention_kernel<__half, 64><<<grid, 128, 0, ctx->stream>>>(p);
    if (dtype == ML2_BF16 && head_size == 128) prefix_attention_kernel<__nv_bfloat16, 128><<<grid, 128, 0, ctx->stream>>>(p);
    if (dtype == ML2_BF16 && head_size == 64) prefix_attention_kernel<__nv_bfloat16, 64><<<grid, 128, 0, ctx->stream>>>(p);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return fail(ML2_E_CUDA, "prefix_attention: %s", cudaGetErrorString(e));
    ++ctx->launches;
    return ML2_OK;
}

}  // extern "C"
