// RMS norm of every query and key head, rotation by position and the write of keys and values into cache rows, in one
// pass over a batch of tokens (ml2_qk_norm_rope).
//
//   y = x * w / sqrt(mean(x^2) + eps)                       per head, when weights are given
//   (y[i], y[i + h]) -> (y[i] c - y[i + h] s, y[i] s + y[i + h] c),  h = rotary / 2, i < h, angle = pos * theta^(-2 i / rotary)
//
// Every element is read once and written once. With many tokens instruction issue is as near as HBM (4032 tokens of 64 / 8 heads
// of 128: 165 MB in 37 us, 4.5 TB/s, 72 % of the issue slots); with few it is the latency of one launch (one token 2.7 us).
// The angle is reduced in 64 bits (turns = pos * freq / 2 pi, minus the nearest whole number): in 32 bits a position of
// 100000 alone leaves an error of 0.004 in the angle. All else is 32-bit arithmetic with one rounding at the store.
#include "../../include/ml2b200.h"

#include "batch_common.cuh"
#include "host_common.hpp"

#include <cmath>

namespace ml2 {

constexpr int kRopeThreads = 320;  // of a block at most
constexpr int kRopeMaxHead = 256;

struct RopeParams {
    void* q_out;
    void* k_cache;
    void* v_cache;
    const void *q, *k, *v, *qw, *kw;
    const int *positions, *slots;
    DeviceStatus* status;
    long long q_out_stride, cache_stride, q_stride, k_stride, v_stride, n_slots;
    int n_heads, n_kv, head, rotary, lanes, lanes_log2;  // lanes: threads of one head, a power of two
    float eps, per_head;                     // per_head: 1 / head
    double turns[kRopeMaxHead / 2];          // theta^(-2 i / rotary) / (2 pi)
};

// A head of `head` elements is head / 16 lanes, 16 elements each: two 16-byte vectors that hold the two halves of eight
// rotated pairs (lanes below rotary / 16), or two neighbouring vectors of the part that is not rotated. A block takes one
// token, all of it in one pass where the heads fit its threads; the first vectors are asked for before the angles are
// computed, which hides most of either behind the other.
template <typename T>
__global__ void __launch_bounds__(kRopeThreads, 4) qk_norm_rope_kernel(const __grid_constant__ RopeParams p)
{
    __shared__ float2 s_unit[kRopeMaxHead / 2];
    const long long t = blockIdx.x;
    const int lane = threadIdx.x & (p.lanes - 1), per_block = blockDim.x >> p.lanes_log2, units = p.head >> 4, turned = p.rotary >> 4, half = p.rotary >> 1;
    const int at0 = lane < turned ? 8 * lane : 16 * lane, at1 = lane < turned ? 8 * lane + half : 16 * lane + 8;
    const int heads = p.n_heads + 2 * p.n_kv;
    auto source = [&](int h) {
        if (h < p.n_heads) return static_cast<const T*>(p.q) + t * p.q_stride + (long long)h * p.head;
        h -= p.n_heads;
        if (h < p.n_kv) return static_cast<const T*>(p.k) + t * p.k_stride + (long long)h * p.head;
        return static_cast<const T*>(p.v) + t * p.v_stride + (long long)(h - p.n_kv) * p.head;
    };
    pdl_wait();
    int h = blockIdx.y * per_block + (threadIdx.x >> p.lanes_log2);
    uint4 x0 = make_uint4(0, 0, 0, 0), x1 = x0;
    if (lane < units && h < heads) {
        const T* in = source(h);
        x0 = *reinterpret_cast<const uint4*>(in + at0);
        x1 = *reinterpret_cast<const uint4*>(in + at1);
    }
    const int slot = p.slots[t];
    if (slot < 0) return;  // padding
    if (slot >= p.n_slots) {
        if (threadIdx.x == 0) report_input_error(p.status, kInputSlot, (int)t);
        return;
    }
    const double pos = (double)p.positions[t];
    for (int i = threadIdx.x; i < half; i += blockDim.x) {
        const double a = pos * p.turns[i];
        const float r = 2.f * (float)(a - rint(a));
        s_unit[(i & 7) * turned + (i >> 3)] = make_float2(cospif(r), sinpif(r));  // neighbouring lanes read neighbouring entries
    }
    __syncthreads();

    for (int base = blockIdx.y * per_block; base < heads; base += gridDim.y * per_block) {
        const bool here = lane < units && h < heads;
        const int next = h + gridDim.y * per_block;
        T* out;
        const T* w;
        if (h < p.n_heads) {
            out = static_cast<T*>(p.q_out) + t * p.q_out_stride + (long long)h * p.head;
            w = static_cast<const T*>(p.qw);
        } else if (h < p.n_heads + p.n_kv) {
            out = static_cast<T*>(p.k_cache) + (long long)slot * p.cache_stride + (long long)(h - p.n_heads) * p.head;
            w = static_cast<const T*>(p.kw);
        } else {
            out = static_cast<T*>(p.v_cache) + (long long)slot * p.cache_stride + (long long)(h - p.n_heads - p.n_kv) * p.head;
            w = nullptr;
        }
        float a[8], b[8];
        unpack8<T>(x0, a);
        unpack8<T>(x1, b);
        if (p.qw) {
            float ss = 0.f, st = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                ss = fmaf(a[e], a[e], ss);
                st = fmaf(b[e], b[e], st);
            }
            ss += st;
            for (int o = p.lanes >> 1; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            if (here && w) {
                const float inv = rsqrtf(ss * p.per_head + p.eps);
                float wa[8], wb[8];
                unpack8<T>(*reinterpret_cast<const uint4*>(w + at0), wa);
                unpack8<T>(*reinterpret_cast<const uint4*>(w + at1), wb);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    a[e] = a[e] * inv * wa[e];
                    b[e] = b[e] * inv * wb[e];
                }
            }
        }
        uint4 y0 = x0, y1 = x1;
        if (h < p.n_heads + p.n_kv) {
            if (lane < turned) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float2 u = s_unit[e * turned + lane];
                    const float r0 = a[e] * u.x - b[e] * u.y, r1 = a[e] * u.y + b[e] * u.x;
                    a[e] = r0;
                    b[e] = r1;
                }
            }
            y0 = pack8<T>(a);
            y1 = pack8<T>(b);
        }
        if (lane < units && next < heads) {
            const T* in = source(next);
            x0 = *reinterpret_cast<const uint4*>(in + at0);
            x1 = *reinterpret_cast<const uint4*>(in + at1);
        }
        if (here) {
            *reinterpret_cast<uint4*>(out + at0) = y0;
            *reinterpret_cast<uint4*>(out + at1) = y1;
        }
        h = next;
    }
}

}  // namespace ml2

using namespace ml2;

extern "C" int ml2_qk_norm_rope(ml2_ctx* h, const ml2_qk_norm_rope_args* args)
{
    Ctx* ctx = reinterpret_cast<Ctx*>(h);
    if (!ctx || !args) return fail(ML2_E_INVALID, "qk_norm_rope: null argument");
    const auto [query_out, key_cache, value_cache, query, key, value, query_weight, key_weight, positions, slots, query_out_stride, cache_stride,
                cache_rows, query_stride, key_stride, value_stride, dtype, n_tokens, n_heads, n_kv_heads, head_size, rotary_size, theta, eps] = *args;
    if (dtype != ML2_F16 && dtype != ML2_BF16) return fail(ML2_E_INVALID, "qk_norm_rope: dtype=%d is neither ML2_F16 nor ML2_BF16", dtype);
    if (n_tokens < 0) return fail(ML2_E_INVALID, "qk_norm_rope: n_tokens=%d", n_tokens);
    if (n_heads < 1 || n_kv_heads < 1 || n_heads % n_kv_heads || n_heads > 65536)
        return fail(ML2_E_INVALID, "qk_norm_rope: n_heads=%d must be a multiple of n_kv_heads=%d", n_heads, n_kv_heads);
    if (head_size < 16 || head_size > kRopeMaxHead || head_size % 16 || rotary_size < 0 || rotary_size > head_size || rotary_size % 16)
        return fail(ML2_E_INVALID, "qk_norm_rope: head_size=%d (16..%d) and rotary_size=%d (0..head_size) must be multiples of 16", head_size,
                    kRopeMaxHead, rotary_size);
    if (!(theta > 0.f) || !std::isfinite(theta) || !(eps >= 0.f)) return fail(ML2_E_INVALID, "qk_norm_rope: theta=%g eps=%g", (double)theta, (double)eps);
    if (!query_weight != !key_weight) return fail(ML2_E_INVALID, "qk_norm_rope: query and key weights come together or not at all");
    if (n_tokens == 0) return ML2_OK;
    if (!query_out || !query || !key || !value || !positions || !slots || !key_cache || !value_cache)
        return fail(ML2_E_INVALID, "qk_norm_rope: null argument");
    const long long q_width = (long long)n_heads * head_size, kv_width = (long long)n_kv_heads * head_size;
    if (query_out_stride < q_width || query_stride < q_width || key_stride < kv_width || value_stride < kv_width || cache_stride < kv_width)
        return fail(ML2_E_INVALID, "qk_norm_rope: a row stride is shorter than the row");
    if (query_out == query && query_out_stride != query_stride && n_tokens > 1)
        return fail(ML2_E_INVALID, "qk_norm_rope: queries over themselves need one row stride, not %lld and %lld", query_stride, query_out_stride);
    if (cache_rows < 1 || cache_rows > INT32_MAX) return fail(ML2_E_INVALID, "qk_norm_rope: the cache has %lld rows", cache_rows);
    if ((query_out_stride | query_stride | key_stride | value_stride | cache_stride) % 8 || !aligned_to(16, query_out, query, key, value) ||
        !aligned_to(16, key_cache, value_cache) || !aligned_to(16, query_weight, key_weight) || !aligned_to(4, positions, slots))
        return fail(ML2_E_INVALID, "qk_norm_rope: pointers must be 16-byte aligned (int arrays 4) and row strides multiples of 8 elements");
    if (int rc = use_callers_stream(ctx)) return rc;

    RopeParams p{};
    p.q_out = query_out; p.k_cache = key_cache; p.v_cache = value_cache;
    p.q = query; p.k = key; p.v = value; p.qw = query_weight; p.kw = key_weight;
    p.positions = positions; p.slots = slots; p.status = input_status(ctx);
    p.q_out_stride = query_out_stride; p.cache_stride = cache_stride;
    p.q_stride = query_stride; p.k_stride = key_stride; p.v_stride = value_stride; p.n_slots = cache_rows;
    p.n_heads = n_heads; p.n_kv = n_kv_heads; p.head = head_size; p.rotary = rotary_size; p.eps = eps; p.per_head = 1.0f / (float)head_size;
    p.lanes = 1;
    while (p.lanes * 16 < head_size) {
        p.lanes *= 2;
        ++p.lanes_log2;
    }
    if (rotary_size) {
        // one pow, then products: i of them leave a relative error of i 2^-53, far below what the angle needs
        const double ratio = std::pow((double)theta, -2.0 / rotary_size);
        double f = 0.15915494309189533577;  // 1 / (2 pi)
        for (int i = 0; i < rotary_size / 2; ++i, f *= ratio) p.turns[i] = f;
    }
    // Up to kRopeThreads threads a token; while the tokens do not fill the SMs, their heads are cut over blocks of 256 threads (40
    // heads of 128: 1 token 2.8 us instead of 4.1, 128 tokens 4.1 instead of 4.6, 256 tokens 5.7 against 5.4).
    const int lanes = (n_heads + 2 * n_kv_heads) * p.lanes;
    const bool few = n_tokens <= ctx->sm_count;
    const int threads = std::min(few ? 256 : kRopeThreads, ceil_div(lanes, 32) * 32);
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)n_tokens, few ? (unsigned)std::min(ceil_div(lanes, threads), std::max(1, 2 * ctx->sm_count / n_tokens)) : 1u);
    cfg.blockDim = dim3(threads);
    cfg.stream = ctx->stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = ctx->pdl ? 1 : 0;
    const cudaError_t e = dtype == ML2_F16 ? cudaLaunchKernelEx(&cfg, qk_norm_rope_kernel<__half>, p)
                                           : cudaLaunchKernelEx(&cfg, qk_norm_rope_kernel<__nv_bfloat16>, p);
    if (e != cudaSuccess) return fail(ML2_E_CUDA, "qk_norm_rope: %s", cudaGetErrorString(e));
    ++ctx->launches;
    return ML2_OK;
}
