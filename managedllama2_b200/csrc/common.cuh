// Shared device helpers for the sm_100a decode kernels: mbarrier / bulk-copy / programmatic
// dependent launch wrappers (inline PTX), the mixed-precision FMA, and small reductions.
#pragma once

#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <cstdint>

namespace ml2 {

constexpr int kGroup = 128;           // AWQ group size along d_in (native/mat_vec_kernel.cu:96 in the reference)
constexpr uint32_t kSpinLimit = 1u << 22;  // bounded mbarrier waits: ~seconds, then flag an error and bail out

// Error word written by kernels whose bounded wait expired (host reads it; the device never traps).
struct DeviceStatus {
    unsigned int error;   // 0 = ok; otherwise a code from the kernel that gave up
    unsigned int detail;
};

// What a batched-decoding operator found wrong in device tables (second status word of the context). The
// first finding is kept; the element is left out (its row, token or page counts as absent) and the kernel goes on.
enum InputError : unsigned int {
    kInputFreeCount = 0x101,     // count of the free pages outside 0..n_pages; detail = the count
    kInputFreeOverflow = 0x102,  // more pages given back than the free stack holds; detail = pages given back
    kInputPage = 0x103,          // page number outside the cache; detail = request
    kInputSlot = 0x104,          // slot outside the cache; detail = token
    kInputLength = 0x105,        // length above max_length or negative, or query rows out of order; detail = request
    kAttentionGaveUp = 0x106,    // no fault of the input: a wait inside the prefix kernel ran out; detail = CTA
};

__host__ __device__ constexpr int ceil_div(int a, int b) { return (a + b - 1) / b; }

// ---- shared-memory addresses -------------------------------------------------------------
__device__ __forceinline__ uint32_t smem_u32(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

__device__ __forceinline__ void report_input_error(DeviceStatus* st, unsigned int code, int detail)
{
    if (atomicCAS(&st->error, 0u, code) == 0u) st->detail = (unsigned int)detail;
}

// ---- mbarrier ----------------------------------------------------------------------------
__device__ __forceinline__ void mbar_init(uint64_t* bar, uint32_t count)
{
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_fence_init() { asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory"); }
__device__ __forceinline__ void mbar_arrive(uint64_t* bar)
{
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void mbar_arrive_expect_tx(uint64_t* bar, uint32_t bytes)
{
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool mbar_try_wait(uint64_t* bar, uint32_t parity)
{
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return ok != 0;
}
// try_wait that lets the hardware suspend the thread for up to `ns` nanoseconds while the phase is pending:
// a waiting warp then costs almost no issue slots (used by the roles that are not on the critical path).
__device__ __forceinline__ bool mbar_try_wait_suspend(uint64_t* bar, uint32_t parity, uint32_t ns)
{
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity), "r"(ns)
        : "memory");
    return ok != 0;
}
// Bounded wait. Returns false when the limit ran out (caller records the error and leaves).
__device__ __forceinline__ bool mbar_wait(uint64_t* bar, uint32_t parity)
{
    for (uint32_t i = 0; i < kSpinLimit; ++i)
        if (mbar_try_wait(bar, parity)) return true;
    return false;
}

// ---- 1-D bulk async copy global -> shared (TMA engine, no tensor map, no multicast) ---------
// dst/src 16-byte aligned, bytes a multiple of 16. Completion is signalled on `bar` as transaction bytes.
__device__ __forceinline__ void bulk_g2s(void* dst_smem, const void* src_gmem, uint32_t bytes, uint64_t* bar, uint64_t policy)
{
    asm volatile(
        "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1], %2, [%3], %4;" ::"r"(
            smem_u32(dst_smem)),
        "l"(src_gmem), "r"(bytes), "r"(smem_u32(bar)), "l"(policy)
        : "memory");
}
__device__ __forceinline__ uint64_t policy_evict_first()
{
    uint64_t p;
    asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(p));
    return p;
}
__device__ __forceinline__ uint64_t policy_evict_last()
{
    uint64_t p;
    asm volatile("createpolicy.fractional.L2::evict_last.b64 %0, 1.0;" : "=l"(p));
    return p;
}

// ---- programmatic dependent launch --------------------------------------------------------
// wait: blocks until the kernel this one depends on has completed and its writes are visible.
// launch_dependents: lets the next kernel in the stream start its independent prologue.
// Both are no-ops when the launch carries no programmatic dependency.
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void pdl_launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// ---- named barrier among a subset of the CTA's warps ---------------------------------------
__device__ __forceinline__ void named_bar_sync(int id, int nthreads)
{
    asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(nthreads) : "memory");
}

// ---- mixed-precision FMA (sm_100+): d = a(f16) * b(f16) + c(f32), product exact, one rounding ----
__device__ __forceinline__ float fma_f16_f32(unsigned short a, unsigned short b, float c)
{
    float d;
    asm("fma.rn.f32.f16 %0, %1, %2, %3;" : "=f"(d) : "h"(a), "h"(b), "f"(c));
    return d;
}
__device__ __forceinline__ unsigned short lo16(uint32_t v) { return static_cast<unsigned short>(v & 0xffffu); }
__device__ __forceinline__ unsigned short hi16(uint32_t v) { return static_cast<unsigned short>(v >> 16); }

__device__ __forceinline__ float warp_sum(float v)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ float warp_max(float v)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

// streaming 16-byte load that does not allocate in L1
__device__ __forceinline__ uint4 ld_nc_v4(const void* p)
{
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

}  // namespace ml2
