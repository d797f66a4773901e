// Host-side types shared by the C-ABI translation units.
#pragma once

#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "common.cuh"

namespace ml2 {

struct Ctx {
    int device = 0;
    int sm_count = 0;
    cudaStream_t stream = nullptr;         // of the next launch: the caller's, or a model's own once that has run
    cudaStream_t caller_stream = nullptr;  // what ml2_ctx_set_stream was given last
    bool callers_calls = false;            // a batched-decoding call has come back to it since a model ran
    bool pdl = false;
    DeviceStatus* status_dev = nullptr;   // [0] waits of a model that ran out, [1] what a batched-decoding operator met
    void* scratch = nullptr;          // host-buffer entry points stage their vectors here
    size_t scratch_bytes = 0;
    long long launches = 0;
    bool attention_ready[2][2] = {};  // prefix_attention.cu: kernels of either type and head size may be launched
    long long wait_cycles = 20000000000ll;   // budget of every device-side wait, in SM clock cycles (about ten seconds)
};

struct MatVecPlan {
    int wsize, zsize, ssize, units;
    int kw, mw, rw, nstage;
    int chunk_bytes, woff_z, woff_s;
    int smem_bytes, ntiles, grid, threads;
};

enum class Fmt : int;
enum class Epi : int;
enum class Pro : int;
struct MatVecParams;

int fail(int code, const char* fmt, ...);
// Makes the context's device current for the calling thread (every entry point does this first: a thread may hold
// several contexts, or may have switched device in between).
int use_device(const Ctx* ctx);
// The same, and the context's launches go to the caller's stream again, behind what a model of the context has queued on its own:
// a caller's tensors are ordered by the caller's stream.
int use_callers_stream(Ctx* ctx);
// The other way: a model's next launches, on its own stream, come behind such calls, which may still read its caches.
int use_model_stream(Ctx* ctx, cudaStream_t stream);
int plan_matvec(const Ctx* ctx, Fmt fmt, Epi epi, int rows, int cols, int nmat, MatVecPlan* pl);
int launch_matvec(Ctx* ctx, Fmt fmt, Epi epi, Pro pro, const MatVecPlan& pl, MatVecParams prm, bool pdl);

// What an operator finds wrong in device tables, or its own waits that ran out, go here: apart from the word of a model's waits,
// which stops the persistent kernel.
inline DeviceStatus* input_status(const Ctx* ctx) { return ctx->status_dev + 1; }

constexpr int kMaxPageSize = 1024;
constexpr int kMaxRequests = 8192;
// log2 of a page size, -1 when it is not a power of two in 1..kMaxPageSize
inline int page_shift(int page_size)
{
    for (int s = 0; (1 << s) <= kMaxPageSize; ++s)
        if (page_size == (1 << s)) return s;
    return -1;
}
template <typename... P>
inline bool aligned_to(size_t bytes, const P*... p)
{
    return ((reinterpret_cast<uintptr_t>(p) | ...) & (bytes - 1)) == 0;
}

// sampling chain (sampler.cu): Sampler.Sample for temperature != 0 on `st`; the logits are consumed in place
int sampler_chain(cudaStream_t st, int device, void* logits, int* indices, int size, float temperature, float top_p, float coin, int* tokens,
                  int next_pos);

}  // namespace ml2
