// Block tables and slot maps of a paged KV cache, built on the GPU from request lengths (ml2_block_tables).
//
// With pages(x) = ceil(x / page_size), a step that takes request r from old[r] to new[r] tokens is four prefix sums over
// the requests and three lists whose elements do not depend on one another:
//   pushes  pages(new) .. pages(old) - 1 of every request that shrinks go on top of the free stack,
//   pops    every request that grows takes pages(new) - pages(old) pages off the top,
//   tokens  token old[r] + j of a growing request gets row start[r] + j of the slot map.
// One CTA does the sums in shared memory, then the lists, cut evenly over its threads, each element finding its request by
// bisection of the sums. A page number that is none of the cache's is reported where it is met; it stays off the free stack,
// and the table that would have it gets -1. What bounds it is latency: loads of the lengths, the scan's barriers, dependent loads and the store.
// Where the tokens are many (a step that brings prompts), a second kernel of many CTAs writes the slot map from the finished
// table: 186000 tokens of 512 requests take 15.6 us, 13 of them the first kernel's; one CTA alone took 150. 64 requests that grow
// by one token take 3.6 us.
#include "../../include/ml2b200.h"

#include "batch_common.cuh"
#include "host_common.hpp"

namespace ml2 {

constexpr int kTablesThreads = 1024;
// Up to this many rows one CTA writes the slot map. One kernel / two: 4096 rows 5.0 / 7.4 us, 8192 7.4 / 9.2, 32768 18.5 / 10.2.
constexpr int kTablesFill = 8192;

struct TablesParams {
    const int* lengths;
    const int* new_lengths;
    int* table;
    int* free_pages;
    const int* free_count;
    int* lengths_out;
    int* free_count_out;
    int* query_start;
    int* slots;
    int* positions;
    int* refused;
    DeviceStatus* status;
    int n, page_shift, width, n_pages, max_tokens, offset;
    int fill;  // rows of the slot map that the first kernel writes: all of them or none
};

struct Sums {
    long long tokens;
    int back, need;
};
__device__ __forceinline__ Sums operator+(const Sums& a, const Sums& b) { return {a.tokens + b.tokens, a.back + b.back, a.need + b.need}; }

// Exclusive sum over the CTA's threads in thread order; `total` gets the sum of all. s: one entry per warp and one more.
__device__ __forceinline__ Sums block_scan(Sums v, Sums* s, Sums* total)
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
    Sums incl = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        Sums u;
        u.tokens = __shfl_up_sync(0xffffffffu, incl.tokens, o);
        u.back = __shfl_up_sync(0xffffffffu, incl.back, o);
        u.need = __shfl_up_sync(0xffffffffu, incl.need, o);
        if (lane >= o) incl = incl + u;
    }
    __syncthreads();  // s may still be read from an earlier scan
    if (lane == 31) s[warp] = incl;
    __syncthreads();
    if (warp == 0) {
        const Sums mine = lane < nw ? s[lane] : Sums{0, 0, 0};
        Sums w = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            Sums u;
            u.tokens = __shfl_up_sync(0xffffffffu, w.tokens, o);
            u.back = __shfl_up_sync(0xffffffffu, w.back, o);
            u.need = __shfl_up_sync(0xffffffffu, w.need, o);
            if (lane >= o) w = w + u;
        }
        if (lane < nw) s[lane] = Sums{w.tokens - mine.tokens, w.back - mine.back, w.need - mine.need};
        if (lane == 31) s[32] = w;
    }
    __syncthreads();
    *total = s[32];
    const Sums base = s[warp];
    return {base.tokens + incl.tokens - v.tokens, base.back + incl.back - v.back, base.need + incl.need - v.need};
}

// The r with s[r] <= x < s[r + 1], for x in [0, s[n]): entries that are empty are passed over.
__device__ __forceinline__ int bisect(const int* s, int n, int x)
{
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (s[mid + 1] > x) hi = mid;
        else lo = mid + 1;
    }
    return lo;
}

__global__ void __launch_bounds__(kTablesThreads) block_tables_kernel(const TablesParams p)
{
    extern __shared__ int s_all[];        // four arrays of n and three entries: 128 KB for the most requests
    __shared__ Sums s_scan[33];
    int* s_start = s_all;                 // rows of the slot map before request r
    int* s_pop = s_start + p.n + 1;       // pages taken before request r
    int* s_push = s_pop + p.n + 1;        // pages given back before request r
    int* s_old = s_push + p.n + 1;

    pdl_wait();

    const int per = ceil_div(p.n, (int)blockDim.x), r0 = min((int)threadIdx.x * per, p.n), r1 = min(r0 + per, p.n);
    const int mask = (1 << p.page_shift) - 1;
    auto pages = [&](int x) { return (x >> p.page_shift) + ((x & mask) ? 1 : 0); };
    auto valid = [&](int a, int b) { return a >= 0 && b >= 0 && pages(a) <= p.width && pages(b) <= p.width; };
    auto change = [&](int r) {
        const int a = p.lengths[r], b = p.new_lengths[r];
        Sums v{0, 0, 0};
        if (valid(a, b)) {
            v.tokens = max(b - a, 0);
            v.back = max(pages(a) - pages(b), 0);
            v.need = max(pages(b) - pages(a), 0);
        }
        return v;
    };

    Sums mine{0, 0, 0}, total;
    for (int r = r0; r < r1; ++r) mine = mine + change(r);
    Sums before = block_scan(mine, s_scan, &total);

    int count = *p.free_count;
    if (count < 0 || count > p.n_pages) {
        if (threadIdx.x == 0) report_input_error(p.status, kInputFreeCount, count);
        count = min(max(count, 0), p.n_pages);
    }
    const int threads = (int)blockDim.x, me = (int)threadIdx.x, room = p.n_pages - count;
    {
        int push = before.back;
        for (int r = r0; r < r1; ++r) {
            s_push[r] = push;
            s_old[r] = p.lengths[r];
            push += change(r).back;
        }
    }
    if (total.back) {
        __syncthreads();
        bool broken = false;
        for (unsigned x = me; x < (unsigned)total.back; x += threads) {
            const int r = bisect(s_push, p.n, x), id = p.table[(size_t)r * p.width + pages(p.new_lengths[r]) + (x - s_push[r])];
            if (id < 0 || id >= p.n_pages) {
                report_input_error(p.status, kInputPage, r);
                broken = true;
            } else if ((int)x < room) {
                p.free_pages[count + x] = id;
            }
        }
        // pages that are none stay off the stack: the others move together, each thread those of its requests
        if (__syncthreads_or(broken)) {
            auto given = [&](auto&& f) {
                for (int r = r0; r < r1; ++r)
                    for (int left = change(r).back, i = pages(p.new_lengths[r]); left > 0; --left, ++i) {
                        const int id = p.table[(size_t)r * p.width + i];
                        if (id >= 0 && id < p.n_pages) f(id);
                    }
            };
            Sums part{0, 0, 0}, sound;
            given([&](int) { ++part.back; });
            int at = block_scan(part, s_scan, &sound).back;
            given([&](int id) {
                if (at < room) p.free_pages[count + at] = id;
                ++at;
            });
            total.back = sound.back;
        }
    }
    if (total.back > room && threadIdx.x == 0) report_input_error(p.status, kInputFreeOverflow, total.back);
    const int have = count + min(total.back, room);
    const bool all_fit = total.tokens <= p.max_tokens && total.need <= have;

    // Exclusive sums of what is served. The usual case takes them from the scan above; when something does not fit, the
    // two cuts (tokens first, then pages among the rest) each move the sums behind them, so they are scanned again.
    if (all_fit) {
        for (int r = r0; r < r1; ++r) {
            const Sums v = change(r);
            s_start[r] = (int)before.tokens;
            s_pop[r] = before.need;
            before = before + v;
            p.refused[r] = valid(s_old[r], p.new_lengths[r]) ? 0 : ML2_REFUSED_LENGTH;
        }
    } else {
        const long long tokens_before = before.tokens;
        auto over = [&](const Sums& v, long long sum) { return v.tokens > 0 && sum > p.max_tokens; };
        Sums part{0, 0, 0}, unused;
        long long sum = tokens_before;
        for (int r = r0; r < r1; ++r) {
            const Sums v = change(r);
            sum += v.tokens;
            if (!over(v, sum)) part.need += v.need;
        }
        const Sums need_before = block_scan(part, s_scan, &unused);
        // pages, then tokens, of what is left
        Sums served{0, 0, 0};
        sum = tokens_before;
        int need = need_before.need;
        for (int r = r0; r < r1; ++r) {
            const Sums v = change(r);
            sum += v.tokens;
            int code = valid(s_old[r], p.new_lengths[r]) ? 0 : ML2_REFUSED_LENGTH;
            if (over(v, sum)) code = ML2_REFUSED_TOKENS;
            else if (v.need > 0) {
                need += v.need;
                if (need > have) code = ML2_REFUSED_PAGES;
            }
            if (!code) {
                served.tokens += v.tokens;
                served.need += v.need;
            }
            s_start[r] = code;  // this thread's own entry, replaced below
        }
        before = block_scan(served, s_scan, &total);
        for (int r = r0; r < r1; ++r) {
            const int code = s_start[r];
            const Sums v = change(r);
            s_start[r] = (int)before.tokens;
            s_pop[r] = before.need;
            if (!code) {
                before.tokens += v.tokens;
                before.need += v.need;
            }
            p.refused[r] = code;
        }
    }
    if (threadIdx.x == 0) {
        s_start[p.n] = (int)total.tokens;
        s_pop[p.n] = total.need;
    }
    // Pages given back are taken again below, and the lengths may be written over the ones read above: everybody is done
    // reading and pushing first.
    __syncthreads();

    const int n_pop = total.need, n_tokens = (int)total.tokens;
    for (unsigned x = me; x < (unsigned)n_pop; x += threads) {
        const int r = bisect(s_pop, p.n, x);
        int id = p.free_pages[have - 1 - x];
        if (id < 0 || id >= p.n_pages) {
            report_input_error(p.status, kInputPage, r);
            id = -1;
        }
        p.table[(size_t)r * p.width + pages(s_old[r]) + (x - s_pop[r])] = id;
    }
    for (int t = me; t < p.fill; t += threads) {
        int slot = -1, position = 0;
        if (t < n_tokens) {
            const int r = bisect(s_start, p.n, t), old = s_old[r], at = old + (t - s_start[r]);
            const int page = at >> p.page_shift, held = pages(old);
            // a page taken in this call is read from the stack: its table entry may not be written yet
            const int id = page < held ? p.table[(size_t)r * p.width + page] : p.free_pages[have - 1 - (s_pop[r] + page - held)];
            if (id >= 0 && id < p.n_pages) slot = (id << p.page_shift) + (at & mask);
            else report_input_error(p.status, kInputPage, r);
            position = p.offset + at;
        }
        p.slots[t] = slot;
        p.positions[t] = position;
    }
    for (int r = r0; r < r1; ++r) {
        // a request that keeps its rows keeps its length: growth is seen in the served sums, all else in the lengths
        const int a = s_old[r], b = p.new_lengths[r];
        const bool grows = b > a, served = s_start[r + 1] > s_start[r];
        p.query_start[r] = s_start[r];
        p.lengths_out[r] = !valid(a, b) || (grows && !served) ? a : b;
    }
    if (threadIdx.x == 0) {
        p.query_start[p.n] = n_tokens;
        *p.free_count_out = have - n_pop;
    }
}

// The slot map of many tokens, four a thread: request by bisection of query_start, its old length from the new one.
__global__ void __launch_bounds__(256) slot_map_kernel(const TablesParams p)
{
    pdl_wait();
    const int n_tokens = p.query_start[p.n], t0 = (blockIdx.x * 256 + threadIdx.x) * 4;
    if (t0 >= p.max_tokens) return;
    int r = 0, start = 0, end = 0, old = 0;
    for (int t = t0; t < min(t0 + 4, p.max_tokens); ++t) {
        int slot = -1, position = 0;
        if (t < n_tokens) {
            if (t >= end) {
                r = bisect(p.query_start, p.n, t);
                start = p.query_start[r];
                end = p.query_start[r + 1];
                old = p.new_lengths[r] - (end - start);
            }
            const int at = old + (t - start), id = p.table[(size_t)r * p.width + (at >> p.page_shift)];
            if (id >= 0 && id < p.n_pages) slot = (id << p.page_shift) + (at & ((1 << p.page_shift) - 1));
            else report_input_error(p.status, kInputPage, r);
            position = p.offset + at;
        }
        p.slots[t] = slot;
        p.positions[t] = position;
    }
}

}  // namespace ml2

using namespace ml2;

extern "C" int ml2_block_tables(ml2_ctx* h, const ml2_block_tables_args* args)
{
    Ctx* ctx = reinterpret_cast<Ctx*>(h);
    if (!ctx || !args) return fail(ML2_E_INVALID, "block_tables: null argument");
    const auto [lengths, new_lengths, table, free_pages, free_count, lengths_out, free_count_out, query_start, slots, positions, refused, n_requests,
                page_size, table_stride, n_pages, max_tokens, position_offset] = *args;
    if (!lengths || !new_lengths || !table || !free_pages || !free_count || !lengths_out || !free_count_out || !query_start || !refused)
        return fail(ML2_E_INVALID, "block_tables: null argument");
    if (!aligned_to(4, lengths, new_lengths, table, free_pages, free_count) || !aligned_to(4, lengths_out, free_count_out, query_start, slots, positions, refused))
        return fail(ML2_E_INVALID, "block_tables: arrays must be 4-byte aligned");
    if (max_tokens < 0 || max_tokens > INT32_MAX / 2 || (max_tokens > 0 && (!slots || !positions)))
        return fail(ML2_E_INVALID, "block_tables: max_tokens=%d with slots=%p positions=%p", max_tokens, (void*)slots, (void*)positions);
    if (n_requests < 1 || n_requests > kMaxRequests)
        return fail(ML2_E_INVALID, "block_tables: n_requests=%d must be 1..%d", n_requests, kMaxRequests);
    const int shift = page_shift(page_size);
    if (shift < 0) return fail(ML2_E_INVALID, "block_tables: page_size=%d must be a power of two, at most %d", page_size, kMaxPageSize);
    if (table_stride < 1 || n_pages < 1) return fail(ML2_E_INVALID, "block_tables: table_stride=%d n_pages=%d must be positive", table_stride, n_pages);
    const long long longest = (long long)table_stride * page_size;
    if (position_offset < 0 || longest + position_offset > INT32_MAX || (long long)n_requests * table_stride > INT32_MAX ||
        (long long)n_pages * page_size > INT32_MAX)
        return fail(ML2_E_INVALID, "block_tables: positions, pages or slots pass 32 bits (table %d x %d, page_size=%d, n_pages=%d, offset=%d)",
                    n_requests, table_stride, page_size, n_pages, position_offset);
    if (new_lengths == lengths_out || new_lengths == lengths)
        return fail(ML2_E_INVALID, "block_tables: new_lengths must be an array of its own");
    if (int rc = use_callers_stream(ctx)) return rc;

    TablesParams p{};
    p.lengths = lengths; p.new_lengths = new_lengths; p.table = table; p.free_pages = free_pages; p.free_count = free_count;
    p.lengths_out = lengths_out; p.free_count_out = free_count_out; p.query_start = query_start; p.slots = slots; p.positions = positions;
    p.refused = refused; p.status = input_status(ctx);
    p.n = n_requests; p.page_shift = shift; p.width = table_stride; p.n_pages = n_pages; p.max_tokens = max_tokens; p.offset = position_offset;
    p.fill = max_tokens <= kTablesFill ? max_tokens : 0;

    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(1);
    // few requests and rows: the barriers of 8 warps cost less than those of 32 (64 requests 3.6 us instead of 4.1)
    cfg.blockDim = dim3(n_requests <= 256 && p.fill <= 1024 ? 256 : kTablesThreads);
    cfg.dynamicSmemBytes = (4 * (size_t)n_requests + 3) * sizeof(int);
    cfg.stream = ctx->stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = ctx->pdl ? 1 : 0;
    cudaError_t e = cudaSuccess;
    // 48 KB of a block without this, the kernel's static shared memory among them
    if (cfg.dynamicSmemBytes + sizeof(Sums) * 33 > 48 * 1024)
        e = cudaFuncSetAttribute(block_tables_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)((4 * kMaxRequests + 3) * sizeof(int)));
    if (e == cudaSuccess) e = cudaLaunchKernelEx(&cfg, block_tables_kernel, p);
    if (e == cudaSuccess) {
        ++ctx->launches;
        if (p.fill < max_tokens) {
            cfg.gridDim = dim3((unsigned)ceil_div(max_tokens, 1024));
            cfg.blockDim = dim3(256);
            cfg.dynamicSmemBytes = 0;
            cfg.numAttrs = 1;  // is set up while the first kernel runs, and waits for it
            if ((e = cudaLaunchKernelEx(&cfg, slot_map_kernel, p)) == cudaSuccess) ++ctx->launches;
        }
    }
    if (e != cudaSuccess) return fail(ML2_E_CUDA, "block_tables: %s", cudaGetErrorString(e));
    return ML2_OK;
}
