// Attention of a batch whose requests share a prefix: every query row sees the shared rows, which lie in one contiguous
// cache, and the rows of its own request, which lie in pages (ml2_prefix_attention).
//
//   o = sum_j p_j v_j,  p_j = exp(scale q.k_j - lse),  lse = log sum_j exp(scale q.k_j),  j over the prefix and own rows 0..last
//
// with last = length - queries + i for query i of a request that has `queries` rows in this call.
#include "../../include/ml2b200.h"

#include "batch_common.cuh"
#include "host_common.hpp"
#include "tcgen05.cuh"

#include <cmath>
#include <type_traits>

namespace ml2 {

struct AttnBatch {
    void* out;
    float* lse;
    const void *q, *pk, *pv, *k, *v;
    const int *table, *lengths, *query_start;
    DeviceStatus* status;
    // Partial results, for a row and head the sum o = sum of exp2(score - m) v over some of the keys [head], and (m, l): a
    // reference up to 2^15 below the largest score (in powers of two) and l = sum of exp2(score - m). One without keys has m = -inf, l = 0
    // and an o that is not read. pre: of the prefix by blocks, [segments][rows that are there][n_heads]; run: of the warps' runs.
    float *pre_o, *run_o;
    float2 *pre_ml, *run_ml;
    int* run_base;      // [n_requests + 1]: places before request r, of all requests; then the places of a run, negative where
                        // the requests have more than own_places
    int own_places;     // of all requests at most, whose query rows do not overlap
    long long wait_cycles;
    long long out_stride, q_stride, prefix_stride, cache_stride;
    int n_requests, n_rows, prefix, max_length, n_pages, table_stride, page_shift, n_heads, n_kv, group;
    int prefix_ctas;    // of the kernel that does the prefix by blocks, 0 where the runs do it
    int run_ctas;       // of the kernel of runs, 0 without it
    float scale_log2;   // scale * log2(e)
};

// Query rows [first, first + count) and own tokens of request r; a request whose entries cannot be has none of either.
struct Span {
    int first, count, length;
    bool good;
};
__device__ __forceinline__ Span request_span(const AttnBatch& p, int r)
{
    const int a = p.query_start[r], b = p.query_start[r + 1], length = p.lengths[r];
    const bool good = a >= 0 && (r > 0 || a == 0) && b >= a && b <= p.n_rows && length >= 0 && length <= p.max_length;
    return good ? Span{a, b - a, length, true} : Span{0, 0, 0, false};
}

constexpr int kTile = 16;      // keys of a tile: the k of one m16n8k16 product with the values
// tiles of a warp's ring: 24 KB at either head size, so that two blocks of four warps share an SM
constexpr int stages(int head) { return head == 128 ? 3 : 6; }
constexpr int kAttnWarps = 4;
constexpr int kAttnThreads = 32 * kAttnWarps;
// The reference point m of a row is set kLower powers of two below a score and moves only when one exceeds it by more than
// kSlack: weights of at most 2^15 fit fp16 and sums are fp32, so the sums are rescaled a few times in all instead of at most
// tiles. Set as low as that, it leaves fp16 (whose smallest number is 2^-24) the weights down to 2^-32 of the largest: 65536
// keys of 2^-25.06 each beside one of 1 had no part in the output at all with m at the score itself. (The difference t - m is
// exact where it matters; t > m + kSlack could let 2^16 pass, which is infinite in fp16, where scores of 2^24 are 2 apart.)
constexpr float kSlack = 15.f, kLower = 7.f;
// Places of a run at least, where the longest sequence has n: a lone warp needs 0.7 us a place and the join 0.1 us a result, so
// that n places are best left to 2 sqrt(n) runs. One place a run where there are more warps than places: 19.8 us instead of 13.3
// for 8 heads of 8 and 1024 keys, 13.5 instead of 12.2 for 5 heads and 512; ten places: 17.1 and 15.9.
__device__ __forceinline__ int shortest_run(int n) { return max(1, (int)(0.5f * sqrtf((float)n) + 0.5f)); }
constexpr int kOpen = 1;       // what it costs to begin a sequence (its queries, its result), in key tiles: 2300 cycles against 2200

template <typename T> __device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t at)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t at)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
// 16 bytes to shared memory without passing registers; `bytes` 0 writes zeros and reads nothing
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int bytes)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ float exp2_fast(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// 0x8000 for either of two 16-bit values that is infinite or NaN: an exponent of ones carries over
template <typename T> __device__ __forceinline__ uint32_t not_finite(uint32_t w)
{
    constexpr bool kHalf = std::is_same<T, __half>::value;
    return ((w & (kHalf ? 0x7c007c00u : 0x7f807f80u)) + (kHalf ? 0x04000400u : 0x00800080u)) & 0x80008000u;
}
template <typename T> __device__ __forceinline__ uint32_t times_zero(uint32_t w) { return (not_finite<T>(w) >> 15) * 0x7fffu; }  // 0 or NaN

// A weight as the sum of two 16-bit numbers, 22 bits of it in fp16 and 16 in bf16: the products with the values then lose nothing
// that the output's own rounding leaves to see (with one, the error against 64 bits was 1.3 times that rounding's, 2.8e-4 against
// 2.1e-4 in fp16). The first lies below the weight, by cutting off the number before it, so that the second is above 0: a weight
// times an infinite value is infinite, not 0 times infinity. (Weights below 2^-13 in fp16 may have a second part of 0.)
template <typename T> __device__ __forceinline__ uint32_t below2(float a, float b)
{
    const int x = max(__float_as_int(a) - 1, 0), y = max(__float_as_int(b) - 1, 0);
    if constexpr (std::is_same<T, __half>::value) {
        uint32_t w;
        asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(__int_as_float(y)), "f"(__int_as_float(x)));
        return w;
    } else {
        return __byte_perm(x, y, 0x7632);
    }
}
template <typename T> __device__ __forceinline__ uint32_t rest2(uint32_t w, float a, float b)
{
    const float2 f = unpack2<T>(w);
    return pack2<T>(a - f.x, b - f.y);
}

// Rows of a request that has `count` queries (or of the prefix, which all see), counted 16 at a time.
__device__ __forceinline__ int row_tiles(const AttnBatch& p, int count) { return (count * p.group + 15) >> 4; }
// Key tiles that the 16 rows from row0 on look at: as many as the last of them sees.
__device__ __forceinline__ int tiles_seen(const AttnBatch& p, int count, int length, int row0, int rows)
{
    const int last = (row0 + rows - 1) / p.group, seen = min(length, length - count + last + 1);
    return seen > 0 ? (seen + kTile - 1) / kTile : 0;
}
// A request's share of the runs: `seqs` row tiles for each key head, the first of which sees `low` key tiles and the last `high`.
// Places before row tile rt, for one key head: kOpen and the key tiles of each row tile, the latter taken to grow evenly from low
// to high and, where they grow, two more, which covers every row tile (checked for groups of up to 65536 heads; 7 % more
// places than are needed, where `high` for all would be 70 % more).
struct Share {
    int seqs, low, high;
};
__device__ __forceinline__ Share request_share(const AttnBatch& p, int count, int length)
{
    const int n = row_tiles(p, count);
    if (!n) return {0, 0, 0};
    return {n, tiles_seen(p, count, length, 0, min(16, count * p.group)), tiles_seen(p, count, length, 16 * (n - 1), count * p.group - 16 * (n - 1))};
}
__device__ __forceinline__ int places_before(const Share& s, int rt)
{
    if (!s.high) return 0;
    long long n = (long long)rt * (kOpen + s.low);
    if (s.high > s.low) n += 2 * rt + (long long)(s.high - s.low) * rt * (rt - 1) / (2 * (s.seqs - 1));
    return (int)n;
}
// Where the result of run `run` for the 16 rows from row0 on of a key head begins: runs and rows are numbered through, so that
// no two results meet and all need no more than one entry per row and head, and 16 per run.
__device__ __forceinline__ long long result_row(const AttnBatch& p, bool prefix, int first, int row0, int rows, int kvh, int run)
{
    return (prefix ? (long long)p.n_rows * p.n_heads : 0) + ((long long)first * p.group + row0) * p.n_kv + kvh * rows + 16ll * run;
}

// a + b of numbers that are not negative, 2^31 - 1 at most
__device__ __forceinline__ int add_up_to(int a, int b) { return (int)min((unsigned)a + (unsigned)b, 0x7fffffffu); }

// A walk over one run: 16 rows of one key head and request (a sequence), kOpen places for its beginning and one for each of its
// key tiles, then the next sequence.
struct Walk {
    int pos, end;              // of all tiles
    int request;               // n_requests: the prefix
    int rt, kvh, k;            // row tile, key head, place in the sequence
    int first, count, length;  // query rows and keys of the request
    Share share;
    int places, need, rows;    // places of a sequence, those up to the last key tile that its rows see, its rows
};
__device__ __forceinline__ void open_request(const AttnBatch& p, Walk& w, int total_rows)
{
    if (w.request == p.n_requests) {
        w.first = 0;
        w.count = total_rows;
        w.length = p.prefix;
    } else {
        const Span s = request_span(p, w.request);
        w.first = s.first;
        w.count = s.count;
        w.length = s.length;
    }
    const int all = (w.length + kTile - 1) / kTile;
    w.share = w.request == p.n_requests ? Share{row_tiles(p, w.count), all, all} : request_share(p, w.count, w.length);
}
__device__ __forceinline__ void open_rows(const AttnBatch& p, Walk& w)
{
    w.rows = min(16, w.count * p.group - w.rt * 16);
    w.places = places_before(w.share, w.rt + 1) - places_before(w.share, w.rt);
    w.need = w.request == p.n_requests ? w.places : kOpen + tiles_seen(p, w.count, w.length, w.rt * 16, w.rows);
}
__device__ __forceinline__ void open_walk(const AttnBatch& p, const int* s_base, int total_rows, Walk& w)
{
    if (w.pos >= w.end) return;
    int lo = 0, hi = p.n_requests;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (s_base[mid + 1] > w.pos) hi = mid;
        else lo = mid + 1;
    }
    w.request = lo;
    open_request(p, w, total_rows);
    const int local = w.pos - s_base[lo];
    int rt = 0;
    for (int n = w.share.seqs; n > 1;) {
        const int half = n >> 1;
        if (places_before(w.share, rt + half) * p.n_kv <= local) rt += half;
        n -= half;
    }
    w.rt = rt;
    open_rows(p, w);
    // key heads, next to one another in the cache, go to neighbouring runs
    const int rest = local - places_before(w.share, rt) * p.n_kv;
    w.kvh = rest / w.places;
    w.k = rest - w.kvh * w.places;
}
// Moves to the next key tile that somebody sees; false at the end of the run.
__device__ __forceinline__ bool settle(const AttnBatch& p, const int* s_base, int total_rows, Walk& w)
{
    while (w.pos < w.end) {
        if (w.k < kOpen) {
            const int n = min(kOpen - w.k, w.end - w.pos);
            w.k += n;
            w.pos += n;
            continue;
        }
        if (w.k < w.need) return true;
        w.pos += w.places - w.k;
        w.k = 0;
        if (w.pos >= w.end) return false;
        if (++w.kvh < p.n_kv) continue;
        w.kvh = 0;
        if (++w.rt == w.share.seqs) {
            w.rt = 0;
            do ++w.request;
            while (s_base[w.request + 1] == s_base[w.request]);
            open_request(p, w, total_rows);
        }
        open_rows(p, w);
    }
    return false;
}

// Every warp works for itself: the key tiles of all requests, one after the other, and one place more for every sequence, are
// cut into runs of the same length, one a warp (without that place runs through short requests took 1.5 times as long). It
// streams its tiles through a ring of its own (cp.async; the next ones are under way while one is used, across the borders of
// sequences) and leaves a result for every sequence that it has a part of. 16 rows are all the tensor core's m16 has, so a tile of
// 16 keys (8 KB at head 128) costs 48 products however few rows are real: with one row a request HBM bounds it (64 requests of 135
// tokens, 40 heads of 128: 173 MB in 37 us, 4.7 TB/s), with many the instructions and their latency (1229 queries of 8 requests,
// 32 heads: 53000 tiles in 70 us, the keys read again for every 16 queries).
template <typename T, int kHead>
__global__ void __launch_bounds__(kAttnThreads, 2) attention_runs_kernel(const __grid_constant__ AttnBatch p)
{
    constexpr int kRowBytes = kHead * 2, kChunks = kHead / 8, kTileBytes = kTile * kRowBytes, kSteps = kHead / 16, kStages = stages(kHead);
    extern __shared__ __align__(128) unsigned char s_mem[];
    __shared__ unsigned s_valid[kAttnWarps][kStages];
    __shared__ int s_sum[kAttnWarps], s_long[kAttnWarps];
    int* s_base = reinterpret_cast<int*>(s_mem + kAttnWarps * kStages * 2 * kTileBytes);  // places before request r; the prefix last

    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    // After the prefix kernel this one starts beside it, and reads queries, pages and tables without a wait of its own: every block of
    // that kernel has come past its own wait, for all that precedes both, before it lets this one start. (It waits for the prefix
    // kernel at its end.)
    if (!p.prefix_ctas) pdl_wait();
    pdl_launch_dependents();  // every block is resident by the time the join's come, which look up their rows meanwhile
    const int total_rows = min(max(p.query_start[p.n_requests], 0), p.n_rows);
    bool too_many;
    int longest = kOpen + (p.prefix_ctas ? 0 : (p.prefix + kTile - 1) / kTile);
    // ---- how many places every request has -----------------------------------------------------------------------------
    {
        const int per = ceil_div(p.n_requests, kAttnThreads), r0 = min((int)threadIdx.x * per, p.n_requests), r1 = min(r0 + per, p.n_requests);
        int mine = 0;
        for (int r = r0; r < r1; ++r) {
            const Span s = request_span(p, r);
            if (!s.good && blockIdx.x == 0) report_input_error(p.status, kInputLength, r);
            s_base[r] = mine;
            const Share share = request_share(p, s.count, s.length);
            mine = add_up_to(mine, places_before(share, share.seqs) * p.n_kv);
            longest = max(longest, kOpen + share.high);
        }
        // Rows that several requests lay claim to (query rows out of order, reported above) count for each of them: their sum may pass
        // what the host saw fits, and 32 bits. Nobody has own tokens then.
        int incl = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl = add_up_to(incl, v);
        }
        int before = __shfl_up_sync(0xffffffffu, incl, 1);
        if (lane == 0) before = 0;
        longest = __reduce_max_sync(0xffffffffu, longest);
        if (lane == 31) {
            s_sum[warp] = incl;
            s_long[warp] = longest;
        }
        __syncthreads();
        int base = before, all = 0;
#pragma unroll
        for (int w = 0; w < kAttnWarps; ++w) {
            if (w < warp) base = add_up_to(base, s_sum[w]);
            all = add_up_to(all, s_sum[w]);
            longest = max(longest, s_long[w]);
        }
        too_many = all > p.own_places;
        if (too_many) all = 0;
        for (int r = r0; r < r1; ++r) s_base[r] = too_many ? 0 : s_base[r] + base;
        if (threadIdx.x == 0) {
            s_base[p.n_requests] = all;
            s_base[p.n_requests + 1] = all + (p.prefix_ctas || !p.prefix ? 0 : row_tiles(p, total_rows) * p.n_kv * (kOpen + (p.prefix + kTile - 1) / kTile));
        }
        __syncthreads();
    }
    const int all = s_base[p.n_requests + 1], per = max(shortest_run(longest), (all + (int)gridDim.x * kAttnWarps - 1) / ((int)gridDim.x * kAttnWarps)), run = blockIdx.x * kAttnWarps + warp;
    if (blockIdx.x == 0) {  // the join finds the results by these
        for (int r = threadIdx.x; r <= p.n_requests; r += kAttnThreads) p.run_base[r] = s_base[r];
        if (threadIdx.x == 0) p.run_base[p.n_requests + 1] = too_many ? -per : per;
    }

    unsigned char* ring = s_mem + warp * kStages * 2 * kTileBytes;
    const uint32_t ring_u32 = smem_u32(ring);
    const int page_mask = (1 << p.page_shift) - 1;

    // ---- where the loads stand: the next tile to ask for ----------------------------------------------------------------
    Walk ld{};
    ld.pos = min(run * per, all);
    ld.end = min(ld.pos + per, all);
    open_walk(p, s_base, total_rows, ld);
    Walk w = ld;
    bool more = settle(p, s_base, total_rows, ld);
    int row = -1;  // lanes 0..15: cache row of the tile's key `lane`, -1 for none
    auto find_rows = [&]() {
        const int key = (ld.k - kOpen) * kTile + (lane & 15);
        row = -1;
        if (key < ld.length) {
            if (ld.request == p.n_requests) row = key;
            else {
                const int page = p.table[(long long)ld.request * p.table_stride + (key >> p.page_shift)];
                if (page >= 0 && page < p.n_pages) row = (page << p.page_shift) + (key & page_mask);
                else report_input_error(p.status, kInputPage, ld.request);
            }
        }
    };
    auto load_tile = [&](int stage) {
        if (more) {
            const bool prefix = ld.request == p.n_requests;
            const char* kb = static_cast<const char*>(prefix ? p.pk : p.k) + (ld.kvh * kHead + lane % kChunks * 8) * 2;
            const char* vb = static_cast<const char*>(prefix ? p.pv : p.v) + (ld.kvh * kHead + lane % kChunks * 8) * 2;
            const unsigned step = (unsigned)(prefix ? p.prefix_stride : p.cache_stride) * 2u;  // bytes, below 2^32
            const unsigned valid = __ballot_sync(0xffffffffu, row >= 0) & 0xffffu;
            if (lane == 0) s_valid[warp][stage] = valid;
            const uint32_t dst = ring_u32 + stage * 2 * kTileBytes + lane / kChunks * kRowBytes;
#pragma unroll
            for (int i = 0; i < kChunks / 2; ++i) {
                const int key = i * (32 / kChunks) + lane / kChunks, r = __shfl_sync(0xffffffffu, row, key), bytes = r < 0 ? 0 : 16;
                const unsigned long long off = (unsigned long long)(unsigned)max(r, 0) * step;
                const uint32_t to = dst + i * (32 / kChunks) * kRowBytes + (((lane % kChunks) ^ (key & 7)) << 4);
                cp_async16(to, kb + off, bytes);
                cp_async16(to + kTileBytes, vb + off, bytes);
            }
            ++ld.k;
            ++ld.pos;
            more = settle(p, s_base, total_rows, ld);
            if (more) find_rows();  // the table is asked one tile ahead
        }
        cp_async_commit();
    };

    if (more) find_rows();
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) load_tile(i);

    int stage = 0;
    const int g = lane >> 2, t4 = lane & 3;
    while (settle(p, s_base, total_rows, w)) {
        const bool prefix = w.request == p.n_requests;
        const int n_tiles = min(w.need - w.k, w.end - w.pos), key0 = (w.k - kOpen) * kTile, row0 = w.rt * 16;
        w.pos += n_tiles;
        w.k += n_tiles;

        // rows g and g + 8 of the tile: query row, head, and the keys they see
        const int m0 = row0 + g, m1 = m0 + 8;
        const bool live0 = g < w.rows, live1 = g + 8 < w.rows;
        const int i0 = m0 / p.group, i1 = m1 / p.group;
        const int h0 = w.kvh * p.group + m0 % p.group, h1 = w.kvh * p.group + m1 % p.group;
        const int seen0 = prefix ? w.length : w.length - w.count + i0 + 1, seen1 = prefix ? w.length : w.length - w.count + i1 + 1;
        const int seen_by_all = prefix || w.count == 1 ? w.length : w.length - w.count + row0 / p.group + 1;

        uint32_t qf[kSteps][4];
        {
            const T* q0 = static_cast<const T*>(p.q) + (long long)(w.first + i0) * p.q_stride + (long long)h0 * kHead + t4 * 2;
            const T* q1 = static_cast<const T*>(p.q) + (long long)(w.first + i1) * p.q_stride + (long long)h1 * kHead + t4 * 2;
#pragma unroll
            for (int k = 0; k < kSteps; ++k) {
                qf[k][0] = live0 ? *reinterpret_cast<const uint32_t*>(q0 + k * 16) : 0u;
                qf[k][1] = live1 ? *reinterpret_cast<const uint32_t*>(q1 + k * 16) : 0u;
                qf[k][2] = live0 ? *reinterpret_cast<const uint32_t*>(q0 + k * 16 + 8) : 0u;
                qf[k][3] = live1 ? *reinterpret_cast<const uint32_t*>(q1 + k * 16 + 8) : 0u;
            }
        }
        float acc[kHead / 8][4];
#pragma unroll
        for (int n = 0; n < kHead / 8; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
        float mx0 = -INFINITY, mx1 = -INFINITY, l0 = 0.f, l1 = 0.f;

        for (int key = key0; key < key0 + n_tiles * kTile; key += kTile) {
            cp_async_wait<kStages - 2>();
            __syncwarp();
            const uint32_t kt = ring_u32 + stage * 2 * kTileBytes, vt = kt + kTileBytes;
            const unsigned valid = s_valid[warp][stage];

            float s[2][4] = {};
            {
                float odd[2][4] = {};  // the steps alternate between two sums: half as long a chain of products
                const int kr = (lane & 7) + ((lane >> 4) & 1) * 8, kc = (lane >> 3) & 1;
#pragma unroll
                for (int k = 0; k < kSteps; ++k) {
                    uint32_t b[4];
                    ldsm4(b, kt + kr * kRowBytes + (((2 * k + kc) ^ (kr & 7)) << 4));
                    mma16816<T>(k & 1 ? odd[0] : s[0], qf[k], b[0], b[1]);
                    mma16816<T>(k & 1 ? odd[1] : s[1], qf[k], b[2], b[3]);
                }
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[n][e] += odd[n][e];
            }
            const bool causal = key + kTile > seen_by_all && seen_by_all < w.length, masked = valid != 0xffffu || causal;
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    s[n][e] *= p.scale_log2;
                    if (masked) {
                        const int j = n * 8 + t4 * 2 + (e & 1);
                        if (!((valid >> j) & 1u) || key + j >= (e < 2 ? seen0 : seen1)) s[n][e] = -INFINITY;
                    }
                }
            float t0 = fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[1][0], s[1][1]));
            float t1 = fmaxf(fmaxf(s[0][2], s[0][3]), fmaxf(s[1][2], s[1][3]));
            t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, 1));
            t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, 1));
            t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, 2));
            t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, 2));
            if (__any_sync(0xffffffffu, t0 - mx0 > kSlack || t1 - mx1 > kSlack)) {  // a much larger score: what was summed shrinks
                const float n0 = t0 - mx0 > kSlack ? t0 - kLower : mx0, n1 = t1 - mx1 > kSlack ? t1 - kLower : mx1;
                const float c0 = n0 == mx0 ? 1.f : exp2_fast(mx0 - n0), c1 = n1 == mx1 ? 1.f : exp2_fast(mx1 - n1);
                l0 *= c0;
                l1 *= c1;
#pragma unroll
                for (int n = 0; n < kHead / 8; ++n) {
                    acc[n][0] *= c0;
                    acc[n][1] *= c0;
                    acc[n][2] *= c1;
                    acc[n][3] *= c1;
                }
                mx0 = n0;
                mx1 = n1;
            }
            const float b0 = mx0 == -INFINITY ? 0.f : mx0, b1 = mx1 == -INFINITY ? 0.f : mx1;
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                s[n][0] = exp2_fast(s[n][0] - b0);
                s[n][1] = exp2_fast(s[n][1] - b0);
                s[n][2] = exp2_fast(s[n][2] - b1);
                s[n][3] = exp2_fast(s[n][3] - b1);
                l0 += s[n][0] + s[n][1];
                l1 += s[n][2] + s[n][3];
            }
            if (causal) {
                // Weight 0 times a value that is not finite would be NaN in the rows that do not see its key. Such keys are
                // taken out of the product and added to the rows that see them one by one.
                unsigned odd = 0;
                for (int i = 0; i < kChunks / 2; ++i) {
                    const int at = i * 32 + lane;  // 16 bytes of key at / kChunks
                    uint32_t v[4];
                    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(vt + at * 16) : "memory");
                    bool bad = false;
#pragma unroll
                    for (int e = 0; e < 4; ++e) bad |= not_finite<T>(v[e]) != 0;
                    if (bad) odd |= 1u << (at / kChunks);
                }
                odd = __reduce_or_sync(0xffffffffu, odd);
                for (unsigned left = odd; left; left &= left - 1) {
                    const int j = __ffs(left) - 1, n = j >> 3, src = (lane & ~3) | ((j & 7) >> 1);
                    const float pa = (j & 1) ? s[n][1] : s[n][0], pb = (j & 1) ? s[n][3] : s[n][2];
                    const float p0 = __shfl_sync(0xffffffffu, pa, src), p1 = __shfl_sync(0xffffffffu, pb, src);
                    const bool in0 = key + j < seen0, in1 = key + j < seen1;
#pragma unroll
                    for (int d = 0; d < kHead / 8; ++d) {
                        const uint32_t at = vt + j * kRowBytes + (((d ^ (j & 7)) << 4) | (t4 << 2));
                        uint32_t v;
                        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
                        const float2 f = unpack2<T>(v);
                        if (in0) { acc[d][0] += p0 * f.x; acc[d][1] += p0 * f.y; }
                        if (in1) { acc[d][2] += p1 * f.x; acc[d][3] += p1 * f.y; }
                    }
                }
                if (odd) {
                    __syncwarp();
                    for (unsigned left = odd; left; left &= left - 1) {
                        const int j = __ffs(left) - 1;
                        for (int c = lane; c < kHead / 2; c += 32)
                            asm volatile("st.shared.u32 [%0], %1;" ::"r"(vt + j * kRowBytes + c * 4), "r"(0u) : "memory");
                    }
                    __syncwarp();
                }
            }
            // both parts of the weights: 16 more products a tile, hidden behind loads in all but the largest calls (own tokens of 1229
            // queries: 3 % more)
            const uint32_t pf[4] = {below2<T>(s[0][0], s[0][1]), below2<T>(s[0][2], s[0][3]), below2<T>(s[1][0], s[1][1]), below2<T>(s[1][2], s[1][3])};
            const uint32_t pr[4] = {rest2<T>(pf[0], s[0][0], s[0][1]), rest2<T>(pf[1], s[0][2], s[0][3]), rest2<T>(pf[2], s[1][0], s[1][1]),
                                    rest2<T>(pf[3], s[1][2], s[1][3])};
            {
                const int vr = (lane & 7) + ((lane >> 3) & 1) * 8, vc = lane >> 4;
#pragma unroll
                for (int d = 0; d < kHead / 16; ++d) {
                    uint32_t b[4];
                    ldsm4_t(b, vt + vr * kRowBytes + (((2 * d + vc) ^ (vr & 7)) << 4));
                    mma16816<T>(acc[2 * d], pf, b[0], b[1]);
                    mma16816<T>(acc[2 * d + 1], pf, b[2], b[3]);
                    mma16816<T>(acc[2 * d], pr, b[0], b[1]);
                    mma16816<T>(acc[2 * d + 1], pr, b[2], b[3]);
                }
            }
            __syncwarp();  // everybody has read the tile that the next load writes over one turn from now
            load_tile(stage == 0 ? kStages - 1 : stage - 1);
            stage = stage == kStages - 1 ? 0 : stage + 1;
        }
        l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
        l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
        l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
        l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
        const long long at0 = result_row(p, prefix, w.first, row0, w.rows, w.kvh, run) + g, at1 = at0 + 8;
        if (live0) {
            if (t4 == 0) p.run_ml[at0] = make_float2(mx0, l0);
#pragma unroll
            for (int n = 0; n < kHead / 8; ++n) *reinterpret_cast<float2*>(p.run_o + at0 * kHead + n * 8 + t4 * 2) = make_float2(acc[n][0], acc[n][1]);
        }
        if (live1) {
            if (t4 == 0) p.run_ml[at1] = make_float2(mx1, l1);
#pragma unroll
            for (int n = 0; n < kHead / 8; ++n) *reinterpret_cast<float2*>(p.run_o + at1 * kHead + n * 8 + t4 * 2) = make_float2(acc[n][2], acc[n][3]);
        }
    }
    cp_async_wait<0>();
    if (p.prefix_ctas) pdl_wait();  // the join follows this kernel: it may start when the prefix is done too
}

// ---- the prefix, with many rows: fifth-generation tensor core ------------------------------------------------------------
//
// A block is 256 rows (query row, head of the group) of one key head, as two tiles of 128; blocks x key tiles of 64 keys are
// cut into one contiguous run per CTA, so all CTAs do the same work within one tile and a block's runs ("segments") are
// joined afterwards. Two streams of a CTA alternate on the tensor core:
//   S = Q K^T (operands in shared memory, S in TMEM, two of them a stream: one is filled while the other is used),
//   P = exp2(S - m), in 16 bits, over S in TMEM           (256 threads, half a row each)
//   O += P V (P from TMEM, V as it lies: MN-major)
// With more than 128 rows both streams use each key tile, the first with rows 0..127, the second with 128..255. With fewer,
// both have the same rows and take the key tiles in turn: then HBM bounds the kernel and eight tiles of 16 KB are under way
// (64 rows of 40 heads, 4032 keys: 83 MB in 25 us from a cold start). With many rows the products themselves (N = 64 reads its
// operands from shared memory at 47 cycles a product instead of 32) and the instructions of the warps that queue them bound it:
// 1024 rows of 8 heads, 16384 keys: 69 GFLOP in 68 to 78 us (of different GPUs), the tensor pipe 55 % active. Without the softmax
// it took 12 us less, without seven of eight products 31 us less. S tiles of 128 keys, one a stream, were tried when one lane
// alone ran the code that queues the products (64 samples of 40 heads: 100 us a call instead of 83), and not since.
constexpr int kBlockRows = 256;
constexpr int kKeyTile = 64;
constexpr int kRing = 4;                 // key tiles in shared memory, and value tiles
constexpr int kBlockThreads = 608;       // per stream 8 softmax warps and one that feeds the tensor core; load warp
// From which length on the prefix is done by blocks, not by runs, with up to 16 rows of a key head and with more. Measured, at up to
// 512 rows of a key head (with more the runs' time grows and the blocks' hardly does, so that these are better earlier) (us by
// blocks / by runs): 1 row of 40 heads, 1024 keys 17.8 / 14.9, 4096 27.0 / 27.9, 8192 38.9 / 41.6; 64 rows of 40 heads, 512 keys
// 26.2 / 21.7, 1024 28.6 / 28.1, 2048 33.0 / 37.3; 512 rows of 8 heads, 512 keys 23.6 / 22.0, 1024 24.3 / 30.5, 4096 32.2 / 84.4.
constexpr int kBlockPrefixFewRows = 4096, kBlockPrefix = 1024;

// Up to this many rows of a key head both parts of the weights are multiplied (the second lies behind the first, over S as well):
// HBM bounds the kernel then (the call of 64 rows of 40 heads behind 4032 keys takes 69 us instead of 67). With more rows the
// products do: that of 1024 rows of 8 heads behind 16384 keys would take 130 us instead of 114, so the weights are rounded to 16
// bits, for an error against 64 bits of 2.3e-3 instead of 1.7e-3 in bf16.
constexpr int kWholeRows = kBlockRows / 2;

struct PrefixMaps {
    CUtensorMap k, v;
};
struct PrefixRuns {  // how blocks and key tiles are cut, from the rows that are there: the same in both kernels
    int rows, blocks, key_tiles, per;    // rows of a key head, blocks of them, key tiles of one block, tiles of a CTA
    int tiles;                           // n_kv * blocks * key_tiles, below 2^31 (the host sees to it)
};
__host__ __device__ __forceinline__ PrefixRuns prefix_runs(int total_rows, int group, int n_kv, int prefix, int ctas)
{
    PrefixRuns r{};
    r.rows = total_rows * group;
    r.blocks = ceil_div(r.rows, kBlockRows);
    r.key_tiles = ceil_div(prefix, kKeyTile);
    r.tiles = n_kv * r.blocks * r.key_tiles;
    r.per = ceil_div(r.tiles, ctas);
    return r;
}
// Segments of a block: the CTAs first .. last have a part of it; two results each where the streams take turns.
__device__ __forceinline__ void block_segments(const PrefixRuns& r, int kvh, int block, int* first, int* results)
{
    const unsigned a = (unsigned)(kvh * r.blocks + block) * r.key_tiles;
    *first = (int)(a / (unsigned)r.per);
    const int n = (int)((a + r.key_tiles - 1) / (unsigned)r.per) - *first + 1;
    *results = r.rows - block * kBlockRows <= kBlockRows / 2 ? 2 * n : n;
}

template <int kHead> struct BlockSmem {
    static constexpr int kQHalf = 128 * 128, kQBytes = kQHalf * (kHead / 64);            // 64 dims of 128 rows, 128-byte swizzle
    static constexpr int kHalf = kKeyTile * 128, kTileBytes = kHalf * (kHead / 64);      // 64 dims of a key or value tile
    static constexpr int kBytes = 1024 + 2 * kQBytes + 2 * kRing * kTileBytes;
};

// a * b + c, a + b on two fp32 values at once
__device__ __forceinline__ uint64_t two(float x, float y) { return (uint64_t)__float_as_uint(y) << 32 | __float_as_uint(x); }
__device__ __forceinline__ float2 apart(uint64_t v) { return make_float2(__uint_as_float((uint32_t)v), __uint_as_float((uint32_t)(v >> 32))); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c)
{
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b)
{
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

// Barrier of the two warps `id`; true when `flag` is for any thread of them.
__device__ __forceinline__ bool pair_any(int id, bool flag)
{
    uint32_t any;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 q, %3, 0;\n\tbar.red.or.pred p, %1, %2, q;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(any)
                 : "r"(id), "r"(64), "r"((uint32_t)flag)
                 : "memory");
    return any != 0;
}

template <typename T, int kHead, bool kWhole>
__global__ void __launch_bounds__(kBlockThreads, 1) attention_prefix_kernel(const __grid_constant__ AttnBatch p, const __grid_constant__ PrefixMaps maps)
{
    using S = BlockSmem<kHead>;
    constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
    extern __shared__ unsigned char s_raw[];
    // Tile g of the CTA's run (counted over all segments) has key and value slot g % kRing. b_k, b_v: it has landed. b_s, b_o, for
    // each stream: its scores or its product with the values are done, which also frees the slot; a stream that does not use the
    // tile arrives there as well. A commit costs the feeding thread 90 cycles, so each serves both ends.
    __shared__ uint64_t b_k[kRing], b_v[kRing], b_s[2][kRing], b_o[2][kRing], b_q[2], b_p[2][2], b_end[2];
    __shared__ float s_top[2][2][128];  // of a stream's half rows, when they have to agree on m, and their sums
    __shared__ uint32_t s_tmem;
    __shared__ int s_abort;
    const uint32_t q_base = (smem_u32(s_raw) + 1023u) & ~1023u, k_ring = q_base + 2 * S::kQBytes, v_ring = k_ring + kRing * S::kTileBytes;
    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;  // uniform, and known to be

    if (threadIdx.x == 0) {
        for (int i = 0; i < kRing; ++i) {
            mbar_init(&b_k[i], 1);
            mbar_init(&b_v[i], 1);
            for (int j = 0; j < 2; ++j) {
                mbar_init(&b_s[j][i], 1);
                mbar_init(&b_o[j][i], 1);
            }
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&b_q[i], 8);  // one arrival a warp
            mbar_init(&b_p[i][0], 8);
            mbar_init(&b_p[i][1], 8);
            mbar_init(&b_end[i], 1);
        }
        s_abort = 0;
        mbar_fence_init();
    }
    if (warp == 16) tmem_alloc(&s_tmem, 512);
    if (warp == 18 && lane == 0) {
        tma_prefetch_map(&maps.k);
        tma_prefetch_map(&maps.v);
    }
    pdl_wait();
    pdl_launch_dependents();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem;  // columns: S of stream 0 (2 x 64), of stream 1, O of stream 0 (128), of stream 1

    const int total_rows = min(max(p.query_start[p.n_requests], 0), p.n_rows);
    const PrefixRuns runs = prefix_runs(total_rows, p.group, p.n_kv, p.prefix, gridDim.x);
    const int begin = min((int)blockIdx.x * runs.per, runs.tiles), end = min(begin + runs.per, runs.tiles);

    // a CTA's run, block by block: f(kvh, block, first key tile, tiles)
    auto for_segments = [&](auto&& f) {
        if (begin >= end) return true;
        int kvh = begin / runs.key_tiles, tile = begin - kvh * runs.key_tiles, block = kvh % runs.blocks;
        kvh /= runs.blocks;
        for (int left = end - begin; left > 0;) {
            const int n = min(runs.key_tiles - tile, left);
            if (!f(kvh, block, tile, n)) return false;
            left -= n;
            tile = 0;
            if (++block == runs.blocks) {
                block = 0;
                ++kvh;
            }
        }
        return true;
    };
    // tiles of a stream in a segment
    auto share = [](bool turns, int n, int stream) { return turns ? (n + 1 - stream) >> 1 : n; };

    if (warp == 18) {
        // ---- loads, in the order of their first use ------------------------------------------------------------------
        if (lane == 0) {
            unsigned base = 0, keys = 0, vals = 0;  // first tile of the segment; tiles asked for
            auto load = [&](bool key, int kvh, int tile, unsigned g) {
                const unsigned slot = g % kRing, parity = (g / kRing & 1) ^ 1;
                for (int s = 0; s < 2; ++s)
                    if (!mbar_wait_for(key ? &b_s[s][slot] : &b_o[s][slot], parity, p.wait_cycles, &s_abort)) return false;
                uint64_t* full = key ? &b_k[slot] : &b_v[slot];
                mbar_arrive_expect_tx(full, S::kTileBytes);
#pragma unroll
                for (int h = 0; h < kHead / 64; ++h)
                    tma_load_2d((key ? k_ring : v_ring) + slot * S::kTileBytes + h * S::kHalf, key ? &maps.k : &maps.v, kvh * kHead + h * 64,
                                tile * kKeyTile, full);
                ++(key ? keys : vals);
                return true;
            };
            for_segments([&](int kvh, int block, int tile, int n) {
                const int step = runs.rows - block * kBlockRows <= kBlockRows / 2 ? 2 : 1;
                auto loads = [&](bool key, int j) {
                    for (int t = j * step; t < min(n, (j + 1) * step); ++t)
                        if (!load(key, kvh, tile + t, base + t)) return false;
                    return true;
                };
                if (!loads(true, 0)) return false;
                for (int j = 0; j * step < n; ++j)
                    if (!loads(true, j + 1) || !loads(false, j)) return false;
                base += n;
                return true;
            });
            // Copies that are under way land before this CTA leaves: not only where this thread has given up, for those who would
            // wait for the last ones may have.
            auto land = [&](uint64_t* full, unsigned n) {
                for (unsigned g = n > kRing ? n - kRing : 0; g < n; ++g)
                    for (int i = 0; i < 1 << 20 && !mbar_try_wait(&full[g % kRing], g / kRing & 1); ++i) {}
            };
            land(b_k, keys);
            land(b_v, vals);
        }
        __syncwarp();
    } else if (warp >= 16) {
        // ---- the tensor core's queue, one warp for each stream ---------------------------------------------------------
        // (One warp for both was slower than the products.) The whole warp goes through the loops and one lane issues: operands
        // then lie in uniform registers, 22 cycles a product instead of 47 and more with one lane running all of it.
        {
            const bool leader = elect_one();
            constexpr uint32_t kShapeS = tc_shape(128, kKeyTile, kBf16, false), kShapeO = tc_shape(128, kHead, kBf16, true);
            const int s = warp - 16;
            auto same = [](uint32_t v) { return __shfl_sync(0xffffffffu, v, 0); };  // a value known to be that of the whole warp
            const uint32_t q_op = same(tc_operand_low(q_base + s * S::kQBytes, 16)), k_op = tc_operand_low(k_ring, 16), v_op = tc_operand_low(v_ring, S::kHalf);
            const uint32_t t_s = tmem + s * 128, t_o = same(tmem + 256 + s * 128);
            auto wait = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait_for(bar, parity, p.wait_cycles, &s_abort)) != 0; };
            unsigned base = 0;                // first tile of the segment
            unsigned asked = 0, added = 0;    // S tiles queued since the start, and P tiles used
            unsigned turn_q = 0;              // Q tiles taken
            for_segments([&](int, int block, int, int n) {
                const bool turns = runs.rows - block * kBlockRows <= kBlockRows / 2;
                const int step = turns ? 2 : 1;
                // Step j's key or value tiles. Each stream looks at every tile, and lets go at once of one that is the other's: who
                // skipped a tile could take an earlier phase of its barrier for a later one.
                auto scores = [&](int j) {
                    for (int t = j * step; t < min(n, (j + 1) * step); ++t) {
                        const unsigned g = base + t, slot = g % kRing;
                        if (!wait(&b_k[slot], g / kRing & 1)) return false;
                        if (turns && (t & 1) != s) {
                            if (leader) mbar_arrive(&b_s[s][slot]);
                            continue;
                        }
                        tc_fence_after();
                        const uint32_t k = same(k_op + slot * (S::kTileBytes >> 4)), to = same(t_s + (asked++ & 1) * 64);
                        if (leader) {
#pragma unroll
                            for (int i = 0; i < kHead / 16; ++i)
                                tc_mma_ss(to, tc_operand_at(q_op + (i / 4) * (S::kQHalf >> 4) + (i % 4) * 2),
                                          tc_operand_at(k + (i / 4) * (S::kHalf >> 4) + (i % 4) * 2), kShapeS, i > 0);
                            tc_commit(&b_s[s][slot]);
                        }
                        __syncwarp();
                    }
                    return true;
                };
                uint32_t add = 0;
                auto values = [&](int j) {
                    for (int t = j * step; t < min(n, (j + 1) * step); ++t) {
                        const unsigned g = base + t, slot = g % kRing;
                        if (!wait(&b_v[slot], g / kRing & 1)) return false;
                        if (turns && (t & 1) != s) {
                            if (leader) mbar_arrive(&b_o[s][slot]);
                            continue;
                        }
                        if (!wait(&b_p[s][added & 1], added >> 1 & 1)) return false;
                        tc_fence_after();
                        const uint32_t v = same(v_op + slot * (S::kTileBytes >> 4)), from = same(t_s + (added++ & 1) * 64), more = same(add);
                        if (leader) {
                            tc_mma_ts(t_o, from, tc_operand_at(v), kShapeO, more);
#pragma unroll
                            for (int k = 1; k < kKeyTile / 16 * (kWhole ? 2 : 1); ++k)
                                tc_mma_ts(t_o, from + k * 8, tc_operand_at(v + k % (kKeyTile / 16) * (2048 >> 4)), kShapeO, 1);
                            tc_commit(&b_o[s][slot]);
                        }
                        __syncwarp();
                        add = 1;
                    }
                    return true;
                };
                // a stream without tiles hands over no Q: it could be two phases ahead of this wait otherwise
                if (share(turns, n, s) && !wait(&b_q[s], turn_q++ & 1)) return false;
                if (!scores(0)) return false;
                // S of the next step goes where P of the one before lay: behind the product that reads it
                for (int j = 0; j * step < n; ++j)
                    if (!scores(j + 1) || !values(j)) return false;
                base += n;
                return true;
            });
            // products that are under way end before the TMEM is given back, whoever has given up
            if (leader) tc_commit(&b_end[s]);
            for (int i = 0; i < 1 << 20 && !mbar_try_wait(&b_end[s], 0); ++i) {}
        }
        __syncwarp();
    } else {
        // ---- softmax: half a row a thread, two warps for 32 rows -----------------------------------------------------------
        // These warps never leave early: after a wait that ran out they go through the rest without waiting and write nothing,
        // so that nobody is missed at the barriers of two warps.
        const int s = warp >> 3, half = (warp >> 2) & 1, quarter = warp & 3, row = quarter * 32 + lane, pair = 1 + s * 4 + quarter;
        const uint32_t lanes = (uint32_t)quarter << 21, t_o = tmem + 256 + s * 128 + half * (kHead / 2) + lanes;
        const uint32_t q_tile = q_base + s * S::kQBytes;
        // its sign goes into Q, so that the largest S is the largest score; so does a scale of 0 (masked keys have -inf to keep)
        const float scale = p.scale_log2 == 0.f ? 1.f : fabsf(p.scale_log2);
        const uint32_t sign = p.scale_log2 < 0.f ? 0x80008000u : 0u;
        const uint64_t scale2 = two(scale, scale), lower2 = two(kLower, kLower);
        unsigned used = 0;  // S tiles of this stream since the start
        bool dead = false;
        auto wait = [&](uint64_t* bar, uint32_t parity) {
            if (!dead) dead = !__all_sync(0xffffffffu, mbar_wait_for(bar, parity, p.wait_cycles, &s_abort));
        };
        unsigned base = 0;  // first tile of the segment
        // The stream's product with the values of tile g is done. Not asked for before the one of tile g - 4 is seen to be done, and
        // the slot is not used again before this: a block has more than eight tiles (kBlockPrefix), so that a stream has no tile only
        // in a run's first or last segment.
        auto o_done = [&](unsigned g) { wait(&b_o[s][g % kRing], g / kRing & 1); };
        for_segments([&](int kvh, int block, int tile, int n) {
            const bool turns = runs.rows - block * kBlockRows <= kBlockRows / 2;
            const int ns = share(turns, n, s);
            const int first_row = block * kBlockRows + (turns ? 0 : s * 128), rows = min(128, runs.rows - first_row);
            // this thread's row, and what lies before it in the queries and in the results; others ask for theirs by shuffle
            const int mrow = first_row + row, trow = mrow / p.group, hrow = kvh * p.group + mrow % p.group;
            const long long q_at = trow * p.q_stride + (long long)hrow * kHead, at_row = (long long)trow * p.n_heads + hrow;
            // this warp's 16 rows of Q, sixteen bytes a lane: what the stream's earlier products read is done with
            if (ns) {
                constexpr int kVec = kHead / 8, kLoads = kVec / 2;  // 16-byte vectors of a row; 16 rows of them are kVec / 2 a lane
                uint4 v[kLoads];
#pragma unroll
                for (int i = 0; i < kLoads; ++i) {
                    const int r = half * 16 + (i * 32 + lane) / kVec, c = lane % kVec;
                    const long long at = __shfl_sync(0xffffffffu, q_at, r);
                    v[i] = make_uint4(0, 0, 0, 0);
                    if (quarter * 32 + r < rows) v[i] = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.q) + at + c * 8);
                    if (p.scale_log2 == 0.f) v[i] = make_uint4(times_zero<T>(v[i].x), times_zero<T>(v[i].y), times_zero<T>(v[i].z), times_zero<T>(v[i].w));
                }
#pragma unroll
                for (int i = 0; i < kLoads; ++i) {
                    const int r = quarter * 32 + half * 16 + (i * 32 + lane) / kVec, c = lane % kVec;
                    const uint32_t to = q_tile + (c >> 3) * S::kQHalf + r * 128 + (((c & 7) ^ (r & 7)) << 4);
                    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(to), "r"(v[i].x ^ sign), "r"(v[i].y ^ sign), "r"(v[i].z ^ sign),
                                 "r"(v[i].w ^ sign)
                                 : "memory");
                }
                fence_async_shared();
                __syncwarp();
                if (lane == 0) mbar_arrive(&b_q[s]);
            }

            const bool busy = quarter * 32 < rows;  // warps without rows only keep step
            // Largest S so far but for kSlack - kLower, before the scale. S - m comes first: score * scale less a rounded m would be off
            // by half a step of m, which is no weight at all or an infinite one where scores are huge.
            float m = -INFINITY;
            uint64_t sum[2] = {0, 0};
            for (int j = 0; j < ns; ++j, ++used) {
                const unsigned g = base + (turns ? 2 * j + s : j);
                wait(&b_s[s][g % kRing], g / kRing & 1);
                tc_fence_after();
                if (busy) {
                    const uint32_t t_s = tmem + s * 128 + (used & 1) * 64 + lanes;
                    uint32_t x[32];
                    tmem_ld32(t_s + half * 32, x);
                    tmem_wait_ld();
                    const int left = p.prefix - (tile + (turns ? 2 * j + s : j)) * kKeyTile - half * 32;  // keys from these on
                    if (left < 32) {
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            if (e >= left) x[e] = 0xff800000u;
                    }
                    float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int e = 0; e < 32; e += 8)
#pragma unroll
                        for (int i = 0; i < 4; ++i) top[i] = fmaxf(fmaxf(top[i], __uint_as_float(x[e + 2 * i])), __uint_as_float(x[e + 2 * i + 1]));
                    float t = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
                    // both halves have their S in registers after this barrier, so P may go over it
                    if (pair_any(pair, (t - m) * scale > kSlack - kLower)) {
                        s_top[s][half][row] = t;
                        named_bar_sync(pair, 64);
                        t = fmaxf(t, s_top[s][half ^ 1][row]);
                        const bool move = (t - m) * scale > kSlack - kLower;
                        const float c = move ? exp2_fast((m - t) * scale) : 1.f;
                        m = move ? t : m;
                        const uint64_t c2 = two(c, c);
                        sum[0] = fma2(sum[0], c2, 0);
                        sum[1] = fma2(sum[1], c2, 0);
                        if (j > 0) {
                            // O is at rest between the product before (waited for here) and the one that waits for this P
                            o_done(g - (turns ? 2 : 1));
                            tc_fence_after();
#pragma unroll 1
                            for (int d = 0; d < kHead / 2; d += 32) {
                                uint32_t o[32];
                                tmem_ld32(t_o + d, o);
                                tmem_wait_ld();
#pragma unroll
                                for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * c);
                                tmem_st32(t_o + d, o);
                            }
                        }
                    }
                    const float ref = m == -INFINITY ? 0.f : -m;
                    const uint64_t ref2 = two(ref, ref);
                    uint32_t w[16], w2[kWhole ? 16 : 1];
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const float2 y = apart(fma2(add2((uint64_t)x[2 * e + 1] << 32 | x[2 * e], ref2), scale2, lower2));
                        const float a = exp2_fast(y.x), b = exp2_fast(y.y);
                        sum[e & 1] = add2(sum[e & 1], two(a, b));
                        w[e] = kWhole ? below2<T>(a, b) : pack2<T>(a, b);
                        if constexpr (kWhole) w2[e] = rest2<T>(w[e], a, b);
                    }
                    tmem_st16(t_s + half * 16, w);
                    if constexpr (kWhole) tmem_st16(t_s + 32 + half * 16, w2);
                    tmem_wait_st();
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&b_p[s][used & 1]);
            }

            // ---- the segment's result --------------------------------------------------------------------------------------
            int first, results;
            block_segments(runs, kvh, block, &first, &results);
            const int split = turns ? 2 * ((int)blockIdx.x - first) + s : (int)blockIdx.x - first;
            if (ns) {
                o_done(base + (turns ? 2 * (ns - 1) + s : ns - 1));
                tc_fence_after();
            }
            base += n;
            if (busy) {
                const long long results_at = (long long)split * total_rows * p.n_heads;
                const float2 l2 = apart(add2(sum[0], sum[1]));
                if (half) s_top[s][1][row] = l2.x + l2.y;
                named_bar_sync(pair, 64);
                if (!half && row < rows && !dead) p.pre_ml[results_at + at_row] = make_float2(m * scale - kLower, l2.x + l2.y + s_top[s][1][row]);
                named_bar_sync(pair, 64);
                if (ns) {
                    // through this warp's own 16 rows of the Q tile (others may have the next segment's rows in theirs), 16 dims
                    // at a time, so that rows leave in pieces of 64 bytes
                    const uint32_t mine = q_tile + quarter * 32 * 128 + half * 16 * 128;
#pragma unroll 1
                    for (int d = 0; d < kHead / 2; d += 16) {
                        uint32_t o[16];
                        tmem_ld16(t_o + d, o);
                        tmem_wait_ld();
#pragma unroll
                        for (int e = 0; e < 16; e += 4)
                            asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(mine + lane * 64 + (((e >> 2) ^ ((lane >> 1) & 3)) << 4)), "r"(o[e]),
                                         "r"(o[e + 1]), "r"(o[e + 2]), "r"(o[e + 3])
                                         : "memory");
                        __syncwarp();
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int r = i * 8 + (lane >> 2), c = lane & 3;
                            const long long at = __shfl_sync(0xffffffffu, at_row, r);
                            uint4 v;
                            asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                                         : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                                         : "r"(mine + r * 64 + ((c ^ ((r >> 1) & 3)) << 4))
                                         : "memory");
                            if (quarter * 32 + r < rows && !dead)
                                *reinterpret_cast<uint4*>(p.pre_o + (results_at + at) * kHead + half * (kHead / 2) + d + c * 4) = v;
                        }
                        __syncwarp();
                    }
                }
            }
            tc_fence_before();  // O has been read before the next segment's first product, which waits for this thread's P
            return true;
        });
    }
    __syncthreads();
    if (threadIdx.x == 0 && s_abort) report_input_error(p.status, kAttentionGaveUp, blockIdx.x);
    tc_fence_after();
    if (warp == 16) tmem_free(tmem, 512);
}

// Joins the partial results of one row and head: o = sum_s 2^(m_s - m) o_s / sum_s 2^(m_s - m) l_s. A block takes one row and
// some of its heads: the row's request is looked up once, the warps then go from head to head. (One warp for each row and head,
// all of them looking up: 50 us instead of 36 for 1229 rows of 32 heads, cold.)
constexpr int kJoinWarps = 8;
template <typename T, int kHead>
__global__ void __launch_bounds__(32 * kJoinWarps) attention_join_kernel(const __grid_constant__ AttnBatch p)
{
    constexpr int kPer = kHead / 32;
    __shared__ int s_row[6];  // first query row, queries, length, places before the request, before the prefix, of a run
    // what stood in these arrays before the call's first kernel is there already: that kernel has waited for it
    const int t = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (!p.run_ctas && !p.prefix_ctas) pdl_wait();
    const int total_rows = min(p.query_start[p.n_requests], p.n_rows);
    if (t >= total_rows) {
        pdl_wait();  // all the same: what follows in the stream follows this kernel
        return;
    }
    if (warp == 0) {
        // the request of this row: the lanes look at 32 places at a time
        int lo = 0;
        for (int n = p.n_requests; n > 1;) {
            const int step = (n + 31) >> 5, at = lo + lane * step;
            const unsigned below = __ballot_sync(0xffffffffu, lane * step < n && p.query_start[at] <= t);
            const int k = below ? 31 - __clz(below) : 0;
            lo += k * step;
            n = min(step, n - k * step);
        }
        const Span s = request_span(p, lo);
        if (!s.good && lane == 0) report_input_error(p.status, kInputLength, lo);
        bool own = p.run_ctas && s.good && t >= s.first && t < s.first + s.count;
        pdl_wait();
        if (lane == 0) {
            const int per = p.run_ctas ? p.run_base[p.n_requests + 1] : 1;
            own = own && per > 0;
            s_row[0] = s.first;
            s_row[1] = s.count;
            s_row[2] = own ? s.length : 0;
            s_row[3] = own ? p.run_base[lo] : 0;
            s_row[4] = p.run_ctas ? p.run_base[p.n_requests] : 0;
            s_row[5] = max(abs(per), 1);
        }
    }
    pdl_wait();  // the results, from here on
    __syncthreads();
    const int first_row = s_row[0], count = s_row[1], length = s_row[2], per = s_row[5];
    // what the heads have in common (integer divisions are most of this kernel's instructions)
    const PrefixRuns runs = p.prefix_ctas ? prefix_runs(total_rows, p.group, p.n_kv, p.prefix, p.prefix_ctas) : PrefixRuns{};
    const Share share = length > 0 ? request_share(p, count, length) : Share{0, 0, 0};
    int row_tile = -1, before = 0, here_places = 0, need = 0, rows16 = 0;  // of the row tile last seen
    for (int h = blockIdx.y * kJoinWarps + warp; h < p.n_heads; h += gridDim.y * kJoinWarps) {
        const long long id = (long long)t * p.n_heads + h;
        const int kvh = h / p.group, g = h - kvh * p.group;
        // results: of the prefix (by blocks: `step` apart; by runs), then of the own tokens
        long long pre_at = 0, pre_step = 0, own_at = 0;
        int pre = 0, own = 0;
        const float *pre_o = p.pre_o, *own_o = p.run_o;
        const float2 *pre_ml = p.pre_ml, *own_ml = p.run_ml;
        if (p.prefix_ctas) {
            int first;
            block_segments(runs, kvh, (t * p.group + g) / kBlockRows, &first, &pre);
            pre_at = id;
            pre_step = (long long)total_rows * p.n_heads;
        } else if (p.prefix) {
            const int m = t * p.group + g, row0 = m & ~15, rows = min(16, total_rows * p.group - row0), n = kOpen + (p.prefix + kTile - 1) / kTile;
            const int a = s_row[4] + ((row0 >> 4) * p.n_kv + kvh) * n, first = (a + kOpen) / per;
            pre = (a + n - 1) / per - first + 1;
            pre_at = result_row(p, true, 0, row0, rows, kvh, first) + (m & 15);
            pre_step = 16;
            pre_o = p.run_o;
            pre_ml = p.run_ml;
        }
        if (length > 0) {
            const int m = (t - first_row) * p.group + g, row0 = m & ~15;
            if (row0 >> 4 != row_tile) {
                row_tile = row0 >> 4;
                rows16 = min(16, count * p.group - row0);
                before = places_before(share, row_tile);
                here_places = places_before(share, row_tile + 1) - before;
                need = tiles_seen(p, count, length, row0, rows16);
            }
            const int a = s_row[3] + before * p.n_kv + kvh * here_places + kOpen, first = a / per;
            own = need ? (a + need - 1) / per - first + 1 : 0;
            own_at = result_row(p, false, first_row, row0, rows16, kvh, first) + (m & 15);
        }
        const int splits = pre + own;

        float m = -INFINITY, l = 0.f, acc[kPer] = {};
        for (int base = 0; base < splits; base += 32) {
            const int mine = base + lane;
            float2 ml = make_float2(-INFINITY, 0.f);
            if (mine < pre) ml = pre_ml[pre_at + mine * pre_step];
            else if (mine < splits) ml = own_ml[own_at + (mine - pre) * 16];
            const float mn = fmaxf(m, warp_max(ml.x)), to = mn == -INFINITY ? 0.f : mn;
            const float c = exp2_fast(m - to), w = exp2_fast(ml.x - to);
            l = l * c + warp_sum(ml.y * w);
#pragma unroll
            for (int e = 0; e < kPer; ++e) acc[e] *= c;
            m = mn;
            const int here = min(32, splits - base);
            for (int i = 0; i < here; i += 4) {  // four at a time are under way
                float v[4][kPer], wi[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int at = base + i + k;
                    wi[k] = __shfl_sync(0xffffffffu, w, (i + k) & 31);
                    if (i + k >= here) wi[k] = 0.f;
#pragma unroll
                    for (int e = 0; e < kPer; ++e) v[k][e] = 0.f;
                    if (wi[k] != 0.f) {
                        const float* o = (at < pre ? pre_o + (pre_at + at * pre_step) * kHead : own_o + (own_at + (at - pre) * 16ll) * kHead) + lane * kPer;
                        if constexpr (kPer == 4) {
                            const float4 x = *reinterpret_cast<const float4*>(o);
                            v[k][0] = x.x; v[k][1] = x.y; v[k][2] = x.z; v[k][3] = x.w;
                        } else {
                            const float2 x = *reinterpret_cast<const float2*>(o);
                            v[k][0] = x.x; v[k][1] = x.y;
                        }
                    }
                }
#pragma unroll
                for (int k = 0; k < 4; ++k)
#pragma unroll
                    for (int e = 0; e < kPer; ++e) acc[e] += wi[k] * v[k][e];
            }
        }
        const float inv = l == 0.f ? 0.f : 1.f / l;
        T* o = static_cast<T*>(p.out) + (long long)t * p.out_stride + (long long)h * kHead + lane * kPer;
        if constexpr (kPer == 4)
            *reinterpret_cast<uint2*>(o) = make_uint2(pack2<T>(acc[0] * inv, acc[1] * inv), pack2<T>(acc[2] * inv, acc[3] * inv));
        else
            *reinterpret_cast<uint32_t*>(o) = pack2<T>(acc[0] * inv, acc[1] * inv);
        if (p.lse && lane == 0) p.lse[id] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.69314718055994530942f;
    }
}

// Which kernels run, and the workspace's layout.
struct AttnPlan {
    int prefix_ctas, run_ctas;
    long long tiles;   // key tiles of either kernel, at most
    long long own_places;  // of the runs, without the prefix, at most
    size_t run_o, pre_ml, run_ml, run_base, bytes;  // offsets into the workspace (pre_o comes first), and its size
};
static AttnPlan plan_attention(const Ctx* ctx, int n_rows, int n_requests, int prefix, int max_length, int n_heads, int n_kv, int head)
{
    AttnPlan pl{};
    if (!n_rows) return pl;
    const int sms = std::max(1, ctx->sm_count);
    const long long rows = (long long)n_rows * (n_heads / n_kv);  // of a key head
    long long pre_rows = 0, run_rows = 0, run_tiles = (n_requests + rows / 16) * n_kv * (max_length ? kOpen + ceil_div(max_length, kTile) + 3 : 0);
    pl.own_places = run_tiles;
    if (prefix >= (rows <= 16 ? kBlockPrefixFewRows : kBlockPrefix)) {
        const long long blocks = (rows + kBlockRows - 1) / kBlockRows, key_tiles = ceil_div(prefix, kKeyTile);
        pl.tiles = blocks * n_kv * key_tiles;
        pl.prefix_ctas = (int)std::min<long long>(sms, pl.tiles);
        // Any number of rows up to n_rows may be there. With b blocks of a key head a CTA has at least n_kv b key_tiles / ctas
        // tiles, a block at most ctas / (n_kv b) + 2 segments and never more than key tiles, and a segment two results.
        pre_rows = std::min(512ll * pl.prefix_ctas + 1024ll * blocks * n_kv, 2 * key_tiles * n_rows * n_heads);
    } else {
        run_tiles += (rows + 15) / 16 * n_kv * (prefix ? kOpen + ceil_div(prefix, kTile) : 0);
    }
    pl.tiles = std::max(pl.tiles, run_tiles);
    pl.run_ctas = (int)std::min<long long>(2 * sms, (run_tiles + kAttnWarps - 1) / kAttnWarps);
    if (pl.run_ctas) run_rows = 2ll * n_rows * n_heads + 16ll * pl.run_ctas * kAttnWarps;
    pl.run_o = (size_t)pre_rows * head * sizeof(float);
    pl.pre_ml = pl.run_o + (size_t)run_rows * head * sizeof(float);
    pl.run_ml = pl.pre_ml + (size_t)pre_rows * sizeof(float2);
    pl.run_base = pl.run_ml + (size_t)run_rows * sizeof(float2);
    pl.bytes = pl.run_base + (pl.run_ctas ? (n_requests + 2) * sizeof(int) : 0);
    return pl;
}

// Tensor map of the prefix's keys or values: boxes of 64 columns and kKeyTile rows in 128-byte swizzle, rows behind the end
// read as zeros.
static bool make_map(CUtensorMap* map, int dtype, const void* base, long long row_stride, int columns, int rows)
{
    using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static const Encode encode = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult found;
        const cudaError_t e = cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &found);
        return e == cudaSuccess && found == cudaDriverEntryPointSuccess ? reinterpret_cast<Encode>(f) : nullptr;
    }();
    if (!encode) return false;
    const cuuint64_t size[2] = {(cuuint64_t)columns, (cuuint64_t)rows}, stride[1] = {(cuuint64_t)row_stride * 2};
    const cuuint32_t box[2] = {64, kKeyTile}, step[2] = {1, 1};
    return encode(map, dtype == ML2_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base), size, stride,
                  box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int kHead>
static cudaError_t launch_attention(Ctx* ctx, const AttnBatch& p, const AttnPlan& pl, const PrefixMaps& maps)
{
    bool& ready = ctx->attention_ready[std::is_same<T, __half>::value][kHead == 128];  // shared-memory limits are set once
    cudaError_t e = cudaSuccess;
    const auto whole = attention_prefix_kernel<T, kHead, true>, rounded = attention_prefix_kernel<T, kHead, false>;
    if (!ready) {
        e = cudaFuncSetAttribute(attention_runs_kernel<T, kHead>, cudaFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(whole, cudaFuncAttributeMaxDynamicSharedMemorySize, BlockSmem<kHead>::kBytes);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(rounded, cudaFuncAttributeMaxDynamicSharedMemorySize, BlockSmem<kHead>::kBytes);
        if (e != cudaSuccess) return e;
        ready = true;
    }
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.stream = ctx->stream;
    cfg.attrs = attr;
    cfg.numAttrs = ctx->pdl ? 1 : 0;
    if (pl.prefix_ctas) {
        cfg.gridDim = dim3(pl.prefix_ctas);
        cfg.blockDim = dim3(kBlockThreads);
        cfg.dynamicSmemBytes = BlockSmem<kHead>::kBytes;
        if ((e = cudaLaunchKernelEx(&cfg, p.n_rows * p.group <= kWholeRows ? whole : rounded, p, maps)) != cudaSuccess) return e;
        ++ctx->launches;
        cfg.numAttrs = 1;  // what follows starts as this kernel's CTAs leave
    }
    if (pl.run_ctas) {
        cfg.gridDim = dim3(pl.run_ctas);
        cfg.blockDim = dim3(kAttnThreads);
        cfg.dynamicSmemBytes = kAttnWarps * stages(kHead) * 2 * kTile * kHead * 2 + (p.n_requests + 2) * sizeof(int);
        if ((e = cudaLaunchKernelEx(&cfg, attention_runs_kernel<T, kHead>, p)) != cudaSuccess) return e;
        ++ctx->launches;
        cfg.numAttrs = 1;
    }
    cfg.gridDim = dim3((unsigned)p.n_rows, (unsigned)std::min(ceil_div(p.n_heads, kJoinWarps), std::max(1, 6 * ctx->sm_count / p.n_rows)));
    cfg.blockDim = dim3(32 * kJoinWarps);
    cfg.dynamicSmemBytes = 0;
    if ((e = cudaLaunchKernelEx(&cfg, attention_join_kernel<T, kHead>, p)) == cudaSuccess) ++ctx->launches;
    return e;
}

static int check_sizes(const char* what, int n_rows, int n_requests, int prefix, int max_length, int n_heads, int n_kv, int head_size)
{
    if (n_rows < 0 || n_requests < 1 || n_requests > kMaxRequests)
        return fail(ML2_E_INVALID, "%s: n_rows=%d n_requests=%d (1..%d)", what, n_rows, n_requests, kMaxRequests);
    constexpr int kMost = INT32_MAX - 63;  // whole tiles of keys stay below 2^31
    if (prefix < 0 || max_length < 0 || prefix > kMost || max_length > kMost)
        return fail(ML2_E_INVALID, "%s: prefix of %d rows, max_length=%d", what, prefix, max_length);
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
    *bytes = plan_attention(reinterpret_cast<Ctx*>(h), n_rows, n_requests, prefix_length, max_length, n_heads, n_kv_heads, head_size).bytes;
    return ML2_OK;
}

int ml2_prefix_attention(ml2_ctx* h, const ml2_prefix_attention_args* args)
{
    Ctx* ctx = reinterpret_cast<Ctx*>(h);
    if (!ctx || !args) return fail(ML2_E_INVALID, "prefix_attention: null argument");
    const auto [out, lse, query, prefix_key, prefix_value, key_cache, value_cache, table, lengths, query_start, workspace, workspace_bytes, out_stride,
                query_stride, prefix_stride, cache_stride, cache_rows, dtype, n_rows, n_requests, prefix_length, max_length, page_size, table_stride, n_heads,
                n_kv_heads, head_size, scale] = *args;
    if (dtype != ML2_F16 && dtype != ML2_BF16) return fail(ML2_E_INVALID, "prefix_attention: dtype=%d is neither ML2_F16 nor ML2_BF16", dtype);
    if (cache_rows < 1 || cache_rows > INT32_MAX) return fail(ML2_E_INVALID, "prefix_attention: the cache has %lld rows", cache_rows);
    if (int rc = check_sizes("prefix_attention", n_rows, n_requests, prefix_length, max_length, n_heads, n_kv_heads, head_size)) return rc;
    const int shift = page_shift(page_size);
    if (shift < 0) return fail(ML2_E_INVALID, "prefix_attention: page_size=%d must be a power of two, at most %d", page_size, kMaxPageSize);
    if (table_stride < 1 || (long long)table_stride * page_size > INT32_MAX)
        return fail(ML2_E_INVALID, "prefix_attention: table_stride=%d with page_size=%d", table_stride, page_size);
    if (max_length > table_stride * page_size)
        return fail(ML2_E_INVALID, "prefix_attention: max_length=%d passes the table's %d pages of %d", max_length, table_stride, page_size);
    constexpr float kLog2e = 1.44269504088896340736f;
    if (!std::isfinite(scale * kLog2e)) return fail(ML2_E_INVALID, "prefix_attention: scale=%g", (double)scale);
    if (n_rows == 0) return ML2_OK;
    if (!out || !query || !table || !lengths || !query_start || !key_cache || !value_cache || (prefix_length && (!prefix_key || !prefix_value)))
        return fail(ML2_E_INVALID, "prefix_attention: null argument");
    const long long q_width = (long long)n_heads * head_size, kv_width = (long long)n_kv_heads * head_size;
    if (out_stride < q_width || query_stride < q_width || cache_stride < kv_width || (prefix_length && prefix_stride < kv_width))
        return fail(ML2_E_INVALID, "prefix_attention: a row stride is shorter than the row");
    if ((out_stride | query_stride | cache_stride | prefix_stride) % 8 || !aligned_to(16, out, query, key_cache, value_cache) ||
        !aligned_to(16, prefix_key, prefix_value, workspace) || !aligned_to(4, lse, table, lengths, query_start))
        return fail(ML2_E_INVALID, "prefix_attention: pointers must be 16-byte aligned (lse and int arrays 4) and row strides multiples of 8 elements");
    if (cache_stride > INT32_MAX / 2 || prefix_stride > INT32_MAX / 2)
        return fail(ML2_E_INVALID, "prefix_attention: cache rows are further apart than 2^30 elements");
    const AttnPlan pl = plan_attention(ctx, n_rows, n_requests, prefix_length, max_length, n_heads, n_kv_heads, head_size);
    if (pl.tiles > INT32_MAX / 2 || (long long)n_rows * (n_heads / n_kv_heads) > INT32_MAX / 2 || (long long)n_rows * n_heads > INT32_MAX)
        return fail(ML2_E_INVALID, "prefix_attention: n_rows=%d with %d heads is too much for one call", n_rows, n_heads);
    if (workspace_bytes < pl.bytes || (pl.bytes && !workspace))
        return fail(ML2_E_INVALID, "prefix_attention: the workspace has %zu bytes, %zu are needed", workspace_bytes, pl.bytes);
    if (int rc = use_callers_stream(ctx)) return rc;
    AttnBatch p{};
    p.out = out; p.lse = lse; p.q = query; p.pk = prefix_key; p.pv = prefix_value; p.k = key_cache; p.v = value_cache;
    p.table = table; p.lengths = lengths; p.query_start = query_start; p.status = input_status(ctx);
    p.out_stride = out_stride; p.q_stride = query_stride; p.prefix_stride = prefix_stride; p.cache_stride = cache_stride;
    p.n_requests = n_requests; p.n_rows = n_rows; p.prefix = prefix_length; p.max_length = max_length; p.n_pages = (int)(cache_rows >> shift);
    p.table_stride = table_stride; p.page_shift = shift; p.n_heads = n_heads; p.n_kv = n_kv_heads; p.group = n_heads / n_kv_heads;
    p.scale_log2 = scale * kLog2e;
    char* ws = static_cast<char*>(workspace);
    p.pre_o = reinterpret_cast<float*>(ws); p.run_o = reinterpret_cast<float*>(ws + pl.run_o);
    p.pre_ml = reinterpret_cast<float2*>(ws + pl.pre_ml); p.run_ml = reinterpret_cast<float2*>(ws + pl.run_ml);
    p.run_base = reinterpret_cast<int*>(ws + pl.run_base);
    p.prefix_ctas = pl.prefix_ctas; p.run_ctas = pl.run_ctas; p.own_places = (int)pl.own_places;
    p.wait_cycles = ctx->wait_cycles;
    PrefixMaps maps{};
    auto make_maps = [&] {
        return make_map(&maps.k, dtype, prefix_key, prefix_stride, (int)kv_width, p.prefix) &&
               make_map(&maps.v, dtype, prefix_value, prefix_stride, (int)kv_width, p.prefix);
    };
    // The driver makes no map in a thread that has not used the device yet (the runtime's own calls bind it as they need it).
    if (pl.prefix_ctas && !make_maps() && (cudaSetDevice(ctx->device) != cudaSuccess || !make_maps()))
        return fail(ML2_E_CUDA, "prefix_attention: no tensor map for a prefix of %d rows of %lld, stride %lld", p.prefix, kv_width, prefix_stride);
    cudaError_t e;
    if (head_size == 128) e = dtype == ML2_F16 ? launch_attention<__half, 128>(ctx, p, pl, maps) : launch_attention<__nv_bfloat16, 128>(ctx, p, pl, maps);
    else e = dtype == ML2_F16 ? launch_attention<__half, 64>(ctx, p, pl, maps) : launch_attention<__nv_bfloat16, 64>(ctx, p, pl, maps);
    if (e != cudaSuccess) return fail(ML2_E_CUDA, "prefix_attention: %s", cudaGetErrorString(e));
    return ML2_OK;
}

}  // extern "C"
