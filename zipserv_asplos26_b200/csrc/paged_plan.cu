// Step plan of a paged KV cache: block tables, slots and positions from request
// lengths, on the GPU (zs_plan_step).
//
// With page size P, request r of length len[r] gets new[r] tokens (negative: it
// has ended). In request order:
//   back[r]  = pages of an ended request, appended to the free list
//   fits[r]  = its tokens fit the step's room, its pages the table's width, and
//              its new pages the free list (by inclusive prefix sums)
//   need[r]  = ceil((len + new) / P) - ceil(len / P) where it fits
//   page j of the step (exclusive prefix of need) = free[have - 1 - j]
//   token t of the step: request by the prefix sums of the admitted tokens,
//   position len + rank, slot = table[r][pos / P] * P + pos % P.
//
// What bounds it: nothing but latency (16 bytes a token; 131 thousand tokens
// are 2 MB, 0.3 us of HBM). So it is one launch: every CTA repeats the three
// prefix sums over the requests in shared memory, each thread holding a
// contiguous run of them (three block scans whatever the request count), and
// then writes its share of the tokens, table entries and free-list entries by
// binary search in the prefix sums. No CTA reads what another writes: inputs
// `lens` and `count` are not updated in place, taken pages are looked up by
// formula and not in the table, and a taken page that was given back in the
// same step is found in the ended request's row and not in the free list.
//
// Measured: 3 requests 3.4 us, 256 requests with 16 thousand tokens 5.3, 37
// prompts of 131 thousand tokens in all 4.9, of which an empty launch is some 2.
#include <algorithm>

#include "paged.cuh"

namespace zs {
namespace {

constexpr int kPlanThreads = 512;
constexpr int kPlanWarps = kPlanThreads / 32;
constexpr int kPlanMaxRequests = 8192;

struct PlanArgs {
    int* table;
    long long table_stride;
    int R, width, page_shift, max_tokens, capacity;
    const int* lens;
    const int* fresh;
    int* free_list;
    const int* count;
    int* out_lens;
    int* out_count;
    int* out_cu;
    long long* slots;
    int* token_seq;
    int* positions;
    uint8_t* refused;
    unsigned* err;
};

// Exclusive prefixes of N values over the block's threads, their sums in total.
// `part` is this scan's own N * kPlanWarps entries of shared memory.
template <int N>
__device__ __forceinline__ void block_scan(long long (&v)[N], long long* part, long long (&total)[N]) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    long long inc[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        inc[i] = v[i];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long u = __shfl_up_sync(~0u, inc[i], o);
            if (lane >= o) inc[i] += u;
        }
        if (lane == 31) part[i * kPlanWarps + warp] = inc[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
        long long w = lane < kPlanWarps ? part[i * kPlanWarps + lane] : 0;
#pragma unroll
        for (int o = 1; o < kPlanWarps; o <<= 1) {
            const long long u = __shfl_up_sync(~0u, w, o);
            if (lane >= o) w += u;
        }
        const long long before = __shfl_sync(~0u, w, warp ? warp - 1 : 0);
        total[i] = __shfl_sync(~0u, w, kPlanWarps - 1);
        v[i] = inc[i] - v[i] + (warp ? before : 0);
    }
}

// Largest r in [0, n) with pre[r] <= x (pre ascending, pre[0] == 0).
__device__ __forceinline__ int owner(const int* pre, int n, int x) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (pre[mid] <= x) lo = mid; else hi = mid;
    }
    return lo;
}

__global__ void __launch_bounds__(kPlanThreads) plan_kernel(const PlanArgs a) {
    extern __shared__ int plan_smem[];
    __shared__ long long parts[4 * kPlanWarps];
    __shared__ int s_taken;            // pages taken by the step
    const int R = a.R, sh = a.page_shift, P1 = (1 << sh) - 1;
    int* cu = plan_smem;               // [R + 1] admitted tokens before request r
    int* back0 = cu + R + 1;           // [R + 1] pages given back before request r
    int* need0 = back0 + R + 1;        // [R] pages taken before request r
    int* lens = need0 + R;             // [R] lengths before the step
    int* fresh = lens + R;             // [R] tokens asked for, negative: ended
    const int count_in = *a.count;
    // what a row of the table holds, and a position can be
    const int len_cap = (int)min((long long)a.width << sh, (long long)INT_MAX - P1);
    for (int r = threadIdx.x; r < R; r += kPlanThreads) {
        lens[r] = max(0, min(a.lens[r], len_cap));
        fresh[r] = a.fresh[r];
    }
    if (threadIdx.x == 0) s_taken = 0;
    __syncthreads();
    const int per = (R + kPlanThreads - 1) / kPlanThreads;
    const int r0 = min(R, (int)threadIdx.x * per), r1 = min(R, r0 + per);
    // 1. pages given back, tokens asked for
    long long first_sums[2] = {0, 0}, first_totals[2];
    for (int r = r0; r < r1; ++r) {
        if (fresh[r] < 0) first_sums[0] += (lens[r] + P1) >> sh;
        else first_sums[1] += fresh[r];
    }
    block_scan(first_sums, parts, first_totals);
    long long back = first_sums[0];
    const long long want = first_sums[1], back_total = first_totals[0];
    const int count0 = max(0, min(count_in, a.capacity));
    const long long have = min((long long)count0 + back_total, (long long)a.capacity);
    // 2. pages needed by the requests that fit the step and the table
    auto pages_needed = [&](int r, long long want_end) -> int {
        const int f = fresh[r], len = lens[r];
        const long long end = (long long)len + max(f, 0);
        if (f < 0 || want_end > a.max_tokens || end > len_cap) return -1;
        return (int)(((end + P1) >> sh) - ((len + P1) >> sh));
    };
    long long need[1] = {0}, need_total[1];
    long long w = want;
    for (int r = r0; r < r1; ++r) {
        w += max(fresh[r], 0);
        need[0] += max(pages_needed(r, w), 0);
    }
    block_scan(need, parts + 2 * kPlanWarps, need_total);
    // 3. admitted tokens
    long long got_sum[1] = {0}, got_total[1];
    w = want;
    long long n = need[0];
    for (int r = r0; r < r1; ++r) {
        const int f = fresh[r];
        w += max(f, 0);
        const int p = pages_needed(r, w);
        n += max(p, 0);
        if (p == 0 || (p > 0 && n <= have)) got_sum[0] += f;
    }
    block_scan(got_sum, parts + 3 * kPlanWarps, got_total);
    long long got = got_sum[0];
    w = want;
    n = need[0];
    const bool first = blockIdx.x == 0;
    bool any_refused = false;
    int end = 0;
    for (int r = r0; r < r1; ++r) {
        const int f = fresh[r], len = lens[r];
        w += max(f, 0);
        const int p = pages_needed(r, w);
        const bool ok = p == 0 || (p > 0 && n + p <= have);
        cu[r] = (int)got;
        need0[r] = (int)min(n, have);       // exact for every admitted request that takes pages
        back0[r] = (int)back;
        if (first) {
            a.out_lens[r] = f < 0 ? 0 : len + (ok ? f : 0);
            a.out_cu[r] = (int)got;
            a.refused[r] = !ok && f > 0;
        }
        any_refused |= !ok && f > 0;
        n += max(p, 0);
        if (ok && p > 0) end = (int)n;
        if (ok) got += f;
        if (f < 0) back += (len + P1) >> sh;
    }
    // Admission is by inclusive prefix, so the requests refused for want of
    // pages are the last ones that need any: the pages taken end where the last
    // admitted request's do.
    if (end) atomicMax(&s_taken, end);
    if (threadIdx.x == 0) {
        cu[R] = (int)got_total[0];
        back0[R] = (int)back_total;
    }
    if (first && any_refused) set_err(a.err, kErrPagedFull);
    __syncthreads();
    const int used = s_taken;
    if (first && threadIdx.x == 0) {
        a.out_cu[R] = cu[R];
        *a.out_count = (int)have - used;
        if (count_in != count0 || back_total + count0 > a.capacity) set_err(a.err, kErrPagedIndex);
    }

    // the page at position x of the free list once the ended requests' pages are on it
    auto free_page = [&](int x) -> int {
        if (x < count0) return a.free_list[x];
        const int b = x - count0;
        const int r = owner(back0, R, b);
        return a.table[(long long)r * a.table_stride + (b - back0[r])];
    };
    // One index space for the pages given back (the free list has room for every
    // page of the pool), the new table entries and the tokens, so that their
    // lookups are in flight together. The pool's size is not known here: a page
    // below 0 (one that a table or the free list does not have) is flagged, and its
    // tokens get no slot; the rotary write flags slots past the pool.
    const int nback = (int)(have - count0), tokens = cu[R];
    const long long items = (long long)nback + used + a.max_tokens;
    bool bad = false;
    for (long long i = blockIdx.x * kPlanThreads + threadIdx.x; i < items; i += gridDim.x * kPlanThreads) {
        if (i < nback) {
            const int blk = free_page(count0 + (int)i);
            bad |= blk < 0;
            a.free_list[count0 + i] = blk;
        } else if (i < nback + (long long)used) {
            const int j = (int)(i - nback), r = owner(need0, R, j);
            const int col = ((lens[r] + P1) >> sh) + (j - need0[r]);
            const int blk = free_page((int)have - 1 - j);
            bad |= blk < 0;
            a.table[(long long)r * a.table_stride + col] = blk;
        } else {
            const int t = (int)(i - nback - used);
            long long slot = -1;
            int r = -1, pos = 0;
            if (t < tokens) {
                r = owner(cu, R, t);
                const int len = lens[r];
                pos = len + (t - cu[r]);
                const int col = pos >> sh, old = (len + P1) >> sh;
                const int blk = col < old ? a.table[(long long)r * a.table_stride + col]
                                          : free_page((int)have - 1 - (need0[r] + col - old));
                bad |= blk < 0;
                slot = blk < 0 ? -1 : ((long long)blk << sh) + (pos & P1);
            }
            a.slots[t] = slot;
            a.token_seq[t] = r;
            a.positions[t] = pos;
        }
    }
    if (bad) set_err(a.err, kErrPagedIndex);
}

}  // namespace
}  // namespace zs

extern "C" int zs_plan_step(const ZsPlanStep* p) {
    using namespace zs;
    if (!p || p->R <= 0 || p->R > kPlanMaxRequests || p->width <= 0 || p->capacity <= 0 || p->max_tokens < 0 ||
        p->max_tokens > (1 << 30))
        return cudaErrorInvalidValue;
    const int R = p->R, page_size = p->page_size, max_tokens = p->max_tokens;
    if ((int64_t)R * p->width > INT32_MAX || p->table_stride < p->width) return cudaErrorInvalidValue;
    if (page_size < 16 || page_size > 256 || (page_size & (page_size - 1))) return cudaErrorInvalidValue;
    if (!p->block_table || !p->seq_lens || !p->new_lens || !p->free_blocks || !p->free_count || !p->out_lens ||
        !p->out_count || !p->out_cu || !p->refused || (max_tokens && (!p->slots || !p->token_seq || !p->positions)))
        return cudaErrorInvalidValue;
    // every CTA repeats the prefix sums from these; the outputs are other buffers
    if (p->out_lens == p->seq_lens || p->out_lens == p->new_lens || p->out_count == p->free_count)
        return cudaErrorInvalidValue;
    PlanArgs a{p->block_table, p->table_stride, R, p->width, 0, max_tokens, p->capacity, p->seq_lens, p->new_lens,
               p->free_blocks, p->free_count, p->out_lens, p->out_count, p->out_cu,
               reinterpret_cast<long long*>(p->slots), p->token_seq, p->positions, p->refused, p->err};
    while ((1 << a.page_shift) < page_size) ++a.page_shift;
    const size_t smem = sizeof(int) * (5 * (size_t)R + 2);
    if (smem > 40 * 1024) {    // the same limit every time: threads may call with different sizes
        const cudaError_t e = cudaFuncSetAttribute(plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                   (int)sizeof(int) * (5 * kPlanMaxRequests + 2));
        if (e != cudaSuccess) return e;
    }
    // a thread a token, with some more for pages
    const long long items = max_tokens + ((long long)max_tokens >> a.page_shift) + 2ll * R;
    const int grid = (int)std::min(148ll, (items + kPlanThreads - 1) / kPlanThreads);
    plan_kernel<<<grid, kPlanThreads, smem, (cudaStream_t)p->stream>>>(a);
    return cudaGetLastError();
}

// The argument structs' sizes, as bindings pack them.
static_assert(sizeof(ZsPagePool) == 56 && sizeof(ZsPlanStep) == 144 && sizeof(ZsRopeWrite) == 280 &&
                  sizeof(ZsPagedAttention) == 232 && sizeof(ZsPageBounds) == 136 && sizeof(ZsSelectPages) == 128,
              "argument struct layout");
