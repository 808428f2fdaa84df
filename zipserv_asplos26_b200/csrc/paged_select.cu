// Bounds of complete pages in 8 bits (zs_page_bounds) and the choice of a
// sequence's pages by those bounds (zs_select_pages).
//
// Bounds, per page and KV head, from its keys k[t][d]: with
//   s    = 2^floor(log2 max |k|) / 64            (a power of two: dividing by it is exact)
//   up_d = ceil(max_t k[t][d] / s), lo_d = floor(min_t k[t][d] / s), within +-127
// so up_d * s and lo_d * s bound every key of the page but for the clamp.
//
// Score of a page for a query group of G heads sharing the KV head: with q
// rounded to whole numbers within +-127 by a power of two common to the group,
//   score = max_g sum_d (q_gd > 0 ? q_gd * up_d : q_gd * lo_d) * s.
// The sums are whole numbers below 2^24 for head dims up to 512 and s is a power
// of two, so a score is exact in fp32 in any order of summation and the choice
// is the same on every run and in every implementation. A page with a NaN or an
// infinity has s = inf and is chosen before all scored ones.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "paged.cuh"

namespace zs {
namespace {

// ------------------------------------------------------------------ bounds
// One warp reduces one page of one KV head: a lane holds 8 channels of every
// (32 / (D / 8))-th token, running maximum and minimum as packed 16-bit pairs
// (exact), 16-byte loads in full batches of eight. Bound by HBM: the keys are read
// once. A warp a CTA, so that an SM takes new pages a warp at a time: 12 thousand
// pages and heads of 16 KB (207 MB) in 33.4 us, 6.2 TB/s (35.7 with four warps).
constexpr int kBoundsThreads = 32;
constexpr int kBoundsBatch = 8;

struct BoundsArgs {
    PoolView kp;
    const int* table;
    long long table_stride;
    int B, width;
    int per_seq;       // tasks a sequence, or 0: tasks are the complete pages in order
    const int* before;
    const int* lens;
    int8_t* codes;     // [num_blocks][heads][2][D]
    float* scales;     // [num_blocks][heads]
    unsigned* err;
};

__device__ __forceinline__ uint32_t max2_nan(uint32_t a, uint32_t b, __nv_bfloat16) {
    const __nv_bfloat162 r = __hmax2_nan(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t min2_nan(uint32_t a, uint32_t b, __nv_bfloat16) {
    const __nv_bfloat162 r = __hmin2_nan(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t max2_nan(uint32_t a, uint32_t b, __half) {
    const __half2 r = __hmax2_nan(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t min2_nan(uint32_t a, uint32_t b, __half) {
    const __half2 r = __hmin2_nan(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
}

template <typename T, int D>
__global__ void __launch_bounds__(kBoundsThreads, 32) page_bounds_kernel(const BoundsArgs a) {
    constexpr int kLanes = D / 8;            // lanes a token
    constexpr int kRows = 32 / kLanes;       // tokens a pass
    const int lane = threadIdx.x & 31;
    const long long warp = (long long)blockIdx.x * (kBoundsThreads / 32) + (threadIdx.x >> 5);
    const int h = (int)(warp % a.kp.heads);
    const long long task = warp / a.kp.heads;
    const int sh = a.kp.page_shift;
    // pages [before / P, len / P) of a sequence became complete
    auto range = [&](int b, int& first) {
        first = max(a.before[b], 0) >> sh;
        return max(0, min(a.lens[b] >> sh, a.width) - first);
    };
    int b, p;
    if (a.per_seq) {                         // a rectangle of tasks
        b = (int)(task / a.per_seq);
        p = (int)(task % a.per_seq);
        if (b >= a.B) return;
        int first;
        if (p >= range(b, first)) return;
        p += first;
    } else {                                 // the complete pages in order: found by a prefix over the sequences
        const int per = (a.B + 31) / 32;
        long long mine = 0;
        int first;
        for (int i = 0; i < per; ++i)
            if (lane * per + i < a.B) mine += range(lane * per + i, first);
        long long inc = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long u = __shfl_up_sync(~0u, inc, o);
            if (lane >= o) inc += u;
        }
        const unsigned past = __ballot_sync(~0u, inc > task);
        if (!past) return;
        const int owner = __ffs(past) - 1;
        long long left = task - __shfl_sync(~0u, inc - mine, owner);
        for (b = owner * per;; ++b) {
            const int n = range(b, first);
            if (left < n) break;
            left -= n;
        }
        p = first + (int)left;
    }
    const int blk = a.table[b * a.table_stride + p];
    if (blk < 0 || blk >= a.kp.num_blocks) {
        if (lane == 0) set_err(a.err, kErrPagedIndex);
        return;
    }
    const int c = lane % kLanes, r0 = lane / kLanes;
    const uint16_t* base = static_cast<const uint16_t*>(a.kp.data) + blk * a.kp.s_block + h * a.kp.s_head + c * 8;
    // (-inf, +inf) pairs of the type
    const uint32_t ninf = std::is_same<T, __nv_bfloat16>::value ? 0xFF80FF80u : 0xFC00FC00u, pinf = ninf & 0x7FFF7FFFu;
    uint4 hi = make_uint4(ninf, ninf, ninf, ninf), lo = make_uint4(pinf, pinf, pinf, pinf);
    auto fold = [&](const uint4& x) {
        hi.x = max2_nan(hi.x, x.x, T()); hi.y = max2_nan(hi.y, x.y, T());
        hi.z = max2_nan(hi.z, x.z, T()); hi.w = max2_nan(hi.w, x.w, T());
        lo.x = min2_nan(lo.x, x.x, T()); lo.y = min2_nan(lo.y, x.y, T());
        lo.z = min2_nan(lo.z, x.z, T()); lo.w = min2_nan(lo.w, x.w, T());
    };
    // batches of loads in flight; a page is 4 passes (16 tokens of 64 channels) or a multiple of 8
    const int passes = (1 << sh) / kRows;
    const uint16_t* at = base + r0 * a.kp.s_token;
    const long long step = kRows * a.kp.s_token;
    if (passes < kBoundsBatch) {
#pragma unroll
        for (int i = 0; i < 4; ++i) fold(ld_stream16(at + i * step));
    } else {
        for (int i = 0; i < passes; i += kBoundsBatch) {
            uint4 x[kBoundsBatch];
#pragma unroll
            for (int j = 0; j < kBoundsBatch; ++j) x[j] = ld_stream16(at + (i + j) * step);
#pragma unroll
            for (int j = 0; j < kBoundsBatch; ++j) fold(x[j]);
        }
    }
#pragma unroll
    for (int o = kLanes; o < 32; o <<= 1) {
        hi.x = max2_nan(hi.x, __shfl_xor_sync(~0u, hi.x, o), T()); hi.y = max2_nan(hi.y, __shfl_xor_sync(~0u, hi.y, o), T());
        hi.z = max2_nan(hi.z, __shfl_xor_sync(~0u, hi.z, o), T()); hi.w = max2_nan(hi.w, __shfl_xor_sync(~0u, hi.w, o), T());
        lo.x = min2_nan(lo.x, __shfl_xor_sync(~0u, lo.x, o), T()); lo.y = min2_nan(lo.y, __shfl_xor_sync(~0u, lo.y, o), T());
        lo.z = min2_nan(lo.z, __shfl_xor_sync(~0u, lo.z, o), T()); lo.w = min2_nan(lo.w, __shfl_xor_sync(~0u, lo.w, o), T());
    }
    float up[8], dn[8];
    const uint32_t hw[4] = {hi.x, hi.y, hi.z, hi.w}, lw[4] = {lo.x, lo.y, lo.z, lo.w};
    uint32_t most = 0;       // bits of max |k|: unsigned order is magnitude order, NaN above infinity
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 u = unpack2<T>(hw[i]), w = unpack2<T>(lw[i]);
        up[2 * i] = u.x; up[2 * i + 1] = u.y;
        dn[2 * i] = w.x; dn[2 * i + 1] = w.y;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        most = max(most, max(__float_as_uint(up[i]) & 0x7FFFFFFFu, __float_as_uint(dn[i]) & 0x7FFFFFFFu));
    most = __reduce_max_sync(~0u, most);
    const bool finite = most < 0x7F800000u;
    const float power = __uint_as_float(most & 0x7F800000u);      // 2^floor(log2 max), 0 for zero and subnormals
    const bool live = finite && power > 0.f;
    const float s = finite ? power * 0.015625f : INFINITY;
    if (r0 == 0) {
        uint32_t cu[2] = {0, 0}, cl[2] = {0, 0};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float d = live ? s : 1.f;
            const int u = live ? max(-127, min(127, (int)ceilf(up[i] / d))) : 0;
            const int w = live ? max(-127, min(127, (int)floorf(dn[i] / d))) : 0;
            cu[i / 4] |= (uint32_t)(u & 0xFF) << (8 * (i % 4));
            cl[i / 4] |= (uint32_t)(w & 0xFF) << (8 * (i % 4));
        }
        int8_t* out = a.codes + ((long long)blk * a.kp.heads + h) * (2 * D) + c * 8;
        *reinterpret_cast<uint2*>(out) = make_uint2(cu[0], cu[1]);
        *reinterpret_cast<uint2*>(out + D) = make_uint2(cl[0], cl[1]);
    }
    if (lane == 0) a.scales[(long long)blk * a.kp.heads + h] = s;
}

// ------------------------------------------------------------------ choice
// A cluster of CTAs a (sequence, KV head): each scores its share of the pages and
// stores the scores, as order-preserving 32-bit keys, in the first CTA's shared
// memory; that one finds the K-th largest key by histograms over the range of the
// keys (1024 bins of it, then of the bin that holds the K-th, until a bin ends at
// the K-th or is one key wide) and writes the chosen pages in ascending order,
// ties to the lowest page. Scores are 8-bit matrix products (16 heads x 32 codes x
// 8 pages): a loop of 4-way dot products over the heads took 14 thousand cycles
// where the products take 7.5, which is what the codes take to arrive. Bound by
// HBM while scoring (2 D + 4 bytes a page and head), then by the latency of some
// ten barriers: 64 of up to 2049 pages for 64 (sequence, head) pairs, 26 MB, 12 us
// (4 of them the bytes); 48 of 513 pages for 8 pairs 5.7 us.
constexpr int kSelectThreads = 256;
constexpr int kSelectWarps = kSelectThreads / 32;
constexpr int kSelectMaxPages = 32768;
constexpr int kSelectMaxGroup = 128;
constexpr int kSelectBins = 1024;        // four a thread
constexpr int kSelectMaxCluster = 8;

struct SelectArgs {
    const uint16_t* q;       // [B][Hq][D]
    const int8_t* codes;
    const float* scales;
    const int* table;
    long long table_stride;
    const int* lens;
    int B, Hq, Hkv, width, page_shift, num_blocks, top, sinks, local;
    int* pages;              // [B][Hkv][top]
    int* counts;             // [B][Hkv]
    unsigned* err;
};

__device__ __forceinline__ uint32_t order_key(float f) {
    const uint32_t u = __float_as_uint(f + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ void st_cluster(uint32_t addr, uint32_t v) {
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}

__device__ __forceinline__ void red_cluster_min(uint32_t addr, uint32_t v) {
    asm volatile("red.relaxed.cluster.shared::cluster.min.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ void red_cluster_max(uint32_t addr, uint32_t v) {
    asm volatile("red.relaxed.cluster.shared::cluster.max.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}

__device__ __forceinline__ void mma_s8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, "
        "%3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Exclusive prefix of a 32-bit value over the block's threads.
__device__ __forceinline__ uint32_t select_scan(uint32_t v, uint32_t* part) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t u = __shfl_up_sync(~0u, inc, o);
        if (lane >= o) inc += u;
    }
    if (lane == 31) part[warp] = inc;
    __syncthreads();
    uint32_t w = lane < kSelectWarps ? part[lane] : 0;
#pragma unroll
    for (int o = 1; o < kSelectWarps; o <<= 1) {
        const uint32_t u = __shfl_up_sync(~0u, w, o);
        if (lane >= o) w += u;
    }
    const uint32_t before = __shfl_sync(~0u, w, warp ? warp - 1 : 0);
    return inc - v + (warp ? before : 0);
}

template <typename T, int D>
__global__ void __launch_bounds__(kSelectThreads, 2) select_kernel(const SelectArgs a, int cluster) {
    constexpr int kPieces = 2 * D / 16;              // 16-byte pieces of a page's codes
    constexpr int kLanes = 4;                        // lanes a page
    constexpr int kLoads = kPieces / kLanes;
    constexpr int kPages = 32 / kLanes;              // pages scored together
    constexpr int kGroups = D <= 128 ? 4 : 2;        // of them a warp pass, loads in flight together
    extern __shared__ uint4 select_smem[];
    __shared__ __align__(16) uint32_t s_hist[kSelectBins];
    __shared__ uint32_t s_part[2][kSelectWarps], s_pick[3], s_lo, s_hi;
    const int unit = blockIdx.x / cluster, rank = blockIdx.x % cluster;
    const int b = unit / a.Hkv, h = unit % a.Hkv;
    const int G = a.Hq / a.Hkv, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int sh = a.page_shift;
    grid_dep_launch();
    grid_dep_wait();
    const uint32_t* q = reinterpret_cast<const uint32_t*>(a.q + ((long long)b * a.Hq + (long long)h * G) * D);
    // q's largest magnitude, by every warp for itself, beside the length
    uint32_t most = 0;
#pragma unroll 4
    for (int i = lane; i < G * D / 2; i += 32) {
        const float2 f = unpack2<T>(q[i]);
        most = max(most, max(__float_as_uint(f.x) & 0x7FFFFFFFu, __float_as_uint(f.y) & 0x7FFFFFFFu));
    }
    const int len = max(0, min(a.lens[b], (int)min((long long)a.width << sh, (long long)INT_MAX)));
    const int n = (int)(((long long)len + (1 << sh) - 1) >> sh);
    int* out = a.pages + (long long)unit * a.top;
    if (rank == 0 && tid == 0) a.counts[unit] = min(n, a.top);
    if (n <= a.top) {                                // the same for the whole cluster
        for (int i = rank * kSelectThreads + tid; i < a.top; i += cluster * kSelectThreads) out[i] = i < n ? i : -1;
        return;
    }
    // This CTA's pages; a warp passes over `pass` of them at a time, few where
    // there are few. The blocks of the first pass are on their way during q's
    // rounding.
    const int share = (n + cluster - 1) / cluster;
    const int p_end = min(n, (rank + 1) * share);
    const int groups = min(kGroups, (share + kSelectWarps * kPages - 1) / (kSelectWarps * kPages));
    const int pass = groups * kPages;
    const int* row = a.table + b * a.table_stride;
    int p0 = rank * share + warp * pass;
    int blk = lane < pass && p0 + lane < p_end ? row[p0 + lane] : -1;
    int8_t* q8 = reinterpret_cast<int8_t*>(select_smem);              // [G][2 D]: positive part, negative part
    uint32_t* keys = reinterpret_cast<uint32_t*>(select_smem + G * kPieces);
    // No CTA writes into the first one's shared memory before that one has set this
    // up: waited for before the scores.
    if (tid == 0) {
        s_lo = 0xFFFFFFFFu;
        s_hi = 0;
    }
    if (tid < 3) keys[n + tid] = 0;                  // up to a multiple of four; no page's key is 0
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    // q to whole numbers
    most = __reduce_max_sync(~0u, most);
    const float step = __uint_as_float(most & 0x7F800000u) * 0.015625f;
    const bool live = most < 0x7F800000u && step > 0.f;
    for (int i = tid; i < G * D / 2; i += kSelectThreads) {
        const float2 f = unpack2<T>(q[i]);
        const int x = live ? max(-127, min(127, (int)rintf(f.x / step))) : 0;
        const int y = live ? max(-127, min(127, (int)rintf(f.y / step))) : 0;
        char2* at = reinterpret_cast<char2*>(q8 + (i / (D / 2)) * 2 * D + i % (D / 2) * 2);
        at[0] = make_char2((signed char)max(x, 0), (signed char)max(y, 0));
        at[D / 2] = make_char2((signed char)min(x, 0), (signed char)min(y, 0));
    }
    __syncthreads();
    const uint32_t keys0 = mapa_shared(smem_u32(keys), 0);
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    // scores, kLanes lanes a page
    const int sub = lane / kLanes, l4 = lane % kLanes;
    uint32_t lo = 0xFFFFFFFFu, hi = 0;               // range of the scored keys
    for (; p0 < p_end; p0 += kSelectWarps * pass) {
        const int p = p0 + lane;
        const bool mine = lane < pass && p < p_end;
        if (mine && (blk < 0 || blk >= a.num_blocks)) {
            set_err(a.err, kErrPagedIndex);
            blk = -1;
        }
        const long long at = blk >= 0 ? (long long)blk * a.Hkv + h : -1;
        const float s = at >= 0 ? a.scales[at] : 0.f;
        uint4 c[kGroups][kLoads];
#pragma unroll
        for (int j = 0; j < kGroups; ++j) {
            const long long from = __shfl_sync(~0u, at, (j * kPages + sub) & 31);
#pragma unroll
            for (int i = 0; i < kLoads; ++i)
                c[j][i] = j < groups && from >= 0 ? ld_nc16(a.codes + from * (2 * D) + (i * kLanes + l4) * 16)
                                                  : make_uint4(0, 0, 0, 0);
        }
        const int ahead = p0 + kSelectWarps * pass + lane;
        blk = lane < pass && ahead < p_end ? row[ahead] : -1;
        // Products of 8-bit matrices, 16 heads x 32 codes x 8 pages: as the order of
        // the codes does not matter, a lane's 16-byte pieces are used as they lie.
        int best = INT_MIN;
        for (int g0 = 0; g0 < G; g0 += 16) {
            int sum[kGroups][4];
#pragma unroll
            for (int j = 0; j < kGroups; ++j)
#pragma unroll
                for (int x = 0; x < 4; ++x) sum[j][x] = 0;
            const bool r0 = g0 + sub < G, r1 = g0 + sub + 8 < G;
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                const uint4 zero = make_uint4(0, 0, 0, 0);
                const uint4 w0 = r0 ? select_smem[(g0 + sub) * kPieces + i * kLanes + l4] : zero;
                const uint4 w1 = r1 ? select_smem[(g0 + sub + 8) * kPieces + i * kLanes + l4] : zero;
#pragma unroll
                for (int j = 0; j < kGroups; ++j) {
                    mma_s8(sum[j], w0.x, w1.x, w0.y, w1.y, c[j][i].x, c[j][i].y);
                    mma_s8(sum[j], w0.z, w1.z, w0.w, w1.w, c[j][i].z, c[j][i].w);
                }
            }
            // heads sub and sub + 8, pages 2 l4 and 2 l4 + 1 of each group
#pragma unroll
            for (int j = 0; j < kGroups; ++j) {
                int x = max(r0 ? sum[j][0] : INT_MIN, r1 ? sum[j][2] : INT_MIN);
                int y = max(r0 ? sum[j][1] : INT_MIN, r1 ? sum[j][3] : INT_MIN);
#pragma unroll
                for (int o = kLanes; o < 32; o <<= 1) {
                    x = max(x, __shfl_xor_sync(~0u, x, o));
                    y = max(y, __shfl_xor_sync(~0u, y, o));
                }
                // lane j * kPages + i keeps page i of group j
                const int from = (lane % kPages) / 2;
                const int gx = __shfl_sync(~0u, x, from), gy = __shfl_sync(~0u, y, from);
                if (lane / kPages == j) best = max(best, lane & 1 ? gy : gx);
            }
        }
        if (mine) {
            uint32_t key = 0xFFFFFFFFu;              // the first and last pages are chosen in any case
            if (p >= a.sinks && p < n - a.local) {
                key = order_key(s < INFINITY ? (float)best * s : INFINITY);
                lo = min(lo, key);
                hi = max(hi, key);
            }
            st_cluster(keys0 + p * 4, key);
        }
    }
    lo = __reduce_min_sync(~0u, lo);
    hi = __reduce_max_sync(~0u, hi);
    if (lane == 0 && hi) {
        red_cluster_min(mapa_shared(smem_u32(&s_lo), 0), lo);
        red_cluster_max(mapa_shared(smem_u32(&s_hi), 0), hi);
    }
    cluster_sync();
    if (rank) return;
    lo = s_lo;
    hi = s_hi;
    const uint4* keys4 = reinterpret_cast<const uint4*>(keys);
    const int n4 = (n + 3) / 4;
    // top < n and the forced pages are sinks + local <= top, all different, so
    // at least one page is scored and `want` of the scored ones are chosen
    uint32_t want = (uint32_t)(a.top - a.sinks - a.local);
    while (want && lo != hi) {
        const int shift = max(0, 22 - __clz(hi - lo));          // (hi - lo) >> shift is below 1024
        static_assert(kSelectBins == 4 * kSelectThreads, "four bins a thread");
        reinterpret_cast<uint4*>(s_hist)[tid] = make_uint4(0, 0, 0, 0);
        __syncthreads();
        auto count = [&](uint32_t k) {
            if (k >= lo && k <= hi) atomicAdd(&s_hist[(k - lo) >> shift], 1u);
        };
        for (int i = tid; i < n4; i += kSelectThreads) {
            const uint4 k = keys4[i];
            count(k.x);
            count(k.y);
            count(k.z);
            count(k.w);
        }
        __syncthreads();
        // thread t looks at four bins, from kSelectBins - 1 - 4 t down
        const uint4 bins = reinterpret_cast<const uint4*>(s_hist)[kSelectThreads - 1 - tid];
        uint32_t above = select_scan(bins.x + bins.y + bins.z + bins.w, s_part[0]);
        const uint32_t held[4] = {bins.w, bins.z, bins.y, bins.x};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (above < want && above + held[i] >= want) {
                s_pick[0] = kSelectBins - 1 - 4 * tid - i;
                s_pick[1] = want - above;
                s_pick[2] = held[i];
            }
            above += held[i];
        }
        __syncthreads();
        const uint32_t from = lo + (s_pick[0] << shift);
        want = s_pick[1];
        if (want == s_pick[2]) {        // the whole bin is chosen: everything from its start on
            lo = from - 1;
            want = 0;
            break;
        }
        hi = min(hi, from + ((1u << shift) - 1));
        lo = from;
        __syncthreads();                // before the bins and the pick are written again
    }
    // keys above lo are in; of its equals the first `want` pages
    if (a.top == a.sinks + a.local) lo = 0xFFFFFFFEu;
    const int per = (n4 + kSelectThreads - 1) / kSelectThreads;
    const int i0 = min(n4, tid * per), i1 = min(n4, i0 + per);
    uint32_t above = 0, equal = 0;
    for (int i = i0; i < i1; ++i) {
        const uint4 k = keys4[i];
        above += (k.x > lo) + (k.y > lo) + (k.z > lo) + (k.w > lo);
        equal += (k.x == lo) + (k.y == lo) + (k.z == lo) + (k.w == lo);
    }
    const uint32_t before = select_scan(above << 16 | equal, s_part[1]);
    uint32_t at_above = before >> 16, at_equal = before & 0xFFFFu;
    auto emit = [&](uint32_t k, int i) {
        const bool gt = k > lo, eq = k == lo;
        if (gt || (eq && at_equal < want)) out[at_above + min(at_equal, want)] = i;
        at_above += gt;
        at_equal += eq;
    };
    for (int i = i0; i < i1; ++i) {
        const uint4 k = keys4[i];
        emit(k.x, 4 * i);
        emit(k.y, 4 * i + 1);
        emit(k.z, 4 * i + 2);
        emit(k.w, 4 * i + 3);
    }
}

template <typename T>
cudaError_t launch_select(const SelectArgs& a, int D, cudaStream_t s) {
    const int G = a.Hq / a.Hkv;
    const size_t smem = (size_t)G * 2 * D + sizeof(uint32_t) * ((size_t)a.width + 3);
    // CTAs a (sequence, KV head): as many as the GPU holds at once (two an SM), while
    // each still has 64 pages for its eight warps
    int cluster = 1;
    while (cluster < kSelectMaxCluster && (long long)a.B * a.Hkv * cluster * 2 <= 296 && a.width / (2 * cluster) >= 64) cluster *= 2;
    if ((long long)a.B * a.Hkv * cluster > INT32_MAX) return cudaErrorInvalidValue;
    auto go = [&](auto kernel) -> cudaError_t {
        if (smem > 40 * 1024) {    // the same limit every time: threads may call with different sizes
            const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                       kSelectMaxGroup * 2 * D + 4 * (kSelectMaxPages + 3));
            if (e != cudaSuccess) return e;
        }
        cudaLaunchConfig_t cfg;
        cudaLaunchAttribute attr[2];
        pdl_config(&cfg, attr, dim3((unsigned)(a.B * a.Hkv * cluster)), dim3(kSelectThreads), smem, s);
        attr[1].id = cudaLaunchAttributeClusterDimension;
        attr[1].val.clusterDim.x = cluster;
        attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
        cfg.numAttrs = 2;
        return cudaLaunchKernelEx(&cfg, kernel, a, cluster);
    };
    switch (D) {
        case 64: return go(select_kernel<T, 64>);
        case 128: return go(select_kernel<T, 128>);
        case 256: return go(select_kernel<T, 256>);
    }
    return cudaErrorInvalidValue;
}

}  // namespace
}  // namespace zs

extern "C" int zs_page_bounds(const ZsPageBounds* p) {
    using namespace zs;
    BoundsArgs a{};
    if (!p || !make_pool(&p->k_pool, &a.kp) || p->B < 0 || p->width <= 0 || p->table_stride < p->width ||
        p->max_new < 0 || p->max_total < 0)
        return cudaErrorInvalidValue;
    if (a.kp.dim != 64 && a.kp.dim != 128 && a.kp.dim != 256) return cudaErrorInvalidValue;
    if (p->B == 0 || p->max_new == 0) return cudaSuccess;
    if (!p->block_table || !p->lens_before || !p->seq_lens || !p->codes || !p->scales || !aligned16p(p->codes))
        return cudaErrorInvalidValue;
    const int B = p->B;
    a.table = p->block_table;
    a.table_stride = p->table_stride;
    a.B = B;
    a.width = p->width;
    // max_new tokens complete at most this many pages of a sequence; max_total
    // tokens in all at most one a sequence more than their pages. The second
    // bound is the smaller one where a few of many sequences got a prompt: then
    // each warp looks its page up.
    const int page = 1 << a.kp.page_shift;
    const long long per_seq = std::min<long long>(p->width, ((long long)p->max_new + page - 1) / page);
    long long tasks = per_seq * B;
    a.per_seq = (int)per_seq;
    if (p->max_total > 0 && p->max_total / page + B < tasks / 2) {
        tasks = p->max_total / page + B;
        a.per_seq = 0;
    }
    a.before = p->lens_before;
    a.lens = p->seq_lens;
    a.codes = p->codes;
    a.scales = p->scales;
    a.err = p->err;
    const long long warps = tasks * a.kp.heads;
    const long long grid = (warps + kBoundsThreads / 32 - 1) / (kBoundsThreads / 32);
    if (grid > INT32_MAX) return cudaErrorInvalidValue;
    cudaStream_t s = (cudaStream_t)p->stream;
    const bool bf = p->k_pool.dtype == ZS_BF16;
    switch (a.kp.dim) {
        case 64:
            if (bf) page_bounds_kernel<__nv_bfloat16, 64><<<(unsigned)grid, kBoundsThreads, 0, s>>>(a);
            else page_bounds_kernel<__half, 64><<<(unsigned)grid, kBoundsThreads, 0, s>>>(a);
            break;
        case 128:
            if (bf) page_bounds_kernel<__nv_bfloat16, 128><<<(unsigned)grid, kBoundsThreads, 0, s>>>(a);
            else page_bounds_kernel<__half, 128><<<(unsigned)grid, kBoundsThreads, 0, s>>>(a);
            break;
        case 256:
            if (bf) page_bounds_kernel<__nv_bfloat16, 256><<<(unsigned)grid, kBoundsThreads, 0, s>>>(a);
            else page_bounds_kernel<__half, 256><<<(unsigned)grid, kBoundsThreads, 0, s>>>(a);
            break;
        default: return cudaErrorInvalidValue;
    }
    return cudaGetLastError();
}

extern "C" int zs_select_pages(const ZsSelectPages* p) {
    using namespace zs;
    if (!p) return cudaErrorInvalidValue;
    const int B = p->B, Hq = p->Hq, Hkv = p->Hkv, page_size = p->page_size;
    if (B < 0 || Hkv <= 0 || Hq <= 0 || Hq % Hkv || Hq / Hkv > kSelectMaxGroup || p->width <= 0 ||
        p->width > kSelectMaxPages || p->table_stride < p->width || p->num_blocks <= 0)
        return cudaErrorInvalidValue;
    if (page_size < 16 || page_size > 256 || (page_size & (page_size - 1))) return cudaErrorInvalidValue;
    if (p->sinks < 0 || p->local < 1 || p->top < (long long)p->sinks + p->local ||
        (p->dtype != ZS_BF16 && p->dtype != ZS_FP16) || (p->D != 64 && p->D != 128 && p->D != 256))
        return cudaErrorInvalidValue;
    if ((long long)B * Hkv > INT32_MAX) return cudaErrorInvalidValue;
    if (B == 0) return cudaSuccess;
    if (!p->q || !p->codes || !p->scales || !p->block_table || !p->seq_lens || !p->pages || !p->counts ||
        !aligned16p(p->codes) || !aligned16p(p->q))
        return cudaErrorInvalidValue;
    SelectArgs a{p->q, p->codes, p->scales, p->block_table, p->table_stride, p->seq_lens, B, Hq, Hkv, p->width, 0,
                 p->num_blocks, p->top, p->sinks, p->local, p->pages, p->counts, p->err};
    while ((1 << a.page_shift) < page_size) ++a.page_shift;
    return p->dtype == ZS_BF16 ? launch_select<__nv_bfloat16>(a, p->D, (cudaStream_t)p->stream)
                               : launch_select<__half>(a, p->D, (cudaStream_t)p->stream);
}
