// One token per row of logits from a given random number (zs_sample).
//
// With x the row, T its temperature, w_i = exp((x_i - max x) / T) and the tokens in the
// order of x, largest first and equal ones by index:
//   top_k   keeps the first top_k tokens,
//   top_p   of these the shortest beginning whose weights reach top_p of theirs,
//   min_p   the tokens with w_i >= min_p,
// each a beginning of that order, so the shortest one is what is kept: all tokens whose x
// is above a border, and the first few (by index) of those on it. The token is the first,
// by index, at which the running sum of the kept weights passes u times their sum.
//
// A token must not depend on the order of sums, so weights are whole numbers, rounded from
// 64-bit floats to steps of 2^-S of the largest (S = 62 - log2 of the vocabulary's size,
// 50 at most): every sum is exact, and products with top_p and u are taken in 128 bits.
// Of the weights themselves 2^-49 is lost in 2^(-t): t's nearest multiple of 1 / 2048 from
// a table, the rest by a polynomial of degree three.
//
// Borders are found by the logits' order, its first 12 bits first: a histogram in shared
// memory of how many, or how much weight, the tokens hold. The next reading, where there is
// one border, sums the weights above its 4096th part of the order, for each block of 1024
// tokens, and gathers the tokens in it; their next 12 and 8 bits find the border. With two
// borders it gathers all tokens from the first one's part on; up to 4096 of them are all that
// remains to be looked at, up to 512 each against all others. Where more are gathered,
// further readings find the other bits, and the sums. In the end the block in which the
// running sum passes its target is read once more. All readings but the first come from L2. A row goes to a cluster of up to 8 CTAs
// where there are few, its histograms joined through distributed shared memory. Bound by
// instructions: some 30 for a weight, 10 of them in 64 bits.
//
// Measured: 256 rows of 131071 in fp32, nuclei of tens of thousands of tokens (two weights
// for each) 246 us, 134 instructions a logit issued in 56% of the cycles, HBM read once; 64
// rows of 128000 in bf16 with settings of their own 62; 3 of 32000 with top_k = 50 and top_p
// = 0.95 19, a chain of some ten steps between barriers, 500 to 5000 cycles each.
#include <algorithm>
#include <atomic>
#include <cfloat>
#include <climits>
#include <cmath>
#include <type_traits>

#include "paged.cuh"

namespace zs {
namespace {

constexpr int kSampThreads = 512;
constexpr int kSampWarps = kSampThreads / 32;
constexpr int kSampBlock = 1024;            // tokens of a sum
constexpr int kSampMaxBlocks = 1024;        // so 2^20 tokens at most
constexpr int kBins = 4096;
constexpr int kPowers = 2048;
constexpr int kList = 4096;                 // gathered tokens of a CTA, at most
constexpr int kFew = kSampThreads;          // of a row, so few that each is held against all others
constexpr unsigned kErrSampleNothing = 8u;  // a row had nothing to choose from
constexpr unsigned kOrderOfMost = 0xFF7FFFFFu, kOrderOfMinusInf = 0x007FFFFFu;     // of the largest finite number
using u64 = unsigned long long;

struct SampArgs {
    const void* logits;
    long long stride;
    const float* u;
    const float* temperature;     // nullable, as the next three: else the value for all rows
    const int* top_k;
    const float* top_p;
    const float* min_p;
    double temperature1, top_p1, min_p1;
    int top_k1;
    long long* out;
    unsigned* err;
    int V, blocks, steps;         // blocks a CTA; S
};

struct SampShared {
    double powers[kPowers];                 // 2^(-j / 2048)
    union {
        unsigned count[kBins];
        struct {
            unsigned lo[kBins], hi[kBins];
        };
        ulonglong2 few[kSampThreads];       // a few gathered tokens: place in the order, weight
    };
    u64 mass[kSampMaxBlocks];               // of the CTA's blocks (the row's, from a list): weights above the border
    unsigned ties[kSampMaxBlocks];          // and tokens on it
    unsigned list_key[kList];
    int list_at[kList];
    int listed;                             // tokens that the CTA gathered, more than kList where they did not fit
    u64 part[kSampWarps], part2[kSampWarps];
    float peak;                             // the CTA's largest logit, NaN where it has one
    int first;                              // its first token of the largest logit
    // what the first CTA found, for the others
    unsigned bin;
    u64 rest, total;
};

// Logits in their order as unsigned numbers; both zeros are one.
__device__ __forceinline__ unsigned order_of(float x) {
    const int b = __float_as_int(x + 0.f);
    return (unsigned)(b ^ (b >> 31 | INT_MIN));
}
__device__ __forceinline__ float value_of(unsigned k) { return __uint_as_float(k >> 31 ? k & 0x7FFFFFFFu : ~k); }

__device__ __forceinline__ float max_nan(float a, float b) {         // NaN where one is
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

struct Weigher {
    const double* powers;
    double peak, rate, least;      // largest logit; log2(e) / T; min_p in steps
    float top, cut;                // peak; a logit whose weight is 0, as are those below
    int steps;

    // The weight of a logit in steps of 2^-S; with kMin, 0 where min_p leaves it out.
    template <bool kMin = false>
    __device__ __forceinline__ u64 of(float x) const {
        const double t = (peak - (double)fminf(fmaxf(x, cut), top)) * rate;    // below 131
        const double m = fma(t, (double)kPowers, 6755399441055744.0);          // 1.5 2^52: rounds to a whole number
        const int k = __double2loint(m);
        const double r = fma(m - 6755399441055744.0, -1.0 / kPowers, t);
        // 2^(-r) - 1
        const double e = r * fma(r, fma(r, -0.05550410866482158, 0.2402265069591007), -0.6931471805599453);
        const double p = powers[k & (kPowers - 1)];
        const double v = fma(p, e, p);
        const double w = __hiloint2double(__double2hiint(v) + ((steps - (k >> 11)) << 20), __double2loint(v));
        const double whole = w + 4503599627370496.0;    // 2^52: its low bits are w rounded
        const u64 n = (u64)__double_as_longlong(whole) & 0xFFFFFFFFFFFFFull;
        return kMin && w < least ? 0ull : n;
    }
    __device__ __forceinline__ u64 of_kept(float x) const { return least > 0.0 ? of<true>(x) : of<false>(x); }
};

// Inclusive prefix over the block's threads, and the total.
__device__ __forceinline__ u64 block_prefix(u64 v, u64* part, u64& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const u64 x = __shfl_up_sync(~0u, v, o);
        if (lane >= o) v += x;
    }
    __syncthreads();
    if (lane == 31) part[warp] = v;
    __syncthreads();
    u64 before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kSampWarps; ++w) {
        if (w < warp) before += part[w];
        all += part[w];
    }
    total = all;
    return v + before;
}

// floor(f * n), or ceil(f * n), for 0 <= f < 1 and n < 2^62: f = m 2^-q, q from 53 on.
__device__ __forceinline__ u64 times(double f, u64 n, bool up) {
    const u64 b = (u64)__double_as_longlong(f);
    const int e = (int)(b >> 52);
    const u64 m = (b & 0xFFFFFFFFFFFFFull) | (e ? 1ull << 52 : 0ull);
    const int q = 1075 - max(e, 1);
    const u64 hi = __umul64hi(m, n), lo = m * n;         // below 2^115
    u64 r = 0, cut = hi | lo;
    if (q < 64) {
        r = hi << (64 - q) | lo >> q;
        cut = lo & ((1ull << q) - 1);
    } else if (q < 128) {
        r = hi >> (q - 64);
        cut = lo | (hi & ((1ull << (q - 64)) - 1));
    }
    return r + (up && cut ? 1 : 0);
}

__device__ __forceinline__ u64 ld_peer64(const void* mine, unsigned rank) {
    u64 v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(mapa_shared(smem_u32(mine), rank)) : "memory");
    return v;
}
__device__ __forceinline__ unsigned ld_peer32(const void* mine, unsigned rank) {
    unsigned v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(mapa_shared(smem_u32(mine), rank)) : "memory");
    return v;
}

template <typename T>
__device__ __forceinline__ float to_float(T x) {
    if constexpr (std::is_same<T, float>::value) return x;
    else if constexpr (std::is_same<T, __half>::value) return __half2float(x);
    else return __bfloat162float(x);
}

template <typename T, int kVec>
struct alignas(sizeof(T) * kVec) Several {
    T x[kVec];
};

template <typename T>
__global__ void __launch_bounds__(kSampThreads, 2) sample_kernel(const SampArgs a) {
    extern __shared__ __align__(16) uint8_t samp_smem[];
    SampShared& sh = *reinterpret_cast<SampShared*>(samp_smem);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    unsigned size;
    asm("mov.u32 %0, %cluster_nctarank;" : "=r"(size));
    const unsigned rank = cluster_ctarank();
    const long long row = blockIdx.x / size;
    const T* x = static_cast<const T*>(a.logits) + row * a.stride;
    const int e0 = min(a.V, (int)rank * a.blocks * kSampBlock), e1 = min(a.V, e0 + a.blocks * kSampBlock);
    auto all_sync = [&] {
        if (size > 1) cluster_sync();
        else __syncthreads();
    };
    // f(logit, index) for the logits from `from` to `to`, by `threads` threads, this one being
    // `me` of them: four a load between the first and the last boundary of four, two loads on
    // their way (four, of 16 bytes, were no faster and made the kernel several times as long).
    auto each = [&](int from, int to, int me, int threads, auto&& f) {
        constexpr int kVec = 4;
        using Vec = Several<T, kVec>;
        const int off = (int)(reinterpret_cast<uintptr_t>(x + from) % sizeof(Vec)) / (int)sizeof(T);
        const int head = min(to - from, off ? kVec - off : 0);
        const int start = from + head, vecs = (to - start) / kVec, last = start + vecs * kVec;
        const Vec* p = reinterpret_cast<const Vec*>(x + start);
#pragma unroll 1
        for (int i = me; i < vecs; i += 2 * threads) {
            const int two = i + threads < vecs ? threads : 0;          // else the first again, not looked at
            const Vec v = p[i], w = p[i + two];
#pragma unroll
            for (int j = 0; j < kVec; ++j) f(to_float<T>(v.x[j]), start + i * kVec + j);
            if (two) {
#pragma unroll
                for (int j = 0; j < kVec; ++j) f(to_float<T>(w.x[j]), start + (i + threads) * kVec + j);
            }
        }
        // before the first boundary and behind the last
        const int at = me < head ? from + me : last + me - head;
        if (me < head + to - last) f(to_float<T>(x[at]), at);
    };

    // ---- the largest logit, NaN if any is
    float peak = -INFINITY;
    each(e0, e1, tid, kSampThreads, [&](float v, int) { peak = max_nan(peak, v); });
#pragma unroll
    for (int o = 16; o; o >>= 1) peak = max_nan(peak, __shfl_xor_sync(~0u, peak, o));
    float* peaks = reinterpret_cast<float*>(sh.part);
    if (lane == 0) peaks[warp] = peak;
    __syncthreads();
    if (tid == 0) {
        for (int w = 0; w < kSampWarps; ++w) peak = max_nan(peak, peaks[w]);
        sh.peak = peak;
        sh.first = INT_MAX;
        sh.listed = 0;
    }
    all_sync();
    peak = sh.peak;
    for (unsigned r = 0; r < size && size > 1; ++r) peak = max_nan(peak, __uint_as_float(ld_peer32(&sh.peak, r)));
    const bool bad = isnan(peak) || peak == -INFINITY;
    const double temperature = a.temperature ? (double)a.temperature[row] : a.temperature1;
    const int top_k = a.top_k ? a.top_k[row] : a.top_k1;
    const double top_p = a.top_p ? (double)a.top_p[row] : a.top_p1;
    const double min_p = a.min_p ? (double)a.min_p[row] : a.min_p1;
    if (bad || !(temperature > 0.0) || top_k == 1 || top_p <= 0.0) {           // the same for the row
        int first = INT_MAX;
        if (!bad) each(e0, e1, tid, kSampThreads, [&](float v, int i) { first = min(first, v == peak ? i : INT_MAX); });
        first = __reduce_min_sync(~0u, first);
        if (lane == 0) atomicMin(&sh.first, first);
        all_sync();
        if (rank == 0 && tid == 0) {
            first = sh.first;
            for (unsigned r = 1; r < size; ++r) first = min(first, (int)ld_peer32(&sh.first, r));
            if (bad) set_err(a.err, kErrSampleNothing);
            a.out[row] = bad ? -1 : first;
        }
        if (size > 1) cluster_sync();                                         // the first CTA has read the others' numbers
        return;
    }

    // 2^(-j / 2048) as products of 2^(-i / 32) and 2^(-i / 2048)
    double* few = reinterpret_cast<double*>(sh.count);
    if (tid < 96) few[tid] = exp2(-(tid < 32 ? (double)tid / 32 : (double)(tid - 32) / kPowers));
    __syncthreads();
    for (int j = tid; j < kPowers; j += kSampThreads) sh.powers[j] = few[j >> 6] * few[32 + (j & 63)];
    __syncthreads();
    Weigher weigh;
    weigh.powers = sh.powers;
    // Logits 64 T ln 2 below the largest, and -inf, weigh nothing. A T so small that the next
    // number below the largest is further down than that counts as one that puts it at 130.
    unsigned none = kOrderOfMinusInf;          // logits up to here are not weighed at all
    weigh.peak = (double)peak;
    weigh.top = peak;
    weigh.cut = __double2float_rd((double)peak - 44.3614195558365 * temperature);
    weigh.cut = fmaxf(fminf(weigh.cut, nextafterf(peak, -INFINITY)), -FLT_MAX);
    weigh.rate = fmin(1.4426950408889634 / temperature, 130.0 / ((double)peak - (double)weigh.cut));
    weigh.rate = fmin(weigh.rate, DBL_MAX);    // a row of -FLT_MAX, which has no number below, and T below 2^-1023
    if (isinf(peak)) {                         // infinite ones weigh 1, others nothing
        none = kOrderOfMost;
        weigh.peak = weigh.top = weigh.cut = 0.f;
        weigh.rate = 0.0;
    }
    weigh.steps = a.steps;
    weigh.least = min_p > 0.0 ? fmin(min_p, 1.0) * __hiloint2double((1023 + a.steps) << 20, 0) : 0.0;
    constexpr int kLevels = std::is_same<T, float>::value ? 3 : 2;            // 16-bit types: 24 bits tell all apart
    constexpr int kDigit[3] = {20, 8, 0}, kWidth[3] = {12, 12, 8};
    // One digit of a border in the order, `found` being the digits before it. Count: of the
    // `want`-th token; else where weights, of the tokens above `floor` and floor_ties times the
    // one on it, reach `want` (at the first digit: top_p of their sum). The tokens are the
    // CTA's share of the row or, with listed >= 0, so many of its list; `many` CTAs take part.
    auto digit = [&](auto count_c, unsigned many, int level, int listed, unsigned floor, u64 floor_ties, unsigned& found,
                     u64& want) {
        constexpr bool kCount = decltype(count_c)::value;
        const int shift = kDigit[level], width = kWidth[level], bins = 1 << width;
        auto sync = [&] {
            if (many > 1) cluster_sync();
            else __syncthreads();
        };
        for (int j = tid; j < bins; j += kSampThreads) {
            if constexpr (kCount) sh.count[j] = 0;
            else sh.lo[j] = sh.hi[j] = 0;
        }
        __syncthreads();
        auto put = [&](unsigned k, u64 w) {
            const unsigned b = k >> shift & (bins - 1);
            if constexpr (kCount) atomicAdd(&sh.count[b], 1u);
            else if (w) {
                const unsigned lo = (unsigned)w, old = atomicAdd(&sh.lo[b], lo);
                const unsigned hi = (unsigned)(w >> 32) + (old + lo < old ? 1u : 0u);
                if (hi) atomicAdd(&sh.hi[b], hi);
            }
        };
        auto take = [&](unsigned k, float v) {
            if (level && k >> (shift + width) != found) return;
            if constexpr (kCount) put(k, 0);
            else {
                const u64 w = weigh.of(v);             // without a branch around it
                put(k, k > floor ? w : 0ull);
            }
        };
        if (listed < 0) each(e0, e1, tid, kSampThreads, [&](float v, int) { take(order_of(v), v); });
        else
#pragma unroll 1
            for (int i = tid; i < listed; i += kSampThreads) take(sh.list_key[i], value_of(sh.list_key[i]));
        if (!kCount && rank == 0 && tid == 0 && floor_ties && (!level || floor >> (shift + width) == found))
            put(floor, weigh.of(value_of(floor)) * floor_ties);
        sync();
        if (rank == 0) {
            if (many > 1) {                    // the others' histograms to the first CTA's
                constexpr int kEach = kBins / kSampThreads;
                u64 n[kEach];
#pragma unroll
                for (int i = 0; i < kEach; ++i) n[i] = 0;
#pragma unroll 1
                for (unsigned r = 0; r < many; ++r)
#pragma unroll
                    for (int i = 0; i < kEach; ++i) {                  // all on their way together
                        const int b = i * kSampThreads + tid;
                        if (b >= bins) continue;
                        if constexpr (kCount) n[i] += ld_peer32(&sh.count[b], r);
                        else n[i] += ((u64)ld_peer32(&sh.hi[b], r) << 32) + ld_peer32(&sh.lo[b], r);
                    }
#pragma unroll
                for (int i = 0; i < kEach; ++i) {
                    const int b = i * kSampThreads + tid;
                    if (b >= bins) continue;
                    if constexpr (kCount) sh.count[b] = (unsigned)n[i];
                    else {
                        sh.lo[b] = (unsigned)n[i];
                        sh.hi[b] = (unsigned)(n[i] >> 32);
                    }
                }
                __syncthreads();
            }
            // a warp's bins from the highest down, neighbouring ones a lane
            constexpr int kEach = kBins / kSampThreads;
            const int per = max(1, bins / kSampThreads), end = bins - 1 - (warp * (bins / kSampWarps) + lane * per);
            u64 v[kEach], mine = 0;
#pragma unroll
            for (int i = 0; i < kEach; ++i) {
                v[i] = 0;
                if (i < per && lane * per < bins / kSampWarps) {
                    if constexpr (kCount) v[i] = sh.count[end - i];
                    else v[i] = ((u64)sh.hi[end - i] << 32) + sh.lo[end - i];
                }
                mine += v[i];
            }
            u64 total;
            u64 before = block_prefix(mine, sh.part, total) - mine;
            if (!kCount && level == 0) want = times(top_p, total, true);
            if (before < want && want <= before + mine) {
#pragma unroll
                for (int i = 0; i < kEach; ++i) {
                    if (before < want && want <= before + v[i]) {
                        sh.bin = end - i;
                        sh.rest = want - before;
                    }
                    before += v[i];
                }
            }
        }
        sync();
        const unsigned bin = many > 1 ? ld_peer32(&sh.bin, 0) : sh.bin;
        want = many > 1 ? ld_peer64(&sh.rest, 0) : sh.rest;
        found = found << width | bin;
    };
    const bool by_count = top_k > 0 && top_k < a.V, by_weight = top_p < 1.0;
    unsigned edge = none;          // tokens above it are kept, and of those on it the first `ties`
    u64 ties = 0;

    auto gather = [&](unsigned k, int i) {
        const int at = atomicAdd(&sh.listed, 1);
        if (at < kList) {
            sh.list_key[at] = k;
            sh.list_at[at] = i;
        }
    };
    // Sums of blocks, a warp a block: weights above `high`; tokens from `low` to `high` are
    // gathered, or counted.
    auto sum_blocks = [&](unsigned low, unsigned high, bool gathers) {
        for (int b = warp; b < a.blocks; b += kSampWarps) {
            const int from = e0 + b * kSampBlock;
            u64 m = 0;
            unsigned t = 0;
            // where more were gathered than fit, another reading follows
            if (from < e1 && !(gathers && *static_cast<volatile int*>(&sh.listed) > kList))
                each(from, min(from + kSampBlock, e1), lane, 32, [&](float v, int i) {
                    const unsigned k = order_of(v);
                    if (k < low) return;
                    if (k > high) {
                        if (k > none) m += weigh.of_kept(v);
                    } else if (gathers) {
                        gather(k, i);
                    } else {
                        ++t;
                    }
                });
#pragma unroll
            for (int o = 16; o; o >>= 1) {
                m += __shfl_xor_sync(~0u, m, o);
                t += __shfl_xor_sync(~0u, t, o);
            }
            if (lane == 0) {
                sh.mass[b] = m;
                sh.ties[b] = t;
            }
        }
    };

    // ---- the borders. After the first digit of the first one: with one border the sums above
    // its part of the order and the tokens in it; with two the tokens from its part on, which
    // the first CTA goes on with alone.
    bool summed = false, alone = false;
    auto clear_blocks = [&] {
        for (int b = tid; b < (int)size * a.blocks; b += kSampThreads) {
            sh.mass[b] = 0;
            sh.ties[b] = 0;
        }
        __syncthreads();
    };
    int listed = -1;
    if (by_count || by_weight) {
        unsigned found = 0, floor = none, many = size;
        u64 want = (u64)top_k, floor_ties = 0;
        bool weighing = !by_count, first = true;
        int level = 0;
#pragma unroll 1
        while (true) {
            if (weighing) digit(std::false_type(), many, level, listed, floor, floor_ties, found, want);
            else digit(std::true_type(), many, level, listed, floor, floor_ties, found, want);
            if (first) {
                first = false;
                const unsigned low = found << kDigit[0];
                const bool one = by_count != by_weight;
                if (one) sum_blocks(low, low | ((1u << kDigit[0]) - 1), true);
                else each(e0, e1, tid, kSampThreads, [&](float v, int i) {
                    const unsigned k = order_of(v);
                    if (k >= low && *static_cast<volatile int*>(&sh.listed) <= kList) gather(k, i);
                });
                all_sync();
                int before[9];                 // tokens that the CTAs before gathered
                bool fits = true;
                before[0] = 0;
#pragma unroll
                for (unsigned r = 0; r < 8; ++r) {
                    const int n = r >= size ? 0 : size > 1 ? (int)ld_peer32(&sh.listed, r) : sh.listed;
                    fits &= n <= kList;
                    before[r + 1] = before[r] + min(n, kList + 1);
                }
                const int total = before[8];
                const bool few = total <= kFew;
                if (rank == 0 && (few || (!one && total <= kList))) {          // the others' tokens behind its own
                    for (int i = before[1] + tid; i < total; i += kSampThreads) {
                        int r = 1, off = before[1];
#pragma unroll
                        for (int y = 2; y < 8; ++y)
                            if (i >= before[y]) {
                                r = y;
                                off = before[y];
                            }
                        sh.list_key[i] = ld_peer32(&sh.list_key[i - off], r);
                        sh.list_at[i] = (int)ld_peer32(&sh.list_at[i - off], r);
                    }
                    __syncthreads();
                }
                if (few) {
                    // ---- each token against all others: how many come before it, of what weight
                    if (rank == 0) {
                        const bool on = tid < total;
                        const unsigned key = on ? sh.list_key[tid] : 0u;
                        const int at = on ? sh.list_at[tid] : INT_MAX;
                        const u64 w = on && key > none ? weigh.of(value_of(key)) : 0ull;
                        const u64 place = (u64)key << 32 | (unsigned)~at;              // larger comes first
                        if (on) sh.few[tid] = make_ulonglong2(place, w);
                        if (tid == 0) {
                            sh.bin = 0xFFFFFFFFu;
                            sh.rest = 0;
                        }
                        __syncthreads();
                        u64 w_before = 0;
                        unsigned n_before = 0;
#pragma unroll 4
                        for (int j = 0; j < total; ++j) {
                            const ulonglong2 f = sh.few[j];
                            const bool before = f.x > place;
                            n_before += before;
                            w_before += before ? f.y : 0ull;
                        }
                        // with one border `want` counts from the border's part on, as the list does
                        bool kept = on && (by_count ? n_before < (one ? want : (u64)top_k) : w_before < want);
                        if (by_count && by_weight) {
                            u64 sum;
                            block_prefix(kept ? w : 0ull, sh.part, sum);
                            kept = kept && w_before < times(top_p, sum, true);
                        }
                        if (kept) atomicMin(&sh.bin, max(key, none));
                        __syncthreads();
                        if (kept && key > none && key == sh.bin) atomicAdd(&sh.rest, 1ull);
                    }
                    if (one) all_sync();
                    else if (rank == 0) __syncthreads();
                    alone = !one;
                    summed = one;
                    if (alone && rank != 0) break;
                    edge = one && size > 1 ? ld_peer32(&sh.bin, 0) : sh.bin;
                    ties = one && size > 1 ? ld_peer64(&sh.rest, 0) : sh.rest;
                    listed = one ? sh.listed : total;
                    if (!one) clear_blocks();
                    break;
                }
                if (one && fits) {
                    listed = sh.listed;
                    summed = true;
                } else if (!one && total <= kList) {
                    alone = true;
                    if (rank != 0) break;
                    clear_blocks();
                    listed = total;
                    many = 1;
                }
            }
            if (++level < kLevels) continue;
            // 16-bit types: the last 8 bits follow from the sign
            edge = kLevels == 3 ? found : found << 8 | (found >> 23 ? 0u : 0xFFu);
            if (weighing) {
                const u64 w = weigh.of(value_of(edge));
                ties = (want + w - 1) / w;
                break;
            }
            ties = edge > none ? want : 0;                 // weights begin above `none`
            edge = max(edge, none);
            if (!by_weight) break;
            weighing = true;
            level = 0;
            found = 0;
            floor = edge;
            floor_ties = ties;
        }
    }
    const u64 on_edge = weigh.of_kept(value_of(edge));
    if (!summed && !alone) sum_blocks(edge, edge, false);
    else
        for (int i = tid; i < listed; i += kSampThreads) {
            const unsigned k = sh.list_key[i];
            const int b = (sh.list_at[i] - (alone ? 0 : e0)) / kSampBlock;
            if (k > edge) atomicAdd(&sh.mass[b], weigh.of_kept(value_of(k)));
            else if (k == edge) atomicAdd(&sh.ties[b], 1u);
        }
    if (alone) __syncthreads();
    else all_sync();
    if (rank == 0) {
        // a thread's blocks in order; the block in which the running sum passes u times the sum
        const int all = (int)size * a.blocks, per = (all + kSampThreads - 1) / kSampThreads;
        auto at = [&](int b, u64& m, unsigned& t) {
            const int r = b / a.blocks, i = b % a.blocks;
            const bool own = size == 1 || alone;
            m = own ? sh.mass[alone ? b : i] : ld_peer64(&sh.mass[i], r);
            t = own ? sh.ties[alone ? b : i] : ld_peer32(&sh.ties[i], r);
        };
        u64 sum = 0, tied = 0, total;
        for (int b = tid * per; b < min(all, (tid + 1) * per); ++b) {
            u64 m;
            unsigned t;
            at(b, m, t);
            tied += t;
        }
        const u64 tied_before = block_prefix(tied, sh.part, total) - tied;
        u64 used = tied_before;
        for (int b = tid * per; b < min(all, (tid + 1) * per); ++b) {
            u64 m;
            unsigned t;
            at(b, m, t);
            sum += m + (min(used + t, ties) - min(used, ties)) * on_edge;
            used += t;
        }
        u64 before = block_prefix(sum, sh.part2, total) - sum;
        const float u = a.u[row];
        const u64 target = min(u > 0.f ? u < 1.f ? times((double)u, total, false) : total : 0ull, total - 1);
        used = tied_before;
        if (tid == 0) sh.bin = 0;
        __syncthreads();
        for (int b = tid * per; b < min(all, (tid + 1) * per); ++b) {
            u64 m;
            unsigned t;
            at(b, m, t);
            const u64 s = m + (min(used + t, ties) - min(used, ties)) * on_edge;
            if (before <= target && target < before + s) {
                sh.bin = b;
                sh.rest = target - before;
                sh.total = used;
            }
            before += s;
            used += t;
        }
        __syncthreads();
        // ---- the token in the block: two neighbouring ones a thread
        const int first = (int)sh.bin * kSampBlock + tid * 2;
        const u64 want = sh.rest;
        unsigned key[2];
        u64 w[2], here = 0;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            key[j] = 0;
            w[j] = 0;
            if (first + j < a.V) {
                const float v = to_float<T>(x[first + j]);
                key[j] = order_of(v);
                w[j] = key[j] > edge ? weigh.of_kept(v) : 0ull;
                here += key[j] == edge;
            }
        }
        u64 rank_of = sh.total + block_prefix(here, sh.part, total) - here;
#pragma unroll
        for (int j = 0; j < 2; ++j)
            if (key[j] == edge) {
                if (rank_of < ties) w[j] = on_edge;
                ++rank_of;
            }
        u64 up_to = block_prefix(w[0] + w[1], sh.part2, total) - (w[0] + w[1]);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            if (up_to <= want && want < up_to + w[j]) a.out[row] = first + j;
            up_to += w[j];
        }
    }
    if (size > 1) cluster_sync();          // the first CTA has read the others' sums
}

template <typename T>
cudaError_t launch_sample(const SampArgs& a, int B, int cluster, cudaStream_t s) {
    const auto kernel = sample_kernel<T>;
    static std::atomic<unsigned long long> ready{0};      // a bit a device
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    if (!(ready.load(std::memory_order_acquire) >> dev & 1)) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(SampShared));
        if (e != cudaSuccess) return e;
        ready.fetch_or(1ull << dev, std::memory_order_release);
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(B * cluster));
    cfg.blockDim = dim3(kSampThreads);
    cfg.dynamicSmemBytes = sizeof(SampShared);
    cfg.stream = s;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = cluster;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, a);
}

}  // namespace
}  // namespace zs

extern "C" int zs_sample(const ZsSample* p) {
    using namespace zs;
    if (!p || p->B < 0 || p->V <= 0 || p->V > kSampBlock * kSampMaxBlocks || p->row_stride < 0 ||
        (p->dtype != ZS_BF16 && p->dtype != ZS_FP16 && p->dtype != ZS_FP32))
        return cudaErrorInvalidValue;
    if (p->B == 0) return cudaSuccess;
    if (p->B > INT32_MAX / 8 || !p->logits || !p->u || !p->out ||
        reinterpret_cast<uintptr_t>(p->logits) % (p->dtype == ZS_FP32 ? 4 : 2))
        return cudaErrorInvalidValue;
    SampArgs a{};
    a.logits = p->logits;
    a.stride = p->row_stride;
    a.u = p->u;
    a.temperature = p->temperature;
    a.top_k = p->top_k;
    a.top_p = p->top_p;
    a.min_p = p->min_p;
    a.temperature1 = p->temperature1;
    a.top_k1 = p->top_k1;
    a.top_p1 = p->top_p1;
    a.min_p1 = p->min_p1;
    a.out = reinterpret_cast<long long*>(p->out);
    a.err = p->err;
    a.V = p->V;
    int log2v = 0;
    while ((1 << log2v) < p->V) ++log2v;
    a.steps = std::min(50, 62 - log2v);
    // A CTA has eight blocks or more, and either all CTAs fit the GPU (two an SM), or the rows
    // at hand L2 (256 rows of 131071 in fp32: 681 MB read from HBM where all were).
    const int blocks = (p->V + kSampBlock - 1) / kSampBlock;
    const long long row_bytes = (long long)p->V * (p->dtype == ZS_FP32 ? 4 : 2);
    int cluster = 1;
    while (cluster < 8 && blocks >= cluster * 16 &&
           ((long long)p->B * cluster * 2 <= 296 || std::min<long long>(p->B, 296 / cluster) * row_bytes > (96ll << 20)))
        cluster *= 2;
    a.blocks = (blocks + cluster - 1) / cluster;
    cudaStream_t s = (cudaStream_t)p->stream;
    switch (p->dtype) {
        case ZS_BF16: return launch_sample<__nv_bfloat16>(a, p->B, cluster, s);
        case ZS_FP16: return launch_sample<__half>(a, p->B, cluster, s);
        default: return launch_sample<float>(a, p->B, cluster, s);
    }
}
