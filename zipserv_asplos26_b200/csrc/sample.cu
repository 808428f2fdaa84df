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
// Borders are found by three passes over 12, 12 and 8 bits of the logits' order (16-bit
// logits: two), each a histogram in shared memory of how many, or how much weight, the
// tokens hold that share the bits found so far. A row is read once for its maximum, twice
// or three times for each border, and once for sums of blocks of 1024, from which the
// token's block is found; all but the first come from L2. A row goes to a cluster of up to
// 8 CTAs where there are few, its histograms joined through distributed shared memory.
// Bound by instructions: some 30 for a weight in a histogram, 10 of them in 64 bits.
#include <algorithm>
#include <atomic>
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
constexpr unsigned kErrSampleNothing = 8u;  // a row had nothing to choose from
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
    };
    u64 mass[kSampMaxBlocks];               // of the CTA's blocks: weights above the border
    unsigned ties[kSampMaxBlocks];          // and tokens on it
    u64 part[kSampWarps], part2[kSampWarps];
    u64 best;                               // the CTA's first largest token
    int bad;
    // what the first CTA found, for the others
    unsigned bin;
    u64 rest, total;
};

// Logits in their order as unsigned numbers; both zeros are one.
__device__ __forceinline__ unsigned order_of(float x) {
    const unsigned b = __float_as_uint(x + 0.f);
    return b >> 31 ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(unsigned k) { return __uint_as_float(k >> 31 ? k & 0x7FFFFFFFu : ~k); }
constexpr unsigned kOrderInf = 0xFF800000u, kOrderMinusInf = 0x007FFFFFu;

struct Weigher {
    const double* powers;
    double peak, rate, least;      // largest logit; log2(e) / T; min_p in steps
    int steps;

    // The weight of a logit in steps of 2^-S; 0 where min_p leaves it out.
    __device__ __forceinline__ u64 operator()(float x) const {
        const double d = peak - (double)x;              // NaN where both are infinite: not below 0
        const double t = d * rate;
        if (!(d > 0.0)) return 1ull << steps;
        if (!(t < 64.0)) return 0ull;                   // x is -inf among them
        const double m = fma(t, (double)kPowers, 6755399441055744.0);          // 1.5 2^52: rounds to a whole number
        const int k = __double2loint(m);
        const double r = fma(m - 6755399441055744.0, -1.0 / kPowers, t);
        // 2^(-r) - 1
        const double e = r * fma(r, fma(r, -0.05550410866482158, 0.2402265069591007), -0.6931471805599453);
        const double p = powers[k & (kPowers - 1)];
        const double v = fma(p, e, p);
        const double w = __hiloint2double(__double2hiint(v) + ((steps - (k >> 11)) << 20), __double2loint(v));
        if (w < least) return 0ull;
        const double whole = w + 4503599627370496.0;    // 2^52: its low bits are w rounded
        return (u64)__double_as_longlong(whole) & 0xFFFFFFFFFFFFFull;
    }
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

// kVec logits a load where rows start on 16 bytes, else one.
template <typename T, int kVec>
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
    for (int j = tid; j < kPowers; j += kSampThreads) sh.powers[j] = exp2(-(double)j / kPowers);

    // f(logit, index) for the logits from `from` to `to`, four loads on their way.
    auto each = [&](int from, int to, int first, int threads, auto&& f) {
        constexpr int kBatch = kVec > 1 ? 4 : 8;
        for (int i = from + first * kVec; i < to; i += kBatch * threads * kVec) {
            Several<T, kVec> v[kBatch];
#pragma unroll
            for (int y = 0; y < kBatch; ++y) {
                const int at = i + y * threads * kVec;
                if (at + kVec <= to) v[y] = *reinterpret_cast<const Several<T, kVec>*>(x + at);
                else
#pragma unroll
                    for (int j = 0; j < kVec; ++j)
                        if (at + j < to) v[y].x[j] = x[at + j];
            }
#pragma unroll
            for (int y = 0; y < kBatch; ++y)
#pragma unroll
                for (int j = 0; j < kVec; ++j) {
                    const int at = i + y * threads * kVec + j;
                    if (at < to) f(to_float<T>(v[y].x[j]), at);
                }
        }
    };

    // ---- the first of the largest tokens; whether there is a NaN
    u64 best = 0;
    bool nan = false;
    each(e0, e1, tid, kSampThreads, [&](float v, int i) {
        const unsigned k = order_of(v);
        nan |= isnan(v);
        best = max(best, (u64)k << 32 | (unsigned)~i);
    });
#pragma unroll
    for (int o = 16; o; o >>= 1) best = max(best, __shfl_xor_sync(~0u, best, o));
    nan = __syncthreads_or(nan);
    if (lane == 0) sh.part[warp] = best;
    __syncthreads();
    if (tid == 0) {
        for (int w = 0; w < kSampWarps; ++w) best = max(best, sh.part[w]);
        sh.best = best;
        sh.bad = nan;
    }
    all_sync();
    best = sh.best;
    bool bad = sh.bad;
    for (unsigned r = 0; r < size && size > 1; ++r) {
        best = max(best, ld_peer64(&sh.best, r));
        bad |= ld_peer32(&sh.bad, r) != 0;
    }
    const unsigned top = (unsigned)(best >> 32);
    bad |= top <= kOrderMinusInf;
    const double temperature = a.temperature ? (double)a.temperature[row] : a.temperature1;
    const int top_k = a.top_k ? a.top_k[row] : a.top_k1;
    const double top_p = a.top_p ? (double)a.top_p[row] : a.top_p1;
    const double min_p = a.min_p ? (double)a.min_p[row] : a.min_p1;
    if (bad || !(temperature > 0.0) || top_k == 1 || top_p <= 0.0) {           // the same for the row
        if (rank == 0 && tid == 0) {
            if (bad) set_err(a.err, kErrSampleNothing);
            a.out[row] = bad ? -1 : (long long)(unsigned)~(unsigned)best;
        }
        if (size > 1) cluster_sync();                                         // peers read this CTA's numbers
        return;
    }

    Weigher weigh;
    weigh.powers = sh.powers;
    weigh.peak = (double)value_of(top);
    weigh.rate = 1.4426950408889634 / temperature;
    weigh.steps = a.steps;
    weigh.least = 0.0;
    constexpr int kLevels = std::is_same<T, float>::value ? 3 : 2;            // 16-bit types: 24 bits tell all apart
    constexpr int kDigit[3] = {20, 8, 0}, kWidth[3] = {12, 12, 8};

    // The place of a border in the order: kCount: of the `want`-th token; else where weights,
    // of the tokens above `floor_key` and floor_ties times the one on it, reach top_p of their
    // sum. rest: what is wanted of the tokens on the border (tokens, or weight).
    auto border = [&](auto count_c, u64 want, unsigned floor_key, u64 floor_ties, u64& rest) {
        constexpr bool kCount = decltype(count_c)::value;
        unsigned found = 0;
#pragma unroll 1
        for (int level = 0; level < kLevels; ++level) {
            const int shift = kDigit[level], width = kWidth[level], bins = 1 << width;
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
            each(e0, e1, tid, kSampThreads, [&](float v, int) {
                const unsigned k = order_of(v);
                if (level && k >> (shift + width) != found) return;
                if constexpr (kCount) put(k, 0);
                else if (k > floor_key) put(k, weigh(v));
            });
            if (!kCount && rank == 0 && tid == 0 && floor_ties && (!level || floor_key >> (shift + width) == found))
                put(floor_key, weigh(value_of(floor_key)) * floor_ties);
            all_sync();
            if (rank == 0) {
                // a thread's bins, from the highest down
                const int per = max(1, bins / kSampThreads);
                const int high = bins - 1 - tid * per;
                u64 sum = 0, each_bin[kBins / kSampThreads];
#pragma unroll
                for (int j = 0; j < kBins / kSampThreads; ++j) {
                    each_bin[j] = 0;
                    if (j >= per || high - j < 0) continue;
                    for (unsigned r = 0; r < size; ++r) {
                        if constexpr (kCount) each_bin[j] += size > 1 ? ld_peer32(&sh.count[high - j], r) : sh.count[high - j];
                        else if (size > 1)
                            each_bin[j] += (u64)ld_peer32(&sh.hi[high - j], r) << 32;
                        else each_bin[j] += (u64)sh.hi[high - j] << 32;
                        if constexpr (!kCount) each_bin[j] += size > 1 ? ld_peer32(&sh.lo[high - j], r) : sh.lo[high - j];
                    }
                    sum += each_bin[j];
                }
                u64 total;
                u64 before = block_prefix(sum, sh.part, total) - sum;
                if (!kCount && level == 0) want = times(top_p, total, true);
#pragma unroll
                for (int j = 0; j < kBins / kSampThreads; ++j) {
                    if (before < want && want <= before + each_bin[j]) {
                        sh.bin = high - j;
                        sh.rest = want - before;
                    }
                    before += each_bin[j];
                }
            }
            all_sync();
            const unsigned bin = size > 1 ? ld_peer32(&sh.bin, 0) : sh.bin;
            want = size > 1 ? ld_peer64(&sh.rest, 0) : sh.rest;
            found = found << width | bin;
        }
        // peers have read the first CTA's numbers before it writes new ones: its histogram
        // and the next all_sync lie in between
        rest = want;
        if constexpr (kLevels == 2) found = found << 8 | (found >> 23 ? 0u : 0xFFu);
        return found;
    };

    unsigned edge = 0;             // tokens above it are kept, and of those on it the first `ties`
    u64 ties = 0, rest;
    if (top_k > 0 && top_k < a.V) {
        edge = border(std::true_type(), (u64)top_k, 0u, 0ull, rest);
        ties = rest;
    }
    if (top_p < 1.0) {
        const unsigned e = border(std::false_type(), 0ull, edge, ties, rest);
        const u64 w = weigh(value_of(e));
        ties = (rest + w - 1) / w;
        edge = e;
    }
    if (min_p > 0.0) weigh.least = fmin(min_p, 1.0) * __hiloint2double((1023 + a.steps) << 20, 0);

    // ---- sums of blocks, a warp a block
    const u64 on_edge = edge ? weigh(value_of(edge)) : 0ull;
    for (int b = warp; b < a.blocks; b += kSampWarps) {
        const int from = e0 + b * kSampBlock;
        if (from >= e1) {
            if (lane == 0) {
                sh.mass[b] = 0;
                sh.ties[b] = 0;
            }
            continue;
        }
        u64 m = 0;
        unsigned t = 0;
        each(from, min(from + kSampBlock, e1), lane, 32, [&](float v, int) {
            const unsigned k = order_of(v);
            if (k > edge) m += weigh(v);
            t += k == edge;
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
    all_sync();
    if (rank == 0) {
        // a thread's blocks in order; the block in which the running sum passes u times the sum
        const int all = (int)size * a.blocks, per = (all + kSampThreads - 1) / kSampThreads;
        auto at = [&](int b, u64& m, unsigned& t) {
            const int r = b / a.blocks, i = b % a.blocks;
            m = size > 1 ? ld_peer64(&sh.mass[i], r) : sh.mass[i];
            t = size > 1 ? ld_peer32(&sh.ties[i], r) : sh.ties[i];
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
                w[j] = key[j] > edge ? weigh(v) : 0ull;
                here += edge && key[j] == edge;
            }
        }
        u64 rank_of = sh.total + block_prefix(here, sh.part, total) - here;
#pragma unroll
        for (int j = 0; j < 2; ++j)
            if (edge && key[j] == edge) {
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

template <typename T, int kVec>
cudaError_t launch_sample(const SampArgs& a, int B, int cluster, cudaStream_t s) {
    const auto kernel = sample_kernel<T, kVec>;
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

template <typename T>
cudaError_t launch_type(const SampArgs& a, int B, int cluster, cudaStream_t s) {
    constexpr int kVec = 16 / sizeof(T);
    const bool aligned = aligned16p(a.logits) && (B == 1 || a.stride % kVec == 0);
    return aligned ? launch_sample<T, kVec>(a, B, cluster, s) : launch_sample<T, 1>(a, B, cluster, s);
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
    // a CTA has four blocks or more, and all CTAs fit the GPU (two an SM)
    const int blocks = (p->V + kSampBlock - 1) / kSampBlock;
    int cluster = 1;
    while (cluster < 8 && (long long)p->B * cluster * 2 <= 296 && blocks >= cluster * 8) cluster *= 2;
    a.blocks = (blocks + cluster - 1) / cluster;
    cudaStream_t s = (cudaStream_t)p->stream;
    switch (p->dtype) {
        case ZS_BF16: return launch_type<__nv_bfloat16>(a, p->B, cluster, s);
        case ZS_FP16: return launch_type<__half>(a, p->B, cluster, s);
        default: return launch_type<float>(a, p->B, cluster, s);
    }
}
