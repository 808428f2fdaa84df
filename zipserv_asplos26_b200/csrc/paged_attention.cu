// Attention of one new token per sequence over a paged KV cache, the whole
// cache or a chosen list of its pages (zs_paged_attention).
//
//   out[b][i] = sum_t exp(s_t - m) v_t / sum_t exp(s_t - m),  s_t = scale q[b][i] . k_t,
// t over the sequence's tokens (of the listed pages), k and v of KV head
// i / (Hq / Hkv), m = max s_t; zero where nothing is attended. One pass: every
// warp keeps a running maximum, sum and unnormalised output in fp32 registers.
//
// Bound by HBM: each K and V row is read once for every 16 query heads that share
// it. The work is cut into chunks of 16 tokens of a unit (sequence, KV head, tile
// of up to 16 query heads), a warp's step, and dealt in one of two ways, chosen by
// sizes that the host has (unit_warps). Tiles do not share their reads: 64 sequences
// of 8193 with one KV head take 51 us for 16 query heads, 82 for 32 and 163 for 64
// (their keys and values once: 41).
//
// A warp copies its chunks' K and V rows with 16-byte cp.async into a ring of its
// own, ahead of the chunk it works on (rows past the length are zero-filled and
// never read), so there is no barrier in the loop and copies run on while a unit
// ends and the next begins. The products are m16n8k16 ones: a decode step has 1 to
// 16 query heads a KV head, far below a tcgen05 tile's 128 rows. Up to 8 heads they
// are the columns (PaNarrow), up to 16 the rows (PaWide); the tensor pipe is busy
// 14% of the time with 4 heads. P is fed as a 16-bit high part plus its 16-bit
// remainder (at most 2^-16 of a bf16 weight is left out, 2^-22 of an fp16 one), so that
// rounding P adds nothing to the output's own rounding. An infinite value would meet a
// remainder of zero or of the other sign there and give NaN: outputs that are not finite
// are looked at again (odd_values).
//
// Measured in long runs, at the power cap that they reach (bf16, 32 query and 8 KV
// heads of 128, pages of 64): B=32 T=4129 87.5 us, 6.19 TB/s; B=1 T=131105 89, 6.0;
// 61 sequences of 0..16417 (fp16, 64 query heads, pages of 16) 319, 6.5; B=1 T=97
// 4.8. A plain copy does 6.56 TB/s. DRAM reads are the algorithm's bytes (541.5 MB).
#include "paged_runs.cuh"

namespace zs {
namespace {

// P is computed as 2^(s - m + bias): for fp16 the bias keeps probabilities down
// to 2^-39 of the largest above fp16's smallest step (long tails of a long cache
// would vanish otherwise); bf16 has fp32's exponents.
template <typename T>
constexpr float kPBias = 0.f;
template <>
constexpr float kPBias<__half> = 15.f;

template <int D>
struct PaTile {
    static constexpr int kRowBytes = D * 2;
    static constexpr int kTile = kPaChunk * kRowBytes;             // one K or V chunk
};

// CTAs an SM and chunks of a warp's ring. What counts is how much is on its way:
// some 96 KB an SM read fastest where the products leave the time (the form for 8
// heads), from more warps rather than deeper rings. B=32 T=4129 in a long run under
// the power cap: 12 warps of 2 chunks 87.3 us, 8 of 3 91.4; D = 64: 16 of 2 90.9,
// 16 of 3 95.0, 12 of 4 95.6. The form for 16 heads holds twice the registers: 8
// warps of 2 chunks at D = 128 (90.0 us with 16 heads a KV head, 93.0 with 3), 12 of
// 3 at 64.
template <int D, bool kNarrow>
struct PaCfg : PaTile<D> {
    static constexpr int kCtas = kNarrow ? (D <= 64 ? 4 : 3) : (D <= 64 ? 3 : 2);
    static constexpr int kStages = !kNarrow && D <= 64 ? 3 : 2;
    static constexpr int kRing = kStages * 2 * PaTile<D>::kTile;   // bytes of a warp's ring
    static constexpr int kSmem = kPaWarps * kRing;
};

// Starts the copies of one chunk (its rows past `lim` are zeros).
template <int D>
__device__ __forceinline__ void copy_chunk(const PaArgs& a, uint32_t dst, int blk, int ch, int h, int lim,
                                           uint64_t policy) {
    using C = PaTile<D>;
    constexpr int kPieces = D / 8;                 // 16-byte pieces a row
    const int lane = threadIdx.x & 31;
    const int row0 = (ch & ((1 << (a.kp.page_shift - 4)) - 1)) * kPaChunk;
    const uint16_t* ks =
        static_cast<const uint16_t*>(a.kp.data) + h * a.kp.s_head + blk * a.kp.s_block + row0 * a.kp.s_token;
    const uint16_t* vs =
        static_cast<const uint16_t*>(a.vp.data) + h * a.vp.s_head + blk * a.vp.s_block + row0 * a.vp.s_token;
#pragma unroll
    for (int i = 0; i < kPaChunk * kPieces / 32; ++i) {
        const int x = i * 32 + lane, r = x / kPieces, pc = x % kPieces;
        const uint32_t to = dst + r * C::kRowBytes + ((pc ^ (r & 7)) * 16);
        cp16(to, ks + r * a.kp.s_token + pc * 8, r < lim, policy);
        cp16(to + C::kTile, vs + r * a.vp.s_token + pc * 8, r < lim, policy);
    }
}

// A weight of a finite score is positive, however small, so an output channel whose
// values include an infinity is that infinity, and NaN only where they include both
// signs or a NaN. The products cannot tell (0 * inf is NaN, and the remainder of a
// weight may be zero or negative), so where a finished output is not finite although
// the sum of its weights is a number, the values of its pieces that are not finite are
// read once more, here `count` chunks from `first` on. Adds to `seen`, for each of the
// kCount channels from c0 on, three bits: an infinity is there, a negative one, a NaN.
// Nothing of this runs while outputs are finite; to see that they are costs 0.1 us of
// 4.0 at B=1 T=97 and nothing in long runs. One infinity among B=32 T=4129: 160 us
// (finite 83), B=1 T=131105: 209 (83); with all of a unit read again it was 520 and
// 14186.
template <typename T, int kCount, bool kListed>
__device__ __forceinline__ void odd_values_of(const PaArgs& a, int e, int b, int h, int first, int count, int c0,
                                              uint32_t& seen) {
    constexpr uint32_t kInf = std::is_same<T, __nv_bfloat16>::value ? 0x7F80u : 0x7C00u;
    const int len = min(a.lens[b], (int)min((long long)a.width << a.kp.page_shift, (long long)INT_MAX));
    const uint16_t* base = static_cast<const uint16_t*>(a.vp.data) + h * a.vp.s_head + c0;
#pragma unroll 1
    for (int ch = first; ch < first + count; ++ch) {
        int blk, lim;
        look_chunk<kListed>(a, e, b, ch, len, blk, lim);
        const int row0 = (ch & ((1 << (a.kp.page_shift - 4)) - 1)) * kPaChunk;
        const uint16_t* v = base + blk * a.vp.s_block + row0 * a.vp.s_token;
#pragma unroll 4
        for (int r = 0; r < kPaChunk; ++r) {
            if (r >= lim) break;
            uint32_t w[2] = {0u, 0u};
            if constexpr (kCount == 4) *reinterpret_cast<uint2*>(w) = *reinterpret_cast<const uint2*>(v + r * a.vp.s_token);
            else w[0] = *reinterpret_cast<const uint32_t*>(v + r * a.vp.s_token);
#pragma unroll
            for (int j = 0; j < kCount; ++j) {
                const uint32_t x = w[j / 2] >> (j % 2 * 16) & 0xFFFFu, mag = x & 0x7FFFu;
                seen |= (mag > kInf ? 4u : mag < kInf ? 0u : x >> 15 ? 2u : 1u) << (3 * j);
            }
        }
    }
}
// What a warp holds of a unit: q as product fragments, running maximum (base 2),
// sum and output. Two forms: 16 heads as the rows of S and O (here; a lane has rows
// lane / 4 and lane / 4 + 8), or up to 8 heads as the columns of S^T and O^T.
template <typename T, int D>
struct PaWide {
    uint32_t qf[D / 16][4];
    float o[D / 8][4], m[2], l[2];
    struct Scores {
        float v[2][4];
    };
    struct Weights {
        uint32_t hi[4], lo[4];
    };

    __device__ __forceinline__ void start(const uint16_t* q, int rows) {
        const int lane = threadIdx.x & 31, r = lane >> 2, cc = (lane & 3) * 2;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int row = r + (i & 1) * 8, col = ks * 16 + (i >> 1) * 8 + cc;
                qf[ks][i] = row < rows ? *reinterpret_cast<const uint32_t*>(q + (long long)row * D + col) : 0u;
            }
#pragma unroll
        for (int i = 0; i < D / 8; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) o[i][j] = 0.f;
        m[0] = m[1] = -INFINITY;
        l[0] = l[1] = 0.f;
    }

    // S = Q K^T of a chunk's keys at kt: 16 heads x 16 tokens.
    __device__ __forceinline__ void scores(uint32_t kt, Scores& s) {
        auto& sc = s.v;
        const int lane = threadIdx.x & 31, r = (lane & 7) + ((lane >> 4) << 3), half = (lane >> 3) & 1;
        const uint32_t row = kt + r * PaTile<D>::kRowBytes;
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) sc[j][i] = 0.f;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
            uint32_t f[4];
            ldsm4(f, row + (((ks * 2 + half) ^ (r & 7)) * 16));
            mma16816(sc[0], qf[ks], f[0], f[1], T());
            mma16816(sc[1], qf[ks], f[2], f[3], T());
        }
    }

    // Running maximum and sum; P = 2^(S - m) as fragments of two 16-bit parts.
    __device__ __forceinline__ void weigh(const Scores& s, int lim, float scale2, Weights& w) {
        const auto& sc = s.v;
        const int t = (threadIdx.x & 3) * 2;
        float p[2][4];
        bool grew = false;
        float keep[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            float mx = -INFINITY;
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float x = j * 8 + t + i < lim ? sc[j][r * 2 + i] * scale2 : -INFINITY;
                    p[j][r * 2 + i] = x;
                    mx = fmaxf(mx, x);
                }
            mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, 2));
            const float mn = fmaxf(m[r], mx);
            grew |= mn > m[r];
            const float ref = mn == -INFINITY ? 0.f : mn;
            keep[r] = exp2f(m[r] - ref);
            m[r] = mn;
            float sum = 0.f;
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float x = exp2f(p[j][r * 2 + i] - ref + kPBias<T>);
                    p[j][r * 2 + i] = x;
                    sum += x;
                }
            l[r] = l[r] * keep[r] + sum;
        }
        if (__any_sync(~0u, grew)) {
#pragma unroll
            for (int i = 0; i < D / 8; ++i) {
                o[i][0] *= keep[0];
                o[i][1] *= keep[0];
                o[i][2] *= keep[1];
                o[i][3] *= keep[1];
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float x = p[i >> 1][(i & 1) * 2], y = p[i >> 1][(i & 1) * 2 + 1];
            w.hi[i] = pack2<T>(x, y);
            const float2 back = unpack2<T>(w.hi[i]);
            w.lo[i] = pack2<T>(x - back.x, y - back.y);
        }
    }

    // O += P V of a chunk's values at vt.
    __device__ __forceinline__ void add(uint32_t vt, const Weights& w) {
        const int lane = threadIdx.x & 31, r = lane & 15, half = lane >> 4;
        const uint32_t row = vt + r * PaTile<D>::kRowBytes;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
            uint32_t f[4];
            ldsm4t(f, row + (((ks * 2 + half) ^ (r & 7)) * 16));
            mma16816(o[ks * 2], w.hi, f[0], f[1], T());
            mma16816(o[ks * 2 + 1], w.hi, f[2], f[3], T());
            mma16816(o[ks * 2], w.lo, f[0], f[1], T());
            mma16816(o[ks * 2 + 1], w.lo, f[2], f[3], T());
        }
    }

    // The sums of a row's four lanes.
    __device__ __forceinline__ void finish() {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            l[r] += __shfl_xor_sync(~0u, l[r], 1);
            l[r] += __shfl_xor_sync(~0u, l[r], 2);
        }
    }
    // Whether any lane's output is odd, and the odd ones from what each lane saw of D / 32 channels.
    __device__ __forceinline__ bool odd() const {
        float x[4] = {0.f, 0.f, 0.f, 0.f}, y[4] = {0.f, 0.f, 0.f, 0.f};       // short chains
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
            x[i % 2 * 2] += o[i][0] * 0.f;
            x[i % 2 * 2 + 1] += o[i][1] * 0.f;
            y[i % 2 * 2] += o[i][2] * 0.f;
            y[i % 2 * 2 + 1] += o[i][3] * 0.f;
        }
        return __any_sync(~0u, is_odd((x[0] + x[1]) + (x[2] + x[3]), l[0]) || is_odd((y[0] + y[1]) + (y[2] + y[3]), l[1]));
    }
    __device__ __forceinline__ void mend(uint32_t seen) {
        const int d0 = (threadIdx.x & 3) * 2;
#pragma unroll
        for (int i = 0; i < D / 8; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int c = i * 8 + d0 + (j & 1);
                const float x = odd_output(__shfl_sync(~0u, seen, c / (D / 32)), c % (D / 32), o[i][j]);
                if (!isnan(l[j >> 1])) o[i][j] = x;
            }
    }
    // The finished rows, to the output [rows][D].
    __device__ __forceinline__ void write(uint16_t* out, float* lse, int rows) const {
        const int lane = threadIdx.x & 31, d0 = (lane & 3) * 2;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int row = (lane >> 2) + r * 8;
            if (row >= rows) continue;
            const float inv = l[r] == 0.f ? 0.f : 1.f / l[r];
#pragma unroll
            for (int i = 0; i < D / 8; ++i)
                *reinterpret_cast<uint32_t*>(out + row * D + i * 8 + d0) = pack2<T>(o[i][r * 2] * inv, o[i][r * 2 + 1] * inv);
            if (lse && d0 == 0) lse[row] = log_sum(m[r], l[r], kPBias<T>);
        }
    }
    // A piece: unnormalised rows [rows][D], and [rows][2] maxima and sums.
    __device__ __forceinline__ void park(float* po, float* ml, int rows) const {
        const int lane = threadIdx.x & 31, d0 = (lane & 3) * 2;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int row = (lane >> 2) + r * 8;
            if (row >= rows) continue;
#pragma unroll
            for (int i = 0; i < D / 8; ++i)
                *reinterpret_cast<float2*>(po + row * D + i * 8 + d0) = make_float2(o[i][r * 2], o[i][r * 2 + 1]);
            if (d0 == 0) *reinterpret_cast<float2*>(ml + row * 2) = make_float2(m[r], l[r]);
        }
    }
};

// Up to 8 heads: the keys are the rows of S^T = K Q^T (16 tokens x 8 heads) and the
// channels those of O^T += V^T P^T, half the products and half the exponentials of
// the form above. A lane has heads 2 (lane % 4) and the next, of S^T tokens lane / 4
// and lane / 4 + 8, of O^T channels likewise; P^T gets its fragment by transposing
// 8 x 8 blocks in registers.
template <typename T, int D>
struct PaNarrow {
    uint32_t qf[D / 16][2];
    float o[D / 16][4], m[2], l[2];
    struct Scores {
        float v[4];
    };
    struct Weights {
        uint32_t hi[2], lo[2];
    };

    __device__ __forceinline__ void start(const uint16_t* q, int rows) {
        const int lane = threadIdx.x & 31, head = lane >> 2, cc = (lane & 3) * 2;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks)
#pragma unroll
            for (int i = 0; i < 2; ++i)
                qf[ks][i] = head < rows ? *reinterpret_cast<const uint32_t*>(q + head * D + ks * 16 + i * 8 + cc) : 0u;
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) o[i][j] = 0.f;
        m[0] = m[1] = -INFINITY;
        l[0] = l[1] = 0.f;
    }

    __device__ __forceinline__ void scores(uint32_t kt, Scores& s) {
        const int lane = threadIdx.x & 31, r = lane & 15, half = lane >> 4;
        const uint32_t row = kt + r * PaTile<D>::kRowBytes;
        // two sums: the products of a chain wait for one another
        float odd[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < 4; ++i) s.v[i] = 0.f;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
            uint32_t f[4];
            ldsm4(f, row + (((ks * 2 + half) ^ (r & 7)) * 16));
            mma16816(ks & 1 ? odd : s.v, f, qf[ks][0], qf[ks][1], T());
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) s.v[i] += odd[i];
    }

    __device__ __forceinline__ void weigh(const Scores& s, int lim, float scale2, Weights& w) {
        const int t = (threadIdx.x & 31) >> 2;
        float p[4], keep[2];
        bool grew = false;
#pragma unroll
        for (int j = 0; j < 2; ++j) {               // head
            const float x = t < lim ? s.v[j] * scale2 : -INFINITY;
            const float y = t + 8 < lim ? s.v[2 + j] * scale2 : -INFINITY;
            float mx = fmaxf(x, y);
#pragma unroll
            for (int k = 4; k < 32; k <<= 1) mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, k));
            const float mn = fmaxf(m[j], mx);
            grew |= mn > m[j];
            const float ref = mn == -INFINITY ? 0.f : mn;
            keep[j] = exp2f(m[j] - ref);
            m[j] = mn;
            p[j] = exp2f(x - ref + kPBias<T>);
            p[2 + j] = exp2f(y - ref + kPBias<T>);
            l[j] = l[j] * keep[j] + (p[j] + p[2 + j]);
        }
        if (__any_sync(~0u, grew)) {
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
                o[i][0] *= keep[0];
                o[i][1] *= keep[1];
                o[i][2] *= keep[0];
                o[i][3] *= keep[1];
            }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t hi = pack2<T>(p[2 * i], p[2 * i + 1]);
            const float2 back = unpack2<T>(hi);
            w.hi[i] = transpose8(hi);
            w.lo[i] = transpose8(pack2<T>(p[2 * i] - back.x, p[2 * i + 1] - back.y));
        }
    }

    __device__ __forceinline__ void add(uint32_t vt, const Weights& w) {
        const int lane = threadIdx.x & 31, r = (lane & 7) + ((lane >> 4) << 3), half = (lane >> 3) & 1;
        const uint32_t row = vt + r * PaTile<D>::kRowBytes;
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
            uint32_t f[4];
            ldsm4t(f, row + (((i * 2 + half) ^ (r & 7)) * 16));
            mma16816(o[i], f, w.hi[0], w.hi[1], T());
            mma16816(o[i], f, w.lo[0], w.lo[1], T());
        }
    }

    __device__ __forceinline__ void finish() {
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int k = 4; k < 32; k <<= 1) l[j] += __shfl_xor_sync(~0u, l[j], k);
    }
    __device__ __forceinline__ bool odd() const {
        float x[4] = {0.f, 0.f, 0.f, 0.f}, y[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
            x[i % 2 * 2] += o[i][0] * 0.f;
            x[i % 2 * 2 + 1] += o[i][2] * 0.f;
            y[i % 2 * 2] += o[i][1] * 0.f;
            y[i % 2 * 2 + 1] += o[i][3] * 0.f;
        }
        return __any_sync(~0u, is_odd((x[0] + x[1]) + (x[2] + x[3]), l[0]) || is_odd((y[0] + y[1]) + (y[2] + y[3]), l[1]));
    }
    __device__ __forceinline__ void mend(uint32_t seen) {
        const int d0 = (threadIdx.x & 31) >> 2;
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int c = i * 16 + (j >> 1) * 8 + d0;
                const float x = odd_output(__shfl_sync(~0u, seen, c / (D / 32)), c % (D / 32), o[i][j]);
                if (!isnan(l[j & 1])) o[i][j] = x;
            }
    }
    __device__ __forceinline__ void write(uint16_t* out, float* lse, int rows) const {
        const int lane = threadIdx.x & 31, d0 = lane >> 2;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int row = (lane & 3) * 2 + j;
            if (row >= rows) continue;
            const float inv = l[j] == 0.f ? 0.f : 1.f / l[j];
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
                const uint32_t v = pack2<T>(o[i][j] * inv, o[i][2 + j] * inv);
                out[row * D + i * 16 + d0] = (uint16_t)v;
                out[row * D + i * 16 + 8 + d0] = (uint16_t)(v >> 16);
            }
            if (lse && d0 == 0) lse[row] = log_sum(m[j], l[j], kPBias<T>);
        }
    }
    __device__ __forceinline__ void park(float* po, float* ml, int rows) const {
        const int lane = threadIdx.x & 31, d0 = lane >> 2;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int row = (lane & 3) * 2 + j;
            if (row >= rows) continue;
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
                po[row * D + i * 16 + d0] = o[i][j];
                po[row * D + i * 16 + 8 + d0] = o[i][2 + j];
            }
            if (d0 == 0) *reinterpret_cast<float2*>(ml + row * 2) = make_float2(m[j], l[j]);
        }
    }
};

template <typename T, int D, bool kNarrow>
struct PaStateOf {
    using type = PaWide<T, D>;
};
template <typename T, int D>
struct PaStateOf<T, D, true> {
    using type = PaNarrow<T, D>;
};

// A warp's ring: kStages - 1 chunks are on their way while one is worked on.
// find(blk, ch, h, s) gives the place of the chunk of step s and returns its number
// of valid tokens. (Keys and values apart, each slot filled again as soon as it is
// used, kept 2 1/2 chunks on their way and was 3% slower.)
template <int D, bool kNarrow>
struct PaRing {
    using C = PaCfg<D, kNarrow>;
    uint32_t base;
    uint64_t policy;
    int steps;
    int lims[C::kStages - 1];      // of the chunks on their way, oldest first

    __device__ __forceinline__ void start(const PaArgs&, uint32_t at, int n) {
        base = at;
        policy = evict_first_policy();
        steps = n;
    }
    __device__ __forceinline__ uint32_t slot(int s) const { return base + (s % C::kStages) * 2 * C::kTile; }
    template <typename Find>
    __device__ __forceinline__ void ask(const PaArgs& a, int s, Find&& find) {
        int lim = 0;
        if (s < steps) {
            int blk, ch, h;
            lim = find(blk, ch, h, s, 0);
            copy_chunk<D>(a, slot(s), blk, ch, h, lim, policy);
        }
        cp_commit();
#pragma unroll
        for (int i = 0; i + 2 < C::kStages; ++i) lims[i] = lims[i + 1];
        lims[C::kStages - 2] = lim;
    }
    // Step s of a unit.
    template <typename State, typename Find>
    __device__ __forceinline__ void step(const PaArgs& a, int s, State& st, Find&& find) {
        typename State::Scores sc;
        typename State::Weights w;
        cp_wait<C::kStages - 2>();
        __syncwarp();
        const int lim = lims[0];
        ask(a, s + C::kStages - 1, find);
        st.scores(slot(s), sc);
        st.weigh(sc, lim, a.scale2, w);
        st.add(slot(s) + C::kTile, w);
        __syncwarp();
    }
};

// The form of a call (paged_runs.cuh).
template <typename T_, int D_, bool kListed_>
struct PaBase {
    using T = T_;
    using Args = PaArgs;
    static constexpr int D = D_, kParts = 1;
    static constexpr bool kListed = kListed_, kOdd = true, kGrouped = false;
    static constexpr float kBias = kPBias<T>;
    template <int kCount>
    __device__ __forceinline__ static void odd_values(const PaArgs& a, int e, int b, int h, int first, int count, int c0,
                                                      uint32_t& seen) {
        odd_values_of<T, kCount, kListed>(a, e, b, h, first, count, c0, seen);
    }
};
template <typename T, int D, bool kListed, bool kNarrow>
struct PaForm : PaBase<T, D, kListed>, PaCfg<D, kNarrow> {
    using Joined = PaBase<T, D, kListed>;
    using State = typename PaStateOf<T, D, kNarrow>::type;
    using Ring = PaRing<D, kNarrow>;
    __device__ __forceinline__ static void start(State& st, const PaArgs&, const uint16_t* q, int rows) { st.start(q, rows); }
};

// CTAs of the run kernel, at most.
inline int pa_max_ctas(int D, int G) {
    if (G <= 8) return 148 * (D <= 64 ? PaCfg<64, true>::kCtas : PaCfg<128, true>::kCtas);
    return 148 * (D <= 64 ? PaCfg<64, false>::kCtas : PaCfg<128, false>::kCtas);
}

template <class F>
cudaError_t launch_form(const PaArgs& a, int W, cudaStream_t s) {
    return launch_paged<F, F>(a, W, s);
}

template <typename T, bool kListed>
cudaError_t dispatch_dim(const PaArgs& a, int W, cudaStream_t s) {
    switch (a.kp.dim) {
        case 64:
            return a.G <= 8 ? launch_form<PaForm<T, 64, kListed, true>>(a, W, s)
                            : launch_form<PaForm<T, 64, kListed, false>>(a, W, s);
        case 128:
            return a.G <= 8 ? launch_form<PaForm<T, 128, kListed, true>>(a, W, s)
                            : launch_form<PaForm<T, 128, kListed, false>>(a, W, s);
    }
    return cudaErrorInvalidValue;
}

}  // namespace
}  // namespace zs

extern "C" size_t zs_paged_attention_workspace_bytes(int B, int Hq, int Hkv, int D) {
    using namespace zs;
    if (B <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || D <= 0) return 0;
    const long long tiles = (Hq / Hkv + kPaRows - 1) / kPaRows;
    const int prow = std::min(Hq / Hkv, kPaRows);
    // G is bounded by prow where it matters (both are above 8, or equal)
    return run_workspace_bytes((long long)B * Hkv * tiles, pa_max_ctas(D, prow), prow, D);
}

namespace zs {
namespace {

// The checked arguments of a call, but for its workspace.
bool attention_args(const ZsPagedAttention* p, PaArgs* a) {
    if (!p || !make_pool(&p->k_pool, &a->kp) || !make_pool(&p->v_pool, &a->vp) || !same_pools(p->k_pool, p->v_pool))
        return false;
    const int B = p->B, Hq = p->Hq, Hkv = a->kp.heads, D = a->kp.dim, top = p->top;
    if (B < 0 || Hq <= 0 || Hq % Hkv || p->width <= 0 || p->table_stride < p->width ||
        !std::isfinite(p->softmax_scale) || (D != 64 && D != 128))
        return false;
    if ((long long)B * Hq > INT32_MAX || (long long)p->width << a->kp.page_shift > INT32_MAX) return false;
    if (B && (!p->q || !p->block_table || !p->seq_lens || !p->out || !aligned16p(p->q) || !aligned16p(p->out)))
        return false;
    if (!p->pages != !p->counts || (p->pages && (top <= 0 || (long long)top << a->kp.page_shift > INT32_MAX)))
        return false;
    a->G = Hq / Hkv;
    a->tiles = (a->G + kPaRows - 1) / kPaRows;
    a->prow = std::min(a->G, kPaRows);
    a->q = p->q;
    a->table = p->block_table;
    a->table_stride = p->table_stride;
    a->lens = p->seq_lens;
    a->pages = p->pages;
    a->counts = p->counts;
    a->B = B; a->Hq = Hq; a->Hkv = Hkv; a->width = p->width; a->top = top;
    a->max_len = std::max(p->max_seqlen, 0);
    a->scale2 = p->softmax_scale * kLog2e;
    a->out = p->out;
    a->lse = p->lse;
    a->err = p->err;
    return true;
}

}  // namespace
}  // namespace zs

extern "C" size_t zs_paged_attention_workspace(const ZsPagedAttention* p) {
    using namespace zs;
    PaArgs a{};
    if (!attention_args(p, &a) || a.B == 0 || unit_warps(a, a.pages != nullptr, pa_max_ctas(a.kp.dim, a.G), 1)) return 0;
    return zs_paged_attention_workspace_bytes(a.B, a.Hq, a.Hkv, a.kp.dim);
}

extern "C" int zs_paged_attention(const ZsPagedAttention* p) {
    using namespace zs;
    PaArgs a{};
    if (!attention_args(p, &a)) return cudaErrorInvalidValue;
    if (a.B == 0) return cudaSuccess;
    const int max_ctas = pa_max_ctas(a.kp.dim, a.G), W = unit_warps(a, a.pages != nullptr, max_ctas, 1);
    if (!W) {
        if (!p->ws || !aligned16p(p->ws) ||
            p->ws_bytes < zs_paged_attention_workspace_bytes(a.B, a.Hq, a.Hkv, a.kp.dim))
            return cudaErrorInvalidValue;
        lay_workspace(&a, p->ws, max_ctas);
    }
    cudaStream_t s = (cudaStream_t)p->stream;
    if (p->k_pool.dtype == ZS_BF16)
        return a.pages ? dispatch_dim<__nv_bfloat16, true>(a, W, s) : dispatch_dim<__nv_bfloat16, false>(a, W, s);
    return a.pages ? dispatch_dim<__half, true>(a, W, s) : dispatch_dim<__half, false>(a, W, s);
}
