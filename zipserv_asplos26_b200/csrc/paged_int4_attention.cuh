// Attention of one new token per sequence over a 4-bit paged KV cache (format:
// paged_int4.cuh), the whole cache or a list of its pages; dealt to the GPU and joined
// as paged_runs.cuh says.
//
//   out[b][i] = sum_t exp(s_t - m) v_t / sum_t exp(s_t - m),  s_t = scale q[b][i] . k_t,
// k and v as their codes say, c + s (u - 8), in fp32 but for the products' operands.
//
// Bound between HBM and the instructions that unpack: 4.5 bits a value leave 3.5 times
// less to read than 16, and the same products. So the codes go to the tensor cores as
// they are, and scales and centres are applied to sums:
//   * Four bits anywhere in the low eight of a 16-bit float are a whole number times its
//     smallest step (2^-133 for bf16, 2^-24 for fp16), exact in a product: one AND makes
//     two operands, with one shift for every four. What sits four bits up counts 16-fold,
//     and meets a q of a sixteenth (scores) or has sums of its own (outputs).
//   * Scores: sum_g s_g (q_g . u_g) + sum_g (c_g - 8 s_g) sum(q_g). The second part is a
//     product too, of the row of parameters with q's sums (in three bf16 parts, 24 bits).
//     Keys are the rows (16 tokens), heads the columns, 8 or twice 8. q is scaled by a
//     power of two (bf16: 2^64; fp16: to its type's top), which loses nothing that counts.
//   * Outputs: sum_t (p_t s_t) (u_t - 8) + sum_t p_t c_t. p s goes in as fp16, scaled by a
//     power of two that follows the largest scale so far, so that it has all 11 bits from
//     there down to 2^-26 of it and vanishes below 2^-37, and its remainder follows as a
//     second part: 22 bits, as rounding a weight must add nothing to outputs that are what
//     is left of values that cancel (one part: 38.8 us for 42.8 at B=32 T=4129 in bf16, and
//     such outputs off by an eighth). The centres meet p in two bf16 parts.
//     The codes are centred by a f16x2 add, exact: sums of codes from 0 to 15 would in the
//     end be far larger than the outputs that are left of them, and a tensor core's sums
//     lose low bits. (Centring the sums every 128 tokens instead took as long.)
//
// The maximum that exponents refer to follows the scores only where one passes it by 2
// or more (base 2), so that most steps need no maximum over their lanes.
//
// Measured in a graph (bf16, 32 query and 8 KV heads of 128, groups of 64, pages of 64):
// B=32 T=4129 42.8 us, 3.6 TB/s (16-bit pages 85.5 us); B=128 137, 4.5 TB/s: 4.9 as a rate
// (75% of a plain copy's) and some 12 us of start, first lookups and join. B=1 T=131105
// 41.5; 61 sequences of 0..16417 (fp16, 64 query heads, groups of 32, pages of 16 by token)
// 176 to 185, 3.6 TB/s. 316 warp instructions for 16 tokens of a head, issued in half of the
// cycles: a warp waits for its own results, and two warps a scheduler hide part of it;
// arithmetic (ALU) 42% busy, tensor cores 35%. DRAM reads are the algorithm's bytes (152.7
// MB), but where rows lie by token 747 MB for 643.
#pragma once

#include "paged_int4.cuh"
#include "paged_runs.cuh"

namespace zs {

// Rows by place: strides in bytes, below 2^32, so that an address is a few multiply-adds.
struct Q4Places {
    const uint8_t* base;
    uint32_t block, token, head;
};
struct Q4Args : PaArgs {          // kp and vp: the codes (for page size, blocks and heads)
    Q4Places kcode, vcode, kpar, vpar;
    int packed;                   // rows of a page's head follow one another
};

namespace {

constexpr int kPaChunkShift = 4;
// The power of two that the values' scales stay below: at least 2^-40, since the weights
// go up to 2^15 over it and meet centres too, those of groups without a range among them.
constexpr int kNoTop = -40, kMostTop = 100;
constexpr uint32_t kLowCodes = 0x000F000Fu, kHighCodes = 0x00F000F0u;

template <int D>
struct Q4Tile {
    static constexpr int kRow = D / 2;                       // bytes of a row's codes
    static constexpr int kCodes = kPaChunk * kRow;
    static constexpr int kParams = kPaChunk * 16;            // a row's parameters in 16 bytes
    static constexpr int kTile = kCodes + kParams;           // keys or values of a part
    // the 16-byte piece of a row in shared memory: eight rows' pieces fill all banks
    __device__ __forceinline__ static int place(int r, int piece) {
        return r * kRow + (piece ^ (D == 128 ? (r >> 1) & 3 : (r >> 2) & 1)) * 16;
    }
};

// A step's parts, CTAs an SM and stages of a warp's ring. In runs of up to 8 heads a step
// takes 64 tokens: what it costs beside the products counts once for four parts, and the
// parts' sums do not wait for one another (B=32 T=4129: 42.8 us with 8 warps an SM, 45.7
// with 12 of 32 tokens, 54.9 with 16 of 16). With 16 heads the registers hold two parts.
// Units are short and get two parts, so that more warps share them.
template <int D, int NT, bool kUnits>
struct Q4Cfg {
    static constexpr int kParts = NT == 1 && !kUnits ? 4 : 2;
    static constexpr int kCtas = NT == 1 && kUnits ? 3 : 2;
    static constexpr int kStages = kParts == 4 ? 2 : 3;
    static constexpr int kPartBytes = 2 * Q4Tile<D>::kTile;
    static constexpr int kChunkBytes = kParts * kPartBytes;
    static constexpr int kPiece = kPaRows * (D + 2) * 4;     // a warp's piece in the units kernel
    static constexpr int kRing = kStages * kChunkBytes > kPiece ? kStages * kChunkBytes : kPiece;
    static constexpr int kSmem = kPaWarps * kRing;
};

__device__ __forceinline__ float exp2_fast(float x) {        // 2 ulp; below 2^-126 it is zero
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// 16 bytes, or zeros; without a hint to fetch what lies around (other heads' rows, where
// rows do not follow one another).
__device__ __forceinline__ void cp16_row(uint32_t dst, const void* src, bool on, uint64_t policy) {
    asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2, %3;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0),
                 "l"(policy)
                 : "memory");
}
__device__ __forceinline__ uint64_t evict_normal_policy() {
    uint64_t p;
    asm volatile("createpolicy.fractional.L2::evict_normal.b64 %0, 1.0;" : "=l"(p));
    return p;
}
__device__ __forceinline__ void cp16_all(uint32_t dst, const void* src, uint64_t policy) {
    asm volatile("cp.async.cg.shared.global.L2::cache_hint.L2::256B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "l"(policy)
                 : "memory");
}
// kBytes bytes (4, 8 or 16) of parameters.
template <int kBytes>
__device__ __forceinline__ void cp_params(uint32_t dst, const void* src, bool on, uint64_t policy) {
    if constexpr (kBytes == 16)
        asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2, %3;" ::"r"(dst), "l"(src),
                     "r"(on ? 16 : 0), "l"(policy)
                     : "memory");
    else
        asm volatile("cp.async.ca.shared.global.L2::cache_hint [%0], [%1], %2, %3, %4;" ::"r"(dst), "l"(src),
                     "n"(kBytes), "r"(on ? kBytes : 0), "l"(policy)
                     : "memory");
}
// The kN scales (bf16) at the start of a row of parameters: two a word, and one of them in fp32.
template <int kN>
__device__ __forceinline__ void ld_scales(uint32_t (&w)[(kN + 1) / 2], uint32_t at) {
    if constexpr (kN == 4)
        asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(at) : "memory");
    else if constexpr (kN == 2)
        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[0]) : "r"(at) : "memory");
    else {
        uint16_t x;
        asm volatile("ld.shared.u16 %0, [%1];" : "=h"(x) : "r"(at) : "memory");
        w[0] = x;
    }
}
template <int kN>
__device__ __forceinline__ float scale_of(const uint32_t (&w)[(kN + 1) / 2], int g) {
    return g & 1 ? __uint_as_float(w[g / 2] & 0xFFFF0000u) : bf16_bits_to_float(w[g / 2]);
}
// The larger of each of two bf16 numbers that are not negative.
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.u16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
// mma16816, free to move among other work, and from sums of a column's own.
__device__ __forceinline__ void product(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __nv_bfloat16) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, "
        "%2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void product(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __half) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, "
        "%2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void first_product(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, float c0,
                                              float c1, __nv_bfloat16) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, "
        "%10, %11};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1));
}
__device__ __forceinline__ void first_product(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, float c0,
                                              float c1, __half) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, "
        "%10, %11};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1));
}
__device__ __forceinline__ uint32_t add_f16x2(uint32_t a, uint32_t b) {
    const __half2 r = __hadd2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ float power_of_two(int e) { return __int_as_float((e + 127) << 23); }   // e from -126 to 127

// What a warp holds of a unit of up to NT x 8 heads. A lane has heads 2 (lane % 4) and
// the next of each eight; of scores, tokens lane / 4 and lane / 4 + 8; of outputs the
// four channels from 4 (lane / 4) on of each 32.
template <typename T, int D, int NG, int NT, int kParts>
struct Q4State {
    static constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
    static constexpr int kBlocks = D / 32, kPer = kBlocks / NG;      // 32 channels: a 16-byte piece of a row
    using Bf = __nv_bfloat16;
    uint32_t qf[NT][kBlocks][2][2];    // q of the even, odd channels (these a sixteenth)
    uint32_t zf[NT][3];                // of what meets the parameters: -8 sum(q_g), sum(q_g), times scale2, in three parts
    float unit[NT][2];                 // of the sums over codes, with scale2
    float o[NT][kBlocks][2][4];        // sums of the even, odd channels
    float z[NT][4];                    // sums of p times the parameters
    float m[NT][2], l[NT][2];          // largest score, sum of weights
    float less[NT][2], most[NT][2];    // scores count from ref = m + top - 13 = -less; at most `most` from there
    int top;                           // scales of values are below 2^top, weights times them below 2^15

    using Four = float[NT][4];         // of a lane's tokens of a part and heads

    __device__ __forceinline__ void start(const uint16_t* q, int rows, float scale2) {
        const int lane = threadIdx.x & 31;
        top = kNoTop;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int head = nt * 8 + (lane >> 2);
            uint32_t w[kBlocks][4];
            float sum[NG], peak = 0.f;
#pragma unroll
            for (int g = 0; g < NG; ++g) sum[g] = 0.f;
#pragma unroll
            for (int b = 0; b < kBlocks; ++b) {
                uint4 x = make_uint4(0u, 0u, 0u, 0u);
                if (head < rows) x = *reinterpret_cast<const uint4*>(q + (long long)head * D + b * 32 + (lane & 3) * 8);
                w[b][0] = x.x;
                w[b][1] = x.y;
                w[b][2] = x.z;
                w[b][3] = x.w;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 f = unpack2<T>(w[b][i]);
                    sum[b / kPer] += f.x + f.y;
                    peak = fmaxf(peak, fmaxf(fabsf(f.x), fabsf(f.y)));
                }
            }
            // bf16: 2^64; fp16: the head's largest below 2^15 (even channels) and 2^11 (odd ones)
            int e = 64;
            if constexpr (!kBf16) {
                peak = fmaxf(peak, __shfl_xor_sync(~0u, peak, 1));
                peak = fmaxf(peak, __shfl_xor_sync(~0u, peak, 2));
                e = 14 - ((__float_as_int(peak) >> 23) - 127);
                e = min(e, 60);                          // a head of zeros
                if (e < -1) e = 0;                       // a head with infinities or NaN
            }
            const float even = power_of_two(e), odd = power_of_two(e - 4);
            // codes in steps of 2^-133 or 2^-24; of the lane's heads
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int ej = __shfl_sync(~0u, e, ((lane & 3) * 2 + j) * 4);
                unit[nt][j] = kBf16 ? scale2 * power_of_two(69) : scale2 * power_of_two(24 - ej);
            }
#pragma unroll
            for (int b = 0; b < kBlocks; ++b) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {            // channels 2i (even) and 2i + 1 (odd)
                    const float2 f = unpack2<T>(w[b][i]);
                    w[b][i] = pack2<T>(f.x * even, f.y * odd);
                }
                // codes of channels i and i + 4 lie 16 bits apart
                qf[nt][b][0][0] = __byte_perm(w[b][0], w[b][2], 0x5410);
                qf[nt][b][0][1] = __byte_perm(w[b][1], w[b][3], 0x5410);
                qf[nt][b][1][0] = __byte_perm(w[b][0], w[b][2], 0x7632);
                qf[nt][b][1][1] = __byte_perm(w[b][1], w[b][3], 0x7632);
            }
            float y[2] = {0.f, 0.f};                     // of parameters 2 (lane % 4) and the next
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                sum[g] += __shfl_xor_sync(~0u, sum[g], 1);
                sum[g] += __shfl_xor_sync(~0u, sum[g], 2);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    if ((lane & 3) * 2 + i == g) y[i] = -8.f * (sum[g] * scale2);
                    if ((lane & 3) * 2 + i == NG + g) y[i] = sum[g] * scale2;
                }
            }
#pragma unroll
            for (int i = 0; i < 3; ++i) {
                zf[nt][i] = pack2<Bf>(y[0], y[1]);
                const float2 back = unpack2<Bf>(zf[nt][i]);
                y[0] -= back.x;
                y[1] -= back.y;
            }
#pragma unroll
            for (int b = 0; b < kBlocks; ++b)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[nt][b][0][i] = o[nt][b][1][i] = 0.f;
#pragma unroll
            for (int i = 0; i < 4; ++i) z[nt][i] = 0.f;
            m[nt][0] = m[nt][1] = -INFINITY;
            less[nt][0] = less[nt][1] = 0.f;
            most[nt][0] = most[nt][1] = -INFINITY;
            l[nt][0] = l[nt][1] = 0.f;
        }
    }

    // The scales of a part's keys or values, at `at`: of a lane's two tokens.
    using Scales = uint32_t[2][(NG + 1) / 2];
    __device__ __forceinline__ void look(uint32_t at, Scales& v) {
        const uint32_t par = at + Q4Tile<D>::kCodes + ((threadIdx.x & 31) >> 2) * 16;
        ld_scales<NG>(v[0], par);
        ld_scales<NG>(v[1], par + 8 * 16);
    }

    // Scores (times scale2, from ref on) of the part whose keys are at kt.
    __device__ __forceinline__ void scores(uint32_t kt, Four& x) {
        const int lane = threadIdx.x & 31, r = lane & 15, half = lane >> 4;
        const uint32_t par = kt + Q4Tile<D>::kCodes;
        float c[NT][4], s[NT][4];
        Scales sc;
        look(kt, sc);
        // the rows of parameters twice over: what they meet is in the two halves of the depth
        uint32_t pr[4];
        ldsm4(pr, par + r * 16);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            first_product(c[nt], pr, zf[nt][0], zf[nt][1], less[nt][0], less[nt][1], Bf());
            product(c[nt], pr, zf[nt][2], 0u, Bf());
        }
        float e[NT][4];
#pragma unroll
        for (int b2 = 0; b2 < kBlocks / 2; ++b2) {
            uint32_t f[4];
            ldsm4(f, kt + Q4Tile<D>::place(r, b2 * 2 + half));
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int b = b2 * 2 + i, g = b / kPer;
                const uint32_t u = f[i * 2], w = f[i * 2 + 1], u8 = u >> 8, w8 = w >> 8;
                const uint32_t lo[4] = {u & kLowCodes, w & kLowCodes, u8 & kLowCodes, w8 & kLowCodes};
                const uint32_t hi[4] = {u & kHighCodes, w & kHighCodes, u8 & kHighCodes, w8 & kHighCodes};
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    if (b % kPer == 0) first_product(e[nt], lo, qf[nt][b][0][0], qf[nt][b][0][1], 0.f, 0.f, T());
                    else product(e[nt], lo, qf[nt][b][0][0], qf[nt][b][0][1], T());
                    product(e[nt], hi, qf[nt][b][1][0], qf[nt][b][1][1], T());
                    if (b % kPer == kPer - 1) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const float k = scale_of<NG>(sc[j >> 1], g);
                            s[nt][j] = g ? s[nt][j] + k * e[nt][j] : k * e[nt][j];
                        }
                    }
                }
            }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i) x[nt][i] = s[nt][i] * unit[nt][i & 1] + c[nt][i];
    }

    // From scores x - ref to weights 2^(x - ref), of the first lim[i] tokens of each part, whose
    // values have the scales v.
    __device__ __forceinline__ void weigh(Four (&x)[kParts], const int (&lim)[kParts], const Scales (&v)[kParts]) {
        const int t = (threadIdx.x & 31) >> 2;
        uint32_t big = 0u;
#pragma unroll
        for (int i = 0; i < kParts; ++i)
#pragma unroll
            for (int w = 0; w < (NG + 1) / 2; ++w) big = max2(big, max2(v[i][0][w], v[i][1][w]));
        const uint32_t room = (uint32_t)(((top + 127) << 7) - 1) * 0x10001u;       // the largest bf16 below 2^top
        bool up = max2(big, room) != room;
#pragma unroll
        for (int i = 0; i < kParts; ++i) {
            if (lim[i] < kPaChunk) {                   // the same for the warp: a unit's last part
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (t + (j >> 1) * 8 >= lim[i]) x[i][nt][j] = -INFINITY;
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int j = 0; j < 4; ++j) up |= x[i][nt][j] > most[nt][j & 1];
        }
        if (__any_sync(~0u, up)) {
#pragma unroll
            for (int k = 4; k < 32; k <<= 1) big = max2(big, __shfl_xor_sync(~0u, big, k));
            top = min(max((int)(max(big & 0xFFFFu, big >> 16) >> 7) - 126, top), kMostTop);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    float mx = -INFINITY;
#pragma unroll
                    for (int i = 0; i < kParts; ++i) mx = fmaxf(mx, fmaxf(x[i][nt][j], x[i][nt][2 + j]));
#pragma unroll
                    for (int k = 4; k < 32; k <<= 1) mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, k));
                    const bool held = m[nt][j] != -INFINITY;           // the same for a head's lanes
                    m[nt][j] = fmaxf(m[nt][j], mx - less[nt][j]);
                    const bool none = m[nt][j] == -INFINITY;
                    const float now = (none ? 0.f : m[nt][j]) + (float)(top - 13);
                    const float by = -less[nt][j] - now, keep = exp2_fast(by);
                    less[nt][j] = -now;
                    most[nt][j] = none ? -INFINITY : (float)(15 - top);
#pragma unroll
                    for (int i = 0; i < kParts; ++i) {
                        x[i][nt][j] += by;
                        x[i][nt][2 + j] += by;
                    }
                    if (held) {                // by any lane: o and z sum all lanes' tokens, l this lane's
                        l[nt][j] *= keep;
                        z[nt][j] *= keep;
#pragma unroll
                        for (int b = 0; b < kBlocks; ++b)
#pragma unroll
                            for (int y = 0; y < 2; ++y) {
                                o[nt][b][y][j] *= keep;
                                o[nt][b][y][2 + j] *= keep;
                            }
                    }
                }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < kParts; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    x[i][nt][j] = exp2_fast(x[i][nt][j]);
                    x[i][nt][2 + j] = exp2_fast(x[i][nt][2 + j]);
                    l[nt][j] += x[i][nt][j] + x[i][nt][2 + j];
                }
    }

    // Four weights (a lane's tokens and heads) as fragments of two 16-bit numbers that add up.
    template <typename P>
    __device__ __forceinline__ static void split(float a, float b, float c, float d, uint32_t (&f)[2][2]) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t x = pack2<P>(a, b), y = pack2<P>(c, d);
            f[i][0] = transpose8(x);
            f[i][1] = transpose8(y);
            if (i == 0) {
                const float2 xb = unpack2<P>(x), yb = unpack2<P>(y);
                a -= xb.x;
                b -= xb.y;
                c -= yb.x;
                d -= yb.y;
            }
        }
    }

    // Adds the part whose values are at vt, of scales sc, by weights w.
    __device__ __forceinline__ void add(uint32_t vt, const Four& w, const Scales& sc) {
        const int lane = threadIdx.x & 31, r = lane & 15, half = lane >> 4;
        // the rows of parameters as columns, twice over: rows 8 to 15 of z are not looked at
        uint32_t pr[4];
        ldsm4t(pr, vt + Q4Tile<D>::kCodes + ((lane & 7) + half * 8) * 16);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            uint32_t f[2][2];
            split<Bf>(w[nt][0], w[nt][1], w[nt][2], w[nt][3], f);
            product(z[nt], pr, f[0][0], f[0][1], Bf());
            product(z[nt], pr, f[1][0], f[1][1], Bf());
        }
        uint32_t f[NT][2][2];
#pragma unroll
        for (int b2 = 0; b2 < kBlocks / 2; ++b2) {
            uint32_t v[4];
            ldsm4t(v, vt + Q4Tile<D>::place(r, b2 * 2 + half));
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int b = b2 * 2 + i, g = b / kPer;
                if (b % kPer == 0) {
                    const float s0 = scale_of<NG>(sc[0], g), s1 = scale_of<NG>(sc[1], g);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
                        split<__half>(w[nt][0] * s0, w[nt][1] * s0, w[nt][2] * s1, w[nt][3] * s1, f[nt]);
                }
                const uint32_t t[4] = {v[i * 2], v[i * 2] >> 8, v[i * 2 + 1], v[i * 2 + 1] >> 8};
                uint32_t lo[4], hi[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    lo[j] = add_f16x2(t[j] & kLowCodes, 0x80088008u);        // - 8 steps
                    hi[j] = add_f16x2(t[j] & kHighCodes, 0x80808080u);       // - 128 steps
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        product(o[nt][b][0], lo, f[nt][x][0], f[nt][x][1], __half());
                        product(o[nt][b][1], hi, f[nt][x][0], f[nt][x][1], __half());
                    }
            }
        }
    }

    // The sums of a head's eight lanes, and the outputs (unnormalised) from the sums.
    __device__ __forceinline__ void finish() {
        const int lane = threadIdx.x & 31;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
#pragma unroll
                for (int k = 4; k < 32; k <<= 1) l[nt][j] += __shfl_xor_sync(~0u, l[nt][j], k);
#pragma unroll
                for (int b = 0; b < kBlocks; ++b) {
                    const float c = __shfl_sync(~0u, z[nt][j], (NG + b / kPer) * 4 + (lane & 3));
#pragma unroll
                    for (int y = 0; y < 2; ++y) {
                        const float by = y ? power_of_two(20) : power_of_two(24);
                        o[nt][b][y][j] = o[nt][b][y][j] * by + c;
                        o[nt][b][y][2 + j] = o[nt][b][y][2 + j] * by + c;
                    }
                }
            }
    }

    // The finished rows, to the output [rows][D].
    __device__ __forceinline__ void write(uint16_t* out, float* lse, int rows) const {
        const int lane = threadIdx.x & 31;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int row = nt * 8 + (lane & 3) * 2 + j;
                if (row >= rows) continue;
                const float inv = l[nt][j] == 0.f ? 0.f : 1.f / l[nt][j];
#pragma unroll
                for (int b = 0; b < kBlocks; ++b)
                    *reinterpret_cast<uint2*>(out + row * D + b * 32 + (lane >> 2) * 4) =
                        make_uint2(pack2<T>(o[nt][b][0][j] * inv, o[nt][b][1][j] * inv),
                                   pack2<T>(o[nt][b][0][2 + j] * inv, o[nt][b][1][2 + j] * inv));
                if (lse && lane < 4) lse[row] = log_sum(-less[nt][j], l[nt][j], 0.f);
            }
    }
    // A piece: unnormalised rows [rows][D], and [rows][2] references and sums. Where nothing
    // weighs the reference is minus infinity, as the other pieces may lie far below zero.
    __device__ __forceinline__ void park(float* po, float* ml, int rows) const {
        const int lane = threadIdx.x & 31;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int row = nt * 8 + (lane & 3) * 2 + j;
                if (row >= rows) continue;
#pragma unroll
                for (int b = 0; b < kBlocks; ++b)
                    *reinterpret_cast<float4*>(po + row * D + b * 32 + (lane >> 2) * 4) =
                        make_float4(o[nt][b][0][j], o[nt][b][1][j], o[nt][b][0][2 + j], o[nt][b][1][2 + j]);
                if (lane < 4)
                    *reinterpret_cast<float2*>(ml + row * 2) =
                        make_float2(m[nt][j] == -INFINITY ? -INFINITY : -less[nt][j], l[nt][j]);
            }
    }
};

// A warp's ring: kStages - 1 chunks are on their way while one is worked on.
template <int D, int NG, int NT, bool kUnits>
struct Q4Ring {
    using C = Q4Cfg<D, NT, kUnits>;
    using Tile = Q4Tile<D>;
    static constexpr int kParts = C::kParts;
    static constexpr int kPieces = D / 32;             // 16-byte pieces a row
    static constexpr int kEach = kPaChunk * kPieces / 32;      // of K, and of V, a lane and part
    uint32_t base;
    uint64_t policy;
    int steps, head;
    const uint8_t *kfrom, *vfrom, *pfrom;              // a lane's places in the present head's rows
    int lims[C::kStages - 1][kParts];                // of the chunks on their way, oldest first

    // Rows that follow one another pass through L2 once; of others, the lines are shared with
    // other heads' rows (61 sequences of 0..16417 in pages by token, marked to leave first and
    // fetched 256 bytes at a time: 1.96 GB read for 0.65).
    __device__ __forceinline__ void start(const Q4Args& a, uint32_t at, int n) {
        base = at;
        policy = a.packed ? evict_first_policy() : evict_normal_policy();
        steps = n;
        head = -1;
        // rows of parameters shorter than 16 bytes end in zeros
        if constexpr (NG < 4) {
            const int lane = threadIdx.x & 31;
#pragma unroll
            for (int s = 0; s < C::kStages * kParts; ++s)
                asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(
                                 base + s * C::kPartBytes + (lane >> 4) * Tile::kTile + Tile::kCodes + (lane & 15) * 16),
                             "r"(0)
                             : "memory");
            __syncwarp();
        }
    }
    __device__ __forceinline__ uint32_t slot(int s) const { return base + (s % C::kStages) * C::kChunkBytes; }
    __device__ __forceinline__ static const uint8_t* at(const uint8_t* p, uint32_t n, uint32_t stride) {
        return p + (uint64_t)n * stride;
    }
    // To the present head's rows, where it is another one (the same for the warp).
    __device__ __forceinline__ void turn_to(const Q4Args& a, int h) {
        if (h == head) return;
        head = h;
        const int lane = threadIdx.x & 31, r0 = lane / kPieces, pc = lane % kPieces;
        kfrom = at(at(a.kcode.base, h, a.kcode.head), r0, a.kcode.token) + pc * 16;
        vfrom = at(at(a.vcode.base, h, a.vcode.head), r0, a.vcode.token) + pc * 16;
        // a row of parameters a lane, the keys' first
        if (lane < 16) pfrom = at(at(a.kpar.base, h, a.kpar.head), lane, a.kpar.token);
        else pfrom = at(at(a.vpar.base, h, a.vpar.head), lane - 16, a.vpar.token);
    }
    static constexpr int kStep = 32 / kPieces;                 // rows that a warp's 16-byte pieces make
    // A lane's places in a part at dst: of its first piece of a key row (8 or 16 rows on, a
    // piece's place is as many rows on), and of its row of parameters.
    __device__ __forceinline__ static uint32_t piece_place(uint32_t dst) {
        const int lane = threadIdx.x & 31;
        return dst + Tile::place(lane / kPieces, lane % kPieces);
    }
    __device__ __forceinline__ static uint32_t params_place(uint32_t dst) {
        const int lane = threadIdx.x & 31;
        return dst + (lane >> 4) * Tile::kTile + Tile::kCodes + (lane & 15) * 16;
    }
    // The parts of a chunk. In pages that hold whole chunks the parts' rows follow one another.
    __device__ __forceinline__ void copy(const Q4Args& a, uint32_t dst, const int (&blk)[kParts], int ch,
                                         const int (&lim)[kParts]) {
        const bool key = (threadIdx.x & 31) < 16;
        const uint32_t p_block = key ? a.kpar.block : a.vpar.block, p_token = key ? a.kpar.token : a.vpar.token;
        const uint32_t row0 = (ch & ((1 << (a.kp.page_shift - 4)) - 1)) * kPaChunk;
        const uint8_t* ks = at(at(kfrom, blk[0], a.kcode.block), row0, a.kcode.token);
        const uint8_t* vs = at(at(vfrom, blk[0], a.vcode.block), row0, a.vcode.token);
        const uint8_t* ps = at(at(pfrom, blk[0], p_block), row0, p_token);
        if (a.packed && a.kp.page_shift >= kPaChunkShift + (kParts == 4 ? 2 : 1) && lim[kParts - 1] == kPaChunk) {       // whole chunks whose rows follow one another
#pragma unroll
            for (int j = 0; j < kParts; ++j) {
                const uint32_t to = piece_place(dst) + j * C::kPartBytes;
#pragma unroll
                for (int i = 0; i < kEach; ++i) {
                    const int on = (j * kPaChunk + i * kStep) * Tile::kRow;
                    cp16_all(to + i * kStep * Tile::kRow, ks + on, policy);
                    cp16_all(to + i * kStep * Tile::kRow + Tile::kTile, vs + on, policy);
                }
                cp_params<4 * NG>(params_place(dst) + j * C::kPartBytes, ps + j * kPaChunk * 4 * NG, true, policy);
            }
            return;
        }
        const int r0 = (threadIdx.x & 31) / kPieces;
#pragma unroll
        for (int j = 0; j < kParts; ++j) {
            if (j > 0) {
                const uint32_t row = ((ch + j) & ((1 << (a.kp.page_shift - 4)) - 1)) * kPaChunk;
                ks = at(at(kfrom, blk[j], a.kcode.block), row, a.kcode.token);
                vs = at(at(vfrom, blk[j], a.vcode.block), row, a.vcode.token);
                ps = at(at(pfrom, blk[j], p_block), row, p_token);
            }
            const uint32_t to = piece_place(dst) + j * C::kPartBytes;
#pragma unroll
            for (int i = 0; i < kEach; ++i) {
                const bool on = r0 + i * kStep < lim[j];
                cp16_row(to + i * kStep * Tile::kRow, at(ks, i * kStep, a.kcode.token), on, policy);
                cp16_row(to + i * kStep * Tile::kRow + Tile::kTile, at(vs, i * kStep, a.vcode.token), on, policy);
            }
            cp_params<4 * NG>(params_place(dst) + j * C::kPartBytes, ps, (int)(threadIdx.x & 15) < lim[j], policy);
        }
    }
    template <typename Find>
    __device__ __forceinline__ void ask(const Q4Args& a, int s, Find&& find) {
        int lim[kParts] = {};
        if (s < steps) {
            int blk[kParts], ch0 = 0;
#pragma unroll
            for (int j = 0; j < kParts; ++j) {
                int ch, h;
                lim[j] = find(blk[j], ch, h, s, j);
                if (j == 0) {
                    ch0 = ch;
                    turn_to(a, h);
                }
            }
            copy(a, slot(s), blk, ch0, lim);
        }
#pragma unroll
        for (int i = 0; i + 2 < C::kStages; ++i)
#pragma unroll
            for (int j = 0; j < kParts; ++j) lims[i][j] = lims[i + 1][j];
#pragma unroll
        for (int j = 0; j < kParts; ++j) lims[C::kStages - 2][j] = lim[j];
        cp_commit();
    }
    // Step s of a unit.
    template <typename State, typename Find>
    __device__ __forceinline__ void step(const Q4Args& a, int s, State& st, Find&& find) {
        cp_wait<C::kStages - 2>();
        __syncwarp();
        int lim[kParts];
#pragma unroll
        for (int j = 0; j < kParts; ++j) lim[j] = lims[0][j];
        ask(a, s + C::kStages - 1, find);
        typename State::Four x[kParts];
#pragma unroll
        for (int j = 0; j < kParts; ++j) st.scores(slot(s) + j * C::kPartBytes, x[j]);
        typename State::Scales v[kParts];
#pragma unroll
        for (int j = 0; j < kParts; ++j) st.look(slot(s) + j * C::kPartBytes + Tile::kTile, v[j]);
        st.weigh(x, lim, v);
#pragma unroll
        for (int j = 0; j < kParts; ++j) st.add(slot(s) + j * C::kPartBytes + Tile::kTile, x[j], v[j]);
        __syncwarp();
    }
};

template <typename T_, int D_, bool kListed_, int kParts_>
struct Q4Base {
    using T = T_;
    using Args = Q4Args;
    static constexpr int D = D_, kParts = kParts_;
    static constexpr bool kListed = kListed_, kOdd = false, kGrouped = !kListed;
    static constexpr float kBias = 0.f;
};
template <typename T, int D, int NG, int NT, bool kListed, bool kUnits, class C = Q4Cfg<D, NT, kUnits>>
struct Q4Form : Q4Base<T, D, kListed, C::kParts> {
    using Joined = Q4Base<T, D, kListed, C::kParts>;
    using State = Q4State<T, D, NG, NT, C::kParts>;
    using Ring = Q4Ring<D, NG, NT, kUnits>;
    static constexpr int kCtas = C::kCtas, kStages = C::kStages, kRing = C::kRing, kSmem = C::kSmem;
    __device__ __forceinline__ static void start(State& st, const Q4Args& a, const uint16_t* q, int rows) {
        st.start(q, rows, a.scale2);
    }
};

template <typename T, int D, int NG, bool kListed>
cudaError_t launch_heads(const Q4Args& a, int W, cudaStream_t s) {
    return a.G <= 8 ? launch_paged<Q4Form<T, D, NG, 1, kListed, false>, Q4Form<T, D, NG, 1, kListed, true>>(a, W, s)
                    : launch_paged<Q4Form<T, D, NG, 2, kListed, false>, Q4Form<T, D, NG, 2, kListed, true>>(a, W, s);
}

template <typename T, bool kListed>
cudaError_t launch_int4(const Q4Args& a, int groups, int W, cudaStream_t s) {
    if (a.kp.dim == 64) return groups == 1 ? launch_heads<T, 64, 1, kListed>(a, W, s) : launch_heads<T, 64, 2, kListed>(a, W, s);
    return groups == 2 ? launch_heads<T, 128, 2, kListed>(a, W, s) : launch_heads<T, 128, 4, kListed>(a, W, s);
}

}  // namespace

// One translation unit a type and kind (paged_int4_attention_*.cu), which build side by side.
cudaError_t int4_attention_bf16(const Q4Args& a, int groups, int W, cudaStream_t s);
cudaError_t int4_attention_bf16_listed(const Q4Args& a, int groups, int W, cudaStream_t s);
cudaError_t int4_attention_fp16(const Q4Args& a, int groups, int W, cudaStream_t s);
cudaError_t int4_attention_fp16_listed(const Q4Args& a, int groups, int W, cudaStream_t s);

}  // namespace zs
