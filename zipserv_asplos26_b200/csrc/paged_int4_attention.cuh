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
//     two operands, with one shift for every four. What sits four bits up counts 16-fold
//     and has sums of its own.
//   * Scores: sum_g s_g (q_g . u_g) + sum_g (c_g - 8 s_g) sum(q_g). The second part is a
//     product too, of the row of parameters with q's sums (in three bf16 parts, 24 bits).
//     Keys are the rows (16 tokens), heads the columns, 8 or twice 8.
//   * Outputs: sum_t (p_t s_t) (u_t - 8) + sum_t p_t c_t. The codes are centred by a
//     bf16x2 add, exact: sums of codes from 0 to 15 would be far larger than the outputs
//     that are left of them, and a tensor core's sums lose low bits. p s, and p for the
//     centres, are fed as a bf16 high part plus its bf16 remainder (2^-16 is left out).
// q (bf16) and p s are scaled by 2^64 on the way in, so that neither they nor the
// products leave fp32's range; powers of two are exact.
//
// The maximum that exponents refer to follows the scores only where one passes it by 8
// or more (base 2), so that most chunks need no maximum over their lanes.
#pragma once

#include "paged_int4.cuh"
#include "paged_runs.cuh"

namespace zs {

struct Q4Args : PaArgs {          // kp and vp: the codes, strides in bytes
    const uint16_t* kpar;
    const uint16_t* vpar;
    long long kpar_block, kpar_token, kpar_head, vpar_block, vpar_token, vpar_head;
};

namespace {

constexpr float kTwo64 = 18446744073709551616.f;
constexpr float kTwo24 = 16777216.f;
constexpr uint32_t kLowCodes = 0x000F000Fu, kHighCodes = 0x00F000F0u;

template <int D>
struct Q4Tile {
    static constexpr int kRow = D / 2;                       // bytes of a row's codes
    static constexpr int kCodes = kPaChunk * kRow;
    static constexpr int kParams = kPaChunk * 16;            // a row's parameters in 16 bytes
    static constexpr int kTile = kCodes + kParams;           // one K or V chunk
    // the 16-byte piece of a row in shared memory: eight rows' pieces fill all banks
    __device__ __forceinline__ static int place(int r, int piece) {
        return r * kRow + (piece ^ (D == 128 ? (r >> 1) & 3 : (r >> 2) & 1)) * 16;
    }
};

template <int D, int NT>
struct Q4Cfg {
    static constexpr int kCtas = NT == 1 ? 4 : 3;
    static constexpr int kStages = 4;
    static constexpr int kChunkBytes = 2 * Q4Tile<D>::kTile;
    static constexpr int kPiece = kPaRows * (D + 2) * 4;     // a warp's piece in the units kernel
    static constexpr int kRing = kStages * kChunkBytes > kPiece ? kStages * kChunkBytes : kPiece;
    static constexpr int kSmem = kPaWarps * kRing;
};

__device__ __forceinline__ void ldsm2(uint32_t (&r)[2], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x2.shared.b16 {%0, %1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldsm2t(uint32_t (&r)[2], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x2.trans.shared.b16 {%0, %1}, [%2];"
                 : "=r"(r[0]), "=r"(r[1])
                 : "r"(a)
                 : "memory");
}
__device__ __forceinline__ float exp2_fast(float x) {        // 2 ulp; below 2^-126 it is zero
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Bytes bytes (4, 8 or 16) of parameters.
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
// The kN scales (bf16) at the start of a row of parameters, in fp32.
template <int kN>
__device__ __forceinline__ void ld_scales(float (&s)[kN], uint32_t at) {
    uint32_t w[2];
    if constexpr (kN == 4)
        asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(at) : "memory");
    else
        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[0]) : "r"(at) : "memory");
#pragma unroll
    for (int g = 0; g < kN; ++g) s[g] = g & 1 ? __uint_as_float(w[g / 2] & 0xFFFF0000u) : bf16_bits_to_float(w[g / 2]);
}
__device__ __forceinline__ uint32_t add_bf16x2(uint32_t a, uint32_t b) {
    const __nv_bfloat162 r = __hadd2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
}

// What a warp holds of a unit of up to NT x 8 heads. A lane has heads 2 (lane % 4) and
// the next of each eight; of scores, tokens lane / 4 and lane / 4 + 8; of outputs the
// four channels from 4 (lane / 4) on of each 32.
template <typename T, int D, int NG, int NT>
struct Q4State {
    static constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
    static constexpr int kBlocks = D / 32, kPer = kBlocks / NG;      // 32 channels: a 16-byte piece of a row
    using Bf = __nv_bfloat16;
    uint32_t qf[NT][kBlocks][2][2];    // q of the even, odd channels
    uint32_t zf[NT][3];                // of what meets the parameters: -8 sum(q_g), sum(q_g), in three parts
    float o[NT][kBlocks][2][4];        // sums of the even, odd channels
    float z[NT][4];                    // sums of p times the parameters
    float m[NT][2], l[NT][2];

    struct Weights {
        float p[NT][4];
    };

    __device__ __forceinline__ void start(const uint16_t* q, int rows) {
        const int lane = threadIdx.x & 31;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int head = nt * 8 + (lane >> 2);
            float sum[NG];
#pragma unroll
            for (int g = 0; g < NG; ++g) sum[g] = 0.f;
#pragma unroll
            for (int b = 0; b < kBlocks; ++b) {
                uint4 x = make_uint4(0u, 0u, 0u, 0u);
                if (head < rows) x = *reinterpret_cast<const uint4*>(q + (long long)head * D + b * 32 + (lane & 3) * 8);
                uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 f = unpack2<T>(w[i]);
                    sum[b / kPer] += f.x + f.y;
                    if constexpr (kBf16) w[i] = pack2<T>(f.x * kTwo64, f.y * kTwo64);
                }
                // codes of channels i and i + 4 lie 16 bits apart
                qf[nt][b][0][0] = __byte_perm(w[0], w[2], 0x5410);
                qf[nt][b][0][1] = __byte_perm(w[1], w[3], 0x5410);
                qf[nt][b][1][0] = __byte_perm(w[0], w[2], 0x7632);
                qf[nt][b][1][1] = __byte_perm(w[1], w[3], 0x7632);
            }
            float e[2] = {0.f, 0.f};                 // of parameters 2 (lane % 4) and the next
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                sum[g] += __shfl_xor_sync(~0u, sum[g], 1);
                sum[g] += __shfl_xor_sync(~0u, sum[g], 2);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    if ((lane & 3) * 2 + i == g) e[i] = -8.f * sum[g];
                    if ((lane & 3) * 2 + i == NG + g) e[i] = sum[g];
                }
            }
#pragma unroll
            for (int i = 0; i < 3; ++i) {
                zf[nt][i] = pack2<Bf>(e[0], e[1]);
                const float2 back = unpack2<Bf>(zf[nt][i]);
                e[0] -= back.x;
                e[1] -= back.y;
            }
#pragma unroll
            for (int b = 0; b < kBlocks; ++b)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[nt][b][0][i] = o[nt][b][1][i] = 0.f;
#pragma unroll
            for (int i = 0; i < 4; ++i) z[nt][i] = 0.f;
            m[nt][0] = m[nt][1] = -INFINITY;
            l[nt][0] = l[nt][1] = 0.f;
        }
    }

    // Scores (times scale2) of the chunk whose keys are at kt.
    __device__ __forceinline__ void scores(uint32_t kt, float scale2, float (&x)[NT][4]) {
        const int lane = threadIdx.x & 31, r = lane & 15, half = lane >> 4;
        const uint32_t par = kt + Q4Tile<D>::kCodes;
        float sc[2][NG], c[NT][4], s[NT][4];
        ld_scales<NG>(sc[0], par + (lane >> 2) * 16);
        ld_scales<NG>(sc[1], par + ((lane >> 2) + 8) * 16);
        uint32_t pr[2];
        ldsm2(pr, par + r * 16);
        const uint32_t a2[4] = {pr[0], pr[1], pr[0], pr[1]}, a1[4] = {pr[0], pr[1], 0u, 0u};
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int i = 0; i < 4; ++i) s[nt][i] = c[nt][i] = 0.f;
            mma16816(c[nt], a2, zf[nt][0], zf[nt][1], Bf());
            mma16816(c[nt], a1, zf[nt][2], 0u, Bf());
        }
        float e[NT][2][4];
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
                    if (b % kPer == 0) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) e[nt][0][j] = e[nt][1][j] = 0.f;
                    }
                    mma16816(e[nt][0], lo, qf[nt][b][0][0], qf[nt][b][0][1], T());
                    mma16816(e[nt][1], hi, qf[nt][b][1][0], qf[nt][b][1][1], T());
                    if (b % kPer == kPer - 1) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) s[nt][j] += sc[j >> 1][g] * (e[nt][0][j] + e[nt][1][j] * 0.0625f);
                    }
                }
            }
        }
        // codes in steps of 2^-133 against q times 2^64, or in steps of 2^-24
        const float unit = kBf16 ? scale2 * (kTwo64 * 32.f) : scale2 * kTwo24;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i) x[nt][i] = s[nt][i] * unit + c[nt][i] * scale2;
    }

    // Weights 2^(x - m) of a chunk's first `lim` tokens.
    __device__ __forceinline__ void weigh(float (&x)[NT][4], int lim, Weights& w) {
        const int t = (threadIdx.x & 31) >> 2;
        bool up = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (t + (i >> 1) * 8 >= lim) x[nt][i] = -INFINITY;
                up |= x[nt][i] > m[nt][i & 1] + 8.f;
            }
        if (__any_sync(~0u, up)) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    float mx = fmaxf(x[nt][j], x[nt][2 + j]);
#pragma unroll
                    for (int k = 4; k < 32; k <<= 1) mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, k));
                    const float mn = fmaxf(m[nt][j], mx);
                    const float keep = exp2_fast(m[nt][j] - (mn == -INFINITY ? 0.f : mn));
                    m[nt][j] = mn;
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
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const float ref = m[nt][j] == -INFINITY ? 0.f : m[nt][j];
                w.p[nt][j] = exp2_fast(x[nt][j] - ref);
                w.p[nt][2 + j] = exp2_fast(x[nt][2 + j] - ref);
                l[nt][j] += w.p[nt][j] + w.p[nt][2 + j];
            }
    }

    // Four weights (a lane's tokens and heads) as the fragments of their two parts.
    struct Parts {
        uint32_t hi[2], lo[2];
    };
    __device__ __forceinline__ static void split(float a, float b, float c, float d, Parts& f) {
        const uint32_t x = pack2<Bf>(a, b), y = pack2<Bf>(c, d);
        const float2 xb = unpack2<Bf>(x), yb = unpack2<Bf>(y);
        f.hi[0] = transpose8(x);
        f.hi[1] = transpose8(y);
        f.lo[0] = transpose8(pack2<Bf>(a - xb.x, b - xb.y));
        f.lo[1] = transpose8(pack2<Bf>(c - yb.x, d - yb.y));
    }

    // Adds the chunk whose values are at vt.
    __device__ __forceinline__ void add(uint32_t vt, const Weights& w) {
        const int lane = threadIdx.x & 31, r = lane & 15, half = lane >> 4;
        const uint32_t par = vt + Q4Tile<D>::kCodes;
        float sc[2][NG];
        ld_scales<NG>(sc[0], par + (lane >> 2) * 16);
        ld_scales<NG>(sc[1], par + ((lane >> 2) + 8) * 16);
        uint32_t pr[2];
        ldsm2t(pr, par + r * 16);
        const uint32_t a0[4] = {pr[0], 0u, pr[1], 0u};
        Parts f[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            split(w.p[nt][0], w.p[nt][1], w.p[nt][2], w.p[nt][3], f[nt]);
            mma16816(z[nt], a0, f[nt].hi[0], f[nt].hi[1], Bf());
            mma16816(z[nt], a0, f[nt].lo[0], f[nt].lo[1], Bf());
        }
#pragma unroll
        for (int b2 = 0; b2 < kBlocks / 2; ++b2) {
            uint32_t v[4];
            ldsm4t(v, vt + Q4Tile<D>::place(r, b2 * 2 + half));
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int b = b2 * 2 + i, g = b / kPer;
                if (b % kPer == 0) {
                    const float s0 = sc[0][g] * kTwo64, s1 = sc[1][g] * kTwo64;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
                        split(w.p[nt][0] * s0, w.p[nt][1] * s0, w.p[nt][2] * s1, w.p[nt][3] * s1, f[nt]);
                }
                const uint32_t t[4] = {v[i * 2], v[i * 2] >> 8, v[i * 2 + 1], v[i * 2 + 1] >> 8};
                uint32_t lo[4], hi[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    lo[j] = add_bf16x2(t[j] & kLowCodes, 0x80088008u);       // - 8 steps
                    hi[j] = add_bf16x2(t[j] & kHighCodes, 0x80808080u);      // - 128 steps
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    mma16816(o[nt][b][0], lo, f[nt].hi[0], f[nt].hi[1], Bf());
                    mma16816(o[nt][b][1], hi, f[nt].hi[0], f[nt].hi[1], Bf());
                    mma16816(o[nt][b][0], lo, f[nt].lo[0], f[nt].lo[1], Bf());
                    mma16816(o[nt][b][1], hi, f[nt].lo[0], f[nt].lo[1], Bf());
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
                        const float unit = kTwo64 * (y ? 2.f : 32.f);
                        o[nt][b][y][j] = o[nt][b][y][j] * unit + c;
                        o[nt][b][y][2 + j] = o[nt][b][y][2 + j] * unit + c;
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
                if (lse && lane < 4) lse[row] = log_sum(m[nt][j], l[nt][j], 0.f);
            }
    }
    // A piece: unnormalised rows [rows][D], and [rows][2] maxima and sums.
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
                if (lane < 4) *reinterpret_cast<float2*>(ml + row * 2) = make_float2(m[nt][j], l[nt][j]);
            }
    }
};

// A warp's ring: kStages - 1 chunks are on their way while one is worked on.
template <int D, int NG, int NT>
struct Q4Ring {
    using C = Q4Cfg<D, NT>;
    using Tile = Q4Tile<D>;
    uint32_t base;
    uint64_t policy;
    int steps;
    int lims[C::kStages - 1];      // of the chunks on their way, oldest first

    __device__ __forceinline__ void start(uint32_t at, int n) {
        base = at;
        policy = evict_first_policy();
        steps = n;
        // rows of parameters shorter than 16 bytes end in zeros
        if constexpr (NG < 4) {
            const int lane = threadIdx.x & 31;
#pragma unroll
            for (int s = 0; s < C::kStages; ++s)
                asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(
                                 slot(s) + (lane >> 4) * Tile::kTile + Tile::kCodes + (lane & 15) * 16),
                             "r"(0)
                             : "memory");
            __syncwarp();
        }
    }
    __device__ __forceinline__ uint32_t slot(int s) const { return base + (s % C::kStages) * C::kChunkBytes; }
    __device__ __forceinline__ void copy(const Q4Args& a, uint32_t dst, int blk, int ch, int h, int lim) {
        constexpr int kPieces = D / 32;                // 16-byte pieces a row
        const int lane = threadIdx.x & 31;
        const int row0 = (ch & ((1 << (a.kp.page_shift - 4)) - 1)) * kPaChunk;
        const uint8_t* ks = static_cast<const uint8_t*>(a.kp.data) + h * a.kp.s_head + blk * a.kp.s_block + row0 * a.kp.s_token;
        const uint8_t* vs = static_cast<const uint8_t*>(a.vp.data) + h * a.vp.s_head + blk * a.vp.s_block + row0 * a.vp.s_token;
#pragma unroll
        for (int i = 0; i < kPaChunk * kPieces / 32; ++i) {
            const int x = i * 32 + lane, r = x / kPieces, pc = x % kPieces;
            const uint32_t to = dst + Tile::place(r, pc);
            cp16(to, ks + r * a.kp.s_token + pc * 16, r < lim, policy);
            cp16(to + Tile::kTile, vs + r * a.vp.s_token + pc * 16, r < lim, policy);
        }
        // a row of parameters a lane, the keys' first
        const int r = lane & 15;
        const bool v = lane >> 4;
        const uint16_t* src = v ? a.vpar + h * a.vpar_head + blk * a.vpar_block + (row0 + r) * a.vpar_token
                                : a.kpar + h * a.kpar_head + blk * a.kpar_block + (row0 + r) * a.kpar_token;
        cp_params<4 * NG>(dst + (v ? Tile::kTile : 0) + Tile::kCodes + r * 16, src, r < lim, policy);
    }
    template <typename Find>
    __device__ __forceinline__ void ask(const Q4Args& a, int s, Find&& find) {
        int lim = 0;
        if (s < steps) {
            int blk, ch, h;
            lim = find(blk, ch, h, s);
            copy(a, slot(s), blk, ch, h, lim);
        }
        cp_commit();
#pragma unroll
        for (int i = 0; i + 2 < C::kStages; ++i) lims[i] = lims[i + 1];
        lims[C::kStages - 2] = lim;
    }
    // Step s of a unit.
    template <typename State, typename Find>
    __device__ __forceinline__ void step(const Q4Args& a, int s, State& st, Find&& find) {
        typename State::Weights w;
        cp_wait<C::kStages - 2>();
        __syncwarp();
        const int lim = lims[0];
        ask(a, s + C::kStages - 1, find);
        {
            decltype(w.p) x;
            st.scores(slot(s), a.scale2, x);
            st.weigh(x, lim, w);
        }
        st.add(slot(s) + Tile::kTile, w);
        __syncwarp();
    }
};

template <typename T_, int D_, bool kListed_>
struct Q4Base {
    using T = T_;
    using Args = Q4Args;
    static constexpr int D = D_;
    static constexpr bool kListed = kListed_, kOdd = false;
    static constexpr float kBias = 0.f;
};
template <typename T, int D, int NG, int NT, bool kListed>
struct Q4Form : Q4Base<T, D, kListed>, Q4Cfg<D, NT> {
    using Joined = Q4Base<T, D, kListed>;
    using State = Q4State<T, D, NG, NT>;
    using Ring = Q4Ring<D, NG, NT>;
};

template <typename T, int D, int NG, bool kListed>
cudaError_t launch_heads(const Q4Args& a, int W, cudaStream_t s) {
    return a.G <= 8 ? launch_paged<Q4Form<T, D, NG, 1, kListed>>(a, W, s) : launch_paged<Q4Form<T, D, NG, 2, kListed>>(a, W, s);
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
