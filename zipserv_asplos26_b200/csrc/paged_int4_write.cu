// Rotary positions on q and k, and the step's k and v quantised to 4 bits into their
// slots of a paged KV cache (zs_rope_write_int4); rows of such a cache read back
// (zs_read_int4). Format: paged_int4.cuh.
//
// Every value is read once and written once.
//   * Writing goes as in paged_rope.cu (a warp walks a token's heads, 16 channels a
//     lane). The halves of a turned head lie apart, so its fp32 values pass through
//     shared memory and come back 16 neighbouring channels a lane; a group of 32 or 64
//     channels is then 2 or 4 lanes, whose minimum and maximum take one or two shuffles
//     each. k is quantised from the turned fp32 values, whose products are rounded one by
//     one (no fused multiply-add): codes are whole numbers, and the plain formula gives
//     the same ones. (x - c) / s is a product with 1 / s, and a quotient only where one of
//     a lane's is near the middle of two codes, where the two could round apart.
//   * Reading back, a lane turns 8 bytes of codes into 32 bytes, of K and of V.
//
// Measured in a graph (32 query and 8 KV heads of 128, bf16, groups of 64): 16411 tokens
// written 80.5 us (364 MB, 4.5 TB/s; 3440 warp instructions a token, issued in 68% of the
// cycles: quantising costs what is left of HBM; 72 registers, so 28 warps an SM: with 96
// and 20, 96 us), read back 20; 65553 tokens read back 69 (345 MB, 5.0 TB/s); 32 tokens
// 3.6 and 2.3.
#include "paged_int4.cuh"
#include "paged_rope.cuh"

namespace zs {
namespace {

constexpr int kInt4QBatch = 4, kInt4Batch = 1;       // passes (of q, of k and v) whose loads are in flight together

struct RopeInt4Args : RopeArgs {
    Int4View kp, vp;
};

// 16 channels of a row in their places of a head's buffer (20 floats for every 16, so
// that eight lanes' accesses fall on all banks).
constexpr int kHeadWords = 128 / 16 * 20;
__device__ __forceinline__ float* place16(float* head, int channel) { return head + channel / 16 * 20 + channel % 16; }

__device__ __forceinline__ float min_nan(float a, float b) {         // NaN where one is
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

template <typename T, int kLanes>      // kLanes: lanes a group (16 channels each)
__global__ void __launch_bounds__(kRopeThreads, 14) rope_write_int4_kernel(const RopeInt4Args a) {
    __shared__ __align__(16) float s_rows[kRopeThreads / 32][4 * kHeadWords];
    const int lane = threadIdx.x & 31;
    const long long warp = (long long)blockIdx.x * (kRopeThreads / 32) + (threadIdx.x >> 5);
    const long long n = warp / a.parts;
    if (n >= a.N) return;
    const int part = (int)(warp - n * a.parts);
    const int per_head = a.D / 16;            // lanes a head: 4 or 8
    const int heads_per = 32 / per_head;      // heads a pass of the warp
    const int sub = lane / per_head, c = lane - sub * per_head;
    const RopeLane me(a, n, c, true);
    const long long slot = a.slots[n];
    const long long cap = (long long)a.kp.num_blocks << a.kp.page_shift;
    const bool live = slot >= 0 && slot < cap;
    if ((slot < -1 || slot >= cap) && lane == 0) set_err(a.err, kErrPagedIndex);     // -1: padding
    const long long blk = slot >> a.kp.page_shift, row = slot & ((1 << a.kp.page_shift) - 1);
    float* mine = s_rows[threadIdx.x >> 5] + sub * (a.D / 16 * 20);
    // ---- q
    const int q_passes = (a.Hq + heads_per - 1) / heads_per, rows = 2 * a.Hkv;           // heads of k, then v
    int i0 = part;
    for (; i0 < q_passes; i0 += kInt4QBatch * a.parts) {
        uint4 x[kInt4QBatch], y[kInt4QBatch];
#pragma unroll
        for (int u = 0; u < kInt4QBatch; ++u) {
            const int h = (i0 + u * a.parts) * heads_per + sub;
            if (h < a.Hq) {          // plain loads: q may be turned in place
                const uint16_t* src = a.q + n * a.q_tok + h * a.q_head;
                x[u] = __ldcs(reinterpret_cast<const uint4*>(src + me.c0));
                y[u] = __ldcs(reinterpret_cast<const uint4*>(src + me.c1));
            }
        }
#pragma unroll
        for (int u = 0; u < kInt4QBatch; ++u) {
            const int h = (i0 + u * a.parts) * heads_per + sub;
            if (h < a.Hq) {
                if (me.turns) me.turn<T>(x[u], y[u], a.interleaved);
                uint16_t* dst = a.q_out + n * a.qo_tok + h * a.qo_head;
                __stcs(reinterpret_cast<uint4*>(dst + me.c0), x[u]);
                __stcs(reinterpret_cast<uint4*>(dst + me.c1), y[u]);
            }
        }
    }
    if (!live) return;
    // ---- k and v, passes q_passes on of the token's
    const int passes = (rows + heads_per - 1) / heads_per;
    i0 = q_passes <= part ? part - q_passes : (part + a.parts - q_passes % a.parts) % a.parts;
    for (; i0 < passes; i0 += kInt4Batch * a.parts) {
        uint4 x[kInt4Batch], y[kInt4Batch];
#pragma unroll
        for (int u = 0; u < kInt4Batch; ++u) {
            const int h = (i0 + u * a.parts) * heads_per + sub;
            x[u] = y[u] = make_uint4(0u, 0u, 0u, 0u);
            if (h < rows) {
                const bool key = h < a.Hkv;
                const uint16_t* src = key ? a.k + n * a.k_tok + h * a.k_head : a.v + n * a.v_tok + (h - a.Hkv) * a.v_head;
                x[u] = __ldcs(reinterpret_cast<const uint4*>(src + (key ? me.c0 : c * 16)));
                y[u] = __ldcs(reinterpret_cast<const uint4*>(src + (key ? me.c1 : c * 16 + 8)));
            }
        }
#pragma unroll
        for (int u = 0; u < kInt4Batch; ++u) {
            const int pass = i0 + u * a.parts, h = pass * heads_per + sub;
            if (pass >= passes) continue;      // the same for the warp
            // ---- keys and values: 16 neighbouring channels a lane, in fp32
            const bool key = h < a.Hkv;
            float f[16];
            {
                const uint32_t w[8] = {x[u].x, x[u].y, x[u].z, x[u].w, y[u].x, y[u].y, y[u].z, y[u].w};
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float2 p = unpack2<T>(w[j]);
                    f[2 * j] = p.x;
                    f[2 * j + 1] = p.y;
                }
            }
            if (key && me.turns) {
                auto turn = [&](float& p, float& q, int j) {
                    const float pc = __fmul_rn(p, me.cs[j]), qs = __fmul_rn(q, me.sn[j]);
                    const float qc = __fmul_rn(q, me.cs[j]), ps = __fmul_rn(p, me.sn[j]);
                    p = __fsub_rn(pc, qs);
                    q = __fadd_rn(qc, ps);
                };
                if (a.interleaved) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) turn(f[2 * j], f[2 * j + 1], j);
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) turn(f[j], f[8 + j], j);
                }
            }
            if (!a.interleaved && pass * heads_per < a.Hkv) {      // the same for the warp
                const int c0 = key ? me.c0 : c * 16, c1 = key ? me.c1 : c * 16 + 8;
                __syncwarp();
#pragma unroll
                for (int j = 0; j < 8; j += 4) {
                    *reinterpret_cast<float4*>(place16(mine, c0 + j)) = make_float4(f[j], f[j + 1], f[j + 2], f[j + 3]);
                    *reinterpret_cast<float4*>(place16(mine, c1 + j)) =
                        make_float4(f[8 + j], f[9 + j], f[10 + j], f[11 + j]);
                }
                __syncwarp();
#pragma unroll
                for (int j = 0; j < 16; j += 4) {
                    const float4 v = *reinterpret_cast<const float4*>(place16(mine, c * 16 + j));
                    f[j] = v.x;
                    f[j + 1] = v.y;
                    f[j + 2] = v.z;
                    f[j + 3] = v.w;
                }
            }
            // ---- the group's scale and centre
            float low = f[0], high = f[0];             // NaN once a value is
#pragma unroll
            for (int j = 1; j < 16; ++j) {
                low = min_nan(low, f[j]);
                high = max_nan(high, f[j]);
            }
#pragma unroll
            for (int o = 1; o < kLanes; o <<= 1) {
                low = min_nan(low, __shfl_xor_sync(~0u, low, o));
                high = max_nan(high, __shfl_xor_sync(~0u, high, o));
            }
            const float range = __fsub_rn(high, low);
            float s = __bfloat162float(__float2bfloat16_rn(__fdiv_rn(range, 15.f)));
            float centre = __bfloat162float(__float2bfloat16_rn(__fadd_rn(low, 8.f * s)));
            if (s < kSmallestScale) {
                s = 0.f;
                centre = __bfloat162float(__float2bfloat16_rn(low));
            }
            if (!(range < INFINITY)) {
                s = 0.f;
                centre = NAN;
            }
            // ---- codes: rounded by adding 1.5 2^23 (and 8), whose bits add up to as many times a constant
            const float by = s > 0.f ? __fdiv_rn(1.f, s) : 0.f;
            constexpr float kWhole = 12582920.f, kLeast = 12582912.f, kMost = 12582927.f;
            constexpr uint32_t kNone = 0u - 0x4B400000u * 0x11111111u;
            uint32_t code[2] = {kNone, kNone};
            bool close = false;            // to the middle of two codes: products are off by 2^-20 at most
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                f[j] = __fsub_rn(f[j], centre);
                const float m = fmaf(f[j], by, kWhole);
                close |= fabsf(fmaf(f[j], by, kWhole - m)) > 0.499998f;
                code[j / 8] += (uint32_t)__float_as_int(fminf(fmaxf(m, kLeast), kMost)) << (j % 8 * 4);
            }
            if (close) {                   // again, by quotients
                code[0] = code[1] = kNone;
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    const float m = rintf(__fdiv_rn(f[j], s)) + kWhole;
                    code[j / 8] += (uint32_t)__float_as_int(fminf(fmaxf(m, kLeast), kMost)) << (j % 8 * 4);
                }
            }
            if (!(s > 0.f)) code[0] = code[1] = 0x88888888u;
            // ---- the head's groups to its first lane
            const uint32_t sb = __bfloat16_as_ushort(__float2bfloat16_rn(s));
            const uint32_t cb = isnan(centre) ? 0x7FC0u : __bfloat16_as_ushort(__float2bfloat16_rn(centre));
            uint32_t ss[4], cc[4];
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int from = sub * per_head + min(g * kLanes, per_head - 1);
                ss[g] = __shfl_sync(~0u, sb, from);
                cc[g] = __shfl_sync(~0u, cb, from);
            }
            if (h >= rows) continue;
            const Int4View& to = key ? a.kp : a.vp;
            const long long head = h - (key ? 0 : a.Hkv);
            *reinterpret_cast<uint2*>(to.codes + blk * to.c_block + row * to.c_token + head * to.c_head + c * 8) =
                make_uint2(code[0], code[1]);
            if (c == 0) {
                uint16_t* par = to.params + blk * to.p_block + row * to.p_token + head * to.p_head;
                if (to.groups == 1)
                    *reinterpret_cast<uint32_t*>(par) = ss[0] | cc[0] << 16;
                else if (to.groups == 2)
                    *reinterpret_cast<uint2*>(par) = make_uint2(ss[0] | ss[1] << 16, cc[0] | cc[1] << 16);
                else
                    *reinterpret_cast<uint4*>(par) = make_uint4(ss[0] | ss[1] << 16, ss[2] | ss[3] << 16,
                                                                cc[0] | cc[1] << 16, cc[2] | cc[3] << 16);
            }
        }
    }
}

// ---- reading back: a lane has 16 channels of a row of K and of V, 8 bytes of codes each,
// and writes 32 bytes at once
constexpr int kReadThreads = 256;

struct ReadArgs {
    Int4View kp, vp;
    const long long* slots;
    uint16_t* k_out;
    uint16_t* v_out;
    long long items;              // of 16 channels of K and of V
    int per_token;                // items a token
    int piece_shift;              // log2(D / 16)
    int group_shift;              // log2(group / 16)
    unsigned* err;
};

struct Read16 {
    uint2 w;
    uint32_t s, c;                // scale and centre
};

__device__ __forceinline__ Read16 read16(const Int4View& p, long long blk, long long row, int h, int piece, int g) {
    Read16 r;
    r.w = __ldcs(reinterpret_cast<const uint2*>(p.codes + blk * p.c_block + row * p.c_token + h * p.c_head + piece * 8));
    const uint16_t* par = p.params + blk * p.p_block + row * p.p_token + h * p.p_head + g;
    r.s = __ldg(par);
    r.c = __ldg(par + p.groups);
    return r;
}

template <typename T>
__device__ __forceinline__ void write16(uint16_t* to, const Read16& x, bool live) {
    const float s = bf16_bits_to_float(x.s), c = bf16_bits_to_float(x.c);
    uint32_t r[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const uint32_t w = j < 4 ? x.w.x : x.w.y;
        // codes as floats: 2^23 + u, less 2^23 + 8
        const float lo = __uint_as_float((w >> (j % 4 * 8) & 15u) | 0x4B000000u) - 8388616.f;
        const float hi = __uint_as_float((w >> (j % 4 * 8 + 4) & 15u) | 0x4B000000u) - 8388616.f;
        r[j] = live ? pack2<T>(__fmaf_rn(s, lo, c), __fmaf_rn(s, hi, c)) : 0u;       // s times a code is exact
    }
    asm volatile("st.global.cs.v4.b32 [%0], {%1, %2, %3, %4};" ::"l"(to), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]) : "memory");
    asm volatile("st.global.cs.v4.b32 [%0], {%1, %2, %3, %4};" ::"l"(to + 8), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]) : "memory");
}

template <typename T>
__global__ void __launch_bounds__(kReadThreads) read_int4_kernel(const ReadArgs a) {
    const long long item = (long long)blockIdx.x * kReadThreads + threadIdx.x;
    if (item >= a.items) return;
    const long long n = div_nonneg(item, a.per_token);
    const int in_token = (int)(item - n * a.per_token);
    const int h = in_token >> a.piece_shift, piece = in_token & ((1 << a.piece_shift) - 1);
    const long long slot = a.slots[n], cap = (long long)a.kp.num_blocks << a.kp.page_shift;
    const bool live = slot >= 0 && slot < cap;
    Read16 k{}, v{};
    if (live) {
        const long long blk = slot >> a.kp.page_shift, row = slot & ((1 << a.kp.page_shift) - 1);
        k = read16(a.kp, blk, row, h, piece, piece >> a.group_shift);
        v = read16(a.vp, blk, row, h, piece, piece >> a.group_shift);
    } else if (slot != -1) {
        set_err(a.err, kErrPagedIndex);
    }
    write16<T>(a.k_out + item * 16, k, live);
    write16<T>(a.v_out + item * 16, v, live);
}

}  // namespace
}  // namespace zs

extern "C" int zs_rope_write_int4(const ZsRopeWriteInt4* p) {
    using namespace zs;
    RopeInt4Args a{};
    if (!p || (p->dtype != ZS_BF16 && p->dtype != ZS_FP16) || !make_int4_pool(&p->k_pool, &a.kp) ||
        !make_int4_pool(&p->v_pool, &a.vp) || !same_int4_pools(p->k_pool, p->v_pool) ||
        !rope_args(p, a.kp.heads, a.kp.dim, &a))
        return cudaErrorInvalidValue;
    if (a.N == 0) return cudaSuccess;
    cudaStream_t s = (cudaStream_t)p->stream;
    const unsigned grid = rope_grid(&a);
    const bool wide = p->k_pool.group == 64;
    if (p->dtype == ZS_BF16) {
        if (wide) rope_write_int4_kernel<__nv_bfloat16, 4><<<grid, kRopeThreads, 0, s>>>(a);
        else rope_write_int4_kernel<__nv_bfloat16, 2><<<grid, kRopeThreads, 0, s>>>(a);
    } else {
        if (wide) rope_write_int4_kernel<__half, 4><<<grid, kRopeThreads, 0, s>>>(a);
        else rope_write_int4_kernel<__half, 2><<<grid, kRopeThreads, 0, s>>>(a);
    }
    return cudaGetLastError();
}

extern "C" int zs_read_int4(const ZsReadInt4* p) {
    using namespace zs;
    ReadArgs a{};
    if (!p || p->N < 0 || (p->dtype != ZS_BF16 && p->dtype != ZS_FP16) || !make_int4_pool(&p->k_pool, &a.kp) ||
        !make_int4_pool(&p->v_pool, &a.vp) || !same_int4_pools(p->k_pool, p->v_pool))
        return cudaErrorInvalidValue;
    if (p->N == 0) return cudaSuccess;
    if (!p->slots || !p->k_out || !p->v_out || !aligned16p(p->k_out) || !aligned16p(p->v_out)) return cudaErrorInvalidValue;
    const long long len = (long long)p->N * a.kp.heads * a.kp.dim;
    if (rows_meet(p->k_out, 1, 1, len, len, len, p->v_out, len)) return cudaErrorInvalidValue;
    a.slots = reinterpret_cast<const long long*>(p->slots);
    a.k_out = p->k_out;
    a.v_out = p->v_out;
    a.piece_shift = a.kp.dim == 64 ? 2 : 3;
    a.group_shift = p->k_pool.group == 32 ? 1 : 2;
    a.per_token = a.kp.heads << a.piece_shift;
    a.items = (long long)p->N * a.per_token;
    a.err = p->err;
    const long long grid = (a.items + kReadThreads - 1) / kReadThreads;
    if (a.kp.heads > INT32_MAX >> 3 || grid > INT32_MAX) return cudaErrorInvalidValue;
    if (p->dtype == ZS_BF16) read_int4_kernel<__nv_bfloat16><<<(unsigned)grid, kReadThreads, 0, (cudaStream_t)p->stream>>>(a);
    else read_int4_kernel<__half><<<(unsigned)grid, kReadThreads, 0, (cudaStream_t)p->stream>>>(a);
    return cudaGetLastError();
}
