// Rotary positions on q and k, and the step's k and v quantised to 4 bits into their
// slots of a paged KV cache (zs_rope_write_int4); rows of such a cache read back
// (zs_read_int4). Format: paged_int4.cuh.
//
// Both are bound by HBM: every value is read once and written once.
//   * Writing goes as in paged_rope.cu (a warp walks a token's heads, 16 channels a
//     lane). The halves of a turned head lie apart, so its fp32 values pass through
//     shared memory and come back 16 neighbouring channels a lane; a group of 32 or 64
//     channels is then 2 or 4 lanes, whose minimum and maximum take one or two shuffles
//     each. k is quantised from the turned fp32 values, whose products are rounded one by
//     one (no fused multiply-add): codes are whole numbers, and the plain formula gives
//     the same ones. (x - c) / s is a product with 1 / s, and a quotient only near the
//     middle of two codes, where the two could round apart.
//   * Reading back, a lane turns 4 bytes of codes into 16 bytes.
#include "paged_int4.cuh"
#include "paged_rope.cuh"

namespace zs {
namespace {

constexpr int kInt4Batch = 2;       // passes whose loads are in flight together

struct RopeInt4Args : RopeArgs {
    Int4View kp, vp;
};

// 16 channels of a row in their places of a head's buffer (20 floats for every 16, so
// that eight lanes' accesses fall on all banks).
constexpr int kHeadWords = 128 / 16 * 20;
__device__ __forceinline__ float* place16(float* head, int channel) { return head + channel / 16 * 20 + channel % 16; }

template <typename T, int kLanes>      // kLanes: lanes a group (16 channels each)
__global__ void __launch_bounds__(kRopeThreads) rope_write_int4_kernel(const RopeInt4Args a) {
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
    const int rows = a.Hq + 2 * a.Hkv;                       // heads of q, then k, then v
    const int passes = (rows + heads_per - 1) / heads_per;
    for (int i0 = part; i0 < passes; i0 += kInt4Batch * a.parts) {
        uint4 x[kInt4Batch], y[kInt4Batch];
#pragma unroll
        for (int u = 0; u < kInt4Batch; ++u) {
            const int h = (i0 + u * a.parts) * heads_per + sub;
            const uint16_t* src = nullptr;
            int c0 = me.c0, c1 = me.c1;
            if (h < a.Hq) {
                src = a.q + n * a.q_tok + h * a.q_head;
            } else if (h < rows && live) {
                if (h < a.Hq + a.Hkv) {
                    src = a.k + n * a.k_tok + (h - a.Hq) * a.k_head;
                } else {
                    src = a.v + n * a.v_tok + (h - a.Hq - a.Hkv) * a.v_head;
                    c0 = c * 16;
                    c1 = c0 + 8;
                }
            }
            x[u] = y[u] = make_uint4(0u, 0u, 0u, 0u);
            if (src) {               // plain loads: q may be turned in place
                x[u] = __ldcs(reinterpret_cast<const uint4*>(src + c0));
                y[u] = __ldcs(reinterpret_cast<const uint4*>(src + c1));
            }
        }
#pragma unroll
        for (int u = 0; u < kInt4Batch; ++u) {
            const int pass = i0 + u * a.parts, h = pass * heads_per + sub;
            if (h < a.Hq) {
                if (me.turns) me.turn<T>(x[u], y[u], a.interleaved);
                uint16_t* dst = a.q_out + n * a.qo_tok + h * a.qo_head;
                __stcs(reinterpret_cast<uint4*>(dst + me.c0), x[u]);
                __stcs(reinterpret_cast<uint4*>(dst + me.c1), y[u]);
            }
            if (!live || pass >= passes || (pass + 1) * heads_per <= a.Hq) continue;      // the same for the warp
            // ---- keys and values: 16 neighbouring channels a lane, in fp32
            const bool key = h < a.Hq + a.Hkv;
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
            if (!a.interleaved) {              // the same for the warp
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
            float low = f[0], high = f[0], odd = 0.f;
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                low = fminf(low, f[j]);
                high = fmaxf(high, f[j]);
                odd += f[j] * 0.f;             // NaN once a value is not finite
            }
#pragma unroll
            for (int o = 1; o < kLanes; o <<= 1) {
                low = fminf(low, __shfl_xor_sync(~0u, low, o));
                high = fmaxf(high, __shfl_xor_sync(~0u, high, o));
                odd += __shfl_xor_sync(~0u, odd, o);
            }
            const float range = __fsub_rn(high, low);
            float s = __bfloat162float(__float2bfloat16_rn(__fdiv_rn(range, 15.f)));
            float centre = __bfloat162float(__float2bfloat16_rn(__fadd_rn(low, 8.f * s)));
            if (s < kSmallestScale) {
                s = 0.f;
                centre = __bfloat162float(__float2bfloat16_rn(low));
            }
            if (!(odd == 0.f && range < INFINITY)) {
                s = 0.f;
                centre = NAN;
            }
            // ---- codes
            const float by = s > 0.f ? __fdiv_rn(1.f, s) : 0.f;
            uint32_t code[2] = {0u, 0u};
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const float d = __fsub_rn(f[j], centre);
                float t = __fmul_rn(d, by), r = rintf(t);
                if (fabsf(t - r) > 0.4999f) r = rintf(__fdiv_rn(d, s));
                r = s > 0.f ? fminf(fmaxf(r, -8.f), 7.f) : 0.f;
                code[j / 8] |= (uint32_t)((int)r + 8) << (j % 8 * 4);
            }
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
            if (h < a.Hq || h >= rows) continue;
            const Int4View& to = key ? a.kp : a.vp;
            const long long head = h - a.Hq - (key ? 0 : a.Hkv);
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

// ---- reading back
constexpr int kReadThreads = 256;
constexpr int kReadBatch = 4;       // items of a thread, their loads in flight together

struct ReadArgs {
    Int4View kp, vp;
    const long long* slots;
    uint16_t* k_out;
    uint16_t* v_out;
    long long items;              // of 8 channels, of K or of V
    int piece_shift;              // log2(D / 8)
    int group_shift;              // log2(group / 8)
    unsigned* err;
};

template <typename T>
__device__ __forceinline__ uint4 values_of(uint32_t w, float s, float c) {
    uint32_t r[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float lo = (float)((int)(w >> (8 * j) & 15u) - 8), hi = (float)((int)(w >> (8 * j + 4) & 15u) - 8);
        r[j] = pack2<T>(__fadd_rn(c, s * lo), __fadd_rn(c, s * hi));          // s times a code is exact
    }
    return make_uint4(r[0], r[1], r[2], r[3]);
}

template <typename T>
__global__ void __launch_bounds__(kReadThreads) read_int4_kernel(const ReadArgs a) {
    const bool values = blockIdx.y;           // of K, or of V
    const Int4View& p = values ? a.vp : a.kp;
    uint16_t* out = values ? a.v_out : a.k_out;
    const long long cap = (long long)p.num_blocks << p.page_shift;
    const long long first = (long long)blockIdx.x * (kReadThreads * kReadBatch) + threadIdx.x;
    uint32_t w[kReadBatch], s[kReadBatch], c[kReadBatch];
#pragma unroll
    for (int i = 0; i < kReadBatch; ++i) {
        const long long item = first + i * kReadThreads;
        w[i] = s[i] = c[i] = 0u;
        if (item >= a.items) continue;
        const long long head_row = item >> a.piece_shift;      // token and head
        const int piece = (int)(item & ((1 << a.piece_shift) - 1));
        const long long n = div_nonneg(head_row, p.heads), h = head_row - n * p.heads;
        const long long slot = a.slots[n];
        if (slot < 0 || slot >= cap) {
            if (slot != -1) set_err(a.err, kErrPagedIndex);
            continue;
        }
        const long long blk = slot >> p.page_shift, row = slot & ((1 << p.page_shift) - 1);
        w[i] = __ldg(reinterpret_cast<const uint32_t*>(p.codes + blk * p.c_block + row * p.c_token + h * p.c_head + piece * 4));
        const uint16_t* par = p.params + blk * p.p_block + row * p.p_token + h * p.p_head + (piece >> a.group_shift);
        s[i] = __ldg(par);
        c[i] = __ldg(par + p.groups);
    }
#pragma unroll
    for (int i = 0; i < kReadBatch; ++i) {
        const long long item = first + i * kReadThreads;
        if (item < a.items)
            __stcs(reinterpret_cast<uint4*>(out) + item,
                   values_of<T>(w[i], bf16_bits_to_float(s[i]), bf16_bits_to_float(c[i])));
    }
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
    a.slots = reinterpret_cast<const long long*>(p->slots);
    a.k_out = p->k_out;
    a.v_out = p->v_out;
    a.piece_shift = a.kp.dim == 64 ? 3 : 4;
    a.group_shift = p->k_pool.group == 32 ? 2 : 3;
    a.items = ((long long)p->N * a.kp.heads) << a.piece_shift;
    a.err = p->err;
    const long long ctas = (a.items + kReadThreads * kReadBatch - 1) / (kReadThreads * kReadBatch);
    if (ctas > INT32_MAX) return cudaErrorInvalidValue;
    const dim3 grid((unsigned)ctas, 2);
    if (p->dtype == ZS_BF16) read_int4_kernel<__nv_bfloat16><<<grid, kReadThreads, 0, (cudaStream_t)p->stream>>>(a);
    else read_int4_kernel<__half><<<grid, kReadThreads, 0, (cudaStream_t)p->stream>>>(a);
    return cudaGetLastError();
}
