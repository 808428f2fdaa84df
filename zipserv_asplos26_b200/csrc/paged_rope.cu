// Rotary positions with one or several axes on q and k, and the step's k and v
// written to their slots of a paged KV cache (zs_rope_write).
//
// Channel pair j of the first `rot` channels turns by the angle of position
// pos[axis(j)] at frequency j, read from a table row [cos_0.. | sin_0..] in
// fp32: (a, b) -> (a cos - b sin, b cos + a sin), in fp32, rounded once. Pairs
// are (j, j + rot / 2), or (2j, 2j + 1) when interleaved; axis(j) is the section
// that j falls in. Channels past `rot` and all of v are copied.
//
// Bound by HBM: q, k, v are read once and written once. A lane owns 16 channels
// of a head (two 16-byte accesses, eight pairs), so its eight cosines and sines
// stay in registers while its warp walks the token's heads, four passes of loads
// ahead of their stores, both marked as read and written once. CTAs of two warps:
// an SM takes on a new token as soon as one is done (256 threads 68.7 us, 64
// threads 64.8 for 16411 tokens of 32 + 2 x 8 heads of 128, 412 MB, 6.36 TB/s; a
// plain copy does 6.56). 32 tokens take 2.7 us, the launch and two dependent reads.
#include "paged_rope.cuh"

namespace zs {
namespace {

constexpr int kRopeBatch = 4;       // passes whose loads are in flight together

struct RopeWriteArgs : RopeArgs {
    PoolView kp, vp;
};

template <typename T>
__global__ void __launch_bounds__(kRopeThreads) rope_write_kernel(const RopeWriteArgs a) {
    const int lane = threadIdx.x & 31;
    const long long warp = (long long)blockIdx.x * (kRopeThreads / 32) + (threadIdx.x >> 5);
    const long long n = warp / a.parts;
    if (n >= a.N) return;
    const int part = (int)(warp - n * a.parts);
    const int per_head = a.D / 16;            // lanes a head
    const int heads_per = 32 / per_head;      // heads a pass of the warp
    const int sub = lane / per_head, c = lane - sub * per_head;
    const bool on = sub < heads_per;
    const RopeLane me(a, n, c, on);
    const int c0 = me.c0, c1 = me.c1;
    const long long slot = a.slots[n];
    const long long cap = (long long)a.kp.num_blocks << a.kp.page_shift;
    const bool live = slot >= 0 && slot < cap;
    if ((slot < -1 || slot >= cap) && lane == 0) set_err(a.err, kErrPagedIndex);     // -1: padding
    const long long blk = slot >> a.kp.page_shift, row = slot & ((1 << a.kp.page_shift) - 1);
    if (!on) return;
    uint16_t* kdst = static_cast<uint16_t*>(a.kp.data) + blk * a.kp.s_block + row * a.kp.s_token;
    uint16_t* vdst = static_cast<uint16_t*>(a.vp.data) + blk * a.vp.s_block + row * a.vp.s_token;
    const int rows = a.Hq + 2 * a.Hkv;                       // heads of q, then k, then v
    const int passes = (rows + heads_per - 1) / heads_per;
    for (int i0 = part; i0 < passes; i0 += kRopeBatch * a.parts) {
        uint4 x[kRopeBatch], y[kRopeBatch];
        uint16_t* dst[kRopeBatch];
#pragma unroll
        for (int u = 0; u < kRopeBatch; ++u) {
            const int h = (i0 + u * a.parts) * heads_per + sub;
            const uint16_t* src = nullptr;
            dst[u] = nullptr;
            if (h < a.Hq) {
                src = a.q + n * a.q_tok + h * a.q_head;
                dst[u] = a.q_out + n * a.qo_tok + h * a.qo_head;
            } else if (h < rows && live) {
                const int kh = h - a.Hq, vh = kh - a.Hkv;
                if (vh < 0) {
                    src = a.k + n * a.k_tok + kh * a.k_head;
                    dst[u] = kdst + kh * a.kp.s_head;
                } else {
                    src = a.v + n * a.v_tok + vh * a.v_head;
                    dst[u] = vdst + vh * a.vp.s_head;
                }
            }
            if (src) {               // plain loads: q may be turned in place
                x[u] = __ldcs(reinterpret_cast<const uint4*>(src + c0));
                y[u] = __ldcs(reinterpret_cast<const uint4*>(src + c1));
            }
        }
#pragma unroll
        for (int u = 0; u < kRopeBatch; ++u) {
            if (!dst[u]) continue;
            if (me.turns && (i0 + u * a.parts) * heads_per + sub < a.Hq + a.Hkv) me.turn<T>(x[u], y[u], a.interleaved);
            __stcs(reinterpret_cast<uint4*>(dst[u] + c0), x[u]);
            __stcs(reinterpret_cast<uint4*>(dst[u] + c1), y[u]);
        }
    }
}

}  // namespace
}  // namespace zs

extern "C" int zs_rope_write(const ZsRopeWrite* p) {
    using namespace zs;
    RopeWriteArgs a{};
    if (!p || !make_pool(&p->k_pool, &a.kp) || !make_pool(&p->v_pool, &a.vp) || !same_pools(p->k_pool, p->v_pool) ||
        a.kp.dim % 16 || a.kp.dim > 512 || !rope_args(p, a.kp.heads, a.kp.dim, &a))
        return cudaErrorInvalidValue;
    if (a.N == 0) return cudaSuccess;
    cudaStream_t stream = (cudaStream_t)p->stream;
    const unsigned grid = rope_grid(&a);
    if (p->k_pool.dtype == ZS_BF16)
        rope_write_kernel<__nv_bfloat16><<<grid, kRopeThreads, 0, stream>>>(a);
    else
        rope_write_kernel<__half><<<grid, kRopeThreads, 0, stream>>>(a);
    return cudaGetLastError();
}
