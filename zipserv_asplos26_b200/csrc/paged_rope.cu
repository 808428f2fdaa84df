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
#include <algorithm>

#include "paged.cuh"
#include "rows_meet.h"

namespace zs {
namespace {

constexpr int kRopeThreads = 64;
constexpr int kRopeMaxAxes = 4;
constexpr int kRopeBatch = 4;       // passes whose loads are in flight together

struct RopeArgs {
    const uint16_t* q;
    const uint16_t* k;
    const uint16_t* v;
    uint16_t* q_out;
    long long q_tok, q_head, k_tok, k_head, v_tok, v_head, qo_tok, qo_head;   // elements
    const int* positions;
    long long pos_axis;           // elements between axes
    const float* table;
    long long table_stride;
    int table_rows;
    const long long* slots;
    PoolView kp, vp;
    int N, Hq, Hkv, D, rot, interleaved, axes;
    int section_end[kRopeMaxAxes];
    int parts;                    // warps a token
    unsigned* err;
};

template <typename T>
__global__ void __launch_bounds__(kRopeThreads) rope_write_kernel(const RopeArgs a) {
    const int lane = threadIdx.x & 31;
    const long long warp = (long long)blockIdx.x * (kRopeThreads / 32) + (threadIdx.x >> 5);
    const long long n = warp / a.parts;
    if (n >= a.N) return;
    const int part = (int)(warp - n * a.parts);
    const int per_head = a.D / 16;            // lanes a head
    const int heads_per = 32 / per_head;      // heads a pass of the warp
    const int sub = lane / per_head, c = lane - sub * per_head;
    const bool on = sub < heads_per;
    const int rot_lanes = a.rot / 16;
    const bool turns = c < rot_lanes;
    // first and second 8 channels of this lane
    int c0, c1;
    if (!turns) {
        c0 = c * 16;
        c1 = c0 + 8;
    } else if (a.interleaved) {
        c0 = c * 16;
        c1 = c0 + 8;
    } else {
        c0 = c * 8;
        c1 = a.rot / 2 + c * 8;
    }
    float cs[8], sn[8];
    if (on && turns) {
        const int half = a.rot / 2;
        int pos[kRopeMaxAxes];
        bool bad = false;
#pragma unroll
        for (int x = 0; x < kRopeMaxAxes; ++x) {
            pos[x] = x < a.axes ? a.positions[x * a.pos_axis + n] : 0;
            if (pos[x] < 0 || pos[x] >= a.table_rows) {
                bad = true;
                pos[x] = 0;
            }
        }
        if (bad) set_err(a.err, kErrPagedIndex);
        auto row_of = [&](int j) {
            int p = pos[0];
#pragma unroll
            for (int x = 1; x < kRopeMaxAxes; ++x)
                if (x < a.axes && j >= a.section_end[x - 1]) p = pos[x];
            return a.table + (long long)p * a.table_stride;
        };
        const float* first = row_of(c * 8);
        bool same = true;       // no section ends among this lane's pairs (or the axes agree)
#pragma unroll
        for (int j = 1; j < 8; ++j) same &= row_of(c * 8 + j) == first;
        if (same) {
            const float4 x0 = __ldg(reinterpret_cast<const float4*>(first + c * 8));
            const float4 x1 = __ldg(reinterpret_cast<const float4*>(first + c * 8 + 4));
            const float4 y0 = __ldg(reinterpret_cast<const float4*>(first + half + c * 8));
            const float4 y1 = __ldg(reinterpret_cast<const float4*>(first + half + c * 8 + 4));
            cs[0] = x0.x; cs[1] = x0.y; cs[2] = x0.z; cs[3] = x0.w;
            cs[4] = x1.x; cs[5] = x1.y; cs[6] = x1.z; cs[7] = x1.w;
            sn[0] = y0.x; sn[1] = y0.y; sn[2] = y0.z; sn[3] = y0.w;
            sn[4] = y1.x; sn[5] = y1.y; sn[6] = y1.z; sn[7] = y1.w;
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                cs[j] = row_of(c * 8 + j)[c * 8 + j];
                sn[j] = row_of(c * 8 + j)[half + c * 8 + j];
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            cs[j] = 1.f;
            sn[j] = 0.f;
        }
    }
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
            if (turns && (i0 + u * a.parts) * heads_per + sub < a.Hq + a.Hkv) {
                uint32_t xs[4] = {x[u].x, x[u].y, x[u].z, x[u].w}, ys[4] = {y[u].x, y[u].y, y[u].z, y[u].w};
                if (a.interleaved) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float2 f = unpack2<T>(xs[j]), w = unpack2<T>(ys[j]);
                        xs[j] = pack2<T>(f.x * cs[j] - f.y * sn[j], f.y * cs[j] + f.x * sn[j]);
                        ys[j] = pack2<T>(w.x * cs[4 + j] - w.y * sn[4 + j], w.y * cs[4 + j] + w.x * sn[4 + j]);
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float2 f = unpack2<T>(xs[j]), w = unpack2<T>(ys[j]);
                        xs[j] = pack2<T>(f.x * cs[2 * j] - w.x * sn[2 * j], f.y * cs[2 * j + 1] - w.y * sn[2 * j + 1]);
                        ys[j] = pack2<T>(w.x * cs[2 * j] + f.x * sn[2 * j], w.y * cs[2 * j + 1] + f.y * sn[2 * j + 1]);
                    }
                }
                x[u] = make_uint4(xs[0], xs[1], xs[2], xs[3]);
                y[u] = make_uint4(ys[0], ys[1], ys[2], ys[3]);
            }
            __stcs(reinterpret_cast<uint4*>(dst[u] + c0), x[u]);
            __stcs(reinterpret_cast<uint4*>(dst[u] + c1), y[u]);
        }
    }
}

}  // namespace
}  // namespace zs

extern "C" int zs_rope_write(const ZsRopeWrite* p) {
    using namespace zs;
    RopeArgs a{};
    if (!p || p->N < 0 || p->Hq <= 0 || !make_pool(&p->k_pool, &a.kp) || !make_pool(&p->v_pool, &a.vp) ||
        !same_pools(p->k_pool, p->v_pool))
        return cudaErrorInvalidValue;
    const int N = p->N, Hq = p->Hq, D = a.kp.dim, Hkv = a.kp.heads, rot = p->rot, axes = p->axes;
    if (D % 16 || D > 512 || rot <= 0 || rot > D || rot % 16 || axes < 1 || axes > kRopeMaxAxes)
        return cudaErrorInvalidValue;
    if (N == 0) return cudaSuccess;
    if (!p->q || !p->k || !p->v || !p->q_out || !p->positions || !p->cos_sin || !p->slots || p->table_rows <= 0)
        return cudaErrorInvalidValue;
    int end = 0;
    for (int x = 0; x < axes; ++x) {
        if (p->sections[x] < 0 || p->sections[x] > rot) return cudaErrorInvalidValue;
        end += p->sections[x];
        a.section_end[x] = end;
    }
    if (end != rot / 2) return cudaErrorInvalidValue;
    if (!aligned16p(p->q) || !aligned16p(p->k) || !aligned16p(p->v) || !aligned16p(p->q_out) ||
        !aligned16p(p->cos_sin) || ((p->q_tok | p->q_head | p->k_tok | p->k_head | p->v_tok | p->v_head) % 8))
        return cudaErrorInvalidValue;
    if (!q_out_is_apart(p->q_out, N, Hq, Hkv, D, p->q, p->q_tok, p->q_head, p->k, p->k_tok, p->k_head, p->v, p->v_tok,
                        p->v_head))
        return cudaErrorInvalidValue;
    a.q = p->q; a.k = p->k; a.v = p->v; a.q_out = p->q_out;
    a.q_tok = p->q_tok; a.q_head = p->q_head; a.k_tok = p->k_tok; a.k_head = p->k_head;
    a.v_tok = p->v_tok; a.v_head = p->v_head;
    a.qo_tok = (long long)Hq * D; a.qo_head = D;
    a.positions = p->positions; a.pos_axis = p->pos_axis;
    a.table = p->cos_sin; a.table_stride = rot; a.table_rows = p->table_rows;
    a.slots = reinterpret_cast<const long long*>(p->slots);
    a.N = N; a.Hq = Hq; a.Hkv = Hkv; a.D = D; a.rot = rot; a.interleaved = p->interleaved ? 1 : 0; a.axes = axes;
    a.err = p->err;
    cudaStream_t stream = (cudaStream_t)p->stream;
    // A warp a token fills the GPU from about 148 x 32 tokens on; with fewer, the
    // token's heads are dealt to several warps.
    const int heads_per = 32 / (D / 16);
    const int passes = (Hq + 2 * Hkv + heads_per - 1) / heads_per;
    a.parts = std::max(1, std::min(passes, (148 * 32 + N - 1) / N));
    const long long warps = (long long)N * a.parts;
    const unsigned grid = (unsigned)((warps + kRopeThreads / 32 - 1) / (kRopeThreads / 32));
    if (p->k_pool.dtype == ZS_BF16)
        rope_write_kernel<__nv_bfloat16><<<grid, kRopeThreads, 0, stream>>>(a);
    else
        rope_write_kernel<__half><<<grid, kRopeThreads, 0, stream>>>(a);
    return cudaGetLastError();
}
