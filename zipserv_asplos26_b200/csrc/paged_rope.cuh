// Rotary positions as the writes of a step's tokens share them (paged_rope.cu: into 16-bit
// pages; paged_int4_write.cu: into 4-bit ones).
#pragma once

#include <algorithm>

#include "paged.cuh"
#include "rows_meet.h"

namespace zs {

constexpr int kRopeThreads = 64;
constexpr int kRopeMaxAxes = 4;

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
    int N, Hq, Hkv, D, rot, interleaved, axes;
    int section_end[kRopeMaxAxes];
    int parts;                    // warps a token
    unsigned* err;
};

// The 16 channels of a head that a lane turns, eight from c0 and eight from c1 on, and
// the cosines and sines of their pairs.
struct RopeLane {
    bool turns;
    int c0, c1;
    float cs[8], sn[8];

    // Lane c of a head's, for token n; `on`: it has channels.
    __device__ __forceinline__ RopeLane(const RopeArgs& a, long long n, int c, bool on) {
        const int rot_lanes = a.rot / 16;
        turns = c < rot_lanes;
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
    }

    // Turns x (from c0 on) and y (from c1 on), 16-bit values, in fp32, rounded once.
    template <typename T>
    __device__ __forceinline__ void turn(uint4& x, uint4& y, int interleaved) const {
        uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
        if (interleaved) {
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
        x = make_uint4(xs[0], xs[1], xs[2], xs[3]);
        y = make_uint4(ys[0], ys[1], ys[2], ys[3]);
    }
};

// Host: the checked arguments of a call, but for its pools (of Hkv heads of D channels).
template <class P>
inline bool rope_args(const P* p, int Hkv, int D, RopeArgs* a) {
    const int N = p->N, Hq = p->Hq, rot = p->rot, axes = p->axes;
    if (N < 0 || Hq <= 0 || rot <= 0 || rot > D || rot % 16 || axes < 1 || axes > kRopeMaxAxes) return false;
    if (N == 0) return true;
    if (!p->q || !p->k || !p->v || !p->q_out || !p->positions || !p->cos_sin || !p->slots || p->table_rows <= 0)
        return false;
    int end = 0;
    for (int x = 0; x < axes; ++x) {
        if (p->sections[x] < 0 || p->sections[x] > rot) return false;
        end += p->sections[x];
        a->section_end[x] = end;
    }
    if (end != rot / 2) return false;
    if (!aligned16p(p->q) || !aligned16p(p->k) || !aligned16p(p->v) || !aligned16p(p->q_out) ||
        !aligned16p(p->cos_sin) || ((p->q_tok | p->q_head | p->k_tok | p->k_head | p->v_tok | p->v_head) % 8))
        return false;
    if (!q_out_is_apart(p->q_out, N, Hq, Hkv, D, p->q, p->q_tok, p->q_head, p->k, p->k_tok, p->k_head, p->v, p->v_tok,
                        p->v_head))
        return false;
    a->q = p->q; a->k = p->k; a->v = p->v; a->q_out = p->q_out;
    a->q_tok = p->q_tok; a->q_head = p->q_head; a->k_tok = p->k_tok; a->k_head = p->k_head;
    a->v_tok = p->v_tok; a->v_head = p->v_head;
    a->qo_tok = (long long)Hq * D; a->qo_head = D;
    a->positions = p->positions; a->pos_axis = p->pos_axis;
    a->table = p->cos_sin; a->table_stride = rot; a->table_rows = p->table_rows;
    a->slots = reinterpret_cast<const long long*>(p->slots);
    a->N = N; a->Hq = Hq; a->Hkv = Hkv; a->D = D; a->rot = rot; a->interleaved = p->interleaved ? 1 : 0; a->axes = axes;
    a->err = p->err;
    return true;
}

// Sets the warps a token and returns the grid: a warp a token fills the GPU from about
// 148 x 32 tokens on; with fewer, the token's heads are dealt to several warps.
inline unsigned rope_grid(RopeArgs* a) {
    const int heads_per = 32 / (a->D / 16);
    const int passes = (a->Hq + 2 * a->Hkv + heads_per - 1) / heads_per;
    a->parts = std::max(1, std::min(passes, (148 * 32 + a->N - 1) / a->N));
    const long long warps = (long long)a->N * a->parts;
    return (unsigned)((warps + kRopeThreads / 32 - 1) / (kRopeThreads / 32));
}

}  // namespace zs
