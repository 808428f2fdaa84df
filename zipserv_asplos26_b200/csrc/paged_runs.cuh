// How paged attention is dealt to the GPU and joined, whatever the cache holds
// (paged_attention.cu: 16-bit keys and values; paged_int4_attention.cuh: 4-bit ones).
//
// The work is cut into chunks, a warp's step: one to four parts of 16 tokens of a unit
// (sequence, KV head, tile of up to 16 query heads). They are dealt in one of two ways,
// chosen by sizes that the host has (unit_warps):
//   * paged_attn_kernel: all chunks in order go to the warps of the GPU in equal
//     runs, found by a prefix sum over the lengths in the kernel, so ragged
//     batches and single long sequences load every SM alike and no length is
//     needed on the host. A run that ends inside a unit leaves its (m, l, O) in a
//     workspace, and paged_join_kernel joins a unit's pieces in order. Where rows of
//     neighbouring heads share lines, a run goes to a CTA whose warps take the same
//     tokens of a head each (PaArgs::group).
//   * paged_attn_units_kernel: a fixed number of warps a unit, joined through
//     distributed shared memory in the same kernel: short units and page lists.
// Sums are always in the same order for the same sizes on the host and the same
// lengths: a result does not change from run to run. The times at the choices below are
// those of 16-bit keys and values.
//
// A form F says what a warp does: T (of q and the output), D, kListed (page lists),
// kParts (of a chunk), kGrouped (whether PaArgs::group is looked at), Args (PaArgs or more), kCtas, kStages, kRing, kSmem, Ring (start,
// ask, step), State (what a warp holds of a unit: finish, write, park), start (of a
// State), kBias (of its exponentials), kOdd (whether infinite values are looked at again,
// by odd_values and State's odd and mend) and Joined (a form of the same T, D, kListed,
// kParts and odd_values: the one that the join is built for).
#pragma once

#include <algorithm>
#include <atomic>
#include <climits>
#include <cmath>
#include <type_traits>

#include "paged.cuh"

namespace zs {

struct PaArgs {
    const uint16_t* q;        // [B][Hq][D]
    PoolView kp, vp;
    const int* table;
    long long table_stride;
    const int* lens;
    const int* pages;         // nullable: [B][Hkv][top]
    const int* counts;        // with pages: [B][Hkv]
    int B, Hq, Hkv, G, tiles, width, top;
    int max_len;              // host's bound on the lengths, 0: none (chooses the way, and so the order of sums)
    float scale2;             // softmax scale * log2(e)
    uint16_t* out;            // [B][Hq][D]
    float* lse;               // nullable: [B][Hq]
    long long* plan;          // workspace: [0] chunks a warp, [1 + unit] first chunk of the unit
    int prow;                 // rows of a piece: min(G, 16)
    float* part_ml;           // [2 W][prow][2], W warps
    float* part_o;            // [2 W][prow][D]
    unsigned* err;
    int group;                // units that a run's warps take side by side: 1, or a CTA's warps one each
};

namespace {

constexpr int kPaWarps = 4;
constexpr int kPaThreads = kPaWarps * 32;
constexpr int kPaChunk = 16;       // tokens of a chunk's part; pages are multiples of it
constexpr int kPaRows = 16;        // query heads a unit
constexpr float kLog2e = 1.4426950408889634f;

// The keys and values pass through L2 once: marked to leave it first, they do not
// push out what the kernels around share through it (tables, q, pieces, the next
// layer's weights).
__device__ __forceinline__ uint64_t evict_first_policy() {
    uint64_t p;
    asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(p));
    return p;
}
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool on, uint64_t policy) {
    asm volatile("cp.async.cg.shared.global.L2::cache_hint.L2::256B [%0], [%1], 16, %2, %3;" ::"r"(dst), "l"(src),
                 "r"(on ? 16 : 0), "l"(policy)
                 : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(a)
                 : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(a)
                 : "memory");
}
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1,
                                         __nv_bfloat16) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, "
        "%2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __half) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, "
        "%2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Transposes an 8 x 8 matrix of 16-bit values held a row a quad of lanes.
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

__device__ __forceinline__ float2 ld_dsmem_f2(uint32_t addr) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
    return v;
}

// log sum exp of a row from its base-2 maximum and sum of exponentials, which are 2^bias too large.
__device__ __forceinline__ float log_sum(float m, float l, float bias) {
    return l == 0.f ? -INFINITY : (m + log2f(l) - bias) / kLog2e;
}

// Parts of 16 tokens, and chunks, of entry e: a sequence (whole cache) or a (sequence, KV
// head) with a page list.
template <bool kListed>
__device__ __forceinline__ int entry_parts(const PaArgs& a, int e) {
    if (kListed) return max(0, min(a.counts[e], a.top)) << (a.kp.page_shift - 4);
    const int cap = (int)min((long long)a.width << a.kp.page_shift, (long long)INT_MAX - 15);
    return (max(0, min(a.lens[e], cap)) + kPaChunk - 1) / kPaChunk;
}
template <class F>
__device__ __forceinline__ int entry_chunks(const PaArgs& a, int e) {
    return (entry_parts<F::kListed>(a, e) + F::kParts - 1) / F::kParts;
}

// Inclusive prefix over the warp's lanes.
__device__ __forceinline__ long long warp_prefix(long long v) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long u = __shfl_up_sync(~0u, v, o);
        if ((int)(threadIdx.x & 31) >= o) v += u;
    }
    return v;
}

// The block and the number of valid tokens of part `ch` of an entry (lim 0: none).
template <bool kListed>
__device__ __forceinline__ void look_chunk(const PaArgs& a, int e, int b, int ch, int len, int& id, int& lim) {
    const int cps = a.kp.page_shift - 4;                               // log2 chunks a page
    int p = ch >> cps;
    if (kListed) p = a.pages[(long long)e * a.top + p];
    id = lim = 0;
    if (p < 0 || p >= a.width) {
        set_err(a.err, kErrPagedIndex);
        return;
    }
    const int t0 = ((p << cps) + (ch & ((1 << cps) - 1))) * kPaChunk;
    if (t0 >= len) return;
    const int blk = a.table[b * a.table_stride + p];
    if (blk < 0 || blk >= a.kp.num_blocks) {
        set_err(a.err, kErrPagedIndex);
        return;
    }
    id = blk;
    lim = min(kPaChunk, len - t0);
}

// Outputs that are not finite (see a form's odd_values, which adds to `seen` three bits
// for each of its channels: an infinity is there, a negative one, a NaN).
// Whether nothing more can change the outputs of the channels whose bits 3 j are in `odd`.
__device__ __forceinline__ bool odd_decided(uint32_t seen, uint32_t odd) {
    return ((seen >> 2 | (seen & seen >> 1)) & odd) == odd;
}
// Bits 3 j of the channels j that are not finite.
template <int kCount>
__device__ __forceinline__ uint32_t odd_channels(const float (&o)[kCount]) {
    uint32_t f = 0;
#pragma unroll
    for (int j = 0; j < kCount; ++j) f |= (isfinite(o[j]) ? 0u : 1u) << (3 * j);
    return f;
}
// The output of the j-th of these channels; o where nothing odd is among its values.
__device__ __forceinline__ float odd_output(uint32_t seen, int j, float o) {
    const uint32_t f = seen >> (3 * j) & 7u;
    return f == 1 ? INFINITY : f == 2 ? -INFINITY : f ? NAN : o;
}
// Whether an output is not finite although the sum of its weights, l, is a number.
__device__ __forceinline__ bool is_odd(float sum_of_zeros, float l) { return isnan(sum_of_zeros) && !isnan(l); }

// Where a warp is in the sequence of all chunks: chunk `ch` of the n chunks of
// unit `in_e` of entry e.
struct PaCursor {
    int e, n, in_e, ch;
};

// To the next unit that has chunks (there is one: the caller has chunks left).
template <class F>
__device__ __forceinline__ void next_unit(const PaArgs& a, int per_entry, PaCursor& c) {
    c.ch = 0;
    if (++c.in_e < per_entry) return;
    c.in_e = 0;
    do c.n = entry_chunks<F>(a, ++c.e);
    while (c.n == 0);
}

template <class F>
__global__ void __launch_bounds__(kPaThreads, F::kCtas) paged_attn_kernel(const typename F::Args a) {
    using T = typename F::T;
    constexpr int D = F::D;
    constexpr bool kListed = F::kListed;
    extern __shared__ __align__(1024) uint8_t pa_smem[];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    grid_dep_launch();
    grid_dep_wait();

    // ---- each warp's run of chunks
    const int entries = kListed ? a.B * a.Hkv : a.B;
    const int group = F::kGrouped ? a.group : 1;
    const int per_entry = (kListed ? a.tiles : a.Hkv * a.tiles) / group;     // groups of units an entry
    // Each warp by itself: lane i sums the chunks of entries [i per, (i + 1) per),
    // a prefix over the lanes gives the total and the lane whose entries hold the
    // warp's first chunk, a second one over those entries the entry.
    const int per = (entries + 31) / 32;
    long long mine = 0;
    int n1 = 0;                    // the lane's last entry's (its only one up to 32 entries)
#pragma unroll 4
    for (int i = 0; i < per; ++i) {
        const int e = lane * per + i;
        n1 = e < entries ? entry_chunks<F>(a, e) : 0;
        mine += n1;
    }
    const long long inc = warp_prefix(mine);
    const long long total = __shfl_sync(~0u, inc, 31) * per_entry;
    const int warps = gridDim.x * (kPaWarps / group);              // that take runs of their own
    // two chunks or more: pieces of one would double what is joined (48 pages for 8
    // pairs 17.5 us, 16.3 so)
    const long long run = max(div_nonneg(total + warps - 1, warps), 2ll);
    if (blockIdx.x == 0 && tid == 0) a.plan[0] = run;
    // neighbouring runs go to different CTAs, so that few chunks spread over the SMs
    const int mine_of = group > 1 ? warp : 0;                      // the warp's unit of a group
    const int id = (group > 1 ? 0 : warp) * (int)gridDim.x + (int)blockIdx.x;
    const long long c_begin = run * id;
    if (c_begin >= total) return;
    const int steps = (int)min(run, total - c_begin);
    const int owner = __ffs(__ballot_sync(~0u, inc * per_entry > c_begin)) - 1;
    long long lo = __shfl_sync(~0u, inc - mine, owner);            // entry chunks before, per unit
    int entry = owner * per, n = __shfl_sync(~0u, n1, owner);
    if (per > 1) {
        for (;; entry += 32) {
            const int e = entry + lane;
            const int ne = e < min(entries, (owner + 1) * per) ? entry_chunks<F>(a, e) : 0;
            const long long ie = warp_prefix((long long)ne);
            const unsigned past = __ballot_sync(~0u, (lo + ie) * per_entry > c_begin);
            if (past) {
                const int l = __ffs(past) - 1;
                entry += l;
                n = __shfl_sync(~0u, ne, l);
                lo += __shfl_sync(~0u, ie - ne, l);
                break;
            }
            lo += __shfl_sync(~0u, ie, 31);
        }
    }
    const long long into = c_begin - lo * per_entry;               // chunks into the entry

    PaCursor at;                   // of the copies
    at.e = entry;
    at.n = n;
    at.in_e = (int)div_nonneg(into, n);
    at.ch = (int)(into - (long long)at.in_e * n);
    PaCursor cur = at;             // of the products
    long long u_lo = c_begin - at.ch;

    // ---- copies: batches of chunks of one unit, up to 32 parts, a lane holding the
    // block and the number of valid tokens of one part; the next batch is looked up
    // while the present one is copied
    constexpr int kParts = F::kParts;
    const int table_len = (int)min((long long)a.width << a.kp.page_shift, (long long)INT_MAX);
    struct Batch {
        int ids, lims, count, h, ch;
    } now, next;
    int looked = 0;                // chunks looked up
    auto look = [&](Batch& t) {
        t.count = min(32 / kParts, min(at.n - at.ch, steps - looked));
        t.ids = 0;
        t.lims = 0;
        t.ch = at.ch;
        t.h = kListed ? at.e % a.Hkv : (at.in_e * group + mine_of) / a.tiles;
        if (t.count <= 0) return;
        if (lane < t.count * kParts && (kParts == 1 || at.ch * kParts + lane < entry_parts<kListed>(a, at.e))) {
            const int b = kListed ? at.e / a.Hkv : at.e;
            look_chunk<kListed>(a, at.e, b, at.ch * kParts + lane, min(a.lens[b], table_len), t.ids, t.lims);
        }
        looked += t.count;
        at.ch += t.count;
        if (at.ch == at.n && looked < steps) next_unit<F>(a, per_entry, at);
    };
    look(now);
    int in_batch = 0;
    // part `part` of the next chunk (parts in order, from 0)
    auto find = [&](int& blk, int& ch, int& h, int, int part) {
        if (part == 0 && in_batch == now.count * kParts) {
            now = next;
            in_batch = 0;
            look(next);
        }
        blk = __shfl_sync(~0u, now.ids, in_batch);
        ch = now.ch * kParts + in_batch;
        h = now.h;
        return __shfl_sync(~0u, now.lims, in_batch++);
    };
    typename F::Ring ring;
    ring.start(a, smem_u32(pa_smem) + warp * F::kRing, steps);
#pragma unroll
    for (int s = 0; s < F::kStages - 1; ++s) {
        ring.ask(a, s, find);
        if (s == 0) look(next);    // the first chunk is on its way while the next batch is looked up
    }

    int s = 0;
    while (true) {
        // ---- a unit, or the part of it in this run
        const int first = cur.ch, count = min(cur.n - first, steps - s);
        const int b = kListed ? cur.e / a.Hkv : cur.e;
        const int of = cur.in_e * group + mine_of;
        const int h = kListed ? cur.e % a.Hkv : of / a.tiles;
        const int tile = kListed ? cur.in_e : of % a.tiles;
        const int g0 = tile * kPaRows, rows = min(kPaRows, a.G - g0);
        if (first == 0 && lane == 0) a.plan[1 + (b * a.Hkv + h) * a.tiles + tile] = u_lo;
        const long long head0 = (long long)b * a.Hq + (long long)h * a.G + g0;
        typename F::State st;
        F::start(st, a, a.q + head0 * D, rows);
        for (const int end = s + count; s < end; ++s) ring.step(a, s, st, find);
        // ---- out, or to the workspace where the run cuts the unit
        const bool whole = first == 0 && count == cur.n;
        const long long slot = (2ll * id + (s == count ? 0 : 1)) * group + mine_of;    // the run's first part, or its last
        st.finish();
        if (whole) {
            if constexpr (F::kOdd) {
                if (__builtin_expect(st.odd(), false)) {
                    uint32_t seen = 0;
                    F::template odd_values<D / 32>(a, cur.e, b, h, 0, cur.n, lane * (D / 32), seen);
                    st.mend(seen);
                }
            }
            st.write(a.out + head0 * D, a.lse ? a.lse + head0 : nullptr, rows);
        } else st.park(a.part_o + slot * a.prow * D, a.part_ml + slot * a.prow * 2, rows);
        if (s == steps) break;
        u_lo += cur.n;
        next_unit<F>(a, per_entry, cur);
    }
    cp_wait<0>();
}

// ---- Each unit by a fixed number W of warps, 1 to 16: no prefix over the
// lengths, no workspace and no second kernel. Warp w of the unit's W takes chunks
// [n w / W, n (w + 1) / W) of the unit's n, leaves (m, l, O) in its own shared
// memory, and after a cluster barrier the unit's threads join the W pieces
// through distributed shared memory, in order. With W below 4 a CTA has several
// units, from 4 on a cluster of W / 4 CTAs has one.
template <class F>
__global__ void __launch_bounds__(kPaThreads, F::kCtas) paged_attn_units_kernel(const typename F::Args a, int W) {
    using T = typename F::T;
    constexpr int D = F::D;
    constexpr bool kListed = F::kListed;
    extern __shared__ __align__(1024) uint8_t pa_smem[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long long warp_id = (long long)blockIdx.x * kPaWarps + warp;
    const int unit = (int)(warp_id / W), w = (int)(warp_id % W);
    const int units = a.B * a.Hkv * a.tiles;
    const bool on = unit < units;          // the last CTA may have fewer
    const int e = on ? (kListed ? unit / a.tiles : unit / (a.Hkv * a.tiles)) : 0;
    const int b = kListed ? e / a.Hkv : e, h = kListed ? e % a.Hkv : unit / a.tiles % a.Hkv;
    const int g0 = unit % a.tiles * kPaRows, rows = on ? min(kPaRows, a.G - g0) : 0;
    const long long head0 = (long long)b * a.Hq + (long long)h * a.G + g0;
    grid_dep_launch();
    grid_dep_wait();
    const int table_len = (int)min((long long)a.width << a.kp.page_shift, (long long)INT_MAX);
    const int len = min(a.lens[b], table_len), n = on ? entry_chunks<F>(a, e) : 0;
    const int first = (int)((long long)n * w / W), steps = (int)((long long)n * (w + 1) / W) - first;
    typename F::State st;
    int ids = 0, lims = 0;         // of 32 parts, a lane each
    constexpr int kParts = F::kParts;
    const int parts = kParts > 1 && on ? entry_parts<kListed>(a, e) : 0;
    auto find = [&](int& blk, int& ch, int& head, int s, int part) {
        const int x = s * kParts + part;                       // part of the warp's share
        if ((x & 31) == 0) {
            ids = lims = 0;
            const int y = first * kParts + x + lane;
            if (x + lane < steps * kParts && (kParts == 1 || y < parts)) look_chunk<kListed>(a, e, b, y, len, ids, lims);
        }
        blk = __shfl_sync(~0u, ids, x & 31);
        ch = first * kParts + x;
        head = h;
        return __shfl_sync(~0u, lims, x & 31);
    };
    typename F::Ring ring;
    ring.start(a, smem_u32(pa_smem) + warp * F::kRing, steps);
#pragma unroll
    for (int s = 0; s < F::kStages - 1; ++s) ring.ask(a, s, find);
    F::start(st, a, a.q + head0 * D, rows);
    for (int s = 0; s < steps; ++s) ring.step(a, s, st, find);
    cp_wait<0>();
    __syncwarp();
    st.finish();
    // the warp's piece, over its ring: [16][D] outputs, [16][2] maxima and sums
    static_assert(F::kRing >= kPaRows * (D + 2) * 4, "a warp's piece fits its ring");
    float* po = reinterpret_cast<float*>(pa_smem + warp * F::kRing);
    st.park(po, po + kPaRows * D, rows);
    // One warp a unit needs no barrier, several of a CTA the CTA's, more the cluster's
    // (its second one keeps a CTA's shared memory until its peers have read it).
    if (W == 1) __syncwarp();
    else if (W <= kPaWarps) __syncthreads();
    else cluster_sync();
    // four channels a thread
    const uint32_t base = smem_u32(pa_smem);
    const int v0 = W < kPaWarps ? warp / W * W : 0;               // the unit's first warp in its (first) CTA
    const int in_cta = min(W, kPaWarps);
    for (int x = w * 32 + lane; x < rows * (D / 4); x += W * 32) {
        const int row = x / (D / 4), d4 = x % (D / 4) * 4;
        float m = -INFINITY, l = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int r = 0; r < W; r += kPaWarps) {
            const uint32_t peer = W <= kPaWarps ? base : mapa_shared(base, r / kPaWarps);
            float2 ml[kPaWarps];
            float4 o[kPaWarps];
#pragma unroll
            for (int v = 0; v < kPaWarps; ++v) {
                ml[v] = make_float2(-INFINITY, 0.f);
                o[v] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (v < in_cta) {
                    const uint32_t piece = peer + (v0 + v) * F::kRing;
                    ml[v] = ld_dsmem_f2(piece + (kPaRows * D + row * 2) * 4);
                    o[v] = ld_dsmem_f4(piece + (row * D + d4) * 4);
                }
            }
            float mn = m;
#pragma unroll
            for (int v = 0; v < kPaWarps; ++v) mn = fmaxf(mn, ml[v].x);
            const float ref = mn == -INFINITY ? 0.f : mn, f0 = exp2f(m - ref);
            l *= f0;
            acc.x *= f0;
            acc.y *= f0;
            acc.z *= f0;
            acc.w *= f0;
#pragma unroll
            for (int v = 0; v < kPaWarps; ++v) {
                const float f = exp2f(ml[v].x - ref);
                l += ml[v].y * f;
                acc.x += o[v].x * f;
                acc.y += o[v].y * f;
                acc.z += o[v].z * f;
                acc.w += o[v].w * f;
            }
            m = mn;
        }
        if constexpr (F::kOdd) {
            if (__builtin_expect(is_odd((acc.x * 0.f + acc.y * 0.f) + (acc.z * 0.f + acc.w * 0.f), l), false)) {
                const uint32_t odd = odd_channels<4>({acc.x, acc.y, acc.z, acc.w});
                uint32_t seen = 0;
                for (int v = 0; v < W && !odd_decided(seen, odd); ++v) {
                    const uint32_t peer = W <= kPaWarps ? base : mapa_shared(base, v / kPaWarps);
                    const float4 o = ld_dsmem_f4(peer + (v0 + v % kPaWarps) * F::kRing + (row * D + d4) * 4);
                    const int c = (int)((long long)n * v / W), end = (int)((long long)n * (v + 1) / W);
                    if (odd_channels<4>({o.x, o.y, o.z, o.w}))
                        F::template odd_values<4>(a, e, b, h, c, end - c, d4, seen);
                }
                acc.x = odd_output(seen, 0, acc.x);
                acc.y = odd_output(seen, 1, acc.y);
                acc.z = odd_output(seen, 2, acc.z);
                acc.w = odd_output(seen, 3, acc.w);
            }
        }
        const float inv = l == 0.f ? 0.f : 1.f / l;
        *reinterpret_cast<uint2*>(a.out + (head0 + row) * D + d4) =
            make_uint2(pack2<T>(acc.x * inv, acc.y * inv), pack2<T>(acc.z * inv, acc.w * inv));
        if (a.lse && d4 == 0) a.lse[head0 + row] = log_sum(m, l, F::kBias);
    }
    if (W > kPaWarps) cluster_sync();
}

// Joins the pieces of the units that the runs cut and writes zeros where nothing
// is attended. Its time is a few dependent reads of what other SMs wrote, so the
// pieces are read in batches, weights and outputs together. A warp takes a query
// head, D / 32 channels a lane; with few heads (long sequences: up to a piece a
// warp of the attention kernel) the warps of a CTA share a head's pieces and add
// their sums in order. It costs some 6 us of 87 at B=1 T=131105, where a unit is cut
// into 222 pieces (runs of 37 of its 8195 chunks).
constexpr int kJoinWarps = 16;
constexpr int kJoinShare = 148;        // heads joined by a CTA each
constexpr int kJoinBatch = 8;

template <class F>
__global__ void __launch_bounds__(kJoinWarps * 32) paged_join_kernel(const typename F::Args a, int share) {
    using T = typename F::T;
    constexpr int D = F::D, kVec = D / 32;
    constexpr bool kListed = F::kListed;
    __shared__ float s_acc[kJoinWarps][D], s_m[kJoinWarps], s_l[kJoinWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const int head = share ? (int)blockIdx.x : (int)blockIdx.x * warps + warp;
    if (head >= a.B * a.Hq) return;
    const int b = head / a.Hq, i = head % a.Hq, h = i / a.G, g = i % a.G;
    const int tile = g / kPaRows, row = g % kPaRows;
    grid_dep_wait();
    const long long run = a.plan[0], lo = a.plan[1 + (b * a.Hkv + h) * a.tiles + tile];
    const int n = entry_chunks<F>(a, kListed ? b * a.Hkv + h : b);
    const int group = F::kGrouped ? a.group : 1, of = group > 1 ? (h * a.tiles + tile) % group : 0;
    float m = -INFINITY, l = 0.f, acc[kVec];
#pragma unroll
    for (int j = 0; j < kVec; ++j) acc[j] = 0.f;
    if (n > 0) {
        const int w0 = (int)div_nonneg(lo, run), w1 = (int)div_nonneg(lo + n - 1, run);
        if (w0 == w1) return;                   // written whole
        // the first piece is the last of its warp's run unless it starts that run
        const bool second = lo != w0 * run;
        const int by = share ? warps : 1;
        for (int v = w0 + (share ? warp : 0); v <= w1; v += kJoinBatch * by) {
            float2 ml[kJoinBatch];
            float o[kJoinBatch][kVec];
#pragma unroll
            for (int x = 0; x < kJoinBatch; ++x) {
                const int w = v + x * by;
                const long long s = ((2ll * w + (w == w0 && second ? 1 : 0)) * group + of) * a.prow + row;
                ml[x] = make_float2(-INFINITY, 0.f);
#pragma unroll
                for (int j = 0; j < kVec; ++j) o[x][j] = 0.f;
                if (w <= w1) {
                    ml[x] = *reinterpret_cast<const float2*>(a.part_ml + s * 2);
                    const float* src = a.part_o + s * D + lane * kVec;
                    if constexpr (kVec == 4) *reinterpret_cast<float4*>(o[x]) = *reinterpret_cast<const float4*>(src);
                    else *reinterpret_cast<float2*>(o[x]) = *reinterpret_cast<const float2*>(src);
                }
            }
            float mn = m;
#pragma unroll
            for (int x = 0; x < kJoinBatch; ++x) mn = fmaxf(mn, ml[x].x);
            const float ref = mn == -INFINITY ? 0.f : mn, f0 = exp2f(m - ref);
            l *= f0;
#pragma unroll
            for (int j = 0; j < kVec; ++j) acc[j] *= f0;
#pragma unroll
            for (int x = 0; x < kJoinBatch; ++x) {
                const float f = exp2f(ml[x].x - ref);
                l += ml[x].y * f;
#pragma unroll
                for (int j = 0; j < kVec; ++j) acc[j] += o[x][j] * f;
            }
            m = mn;
        }
    }
    if (share) {
#pragma unroll
        for (int j = 0; j < kVec; ++j) s_acc[warp][lane * kVec + j] = acc[j];
        if (lane == 0) {
            s_m[warp] = m;
            s_l[warp] = l;
        }
        __syncthreads();
        if (warp) return;
        const float mw = lane < warps ? s_m[lane] : -INFINITY;
        m = mw;
#pragma unroll
        for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
        const float fw = lane < warps ? exp2f(mw - (m == -INFINITY ? 0.f : m)) : 0.f;
        l = 0.f;
#pragma unroll
        for (int j = 0; j < kVec; ++j) acc[j] = 0.f;
        for (int w = 0; w < warps; ++w) {
            const float f = __shfl_sync(~0u, fw, w);
            l += s_l[w] * f;
#pragma unroll
            for (int j = 0; j < kVec; ++j) acc[j] += s_acc[w][lane * kVec + j] * f;
        }
    }
    if constexpr (F::kOdd) {
        float zeros = 0.f;
    #pragma unroll
        for (int j = 0; j < kVec; ++j) zeros += acc[j] * 0.f;
        if (__builtin_expect(is_odd(zeros, l), false)) {
            const uint32_t odd = odd_channels<kVec>(acc);
            const int w0 = (int)div_nonneg(lo, run), w1 = (int)div_nonneg(lo + n - 1, run);
            uint32_t seen = 0;
            for (int w = w0; w <= w1 && !odd_decided(seen, odd); ++w) {
                const long long s = (2ll * w + (w == w0 && lo != w0 * run ? 1 : 0)) * a.prow + row;
                float o[kVec];
    #pragma unroll
                for (int j = 0; j < kVec; ++j) o[j] = a.part_o[s * D + lane * kVec + j];
                const long long c = max(w * run, lo), end = min((w + 1) * run, lo + n);
                if (odd_channels<kVec>(o))
                    F::template odd_values<kVec>(a, kListed ? b * a.Hkv + h : b, b, h, (int)(c - lo), (int)(end - c),
                                                 lane * kVec, seen);
            }
    #pragma unroll
            for (int j = 0; j < kVec; ++j) acc[j] = odd_output(seen, j, acc[j]);
        }
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    uint32_t* out = reinterpret_cast<uint32_t*>(a.out + (long long)head * D + lane * kVec);
#pragma unroll
    for (int j = 0; j < kVec; j += 2) out[j / 2] = pack2<T>(acc[j] * inv, acc[j + 1] * inv);
    if (a.lse && lane == 0) a.lse[head] = log_sum(m, l, F::kBias);
}

inline size_t plan_bytes(long long units) { return ((size_t)(1 + units) * 8 + 255) / 256 * 256; }
inline size_t piece_ml_bytes(int max_ctas, int prow) { return (size_t)2 * max_ctas * kPaWarps * prow * 2 * 4; }
// Of a call whose run kernel has at most max_ctas CTAs.
inline size_t run_workspace_bytes(long long units, int max_ctas, int prow, int D) {
    return plan_bytes(units) + piece_ml_bytes(max_ctas, prow) + (size_t)2 * max_ctas * kPaWarps * prow * D * 4;
}
// Its parts.
inline void lay_workspace(PaArgs* a, void* ws, int max_ctas) {
    uint8_t* at = static_cast<uint8_t*>(ws);
    a->plan = reinterpret_cast<long long*>(at);
    at += plan_bytes((long long)a->B * a->Hkv * a->tiles);
    a->part_ml = reinterpret_cast<float*>(at);
    a->part_o = reinterpret_cast<float*>(at + piece_ml_bytes(max_ctas, a->prow));
}

// The attention kernel's grid: the CTAs that the GPU holds at once (looked up once per device).
template <class F>
cudaError_t resident_ctas(int* ctas) {
    static std::atomic<int> cached[64];
    const auto kernel = paged_attn_kernel<F>;
    int dev = 0, per = 0, sms = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    if ((*ctas = cached[dev].load(std::memory_order_acquire)) > 0) return cudaSuccess;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, F::kSmem);
    if (e != cudaSuccess) return e;
    e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per, kernel, kPaThreads, F::kSmem);
    if (e != cudaSuccess) return e;
    e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return e;
    if (per < 1) return cudaErrorInvalidConfiguration;
    *ctas = std::min(per * sms, 148 * F::kCtas);
    cached[dev].store(*ctas, std::memory_order_release);
    return cudaSuccess;
}

// Warps a unit for paged_attn_units_kernel, or 0 where runs of chunks are the
// better way. Fixed shares have no second kernel (us in runs and so: B=1 T=97 7.5
// and 4.9, 16 sequences of 300 11.1 and 8.7, 512 of 100..200 59.3 and 54.0), but
// the longest unit's share is the time where one wave of warps holds all units (64
// of 0..1000: 26.4 and 34.6 at 36 chunks a warp; 16 of 2048: 27.1 and 28.5 at 17).
// So they serve units that are bounded to 16 chunks a warp, to 64 for page lists,
// whose units are alike (8 x 64 pages: 43.5 and 39.3), or to 5 where they leave SMs
// idle (B=1 T=4096: 9.6 and 15.6). These are the limits for 16-bit keys and values,
// whose chunks are 16 tokens; other forms bring their own (UnitLimits). W fills the GPU once, with two chunks a warp or
// more; units of unlike lengths in more waves want shares of some 12 chunks (128
// of 0..600: 41.1 us with one warp each, 28.7 with four, 31.4 in runs). Clusters of
// more than 4 CTAs were slower in all of these.
constexpr int kPaMaxUnitWarps = 16;

// A bound on a unit's parts: of the page list, the table or the caller's.
inline long long unit_parts(const PaArgs& a, bool listed) {
    const long long pages = ((long long)(listed ? a.top : a.width)) << (a.kp.page_shift - 4);
    return a.max_len > 0 && !listed ? std::min(pages, ((long long)a.max_len + kPaChunk - 1) / kPaChunk) : pages;
}

struct UnitLimits {
    int whole = 16, listed = 64;       // chunks a warp, at most
};

inline int unit_warps(const PaArgs& a, bool listed, int max_ctas, int parts, UnitLimits limits = {}) {
    const long long units = (long long)a.B * a.Hkv * a.tiles, chunks = (unit_parts(a, listed) + parts - 1) / parts;
    const long long resident = (long long)max_ctas * kPaWarps;
    int W = 1;
    while (W < kPaMaxUnitWarps && units * W * 2 <= resident && W * 4 <= chunks) W *= 2;
    while (!listed && W < kPaWarps && W * 12 < chunks) W *= 2;
    const long long steps = (chunks + W - 1) / W;
    const long long most = units * W < 148 * 4 ? 5 : listed ? limits.listed : limits.whole;
    return steps <= most && units * W <= INT32_MAX ? W : 0;
}

template <class F>
cudaError_t launch_units(const typename F::Args& a, int W, cudaStream_t s) {
    const auto kernel = paged_attn_units_kernel<F>;
    static std::atomic<unsigned long long> ready{0};      // a bit a device
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    if (!(ready.load(std::memory_order_acquire) >> dev & 1)) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, F::kSmem);
        if (e != cudaSuccess) return e;
        ready.fetch_or(1ull << dev, std::memory_order_release);
    }
    const long long warps = (long long)a.B * a.Hkv * a.tiles * W;
    cudaLaunchConfig_t cfg;
    cudaLaunchAttribute attr[2];
    pdl_config(&cfg, attr, dim3((unsigned)((warps + kPaWarps - 1) / kPaWarps)), dim3(kPaThreads), F::kSmem, s);
    if (W > kPaWarps) {
        attr[1].id = cudaLaunchAttributeClusterDimension;
        attr[1].val.clusterDim.x = W / kPaWarps;
        attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
        cfg.numAttrs = 2;
    }
    return cudaLaunchKernelEx(&cfg, kernel, a, W);
}

// a's attention by form F in runs, or by U in units where W, unit_warps' answer, is not 0.
template <class F, class U>
cudaError_t launch_paged(const typename F::Args& a, int W, cudaStream_t s) {
    if (W) return launch_units<U>(a, W, s);
    int ctas = 0;
    cudaError_t e = resident_ctas<F>(&ctas);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg;
    cudaLaunchAttribute attr;
    pdl_config(&cfg, &attr, dim3(ctas), dim3(kPaThreads), F::kSmem, s);
    e = cudaLaunchKernelEx(&cfg, paged_attn_kernel<F>, a);
    if (e != cudaSuccess) return e;
    // a head a CTA while there are SMs for it, else a head a warp in small CTAs
    const int heads = a.B * a.Hq, share = heads <= kJoinShare ? 1 : 0;
    pdl_config(&cfg, &attr, dim3((unsigned)(share ? heads : (heads + 3) / 4)), dim3(share ? kJoinWarps * 32 : 128), 0, s);
    return cudaLaunchKernelEx(&cfg, paged_join_kernel<typename F::Joined>, a, share);
}

}  // namespace
}  // namespace zs
