// Attention of one new token per sequence over a paged KV cache, the whole
// cache or a chosen list of its pages (zs_paged_attention).
//
//   out[b][i] = sum_t exp(s_t - m) v_t / sum_t exp(s_t - m),  s_t = scale q[b][i] . k_t,
// t over the sequence's tokens (of the listed pages), k and v of KV head
// i / (Hq / Hkv), m = max s_t; zero where nothing is attended. One pass: every
// warp keeps a running maximum, sum and unnormalised output in fp32 registers.
//
// Bound by HBM: each K and V row is read once for all the query heads that share
// it. The work is cut into chunks of 16 tokens of a unit (sequence, KV head, tile
// of up to 16 query heads); all chunks in order are dealt to the CTAs in equal
// runs, found by a prefix sum over the lengths in the kernel, so ragged batches
// and single long sequences load every SM alike and no length is needed on the
// host. A run that ends inside a unit leaves its (m, l, O) in a workspace and a
// second kernel joins a unit's pieces in order.
//
// Inside a CTA each warp works on every fourth chunk by itself: it copies its
// chunk's K and V rows with 16-byte cp.async into its own ring (rows past the
// length are zero-filled and never read), so there is no barrier in the loop.
// S = Q K^T and O += P V are m16n8k16 products: the rows are query heads, of
// which a decode step has 1 to 16 a KV head, far below a tcgen05 tile's 128, and
// the tensor work is a third of the memory time even with rows unused.
// P is fed as a 16-bit high part plus its 16-bit remainder, so that rounding P
// adds nothing to the output's own rounding.
#include <algorithm>
#include <atomic>
#include <cmath>

#include "paged.cuh"

namespace zs {
namespace {

constexpr int kPaWarps = 4;
constexpr int kPaThreads = kPaWarps * 32;
constexpr int kPaChunk = 16;       // tokens a warp step; pages are multiples of it
constexpr int kPaRows = 16;        // query heads a unit
constexpr float kLog2e = 1.4426950408889634f;

struct PaArgs {
    const uint16_t* q;        // [B][Hq][D]
    PoolView kp, vp;
    const int* table;
    long long table_stride;
    const int* lens;
    const int* pages;         // nullable: [B][Hkv][top]
    const int* counts;        // with pages: [B][Hkv]
    int B, Hq, Hkv, G, tiles, width, top;
    float scale2;             // softmax scale * log2(e)
    uint16_t* out;            // [B][Hq][D]
    float* lse;               // nullable: [B][Hq]
    long long* plan;          // workspace: [0] chunks a CTA, [1 + unit] first chunk of the unit
    float* part_ml;           // [2 W][16][2]
    float* part_o;            // [2 W][16][D]
    unsigned* err;
};

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool on) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
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

// P is computed as 2^(s - m + bias): for fp16 the bias keeps probabilities down
// to 2^-39 of the largest above fp16's smallest step (long tails of a long cache
// would vanish otherwise); bf16 has fp32's exponents.
template <typename T>
constexpr float kPBias = 0.f;
template <>
constexpr float kPBias<__half> = 15.f;

// Chunks of entry e: a sequence (whole cache) or a (sequence, KV head) with a page list.
template <bool kListed>
__device__ __forceinline__ int entry_chunks(const PaArgs& a, int e) {
    if (kListed) return max(0, min(a.counts[e], a.top)) << (a.kp.page_shift - 4);
    const int cap = (int)min((long long)a.width << a.kp.page_shift, (long long)INT_MAX - 15);
    return (max(0, min(a.lens[e], cap)) + kPaChunk - 1) / kPaChunk;
}

__device__ __forceinline__ long long warp_sum(long long v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
    return v;
}

template <int D>
struct PaCfg {
    static constexpr int kRowBytes = D * 2;
    static constexpr int kTile = kPaChunk * kRowBytes;             // one K or V chunk
    static constexpr int kStages = D <= 64 ? 6 : (D <= 128 ? 3 : 2);
    static constexpr int kRing = kStages * 2 * kTile;              // a warp's ring
    static constexpr int kMerge = kPaWarps * kPaRows * (D + 2) * 4;
    static constexpr int kSmem = kPaWarps * kRing > kMerge ? kPaWarps * kRing : kMerge;
};

template <typename T, int D, bool kListed>
__global__ void __launch_bounds__(kPaThreads) paged_attn_kernel(const PaArgs a) {
    using C = PaCfg<D>;
    constexpr int kPieces = D / 8;                 // 16-byte pieces a row
    constexpr int kKs = D / 16;
    extern __shared__ __align__(1024) uint8_t pa_smem[];
    __shared__ long long s_red[2][kPaWarps];
    __shared__ long long s_lo;
    __shared__ int s_entry, s_chunks;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t ring = smem_u32(pa_smem) + warp * C::kRing;
    grid_dep_launch();
    grid_dep_wait();

    // ---- this CTA's run of chunks
    const int entries = kListed ? a.B * a.Hkv : a.B;
    const int per_entry = kListed ? a.tiles : a.Hkv * a.tiles;     // units an entry
    // chunks in all, and (one load for up to kPaThreads entries) this thread's first entry's
    const int n0 = tid < entries ? entry_chunks<kListed>(a, tid) : 0;
    long long mine = n0;
    for (int e = tid + kPaThreads; e < entries; e += kPaThreads) mine += entry_chunks<kListed>(a, e);
    long long inc0 = n0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long u = __shfl_up_sync(~0u, inc0, o);
        if (lane >= o) inc0 += u;
    }
    mine = entries <= kPaThreads ? __shfl_sync(~0u, inc0, 31) : warp_sum(mine);
    if (lane == 31) s_red[0][warp] = inc0;
    if (lane == 0) s_red[1][warp] = mine;
    __syncthreads();
    long long total = 0;
#pragma unroll
    for (int w = 0; w < kPaWarps; ++w) total += s_red[1][w];
    total *= per_entry;
    const long long run = max(div_nonneg(total + gridDim.x - 1, gridDim.x), (long long)kPaWarps);
    if (blockIdx.x == 0 && tid == 0) a.plan[0] = run;
    const long long c_begin = run * blockIdx.x, c_end = min(total, c_begin + run);
    if (c_begin >= c_end) return;
    // the entry that holds c_begin
    long long base = 0;
    for (int e0 = 0; e0 < entries; e0 += kPaThreads) {
        const int e = e0 + tid;
        int n = n0;
        long long inc = inc0;
        if (e0) {
            __syncthreads();
            n = e < entries ? entry_chunks<kListed>(a, e) : 0;
            inc = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const long long u = __shfl_up_sync(~0u, inc, o);
                if (lane >= o) inc += u;
            }
            if (lane == 31) s_red[0][warp] = inc;
            __syncthreads();
        }
        long long before = base;
        for (int w = 0; w < kPaWarps; ++w) {
            if (w < warp) before += s_red[0][w];
            base += s_red[0][w];
        }
        const long long lo = (before + inc - n) * per_entry, hi = (before + inc) * per_entry;
        if (lo <= c_begin && c_begin < hi) {
            s_entry = e;
            s_chunks = n;
            s_lo = lo;
        }
        if (base * per_entry > c_begin) break;
    }
    __syncthreads();
    int e = s_entry, n = s_chunks;
    long long e_lo = s_lo;

    long long c = c_begin;
    while (c < c_end) {
        while (n == 0 || e_lo + (long long)n * per_entry <= c) {     // next entry with chunks left
            e_lo += (long long)n * per_entry;
            n = entry_chunks<kListed>(a, ++e);
        }
        const int in_e = (int)div_nonneg(c - e_lo, n);                 // unit of the entry
        const long long u_lo = e_lo + (long long)in_e * n;
        const int first = (int)(c - u_lo);
        const int last = (int)min((long long)n, c_end - u_lo);
        const int b = kListed ? e / a.Hkv : e;
        const int h = kListed ? e % a.Hkv : in_e / a.tiles;
        const int tile = kListed ? in_e : in_e % a.tiles;
        const int g0 = tile * kPaRows, rows = min(kPaRows, a.G - g0);
        const int unit = (b * a.Hkv + h) * a.tiles + tile;
        if (first == 0 && tid == 0) a.plan[1 + unit] = u_lo;
        const long long cap = (long long)a.width << a.kp.page_shift;
        const int len = (int)max(0ll, min((long long)a.lens[b], cap));

        // ---- Q fragments (on their way while the first chunks' blocks are looked up)
        uint32_t qf[kKs][4];
        {
            const uint16_t* q = a.q + ((long long)b * a.Hq + (long long)h * a.G + g0) * D;
            const int r = lane >> 2, cc = (lane & 3) * 2;
#pragma unroll
            for (int ks = 0; ks < kKs; ++ks)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int row = r + (i & 1) * 8, col = ks * 16 + (i >> 1) * 8 + cc;
                    qf[ks][i] = row < rows ? *reinterpret_cast<const uint32_t*>(q + (long long)row * D + col) : 0u;
                }
        }
        float o[D / 8][4];
#pragma unroll
        for (int i = 0; i < D / 8; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) o[i][j] = 0.f;
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

        // ---- chunks first + warp, + 4, ...
        const int steps = (last - first - warp + kPaWarps - 1) / kPaWarps;
        const int cps = a.kp.page_shift - 4;                           // log2 chunks a page
        // tokens of the step's chunk that count, and its block; lane 0..31 hold 32 steps' worth
        int ids = 0, lims = 0;
        auto fetch = [&](int s0) {
            const int s = s0 + lane;
            ids = 0;
            lims = 0;
            if (s < steps) {
                const int ch = first + warp + s * kPaWarps;
                int p = ch >> cps;
                if (kListed) p = a.pages[(long long)e * a.top + p];
                const int t0 = ((p << cps) + (ch & ((1 << cps) - 1))) * kPaChunk;
                if (p >= 0 && p < a.width && t0 < len) {
                    ids = a.table[b * a.table_stride + p];
                    lims = min(kPaChunk, len - t0);
                    if (ids < 0 || ids >= a.kp.num_blocks) {
                        set_err(a.err, kErrPagedIndex);
                        ids = 0;
                        lims = 0;
                    }
                }
            }
        };
        const uint16_t* kbase = static_cast<const uint16_t*>(a.kp.data) + h * a.kp.s_head;
        const uint16_t* vbase = static_cast<const uint16_t*>(a.vp.data) + h * a.vp.s_head;
        auto produce = [&](int s) {
            if (s < steps) {
                if (s > 0 && (s & 31) == 0) fetch(s);
                const int blk = __shfl_sync(~0u, ids, s & 31), lim = __shfl_sync(~0u, lims, s & 31);
                const int row0 = ((first + warp + s * kPaWarps) & ((1 << cps) - 1)) * kPaChunk;
                const uint16_t* ks = kbase + blk * a.kp.s_block + row0 * a.kp.s_token;
                const uint16_t* vs = vbase + blk * a.vp.s_block + row0 * a.vp.s_token;
                const uint32_t dst = ring + (s % C::kStages) * 2 * C::kTile;
#pragma unroll
                for (int i = 0; i < kPaChunk * kPieces / 32; ++i) {
                    const int x = i * 32 + lane, r = x / kPieces, pc = x % kPieces;
                    const uint32_t at = dst + r * C::kRowBytes + ((pc ^ (r & 7)) * 16);
                    cp16(at, ks + r * a.kp.s_token + pc * 8, r < lim);
                    cp16(at + C::kTile, vs + r * a.vp.s_token + pc * 8, r < lim);
                }
            }
            cp_commit();
        };
        fetch(0);
        // limits of the steps in flight, oldest first
        int lim_at[C::kStages];
#pragma unroll
        for (int s = 0; s < C::kStages - 1; ++s) {
            produce(s);
            lim_at[s] = __shfl_sync(~0u, lims, s & 31);
        }
        for (int s = 0; s < steps; ++s) {
            cp_wait<C::kStages - 2>();
            __syncwarp();
            produce(s + C::kStages - 1);
            lim_at[C::kStages - 1] = __shfl_sync(~0u, lims, (s + C::kStages - 1) & 31);
            const int lim = lim_at[0];
#pragma unroll
            for (int i = 0; i + 1 < C::kStages; ++i) lim_at[i] = lim_at[i + 1];
            const uint32_t kt = ring + (s % C::kStages) * 2 * C::kTile, vt = kt + C::kTile;
            // S = Q K^T: 16 heads x 16 tokens
            float sc[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
            {
                const int r = (lane & 7) + ((lane >> 4) << 3), half = (lane >> 3) & 1;
                const uint32_t row = kt + r * C::kRowBytes;
#pragma unroll
                for (int ks = 0; ks < kKs; ++ks) {
                    uint32_t f[4];
                    ldsm4(f, row + (((ks * 2 + half) ^ (r & 7)) * 16));
                    mma16816(sc[0], qf[ks], f[0], f[1], T());
                    mma16816(sc[1], qf[ks], f[2], f[3], T());
                }
            }
            // running maximum and sum
            const int t = (lane & 3) * 2;
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
                        const float x = j * 8 + t + i < lim ? sc[j][r * 2 + i] * a.scale2 : -INFINITY;
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
            // O += P V, P in two 16-bit parts
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float x = p[i >> 1][(i & 1) * 2], y = p[i >> 1][(i & 1) * 2 + 1];
                hi[i] = pack2<T>(x, y);
                const float2 back = unpack2<T>(hi[i]);
                lo[i] = pack2<T>(x - back.x, y - back.y);
            }
            {
                const int r = lane & 15, half = lane >> 4;
                const uint32_t row = vt + r * C::kRowBytes;
#pragma unroll
                for (int ks = 0; ks < kKs; ++ks) {
                    uint32_t f[4];
                    ldsm4t(f, row + (((ks * 2 + half) ^ (r & 7)) * 16));
                    mma16816(o[ks * 2], hi, f[0], f[1], T());
                    mma16816(o[ks * 2 + 1], hi, f[2], f[3], T());
                    mma16816(o[ks * 2], lo, f[0], f[1], T());
                    mma16816(o[ks * 2 + 1], lo, f[2], f[3], T());
                }
            }
            __syncwarp();
        }
        cp_wait<0>();
        __syncthreads();
        // ---- join the four warps through shared memory
        float* mo = reinterpret_cast<float*>(pa_smem);                  // [warp][16][D]
        float* ml = mo + kPaWarps * kPaRows * D;                        // [warp][16][2]
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            l[r] += __shfl_xor_sync(~0u, l[r], 1);
            l[r] += __shfl_xor_sync(~0u, l[r], 2);
            const int row = (lane >> 2) + r * 8;
            if ((lane & 3) == 0) {
                ml[(warp * kPaRows + row) * 2] = m[r];
                ml[(warp * kPaRows + row) * 2 + 1] = l[r];
            }
#pragma unroll
            for (int i = 0; i < D / 8; ++i)
                *reinterpret_cast<float2*>(mo + (warp * kPaRows + row) * D + i * 8 + (lane & 3) * 2) =
                    make_float2(o[i][r * 2], o[i][r * 2 + 1]);
        }
        __syncthreads();
        const bool whole = first == 0 && last == n;
        const long long slot = 2ll * blockIdx.x + (c == c_begin ? 0 : 1);
        for (int x = tid; x < rows * (D / 4); x += kPaThreads) {
            const int row = x / (D / 4), d4 = x % (D / 4) * 4;
            float mm = -INFINITY;
#pragma unroll
            for (int w = 0; w < kPaWarps; ++w) mm = fmaxf(mm, ml[(w * kPaRows + row) * 2]);
            const float ref = mm == -INFINITY ? 0.f : mm;
            float ll = 0.f;
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < kPaWarps; ++w) {
                const float f = exp2f(ml[(w * kPaRows + row) * 2] - ref);
                ll += ml[(w * kPaRows + row) * 2 + 1] * f;
                const float4 v = *reinterpret_cast<const float4*>(mo + (w * kPaRows + row) * D + d4);
                acc.x += v.x * f;
                acc.y += v.y * f;
                acc.z += v.z * f;
                acc.w += v.w * f;
            }
            if (whole) {
                const float inv = ll == 0.f ? 0.f : 1.f / ll;
                const long long at = (long long)b * a.Hq + (long long)h * a.G + g0 + row;
                *reinterpret_cast<uint2*>(a.out + at * D + d4) =
                    make_uint2(pack2<T>(acc.x * inv, acc.y * inv), pack2<T>(acc.z * inv, acc.w * inv));
                if (a.lse && d4 == 0) a.lse[at] = ll == 0.f ? -INFINITY : (mm + log2f(ll) - kPBias<T>) / kLog2e;
            } else {
                *reinterpret_cast<float4*>(a.part_o + (slot * kPaRows + row) * D + d4) = acc;
                if (d4 == 0) {
                    a.part_ml[(slot * kPaRows + row) * 2] = mm;
                    a.part_ml[(slot * kPaRows + row) * 2 + 1] = ll;
                }
            }
        }
        __syncthreads();
        c = u_lo + last;
    }
}

// Joins the pieces of the units that the runs cut and writes zeros where nothing
// is attended. A warp takes a query head, D / 32 channels a lane; with few heads
// (long sequences: up to one piece a CTA of the attention kernel) the eight warps
// of a CTA share one head's pieces, so that their loads are in flight together,
// and add their sums in order.
constexpr int kJoinWarps = 8;

template <typename T, int D, bool kListed>
__global__ void __launch_bounds__(kJoinWarps * 32) paged_join_kernel(const PaArgs a, int share) {
    constexpr int kVec = D / 32;
    __shared__ float s_acc[kJoinWarps][D], s_m[kJoinWarps], s_l[kJoinWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int head = share ? (int)blockIdx.x : (int)blockIdx.x * kJoinWarps + warp;
    if (head >= a.B * a.Hq) return;
    const int b = head / a.Hq, i = head % a.Hq, h = i / a.G, g = i % a.G;
    const int tile = g / kPaRows, row = g % kPaRows;
    grid_dep_wait();
    const long long run = a.plan[0], lo = a.plan[1 + (b * a.Hkv + h) * a.tiles + tile];
    const int n = entry_chunks<kListed>(a, kListed ? b * a.Hkv + h : b);
    float m = -INFINITY, l = 0.f, acc[kVec];
#pragma unroll
    for (int j = 0; j < kVec; ++j) acc[j] = 0.f;
    if (n > 0) {
        const int w0 = (int)div_nonneg(lo, run), w1 = (int)div_nonneg(lo + n - 1, run);
        if (w0 == w1) return;                   // written whole
        // the first piece is the last of its CTA's run unless it starts that run
        const bool second = lo != w0 * run;
        const int first = share ? warp : 0, by = share ? kJoinWarps : 1;
#pragma unroll 4
        for (int w = w0 + first; w <= w1; w += by) {
            const long long s = (2ll * w + (w == w0 && second ? 1 : 0)) * kPaRows + row;
            const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + s * 2);
            float o[kVec];
            const float* src = a.part_o + s * D + lane * kVec;
            if constexpr (kVec == 4) *reinterpret_cast<float4*>(o) = *reinterpret_cast<const float4*>(src);
            else *reinterpret_cast<float2*>(o) = *reinterpret_cast<const float2*>(src);
            const float mn = fmaxf(m, ml.x), ref = mn == -INFINITY ? 0.f : mn;
            const float f0 = exp2f(m - ref), f1 = exp2f(ml.x - ref);
            l = l * f0 + ml.y * f1;
#pragma unroll
            for (int j = 0; j < kVec; ++j) acc[j] = acc[j] * f0 + o[j] * f1;
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
        m = s_m[0];
#pragma unroll
        for (int w = 1; w < kJoinWarps; ++w) m = fmaxf(m, s_m[w]);
        const float ref = m == -INFINITY ? 0.f : m;
        l = 0.f;
#pragma unroll
        for (int j = 0; j < kVec; ++j) acc[j] = 0.f;
#pragma unroll
        for (int w = 0; w < kJoinWarps; ++w) {
            const float f = exp2f(s_m[w] - ref);
            l += s_l[w] * f;
#pragma unroll
            for (int j = 0; j < kVec; ++j) acc[j] += s_acc[w][lane * kVec + j] * f;
        }
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    uint32_t* out = reinterpret_cast<uint32_t*>(a.out + (long long)head * D + lane * kVec);
#pragma unroll
    for (int j = 0; j < kVec; j += 2) out[j / 2] = pack2<T>(acc[j] * inv, acc[j + 1] * inv);
    if (a.lse && lane == 0) a.lse[head] = l == 0.f ? -INFINITY : (m + log2f(l) - kPBias<T>) / kLog2e;
}

constexpr int kPaMaxCtas = 148 * 4;      // the workspace's bound on the grid

size_t plan_bytes(long long units) { return ((size_t)(1 + units) * 8 + 255) / 256 * 256; }
size_t ml_bytes() { return (size_t)2 * kPaMaxCtas * kPaRows * 2 * 4; }

// The attention kernel's grid: the CTAs that the GPU holds at once (looked up once per device).
template <typename T, int D, bool kListed>
cudaError_t resident_ctas(int* ctas) {
    static std::atomic<int> cached[64];
    const auto kernel = paged_attn_kernel<T, D, kListed>;
    int dev = 0, per = 0, sms = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    if ((*ctas = cached[dev].load(std::memory_order_acquire)) > 0) return cudaSuccess;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, PaCfg<D>::kSmem);
    if (e != cudaSuccess) return e;
    e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per, kernel, kPaThreads, PaCfg<D>::kSmem);
    if (e != cudaSuccess) return e;
    e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return e;
    if (per < 1) return cudaErrorInvalidConfiguration;
    *ctas = std::min(per * sms, kPaMaxCtas);
    cached[dev].store(*ctas, std::memory_order_release);
    return cudaSuccess;
}

template <typename T, int D, bool kListed>
cudaError_t launch_paged(const PaArgs& a, cudaStream_t s) {
    int ctas = 0;
    cudaError_t e = resident_ctas<T, D, kListed>(&ctas);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg;
    cudaLaunchAttribute attr;
    pdl_config(&cfg, &attr, dim3(ctas), dim3(kPaThreads), PaCfg<D>::kSmem, s);
    e = cudaLaunchKernelEx(&cfg, paged_attn_kernel<T, D, kListed>, a);
    if (e != cudaSuccess) return e;
    // heads enough to fill the GPU by a warp each, or a CTA each
    const int heads = a.B * a.Hq, share = heads < 148 * kJoinWarps ? 1 : 0;
    pdl_config(&cfg, &attr, dim3((unsigned)(share ? heads : (heads + kJoinWarps - 1) / kJoinWarps)),
               dim3(kJoinWarps * 32), 0, s);
    return cudaLaunchKernelEx(&cfg, paged_join_kernel<T, D, kListed>, a, share);
}

template <typename T, bool kListed>
cudaError_t dispatch_dim(const PaArgs& a, cudaStream_t s) {
    switch (a.kp.dim) {
        case 64: return launch_paged<T, 64, kListed>(a, s);
        case 128: return launch_paged<T, 128, kListed>(a, s);
    }
    return cudaErrorInvalidValue;
}

}  // namespace
}  // namespace zs

extern "C" size_t zs_paged_attention_workspace_bytes(int B, int Hq, int Hkv, int D) {
    using namespace zs;
    if (B <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || D <= 0) return 0;
    const long long tiles = (Hq / Hkv + kPaRows - 1) / kPaRows;
    return plan_bytes((long long)B * Hkv * tiles) + ml_bytes() + (size_t)2 * kPaMaxCtas * kPaRows * D * 4;
}

extern "C" int zs_paged_attention(const ZsPagedAttention* p) {
    using namespace zs;
    PaArgs a{};
    if (!p || !make_pool(&p->k_pool, &a.kp) || !make_pool(&p->v_pool, &a.vp) || !same_pools(p->k_pool, p->v_pool))
        return cudaErrorInvalidValue;
    const int B = p->B, Hq = p->Hq, Hkv = a.kp.heads, D = a.kp.dim, top = p->top;
    if (B < 0 || Hq <= 0 || Hq % Hkv || p->width <= 0 || p->table_stride < p->width ||
        !std::isfinite(p->softmax_scale))
        return cudaErrorInvalidValue;
    if (B == 0) return cudaSuccess;
    a.G = Hq / Hkv;
    a.tiles = (a.G + kPaRows - 1) / kPaRows;
    if ((long long)B * Hq > INT32_MAX || (long long)p->width << a.kp.page_shift > INT32_MAX) return cudaErrorInvalidValue;
    if (!p->q || !p->block_table || !p->seq_lens || !p->out || !p->ws || !aligned16p(p->q) || !aligned16p(p->out) ||
        !aligned16p(p->ws) || p->ws_bytes < zs_paged_attention_workspace_bytes(B, Hq, Hkv, D))
        return cudaErrorInvalidValue;
    if (!p->pages != !p->counts || (p->pages && (top <= 0 || (long long)top << a.kp.page_shift > INT32_MAX)))
        return cudaErrorInvalidValue;
    a.q = p->q;
    a.table = p->block_table;
    a.table_stride = p->table_stride;
    a.lens = p->seq_lens;
    a.pages = p->pages;
    a.counts = p->counts;
    a.B = B; a.Hq = Hq; a.Hkv = Hkv; a.width = p->width; a.top = top;
    a.scale2 = p->softmax_scale * kLog2e;
    a.out = p->out;
    a.lse = p->lse;
    uint8_t* ws = static_cast<uint8_t*>(p->ws);
    a.plan = reinterpret_cast<long long*>(ws);
    ws += plan_bytes((long long)B * Hkv * a.tiles);
    a.part_ml = reinterpret_cast<float*>(ws);
    ws += ml_bytes();
    a.part_o = reinterpret_cast<float*>(ws);
    a.err = p->err;
    cudaStream_t s = (cudaStream_t)p->stream;
    if (p->k_pool.dtype == ZS_BF16)
        return a.pages ? dispatch_dim<__nv_bfloat16, true>(a, s) : dispatch_dim<__nv_bfloat16, false>(a, s);
    return a.pages ? dispatch_dim<__half, true>(a, s) : dispatch_dim<__half, false>(a, s);
}
