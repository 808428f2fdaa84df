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
//   * paged_attn_kernel: all chunks in order go to the warps of the GPU in equal
//     runs, found by a prefix sum over the lengths in the kernel, so ragged
//     batches and single long sequences load every SM alike and no length is
//     needed on the host. A run that ends inside a unit leaves its (m, l, O) in a
//     workspace, and paged_join_kernel joins a unit's pieces in order.
//   * paged_attn_units_kernel: a fixed number of warps a unit, joined through
//     distributed shared memory in the same kernel: short units and page lists.
// Sums are always in the same order for the same sizes on the host and the same
// lengths: a result does not change from run to run.
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
#include <algorithm>
#include <atomic>
#include <cmath>
#include <type_traits>

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
    int max_len;              // host's bound on the lengths, 0: none (chooses the way, and so the order of sums)
    float scale2;             // softmax scale * log2(e)
    uint16_t* out;            // [B][Hq][D]
    float* lse;               // nullable: [B][Hq]
    long long* plan;          // workspace: [0] chunks a warp, [1 + unit] first chunk of the unit
    int prow;                 // rows of a piece: min(G, 16)
    float* part_ml;           // [2 W][prow][2], W warps
    float* part_o;            // [2 W][prow][D]
    unsigned* err;
};

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

// P is computed as 2^(s - m + bias): for fp16 the bias keeps probabilities down
// to 2^-39 of the largest above fp16's smallest step (long tails of a long cache
// would vanish otherwise); bf16 has fp32's exponents.
template <typename T>
constexpr float kPBias = 0.f;
template <>
constexpr float kPBias<__half> = 15.f;

__device__ __forceinline__ float2 ld_dsmem_f2(uint32_t addr) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
    return v;
}

// log sum exp of a row from its base-2 maximum and sum.
template <typename T>
__device__ __forceinline__ float log_sum(float m, float l) {
    return l == 0.f ? -INFINITY : (m + log2f(l) - kPBias<T>) / kLog2e;
}

// Chunks of entry e: a sequence (whole cache) or a (sequence, KV head) with a page list.
template <bool kListed>
__device__ __forceinline__ int entry_chunks(const PaArgs& a, int e) {
    if (kListed) return max(0, min(a.counts[e], a.top)) << (a.kp.page_shift - 4);
    const int cap = (int)min((long long)a.width << a.kp.page_shift, (long long)INT_MAX - 15);
    return (max(0, min(a.lens[e], cap)) + kPaChunk - 1) / kPaChunk;
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

// ---- a warp's work on a unit, shared by both kernels

// The block and the number of valid tokens of chunk `ch` of an entry (lim 0: none).
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
__device__ __forceinline__ void odd_values(const PaArgs& a, int e, int b, int h, int first, int count, int c0,
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
            if (lse && d0 == 0) lse[row] = log_sum<T>(m[r], l[r]);
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
            if (lse && d0 == 0) lse[row] = log_sum<T>(m[j], l[j]);
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

    __device__ __forceinline__ uint32_t slot(int s) const { return base + (s % C::kStages) * 2 * C::kTile; }
    template <typename Find>
    __device__ __forceinline__ void ask(const PaArgs& a, int s, Find&& find) {
        int lim = 0;
        if (s < steps) {
            int blk, ch, h;
            lim = find(blk, ch, h, s);
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

// Where a warp is in the sequence of all chunks: chunk `ch` of the n chunks of
// unit `in_e` of entry e.
struct PaCursor {
    int e, n, in_e, ch;
};

// To the next unit that has chunks (there is one: the caller has chunks left).
template <bool kListed>
__device__ __forceinline__ void next_unit(const PaArgs& a, int per_entry, PaCursor& c) {
    c.ch = 0;
    if (++c.in_e < per_entry) return;
    c.in_e = 0;
    do c.n = entry_chunks<kListed>(a, ++c.e);
    while (c.n == 0);
}

template <typename T, int D, bool kListed, bool kNarrow>
__global__ void __launch_bounds__(kPaThreads, PaCfg<D, kNarrow>::kCtas) paged_attn_kernel(const PaArgs a) {
    using C = PaCfg<D, kNarrow>;
    extern __shared__ __align__(1024) uint8_t pa_smem[];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    grid_dep_launch();
    grid_dep_wait();

    // ---- each warp's run of chunks
    const int entries = kListed ? a.B * a.Hkv : a.B;
    const int per_entry = kListed ? a.tiles : a.Hkv * a.tiles;     // units an entry
    // Each warp by itself: lane i sums the chunks of entries [i per, (i + 1) per),
    // a prefix over the lanes gives the total and the lane whose entries hold the
    // warp's first chunk, a second one over those entries the entry.
    const int per = (entries + 31) / 32;
    long long mine = 0;
    int n1 = 0;                    // the lane's last entry's (its only one up to 32 entries)
#pragma unroll 4
    for (int i = 0; i < per; ++i) {
        const int e = lane * per + i;
        n1 = e < entries ? entry_chunks<kListed>(a, e) : 0;
        mine += n1;
    }
    const long long inc = warp_prefix(mine);
    const long long total = __shfl_sync(~0u, inc, 31) * per_entry;
    const int warps = gridDim.x * kPaWarps;
    // two chunks or more: pieces of one would double what is joined (48 pages for 8
    // pairs 17.5 us, 16.3 so)
    const long long run = max(div_nonneg(total + warps - 1, warps), 2ll);
    if (blockIdx.x == 0 && tid == 0) a.plan[0] = run;
    // neighbouring runs go to different CTAs, so that few chunks spread over the SMs
    const int id = warp * (int)gridDim.x + (int)blockIdx.x;
    const long long c_begin = run * id;
    if (c_begin >= total) return;
    const int steps = (int)min(run, total - c_begin);
    const int owner = __ffs(__ballot_sync(~0u, inc * per_entry > c_begin)) - 1;
    long long lo = __shfl_sync(~0u, inc - mine, owner);            // entry chunks before, per unit
    int entry = owner * per, n = __shfl_sync(~0u, n1, owner);
    if (per > 1) {
        for (;; entry += 32) {
            const int e = entry + lane;
            const int ne = e < min(entries, (owner + 1) * per) ? entry_chunks<kListed>(a, e) : 0;
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

    // ---- copies: batches of up to 32 chunks of one unit, a lane holding the block
    // and the number of valid tokens of one chunk; the next batch is looked up
    // while the present one is copied
    const int table_len = (int)min((long long)a.width << a.kp.page_shift, (long long)INT_MAX);
    struct Batch {
        int ids, lims, count, h, ch;
    } now, next;
    int looked = 0;                // chunks looked up
    auto look = [&](Batch& t) {
        t.count = min(32, min(at.n - at.ch, steps - looked));
        t.ids = 0;
        t.lims = 0;
        t.ch = at.ch;
        t.h = kListed ? at.e % a.Hkv : at.in_e / a.tiles;
        if (t.count <= 0) return;
        if (lane < t.count) {
            const int b = kListed ? at.e / a.Hkv : at.e;
            look_chunk<kListed>(a, at.e, b, at.ch + lane, min(a.lens[b], table_len), t.ids, t.lims);
        }
        looked += t.count;
        at.ch += t.count;
        if (at.ch == at.n && looked < steps) next_unit<kListed>(a, per_entry, at);
    };
    look(now);
    int in_batch = 0;
    auto find = [&](int& blk, int& ch, int& h, int) {
        if (in_batch == now.count) {
            now = next;
            in_batch = 0;
            look(next);
        }
        blk = __shfl_sync(~0u, now.ids, in_batch);
        ch = now.ch + in_batch;
        h = now.h;
        return __shfl_sync(~0u, now.lims, in_batch++);
    };
    PaRing<D, kNarrow> ring;
    ring.base = smem_u32(pa_smem) + warp * C::kRing;
    ring.policy = evict_first_policy();
    ring.steps = steps;
#pragma unroll
    for (int s = 0; s < C::kStages - 1; ++s) {
        ring.ask(a, s, find);
        if (s == 0) look(next);    // the first chunk is on its way while the next batch is looked up
    }

    int s = 0;
    while (true) {
        // ---- a unit, or the part of it in this run
        const int first = cur.ch, count = min(cur.n - first, steps - s);
        const int b = kListed ? cur.e / a.Hkv : cur.e;
        const int h = kListed ? cur.e % a.Hkv : cur.in_e / a.tiles;
        const int tile = kListed ? cur.in_e : cur.in_e % a.tiles;
        const int g0 = tile * kPaRows, rows = min(kPaRows, a.G - g0);
        if (first == 0 && lane == 0) a.plan[1 + (b * a.Hkv + h) * a.tiles + tile] = u_lo;
        const long long head0 = (long long)b * a.Hq + (long long)h * a.G + g0;
        typename PaStateOf<T, D, kNarrow>::type st;
        st.start(a.q + head0 * D, rows);
        for (const int end = s + count; s < end; ++s) ring.step(a, s, st, find);
        // ---- out, or to the workspace where the run cuts the unit
        const bool whole = first == 0 && count == cur.n;
        const long long slot = 2ll * id + (s == count ? 0 : 1);       // the run's first part, or its last
        st.finish();
        if (whole) {
            if (__builtin_expect(st.odd(), false)) {
                uint32_t seen = 0;
                odd_values<T, D / 32, kListed>(a, cur.e, b, h, 0, cur.n, lane * (D / 32), seen);
                st.mend(seen);
            }
            st.write(a.out + head0 * D, a.lse ? a.lse + head0 : nullptr, rows);
        } else st.park(a.part_o + slot * a.prow * D, a.part_ml + slot * a.prow * 2, rows);
        if (s == steps) break;
        u_lo += cur.n;
        next_unit<kListed>(a, per_entry, cur);
    }
    cp_wait<0>();
}

// ---- Each unit by a fixed number W of warps, 1 to 16: no prefix over the
// lengths, no workspace and no second kernel. Warp w of the unit's W takes chunks
// [n w / W, n (w + 1) / W) of the unit's n, leaves (m, l, O) in its own shared
// memory, and after a cluster barrier the unit's threads join the W pieces
// through distributed shared memory, in order. With W below 4 a CTA has several
// units, from 4 on a cluster of W / 4 CTAs has one.
template <typename T, int D, bool kListed, bool kNarrow>
__global__ void __launch_bounds__(kPaThreads, PaCfg<D, kNarrow>::kCtas) paged_attn_units_kernel(const PaArgs a, int W) {
    using C = PaCfg<D, kNarrow>;
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
    const int len = min(a.lens[b], table_len), n = on ? entry_chunks<kListed>(a, e) : 0;
    const int first = (int)((long long)n * w / W), steps = (int)((long long)n * (w + 1) / W) - first;
    typename PaStateOf<T, D, kNarrow>::type st;
    int ids = 0, lims = 0;         // of 32 chunks, a lane each
    auto find = [&](int& blk, int& ch, int& head, int s) {
        if ((s & 31) == 0) {
            ids = lims = 0;
            if (s + lane < steps) look_chunk<kListed>(a, e, b, first + s + lane, len, ids, lims);
        }
        blk = __shfl_sync(~0u, ids, s & 31);
        ch = first + s;
        head = h;
        return __shfl_sync(~0u, lims, s & 31);
    };
    PaRing<D, kNarrow> ring;
    ring.base = smem_u32(pa_smem) + warp * C::kRing;
    ring.policy = evict_first_policy();
    ring.steps = steps;
#pragma unroll
    for (int s = 0; s < C::kStages - 1; ++s) ring.ask(a, s, find);
    st.start(a.q + head0 * D, rows);
    for (int s = 0; s < steps; ++s) ring.step(a, s, st, find);
    cp_wait<0>();
    __syncwarp();
    st.finish();
    // the warp's piece, over its ring: [16][D] outputs, [16][2] maxima and sums
    static_assert(C::kRing >= kPaRows * (D + 2) * 4, "a warp's piece fits its ring");
    float* po = reinterpret_cast<float*>(pa_smem + warp * C::kRing);
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
                    const uint32_t piece = peer + (v0 + v) * C::kRing;
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
        if (__builtin_expect(is_odd((acc.x * 0.f + acc.y * 0.f) + (acc.z * 0.f + acc.w * 0.f), l), false)) {
            const uint32_t odd = odd_channels<4>({acc.x, acc.y, acc.z, acc.w});
            uint32_t seen = 0;
            for (int v = 0; v < W && !odd_decided(seen, odd); ++v) {
                const uint32_t peer = W <= kPaWarps ? base : mapa_shared(base, v / kPaWarps);
                const float4 o = ld_dsmem_f4(peer + (v0 + v % kPaWarps) * C::kRing + (row * D + d4) * 4);
                const int c = (int)((long long)n * v / W), end = (int)((long long)n * (v + 1) / W);
                if (odd_channels<4>({o.x, o.y, o.z, o.w})) odd_values<T, 4, kListed>(a, e, b, h, c, end - c, d4, seen);
            }
            acc.x = odd_output(seen, 0, acc.x);
            acc.y = odd_output(seen, 1, acc.y);
            acc.z = odd_output(seen, 2, acc.z);
            acc.w = odd_output(seen, 3, acc.w);
        }
        const float inv = l == 0.f ? 0.f : 1.f / l;
        *reinterpret_cast<uint2*>(a.out + (head0 + row) * D + d4) =
            make_uint2(pack2<T>(acc.x * inv, acc.y * inv), pack2<T>(acc.z * inv, acc.w * inv));
        if (a.lse && d4 == 0) a.lse[head0 + row] = log_sum<T>(m, l);
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

template <typename T, int D, bool kListed>
__global__ void __launch_bounds__(kJoinWarps * 32) paged_join_kernel(const PaArgs a, int share) {
    constexpr int kVec = D / 32;
    __shared__ float s_acc[kJoinWarps][D], s_m[kJoinWarps], s_l[kJoinWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const int head = share ? (int)blockIdx.x : (int)blockIdx.x * warps + warp;
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
        // the first piece is the last of its warp's run unless it starts that run
        const bool second = lo != w0 * run;
        const int by = share ? warps : 1;
        for (int v = w0 + (share ? warp : 0); v <= w1; v += kJoinBatch * by) {
            float2 ml[kJoinBatch];
            float o[kJoinBatch][kVec];
#pragma unroll
            for (int x = 0; x < kJoinBatch; ++x) {
                const int w = v + x * by;
                const long long s = (2ll * w + (w == w0 && second ? 1 : 0)) * a.prow + row;
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
                odd_values<T, kVec, kListed>(a, kListed ? b * a.Hkv + h : b, b, h, (int)(c - lo), (int)(end - c),
                                             lane * kVec, seen);
        }
#pragma unroll
        for (int j = 0; j < kVec; ++j) acc[j] = odd_output(seen, j, acc[j]);
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    uint32_t* out = reinterpret_cast<uint32_t*>(a.out + (long long)head * D + lane * kVec);
#pragma unroll
    for (int j = 0; j < kVec; j += 2) out[j / 2] = pack2<T>(acc[j] * inv, acc[j + 1] * inv);
    if (a.lse && lane == 0) a.lse[head] = log_sum<T>(m, l);
}

// CTAs of the run kernel, at most.
inline int pa_max_ctas(int D, int G) {
    if (G <= 8) return 148 * (D <= 64 ? PaCfg<64, true>::kCtas : PaCfg<128, true>::kCtas);
    return 148 * (D <= 64 ? PaCfg<64, false>::kCtas : PaCfg<128, false>::kCtas);
}

size_t plan_bytes(long long units) { return ((size_t)(1 + units) * 8 + 255) / 256 * 256; }
// G is bounded by prow where it matters (both are above 8, or equal)
size_t ml_bytes(int prow, int D) { return (size_t)2 * pa_max_ctas(D, prow) * kPaWarps * prow * 2 * 4; }

// The attention kernel's grid: the CTAs that the GPU holds at once (looked up once per device).
template <typename T, int D, bool kListed, bool kNarrow>
cudaError_t resident_ctas(int* ctas) {
    static std::atomic<int> cached[64];
    const auto kernel = paged_attn_kernel<T, D, kListed, kNarrow>;
    int dev = 0, per = 0, sms = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    if ((*ctas = cached[dev].load(std::memory_order_acquire)) > 0) return cudaSuccess;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, PaCfg<D, kNarrow>::kSmem);
    if (e != cudaSuccess) return e;
    e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per, kernel, kPaThreads, PaCfg<D, kNarrow>::kSmem);
    if (e != cudaSuccess) return e;
    e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return e;
    if (per < 1) return cudaErrorInvalidConfiguration;
    *ctas = std::min(per * sms, pa_max_ctas(D, kNarrow ? 8 : 16));
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
// idle (B=1 T=4096: 9.6 and 15.6). W fills the GPU once, with two chunks a warp or
// more; units of unlike lengths in more waves want shares of some 12 chunks (128
// of 0..600: 41.1 us with one warp each, 28.7 with four, 31.4 in runs). Clusters of
// more than 4 CTAs were slower in all of these.
constexpr int kPaMaxUnitWarps = 16;

// A bound on a unit's chunks: of the page list, the table or the caller's.
inline long long unit_chunks(const PaArgs& a, bool listed) {
    const long long pages = ((long long)(listed ? a.top : a.width)) << (a.kp.page_shift - 4);
    return a.max_len > 0 && !listed ? std::min(pages, ((long long)a.max_len + kPaChunk - 1) / kPaChunk) : pages;
}

inline int unit_warps(const PaArgs& a, bool listed) {
    const long long units = (long long)a.B * a.Hkv * a.tiles, chunks = unit_chunks(a, listed);
    const long long resident = (long long)pa_max_ctas(a.kp.dim, a.G) * kPaWarps;
    int W = 1;
    while (W < kPaMaxUnitWarps && units * W * 2 <= resident && W * 4 <= chunks) W *= 2;
    while (!listed && W < kPaWarps && W * 12 < chunks) W *= 2;
    const long long steps = (chunks + W - 1) / W;
    const long long most = units * W < 148 * 4 ? 5 : listed ? 64 : 16;
    return steps <= most && units * W <= INT32_MAX ? W : 0;
}

template <typename T, int D, bool kListed, bool kNarrow>
cudaError_t launch_units(const PaArgs& a, int W, cudaStream_t s) {
    const auto kernel = paged_attn_units_kernel<T, D, kListed, kNarrow>;
    static std::atomic<unsigned long long> ready{0};      // a bit a device
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    if (!(ready.load(std::memory_order_acquire) >> dev & 1)) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, PaCfg<D, kNarrow>::kSmem);
        if (e != cudaSuccess) return e;
        ready.fetch_or(1ull << dev, std::memory_order_release);
    }
    const long long warps = (long long)a.B * a.Hkv * a.tiles * W;
    cudaLaunchConfig_t cfg;
    cudaLaunchAttribute attr[2];
    pdl_config(&cfg, attr, dim3((unsigned)((warps + kPaWarps - 1) / kPaWarps)), dim3(kPaThreads), PaCfg<D, kNarrow>::kSmem, s);
    if (W > kPaWarps) {
        attr[1].id = cudaLaunchAttributeClusterDimension;
        attr[1].val.clusterDim.x = W / kPaWarps;
        attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
        cfg.numAttrs = 2;
    }
    return cudaLaunchKernelEx(&cfg, kernel, a, W);
}

template <typename T, int D, bool kListed, bool kNarrow>
cudaError_t launch_paged(const PaArgs& a, cudaStream_t s) {
    if (const int W = unit_warps(a, kListed)) return launch_units<T, D, kListed, kNarrow>(a, W, s);
    int ctas = 0;
    cudaError_t e = resident_ctas<T, D, kListed, kNarrow>(&ctas);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg;
    cudaLaunchAttribute attr;
    pdl_config(&cfg, &attr, dim3(ctas), dim3(kPaThreads), PaCfg<D, kNarrow>::kSmem, s);
    e = cudaLaunchKernelEx(&cfg, paged_attn_kernel<T, D, kListed, kNarrow>, a);
    if (e != cudaSuccess) return e;
    // a head a CTA while there are SMs for it, else a head a warp in small CTAs
    const int heads = a.B * a.Hq, share = heads <= kJoinShare ? 1 : 0;
    pdl_config(&cfg, &attr, dim3((unsigned)(share ? heads : (heads + 3) / 4)), dim3(share ? kJoinWarps * 32 : 128), 0, s);
    return cudaLaunchKernelEx(&cfg, paged_join_kernel<T, D, kListed>, a, share);
}

template <typename T, bool kListed>
cudaError_t dispatch_dim(const PaArgs& a, cudaStream_t s) {
    switch (a.kp.dim) {
        case 64: return a.G <= 8 ? launch_paged<T, 64, kListed, true>(a, s) : launch_paged<T, 64, kListed, false>(a, s);
        case 128: return a.G <= 8 ? launch_paged<T, 128, kListed, true>(a, s) : launch_paged<T, 128, kListed, false>(a, s);
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
    return plan_bytes((long long)B * Hkv * tiles) + ml_bytes(prow, D) + (size_t)2 * pa_max_ctas(D, prow) * kPaWarps * prow * D * 4;
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
    if (!attention_args(p, &a) || a.B == 0 || unit_warps(a, a.pages != nullptr)) return 0;
    return zs_paged_attention_workspace_bytes(a.B, a.Hq, a.Hkv, a.kp.dim);
}

extern "C" int zs_paged_attention(const ZsPagedAttention* p) {
    using namespace zs;
    PaArgs a{};
    if (!attention_args(p, &a)) return cudaErrorInvalidValue;
    if (a.B == 0) return cudaSuccess;
    if (!unit_warps(a, a.pages != nullptr)) {
        if (!p->ws || !aligned16p(p->ws) ||
            p->ws_bytes < zs_paged_attention_workspace_bytes(a.B, a.Hq, a.Hkv, a.kp.dim))
            return cudaErrorInvalidValue;
        uint8_t* ws = static_cast<uint8_t*>(p->ws);
        a.plan = reinterpret_cast<long long*>(ws);
        ws += plan_bytes((long long)a.B * a.Hkv * a.tiles);
        a.part_ml = reinterpret_cast<float*>(ws);
        ws += ml_bytes(a.prow, a.kp.dim);
        a.part_o = reinterpret_cast<float*>(ws);
    }
    cudaStream_t s = (cudaStream_t)p->stream;
    if (p->k_pool.dtype == ZS_BF16)
        return a.pages ? dispatch_dim<__nv_bfloat16, true>(a, s) : dispatch_dim<__nv_bfloat16, false>(a, s);
    return a.pages ? dispatch_dim<__half, true>(a, s) : dispatch_dim<__half, false>(a, s);
}
