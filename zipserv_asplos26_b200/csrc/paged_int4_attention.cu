// Entry points of attention over a 4-bit paged KV cache: checks, the workspace and the
// choice of the kernel (paged_int4_attention.cuh).
#include "paged_int4_attention.cuh"

namespace zs {
namespace {

constexpr float kMostScale = 0x1p57f;        // scores are brought up by 2^69 (Q4State::unit)

// CTAs of the run kernel, at most.
inline int q4_max_ctas(int D, int G) {
    if (G <= 8) return 148 * (D == 64 ? Q4Cfg<64, 1, false>::kCtas : Q4Cfg<128, 1, false>::kCtas);
    return 148 * (D == 64 ? Q4Cfg<64, 2, false>::kCtas : Q4Cfg<128, 2, false>::kCtas);
}
// Warps a unit, or 0 for runs. A chunk is 32 tokens in units, so runs pay from fewer of
// them on than with 16-bit pages (us in runs and in units, bf16, 32 query and 8 KV heads of
// 128, page lists as batch x pages of 64):
//   up to 5 a warp     B=1 T=2000 10.6 and 8.4; B=16 T=1000 12.2 and 12.4; 24 of 0..600
//                      12.8 and 9.3; 8 x 16 12.4 and 10.2
//   8 to 10            B=32 T=1000 16.9 and 19.0, T=800 16.9 and 15.9; B=128 T=300 19.5 and
//                      23.8; 64 of 0..1000 23.3 and 21.0; 300 of 0..600 52.2 and 44.4;
//                      512 of 300 61.3 and 56.1; 8 x 64 18.5 and 21.0
//   12 to 16           B=32 T=1500 21.4 and 26.0, T=2000 26.4 and 33.0; B=64 T=2000 41.9 and
//                      47.6; 100 of 0..1500 39.9 and 37.6; 200 x 8 41.7 and 36.1; 8 x 128
//                      27.9 and 35.0
//   32                 32 x 64 41.7 and 61.4; 128 x 16 47.3 and 62.5; 8 x 256 43.3 and 62.9
// and where units leave SMs idle, 1 x 64 and 2 x 64 (8 chunks) 11.0 and 12.1, 12.3 and 12.6.
inline int q4_unit_warps(const Q4Args& a) {
    using One = Q4Cfg<128, 1, true>;
    using Two = Q4Cfg<128, 2, true>;
    static_assert(One::kParts == 2 && Two::kParts == 2, "units' chunks are two parts");
    UnitLimits limits;
    limits.whole = 10;
    limits.listed = 16;
    return unit_warps(a, a.pages != nullptr, 148 * (a.G <= 8 ? One::kCtas : Two::kCtas), 2, limits);
}

// The checked arguments of a call, but for its workspace.
bool int4_attention_args(const ZsPagedAttentionInt4* p, Q4Args* a, int* groups) {
    Int4View k, v;
    if (!p || !make_int4_pool(&p->k_pool, &k) || !make_int4_pool(&p->v_pool, &v) || !same_int4_pools(p->k_pool, p->v_pool))
        return false;
    const int B = p->B, Hq = p->Hq, Hkv = k.heads, top = p->top;
    if (B < 0 || Hq <= 0 || Hq % Hkv || p->width <= 0 || p->table_stride < p->width || !(std::fabs(p->softmax_scale) < kMostScale) ||
        (p->dtype != ZS_BF16 && p->dtype != ZS_FP16))
        return false;
    if ((long long)B * Hq > INT32_MAX || (long long)p->width << k.page_shift > INT32_MAX) return false;
    if (B && (!p->q || !p->block_table || !p->seq_lens || !p->out || !aligned16p(p->q) || !aligned16p(p->out)))
        return false;
    if (!p->pages != !p->counts || (p->pages && (top <= 0 || (long long)top << k.page_shift > INT32_MAX))) return false;
    a->kp = {k.codes, k.c_block, k.c_token, k.c_head, k.num_blocks, k.page_shift, k.heads, k.dim};
    a->vp = {v.codes, v.c_block, v.c_token, v.c_head, v.num_blocks, v.page_shift, v.heads, v.dim};
    auto places = [](Q4Places* x, const void* base, long long block, long long token, long long head) {
        x->base = static_cast<const uint8_t*>(base);
        x->block = (uint32_t)block;
        x->token = (uint32_t)token;
        x->head = (uint32_t)head;
        return block <= UINT32_MAX && token <= UINT32_MAX && head <= UINT32_MAX;
    };
    if (!places(&a->kcode, k.codes, k.c_block, k.c_token, k.c_head) ||
        !places(&a->vcode, v.codes, v.c_block, v.c_token, v.c_head) ||
        !places(&a->kpar, k.params, 2 * k.p_block, 2 * k.p_token, 2 * k.p_head) ||
        !places(&a->vpar, v.params, 2 * v.p_block, 2 * v.p_token, 2 * v.p_head))
        return false;
    const uint32_t row = k.dim / 2, par = 4 * k.groups;
    a->packed = a->kcode.token == row && a->vcode.token == row && a->kpar.token == par && a->vpar.token == par;
    *groups = k.groups;
    a->G = Hq / Hkv;
    a->tiles = (a->G + kPaRows - 1) / kPaRows;
    a->prow = std::min(a->G, kPaRows);
    a->q = p->q;
    a->table = p->block_table;
    a->table_stride = p->table_stride;
    a->lens = p->seq_lens;
    a->group = !a->packed && !p->pages && Hkv * a->tiles % kPaWarps == 0 ? kPaWarps : 1;
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

size_t int4_workspace(const Q4Args& a) {
    return run_workspace_bytes((long long)a.B * a.Hkv * a.tiles, q4_max_ctas(a.kp.dim, a.G), a.prow, a.kp.dim);
}

}  // namespace
}  // namespace zs

extern "C" size_t zs_paged_attention_int4_workspace(const ZsPagedAttentionInt4* p) {
    using namespace zs;
    Q4Args a{};
    int groups;
    if (!int4_attention_args(p, &a, &groups) || a.B == 0 ||
        q4_unit_warps(a))
        return 0;
    return int4_workspace(a);
}

extern "C" int zs_paged_attention_int4(const ZsPagedAttentionInt4* p) {
    using namespace zs;
    Q4Args a{};
    int groups;
    if (!int4_attention_args(p, &a, &groups)) return cudaErrorInvalidValue;
    if (a.B == 0) return cudaSuccess;
    const int max_ctas = q4_max_ctas(a.kp.dim, a.G), W = q4_unit_warps(a);
    if (!W) {
        if (!p->ws || !aligned16p(p->ws) || p->ws_bytes < int4_workspace(a)) return cudaErrorInvalidValue;
        lay_workspace(&a, p->ws, max_ctas);
    }
    cudaStream_t s = (cudaStream_t)p->stream;
    if (p->dtype == ZS_BF16)
        return a.pages ? int4_attention_bf16_listed(a, groups, W, s) : int4_attention_bf16(a, groups, W, s);
    return a.pages ? int4_attention_fp16_listed(a, groups, W, s) : int4_attention_fp16(a, groups, W, s);
}
