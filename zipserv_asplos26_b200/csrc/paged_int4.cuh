// The 4-bit paged KV cache: its format, shared by the quantising write, the read back
// and the attention over it.
//
// A row (a token's keys or values of one KV head, D channels) is held in groups of 32
// or 64 channels: a 4-bit code u per channel, channel 2i in the low half of byte i, and
// per group a bf16 scale s and a bf16 centre c. A channel stands for c + s (u - 8), and
//   s = bf16((max - min) / 15), c = bf16(min + 8 s), u = clamp(rint((x - c) / s) + 8, 0, 15),
// in fp32. What is lost: half a step s / 2, and at the group's ends up to 15 / 256 s +
// |c| / 256 for the roundings of s and c to bf16, which 5 bits a value (fp32 parameters:
// 6) pays for. The codes are centred, so that sums over many tokens stay small on the
// way. A group whose scale is below the smallest normal number has s = 0, c = bf16(min)
// and codes of 8; one with a value that is not finite, or whose range is not, c = NaN,
// and reads back as NaN.
//
// Codes are bytes [block][token][head][D / 2], parameters bf16 [block][token][head][2]
// [D / group] (scales, then centres), rows contiguous, the other strides free.
#pragma once

#include "paged.cuh"

namespace zs {

constexpr float kSmallestScale = 1.17549435e-38f;      // 2^-126

struct Int4View {
    uint8_t* codes;
    uint16_t* params;
    long long c_block, c_token, c_head;   // bytes
    long long p_block, p_token, p_head;   // bf16 elements
    int num_blocks, page_shift, heads, dim, groups;   // groups a row
};

// Host: checks a pool description; false when a kernel could not use it.
inline bool make_int4_pool(const ZsInt4Pool* p, Int4View* v) {
    if (!p || !p->codes || !p->params || p->num_blocks <= 0 || p->num_heads <= 0) return false;
    if ((p->head_dim != 64 && p->head_dim != 128) || (p->group != 32 && p->group != 64)) return false;
    if (p->page_size < 16 || p->page_size > 256 || (p->page_size & (p->page_size - 1))) return false;
    if (p->codes_block < 0 || p->codes_token < 0 || p->codes_head < 0 || p->params_block < 0 || p->params_token < 0 ||
        p->params_head < 0)
        return false;
    v->groups = p->head_dim / p->group;
    if ((p->codes_block | p->codes_token | p->codes_head) % 16) return false;
    if ((p->params_block | p->params_token | p->params_head) % (2 * v->groups)) return false;
    if (!aligned16p(p->codes) || reinterpret_cast<uintptr_t>(p->params) % (4 * v->groups)) return false;
    v->codes = p->codes;
    v->params = p->params;
    v->c_block = p->codes_block;
    v->c_token = p->codes_token;
    v->c_head = p->codes_head;
    v->p_block = p->params_block;
    v->p_token = p->params_token;
    v->p_head = p->params_head;
    v->num_blocks = p->num_blocks;
    v->heads = p->num_heads;
    v->dim = p->head_dim;
    v->page_shift = 0;
    while ((1 << v->page_shift) < p->page_size) ++v->page_shift;
    return true;
}

// K and V pools of one cache.
inline bool same_int4_pools(const ZsInt4Pool& k, const ZsInt4Pool& v) {
    return k.num_blocks == v.num_blocks && k.page_size == v.page_size && k.num_heads == v.num_heads &&
           k.head_dim == v.head_dim && k.group == v.group;
}

__device__ __forceinline__ float bf16_bits_to_float(uint32_t x) { return __uint_as_float(x << 16); }

}  // namespace zs
