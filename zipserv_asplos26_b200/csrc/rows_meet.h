// Host check of overlapping buffers, shared by the C ABI and the Python binding.
#pragma once
#include <stdint.h>

namespace zs {

// Whether any of the rows base + t * tok + h * head (t < n, h < heads), `dim`
// elements each, shares an element with the `len` elements from `at` on. 16-bit
// elements; strides may be 0 or negative.
inline bool rows_meet(const void* base, int64_t n, int64_t heads, int64_t dim, int64_t tok, int64_t head,
                      const void* at, int64_t len) {
    if (n <= 0 || heads <= 0 || dim <= 0 || len <= 0) return false;
    const int64_t d = (static_cast<int64_t>(reinterpret_cast<intptr_t>(at)) -
                       static_cast<int64_t>(reinterpret_cast<intptr_t>(base))) / 2;
    // a row meets where it starts in [d - dim + 1, d + len - 1]; first by the outermost rows
    const int64_t t_end = (n - 1) * tok, h_end = (heads - 1) * head;
    const int64_t low = (t_end < 0 ? t_end : 0) + (h_end < 0 ? h_end : 0);
    const int64_t high = (t_end > 0 ? t_end : 0) + (h_end > 0 ? h_end : 0);
    if (high < d - dim + 1 || low > d + len - 1) return false;
    const int64_t step = tok < 0 ? -tok : tok;
    for (int64_t h = 0; h < heads; ++h) {
        int64_t from = d - dim + 1 - h * head, to = d + len - 1 - h * head;      // of t * tok
        if (tok < 0) {
            const int64_t x = from;
            from = -to;
            to = -x;
        }
        if (to < 0) continue;
        if (step == 0) {
            if (from <= 0) return true;
            continue;
        }
        const int64_t first = from <= 0 ? 0 : (from + step - 1) / step;
        if (first < n && first * step <= to) return true;
    }
    return false;
}

// Whether a rotary write may put its q, contiguous [n][hq][dim], at q_out: on q itself
// where that is as contiguous, else apart from q, k and v (other warps may still read
// them).
inline bool q_out_is_apart(const void* q_out, int64_t n, int64_t hq, int64_t hkv, int64_t dim, const void* q,
                           int64_t q_tok, int64_t q_head, const void* k, int64_t k_tok, int64_t k_head, const void* v,
                           int64_t v_tok, int64_t v_head) {
    const int64_t len = n * hq * dim;
    const bool on_q = q_out == q && (n == 1 || q_tok == hq * dim) && (hq == 1 || q_head == dim);
    return (on_q || !rows_meet(q, n, hq, dim, q_tok, q_head, q_out, len)) &&
           !rows_meet(k, n, hkv, dim, k_tok, k_head, q_out, len) &&
           !rows_meet(v, n, hkv, dim, v_tok, v_head, q_out, len);
}

}  // namespace zs
