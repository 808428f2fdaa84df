// Attention over a 4-bit cache, bf16 queries over lists of pages (paged_int4_attention.cuh).
#include "paged_int4_attention.cuh"

namespace zs {

cudaError_t int4_attention_bf16_listed(const Q4Args& a, int groups, int W, cudaStream_t s) {
    return launch_int4<__nv_bfloat16, true>(a, groups, W, s);
}

}  // namespace zs
