// Attention over a 4-bit cache, bf16 queries over whole sequences (paged_int4_attention.cuh).
#include "paged_int4_attention.cuh"

namespace zs {

cudaError_t int4_attention_bf16(const Q4Args& a, int groups, int W, cudaStream_t s) {
    return launch_int4<__nv_bfloat16, false>(a, groups, W, s);
}

}  // namespace zs
