// Shared pieces of the uncompressed paged-cache operators (step plan, rotary
// write, paged attention, page bounds and page choice).
//
// One layout throughout: a pool holds num_blocks pages of `page` tokens (a power
// of two, 16..256) of every KV head; element (block, token, head, d) sits at
// block * s_block + token * s_token + head * s_head + d, so pools with the heads
// or the tokens outermost inside a page are the same type. Offsets are 64-bit
// element counts.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "common.cuh"
#include "zipserv_b200.h"

namespace zs {

constexpr unsigned kErrPagedIndex = kErrStreamOverflow;   // an index was out of range; the access was skipped
constexpr unsigned kErrPagedFull = 4u;                    // a request was refused (pages, tokens or table width)

struct PoolView {
    void* data;
    long long s_block, s_token, s_head;   // elements
    int num_blocks, page_shift, heads, dim;
};

inline bool aligned16p(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Host: checks a pool description; false when a kernel could not use it.
inline bool make_pool(const ZsPagePool* p, PoolView* v) {
    if (!p || !p->data || p->num_blocks <= 0 || p->num_heads <= 0 || p->head_dim <= 0) return false;
    if (p->page_size < 16 || p->page_size > 256 || (p->page_size & (p->page_size - 1))) return false;
    if ((p->stride_block | p->stride_token | p->stride_head) % 8) return false;
    if (p->stride_block < 0 || p->stride_token < 0 || p->stride_head < 0) return false;
    if (reinterpret_cast<uintptr_t>(p->data) & 15u) return false;
    if (p->dtype != ZS_BF16 && p->dtype != ZS_FP16) return false;
    v->data = p->data;
    v->s_block = p->stride_block;
    v->s_token = p->stride_token;
    v->s_head = p->stride_head;
    v->num_blocks = p->num_blocks;
    v->heads = p->num_heads;
    v->dim = p->head_dim;
    v->page_shift = 0;
    while ((1 << v->page_shift) < p->page_size) ++v->page_shift;
    return true;
}

// K and V pools of one cache.
inline bool same_pools(const ZsPagePool& k, const ZsPagePool& v) {
    return k.num_blocks == v.num_blocks && k.page_size == v.page_size && k.num_heads == v.num_heads &&
           k.head_dim == v.head_dim && k.dtype == v.dtype;
}

// Launch attributes: a kernel that may start while its predecessor on the
// stream drains (it waits with grid_dep_wait before touching memory).
inline void pdl_config(cudaLaunchConfig_t* c, cudaLaunchAttribute* a, dim3 grid, dim3 block, size_t smem,
                       cudaStream_t s) {
    *c = cudaLaunchConfig_t{};
    c->gridDim = grid;
    c->blockDim = block;
    c->dynamicSmemBytes = smem;
    c->stream = s;
    a->id = cudaLaunchAttributeProgrammaticStreamSerialization;
    a->val.programmaticStreamSerializationAllowed = 1;
    c->attrs = a;
    c->numAttrs = 1;
}

// 16-bit float types as the kernels use them.
template <typename T>
struct Half2Of;
template <>
struct Half2Of<__nv_bfloat16> {
    using type = __nv_bfloat162;
};
template <>
struct Half2Of<__half> {
    using type = __half2;
};

__device__ __forceinline__ float2 to_f2(__nv_bfloat162 v) { return __bfloat1622float2(v); }
__device__ __forceinline__ float2 to_f2(__half2 v) { return __half22float2(v); }
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);   // round to nearest, a in the low half
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
}
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t v) {
    return to_f2(*reinterpret_cast<const typename Half2Of<T>::type*>(&v));
}

__device__ __forceinline__ uint4 ld_nc16(const void* p) { return __ldg(reinterpret_cast<const uint4*>(p)); }

// read once: no place in L1
__device__ __forceinline__ uint4 ld_stream16(const void* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(p));
    return v;
}

__device__ __forceinline__ void set_err(unsigned* err, unsigned bit) {
    if (err) atomicOr(err, bit);
}

}  // namespace zs
