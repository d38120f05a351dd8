// long_context.h -- what the operators for long contexts share: element types, checks of tensors and of a paged cache.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "aig_common.cuh"

inline bool dtype_known(int dtype) { return dtype == AIG_F16 || dtype == AIG_BF16; }
inline bool aligned_to(const void* p, size_t bytes) { return ((uintptr_t)p & (bytes - 1)) == 0; }

// 16-byte accesses to rows of head_dim elements of two bytes
inline bool heads_vectorised(const aig_heads& t) {
  return aligned_to(t.data, 16) && t.token_stride % 8 == 0 && t.head_stride % 8 == 0;
}
inline bool heads_sane(const aig_heads* t) { return t && t->data && t->heads > 0 && t->token_stride >= 0 && t->head_stride >= 0 && aligned_to(t->data, 2); }

inline int check_cache(aig_ctx* ctx, const aig_kv_cache* c, const char* who) {
  AIG_REQUIRE(ctx, c && c->k && c->v, "%s: null cache", who);
  AIG_REQUIRE(ctx, dtype_known(c->dtype), "%s: unknown element type %d", who, c->dtype);
  AIG_REQUIRE(ctx, c->kv_heads > 0 && c->page_size > 0 && c->num_pages > 0 && c->head_dim > 0, "%s: bad cache extents", who);
  AIG_REQUIRE(ctx, c->head_dim % 8 == 0 && c->page_stride % 8 == 0 && c->token_stride % 8 == 0 && c->head_stride % 8 == 0 &&
                       c->page_stride >= 0 && c->token_stride >= 0 && c->head_stride >= 0 && aligned_to(c->k, 16) && aligned_to(c->v, 16),
              "%s: a cache's head_dim and strides are multiples of 8, its data on 16-byte boundaries", who);
  return AIG_OK;
}

// Division of numbers below 2^31 by a constant of the launch: one multiplication
struct Divisor {
  uint32_t magic, shift, by;
  static Divisor of(uint32_t d) {
    uint32_t l = 1;
    while (l < 31 && (1u << l) < d) ++l;
    return Divisor{d == 1 ? 0u : (uint32_t)(((uint64_t)1 << (31 + l)) / d + 1), l - 1, d};
  }
#ifdef __CUDACC__
  __device__ __forceinline__ uint32_t divide(uint32_t n) const { return magic == 0 ? n : __umulhi(n, magic) >> shift; }
#endif
};

#ifdef __CUDACC__
template <class T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// two values as one register, the first in the low half
template <class T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <class T>
__device__ __forceinline__ float2 unpack2(uint32_t v);
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t v) { return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v)); }

// 2^x on the special-function unit (relative error 2^-22; -inf gives 0)
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void note_error(int* gerr, int code) { atomicCAS(gerr, 0, code); }
#endif
