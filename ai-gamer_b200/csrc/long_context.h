// long_context.h -- what the operators for long contexts share: element types, checks of tensors and of a paged cache.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include <type_traits>

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

// ---- warp-level matrices and asynchronous copies
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int bytes) {
  // (bytes = 0: the destination is filled with zeros, nothing is read)
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
template <class T>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// a pair of weights as the sum of two pairs of 16-bit values
template <class T>
__device__ __forceinline__ void split2(float x, float y, uint32_t& hi, uint32_t& lo) {
  hi = pack2<T>(x, y);
  const float2 h = unpack2<T>(hi);
  lo = pack2<T>(x - h.x, y - h.y);
}

// 2^x on the special-function unit (relative error 2^-22; -inf gives 0)
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void note_error(int* gerr, int code) { atomicCAS(gerr, 0, code); }
#endif
