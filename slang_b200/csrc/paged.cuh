// Shared pieces of the paged-cache operators: the two 16-bit element types as
// one template parameter, 16-byte vectors of them, and the cache descriptor's
// host-side checks.
#pragma once

#include <cuda_bf16.h>

#include <type_traits>

#include "common.cuh"

namespace sbp {

// 16-bit pair <-> two f32 (round to nearest even), element i in the low half.
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t w);
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t w) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Softmax weights p = 2^(s - m) rounded to T for the second product are held 2^kLift times as large, as are their sums.
// m lies at most kRise below the largest score, so p < 2^8 and f16 has 2^7 to spare: its smallest weights are
// 2^-31 of the one at m in place of 2^-24, which thousands of them beside one that dominates (an attention sink) would
// lose.  bf16 has the range of f32.
constexpr float kRise = 8.f;
template <typename T>
constexpr float kLift = std::is_same<T, __half>::value ? 7.f : 0.f;

// Eight values at p + 8 * i as f32 (16-byte aligned; two vectors for f32).
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
  const uint4 r = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = unpack2<T>(w[i]);
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
template <>
__device__ __forceinline__ void load8<float>(const float* p, float (&v)[8]) {
  const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
  v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
  v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
  *reinterpret_cast<uint4*>(p) = make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]),
                                            pack2<T>(v[6], v[7]));
}

// The cache as the kernels see it.
struct Pages {
  const void* k;
  const void* v;
  int64_t page_stride, head_stride, token_stride;  // elements
  const int32_t* table;                            // [n_seqs][max_pages]
  int max_pages, n_pages, shift;                   // shift = log2(page_size)
};

inline int log2_of(int x) {
  int s = 0;
  while ((1 << s) < x) ++s;
  return s;
}

// Checks a cache descriptor and its page table for entry point `who`.
inline int check_pages(const char* who, const sb_paged_kv* kv, const int32_t* table, int max_pages, Pages* out) {
  SB_CHECK_ARG(kv, "%s: null cache descriptor", who);
  SB_CHECK_ARG(kv->dtype == SB_F16 || kv->dtype == SB_BF16, "%s: the cache is f16 or bf16", who);
  SB_CHECK_ARG(kv->head_dim == 64 || kv->head_dim == 128 || kv->head_dim == 256 || kv->head_dim == 512,
               "%s: head_dim %d not in {64, 128, 256, 512}", who, kv->head_dim);
  SB_CHECK_ARG(kv->page_size >= 1 && kv->page_size <= (1 << 20) && (kv->page_size & (kv->page_size - 1)) == 0,
               "%s: page_size %d is not a power of two", who, kv->page_size);
  SB_CHECK_ARG(kv->n_kv_heads >= 1 && kv->n_pages >= 0 && max_pages >= 0, "%s: bad cache shape", who);
  SB_CHECK_ARG(static_cast<int64_t>(max_pages) * kv->page_size < (1ll << 31), "%s: a sequence's pages hold 2^31 keys", who);
  SB_CHECK_ARG(kv->n_pages == 0 || (kv->k && kv->v), "%s: null cache pointer", who);
  SB_CHECK_ARG(max_pages == 0 || table, "%s: null page table", who);
  if (!sb::aligned(kv->k, 16) || !sb::aligned(kv->v, 16) || kv->page_stride % 8 || kv->head_stride % 8 ||
      kv->token_stride % 8)
    return sb::fail(SB_ERR_ALIGN, "%s: cache rows must start on 16-byte boundaries", who);
  *out = Pages{kv->k, kv->v, kv->page_stride, kv->head_stride, kv->token_stride, table, max_pages, kv->n_pages,
               log2_of(kv->page_size)};
  return SB_OK;
}

}  // namespace sbp
