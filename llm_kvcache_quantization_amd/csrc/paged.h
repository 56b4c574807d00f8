// Shared parts of the paged cache's kernels (include/kvq_paged.h): element types, page addressing
// and the host's checks of a cache.
#pragma once
#include <hip/hip_runtime.h>

#include <string>

#include "kvq_common.h"
#include "kvq_paged.h"

namespace kvq {

int fail(int code, const std::string& msg);

typedef __bf16 bf16_t;
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float float2v __attribute__((ext_vector_type(2)));
typedef float float16v __attribute__((ext_vector_type(16)));

// 16-bit element types: conversions round to nearest even (two values a v_cvt_pk).
// kUp: where P = exp2(s - m) is rounded to the type, m lies this far below the largest score seen (log2 units; a score
// 6 above that largest moves it).  P in fp16 then has room up to 2^15, and all its bits down to 23 below the largest score,
// which is the sum's own precision.  With m at the largest, tokens 15 bits below it lose bits and those 25 below it are
// lost to the product with V, and many of them are no small part (65536 tokens 25 bits below a first one: 2^-9).  bf16 has
// fp32's range.
struct TF16 {
  using elem = half_t;
  static constexpr uint32_t kInf = 0x7C00;
  static constexpr float kUp = 9.f;
  __device__ __forceinline__ static float to_f(uint16_t b) { return (float)__builtin_bit_cast(half_t, b); }
  __device__ __forceinline__ static uint32_t pack(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((float2v{a, b}), half2v));
  }
  __device__ __forceinline__ static float4v mfma16(u32x4 a, u32x4 b, float4v c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8v, a), __builtin_bit_cast(half8v, b), c, 0, 0, 0);
  }
  __device__ __forceinline__ static float16v mfma32(u32x4 a, u32x4 b, float16v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8v, a), __builtin_bit_cast(half8v, b), c, 0, 0, 0);
  }
};
struct TB16 {
  using elem = bf16_t;
  static constexpr uint32_t kInf = 0x7F80;
  static constexpr float kUp = 0.f;
  __device__ __forceinline__ static float to_f(uint16_t b) { return __builtin_bit_cast(float, (uint32_t)b << 16); }
  __device__ __forceinline__ static uint32_t pack(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((float2v{a, b}), bf16x2));
  }
  __device__ __forceinline__ static float4v mfma16(u32x4 a, u32x4 b, float4v c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
  __device__ __forceinline__ static float16v mfma32(u32x4 a, u32x4 b, float16v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
};

// The cache as the kernels take it: the page size as a shift.
struct PagedCache {
  uint8_t* k;
  uint8_t* v;
  int64_t ksp, ksh, kst, vsp, vsh, vst;  // bytes
  uint8_t* ks;
  uint8_t* vs;
  int64_t kssp, kssh, vssp, vssh;        // bytes
  const int32_t* table;
  int64_t table_stride;
  int32_t num_pages, max_pages, lg, page_mask, kv_heads, batch;
};

// Fills `c` from `p` and checks everything that the kernels' addressing rests on.
inline int paged_cache(const kvq_paged_cache& p, PagedCache& c) {
  if (p.batch < 0 || p.kv_heads <= 0 || p.num_pages < 0 || p.max_pages < 0)
    return fail(KVQ_ERR_INVALID, "paged: negative size");
  if (p.page_size < 16 || p.page_size > 256 || (p.page_size & (p.page_size - 1)))
    return fail(KVQ_ERR_INVALID, "paged: page_size must be 16, 32, 64, 128 or 256");
  if (p.format < KVQ_PAGED_F16 || p.format > KVQ_PAGED_INT8) return fail(KVQ_ERR_INVALID, "paged: unknown format");
  const bool i8 = p.format == KVQ_PAGED_INT8;
  if (p.batch > 0 && p.num_pages > 0 && (!p.k || !p.v || (p.max_pages > 0 && !p.table)))
    return fail(KVQ_ERR_INVALID, "paged: NULL pages or table");
  // token offsets within a page are computed in 32 bits
  const int64_t rows[2] = {p.k_stride_t, p.v_stride_t};
  for (int64_t s : rows)
    if (s < (i8 ? 128 : 256) || s > (1 << 22)) return fail(KVQ_ERR_UNSUPPORTED, "paged: token stride out of range");
  if (((uintptr_t)p.k | (uintptr_t)p.v | (uintptr_t)p.k_stride_p | (uintptr_t)p.k_stride_h | (uintptr_t)p.k_stride_t |
       (uintptr_t)p.v_stride_p | (uintptr_t)p.v_stride_h | (uintptr_t)p.v_stride_t) % 16)
    return fail(KVQ_ERR_INVALID, "paged: pages and their strides must be 16-byte aligned");
  if (i8) {
    if (p.group_size != 32 && p.group_size != 64 && p.group_size != 128)
      return fail(KVQ_ERR_INVALID, "paged: group_size must be 32, 64 or 128");
    if (p.batch > 0 && p.num_pages > 0 && (!p.k_scale || !p.v_scale)) return fail(KVQ_ERR_INVALID, "paged: NULL scales");
    if (((uintptr_t)p.k_scale | (uintptr_t)p.v_scale | (uintptr_t)p.ks_stride_p | (uintptr_t)p.ks_stride_h |
         (uintptr_t)p.vs_stride_p | (uintptr_t)p.vs_stride_h) % 16)
      return fail(KVQ_ERR_INVALID, "paged: scale pages and their strides must be 16-byte aligned");
  }
  if ((int64_t)p.max_pages * p.page_size > (1 << 30)) return fail(KVQ_ERR_UNSUPPORTED, "paged: more than 2^30 token slots a row");
  c = PagedCache{};
  c.k = (uint8_t*)p.k; c.v = (uint8_t*)p.v;
  c.ksp = p.k_stride_p; c.ksh = p.k_stride_h; c.kst = p.k_stride_t;
  c.vsp = p.v_stride_p; c.vsh = p.v_stride_h; c.vst = p.v_stride_t;
  c.ks = (uint8_t*)p.k_scale; c.vs = (uint8_t*)p.v_scale;
  c.kssp = p.ks_stride_p; c.kssh = p.ks_stride_h; c.vssp = p.vs_stride_p; c.vssh = p.vs_stride_h;
  c.table = p.table; c.table_stride = p.table_stride;
  c.num_pages = p.num_pages; c.max_pages = p.max_pages;
  c.lg = __builtin_ctz((unsigned)p.page_size);
  c.page_mask = p.page_size - 1;
  c.kv_heads = p.kv_heads; c.batch = p.batch;
  return KVQ_OK;
}

// Of a cache that is written: its pages and heads have memory of their own.
inline int paged_written(const PagedCache& c) {
  const int64_t pages[4] = {c.ksp, c.vsp, c.kssp, c.vssp}, heads[4] = {c.ksh, c.vsh, c.kssh, c.vssh};
  for (int i = 0; i < (c.ks ? 4 : 2); ++i)
    if ((c.num_pages > 1 && pages[i] == 0) || (c.kv_heads > 1 && heads[i] == 0))
      return fail(KVQ_ERR_INVALID, "paged: pages that are written must have memory of their own, got a stride of 0");
  return KVQ_OK;
}

inline int launched() {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? KVQ_OK : fail(KVQ_ERR_LAUNCH, std::string("launch: ") + hipGetErrorString(e));
}

// No C++ exception leaves a C entry point.
template <class F>
int guarded(F f) noexcept {
  try {
    return f();
  } catch (...) {
    return KVQ_ERR_LAUNCH;
  }
}

}  // namespace kvq
