// Tiles of 64 keys in LDS and what a wave of 32 queries does with them: S^T = K Q^T and O^T = V^T P^T in 32x32x16
// matrix instructions, softmax with a running maximum (used by the attention of prompts and of shared prefixes).
//
// Lane (q, hh) = (lane % 32, lane / 32) of a 32 x 32 result holds rows 8 (i / 4) + 4 hh + i % 4 of column q, i < 16.  The 8
// reduction slots that P^T's operand takes from it are keys 16 mm + {4 hh + r, 8 + 4 hh + r}, r < 4; V^T's operand has the
// same keys from two transposing LDS reads of 4 keys each.
#pragma once
#include "paged.h"

namespace kvq {
namespace {

constexpr int kBN = 64;       // keys a tile

__device__ __forceinline__ float xor32(float x) { return __shfl_xor(x, 32, 64); }

// A tile in LDS.  K: [key][16 chunks of 8 channels], chunk ^ (key % 16); V: the same, chunk ^ 4 (key % 4).
typedef u32x4 LdsTile[kBN * 16];

typedef __attribute__((address_space(3))) uint8_t lds_u8;
typedef __attribute__((address_space(3))) u32x4 lds_u32x4;
typedef const __attribute__((address_space(1))) void* gptr;
typedef short s16x4 __attribute__((ext_vector_type(4)));

template <class T>
struct AttnTile {
  float16v acc[4];
  float m, l;

  // K's operands of keys 32 u .. of the tile.
  static __device__ __forceinline__ void read_k(const LdsTile& ks, int u, u32x4 (&kf)[8]) {
    const int lane = threadIdx.x & 63, ql = lane & 31, hh = lane >> 5;
#pragma unroll
    for (int kk = 0; kk < 8; ++kk) kf[kk] = ks[(32 * u + ql) * 16 + ((2 * kk + hh) ^ (ql & 15))];
  }

  // V^T's operands of keys 32 u + 16 mm .., channels 32 ct .., in vf[4 mm + ct].  16 lanes of a transposing read
  // take 4 keys of 16 channels: lane i brings 4 channels of key i / 4.
  static __device__ __forceinline__ void read_v(const LdsTile& vs, int u, u32x4 (&vf)[8]) {
    const int lane = threadIdx.x & 63, hh = lane >> 5, i = lane & 15;
    const lds_u8* const vt = (const lds_u8*)&vs[0];
    const int vrow = 32 * u + 4 * hh + (i >> 2);
    const int vcol = 32 * ((lane >> 4) & 1) + 8 * (i & 3);  // bytes from the 32 channels' first
#pragma unroll
    for (int mm = 0; mm < 2; ++mm)
#pragma unroll
      for (int ct = 0; ct < 4; ++ct)
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          const int row = 16 * mm + 8 * w + vrow;  // row % 4 = i / 4
          const int at = row * 256 + ((64 * ct + vcol) ^ ((i >> 2) << 6));
          const u32x2 x = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(vt + at)));
          vf[4 * mm + ct][2 * w] = x[0];
          vf[4 * mm + ct][2 * w + 1] = x[1];
        }
  }

  static __device__ __forceinline__ float16v scores(const u32x4 (&kf)[8], const u32x4 (&q)[8]) {
    float16v sc;
#pragma unroll
    for (int j = 0; j < 16; ++j) sc[j] = 0.f;
#pragma unroll
    for (int kk = 0; kk < 8; ++kk) sc = T::mfma32(kf[kk], q[kk], sc);
    return sc;
  }

  // P of 32 keys from the scores times mul; returns this lane's sum of it.  P is rounded to 16 bits for the product with V,
  // as the matrix instructions take it (kUp keeps faint ones); the sum is of the unrounded.
  __device__ __forceinline__ float exps(const float16v& sc, float mul, u32x4 (&pb)[2]) const {
    const float mm = -(m == kNegInf ? 0.f : m);
    float s0 = 0.f, s1 = 0.f;
#pragma unroll
    for (int j = 0; j < 16; j += 2) {
      const float e0 = fast_exp2(fmaf(sc[j], mul, mm)), e1 = fast_exp2(fmaf(sc[j + 1], mul, mm));
      s0 += e0;
      s1 += e1;
      pb[j >> 3][(j >> 1) & 3] = T::pack(e0, e1);
    }
    return s0 + s1;
  }

  // While a lane's sum stays below 64 (2^15 in fp16) so does each of its P: the maximum, kUp below the largest score,
  // follows only where it does not.
  __device__ __forceinline__ void add_sum(float sum, const float16v& sc, float mul, u32x4 (&pb)[2]) {
    if (__any(!(sum <= 64.f * (1 << (int)T::kUp)) || m == kNegInf)) {
      float mx = kNegInf;
#pragma unroll
      for (int j = 0; j < 16; ++j) mx = fmaxf(mx, sc[j] * mul);
      mx = fmaxf(fmaxf(mx, xor32(mx)) - T::kUp, m);
      const float f = fast_exp2(m - (mx == kNegInf ? 0.f : mx));
      l *= f;
#pragma unroll
      for (int ct = 0; ct < 4; ++ct) acc[ct] *= f;
      m = mx;
      sum = exps(sc, mul, pb);
    }
    l += sum;
  }

  __device__ __forceinline__ void add_values(const u32x4 (&vf)[8], const u32x4 (&pb)[2]) {
#pragma unroll
    for (int mm = 0; mm < 2; ++mm)
#pragma unroll
      for (int ct = 0; ct < 4; ++ct) acc[ct] = T::mfma32(vf[4 * mm + ct], pb[mm], acc[ct]);
  }
};

}  // namespace
}  // namespace kvq
