// Attention of a prompt, or of a chunk of one, causal, through a sliding window with a few first tokens
// that stay visible (kvq_prefill_attn).
//
//   out_i = sum_j p_ij v_j,  p_i = softmax over the visible j of sm_scale inv_tau_h q_i.k_j
//
// A work-group of four waves takes 128 queries of one head, a wave 32 of them, and goes through the tiles
// of 64 keys that any of them sees: first those of the sinks, then from the window's first key to the last
// query's own.  S^T = K Q^T and O^T = V^T P^T with 32x32x16 matrix instructions: a lane holds one query
// (its column) of both, so the softmax is lane-local but for one exchange between the half-waves, made
// only where the maximum moves, and P^T's operand is the lane's own scores, rounded to 16 bits.
//
// Lane (q, hh) = (lane % 32, lane / 32) of a 32 x 32 result holds rows 8 (i / 4) + 4 hh + i % 4 of column
// q, i < 16.  The 8 reduction slots that P^T's operand takes from it are keys 16 mm + {4 hh + r, 8 + 4 hh +
// r}, r < 4; V^T's operand has the same keys from two transposing LDS reads of 4 keys each.
//
// K and V tiles go straight from memory into LDS, two buffers each, the next tile's loads under the present
// one's products.  Rows are XOR-swizzled in 16-byte chunks (by the lanes' choice of what they load), so that
// the operands' reads spread over all banks.
//
// What is masked may hold anything.  In the place of keys at or past kv_lens the last key is loaded.  An Inf or
// NaN in a V row that some query of a tile sees and another does not would reach both (0 x NaN): where a
// work-group's result is not finite it runs again with such rows taken out of the products and added query by
// query.
//
// What bounds it: the matrix units (busy for 42% of the CUs' busy cycles) and the vector units (43%, half of it
// exponentials), in turn in each wave.  Measured, us a call: 16384 tokens through a window of 4096, 28 heads, bf16, 958 (879
// TFLOP/s; 912 to 1005 from card to card); 8192 tokens without a window 510 (943 TFLOP/s); a tile of 64 keys takes 1.75 us
// on a CU of its own, 2.3 where two share one.
#include "paged.h"

namespace kvq {
namespace {

constexpr int kBM = 128;      // queries a work-group
constexpr int kBN = 64;       // keys a tile
constexpr int kThreads = 256;

struct PreArgs {
  const uint8_t* q;
  const uint8_t* k;
  const uint8_t* v;
  uint8_t* out;
  int64_t qsb, qsh, qss, ksb, ksh, kss, vsb, vsh, vss, osb, osh, oss;  // bytes
  const int32_t* q_lens;
  const int32_t* kv_lens;
  const float* inv_tau;
  float sm;  // sm_scale * log2(e)
  int32_t batch, q_heads, rep, S, T, window, sinks;
  int32_t blocks;   // of queries, a (row, head)
  int32_t splits;   // of a block's keys
  int64_t units;    // batch * q_heads * blocks * splits
  float* part;      // [units][128][128] accumulators, where splits > 1
  float2* ml;       // [units][128]
};

// The key tiles of queries at positions [p0, p1]: n_sink tiles from key 0, then those from `first` on.
struct KeyTiles {
  int n_sink, first, count;
  __device__ __forceinline__ KeyTiles(int p0, int p1, int window, int sinks) {
    n_sink = first = count = 0;
    if (p1 < 0) return;
    const int end = p1 / kBN + 1;
    const int64_t lo = (int64_t)p0 - window + 1;  // no query sees a key before it but the sinks
    if (window > 0 && lo > 0) {
      n_sink = (int)(((int64_t)min(max(sinks, 0), p1 + 1) + kBN - 1) / kBN);
      first = max((int)(lo / kBN), n_sink);
    }
    count = n_sink + max(end - first, 0);
  }
  __device__ __forceinline__ int key(int i) const { return (i < n_sink ? i : first + i - n_sink) * kBN; }
};

struct Row {
  int b, h, block, split, q_len, kv_len, off, i0;
};

__device__ __forceinline__ Row unit_of(const PreArgs& a, int64_t unit64) {
  Row r;
  uint32_t unit = (uint32_t)unit64;  // fewer than 2^31 of them
  r.split = (int)(unit % (uint32_t)a.splits);
  unit /= (uint32_t)a.splits;
  // blocks from both ends in turn: a part of them has its share of the long ones (the later queries') and the short
  // ones; rows of a batch in turn for the same reason
  const int x = (int)(unit % (uint32_t)a.blocks);
  r.block = x & 1 ? x >> 1 : a.blocks - 1 - (x >> 1);
  unit /= (uint32_t)a.blocks;
  r.b = (int)(unit % (uint32_t)a.batch);
  r.h = (int)(unit / (uint32_t)a.batch);
  r.q_len = a.q_lens ? min(max(a.q_lens[r.b], 0), a.S) : a.S;
  r.kv_len = a.kv_lens ? min(max(a.kv_lens[r.b], 0), a.T) : a.T;
  r.off = r.kv_len - r.q_len;
  r.i0 = r.block * kBM;
  return r;
}

// The unit of a work-group, -1: none.  Work-groups go round the 8 XCDs; each XCD has a run of `per` units, whose heads
// share K and V in its L2.  It takes them by the place of their queries, the last and longest first, so that short
// ones are left for the end.  An XCD's work-groups go round its shader engines in turn, whatever those have left to
// do: the (row, head)s shift by one from place to place, or long and short rows would each have engines of their own.
// us, a (row, head) at a time / without the shift / so, all three before padded queries and halves of tiles were left out:
// 4 padded prompts of up to 2047 tokens, 40 heads, window 1024 168 / 209 / 149 (116 since); 8192 tokens, 28 heads, no
// window 717 / - / 516; 4 x 32 heads of 4096 tokens with K and V of their own 780 / - / 680.
__device__ __forceinline__ int64_t unit_at(const PreArgs& a, uint32_t at) {
  const uint32_t xcd = at & 7, k = at >> 3, depth = (uint32_t)a.blocks * (uint32_t)a.splits;
  const uint32_t per = (uint32_t)((a.units + 7) / 8), start = xcd * per, columns = (per + depth - 1) / depth;
  const uint32_t d = k / columns, column = (k + d) % columns;
  // the place of block (blocks - 1 - d / splits) in its (row, head), and that place's distance from the run's first
  const uint32_t x = d / (uint32_t)a.splits, y = 2 * x < (uint32_t)a.blocks ? 2 * x : 2 * ((uint32_t)a.blocks - 1 - x) + 1;
  const uint32_t z = y * (uint32_t)a.splits + d % (uint32_t)a.splits, z0 = start % depth;
  const uint32_t u = column * depth + (z >= z0 ? z - z0 : z + depth - z0);
  return u < per && start + u < (uint32_t)a.units ? (int64_t)(start + u) : -1;
}

__device__ __forceinline__ bool sees(int p, int key, int window, int sinks) {
  return key <= p && (window <= 0 || key > p - window || key < sinks);
}
__device__ __forceinline__ float xor32(float x) { return __shfl_xor(x, 32, 64); }
// A tile in LDS.  K: [key][16 chunks of 8 channels], chunk ^ (key % 16); V: the same, chunk ^ 4 (key % 4).
typedef u32x4 LdsTile[kBN * 16];
// The buffers are variables of their own, and the loop is written out for both: only so does the compiler know
// that the operands' reads of one need not wait for the loads into the other.
struct Lds {
  LdsTile &k0, &v0, &k1, &v1;
  uint32_t (&bad)[2];  // keys of the tile whose V row is not finite
};

typedef __attribute__((address_space(3))) uint8_t lds_u8;
typedef __attribute__((address_space(3))) u32x4 lds_u32x4;
typedef const __attribute__((address_space(1))) void* gptr;
typedef short s16x4 __attribute__((ext_vector_type(4)));

// One side's tiles of rows key0 .. key0 + 63 into LDS.  A wave instruction loads four rows; a lane takes the
// chunk that belongs at its place, 16 bytes from those of its neighbours.
template <bool V>
struct TileLoad {
  const uint8_t* x;
  int64_t stride;
  uint32_t off;    // this lane's place in the tile's first 16 rows
  int row, kv_len;
  __device__ __forceinline__ TileLoad(const uint8_t* x_, int64_t stride_, int kv_len_) : x(x_), stride(stride_), kv_len(kv_len_) {
    const int lane = threadIdx.x & 63;
    row = 4 * (threadIdx.x >> 6) + (lane >> 4);
    off = (uint32_t)row * (uint32_t)stride + ((lane & 15) ^ (V ? (row & 3) << 2 : row & 15)) * 16;
  }
  __device__ __forceinline__ void operator()(int key0, u32x4* to) const {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint8_t* base = x + key0 * stride;
    if (key0 + kBN <= kv_len) {
#pragma unroll
      for (int u = 0; u < 4; ++u)
        __builtin_amdgcn_global_load_lds((gptr)(base + 16 * u * stride + off),
                                         (__attribute__((address_space(3))) void*)(to + (16 * u + 4 * wave) * 16), 16, 0, 0);
    } else {  // the last tile: its last key in the place of those behind
      for (int u = 0; u < 4; ++u) {
        const int over = max(key0 + 16 * u + row - (kv_len - 1), 0);
        __builtin_amdgcn_global_load_lds((gptr)(base + 16 * u * stride + off - over * stride),
                                         (__attribute__((address_space(3))) void*)(to + (16 * u + 4 * wave) * 16), 16, 0, 0);
      }
    }
  }
};

template <class T>
struct Prefill {
  float16v acc[4];
  float m, l;
  bool seen;

  // V of the second run: rows with an Inf or NaN as zeros, their keys marked
  static __device__ __forceinline__ void load_v_finite(const uint8_t* x, int64_t stride, int key0, int kv_len, const Lds& s) {
    const int t = threadIdx.x;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int row = (t >> 4) + 16 * u;
      u32x4 w = *(const u32x4*)(x + min(key0 + row, kv_len - 1) * stride + (t & 15) * 16);
      bool odd = false;
#pragma unroll
      for (int d = 0; d < 4; ++d)
        odd |= !(fabsf(T::to_f((uint16_t)w[d])) < __builtin_inff()) || !(fabsf(T::to_f((uint16_t)(w[d] >> 16))) < __builtin_inff());
      const uint64_t any = __ballot(odd);  // a row is 16 lanes
      if ((any >> (t & 48)) & 0xFFFF) {
        w = u32x4{0, 0, 0, 0};
        if ((t & 15) == 0) atomicOr(&s.bad[row >> 5], 1u << (row & 31));
      }
      s.v0[row * 16 + ((t & 15) ^ ((row & 3) << 2))] = w;
    }
  }

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

  // Scaled scores with -inf where this lane's query does not see the key.
  __device__ __forceinline__ void mask(float16v& sc, const PreArgs& a, float scale, int key0, int u, int p) {
    // key = first + c, c < 32 a constant: c against this lane's last key, first key and end of the sinks
    const int first = key0 + 32 * u + 4 * ((threadIdx.x & 63) >> 5);
    const int last = p - first, from = a.window > 0 ? p - a.window - first : -1, sink = a.sinks - first;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const int c = 8 * (j >> 2) + (j & 3);
      const bool vis = (c <= last) & ((c > from) | (c < sink));
      seen |= vis;
      sc[j] = vis ? sc[j] * scale : kNegInf;
    }
  }

  // P of 32 keys, in 16 bits, from the scores times mul; returns this lane's sum of it.
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

  // A tile's products, 32 keys at a time.  Operands are read from LDS a step before they are used: V's under
  // the exponentials, the second half's K under the first half's product with V (the scheduling barriers keep
  // the compiler from moving the reads to their uses).
  __device__ __forceinline__ void tile(const LdsTile& ks, const LdsTile& vs, const PreArgs& a, const u32x4 (&q)[8], float scale,
                                       int key0, int p, int pw0, int pw1) {
    u32x4 kf[8], vf[8], pb[2];
    read_k(ks, 0, kf);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      // the wave's queries see none of these 32 keys, or all of them, or some
      const int kb = key0 + 32 * u;
      if (pw1 < kb || (a.window > 0 && kb + 31 <= pw0 - a.window && kb >= a.sinks)) {
        if (u == 0) read_k(ks, 1, kf);
        continue;
      }
      const bool full = kb + 31 <= pw0 && (a.window <= 0 || kb > pw1 - a.window || kb + 32 <= a.sinks);
      const float mul = full ? scale : 1.f;
      seen |= full;
      float16v sc = scores(kf, q);
      read_v(vs, u, vf);
      __builtin_amdgcn_sched_barrier(0);
      if (!full) mask(sc, a, scale, key0, u, p);
      add_sum(exps(sc, mul, pb), sc, mul, pb);
      if (u == 0) read_k(ks, 1, kf);
      __builtin_amdgcn_sched_barrier(0);
      add_values(vf, pb);
    }
  }

  // The V rows taken out of the products: every lane scores its own query against the key again, and adds the
  // row if it sees it.
  __device__ __forceinline__ void add_bad(const Lds& s, const PreArgs& a, const uint8_t* k, const uint8_t* v, const u32x4 (&q)[8],
                                          float scale, int key0, int p, int kv_len) {
    const int hh = (threadIdx.x & 63) >> 5;
    for (int w = 0; w < 2; ++w)
      for (uint32_t left = s.bad[w]; left; left &= left - 1) {
        const int key = key0 + 32 * w + __builtin_ctz(left);
        if (key >= kv_len) break;
        const uint8_t* kr = k + key * a.kss;
        float d = 0.f;
#pragma unroll
        for (int kk = 0; kk < 8; ++kk) {
          const u32x4 x = *(const u32x4*)(kr + (16 * kk + 8 * hh) * 2);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            d = fmaf(T::to_f((uint16_t)q[kk][e]), T::to_f((uint16_t)x[e]), d);
            d = fmaf(T::to_f((uint16_t)(q[kk][e] >> 16)), T::to_f((uint16_t)(x[e] >> 16)), d);
          }
        }
        d += xor32(d);
        if (sees(p, key, a.window, a.sinks)) {
          const float e = fast_exp2(fmaf(d, scale, -(m == kNegInf ? 0.f : m)));
#pragma unroll
          for (int ct = 0; ct < 4; ++ct)
#pragma unroll
            for (int j = 0; j < 16; j += 4) {
              const u32x2 x = *(const u32x2*)(v + key * a.vss + (32 * ct + 2 * j + 4 * hh) * 2);
              acc[ct][j] += e * T::to_f((uint16_t)x[0]);
              acc[ct][j + 1] += e * T::to_f((uint16_t)(x[0] >> 16));
              acc[ct][j + 2] += e * T::to_f((uint16_t)x[1]);
              acc[ct][j + 3] += e * T::to_f((uint16_t)(x[1] >> 16));
            }
        }
      }
  }

  template <bool ROBUST>
  __device__ __forceinline__ void attend(const Lds& s, const PreArgs& a, const Row& r, const u32x4 (&q)[8], float scale,
                                         const KeyTiles& kt, int t0, int t1) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint8_t* k = a.k + r.b * a.ksb + (r.h / a.rep) * a.ksh;
    const uint8_t* v = a.v + r.b * a.vsb + (r.h / a.rep) * a.vsh;
    const TileLoad<false> load_k(k, a.kss, r.kv_len);
    const TileLoad<true> load_v(v, a.vss, r.kv_len);
    const int i0 = r.i0 + 32 * wave, i = i0 + (lane & 31);
    // this lane's position; padded queries are the last one again, or all of a wave's tiles would take the masked path
    // (509 queries over 16381 keys: 219 us, so 157), and are written as zeros
    const int p = r.off + min(i, r.q_len - 1);
    const int pw0 = r.off + i0, pw1 = r.off + min(i0 + 31, r.q_len - 1);
#pragma unroll
    for (int ct = 0; ct < 4; ++ct)
#pragma unroll
      for (int j = 0; j < 16; ++j) acc[ct][j] = 0.f;
    m = kNegInf;
    l = 0.f;
    seen = false;
    if (t0 >= t1) return;
    auto products = [&](const LdsTile& kc, const LdsTile& vc, int key0) {
      const bool none = pw1 < key0 || pw1 < pw0 ||
                        (a.window > 0 && key0 + kBN - 1 <= pw0 - a.window && key0 >= a.sinks);
      if (none) return;  // this wave's queries see nothing of the tile
      tile(kc, vc, a, q, scale, key0, p, pw0, pw1);
      if constexpr (ROBUST) add_bad(s, a, k, v, q, scale, key0, p, r.kv_len);
    };
    // this wave's loads have arrived, and then every wave's; the other buffer is free
    auto arrived = [&]() {
      __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
      __syncthreads();
    };
    __syncthreads();  // a first run's reads
    if constexpr (ROBUST) {
      for (int t = t0; t < t1; ++t) {
        const int key0 = kt.key(t);
        if (threadIdx.x < 2) s.bad[threadIdx.x] = 0;
        __syncthreads();
        load_k(key0, s.k0);
        load_v_finite(v, a.vss, key0, r.kv_len, s);
        arrived();
        products(s.k0, s.v0, key0);
        __syncthreads();
      }
    } else {
      load_k(kt.key(t0), s.k0);
      load_v(kt.key(t0), s.v0);
      for (int t = t0; t < t1; t += 2) {
        arrived();
        if (t + 1 < t1) {
          load_k(kt.key(t + 1), s.k1);
          load_v(kt.key(t + 1), s.v1);
        }
        products(s.k0, s.v0, kt.key(t));
        if (t + 1 == t1) break;
        arrived();
        if (t + 2 < t1) {
          load_k(kt.key(t + 2), s.k0);
          load_v(kt.key(t + 2), s.v0);
        }
        products(s.k1, s.v1, kt.key(t + 1));
      }
    }
    __syncthreads();  // the buffers are free
  }
};

// One unit: its queries over its keys, and the output or the split's part.  Returns whether the result is
// not finite (and then has written nothing), or false.
template <class T, bool ROBUST>
__device__ __forceinline__ bool attend_unit(const Lds& s, const PreArgs& a, int64_t unit) {
  const Row r = unit_of(a, unit);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int ql = lane & 31, hh = lane >> 5;
  const int last = min(r.i0 + kBM, r.q_len) - 1;
  const KeyTiles kt(r.off + r.i0, last < r.i0 ? -1 : r.off + last, a.window, a.sinks);
  const int t0 = kt.count * r.split / a.splits, t1 = kt.count * (r.split + 1) / a.splits;  // at most 2^24 tiles, 32 splits

  u32x4 q[8];
  {
    const int i = max(min(r.i0 + 32 * wave + ql, r.q_len - 1), 0);
    const uint8_t* qp = a.q + r.b * a.qsb + r.h * a.qsh + i * a.qss + 16 * hh;
#pragma unroll
    for (int kk = 0; kk < 8; ++kk) q[kk] = *(const u32x4*)(qp + 32 * kk);
  }
  float scale = a.sm;
  if (a.inv_tau) scale *= a.inv_tau[r.h];

  Prefill<T> f;
  f.template attend<ROBUST>(s, a, r, q, scale, kt, t0, t1);
  if constexpr (!ROBUST) {
    bool odd = false;
#pragma unroll
    for (int ct = 0; ct < 4; ++ct)
#pragma unroll
      for (int j = 0; j < 16; ++j) odd |= !(fabsf(f.acc[ct][j]) < __builtin_inff());
    if (__syncthreads_or(odd)) return true;
  }

  float l = f.l + xor32(f.l);
  const bool seen = __shfl_xor((int)f.seen, 32, 64) | (int)f.seen;
  const int row = 32 * wave + ql;
  if (a.splits > 1) {
    // a sum whose maximum is -inf is none: 1 where something was seen, else 0
    if (f.m == kNegInf && l == l) l = seen ? 1.f : 0.f;
    if (hh == 0) a.ml[unit * kBM + row] = float2{f.m, l};
    float* o = a.part + (unit * kBM + row) * 128 + 4 * hh;
#pragma unroll
    for (int ct = 0; ct < 4; ++ct)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        *(float4v*)(o + 32 * ct + 8 * e) = float4v{f.acc[ct][4 * e], f.acc[ct][4 * e + 1], f.acc[ct][4 * e + 2], f.acc[ct][4 * e + 3]};
    return false;
  }
  // the maximum is -inf where nothing was seen (0), or where all that was seen scored -inf (NaN)
  const float inv = f.m == kNegInf && l == l ? (seen ? __builtin_nanf("") : 0.f) : 1.0f / l;
  // through LDS for whole rows: [query][16 chunks], chunk ^ (query % 16)
  u32x2* const o = (u32x2*)(wave < 2 ? s.k0 : s.k1);
#pragma unroll
  for (int ct = 0; ct < 4; ++ct)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int chunk = 4 * ct + e;  // 8 channels, this lane's half of them
      o[((row & 63) * 16 + (chunk ^ (row & 15))) * 2 + hh] =
          u32x2{T::pack(f.acc[ct][4 * e] * inv, f.acc[ct][4 * e + 1] * inv), T::pack(f.acc[ct][4 * e + 2] * inv, f.acc[ct][4 * e + 3] * inv)};
    }
  __syncthreads();
  const int t = threadIdx.x;
#pragma unroll
  for (int u = 0; u < 8; ++u) {
    const int x = (t >> 4) + 16 * u, i = r.i0 + x;
    if (i < a.S)
      *(u32x4*)(a.out + r.b * a.osb + r.h * a.osh + i * a.oss + (t & 15) * 16) =
          i < r.q_len ? (u < 4 ? s.k0 : s.k1)[(x & 63) * 16 + ((t & 15) ^ (x & 15))] : u32x4{0, 0, 0, 0};
  }
  return false;
}

// the rare second run, kept out of the kernel's own register allocation
template <class T>
__device__ __attribute__((noinline)) void attend_again(const Lds* s, const PreArgs* a, int64_t unit) {
  attend_unit<T, true>(*s, *a, unit);
}

template <class T>
__global__ __launch_bounds__(kThreads, 2) void prefill_kernel(PreArgs a) {
  __shared__ LdsTile k0, v0, k1, v1;
  __shared__ uint32_t bad[2];
  const Lds s{k0, v0, k1, v1, bad};
  const int64_t unit = unit_at(a, blockIdx.x);
  if (unit < 0) return;
  if (attend_unit<T, false>(s, a, unit)) {
    const PreArgs again = a;
    attend_again<T>(&s, &again, unit);
  }
}

// Joins the splits of a block: a wave a query, two channels a lane.  A split's weight is worked out by the lane of its
// number; their parts' loads are four side by side.
template <class T>
__global__ __launch_bounds__(256) void prefill_join_kernel(PreArgs a) {
  const int64_t unit = (int64_t)blockIdx.x * a.splits;
  const Row r = unit_of(a, unit);
  const int row = blockIdx.y * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63, i = r.i0 + row;
  if (i >= a.S) return;
  uint32_t result = 0;
  if (i < r.q_len) {
    const float2 ml = lane < a.splits ? a.ml[(unit + lane) * kBM + row] : float2{kNegInf, 0.f};
    float M = ml.x, x = 0.f, y = 0.f;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor(M, o, 64));
    const float f = fast_exp2(ml.x - (M == kNegInf ? 0.f : M));
    float L = lane < a.splits ? ml.y * (M == kNegInf ? 1.f : f) : 0.f;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) L += __shfl_xor(L, o, 64);
    const float* part = a.part + (unit * kBM + row) * 128 + 2 * lane;
    int s = 0;
    for (; s + 4 <= a.splits; s += 4) {
      float2 o[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) o[u] = *(const float2*)(part + (int64_t)(s + u) * kBM * 128);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const float fs = __shfl(f, s + u, 64);
        x = fmaf(o[u].x, fs, x);
        y = fmaf(o[u].y, fs, y);
      }
    }
    for (; s < a.splits; ++s) {
      const float2 o = *(const float2*)(part + (int64_t)s * kBM * 128);
      const float fs = __shfl(f, s, 64);
      x = fmaf(o.x, fs, x);
      y = fmaf(o.y, fs, y);
    }
    // no maximum: nothing was seen (0), or all that was seen scored -inf (NaN)
    const float inv = M == kNegInf && L == L ? (L > 0.f ? __builtin_nanf("") : 0.f) : 1.0f / L;
    result = T::pack(x * inv, y * inv);
  }
  *(uint32_t*)(a.out + r.b * a.osb + r.h * a.osh + i * a.oss + 4 * lane) = result;
}

// ---------------------------------------------------------------- host

constexpr int kTarget = 512;  // work-groups that fill the GPU: two a CU
constexpr int kMaxSplits = 32;

struct Plan {
  int blocks, splits;
  int64_t units, grid, ml, bytes;
};

Plan plan_of(const kvq_prefill_params& p) {
  Plan w{};
  w.blocks = (p.seq_q + kBM - 1) / kBM;
  const int64_t whole = (int64_t)p.batch * p.q_heads * w.blocks;
  // key tiles of the block that sees most
  int64_t tiles = ((int64_t)p.seq_kv + kBN - 1) / kBN;
  if (p.window > 0) {
    const int64_t some = ((int64_t)p.window + kBM + kBN - 1) / kBN + 1 + ((p.sinks > 0 ? p.sinks : 0) + kBN - 1) / kBN;
    if (some < tiles) tiles = some;
  }
  // Fewer blocks than work-groups fit: the number of splits, of at least four tiles, that takes the least time by what
  // was measured: a tile 2.3 us (1.75 where a work-group has its CU alone), a work-group's start 6, a join 3 and 0.016
  // a part.  Against as many splits as fit at once, us: 1024 queries of 40 heads over 16384 keys 371 (476 in one), 4 x 300
  // of 28 heads over 4096 118 (127), 1024 of 28 heads 29 (37); 512 of 28 heads over 4096 53 (in two rounds 67).
  int64_t s = 1;
  if (whole > 0 && whole < kTarget) {
    float least = 0;
    for (int64_t n = 1; n == 1 || (n <= kMaxSplits && 4 * n <= tiles); ++n) {
      const int64_t units = whole * n, rounds = (units + kTarget - 1) / kTarget;
      const float us = rounds * ((tiles + n - 1) / n * (units <= kTarget / 2 ? 1.75f : 2.3f) + 6.f) + (n > 1 ? 3.f + 0.016f * units : 0.f);
      if (n == 1 || us < least) {
        least = us;
        s = n;
      }
    }
  }
  w.splits = (int)s;
  w.units = whole * s;
  const int64_t depth = w.blocks * s;
  if (depth > 0) w.grid = 8 * (((w.units + 7) / 8 + depth - 1) / depth) * depth;  // whole (row, head)s an XCD
  if (s > 1) {
    w.ml = w.units * kBM * 128 * 4;
    w.bytes = w.ml + w.units * kBM * 8;
  }
  return w;
}

int check(const kvq_prefill_params* p) {
  if (!p) return fail(KVQ_ERR_INVALID, "prefill: NULL params");
  if (p->batch < 0 || p->q_heads <= 0 || p->kv_heads <= 0 || p->seq_q < 0 || p->seq_kv < 0) return fail(KVQ_ERR_INVALID, "prefill: negative size");
  if (p->q_heads % p->kv_heads) return fail(KVQ_ERR_INVALID, "prefill: q_heads must be a multiple of kv_heads");
  if (p->type != KVQ_PAGED_F16 && p->type != KVQ_PAGED_BF16) return fail(KVQ_ERR_INVALID, "prefill: unknown type");
  if (p->seq_q > (1 << 30) || p->seq_kv > (1 << 30)) return fail(KVQ_ERR_UNSUPPORTED, "prefill: more than 2^30 tokens");
  if ((int64_t)p->batch * p->q_heads * ((p->seq_q + kBM - 1) / kBM) > (1 << 26) || plan_of(*p).grid >= (1 << 24))
    return fail(KVQ_ERR_UNSUPPORTED, "prefill: too many queries");  // 2^32 threads are no launch
  return KVQ_OK;
}

int prefill(const kvq_prefill_params* p, hipStream_t st) {
  int rc = check(p);
  if (rc) return rc;
  const Plan w = plan_of(*p);
  if (w.units == 0) return KVQ_OK;
  if (!p->q || !p->out || (p->seq_kv > 0 && (!p->k || !p->v))) return fail(KVQ_ERR_INVALID, "prefill: NULL pointer");
  if (((uintptr_t)p->q | (uintptr_t)p->k | (uintptr_t)p->v | (uintptr_t)p->out) % 16 ||
      (p->q_stride_b | p->q_stride_h | p->q_stride_s | p->k_stride_b | p->k_stride_h | p->k_stride_s | p->v_stride_b |
       p->v_stride_h | p->v_stride_s | p->o_stride_b | p->o_stride_h | p->o_stride_s) % 8)
    return fail(KVQ_ERR_INVALID, "prefill: rows must be 16-byte aligned");
  if (p->k_stride_s < 0 || p->v_stride_s < 0 || p->k_stride_s > (1 << 23) || p->v_stride_s > (1 << 23))
    return fail(KVQ_ERR_UNSUPPORTED, "prefill: token stride out of range");  // 64 of them fit 32 bits
  if (w.bytes && (!p->workspace || p->workspace_bytes < w.bytes || (uintptr_t)p->workspace % 16))
    return fail(KVQ_ERR_INVALID, "prefill: workspace too small or not 16-byte aligned");
  PreArgs a{};
  a.q = (const uint8_t*)p->q; a.k = (const uint8_t*)p->k; a.v = (const uint8_t*)p->v; a.out = (uint8_t*)p->out;
  a.qsb = 2 * p->q_stride_b; a.qsh = 2 * p->q_stride_h; a.qss = 2 * p->q_stride_s;
  a.ksb = 2 * p->k_stride_b; a.ksh = 2 * p->k_stride_h; a.kss = 2 * p->k_stride_s;
  a.vsb = 2 * p->v_stride_b; a.vsh = 2 * p->v_stride_h; a.vss = 2 * p->v_stride_s;
  a.osb = 2 * p->o_stride_b; a.osh = 2 * p->o_stride_h; a.oss = 2 * p->o_stride_s;
  a.q_lens = p->q_lens; a.kv_lens = p->kv_lens; a.inv_tau = p->inv_tau;
  a.sm = p->sm_scale * kLog2e;
  a.batch = p->batch; a.q_heads = p->q_heads; a.rep = p->q_heads / p->kv_heads;
  a.S = p->seq_q; a.T = p->seq_kv; a.window = p->window; a.sinks = p->sinks;
  a.blocks = w.blocks; a.splits = w.splits; a.units = w.units;
  a.part = (float*)p->workspace;
  a.ml = (float2*)((uint8_t*)p->workspace + w.ml);
  const bool b16 = p->type == KVQ_PAGED_BF16;
  const dim3 grid((unsigned)w.grid), block(kThreads);
  if (b16) hipLaunchKernelGGL(prefill_kernel<TB16>, grid, block, 0, st, a);
  else hipLaunchKernelGGL(prefill_kernel<TF16>, grid, block, 0, st, a);
  if ((rc = launched())) return rc;
  if (w.splits > 1) {
    const dim3 jg((unsigned)(w.units / w.splits), kBM / 4);
    if (b16) hipLaunchKernelGGL(prefill_join_kernel<TB16>, jg, dim3(256), 0, st, a);
    else hipLaunchKernelGGL(prefill_join_kernel<TF16>, jg, dim3(256), 0, st, a);
    rc = launched();
  }
  return rc;
}

}  // namespace
}  // namespace kvq

extern "C" int kvq_prefill_attn(const kvq_prefill_params* p, kvq_stream_t stream) {
  return kvq::guarded([&] { return kvq::prefill(p, reinterpret_cast<hipStream_t>(stream)); });
}

extern "C" int64_t kvq_prefill_workspace_bytes(const kvq_prefill_params* p) {
  if (kvq::guarded([&] { return kvq::check(p); })) return 0;
  return kvq::plan_of(*p).bytes;
}
