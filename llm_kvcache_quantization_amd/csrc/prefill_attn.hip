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
// r}, r < 4; V is staged transposed with those keys side by side, 16 bytes a (channel, 16 keys, half).
//
// K and V tiles go through registers into LDS, two buffers each, the next tile's loads under the present
// one's products.  Rows of both are XOR-swizzled in 16-byte chunks so that the operands' reads and the
// stores spread over all banks.
//
// What is masked may hold anything.  Keys at or past kv_lens are staged as zeros.  An Inf or NaN in a V row
// that some query of a tile sees and another does not would reach both (0 x NaN): where a work-group's result
// is not finite it runs again with such rows taken out of the products and added query by query.
//
// What bounds it: the matrix units and the exponentials, about equally.
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

__device__ __forceinline__ Row unit_of(const PreArgs& a, int64_t unit) {
  Row r;
  r.split = (int)(unit % a.splits);
  unit /= a.splits;
  r.block = a.blocks - 1 - (int)(unit % a.blocks);  // the later queries see more keys: first
  unit /= a.blocks;
  r.h = (int)(unit % a.q_heads);
  r.b = (int)(unit / a.q_heads);
  r.q_len = a.q_lens ? min(max(a.q_lens[r.b], 0), a.S) : a.S;
  r.kv_len = a.kv_lens ? min(max(a.kv_lens[r.b], 0), a.T) : a.T;
  r.off = r.kv_len - r.q_len;
  r.i0 = r.block * kBM;
  return r;
}

__device__ __forceinline__ bool sees(int p, int key, int window, int sinks) {
  return key <= p && (window <= 0 || key > p - window || key < sinks);
}
__device__ __forceinline__ float xor32(float x) { return __shfl_xor(x, 32, 64); }
__device__ __forceinline__ uint32_t pk_max_u16(uint32_t a, uint32_t b) {
  typedef uint16_t u16v2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16v2, a), __builtin_bit_cast(u16v2, b)));
}

template <class T>
struct Prefill {
  struct Lds {
    u32x4 k[2][kBN * 16];   // [key][16 chunks of 8 channels], chunk ^ (key % 16)
    u32x4 v[2][128 * 8];    // [channel][8 chunks of 8 keys], chunk ^ swizzle(channel)
    uint32_t bad[2];        // keys of the tile whose V row is not finite
  };
  static __device__ __forceinline__ int vswz(int ch) { return ((ch >> 1) ^ (ch >> 4)) & 7; }

  u32x4 rk[4];
  u32x2 rv[8];

  // this thread's part of the tile at key0: K rows t / 16 + 16 u, chunk t % 16; V: channels 4 (t % 32) .. of
  // the 8 keys of chunk t / 32.  A tile's base is the same for all threads, offsets in it fit 32 bits.
  __device__ __forceinline__ void load(const uint8_t* k, const uint8_t* v, const PreArgs& a, int key0, int kv_len) {
    const int t = threadIdx.x, grp = t >> 5;
    const int krow = t >> 4, vrow = 16 * (grp >> 1) + 4 * (grp & 1);
    const uint32_t ko = (uint32_t)krow * (uint32_t)a.kss + (t & 15) * 16, vo = (uint32_t)vrow * (uint32_t)a.vss + (t & 31) * 8;
    const uint8_t* kb = k + key0 * a.kss;
    const uint8_t* vb = v + key0 * a.vss;
    if (key0 + kBN <= kv_len) {
#pragma unroll
      for (int u = 0; u < 4; ++u) rk[u] = *(const u32x4*)(kb + 16 * u * a.kss + ko);
#pragma unroll
      for (int j = 0; j < 8; ++j) rv[j] = *(const u32x2*)(vb + ((j & 3) + 8 * (j >> 2)) * a.vss + vo);
    } else {
      const int left = kv_len - key0;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        rk[u] = u32x4{0, 0, 0, 0};
        if (krow + 16 * u < left) rk[u] = *(const u32x4*)(kb + 16 * u * a.kss + ko);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        rv[j] = u32x2{0, 0};
        if (vrow + (j & 3) + 8 * (j >> 2) < left) rv[j] = *(const u32x2*)(vb + ((j & 3) + 8 * (j >> 2)) * a.vss + vo);
      }
    }
  }
  template <bool ROBUST>
  __device__ __forceinline__ void store(Lds& s, int buf) {
    const int t = threadIdx.x;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int row = (t >> 4) + 16 * u;
      s.k[buf][row * 16 + ((t & 15) ^ (row & 15))] = rk[u];
    }
    const int grp = t >> 5, c4 = t & 31;
    if constexpr (ROBUST) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        bool odd = false;
#pragma unroll
        for (int d = 0; d < 2; ++d)
          odd |= !(fabsf(T::to_f((uint16_t)rv[j][d])) < __builtin_inff()) ||
                 !(fabsf(T::to_f((uint16_t)(rv[j][d] >> 16))) < __builtin_inff());
        // a row's 32 lanes are one half of the wave
        const uint64_t m = __ballot(odd);
        if ((uint32_t)(threadIdx.x & 32 ? m >> 32 : m)) {
          rv[j] = u32x2{0, 0};
          const int key = 16 * (grp >> 1) + 4 * (grp & 1) + (j & 3) + 8 * (j >> 2);
          if (c4 == 0) atomicOr(&s.bad[key >> 5], 1u << (key & 31));
        }
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int ch = 4 * c4 + e;
      const uint32_t sel = e & 1 ? 0x07060302u : 0x05040100u;
      u32x4 w;
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = perm_b32(rv[2 * j + 1][e >> 1], rv[2 * j][e >> 1], sel);
      s.v[buf][ch * 8 + (grp ^ vswz(ch))] = w;
    }
  }

  float16v acc[4];
  float m, l;
  bool seen;

  template <bool ROBUST>
  __device__ __forceinline__ void attend(Lds& s, const PreArgs& a, const Row& r, const u32x4 (&q)[8], float scale,
                                         const KeyTiles& kt, int t0, int t1) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int ql = lane & 31, hh = lane >> 5;
    const uint8_t* k = a.k + r.b * a.ksb + (r.h / a.rep) * a.ksh;
    const uint8_t* v = a.v + r.b * a.vsb + (r.h / a.rep) * a.vsh;
    const int i = r.i0 + 32 * wave + ql;
    const int p = i < r.q_len ? r.off + i : -1;  // this lane's position; -1 sees nothing
    const int pw0 = r.off + r.i0 + 32 * wave, pw1 = r.off + min(r.i0 + 32 * wave + 31, r.q_len - 1);
#pragma unroll
    for (int ct = 0; ct < 4; ++ct)
#pragma unroll
      for (int j = 0; j < 16; ++j) acc[ct][j] = 0.f;
    m = kNegInf;
    l = 0.f;
    seen = false;
    if (t0 >= t1) return;
    if (ROBUST) {
      __syncthreads();
      if (threadIdx.x < 2) s.bad[threadIdx.x] = 0;
      __syncthreads();
    }
    load(k, v, a, kt.key(t0), r.kv_len);
    store<ROBUST>(s, 0);
    __syncthreads();
    for (int t = t0; t < t1; ++t) {
      const int buf = ROBUST ? 0 : (t - t0) & 1, key0 = kt.key(t);
      const bool more = t + 1 < t1;
      if (more) load(k, v, a, kt.key(t + 1), r.kv_len);
      // what this wave's queries see of the tile: all, some, or nothing
      const bool none = pw1 < key0 || pw1 < pw0 ||
                        (a.window > 0 && key0 + kBN - 1 <= pw0 - a.window && key0 >= a.sinks);
      const bool full = key0 + kBN - 1 <= pw0 && r.i0 + 32 * wave + 31 < r.q_len &&
                        (a.window <= 0 || key0 > pw1 - a.window || key0 + kBN <= a.sinks);
      if (!none) {
        float16v sc[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
#pragma unroll
          for (int j = 0; j < 16; ++j) sc[u][j] = 0.f;
          const int row = 32 * u + ql;
#pragma unroll
          for (int kk = 0; kk < 8; ++kk)
            sc[u] = T::mfma32(s.k[buf][row * 16 + ((2 * kk + hh) ^ (row & 15))], q[kk], sc[u]);
        }
        float mul = scale;
        if (!full) {
          mul = 1.f;
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              const int key = key0 + 32 * u + 8 * (j >> 2) + 4 * hh + (j & 3);
              const bool vis = sees(p, key, a.window, a.sinks);
              seen |= vis;
              sc[u][j] = vis ? sc[u][j] * scale : kNegInf;
            }
        } else {
          seen = true;
        }
        u32x4 pb[2][2];
        auto exps = [&]() {
          const float mm = -(m == kNegInf ? 0.f : m);
          uint32_t top = 0;
          float sum = 0.f;
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int j = 0; j < 16; j += 2) {
              const float e0 = fast_exp2(fmaf(sc[u][j], mul, mm)), e1 = fast_exp2(fmaf(sc[u][j + 1], mul, mm));
              sum += e0 + e1;
              const uint32_t w = T::pack(e0, e1);
              pb[u][j >> 3][(j >> 1) & 3] = w;
              top = pk_max_u16(top, w);
            }
          l += sum;
          return max(top & 0xFFFFu, top >> 16);
        };
        // 64 as a 16-bit value: P's bits order as its values, which are not negative
        const uint32_t limit = T::pack(64.f, 0.f);
        const float l0 = l;
        const uint32_t top = exps();
        if (__any(top > limit || m == kNegInf)) {
          // the maximum moves: rescale, and take the exponentials again
          l = l0;
          float mx = kNegInf;
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int j = 0; j < 16; ++j) mx = fmaxf(mx, sc[u][j] * mul);
          mx = fmaxf(fmaxf(mx, xor32(mx)), m);
          const float f = fast_exp2(m - (mx == kNegInf ? 0.f : mx));
          l *= f;
#pragma unroll
          for (int ct = 0; ct < 4; ++ct) acc[ct] *= f;
          m = mx;
          exps();
        }
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int mm = 0; mm < 2; ++mm)
#pragma unroll
            for (int ct = 0; ct < 4; ++ct) {
              const int ch = 32 * ct + ql;
              acc[ct] = T::mfma32(s.v[buf][ch * 8 + ((4 * u + 2 * mm + hh) ^ vswz(ch))], pb[u][mm], acc[ct]);
            }
        if constexpr (ROBUST) {
          for (int w = 0; w < 2; ++w)
            for (uint32_t left = s.bad[w]; left; left &= left - 1) {
              const int kl = 32 * w + __builtin_ctz(left), key = key0 + kl;
              // every lane makes the products of its own query's scores again, for this key
              const uint8_t* kr = k + key * a.kss;
              float d = 0.f;
              for (int kk = 0; kk < 8; ++kk)
                for (int e = 0; e < 8; ++e) {
                  const uint16_t kb = *(const uint16_t*)(kr + (16 * kk + 8 * hh + e) * 2);
                  uint32_t qb = 0;
#pragma unroll
                  for (int z = 0; z < 8; ++z)
                    if (z == kk) qb = e & 1 ? q[z][e >> 1] >> 16 : q[z][e >> 1] & 0xFFFFu;
                  d = fmaf(T::to_f((uint16_t)qb), T::to_f(kb), d);
                }
              d += xor32(d);
              if (sees(p, key, a.window, a.sinks)) {
                const float e = fast_exp2(fmaf(d, scale, -(m == kNegInf ? 0.f : m)));
                for (int ct = 0; ct < 4; ++ct)
#pragma unroll
                  for (int j = 0; j < 16; ++j) {
                    const int ch = 32 * ct + 8 * (j >> 2) + 4 * hh + (j & 3);
                    const float x = e * T::to_f(*(const uint16_t*)(v + key * a.vss + ch * 2));
#pragma unroll
                    for (int z = 0; z < 4; ++z)
                      if (z == ct) acc[z][j] += x;
                  }
              }
            }
        }
      }
      if constexpr (ROBUST) {
        __syncthreads();
        if (threadIdx.x < 2) s.bad[threadIdx.x] = 0;
        __syncthreads();
      }
      if (more) store<ROBUST>(s, ROBUST ? 0 : buf ^ 1);
      __syncthreads();
    }
  }
};

// One unit: its queries over its keys, and the output or the split's part.  Returns whether the result is
// not finite (and then has written nothing), or false.
template <class T, bool ROBUST>
__device__ __forceinline__ bool attend_unit(typename Prefill<T>::Lds& s, const PreArgs& a, int64_t unit) {
  const Row r = unit_of(a, unit);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int ql = lane & 31, hh = lane >> 5;
  const int last = min(r.i0 + kBM, r.q_len) - 1;
  const KeyTiles kt(r.off + r.i0, last < r.i0 ? -1 : r.off + last, a.window, a.sinks);
  const int t0 = (int)((int64_t)kt.count * r.split / a.splits), t1 = (int)((int64_t)kt.count * (r.split + 1) / a.splits);

  u32x4 q[8];
  {
    const int i = min(r.i0 + 32 * wave + ql, a.S - 1);
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
  // through LDS for whole rows: [query][16 chunks], chunk ^ (query % 16); K's buffers are free
  u32x2* const o = (u32x2*)&s.k[0][0];
#pragma unroll
  for (int ct = 0; ct < 4; ++ct)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int chunk = 4 * ct + e;  // 8 channels, this lane's half of them
      o[(row * 16 + (chunk ^ (row & 15))) * 2 + hh] =
          u32x2{T::pack(f.acc[ct][4 * e] * inv, f.acc[ct][4 * e + 1] * inv), T::pack(f.acc[ct][4 * e + 2] * inv, f.acc[ct][4 * e + 3] * inv)};
    }
  __syncthreads();
  const int t = threadIdx.x;
#pragma unroll
  for (int u = 0; u < 8; ++u) {
    const int x = (t >> 4) + 16 * u, i = r.i0 + x;
    if (i < a.S)
      *(u32x4*)(a.out + r.b * a.osb + r.h * a.osh + i * a.oss + (t & 15) * 16) = ((const u32x4*)o)[x * 16 + ((t & 15) ^ (x & 15))];
  }
  return false;
}

// the rare second run, kept out of the kernel's own register allocation
template <class T>
__device__ __attribute__((noinline)) void attend_again(typename Prefill<T>::Lds* s, const PreArgs* a, int64_t unit) {
  attend_unit<T, true>(*s, *a, unit);
}

template <class T>
__global__ __launch_bounds__(kThreads, 2) void prefill_kernel(PreArgs a) {
  __shared__ typename Prefill<T>::Lds s;
  // work-groups go round the 8 XCDs: each XCD gets a run of units, whose heads share K and V in its L2
  const int64_t per = (a.units + 7) / 8;
  const int64_t unit = (int64_t)(blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if ((int64_t)(blockIdx.x >> 3) >= per || unit >= a.units) return;
  if (attend_unit<T, false>(s, a, unit)) {
    const PreArgs again = a;
    attend_again<T>(&s, &again, unit);
  }
}

// Joins the splits of a block: a wave a query, two channels a lane.
template <class T>
__global__ __launch_bounds__(256) void prefill_join_kernel(PreArgs a) {
  const int64_t unit = (int64_t)blockIdx.x * a.splits;
  const Row r = unit_of(a, unit);
  const int row = blockIdx.y * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63, i = r.i0 + row;
  if (i >= a.S) return;
  float M = kNegInf, L = 0.f, x = 0.f, y = 0.f;
  for (int s = 0; s < a.splits; ++s) M = fmaxf(M, a.ml[(unit + s) * kBM + row].x);
  const float shift = M == kNegInf ? 0.f : M;
  for (int s = 0; s < a.splits; ++s) {
    const float2 p = a.ml[(unit + s) * kBM + row];
    const float2 o = *(const float2*)(a.part + ((unit + s) * kBM + row) * 128 + 2 * lane);
    const float f = fast_exp2(p.x - shift);
    L += p.y * (M == kNegInf ? 1.f : f);
    x = fmaf(o.x, f, x);
    y = fmaf(o.y, f, y);
  }
  const float inv = M == kNegInf && L == L ? (L > 0.f ? __builtin_nanf("") : 0.f) : 1.0f / L;
  *(uint32_t*)(a.out + r.b * a.osb + r.h * a.osh + i * a.oss + 4 * lane) = T::pack(x * inv, y * inv);
}

// ---------------------------------------------------------------- host

constexpr int kTarget = 512;  // work-groups that fill the GPU: two a CU
constexpr int kMaxSplits = 32;

struct Plan {
  int blocks, splits;
  int64_t units, ml, bytes;
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
  int64_t s = 1;
  if (whole > 0 && whole < kTarget) {
    s = kTarget / whole;
    if (s > tiles / 4) s = tiles / 4;  // a split of fewer than four tiles costs more in the join than it gains
    if (s > kMaxSplits) s = kMaxSplits;
    if (s < 1) s = 1;
  }
  w.splits = (int)s;
  w.units = whole * s;
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
  if ((int64_t)p->batch * p->q_heads * ((p->seq_q + kBM - 1) / kBM) > (1 << 26)) return fail(KVQ_ERR_UNSUPPORTED, "prefill: too many queries");
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
  const dim3 grid((unsigned)((w.units + 7) / 8 * 8)), block(kThreads);
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
