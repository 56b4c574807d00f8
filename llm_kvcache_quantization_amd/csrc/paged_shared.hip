// Attention of one new token a row over a paged cache, where the rows of a group share their first tokens
// (kvq_shared_decode).
//
//   out[b,h] = sum_t p_t v_t,  p = softmax over t < n_b of sm_scale inv_tau_h q.k_t,
//   K and V of t < P (the group's prefix) in the pages of the group's first row
//
// The softmax is taken in parts (maximum, sum, accumulator) that a second launch joins: those of the prefix,
// whose K and V are read once for the columns (row, query head) of a KV head together, and those of each row's
// own tokens behind it, its tail.
//
// A work-group of four waves takes up to 128 columns (a prefix's) or a row's heads (a tail's) through a run of tiles of
// 64 tokens, in LDS, two buffers, as the prompts' attention does it.  A wave has 32 columns.  Up to 64 columns
// two waves share them, each with half of a tile's tokens, and join at the end.
//
// Tokens that nobody sees (outside the run's range, pages that are not there) are loaded from a row of zeros, so
// that a masked NaN reaches nobody; all columns of a work-group see the same tokens.  A row that is shorter than its
// group's prefix takes no part in it: its tail begins at its first token, in the pages of the group's first row.
#include <type_traits>

#include "attn_tile.h"
#include "kvq_shared.h"

namespace kvq {
namespace {

constexpr int kThreads = 256;
constexpr int kCols = 128;      // columns a work-group
constexpr int kMaxRows = 4096;  // rows of a call
constexpr int kMaxRep = 128;    // query heads of a KV head
constexpr int kMaxChunks = 64;  // work-groups of a tail

// A prefix's work-group: columns col0 .. of the group whose first row is row0, tiles t0 .. t1 of its first len tokens; its
// parts are slot .. slot + cols - 1 of a KV head's.
struct Unit {
  int32_t row0, col0, cols, t0, t1, len, slot, reserved;
};
// A row's prefix: the group's first row and tokens; columns a work-group takes, columns of the group, runs of tiles; the
// part of column c in run s: slot + (c / per * per) * splits + s * (columns of c's work-group) + c % per.
struct RowPlan {
  int32_t row0, len, slot, splits, per, cols, reserved[2];
};

// nothing writes these while the kernels run: scalar loads
typedef const __attribute__((address_space(4))) int32_t* const_i32;

__device__ __forceinline__ RowPlan plan_of_row(const RowPlan* rows, int b) {
  const const_i32 p = (const_i32)(rows + b);
  return RowPlan{p[0], p[1], p[2], p[3], p[4], p[5], {0, 0}};
}

struct ShArgs {
  PagedCache c;
  const uint16_t* q;
  int64_t qsb, qsh;  // elements
  uint16_t* out;
  const int32_t* lens;
  const float* inv_tau;
  float sm;  // sm_scale * log2(e)
  int32_t q_heads, rep;
  const Unit* units;
  const RowPlan* rows;
  int32_t chunks;        // of a tail, at most
  int32_t prefix_slots;  // parts of the prefixes of a KV head; then those of the tails, [row][chunk][head]
  uint32_t tails;        // work-groups of tails, the launch's first
  int64_t slots;         // parts of a KV head
  float2* ml;            // [kv_heads][slots]
  float* acc;            // [kv_heads][slots][128]
};

constexpr int kTailTiles = 2;  // least tiles of a tail's work-group

// The tiles of a row's own tokens lo .. hi - 1.
struct Tail {
  int lo, hi, first, count, chunks;
  __device__ __forceinline__ Tail(const ShArgs& a, const RowPlan& r, int b) {
    const int64_t cap = (int64_t)a.c.max_pages << a.c.lg;
    hi = (int)min((int64_t)max(((const_i32)a.lens)[b], 0), cap);
    lo = hi >= r.len ? r.len : 0;
    first = lo / kBN;
    count = hi > lo ? (hi + kBN - 1) / kBN - first : 0;
    chunks = min(a.chunks, (count + kTailTiles - 1) / kTailTiles);
  }
  __device__ __forceinline__ int begin(int i) const { return first + (int)((uint32_t)count * (uint32_t)i / (uint32_t)chunks); }
};

__device__ const u32x4 zero_row[16] = {};

// What a work-group reads: tiles of tokens lo .. hi - 1 of one row's pages, for one KV head.
struct Source {
  const uint8_t *k, *v, *ks, *vs;
  const_i32 table;
  int lo, hi;
};

struct Pages {
  int32_t n[4];  // of 16 tokens each
};

__device__ __forceinline__ Pages pages_of(const PagedCache& c, const Source& s, int tile) {
  Pages p;
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int i = (tile * kBN + 16 * u) >> c.lg;
    p.n[u] = i < c.max_pages ? s.table[i] : -1;
  }
  return p;
}

// Bit u: the page of tokens 16 u .. is there.
__device__ __forceinline__ uint32_t there(const PagedCache& c, const Pages& p) {
  uint32_t ok = 0;
#pragma unroll
  for (int u = 0; u < 4; ++u) ok |= (uint32_t)((uint32_t)p.n[u] < (uint32_t)c.num_pages) << u;
  return ok;
}

// A tile's rows from 16-bit pages straight into LDS.  A wave instruction loads four rows of 16; a lane takes the chunk
// that belongs at its place.
struct Direct {
  uint32_t k_off, v_off;
  int row, chunk;
  __device__ __forceinline__ Direct(const PagedCache& c) {
    const int lane = threadIdx.x & 63;
    row = 4 * (threadIdx.x >> 6) + (lane >> 4);
    chunk = lane & 15;
    k_off = (uint32_t)row * (uint32_t)c.kst + (uint32_t)(chunk ^ row) * 16;
    v_off = (uint32_t)row * (uint32_t)c.vst + (uint32_t)(chunk ^ ((row & 3) << 2)) * 16;
  }
  __device__ __forceinline__ void load(const PagedCache& c, const Source& s, int key0, const Pages& p, uint32_t ok, LdsTile& kt,
                                       LdsTile& vt) const {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const bool all = ok == 15 && key0 >= s.lo && key0 + kBN <= s.hi;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int at = 16 * u + 4 * wave;  // the wave's first row
      const uint32_t slot = (uint32_t)((key0 + 16 * u) & c.page_mask);
      const int64_t page = (ok >> u & 1) ? p.n[u] : 0;
      const uint8_t* kp = s.k + page * c.ksp + slot * (uint32_t)c.kst + k_off;
      const uint8_t* vp = s.v + page * c.vsp + slot * (uint32_t)c.vst + v_off;
      if (!all) {
        const int key = key0 + 16 * u + row;
        const bool there = (ok >> u & 1) && key >= s.lo && key < s.hi;
        kp = there ? kp : (const uint8_t*)(zero_row + chunk);
        vp = there ? vp : (const uint8_t*)(zero_row + chunk);
      }
      __builtin_amdgcn_global_load_lds((gptr)kp, (__attribute__((address_space(3))) void*)(&kt[at * 16]), 16, 0, 0);
      __builtin_amdgcn_global_load_lds((gptr)vp, (__attribute__((address_space(3))) void*)(&vt[at * 16]), 16, 0, 0);
    }
  }
};

// A tile's rows from INT8 pages: 16 codes of a row a piece, two pieces of K and of V a thread, in registers while the
// tile before it is worked on, then code x scale in fp16 (the framework's own dequantization) into LDS.
template <int GS>
struct Coded {
  static constexpr int G = 128 / GS;
  u32x4 k[2], v[2];
  uint16_t ks[2], vs[2];
  __device__ __forceinline__ void load(const PagedCache& c, const Source& s, int key0, const Pages& p, uint32_t ok) {
    const int piece = threadIdx.x & 7, half = __builtin_amdgcn_readfirstlane(threadIdx.x >> 7);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int row = (threadIdx.x >> 3) + 32 * e, key = key0 + row;  // of tokens 16 (2 e + half) ..
      const bool up = half != 0, good = (ok >> (2 * e + half)) & 1;
      const int64_t page = good ? (up ? p.n[2 * e + 1] : p.n[2 * e]) : 0;
      const uint32_t slot = (uint32_t)(key & c.page_mask);
      const bool there = good && key >= s.lo && key < s.hi;
      const uint8_t* kp = s.k + page * c.ksp + slot * (uint32_t)c.kst + piece * 16;
      const uint8_t* vp = s.v + page * c.vsp + slot * (uint32_t)c.vst + piece * 16;
      const uint8_t* ksp = s.ks + page * c.kssp + slot * (2 * G) + piece * 16 / GS * 2;
      const uint8_t* vsp = s.vs + page * c.vssp + slot * (2 * G) + piece * 16 / GS * 2;
      const uint8_t* const zero = (const uint8_t*)zero_row;
      k[e] = ld_stream<u32x4>(there ? kp : zero);
      v[e] = ld_stream<u32x4>(there ? vp : zero);
      ks[e] = *(const uint16_t*)(there ? ksp : zero);
      vs[e] = *(const uint16_t*)(there ? vsp : zero);
    }
  }
  static __device__ __forceinline__ void put(u32x4 x, uint16_t scale, u32x4* lo, u32x4* hi) {
    const half2v s = as_h2(scale * 0x00010001u);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      u32x4 y;
#pragma unroll
      for (int d = 0; d < 2; ++d) {
        const uint32_t u = x[2 * h + d] ^ 0x80808080u;
        y[2 * d] = as_u32(as_h2(code_pair(u, 0x04010400u)) * s);
        y[2 * d + 1] = as_u32(as_h2(code_pair(u, 0x04030402u)) * s);
      }
      *(h ? hi : lo) = y;
    }
  }
  __device__ __forceinline__ void store(LdsTile& kt, LdsTile& vt) const {
    const int piece = threadIdx.x & 7;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int row = (threadIdx.x >> 3) + 32 * e;
      put(k[e], ks[e], &kt[row * 16 + ((2 * piece) ^ (row & 15))], &kt[row * 16 + ((2 * piece + 1) ^ (row & 15))]);
      put(v[e], vs[e], &vt[row * 16 + ((2 * piece) ^ ((row & 3) << 2))], &vt[row * 16 + ((2 * piece + 1) ^ ((row & 3) << 2))]);
    }
  }
};

template <class M>
struct Shared : AttnTile<M> {
  using AttnTile<M>::acc;
  using AttnTile<M>::m;
  using AttnTile<M>::l;
  bool seen;

  // A tile's tokens 32 u0 .. 32 u1 - 1.
  __device__ __forceinline__ void tile(const LdsTile& ks, const LdsTile& vs, const Source& s, const u32x4 (&q)[8], float scale,
                                       int key0, uint32_t ok, int u0, int u1) {
    const bool full = ok == 15 && key0 >= s.lo && key0 + kBN <= s.hi;
    const float mul = full ? scale : 1.f;
    seen |= full;
    u32x4 kf[8], vf[8], pb[2];
    this->read_k(ks, u0, kf);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll 1
    for (int u = u0; u < u1; ++u) {
      float16v sc = this->scores(kf, q);
      this->read_v(vs, u, vf);
      __builtin_amdgcn_sched_barrier(0);
      if (!full) {
        const int first = 32 * u + 4 * ((threadIdx.x & 63) >> 5);
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const int at = first + 8 * (j >> 2) + (j & 3);  // in the tile
          const bool vis = key0 + at >= s.lo && key0 + at < s.hi && (ok >> (at >> 4) & 1);
          seen |= vis;
          sc[j] = vis ? sc[j] * scale : kNegInf;
        }
      }
      this->add_sum(this->exps(sc, mul, pb), sc, mul, pb);
      if (u + 1 < u1) this->read_k(ks, u + 1, kf);
      __builtin_amdgcn_sched_barrier(0);
      this->add_values(vf, pb);
    }
  }
};

template <class T, bool I8, int GS>
__global__ __launch_bounds__(kThreads, 2) void shared_decode_kernel(ShArgs a) {
  using M = typename std::conditional<I8, TF16, T>::type;  // the matrix instructions' type
  __shared__ LdsTile k0, v0, k1, v1;
  __shared__ float2 half_ml[2][32];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int ql = lane & 31, hh = lane >> 5, rep = a.rep;
  const PagedCache& pc = a.c;
  const int H = pc.kv_heads;

  int h, row0, col0, cols, t, t1;
  int64_t slot;
  Source s;
  {
    uint32_t at = blockIdx.x;
    if (at < a.tails) {
      h = (int)(at % (uint32_t)H);
      at /= (uint32_t)H;
      const int chunk = (int)(at % (uint32_t)a.chunks), b = (int)(at / (uint32_t)a.chunks);
      const RowPlan r = plan_of_row(a.rows, b);
      const Tail tail(a, r, b);
      if (chunk >= tail.chunks) return;
      row0 = b; col0 = 0; cols = rep;
      t = tail.begin(chunk); t1 = tail.begin(chunk + 1);
      s.lo = tail.lo; s.hi = tail.hi;
      s.table = (const_i32)(pc.table + (tail.lo == r.len ? b : r.row0) * pc.table_stride);
      slot = a.prefix_slots + ((int64_t)b * a.chunks + chunk) * rep;
    } else {
      at -= a.tails;
      h = (int)(at % (uint32_t)H);
      const const_i32 w = (const_i32)(a.units + at / (uint32_t)H);
      const Unit u{w[0], w[1], w[2], w[3], w[4], w[5], w[6], 0};
      row0 = u.row0; col0 = u.col0; cols = u.cols;
      t = u.t0; t1 = u.t1;
      s.lo = 0; s.hi = u.len;
      s.table = (const_i32)(pc.table + u.row0 * pc.table_stride);
      slot = u.slot;
    }
  }
  s.k = pc.k + h * pc.ksh; s.v = pc.v + h * pc.vsh;
  if constexpr (I8) { s.ks = pc.ks + h * pc.kssh; s.vs = pc.vs + h * pc.vssh; }
  t = __builtin_amdgcn_readfirstlane(t);
  t1 = __builtin_amdgcn_readfirstlane(t1);

  // the wave's columns and the halves of a tile that are its own
  const bool halves = cols <= 64;
  const int block = halves ? wave >> 1 : wave, u0 = halves ? wave & 1 : 0, u1 = halves ? u0 + 1 : 2;
  const bool active = 32 * block < cols;

  u32x4 q[8];
  float scale = a.sm;
  const int col = 32 * block + ql;
  {
    const int x = col0 + min(col, cols - 1), row = row0 + x / rep, head = h * rep + x % rep;
    const uint16_t* qp = a.q + row * a.qsb + head * a.qsh + 8 * hh;
#pragma unroll
    for (int kk = 0; kk < 8; ++kk) q[kk] = *(const u32x4*)(qp + 16 * kk);
    if (a.inv_tau) scale *= a.inv_tau[head];
  }

  Shared<M> f;
#pragma unroll
  for (int ct = 0; ct < 4; ++ct)
#pragma unroll
    for (int j = 0; j < 16; ++j) f.acc[ct][j] = 0.f;
  f.m = kNegInf;
  f.l = 0.f;
  f.seen = false;

  Pages p = pages_of(pc, s, t);
  uint32_t ok = there(pc, p);
  if constexpr (!I8) {
    const Direct d(pc);
    auto arrived = [&]() {  // this wave's loads have, and then every wave's; the other buffer is free
      __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
      __syncthreads();
    };
    d.load(pc, s, t * kBN, p, ok, k0, v0);
    p = pages_of(pc, s, min(t + 1, t1 - 1));
    for (; t < t1; t += 2) {
      arrived();
      uint32_t ok1 = there(pc, p);
      if (t + 1 < t1) {
        d.load(pc, s, (t + 1) * kBN, p, ok1, k1, v1);
        p = pages_of(pc, s, min(t + 2, t1 - 1));
      }
      if (active) f.tile(k0, v0, s, q, scale, t * kBN, ok, u0, u1);
      if (t + 1 == t1) break;
      arrived();
      ok = there(pc, p);
      if (t + 2 < t1) {
        d.load(pc, s, (t + 2) * kBN, p, ok, k0, v0);
        p = pages_of(pc, s, min(t + 3, t1 - 1));
      }
      if (active) f.tile(k1, v1, s, q, scale, (t + 1) * kBN, ok1, u0, u1);
    }
  } else {
    Coded<GS> d;
    d.load(pc, s, t * kBN, p, ok);
    p = pages_of(pc, s, min(t + 1, t1 - 1));
    if constexpr (std::is_same<T, TB16>::value) {
      // bf16 values in fp16: exact once the column's largest is scaled to [1, 2) by a power of two (what lies 2^24
      // and more below it loses bits that are below the sum's)
      float top = 0.f;
#pragma unroll
      for (int kk = 0; kk < 8; ++kk)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          top = fmaxf(top, fmaxf(fabsf(TB16::to_f((uint16_t)q[kk][j])), fabsf(TB16::to_f((uint16_t)(q[kk][j] >> 16)))));
      top = fmaxf(top, xor32(top));
      int ex = (int)(__builtin_bit_cast(uint32_t, top) >> 23) - 127;
      if (ex == 128 || ex == -127) ex = 0;  // Inf or NaN stays what it is; zero or a subnormal is 0
      const float g = ldexpf(1.f, -ex);
      scale = ldexpf(scale, ex);
#pragma unroll
      for (int kk = 0; kk < 8; ++kk)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          q[kk][j] = TF16::pack(TB16::to_f((uint16_t)q[kk][j]) * g, TB16::to_f((uint16_t)(q[kk][j] >> 16)) * g);
    }
    d.store(k0, v0);
    for (; t < t1; t += 2) {
      __syncthreads();
      uint32_t ok1 = there(pc, p);
      if (t + 1 < t1) {
        d.load(pc, s, (t + 1) * kBN, p, ok1);
        p = pages_of(pc, s, min(t + 2, t1 - 1));
      }
      if (active) f.tile(k0, v0, s, q, scale, t * kBN, ok, u0, u1);
      if (t + 1 == t1) break;
      d.store(k1, v1);
      __syncthreads();
      ok = there(pc, p);
      if (t + 2 < t1) {
        d.load(pc, s, (t + 2) * kBN, p, ok);
        p = pages_of(pc, s, min(t + 3, t1 - 1));
      }
      if (active) f.tile(k1, v1, s, q, scale, (t + 1) * kBN, ok1, u0, u1);
      if (t + 2 < t1) d.store(k0, v0);
    }
  }

  // a sum whose maximum is -inf is none: 1 where something was seen, else 0
  f.l += xor32(f.l);
  f.seen |= (bool)__shfl_xor((int)f.seen, 32, 64);
  if (f.m == kNegInf && f.l == f.l) f.l = f.seen ? 1.f : 0.f;
  if (halves) {
    __syncthreads();  // the buffers are free
    float4v* const other = (float4v*)(block ? k1 : k0);  // [16][64]
    if (active && u0 == 1) {
      if (hh == 0) half_ml[block][ql] = float2{f.m, f.l};
#pragma unroll
      for (int ct = 0; ct < 4; ++ct)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          other[(4 * ct + e) * 64 + lane] = float4v{f.acc[ct][4 * e], f.acc[ct][4 * e + 1], f.acc[ct][4 * e + 2], f.acc[ct][4 * e + 3]};
    }
    __syncthreads();
    if (!active || u0 == 1) return;
    const float2 o = half_ml[block][ql];
    const float top = fmaxf(f.m, o.x), f0 = part_of(f.m, top), f1 = part_of(o.x, top);
    f.l = sum_in(f.m, f.l, top) + sum_in(o.x, o.y, top);
    f.m = top;
#pragma unroll
    for (int ct = 0; ct < 4; ++ct)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float4v x = other[(4 * ct + e) * 64 + lane];
#pragma unroll
        for (int r = 0; r < 4; ++r) f.acc[ct][4 * e + r] = f.acc[ct][4 * e + r] * f0 + x[r] * f1;
      }
  }
  if (col >= cols) return;
  slot += h * a.slots + col;
  if (hh == 0) a.ml[slot] = float2{f.m, f.l};
  float* const o = a.acc + slot * 128 + 4 * hh;
#pragma unroll
  for (int ct = 0; ct < 4; ++ct)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      *(float4v*)(o + 32 * ct + 8 * e) = float4v{f.acc[ct][4 * e], f.acc[ct][4 * e + 1], f.acc[ct][4 * e + 2], f.acc[ct][4 * e + 3]};
}

// Joins a column's parts: a work-group a (row, query head), 16 parts at a time, 8 channels a thread.
template <class T>
__global__ __launch_bounds__(kThreads) void shared_join_kernel(ShArgs a) {
  __shared__ float part[16][16][10];  // 8 values, maximum, sum
  const int rep = a.rep, cc = threadIdx.x & 15, sl = threadIdx.x >> 4;
  const int head = blockIdx.x, b = blockIdx.y, h = head / rep;
  const RowPlan r = plan_of_row(a.rows, b);
  const Tail tail(a, r, b);
  const int splits = tail.lo == r.len ? r.splits : 0;
  const int c = (b - r.row0) * rep + head % rep, c0 = c / max(r.per, 1) * r.per, width = min(r.per, r.cols - c0);
  const int64_t first = h * a.slots + r.slot + (int64_t)c0 * r.splits + (c - c0);
  const int64_t own = h * a.slots + a.prefix_slots + (int64_t)b * a.chunks * rep + head % rep;
  float m = kNegInf, l = 0.f, o[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) o[k] = 0.f;
  for (int w = sl; w < splits + tail.chunks; w += 16) {
    const int64_t slot = w < splits ? first + (int64_t)w * width : own + (int64_t)(w - splits) * rep;
    const float2 p = a.ml[slot];
    const float4v x = *(const float4v*)(a.acc + slot * 128 + cc * 8), y = *(const float4v*)(a.acc + slot * 128 + cc * 8 + 4);
    const float top = fmaxf(m, p.x), f0 = part_of(m, top), f1 = part_of(p.x, top);
    l = sum_in(m, l, top) + sum_in(p.x, p.y, top);
    m = top;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      o[k] = o[k] * f0 + x[k] * f1;
      o[4 + k] = o[4 + k] * f0 + y[k] * f1;
    }
  }
#pragma unroll
  for (int k = 0; k < 8; ++k) part[sl][cc][k] = o[k];
  part[sl][cc][8] = m;
  part[sl][cc][9] = l;
  __syncthreads();
  if (threadIdx.x >= 128) return;
  const int ch = threadIdx.x, pc = ch >> 3, pk = ch & 7;
  float top = kNegInf, L = 0.f, v = 0.f;
#pragma unroll
  for (int w = 0; w < 16; ++w) top = fmaxf(top, part[w][pc][8]);
#pragma unroll
  for (int w = 0; w < 16; ++w) {
    L += sum_in(part[w][pc][8], part[w][pc][9], top);
    v = fmaf(part_of(part[w][pc][8], top), part[w][pc][pk], v);
  }
  a.out[((int64_t)b * a.q_heads + head) * 128 + ch] = (uint16_t)T::pack(v * inverse_of(top, L), 0.f);
}

// ---------------------------------------------------------------- host

constexpr int kTarget = 512;     // work-groups that fill the GPU: two a CU
constexpr int kMinTiles = 2;     // least tiles of a prefix's work-group
constexpr int kMaxSplits = 256;

int plan(const int32_t* sizes, const int32_t* lens, int32_t groups, int32_t q_heads, int32_t kv_heads, kvq_shared_plan_info* info,
         int32_t* words, int64_t capacity) {
  if (groups < 0 || (groups > 0 && (!sizes || !lens)) || !info) return fail(KVQ_ERR_INVALID, "shared plan: NULL or negative");
  if (q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads) return fail(KVQ_ERR_INVALID, "shared plan: q_heads must be a multiple of kv_heads");
  const int64_t rep = q_heads / kv_heads;
  if (rep > kMaxRep) return fail(KVQ_ERR_UNSUPPORTED, "shared plan: more than 128 query heads a KV head");
  int64_t rows = 0, work = 0;
  for (int g = 0; g < groups; ++g) {
    if (sizes[g] < 1 || lens[g] < 0) return fail(KVQ_ERR_INVALID, "shared plan: a group has at least one row and no negative length");
    if (lens[g] > (1 << 30)) return fail(KVQ_ERR_UNSUPPORTED, "shared plan: more than 2^30 shared tokens");
    rows += sizes[g];
    if (rows > kMaxRows) return fail(KVQ_ERR_UNSUPPORTED, "shared plan: more than 4096 rows");
    work += (sizes[g] * rep + kCols - 1) / kCols * (((int64_t)lens[g] + kBN - 1) / kBN);
  }
  // tiles a work-group: what fills the GPU beside one work-group of each row and KV head for the tails
  int64_t target = kTarget - rows * kv_heads;
  if (target < kTarget / 2) target = kTarget / 2;
  int64_t quota = (work * kv_heads + target - 1) / target;
  if (quota < kMinTiles) quota = kMinTiles;
  int64_t units = 0, slots = 0, row = 0;
  const auto put = [&](int64_t at, const int32_t (&w)[8]) {
    if (words && at * 8 + 8 <= capacity)
      for (int i = 0; i < 8; ++i) words[at * 8 + i] = w[i];
  };
  for (int g = 0; g < groups; ++g) {
    const int64_t cols = sizes[g] * rep, blocks = (cols + kCols - 1) / kCols, tiles = ((int64_t)lens[g] + kBN - 1) / kBN;
    const int64_t per = ((cols + blocks - 1) / blocks + 31) / 32 * 32;  // even blocks of whole waves
    int64_t splits = (tiles + quota - 1) / quota;
    if (splits > kMaxSplits) splits = kMaxSplits;
    for (int i = 0; i < sizes[g]; ++i)
      put(row + i, {(int32_t)row, lens[g], (int32_t)slots, (int32_t)splits, (int32_t)per, (int32_t)cols, 0, 0});
    for (int64_t s = 0; s < splits; ++s)
      for (int64_t c0 = 0; c0 < cols; c0 += per) {
        const int64_t width = cols - c0 < per ? cols - c0 : per;
        put(rows + units, {(int32_t)row, (int32_t)c0, (int32_t)width, (int32_t)(tiles * s / splits), (int32_t)(tiles * (s + 1) / splits),
                           lens[g], (int32_t)(slots + c0 * splits + s * width), 0});
        ++units;
      }
    slots += cols * splits;
    row += sizes[g];
  }
  info->rows = (int32_t)rows;
  info->units = (int32_t)units;
  info->slots = (int32_t)slots;
  info->words = (int32_t)(8 * (rows + units));
  return KVQ_OK;
}

int check(const kvq_shared_decode_params* p, PagedCache& c) {
  if (!p) return fail(KVQ_ERR_INVALID, "shared decode: NULL params");
  const int rc = paged_cache(p->cache, c);
  if (rc) return rc;
  if (p->q_type != KVQ_PAGED_F16 && p->q_type != KVQ_PAGED_BF16) return fail(KVQ_ERR_INVALID, "shared decode: unknown q_type");
  if (p->cache.format != KVQ_PAGED_INT8 && p->cache.format != p->q_type)
    return fail(KVQ_ERR_INVALID, "shared decode: the pages' type is another than q's");
  if (p->q_heads <= 0 || p->q_heads % c.kv_heads) return fail(KVQ_ERR_INVALID, "shared decode: q_heads must be a multiple of kv_heads");
  if (p->q_heads / c.kv_heads > kMaxRep) return fail(KVQ_ERR_UNSUPPORTED, "shared decode: more than 128 query heads a KV head");
  if (p->q_heads > 65535) return fail(KVQ_ERR_UNSUPPORTED, "shared decode: too many heads");
  if (c.batch > kMaxRows) return fail(KVQ_ERR_UNSUPPORTED, "shared decode: more than 4096 rows");
  if (p->plan.rows != c.batch || p->plan.units < 0 || p->plan.slots < 0) return fail(KVQ_ERR_INVALID, "shared decode: the plan is of another batch");
  return KVQ_OK;
}

struct Launch {
  int chunks;             // of a tail
  int64_t slots, acc, bytes;
  int64_t tails, grid;
};

Launch launch_of(const kvq_shared_decode_params& p) {
  Launch w{};
  const int64_t B = p.cache.batch, H = p.cache.kv_heads, rep = p.q_heads / H;
  const int64_t tiles = ((int64_t)p.cache.max_pages * p.cache.page_size + kBN - 1) / kBN;
  int64_t chunks = kTarget / (B > 0 ? B * H : 1);
  const int64_t most = (tiles + kTailTiles - 1) / kTailTiles;
  if (chunks > kMaxChunks) chunks = kMaxChunks;
  if (chunks > most) chunks = most;
  w.chunks = (int)(chunks < 1 ? 1 : chunks);
  w.slots = p.plan.slots + B * w.chunks * rep;
  w.acc = (8 * H * w.slots + 63) / 64 * 64;
  w.bytes = w.acc + 512 * H * w.slots;
  w.tails = B * H * w.chunks;
  w.grid = w.tails + H * p.plan.units;
  return w;
}

template <class T, bool I8, int GS>
int launch(const ShArgs& a, const Launch& w, hipStream_t st) {
  hipLaunchKernelGGL((shared_decode_kernel<T, I8, GS>), dim3((unsigned)w.grid), dim3(kThreads), 0, st, a);
  const int rc = launched();
  if (rc) return rc;
  hipLaunchKernelGGL(shared_join_kernel<T>, dim3((unsigned)a.q_heads, (unsigned)a.c.batch), dim3(kThreads), 0, st, a);
  return launched();
}

int decode(const kvq_shared_decode_params* p, hipStream_t st) {
  ShArgs a{};
  int rc = check(p, a.c);
  if (rc) return rc;
  if (a.c.batch == 0) return KVQ_OK;
  if (!p->q || !p->out || !p->context_lens || !p->plan_words) return fail(KVQ_ERR_INVALID, "shared decode: NULL pointer");
  if (((uintptr_t)p->q | (uintptr_t)p->out) % 16 || (p->q_stride_b | p->q_stride_h) % 8)
    return fail(KVQ_ERR_INVALID, "shared decode: q rows must be 16-byte aligned");
  const Launch w = launch_of(*p);
  if (w.grid >= (1 << 24) || w.slots >= (1 << 30)) return fail(KVQ_ERR_UNSUPPORTED, "shared decode: too many rows and heads");
  if (!p->workspace || p->workspace_bytes < w.bytes || (uintptr_t)p->workspace % 16)
    return fail(KVQ_ERR_INVALID, "shared decode: workspace too small or not 16-byte aligned");
  // without pages every row sees nothing: no column of the table is read
  if (a.c.num_pages == 0) a.c.max_pages = 0;
  a.q = (const uint16_t*)p->q; a.qsb = p->q_stride_b; a.qsh = p->q_stride_h;
  a.out = (uint16_t*)p->out;
  a.lens = p->context_lens;
  a.inv_tau = p->inv_tau;
  a.sm = p->sm_scale * kLog2e;
  a.q_heads = p->q_heads; a.rep = p->q_heads / a.c.kv_heads;
  a.rows = (const RowPlan*)p->plan_words;
  a.units = (const Unit*)(p->plan_words + 8 * (int64_t)p->plan.rows);
  a.chunks = w.chunks;
  a.prefix_slots = p->plan.slots;
  a.tails = (uint32_t)w.tails;
  a.slots = w.slots;
  a.ml = (float2*)p->workspace;
  a.acc = (float*)((uint8_t*)p->workspace + w.acc);
  const bool b16 = p->q_type == KVQ_PAGED_BF16;
  const int gs = p->cache.format == KVQ_PAGED_INT8 ? p->cache.group_size : 0;
#define KVQ_SH(I8, GS) return b16 ? launch<TB16, I8, GS>(a, w, st) : launch<TF16, I8, GS>(a, w, st)
  if (gs == 0) KVQ_SH(false, 128);
  if (gs == 32) KVQ_SH(true, 32);
  if (gs == 64) KVQ_SH(true, 64);
  KVQ_SH(true, 128);
#undef KVQ_SH
}

}  // namespace
}  // namespace kvq

extern "C" int kvq_shared_plan(const int32_t* sizes, const int32_t* lens, int32_t groups, int32_t q_heads, int32_t kv_heads,
                               kvq_shared_plan_info* info, int32_t* words, int64_t capacity) {
  return kvq::guarded([&] { return kvq::plan(sizes, lens, groups, q_heads, kv_heads, info, words, capacity); });
}

extern "C" int kvq_shared_decode(const kvq_shared_decode_params* p, kvq_stream_t stream) {
  return kvq::guarded([&] { return kvq::decode(p, reinterpret_cast<hipStream_t>(stream)); });
}

extern "C" int64_t kvq_shared_decode_workspace_bytes(const kvq_shared_decode_params* p) {
  kvq::PagedCache c;
  if (kvq::guarded([&] { return kvq::check(p, c); })) return 0;
  return kvq::launch_of(*p).bytes;
}
