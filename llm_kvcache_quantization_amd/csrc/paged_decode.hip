// Attention of one new token a row over a paged cache (kvq_paged_decode).
//
//   out[b,h] = sum_t p_t v_t,  p = softmax over the visible t of sm_scale inv_tau_h q.k_t
//
// One pass over K and V with a running maximum and sum.  What bounds it: HBM; every visible K and V row
// is read once for all query heads of its KV head.  Measured, us a call: 8 rows x 8 KV heads x 32768 tokens in fp16 pages of 16
// 175 (6.1 TB/s), of 64 165 (6.5 TB/s); 8 ragged rows of up to 65536 tokens in INT8, groups of 32, 110 (5.8 TB/s); below
// 2048 tokens a row the chain launch, length, page, K, V, join: 9 to 13.
//
// Work: a row's visible tokens are cut into tiles of 32 token slots, and the tiles of all rows of a KV
// head are shared out over the work-groups (Share; long rows of a ragged batch are split, short ones are
// not).  A work-group writes the rows that it has whole; of a row it shares it writes (maximum, sum,
// accumulator), which a second launch joins.
//
// A wave takes a tile by itself: S^T = K Q^T, O^T = V^T P^T with 16x16x32 matrix instructions (the rows
// of a KV head's query group padded to 16).  Lane (g, c) = (lane / 16, lane % 16) of S^T holds head c and,
// with the K rows assigned to matrix rows as below, tokens 8 g .. 8 g + 7: the operand that P^T needs, so P
// never moves between lanes.  V^T's operand, 8 tokens of a channel, is transposed in registers from 8 rows'
// 16-byte loads (channels 8 c .. 8 c + 7).
#include <type_traits>

#include "paged.h"

namespace kvq {
namespace {

constexpr int kTile = 32;        // token slots a tile
constexpr int kMaxRows = 4096;   // rows of a call (the tiles before each lie in LDS)
constexpr int kHeads = 16;       // query heads of a KV head, padded

struct DecArgs {
  PagedCache c;
  const uint16_t* q;
  int64_t qsb, qsh;  // elements
  uint16_t* out;
  const int32_t* lens;
  const float* inv_tau;
  float sm;  // sm_scale * log2(e)
  int32_t window, sinks, q_heads, rep;
  int32_t groups;      // work-groups a KV head
  int32_t min_tiles;   // least tiles of a work-group
  int32_t solo;        // a work-group takes one whole row: nothing to join
  // workspace
  int32_t* pre;        // [batch + 1] tiles before each row, the tiles of a work-group (negative: work-groups of one
                       // row), [batch] the work-groups before each row
  float2* ml;          // [kv_heads][groups][2][rep] maximum (log2 units) and sum of a shared row's part:
                       // the first slot the part its tiles begin with, the second the part they end with
  float* acc;          // [kv_heads][groups][2][rep][128]
  float* lse;          // [batch][q_heads] log2 of the softmax's denominator
  float* scores;       // [kv_heads][tiles_cap][rep][32] scaled scores (log2 units), for the weights
  int64_t tiles_cap;   // tiles a KV head may have
  float* weights;
  int64_t wsb, wsh;
};

// The tiles of a row of n tokens: those of its sinks, then those from the window's first token on.
struct RowTiles {
  int sink_end, lo, sink_tiles, first, count;
  __device__ __forceinline__ RowTiles(int n, int window, int sinks) {
    sink_end = 0;
    lo = 0;
    if (window > 0 && n > window) {
      lo = n - window;
      sink_end = min(max(sinks, 0), n);
    }
    sink_tiles = (sink_end + kTile - 1) / kTile;
    first = max(lo / kTile, sink_tiles);
    count = sink_tiles + max((n + kTile - 1) / kTile - first, 0);
  }
  __device__ __forceinline__ int token(int i) const { return (i < sink_tiles ? i : first + i - sink_tiles) * kTile; }
};

__device__ __forceinline__ int row_len(const DecArgs& a, int b) {
  const int64_t cap = (int64_t)a.c.max_pages << a.c.lg;
  return (int)min((int64_t)max(a.lens[b], 0), cap);
}

// The tiles before each row.  Up to 64 rows every wave has them in its lanes, with the rows' token counts, by a
// scan of its own; more are scanned by the work-group into LDS.
struct Rows {
  int* pre;  // [batch + 1]
  int before, tokens, total;  // lane b: row b's
  bool small;
  __device__ __forceinline__ int start(int b) const { return small ? __builtin_amdgcn_readlane(before, b) : pre[b]; }
  __device__ __forceinline__ int end(int b, int batch) const { return b + 1 < batch ? start(b + 1) : total; }
  __device__ __forceinline__ int length(const DecArgs& a, int b) const {
    return small ? __builtin_amdgcn_readlane(tokens, b) : row_len(a, b);
  }
  // the last row that begins at or before tile t < total: it is not empty
  __device__ __forceinline__ int of(int t, int batch) const {
    if (small) return 63 - __builtin_clzll(__ballot((int)(threadIdx.x & 63) < batch && before <= t));
    int row = 0;
    for (int hi = batch; hi - row > 1;) {
      const int mid = (row + hi) >> 1;
      if (pre[mid] <= t) row = mid; else hi = mid;
    }
    return row;
  }
};

// every thread of the work-group calls it
template <int THREADS>
__device__ __forceinline__ Rows scan_rows(const DecArgs& a, int* lds, int* wsum) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, batch = a.c.batch;
  Rows r;
  r.pre = lds;
  r.small = batch <= 64;
  if (r.small) {
    r.tokens = lane < batch ? row_len(a, lane) : 0;
    const int x = RowTiles(r.tokens, a.window, a.sinks).count;
    const int y = scan64(x);
    r.before = y - x;
    r.total = __builtin_amdgcn_readlane(y, 63);
    return r;
  }
  r.before = r.tokens = 0;
  int base = 0;
  for (int b0 = 0; b0 < batch; b0 += THREADS) {
    const int b = b0 + tid;
    const int x = scan64(RowTiles(b < batch ? row_len(a, b) : 0, a.window, a.sinks).count);
    if (lane == 63) wsum[wave] = x;
    __syncthreads();
    int before = base, all = base;
    for (int w = 0; w < THREADS / 64; ++w) {
      if (w < wave) before += wsum[w];
      all += wsum[w];
    }
    if (b < batch) r.pre[b + 1] = before + x;
    base = all;
    __syncthreads();
  }
  if (tid == 0) r.pre[0] = 0;
  __syncthreads();
  r.total = base;
  return r;
}

// How the rows' tiles are shared out.  `per` tiles a work-group over all rows laid end to end is even, but a
// work-group that ends a row and begins another pays for two prologues and joins (3 to 5 us).  So work-groups of
// one row each, its last one shorter, are taken where they fit with up to 3 more tiles (of 0.65 us) a work-group: 16
// rows x 4 heads of 1500 tokens 16.1 us, end to end 18.4; of 5000 tokens 34.6 and 36.4; but 24 rows of 1500 tokens,
// with 6 more tiles, 23.7 and 22.4.
struct Share {
  int per, parts;  // parts, lane b: those of the rows before row b
  bool by_row;
  __device__ __forceinline__ Share(const DecArgs& a, const Rows& rows) {
    per = max((rows.total + a.groups - 1) / a.groups, a.min_tiles);
    parts = 0;
    by_row = false;
    if (!rows.small || a.solo) return;
    const int lane = threadIdx.x & 63, count = lane < a.c.batch ? RowTiles(rows.tokens, a.window, a.sinks).count : 0;
#pragma unroll 1
    for (int k = 0; k < 4; ++k) {
      const int some = per + k, x = (count + some - 1) / some, y = scan64(x);
      if (__builtin_amdgcn_readlane(y, 63) > a.groups) continue;
      per = some;
      parts = y - x;
      by_row = true;
      return;
    }
  }
};

__device__ __forceinline__ float log_of(float M, float L) {
  return M == kNegInf ? (L > 0.f ? __builtin_nanf("") : __builtin_inff()) : M + __builtin_amdgcn_logf(L);
}
__device__ __forceinline__ float half_of(uint32_t w, int up) {
  return (float)__builtin_bit_cast(half_t, (uint16_t)(up ? w >> 16 : w));
}

typedef const __attribute__((address_space(4))) int32_t* const_i32;

// K rows of a tile: token of matrix row i of half t: 8 (i / 4) + 4 t + i % 4.  V: tokens 8 g .. 8 g + 7,
// channels 8 c .. 8 c + 7.  INT8 K comes by 16 channels a lane: matrix step kk holds channels 64 (kk / 2) + 16 g +
// 8 (kk % 2) ..; groups of 32 then lie in half of the lane groups, and each step is made twice, with Q zero in
// the other half (8 bytes a lane would put a step into one group, but read at 4.0 TB/s where 16 reach 5.7).
template <bool I8>
struct Tile;
template <>
struct Tile<false> {
  u32x4 k[2][4], v[8];
};
template <>
struct Tile<true> {
  u32x2 k[2][4], v[8];
  u32x4 ks[4], vs[4];
};

template <class T, bool I8, int GS, bool WT, int WAVES>
__global__ __launch_bounds__(WAVES * 64, 2) void paged_decode_kernel(DecArgs a) {
  using M = typename std::conditional<I8, TF16, T>::type;  // the matrix instructions' type
  constexpr int G = I8 ? 128 / GS : 1;
  extern __shared__ char lds[];
  __shared__ int wsum[WAVES];
  __shared__ float2 wml[WAVES][kHeads];
  float* const wacc = (float*)lds;                     // [4][32][64]
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int h = blockIdx.y, rep = a.rep;
  const PagedCache& pc = a.c;

  const Rows rows = scan_rows<WAVES * 64>(a, (int*)(lds + 4 * 32 * 64 * 4), wsum);
  const int total = rows.total;
  const Share share(a, rows);
  if ((WT || !a.solo) && blockIdx.x == 0 && h == 0) {
    if (rows.small) {
      if (tid < pc.batch) {
        a.pre[tid] = rows.before;
        a.pre[pc.batch + 2 + tid] = share.parts;
      }
    } else {
      for (int b = tid; b < pc.batch; b += WAVES * 64) a.pre[b] = rows.pre[b];
    }
    if (tid == 0) {
      a.pre[pc.batch] = total;
      a.pre[pc.batch + 1] = share.by_row ? -share.per : share.per;
    }
  }
  // rows that see nothing
  for (int b = blockIdx.x; b < pc.batch; b += gridDim.x)
    if (rows.end(b, pc.batch) == rows.start(b))
      for (int i = tid; i < rep * 64; i += WAVES * 64)
        ((uint32_t*)a.out)[((int64_t)b * a.q_heads + h * rep) * 64 + i] = 0;

  int t, t1, row = blockIdx.x;
  if (a.solo) {
    t = rows.start(row);
    t1 = rows.end(row, pc.batch);
  } else if (share.by_row) {  // the last row whose parts begin here or before; those before the first row with any are 0
    row = 63 - __builtin_clzll(__ballot(lane < pc.batch && share.parts <= (int)blockIdx.x));
    t = rows.start(row) + ((int)blockIdx.x - __builtin_amdgcn_readlane(share.parts, row)) * share.per;
    t1 = min(t + share.per, rows.end(row, pc.batch));
  } else {
    t = (int)min((int64_t)blockIdx.x * share.per, (int64_t)total);
    t1 = (int)min((int64_t)t + share.per, (int64_t)total);
    if (t < t1) row = rows.of(t, pc.batch);
  }
  if (t >= t1) return;

  const uint8_t* const kh = pc.k + h * pc.ksh;
  const uint8_t* const vh = pc.v + h * pc.vsh;
  const int t0 = t;
  for (; t < t1; ++row) {
    row = __builtin_amdgcn_readfirstlane(row);
    const int rs = __builtin_amdgcn_readfirstlane(rows.start(row)), re = __builtin_amdgcn_readfirstlane(rows.end(row, pc.batch));
    if (re == rs) continue;
    const int end = min(t1, re);
    const int n = __builtin_amdgcn_readfirstlane(rows.length(a, row));
    const RowTiles rt(n, a.window, a.sinks);
    const const_i32 tab = (const_i32)(pc.table + row * pc.table_stride);

    // Q^T: head c, channels of this lane's k-slots
    u32x4 q[4];
    float scale = a.sm;
    {
      const int head = h * rep + min(c, rep - 1);
      const uint16_t* qp = a.q + row * a.qsb + head * a.qsh;
      if (a.inv_tau) scale *= a.inv_tau[head];
#pragma unroll
      for (int kk = 0; kk < 4; ++kk)
        q[kk] = *(const u32x4*)(qp + (I8 ? 64 * (kk >> 1) + 16 * g + 8 * (kk & 1) : 32 * kk + 8 * g));
    }
    float m = kNegInf, l = 0.f;
    float4v acc[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] = float4v{0, 0, 0, 0};
    bool any = false;

    // A tile's place: its first token, its pages, this lane's rows and scales in them.  The page numbers are
    // fetched a tile ahead of that, and K and V of a tile while the tile before it is worked on: each operand's
    // registers are loaded again as soon as its products are done.
    struct Place {
      int tok;
      bool full, bad;  // every token of the tile is seen; the page of this lane's V block is not there
      const uint8_t *k, *v, *ks, *vs;
    };
    const int i_end = end - rs;
    auto page_at = [&](int i, int which) {  // of a tile of 32 slots: in one page, or in two of 16
      const int idx = (rt.token(min(i, i_end - 1)) >> pc.lg) + which;
      return idx < pc.max_pages ? tab[idx] : -1;
    };
    auto place = [&](int i, int p0, int p1, bool there) {
      Place w;
      w.tok = __builtin_amdgcn_readfirstlane(rt.token(i));
      if (pc.lg != 4) p1 = p0;
      const bool bad0 = (uint32_t)p0 >= (uint32_t)pc.num_pages, bad1 = (uint32_t)p1 >= (uint32_t)pc.num_pages;
      w.full = !bad0 && !bad1 && w.tok + kTile <= n && (w.tok >= rt.lo || w.tok + kTile <= rt.sink_end);
      if (bad0) p0 = 0;  // read, and masked: page 0 is there
      if (bad1) p1 = 0;
      const int bk = c >> 2;  // this lane's K block of 8 tokens; its V block is g
      int pk = bk >= 2 ? p1 : p0, pv = g >= 2 ? p1 : p0;
      int ko = (w.tok + 8 * bk + (c & 3)) & pc.page_mask, vo = (w.tok + 8 * g) & pc.page_mask;
      if (!there) pk = pv = ko = vo = 0;  // the same few lines for all lanes
      w.bad = g >= 2 ? bad1 : bad0;
      w.k = kh + pk * pc.ksp + (uint32_t)ko * (uint32_t)pc.kst;
      w.v = vh + pv * pc.vsp + (uint32_t)vo * (uint32_t)pc.vst;
      if constexpr (I8) {  // scales of tokens 8 g .. 8 g + 7: [8][G] fp16, dense
        w.ks = pc.ks + h * pc.kssh + pv * pc.kssp + vo * (2 * G);
        w.vs = pc.vs + h * pc.vssh + pv * pc.vssp + vo * (2 * G);
      }
      return w;
    };
    Tile<I8> x;
    auto load_k = [&](const Place& w) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const uint8_t* kr = w.k + u * 4 * pc.kst;
        if constexpr (!I8) {
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) x.k[u][kk] = ld_stream<u32x4>(kr + 64 * kk + 16 * g);
        } else {
#pragma unroll
          for (int kk = 0; kk < 4; kk += 2) {
            const u32x4 y = ld_stream<u32x4>(kr + 32 * kk + 16 * g);
            x.k[u][kk] = u32x2{y[0], y[1]};
            x.k[u][kk + 1] = u32x2{y[2], y[3]};
          }
        }
      }
      if constexpr (I8)
#pragma unroll
        for (int j = 0; j < G; ++j) x.ks[j] = *(const u32x4*)(w.ks + 16 * j);
    };
    auto load_v = [&](const Place& w) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if constexpr (!I8) x.v[j] = ld_stream<u32x4>(w.v + j * pc.vst + 16 * c);
        else x.v[j] = ld_stream<u32x2>(w.v + j * pc.vst + 8 * c);
      }
      if constexpr (I8)
#pragma unroll
        for (int j = 0; j < G; ++j) x.vs[j] = *(const u32x4*)(w.vs + 16 * j);
    };
    int i = t - rs + wave;
    Place w{};
    int n0 = -1, n1 = -1;  // pages of the tile after this
    if (i < i_end) {
      w = place(i, page_at(i, 0), page_at(i, 1), true);
      load_k(w);
      __builtin_amdgcn_sched_barrier(0);  // in the loop's order: what waits for K must not wait for V
      load_v(w);
      n0 = page_at(i + WAVES, 0);
      n1 = page_at(i + WAVES, 1);
    }
    // Q is waited for here, behind the first tile's loads
    if constexpr (I8 && std::is_same<T, TB16>::value) {
      // bf16 values in fp16, the head's largest scaled to [2^14, 2^15) by a power of two: those down to 2^-31 of that power
      // are exact, and smaller ones off by at most 2^-39 of it (fp16's least step is 2^-24)
      float top = 0.f;
#pragma unroll
      for (int kk = 0; kk < 4; ++kk)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          top = fmaxf(top, fmaxf(fabsf(TB16::to_f((uint16_t)q[kk][j])), fabsf(TB16::to_f((uint16_t)(q[kk][j] >> 16)))));
      top = wave_max_xor_groups(top);
      int ex = (int)(__builtin_bit_cast(uint32_t, top) >> 23) - 127;
      ex = ex == 128 || ex == -127 ? 0 : max(ex - 14, -126);  // Inf or NaN stays what it is; zero or a subnormal is 0
      const float f = ldexpf(1.f, -ex);
      scale = ldexpf(scale, ex);
#pragma unroll
      for (int kk = 0; kk < 4; ++kk)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          q[kk][j] = TF16::pack(TB16::to_f((uint16_t)q[kk][j]) * f, TB16::to_f((uint16_t)(q[kk][j] >> 16)) * f);
    }
#pragma unroll
    for (int kk = 0; kk < 4; ++kk)
#pragma unroll
      for (int j = 0; j < 4; ++j) q[kk][j] = c < rep ? q[kk][j] : 0u;
    u32x4 qu[4];  // groups of 32: q for the upper lane groups, q for the lower
    if constexpr (I8 && GS == 32) {
#pragma unroll
      for (int kk = 0; kk < 4; ++kk)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          qu[kk][j] = g >= 2 ? q[kk][j] : 0u;
          q[kk][j] = g < 2 ? q[kk][j] : 0u;
        }
    }
    for (; i < i_end; i += WAVES) {
      // Past the end: page 0's first rows, which nothing uses.  A condition on the loads would have the loop wait for
      // all of them to merge their two values.
      const Place next = place(min(i + WAVES, i_end - 1), n0, n1, i + WAVES < i_end);
      n0 = page_at(i + 2 * WAVES, 0);
      n1 = page_at(i + 2 * WAVES, 1);
      const int tok = w.tok;

      // scores of head c at tokens tok + 8 g + j
      float s[8];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        if constexpr (!I8) {
          float4v d = {0, 0, 0, 0};
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) d = M::mfma16(x.k[u][kk], q[kk], d);
#pragma unroll
          for (int r = 0; r < 4; ++r) s[4 * u + r] = d[r] * scale;
        } else {
          float4v d[G];
#pragma unroll
          for (int j = 0; j < G; ++j) d[j] = float4v{0, 0, 0, 0};
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) {
            const uint32_t lo = x.k[u][kk][0] ^ 0x80808080u, hi = x.k[u][kk][1] ^ 0x80808080u;
            const u32x4 ka = {code_pair(lo, 0x04010400u), code_pair(lo, 0x04030402u), code_pair(hi, 0x04010400u),
                              code_pair(hi, 0x04030402u)};
            if constexpr (GS == 32) {
              d[kk & 2] = M::mfma16(ka, q[kk], d[kk & 2]);
              d[(kk & 2) + 1] = M::mfma16(ka, qu[kk], d[(kk & 2) + 1]);
            } else {
              d[kk * G / 4] = M::mfma16(ka, q[kk], d[kk * G / 4]);
            }
          }
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            float v = 0.f;
#pragma unroll
            for (int j = 0; j < G; ++j) {
              const int at = (4 * u + r) * G + j;  // fp16 scale of token 4 u + r, group j
              const uint32_t w = x.ks[at / 8][at / 2 % 4];
              v = fmaf(d[j][r], half_of(w, at & 1), v);
            }
            s[4 * u + r] = v * scale;
          }
        }
      }
      load_k(next);
      uint32_t seen = 0xFF;  // bit j: token tok + 8 g + j
      if (w.full) {
        any = true;
      } else {
        seen = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int tj = tok + 8 * g + j;
          const bool vis = !w.bad && tj < n && (tj >= rt.lo || tj < rt.sink_end);
          seen |= (uint32_t)vis << j;
          if (!vis) s[j] = kNegInf;
        }
        any |= __any(seen != 0);
      }
      if constexpr (WT) {
        if (c < rep) {
          float* so = a.scores + ((h * a.tiles_cap + rs + i) * rep + c) * kTile + 8 * g;
          *(float4v*)so = float4v{s[0], s[1], s[2], s[3]};
          *(float4v*)(so + 4) = float4v{s[4], s[5], s[6], s[7]};
        }
      }
      // the maximum follows only where a score passes the largest before it by 2^6: P stays below 64 (2^15 in fp16),
      // and the accumulators are seldom rescaled
      float mx = max8f(s[0], s[1], s[2], s[3], s[4], s[5], s[6], s[7]);
      if (__any(mx > m + (6.f + M::kUp))) {
        mx = fmaxf(wave_max_xor_groups(mx) - M::kUp, m);
        const float f = part_of(m, mx);
        l *= f;
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] *= f;
        m = mx;
      }
      const float mm = shift_of(m);
      float p[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        p[j] = fast_exp2(s[j] - mm);
        l += p[j];
      }
      // P in 16 bits: the products' rounding averages out over the tokens; the sum takes the unrounded
      const u32x4 pb = {M::pack(p[0], p[1]), M::pack(p[2], p[3]), M::pack(p[4], p[5]), M::pack(p[6], p[7])};
      __builtin_amdgcn_sched_barrier(0);  // nothing that waits for V above
      if constexpr (!I8) {
        if (!w.full)  // what is masked may hold anything: 0 x NaN is no 0
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (!(seen >> j & 1)) x.v[j] = u32x4{0, 0, 0, 0};
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          u32x4 va;
#pragma unroll
          for (int j = 0; j < 4; ++j)
            va[j] = perm_b32(x.v[2 * j + 1][e >> 1], x.v[2 * j][e >> 1], e & 1 ? 0x07060302u : 0x05040100u);
          acc[e] = M::mfma16(va, pb, acc[e]);
        }
      } else {
        // V's scale of this lane's channel group, tokens in pairs
        uint32_t vsc[4];
        const uint32_t sel = ((8 * c / GS) & 1) ? 0x07060302u : 0x05040100u;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if constexpr (G == 1) {
            vsc[j] = x.vs[0][j];
          } else if constexpr (G == 2) {
            vsc[j] = perm_b32(x.vs[(2 * j + 1) / 4][(2 * j + 1) % 4], x.vs[2 * j / 4][2 * j % 4], sel);
          } else {
            const bool up = c >= 8;
            vsc[j] = perm_b32(up ? x.vs[j][3] : x.vs[j][2], up ? x.vs[j][1] : x.vs[j][0], sel);
          }
        }
        if (!w.full)  // a masked code is finite, its scale may not be
#pragma unroll
          for (int j = 0; j < 4; ++j)
            vsc[j] &= (seen >> 2 * j & 1 ? 0xFFFFu : 0u) | (seen >> (2 * j + 1) & 1 ? 0xFFFF0000u : 0u);
#pragma unroll
        for (int e4 = 0; e4 < 2; ++e4) {
          u32x4 va[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t w0 = x.v[2 * j][e4] ^ 0x80808080u, w1 = x.v[2 * j + 1][e4] ^ 0x80808080u;
            const uint32_t a01 = perm_b32(w1, w0, 0x05010400u), a23 = perm_b32(w1, w0, 0x07030602u);
            // the value code x scale in fp16, as the framework's dequantizers have it
            va[0][j] = as_u32(as_h2(code_pair(a01, 0x04010400u)) * as_h2(vsc[j]));
            va[1][j] = as_u32(as_h2(code_pair(a01, 0x04030402u)) * as_h2(vsc[j]));
            va[2][j] = as_u32(as_h2(code_pair(a23, 0x04010400u)) * as_h2(vsc[j]));
            va[3][j] = as_u32(as_h2(code_pair(a23, 0x04030402u)) * as_h2(vsc[j]));
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[4 * e4 + e] = M::mfma16(va[e], pb, acc[4 * e4 + e]);
        }
      }
      load_v(next);
      w = next;
    }

    // join the waves: acc[e][r] is channel 32 g + 8 r + e of head c
    l = wave_sum_xor_groups(l);
    if (m == kNegInf && l == l) l = any ? 1.f : 0.f;
    if constexpr (WAVES == 8) {  // the upper four first, into the lower four
      if (wave >= 4) {
        if (g == 0) wml[wave][c] = float2{m, l};
#pragma unroll
        for (int e = 0; e < 8; ++e)
#pragma unroll
          for (int r = 0; r < 4; ++r) wacc[((wave - 4) * 32 + r * 8 + e) * 64 + lane] = acc[e][r];
      }
      __syncthreads();
      if (wave < 4) {
        const float2 o = wml[wave + 4][c];
        const float M2 = fmaxf(m, o.x), f0 = part_of(m, M2), f1 = part_of(o.x, M2);
        l = sum_in(m, l, M2) + sum_in(o.x, o.y, M2);
        m = M2;
#pragma unroll
        for (int e = 0; e < 8; ++e)
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[e][r] = acc[e][r] * f0 + wacc[(wave * 32 + r * 8 + e) * 64 + lane] * f1;
      }
      __syncthreads();
    }
    if (wave < 4) {
      if (g == 0) wml[wave][c] = float2{m, l};
#pragma unroll
      for (int e = 0; e < 8; ++e)
#pragma unroll
        for (int r = 0; r < 4; ++r) wacc[(wave * 32 + r * 8 + e) * 64 + lane] = acc[e][r];
    }
    __syncthreads();
    {
      constexpr int NI = 32 / WAVES;  // of the 32 values of a lane, those of this wave
      float mw[4], Mx = kNegInf, L = 0.f, o[NI];
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        mw[w] = wml[w][c].x;
        Mx = fmaxf(Mx, mw[w]);
      }
#pragma unroll
      for (int w = 0; w < 4; ++w) L += sum_in(mw[w], wml[w][c].y, Mx);
#pragma unroll
      for (int k = 0; k < NI; ++k) o[k] = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float f = part_of(mw[w], Mx);
#pragma unroll
        for (int k = 0; k < NI; ++k) o[k] = fmaf(f, wacc[(w * 32 + wave * NI + k) * 64 + lane], o[k]);
      }
      const int ch = 32 * g + wave * NI;  // value k: channel ch + k (r = wave NI / 8)
      const bool whole = t == rs && end == re;
      if (c < rep) {
        if (whole) {
          const float inv = inverse_of(Mx, L);
          const int64_t oh = (int64_t)row * a.q_heads + h * rep + c;
          uint32_t w[NI / 2];
#pragma unroll
          for (int k = 0; k < NI / 2; ++k) w[k] = T::pack(o[2 * k] * inv, o[2 * k + 1] * inv);
          if constexpr (NI == 8) *(u32x4*)(a.out + oh * 128 + ch) = u32x4{w[0], w[1], w[2], w[3]};
          else *(u32x2*)(a.out + oh * 128 + ch) = u32x2{w[0], w[1]};
          if (WT && g == 0 && wave == 0) a.lse[oh] = log_of(Mx, L);
        } else {
          const int64_t slot = (((int64_t)h * a.groups + blockIdx.x) * 2 + (t == t0 ? 0 : 1)) * rep + c;
          if (g == 0 && wave == 0) a.ml[slot] = float2{Mx, L};
#pragma unroll
          for (int k = 0; k < NI; k += 4) *(float4v*)(a.acc + slot * 128 + ch + k) = float4v{o[k], o[k + 1], o[k + 2], o[k + 3]};
        }
      }
    }
    __syncthreads();
    t = end;
  }
}

// A row's part of the shared rows' parts: work-groups first .. last, the slot of each.
struct Parts {
  int first, last, start, per;
  int64_t base;
  __device__ __forceinline__ Parts(const DecArgs& a, int h, int b) {
    start = a.pre[b];
    const int end = a.pre[b + 1];
    per = a.pre[a.c.batch + 1];
    base = (int64_t)h * a.groups * 2;
    if (per < 0) {  // work-groups of one row: always their first part
      first = a.pre[a.c.batch + 2 + b];
      last = end > start ? first + (end - 1 - start) / -per : first;
      start = per = 0;
    } else {
      first = start / per;
      last = end > start ? (end - 1) / per : first;
    }
  }
  __device__ __forceinline__ bool whole() const { return first == last; }  // written by its work-group
  __device__ __forceinline__ int64_t slot(int w) const { return base + 2 * w + ((int64_t)w * per >= start ? 0 : 1); }
};

// Joins a row that several work-groups share: a work-group a (row, query head), 16 parts at a time, 8
// channels a thread.
template <class T>
__device__ __forceinline__ void join_row(const DecArgs& a, int r, int h, int b) {
  __shared__ float part[16][16][10];  // 8 values, maximum, sum
  const int rep = a.rep, cc = threadIdx.x & 15, sl = threadIdx.x >> 4;
  const Parts parts(a, h, b);
  if (parts.whole()) return;
  float m = kNegInf, l = 0.f, o[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) o[k] = 0.f;
  for (int w = parts.first + sl; w <= parts.last; w += 16) {
    const int64_t slot = parts.slot(w) * rep + r;
    const float2 p = a.ml[slot];
    const float4v x = *(const float4v*)(a.acc + slot * 128 + cc * 8), y = *(const float4v*)(a.acc + slot * 128 + cc * 8 + 4);
    const float M = fmaxf(m, p.x), f0 = part_of(m, M), f1 = part_of(p.x, M);
    l = sum_in(m, l, M) + sum_in(p.x, p.y, M);
    m = M;
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
  float M = kNegInf, L = 0.f, v = 0.f;
#pragma unroll
  for (int w = 0; w < 16; ++w) M = fmaxf(M, part[w][pc][8]);
#pragma unroll
  for (int w = 0; w < 16; ++w) {
    L += sum_in(part[w][pc][8], part[w][pc][9], M);
    v = fmaf(part_of(part[w][pc][8], M), part[w][pc][pk], v);
  }
  a.out[((int64_t)b * a.q_heads + h * rep + r) * 128 + ch] = (uint16_t)T::pack(v * inverse_of(M, L), 0.f);
}

// weights[b,g,t] += sum_h p_h(t) from the stored scores and the rows' denominators: eight tiles a work-group, half
// a wave each
__device__ __forceinline__ void add_weights(const DecArgs& a, int chunk, int h, int b) {
  __shared__ float lse[kHeads];
  const int rep = a.rep, n = row_len(a, b);
  const RowTiles rt(n, a.window, a.sinks);
  if (chunk * 8 >= rt.count) return;
  const int r = threadIdx.x >> 4, sl = threadIdx.x & 15;
  bool whole = a.solo;
  if (!whole) {
    const Parts parts(a, h, b);
    whole = parts.whole();
    if (!whole && r < rep) {
      float m = kNegInf, l = 0.f;
      for (int w = parts.first + sl; w <= parts.last; w += 16) {
        const float2 p = a.ml[parts.slot(w) * rep + r];
        const float M = fmaxf(m, p.x);
        l = sum_in(m, l, M) + sum_in(p.x, p.y, M);
        m = M;
      }
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) {
        const float m2 = __shfl_xor(m, o, 16), l2 = __shfl_xor(l, o, 16), M = fmaxf(m, m2);
        l = sum_in(m, l, M) + sum_in(m2, l2, M);
        m = M;
      }
      if (sl == 0) lse[r] = log_of(m, l);
    }
  }
  if (whole && sl == 0 && r < rep) lse[r] = a.lse[(int64_t)b * a.q_heads + h * rep + r];
  __syncthreads();
  const int i = chunk * 8 + (threadIdx.x >> 5), u = threadIdx.x & 31;
  if (i >= rt.count) return;
  const int tok = rt.token(i) + u;
  if (tok >= n) return;
  const float* s = a.scores + (h * a.tiles_cap + a.pre[b] + i) * (int64_t)rep * kTile + u;
  float* w = a.weights + b * a.wsb + h * a.wsh + tok;
  float p = 0.f;
  for (int k = 0; k < rep; ++k) p += fast_exp2(s[k * kTile] - lse[k]);
  if (p != p) {  // a head's softmax is none: that is so for the tokens it sees, and adds nothing to the others of their tile
    const int32_t page = a.c.table[b * a.c.table_stride + (tok >> a.c.lg)];
    if ((uint32_t)page >= (uint32_t)a.c.num_pages || (tok < rt.lo && tok >= rt.sink_end)) return;
  }
  *w += p;
}

// What is left when every part is there, in one launch: the first `joins` work-groups of a (KV head, row) join its
// query heads, the others add the weights.
template <class T, bool WT>
__global__ __launch_bounds__(256) void paged_finish_kernel(DecArgs a, int joins) {
  if ((int)blockIdx.x < joins) join_row<T>(a, blockIdx.x, blockIdx.y, blockIdx.z);
  else if constexpr (WT) add_weights(a, (int)blockIdx.x - joins, blockIdx.y, blockIdx.z);
}

// ---------------------------------------------------------------- host

// Measured on fp16 pages of 16 tokens, 7 query heads a KV head, 4 KV heads, us a call in a graph:
// Work-groups of a launch, one of 4 waves a CU: 64 rows of 2048 tokens 49.3 (512: 52.2, 768: 57.2, 192: 63), 16 of
// 8192 50.4 (51.2, 55.2, 59.4), 1 of 32768 19.8 (22.1, 22.2, 21.2).  8 waves in each: 50.2, 51.2, 20.5.
constexpr int kTargetGroups = 256;
// Least tiles of a work-group.  1 row of 1000 tokens 9.0 (4: 9.6, 8: 10.3, 16: 13), 4 of 700 9.7 (4: 12.6).
constexpr int kMinTiles = 2;
// Rows of at most these tiles are not split: one launch and no workspace.  At 512 tokens 1 row takes 10.0 us and 4
// rows 12.5, split 9.1 and 9.8; but called one by one, where launches count, 10.0 and 13.6.  At 1000 tokens split
// rows win both ways: 9.0 and 9.9 for 17.5 and 19.7.
constexpr int kSoloTiles = 20;

struct Plan {
  int64_t max_tiles;  // of a row
  int groups;
  bool solo;
  int64_t pre, ml, acc, lse, scores, bytes;  // workspace offsets
};

Plan plan_of(const kvq_paged_decode_params& p, bool weights) {
  Plan w{};
  const int64_t cap = (int64_t)p.cache.max_pages * p.cache.page_size;
  const int64_t all = (cap + kTile - 1) / kTile;
  w.max_tiles = all;
  if (p.window > 0) {
    const int64_t sinks = p.sinks > 0 ? p.sinks : 0;
    const int64_t some = (sinks + kTile - 1) / kTile + ((int64_t)p.window + kTile - 1) / kTile + 1;
    if (some < all) w.max_tiles = some;
  }
  const int64_t B = p.cache.batch, H = p.cache.kv_heads, rep = p.q_heads / p.cache.kv_heads;
  w.solo = w.max_tiles <= kSoloTiles;
  const int64_t most = (B * w.max_tiles + kMinTiles - 1) / kMinTiles;
  int64_t g = (kTargetGroups + H - 1) / H;
  if (g > most) g = most;
  w.groups = w.solo ? (int)B : (int)(g > 1 ? g : 1);
  auto take = [&](int64_t bytes) {
    const int64_t at = w.bytes;
    w.bytes += (bytes + 63) / 64 * 64;
    return at;
  };
  if (!w.solo || weights) w.pre = take(4 * (2 * B + 2));
  if (!w.solo) {
    w.ml = take(8 * H * w.groups * 2 * rep);
    w.acc = take(512 * H * w.groups * 2 * rep);
  }
  if (weights) {
    w.lse = take(4 * B * p.q_heads);
    w.scores = take(4 * H * B * w.max_tiles * rep * kTile);
  }
  return w;
}

int check(const kvq_paged_decode_params* p, PagedCache& c) {
  if (!p) return fail(KVQ_ERR_INVALID, "paged decode: NULL params");
  const int rc = paged_cache(p->cache, c);
  if (rc) return rc;
  if (p->q_type != KVQ_PAGED_F16 && p->q_type != KVQ_PAGED_BF16) return fail(KVQ_ERR_INVALID, "paged decode: unknown q_type");
  if (p->cache.format != KVQ_PAGED_INT8 && p->cache.format != p->q_type)
    return fail(KVQ_ERR_INVALID, "paged decode: the pages' type is another than q's");
  if (p->q_heads <= 0 || p->q_heads % p->cache.kv_heads) return fail(KVQ_ERR_INVALID, "paged decode: q_heads must be a multiple of kv_heads");
  if (p->q_heads / p->cache.kv_heads > kHeads) return fail(KVQ_ERR_UNSUPPORTED, "paged decode: more than 16 query heads a KV head");
  if (p->cache.batch > kMaxRows) return fail(KVQ_ERR_UNSUPPORTED, "paged decode: more than 4096 rows");
  if (p->cache.kv_heads > 65535) return fail(KVQ_ERR_UNSUPPORTED, "paged decode: too many heads");
  if (((int64_t)p->cache.max_pages * p->cache.page_size / kTile + 1) * p->cache.batch > (1 << 28))
    return fail(KVQ_ERR_UNSUPPORTED, "paged decode: too many token slots in a batch");
  return KVQ_OK;
}

template <class T, bool I8, int GS, bool WT>
int launch(const DecArgs& a, const Plan& w, hipStream_t st) {
  const int H = a.c.kv_heads, B = a.c.batch;
  const size_t lds = 4 * 32 * 64 * 4 + (B > 64 ? (size_t)(B + 1) * 4 : 0);  // at most 49 KB
  const dim3 grid((unsigned)w.groups, (unsigned)H);
  if (w.solo) hipLaunchKernelGGL((paged_decode_kernel<T, I8, GS, WT, 8>), grid, dim3(512), lds, st, a);
  else hipLaunchKernelGGL((paged_decode_kernel<T, I8, GS, WT, 4>), grid, dim3(256), lds, st, a);
  int rc = launched();
  if (rc) return rc;
  const int joins = w.solo ? 0 : a.rep;
  const int64_t chunks = WT ? (w.max_tiles + 7) / 8 : 0;
  if (joins + chunks > 0) {
    hipLaunchKernelGGL((paged_finish_kernel<T, WT>), dim3((unsigned)(joins + chunks), (unsigned)H, (unsigned)B), dim3(256), 0, st, a, joins);
    rc = launched();
  }
  return rc;
}

int decode(const kvq_paged_decode_params* p, hipStream_t st) {
  DecArgs a{};
  int rc = check(p, a.c);
  if (rc) return rc;
  const int B = a.c.batch;
  if (B == 0) return KVQ_OK;
  if (!p->q || !p->out || !p->context_lens) return fail(KVQ_ERR_INVALID, "paged decode: NULL pointer");
  if (((uintptr_t)p->q | (uintptr_t)p->out) % 16 || (p->q_stride_b | p->q_stride_h) % 8)
    return fail(KVQ_ERR_INVALID, "paged decode: q rows must be 16-byte aligned");
  const Plan w = plan_of(*p, p->weights != nullptr);
  if (w.bytes && (!p->workspace || p->workspace_bytes < w.bytes || (uintptr_t)p->workspace % 16))
    return fail(KVQ_ERR_INVALID, "paged decode: workspace too small or not 16-byte aligned");
  // without pages every row sees nothing: no column of the table is read
  if (a.c.num_pages == 0) a.c.max_pages = 0;
  a.q = (const uint16_t*)p->q; a.qsb = p->q_stride_b; a.qsh = p->q_stride_h;
  a.out = (uint16_t*)p->out;
  a.lens = p->context_lens;
  a.inv_tau = p->inv_tau;
  a.sm = p->sm_scale * kLog2e;
  a.window = p->window; a.sinks = p->sinks;
  a.q_heads = p->q_heads; a.rep = p->q_heads / a.c.kv_heads;
  a.groups = w.groups;
  a.min_tiles = kMinTiles;
  a.solo = w.solo;
  uint8_t* ws = (uint8_t*)p->workspace;
  a.pre = (int32_t*)(ws + w.pre);
  a.ml = (float2*)(ws + w.ml); a.acc = (float*)(ws + w.acc);
  a.lse = (float*)(ws + w.lse); a.scores = (float*)(ws + w.scores);
  a.tiles_cap = (int64_t)B * w.max_tiles;
  a.weights = p->weights; a.wsb = p->w_stride_b; a.wsh = p->w_stride_h;
  const bool b16 = p->q_type == KVQ_PAGED_BF16, wt = p->weights != nullptr;
  const int gs = p->cache.format == KVQ_PAGED_INT8 ? p->cache.group_size : 0;
#define KVQ_DEC(I8, GS)                                                                        \
  return b16 ? (wt ? launch<TB16, I8, GS, true>(a, w, st) : launch<TB16, I8, GS, false>(a, w, st)) \
             : (wt ? launch<TF16, I8, GS, true>(a, w, st) : launch<TF16, I8, GS, false>(a, w, st))
  if (gs == 0) KVQ_DEC(false, 0);
  if (gs == 32) KVQ_DEC(true, 32);
  if (gs == 64) KVQ_DEC(true, 64);
  KVQ_DEC(true, 128);
#undef KVQ_DEC
}

}  // namespace
}  // namespace kvq

extern "C" int kvq_paged_decode(const kvq_paged_decode_params* p, kvq_stream_t stream) {
  return kvq::guarded([&] { return kvq::decode(p, reinterpret_cast<hipStream_t>(stream)); });
}

extern "C" int64_t kvq_paged_decode_workspace_bytes(const kvq_paged_decode_params* p) {
  kvq::PagedCache c;
  if (kvq::guarded([&] { return kvq::check(p, c); })) return 0;
  return kvq::plan_of(*p, p->weights != nullptr).bytes;
}
