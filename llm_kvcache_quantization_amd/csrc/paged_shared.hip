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
// What bounds it: with few tokens and columns a chain of latencies (plan, table, load, the tile's products and
// exponentials one after another: 1.1 + 0.7 + 0.6 + 2.3 us before the first tile, 1.5 a tile of 128 columns), else HBM
// with 16-bit pages (four prompts of up to 16384 tokens with 8 rows of 28 / 4 heads each, 94 MB: 22.8 us; 6.6 TB/s while the
// tiles run, 4.1 with start and end), and with INT8 pages the vector and matrix units in turn (39% and 14% of busy cycles; one
// prompt of 32768, 32 rows of 40 / 8 heads with up to 509 tokens of their own: 78 us, 274 TFLOP/s), two waves a SIMD being all
// that the registers allow.
// The join: 3.3 to 6 us.
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
  int2* map;             // {row, chunk} of the tails' work-groups, -1 for none, where there are more than 64 rows
  int32_t groups;        // work-groups of the tails of a KV head
  int32_t fill;          // work-groups that the tails of a KV head are shared out over (and one more a row, at most)
  int32_t prefix_slots;  // parts of the prefixes of a KV head; then those of the tails, [work-group][head]
  uint32_t tails;        // work-groups of tails, the launch's last
  int4* places;          // [batch] Tails
  int64_t slots;         // parts of a KV head
  float2* ml;            // [kv_heads][slots]
  float* acc;            // [kv_heads][slots][128]
};

// Least tiles of a tail's work-group: 16 rows with 700 tokens behind 8191 shared ones 18.8 us, with one tile 19.0, with six 21.7.
constexpr int kTailTiles = 3;

// The tiles of a row's own tokens lo .. hi - 1.
struct Tail {
  int lo, hi, first, count;
  bool shares;  // the row takes part in its group's prefix
  __device__ __forceinline__ Tail(const ShArgs& a, int len, int n) {
    const int64_t cap = (int64_t)a.c.max_pages << a.c.lg;
    hi = (int)min((int64_t)max(n, 0), cap);
    shares = hi >= len;
    lo = shares ? len : 0;
    first = lo / kBN;
    count = hi > lo ? (hi + kBN - 1) / kBN - first : 0;
  }
  // of `chunks` even runs of tiles, the i-th's first: first + count i / chunks, whose product may pass 32 bits
  __device__ __forceinline__ int begin(int i, int chunks) const {
    const uint32_t n = (uint32_t)chunks, whole = (uint32_t)count / n, rest = (uint32_t)count % n;
    return first + (int)(whole * (uint32_t)i + rest * (uint32_t)i / n);
  }
};

// Which row a tail's work-group is of, and which of its chunks; and, of each row, what the join needs: {first
// work-group, work-groups, whether it shares}.  The tiles of all rows are shared out evenly, whatever their lengths.  Up to 64
// rows are in a wave's lanes, and each work-group finds its own; those of more rows find it in a launch before this.
struct Tails {
  int row, chunk, chunks;
  __device__ __forceinline__ Tails(const ShArgs& a, int at, bool write) {
    const int B = a.c.batch;
    row = -1;
    if (a.map) {
      const const_i32 m = (const_i32)(a.map + at);
      row = m[0];
      chunk = m[1];
      if (row >= 0) chunks = ((const_i32)(a.places + row))[1];
      return;
    }
    const int lane = threadIdx.x & 63;
    int count = 0;
    bool shares = false;
    if (lane < B) {
      const Tail t(a, a.rows[lane].len, a.lens[lane]);
      count = t.count;
      shares = t.shares;
    }
    const int total = __builtin_amdgcn_readlane(scan64(count), 63);
    const int per = max((total + a.fill - 1) / a.fill, kTailTiles);
    const int mine = (count + per - 1) / per, before = scan64(mine) - mine;
    if (write && at == 0 && threadIdx.x < (uint32_t)B) a.places[lane] = {before, mine, shares, 0};
    const uint64_t here = __ballot(lane < B && before <= at && at < before + mine);
    if (!here) return;
    row = __builtin_ctzll(here);
    chunk = at - __builtin_amdgcn_readlane(before, row);
    chunks = __builtin_amdgcn_readlane(mine, row);
  }
};

// Tails of more than 64 rows: a work-group, a run of rows a thread.
__global__ __launch_bounds__(kThreads) void shared_places_kernel(ShArgs a) {
  __shared__ unsigned long long total;
  __shared__ int sums[kThreads / 64];
  const int B = a.c.batch, tid = threadIdx.x, per_thread = (B + kThreads - 1) / kThreads;
  const int b0 = min(tid * per_thread, B), b1 = min(b0 + per_thread, B);
  if (tid == 0) total = 0;
  __syncthreads();
  unsigned long long count = 0;
  for (int b = b0; b < b1; ++b) count += (unsigned long long)Tail(a, a.rows[b].len, a.lens[b]).count;
  atomicAdd(&total, count);
  __syncthreads();
  const int per = max((int)((total + (unsigned)a.fill - 1) / (unsigned)a.fill), kTailTiles);
  int mine = 0;
  for (int b = b0; b < b1; ++b) mine += (Tail(a, a.rows[b].len, a.lens[b]).count + per - 1) / per;
  const int upto = scan64(mine);
  if ((tid & 63) == 63) sums[tid >> 6] = upto;
  __syncthreads();
  int at = upto - mine, all = 0;
  for (int w = 0; w < kThreads / 64; ++w) {
    if (w < tid >> 6) at += sums[w];
    all += sums[w];
  }
  for (int b = b0; b < b1; ++b) {
    const Tail t(a, a.rows[b].len, a.lens[b]);
    const int n = (t.count + per - 1) / per;
    a.places[b] = {at, n, t.shares, 0};
    for (int i = 0; i < n; ++i) a.map[at + i] = {b, i};
    at += n;
  }
  for (int i = all + tid; i < a.groups; i += kThreads) a.map[i] = {-1, 0};
}

__device__ const u32x4 zero_row[16] = {};

// What a work-group reads: tiles of tokens lo .. hi - 1 of one row's pages, for one KV head.
struct Source {
  const uint8_t *k, *v, *ks, *vs;
  const_i32 table;
  int lo, hi;
  // every token of a tile is there and seen (ok: there())
  __device__ __forceinline__ bool whole(int key0, uint32_t ok) const { return ok == 15 && key0 >= lo && key0 + kBN <= hi; }
};

typedef int32_t Pages __attribute__((ext_vector_type(4)));  // of a tile's tokens, 16 each (a vector: registers, whatever picks from it)

__device__ __forceinline__ Pages pages_of(const PagedCache& c, const Source& s, int tile) {
  Pages p;
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int i = (tile * kBN + 16 * u) >> c.lg;
    p[u] = i < c.max_pages ? s.table[i] : -1;
  }
  return p;
}

// Bit u: the page of tokens 16 u .. is there.
__device__ __forceinline__ uint32_t there(const PagedCache& c, const Pages& p) {
  uint32_t ok = 0;
#pragma unroll
  for (int u = 0; u < 4; ++u) ok |= (uint32_t)((uint32_t)p[u] < (uint32_t)c.num_pages) << u;
  return ok;
}

// Where 16 consecutive tokens of a page begin, of one side.  All of it is scalar, and on a wave's way from tile to tile: page
// strides below 2^32 bytes (the host's check) take two instructions to multiply where 64 bits take five.
__device__ __forceinline__ const uint8_t* block_of(const PagedCache& c, const uint8_t* x, int64_t page_stride, int64_t row_stride, int32_t page, int token) {
  return x + (uint64_t)(uint32_t)page * (uint32_t)page_stride + (uint32_t)(token & c.page_mask) * (uint32_t)row_stride;
}

// A tile's rows from 16-bit pages straight into LDS.  A wave instruction loads four rows of 16; a lane takes the chunk
// that belongs at its place.
struct Direct {
  uint32_t k_off, v_off;
  int wave, row, chunk;
  __device__ __forceinline__ Direct(const PagedCache& c, int wave_) : wave(wave_) {
    const int lane = threadIdx.x & 63;
    row = 4 * wave + (lane >> 4);
    chunk = lane & 15;
    k_off = (uint32_t)row * (uint32_t)c.kst + (uint32_t)(chunk ^ row) * 16;
    v_off = (uint32_t)row * (uint32_t)c.vst + (uint32_t)(chunk ^ ((row & 3) << 2)) * 16;
  }
  template <bool ALL>
  __device__ __forceinline__ void load(const PagedCache& c, const Source& s, int key0, const Pages& p, uint32_t ok, LdsTile& kt,
                                       LdsTile& vt) const {
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int at = 16 * u + 4 * wave;  // the wave's first row
      const int32_t page = ALL || (ok >> u & 1) ? p[u] : 0;
      const uint8_t* kp = block_of(c, s.k, c.ksp, c.kst, page, key0 + 16 * u) + k_off;
      const uint8_t* vp = block_of(c, s.v, c.vsp, c.vst, page, key0 + 16 * u) + v_off;
      if constexpr (!ALL) {
        const int key = key0 + 16 * u + row;
        const bool there = (ok >> u & 1) && key >= s.lo && key < s.hi;
        kp = there ? kp : (const uint8_t*)(zero_row + chunk);
        vp = there ? vp : (const uint8_t*)(zero_row + chunk);
      }
      __builtin_amdgcn_global_load_lds((gptr)kp, (__attribute__((address_space(3))) void*)(&kt[at * 16]), 16, 0, 0);
      __builtin_amdgcn_global_load_lds((gptr)vp, (__attribute__((address_space(3))) void*)(&vt[at * 16]), 16, 0, 0);
    }
  }
  __device__ __forceinline__ void operator()(const PagedCache& c, const Source& s, int key0, const Pages& p, uint32_t ok, LdsTile& kt,
                                             LdsTile& vt) const {
    if (s.whole(key0, ok)) load<true>(c, s, key0, p, ok, kt, vt);
    else load<false>(c, s, key0, p, ok, kt, vt);
  }
};

// A tile of INT8 pages as it is, straight into LDS: K's codes [64][128]; V's with the scales of both sides.
typedef u32x4 KCodes[kBN * 8];
template <int G>
struct VCodes {
  u32x4 v[kBN * 8];
  // dwords as they lie in the pages, [pair of groups][token]; of one group, [pair of tokens]
  uint32_t ks[G == 1 ? 64 : kBN * G / 2], vs[G == 1 ? 64 : kBN * G / 2];  // at least a wave's load
};

// A thread's places in a tile of INT8 pages.  A wave instruction loads eight rows of 8 pieces of 16 codes, and a dword of
// scales a lane (a pair of a token's, or two tokens'); waves 0 and 1 take K's scales, 2 and 3 V's, a pair of groups each or
// the same twice.
template <int GS>
struct Coded {
  static constexpr int G = 128 / GS;
  uint32_t k_off, v_off;  // of the wave's rows from the first of their 16
  int wave, row, s_row;   // in the tile: the first piece's (the second's is 32 behind), the scale dword's
  uint32_t k_at, v_at;    // LDS: the first piece's operands
  __device__ __forceinline__ Coded(const PagedCache& c, int wave_) : wave(wave_) {
    const int tid = threadIdx.x, lane = tid & 63;
    row = tid >> 3;
    const uint32_t piece = tid & 7;
    k_off = (uint32_t)(row & 15) * (uint32_t)c.kst + piece * 16;
    v_off = (uint32_t)(row & 15) * (uint32_t)c.vst + piece * 16;
    s_row = G == 1 ? min(2 * lane, kBN - 1) : lane;
    k_at = (uint32_t)row * 256 + ((2 * piece) ^ (uint32_t)(row & 15)) * 16;
    v_at = (uint32_t)row * 256 + ((2 * piece) ^ (uint32_t)((row & 3) << 2)) * 16;
  }

  // The codes of one side: the wave's rows lie in one block of 16 for each piece.
  template <bool V>
  __device__ __forceinline__ void load(const PagedCache& c, const Source& s, int key0, const Pages& p, uint32_t ok, u32x4* to) const {
    const bool upper = wave >= 2;
    if (s.whole(key0, ok)) {
#pragma unroll
      for (int e = 0; e < 2; ++e)
        put<V>(c, s, upper ? p[2 * e + 1] : p[2 * e], key0 + 32 * e + (upper ? 16 : 0), true, to + 256 * e + 64 * wave);
    } else {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const bool good = ok >> (2 * e + upper) & 1;
        const int key = key0 + row + 32 * e;
        put<V>(c, s, good ? (upper ? p[2 * e + 1] : p[2 * e]) : 0, key0 + 32 * e + (upper ? 16 : 0),
               good && key >= s.lo && key < s.hi, to + 256 * e + 64 * wave);
      }
    }
  }
  template <bool V>
  __device__ __forceinline__ void put(const PagedCache& c, const Source& s, int32_t page, int token, bool there, u32x4* to) const {
    const uint8_t* x = V ? block_of(c, s.v, c.vsp, c.vst, page, token) + v_off : block_of(c, s.k, c.ksp, c.kst, page, token) + k_off;
    if (!there) x = (const uint8_t*)zero_row;
    __builtin_amdgcn_global_load_lds((gptr)x, (__attribute__((address_space(3))) void*)to, 16, 0, 0);
  }
  __device__ __forceinline__ void load_scales(const PagedCache& c, const Source& s, int key0, const Pages& p, uint32_t ok, VCodes<G>& to) const {
    const bool v = wave >= 2;
    const uint8_t* const x = v ? s.vs : s.ks;
    const uint32_t page_stride = (uint32_t)(v ? c.vssp : c.kssp);
    uint32_t* const lds = (v ? to.vs : to.ks) + (G == 4 ? 64 * (wave & 1) : 0);
    const uint32_t in_token = G == 4 ? 4 * (wave & 1) : 0;
    if (ok == 15 && c.lg >= 6) {  // a tile of one page
      const uint32_t at = (uint32_t)((key0 & c.page_mask) + s_row) * (2 * G) / 4 * 4 + in_token;
      __builtin_amdgcn_global_load_lds((gptr)(x + (uint64_t)(uint32_t)p[0] * page_stride + at), (__attribute__((address_space(3))) void*)lds, 4, 0, 0);
    } else {
      const int u = s_row >> 4;
      const int32_t n = u < 2 ? (u ? p[1] : p[0]) : u == 2 ? p[2] : p[3];
      const uint32_t at = (uint32_t)((key0 + s_row) & c.page_mask) * (2 * G) / 4 * 4 + in_token;
      const uint8_t* y = x + (uint64_t)(uint32_t)n * page_stride + at;
      if (!(ok >> u & 1)) y = (const uint8_t*)zero_row;
      __builtin_amdgcn_global_load_lds((gptr)y, (__attribute__((address_space(3))) void*)lds, 4, 0, 0);
    }
  }

  // K's operands from its codes: the codes themselves, exact in fp16, whose scales come to the scores.
  __device__ __forceinline__ void decode_k(const KCodes& from, LdsTile& kt) const {
    lds_u8* const to = (lds_u8*)&kt[0];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const u32x4 x = from[threadIdx.x + 256 * e];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        u32x4 k;
#pragma unroll
        for (int d = 0; d < 2; ++d) {
          const uint32_t a = x[2 * h + d] ^ 0x80808080u;
          k[2 * d] = code_pair(a, 0x04010400u);
          k[2 * d + 1] = code_pair(a, 0x04030402u);
        }
        *(lds_u32x4*)(to + (k_at ^ (16 * h)) + 8192 * e) = k;
      }
    }
  }
  // V's operands: code x scale in fp16, the framework's own dequantization, 0 for tokens that nobody sees.
  __device__ __forceinline__ void decode_v(const Source& s, int key0, uint32_t ok, const VCodes<G>& from, LdsTile& vt) const {
    lds_u8* const to = (lds_u8*)&vt[0];
    const bool all = s.whole(key0, ok);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int g = (threadIdx.x & 7) * 16 / GS, at_row = row + 32 * e;
      uint32_t scale = ((const uint16_t*)from.vs)[G == 1 ? at_row : g / 2 * 128 + at_row * 2 + g % 2];
      if (!all) {
        const int at = row + 32 * e, key = key0 + at;
        if (!((ok >> (at >> 4) & 1) && key >= s.lo && key < s.hi)) scale = 0;
      }
      const half2v f = as_h2(scale * 0x00010001u);
      const u32x4 x = from.v[threadIdx.x + 256 * e];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        u32x4 v;
#pragma unroll
        for (int d = 0; d < 2; ++d) {
          const uint32_t a = x[2 * h + d] ^ 0x80808080u;
          v[2 * d] = as_u32(as_h2(code_pair(a, 0x04010400u)) * f);
          v[2 * d + 1] = as_u32(as_h2(code_pair(a, 0x04030402u)) * f);
        }
        *(lds_u32x4*)(to + v_at + 16 * h + 8192 * e) = v;
      }
    }
  }
};

__device__ __forceinline__ float half_of(uint32_t w, int up) {
  return (float)__builtin_bit_cast(half_t, (uint16_t)(up ? w >> 16 : w));
}

// G: groups of an INT8 row's scales; 0 where K's values come as they are.
template <class M, int G>
struct Shared : AttnTile<M> {
  using AttnTile<M>::acc;
  using AttnTile<M>::m;
  using AttnTile<M>::l;
  bool seen;

  // Scores of codes: of each group by itself, times the tokens' scales.  Two groups at a time, whose scales are read for them:
  // all four have no room.
  static __device__ __forceinline__ float16v code_scores(const u32x4 (&kf)[8], const u32x4 (&q)[8], const uint32_t* scales, int u) {
    const int first = 32 * u + 4 * ((threadIdx.x & 63) >> 5);
    float16v sc;
#pragma unroll
    for (int j = 0; j < 16; ++j) sc[j] = 0.f;
    constexpr int N = G < 2 ? G : 2;
#pragma unroll
    for (int g0 = 0; g0 < G; g0 += N) {
      if (g0) __builtin_amdgcn_sched_barrier(0);
      uint32_t w[16];  // token j's, of groups g0 and g0 + 1; of one group, a pair of tokens' in every second
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (G == 1) {
          const u32x2 x = *(const u32x2*)((const uint16_t*)scales + first + 8 * i);
          w[4 * i] = x[0]; w[4 * i + 2] = x[1];
        } else {
          const u32x4 x = *(const u32x4*)(scales + g0 / 2 * 64 + first + 8 * i);
#pragma unroll
          for (int r = 0; r < 4; ++r) w[4 * i + r] = x[r];
        }
      }
#pragma unroll
      for (int g = g0; g < g0 + N; ++g) {
        float16v d;
#pragma unroll
        for (int j = 0; j < 16; ++j) d[j] = 0.f;
#pragma unroll
        for (int kk = 8 * g / G; kk < 8 * (g + 1) / G; ++kk) d = M::mfma32(kf[kk], q[kk], d);
#pragma unroll
        for (int j = 0; j < 16; ++j) sc[j] = fmaf(d[j], G == 1 ? half_of(w[j & ~1], j & 1) : half_of(w[j], g - g0), sc[j]);
      }
    }
    return sc;
  }

  // Scaled scores with -inf for the tokens of a half that nobody sees.
  __device__ __forceinline__ void mask(float16v& sc, const Source& s, float scale, int key0, uint32_t ok, int u) {
    const int first = 32 * u + 4 * ((threadIdx.x & 63) >> 5);
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const int at = first + 8 * (j >> 2) + (j & 3);  // in the tile
      const bool vis = key0 + at >= s.lo && key0 + at < s.hi && (ok >> (at >> 4) & 1);
      seen |= vis;
      sc[j] = vis ? sc[j] * scale : kNegInf;
    }
  }

  // A tile's tokens 32 u0 .. 32 u1 - 1: values as they are.
  __device__ __forceinline__ void tile(const LdsTile& ks, const LdsTile& vs, const Source& s, const u32x4 (&q)[8], float scale,
                                       int key0, uint32_t ok, int u0, int u1) {
    const bool full = s.whole(key0, ok);
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
      if (!full) mask(sc, s, scale, key0, ok, u);
      this->add_sum(this->exps(sc, mul, pb), sc, mul, pb);
      if (u + 1 < u1) this->read_k(ks, u + 1, kf);
      __builtin_amdgcn_sched_barrier(0);
      this->add_values(vf, pb);
    }
  }

  // The same of codes, up to P, and the product with V, pb[half].
  __device__ __forceinline__ void code_probs(const LdsTile& ks, const uint32_t* scales, const Source& s, const u32x4 (&q)[8], float scale,
                                             int key0, uint32_t ok, int u0, int u1, u32x4 (&pb)[2][2]) {
    const bool full = s.whole(key0, ok);
    const float mul = full ? scale : 1.f;
    seen |= full;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int u = u0 + i;
      if (u >= u1) break;
      u32x4 kf[8];
      this->read_k(ks, u, kf);
      float16v sc = code_scores(kf, q, scales, u);
      __builtin_amdgcn_sched_barrier(0);
      if (!full) mask(sc, s, scale, key0, ok, u);
      const float before = m;
      this->add_sum(this->exps(sc, mul, pb[i]), sc, mul, pb[i]);
      // The first half's P stand at the maximum before this one, in 16 bits, and are rounded once more: 2^-11 of a token's
      // weight again, in tiles that raise the maximum.  In fp32 they would take 8 registers more; groups of 32 hold 250 of 256.
      if (i == 1 && __any(m != before)) {
        const float f = fast_exp2(before - shift_of(m));
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int d = 0; d < 4; ++d)
            pb[0][x][d] = M::pack(M::to_f((uint16_t)pb[0][x][d]) * f, M::to_f((uint16_t)(pb[0][x][d] >> 16)) * f);
      }
    }
  }
  __device__ __forceinline__ void code_values(const LdsTile& vs, int u0, int u1, const u32x4 (&pb)[2][2]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (u0 + i >= u1) break;
      u32x4 vf[8];
      this->read_v(vs, u0 + i, vf);
      this->add_values(vf, pb[i]);
    }
  }
};

// A barrier of the work-group for its LDS alone: loads that are under way stay so.
__device__ __forceinline__ void barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

template <class T, bool I8, int GS>
__global__ __launch_bounds__(kThreads, 2) void shared_decode_kernel(ShArgs a) {
  using M = typename std::conditional<I8, TF16, T>::type;  // the matrix instructions' type
  constexpr int G = I8 ? 128 / GS : 0;
  // 16-bit pages: two buffers; INT8: one for the operands, two for codes.  Each is a variable of its own, so that the
  // compiler does not wait for what is being loaded into one where another is read.
  __shared__ LdsTile k0, v0;
  __shared__ typename std::conditional<I8, KCodes, LdsTile>::type k1;
  __shared__ typename std::conditional<I8, VCodes<I8 ? G : 1>, LdsTile>::type v1;
  __shared__ typename std::conditional<I8, KCodes, u32x4[1]>::type k2;
  __shared__ typename std::conditional<I8, VCodes<I8 ? G : 1>, u32x4[1]>::type v2;
  __shared__ float2 half_ml[2][32];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int ql = lane & 31, hh = lane >> 5, rep = a.rep;
  const PagedCache& pc = a.c;
  const int H = pc.kv_heads;

  int h, row0, col0, cols, t, t1;
  int64_t slot;
  Source s;
  {
    // the prefixes first: their runs are the longest
    const uint32_t prefixes = gridDim.x - a.tails;
    uint32_t at = blockIdx.x;
    if (at >= prefixes) {
      at -= prefixes;
      h = (int)(at % (uint32_t)H);
      at /= (uint32_t)H;
      const Tails mine(a, (int)at, h == 0);
      const int b = __builtin_amdgcn_readfirstlane(mine.row);
      if (b < 0) return;
      const RowPlan r = plan_of_row(a.rows, b);
      const Tail tail(a, r.len, ((const_i32)a.lens)[b]);
      row0 = b; col0 = 0; cols = rep;
      t = tail.begin(mine.chunk, mine.chunks); t1 = tail.begin(mine.chunk + 1, mine.chunks);
      s.lo = tail.lo; s.hi = tail.hi;
      s.table = (const_i32)(pc.table + (tail.shares ? b : r.row0) * pc.table_stride);
      slot = a.prefix_slots + (int64_t)at * rep;
    } else {
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

  Shared<M, G> f;
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
    const Direct d(pc, wave);
    auto arrived = [&]() {  // this wave's loads have, and then every wave's; the other buffer is free
      __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
      __syncthreads();
    };
    d(pc, s, t * kBN, p, ok, k0, v0);
    p = pages_of(pc, s, min(t + 1, t1 - 1));
    for (; t < t1; t += 2) {
      arrived();
      uint32_t ok1 = there(pc, p);
      if (t + 1 < t1) {
        d(pc, s, (t + 1) * kBN, p, ok1, k1, v1);
        p = pages_of(pc, s, min(t + 2, t1 - 1));
      }
      if (active) f.tile(k0, v0, s, q, scale, t * kBN, ok, u0, u1);
      if (t + 1 == t1) break;
      arrived();
      ok = there(pc, p);
      if (t + 2 < t1) {
        d(pc, s, (t + 2) * kBN, p, ok, k0, v0);
        p = pages_of(pc, s, min(t + 3, t1 - 1));
      }
      if (active) f.tile(k1, v1, s, q, scale, (t + 1) * kBN, ok1, u0, u1);
    }
  } else {
    // Tiles past the run's end are loaded like any, from the zeros: the waits are the same in every turn.
    const Coded<GS> d(pc, wave);
    u32x4 pb[2][2];
    Pages p1 = pages_of(pc, s, min(t + 1, t1 - 1));
    uint32_t ok1 = t + 1 < t1 ? there(pc, p1) : 0;
    auto load_v = [&](int tile, const Pages& at, uint32_t good, VCodes<G>& to) {
      d.template load<true>(pc, s, tile * kBN, at, good, to.v);
      d.load_scales(pc, s, tile * kBN, at, good, to);
    };
    d.template load<false>(pc, s, t * kBN, p, ok, k1);
    load_v(t, p, ok, v1);
    d.template load<false>(pc, s, (t + 1) * kBN, p1, ok1, k2);
    load_v(t + 1, p1, ok1, v2);
    p = pages_of(pc, s, min(t + 2, t1 - 1));
    if constexpr (std::is_same<T, TB16>::value) {
      // bf16 values in fp16, the column's largest scaled to [2^14, 2^15) by a power of two: those down to 2^-31 of that power
      // are exact, and smaller ones off by at most 2^-39 of it (fp16's least step is 2^-24)
      float top = 0.f;
#pragma unroll
      for (int kk = 0; kk < 8; ++kk)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          top = fmaxf(top, fmaxf(fabsf(TB16::to_f((uint16_t)q[kk][j])), fabsf(TB16::to_f((uint16_t)(q[kk][j] >> 16)))));
      top = fmaxf(top, xor32(top));
      int ex = (int)(__builtin_bit_cast(uint32_t, top) >> 23) - 127;
      ex = ex == 128 || ex == -127 ? 0 : max(ex - 14, -126);  // Inf or NaN stays what it is; zero or a subnormal is 0
      const float g = ldexpf(1.f, -ex);
      scale = ldexpf(scale, ex);
#pragma unroll
      for (int kk = 0; kk < 8; ++kk)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          q[kk][j] = TF16::pack(TB16::to_f((uint16_t)q[kk][j]) * g, TB16::to_f((uint16_t)(q[kk][j] >> 16)) * g);
    }
    __builtin_amdgcn_s_waitcnt(0x0F78);  // vmcnt(8): the first K
    barrier();
    d.decode_k(k1, k0);
    // A wave has two loads of K's codes and three of V's codes and scales under way while it awaits those before them.
    auto arrived = [&]() {
      __builtin_amdgcn_s_waitcnt(0x0F75);  // vmcnt(5)
      barrier();
    };
    arrived();
    // One tile: its scores while V is decoded, its product with V while the next tile's K is.
    auto turn = [&](KCodes& kc, VCodes<G>& vc, const KCodes& next) {
      const uint32_t ok2 = t + 2 < t1 ? there(pc, p) : 0;
      d.template load<false>(pc, s, (t + 2) * kBN, p, ok2, kc);
      d.decode_v(s, t * kBN, ok, vc, v0);
      if (active) f.code_probs(k0, vc.ks, s, q, scale, t * kBN, ok, u0, u1, pb);
      arrived();  // the next K
      load_v(t + 2, p, ok2, vc);
      p = pages_of(pc, s, min(t + 3, t1 - 1));
      d.decode_k(next, k0);
      if (active) f.code_values(v0, u0, u1, pb);
      arrived();  // the next V
      ok = ok1;
      ok1 = ok2;
      ++t;
    };
    while (t + 1 < t1) {  // no way out of its middle: the compiler would wait for all loads at its start
      turn(k1, v1, k2);
      turn(k2, v2, k1);
    }
    if (t < t1) turn(k1, v1, k2);
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): no load may come after the work-group
  }

  // a sum whose maximum is -inf is none: 1 where something was seen, else 0
  f.l += xor32(f.l);
  f.seen |= (bool)__shfl_xor((int)f.seen, 32, 64);
  if (f.m == kNegInf && f.l == f.l) f.l = f.seen ? 1.f : 0.f;
  if (halves) {
    __syncthreads();  // the buffers are free
    float4v* const other = (float4v*)(block ? v0 : k0);  // [16][64]
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
  const const_i32 place = (const_i32)(a.places + b);
  const int chunks = place[1], splits = place[2] ? r.splits : 0;
  const int c = (b - r.row0) * rep + head % rep, c0 = c / max(r.per, 1) * r.per, width = min(r.per, r.cols - c0);
  const int64_t first = h * a.slots + r.slot + (int64_t)c0 * r.splits + (c - c0);
  const int64_t own = h * a.slots + a.prefix_slots + (int64_t)place[0] * rep + head % rep;
  float m = kNegInf, l = 0.f, o[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) o[k] = 0.f;
  const int parts = splits + chunks;
  for (int w = sl; w < parts; w += 64) {  // four parts' loads side by side; past the end the last one again, without weight
    float2 p[4];
    float4v x[4], y[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int i = min(w + 16 * u, parts - 1);
      const int64_t slot = i < splits ? first + (int64_t)i * width : own + (int64_t)(i - splits) * rep;
      p[u] = a.ml[slot];
      x[u] = *(const float4v*)(a.acc + slot * 128 + cc * 8);
      y[u] = *(const float4v*)(a.acc + slot * 128 + cc * 8 + 4);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (w + 16 * u >= parts) break;
      const float top = fmaxf(m, p[u].x), f0 = part_of(m, top), f1 = part_of(p[u].x, top);
      l = sum_in(m, l, top) + sum_in(p[u].x, p[u].y, top);
      m = top;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        o[k] = o[k] * f0 + x[u][k] * f1;
        o[4 + k] = o[4 + k] * f0 + y[u][k] * f1;
      }
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

// Work-groups that fill the GPU, two a CU, and those of them for the prefixes; more of them where each has more than kLong
// tiles, so that the tails matter less.  us in a graph: four prompts of up to 16384 with 8 rows each over 256, 384 and 512 28.9, 27.5,
// 33.3 (then the tails have to wait); one of 32768 with 32 rows, INT8, over 416, 448 and 480 with up to 509 tokens of their own
// 74.7, 80.3, 81.3, with one 77.0, 73.5, 73.5.
constexpr int kTarget = 512;
constexpr int kPrefixTarget = 384;
constexpr int kLongTarget = 448;
constexpr int kLong = 12;
// Least tiles of a prefix's work-group, between a long run and many parts to join: 16 rows over 8191 tokens with 1, 3 and 6
// 21.3, 18.7, 22.3; two rows over 517 10.1, 10.1, 11.0.
constexpr int kMinTiles = 3;
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
  int64_t quota = (work * kv_heads + kPrefixTarget - 1) / kPrefixTarget;  // tiles a work-group
  if (quota > kLong) quota = (work * kv_heads + kLongTarget - 1) / kLongTarget;
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
    // The runs of a block of columns one behind the other: the two work-groups of a CU are then of different blocks where
    // these differ in columns (160 in 96 and 64, INT8, 32768 tokens: 73.5 us, alternating 81.4).
    for (int64_t c0 = 0; c0 < cols; c0 += per)
      for (int64_t s = 0; s < splits; ++s) {
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
  const int64_t strides[4] = {c.ksp, c.vsp, c.kssp, c.vssp};
  for (int64_t x : strides)
    if (x < 0 || x >> 32) return fail(KVQ_ERR_UNSUPPORTED, "shared decode: page stride out of range");
  if (p->plan.rows != c.batch || p->plan.units < 0 || p->plan.slots < 0) return fail(KVQ_ERR_INVALID, "shared decode: the plan is of another batch");
  return KVQ_OK;
}

struct Launch {
  int fill;
  int64_t groups, slots, places, map, acc, bytes;
  int64_t tails, grid;
};

Launch launch_of(const kvq_shared_decode_params& p) {
  Launch w{};
  const int64_t B = p.cache.batch, H = p.cache.kv_heads, rep = p.q_heads / H;
  const int64_t tiles = ((int64_t)p.cache.max_pages * p.cache.page_size + kBN - 1) / kBN;
  const int64_t most = (tiles + kTailTiles - 1) / kTailTiles;  // of a row
  // Long tails in many pieces end together: 32 rows of 40 / 8 heads with up to 4000 tokens of their own behind 32768 shared INT8
  // ones over B, 2 B and 4 B 150, 129 and 123 us; 4 rows with 16000 over 4 B 141, so 79.  Short ones have no more pieces than
  // kTailTiles allows; work-groups that find none are dear where there are many rows.
  int64_t fill = 2 * kTarget / H, rows = B <= 64 ? 4 * B : B;
  if (fill < rows) fill = rows;
  w.fill = (int)fill;
  // what Tails, or the launch before it, makes of that: a piece of each row at the least
  w.groups = fill + B < B * most ? fill + B : B * most;
  if (w.groups < 1) w.groups = 1;  // who writes the places
  w.slots = p.plan.slots + w.groups * rep;
  w.places = (8 * H * w.slots + 63) / 64 * 64;
  w.map = w.places + (16 * B + 63) / 64 * 64;
  w.acc = w.map + (B > 64 ? (8 * w.groups + 63) / 64 * 64 : 0);
  w.bytes = w.acc + 512 * H * w.slots;
  w.tails = H * w.groups;
  w.grid = w.tails + H * p.plan.units;
  return w;
}

template <class T, bool I8, int GS>
int launch(const ShArgs& a, const Launch& w, hipStream_t st) {
  int rc = KVQ_OK;
  if (a.map) {
    hipLaunchKernelGGL(shared_places_kernel, dim3(1), dim3(kThreads), 0, st, a);
    if ((rc = launched())) return rc;
  }
  hipLaunchKernelGGL((shared_decode_kernel<T, I8, GS>), dim3((unsigned)w.grid), dim3(kThreads), 0, st, a);
  if ((rc = launched())) return rc;
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
  a.fill = w.fill; a.groups = (int32_t)w.groups;
  a.prefix_slots = p->plan.slots;
  a.tails = (uint32_t)w.tails;
  a.slots = w.slots;
  a.ml = (float2*)p->workspace;
  a.places = (int4*)((uint8_t*)p->workspace + w.places);
  if (a.c.batch > 64) a.map = (int2*)((uint8_t*)p->workspace + w.map);
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
