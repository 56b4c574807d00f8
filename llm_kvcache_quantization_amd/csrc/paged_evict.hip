// Eviction from a paged cache by accumulated weight (kvq_paged_evict), in two launches.
//
// paged_select_kernel: a work-group a (row, KV head).  The threshold, the need-th largest weight of the
// tokens that are not protected, by three passes of a radix select (11, 11 and 10 bits of a key that orders
// as the floats do) with LDS histograms; then every wave counts what it keeps of its segment of the
// tokens, and writes it from the sum of the segments before it.
//
// paged_move_kernel: the kept rows to the front, in place and in order.  Row j's source lies at or behind
// j, so the rows of a block may be written once the whole block has been read: a work-group that has the
// same bytes of all rows (a slice of one side of one (row, head)) needs one barrier a block and nothing from
// the others, and the next block's loads run under the stores.
//
// What bounds it: the select is a chain of passes over weights that the L2 holds; the move is HBM, or a
// launch's latency where the budget is small.
#include "paged.h"

namespace kvq {
namespace {

constexpr int kSelThreads = 1024;
constexpr int kSelWaves = kSelThreads / 64;
constexpr int kBins = 2048;
constexpr int kMoveThreads = 512;
constexpr int kSlice = 64;                              // bytes of a row a work-group moves
constexpr int kMoveRows = kMoveThreads * 16 / kSlice;   // rows a load of all threads covers
constexpr int kMoveUnroll = 4;

struct EvictArgs {
  PagedCache c;
  const int32_t* lens;
  const float* w;
  int64_t wsb, wsh;
  int32_t* new_lens;
  int32_t* kept;
  float* new_w;
  int32_t w_tokens, budget, sinks, recent;
  int32_t slices;      // of a row of one side
  int32_t scale_bytes; // of a row's scales; 0: none
};

__device__ __forceinline__ int row_len(const EvictArgs& a, int b) {
  return (int)min((int64_t)max(a.lens[b], 0), (int64_t)a.c.max_pages << a.c.lg);
}

// larger key = larger float; NaN below everything, the zeros equal
__device__ __forceinline__ uint32_t key_of(float x) {
  if (x != x) return 0;
  if (x == 0.f) x = 0.f;
  const uint32_t u = __builtin_bit_cast(uint32_t, x + 0.f);
  return u ^ (u >> 31 ? 0xFFFFFFFFu : 0x80000000u);
}

__global__ __launch_bounds__(kSelThreads) void paged_select_kernel(EvictArgs a) {
  __shared__ int hist[kBins];
  __shared__ int wtot[kSelWaves], wgt[kSelWaves], weq[kSelWaves];
  __shared__ int s_bin, s_rank, s_bad;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int h = blockIdx.x, b = blockIdx.y;
  const int n = row_len(a, b);
  const float* w = a.w + b * a.wsb + h * a.wsh;
  const int64_t bh = (int64_t)b * a.c.kv_heads + h;
  int32_t* kept = a.kept + bh * a.budget;
  float* nw = a.new_w + bh * a.w_tokens;
  if (tid == 0) s_bad = 0;
  __syncthreads();
  if (n > a.budget) {
    const int pages = (n + a.c.page_mask) >> a.c.lg;
    bool bad = false;
    for (int i = tid; i < pages; i += kSelThreads)
      bad |= (uint32_t)a.c.table[b * a.c.table_stride + i] >= (uint32_t)a.c.num_pages;
    if (bad) s_bad = 1;
    __syncthreads();
  }
  if (n <= a.budget || s_bad) {  // everything stays
    for (int i = tid; i < a.w_tokens; i += kSelThreads) nw[i] = i < n ? w[i] : 0.f;
    for (int i = tid; i < a.budget; i += kSelThreads) kept[i] = i < n && !s_bad ? i : -1;
    if (h == 0 && tid == 0) a.new_lens[b] = n;
    return;
  }
  const int lo = a.sinks, hi = n - a.recent, need = a.budget - a.sinks - a.recent;
  // the threshold: key of the need-th largest weight in [lo, hi), and how many equal to it are kept
  uint32_t thr = 0xFFFFFFFFu;
  int rank = 0;
  if (need > 0) {
    uint32_t prefix = 0;
    rank = need;  // among the keys that share the prefix
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
      const uint32_t mask = (1u << bits) - 1;
      for (int i = tid; i < kBins; i += kSelThreads) hist[i] = 0;
      __syncthreads();
      for (int i = lo + tid; i < hi; i += kSelThreads) {
        const uint32_t k = key_of(w[i]);
        if (pass == 0 || (k >> (shift + bits)) == prefix) atomicAdd(&hist[(k >> shift) & mask], 1);
      }
      __syncthreads();
      // keys in bins above this thread's two, by a suffix sum: thread t has bins 2 (1023 - t) + 1, + 0
      const int top = 2 * (kSelThreads - 1 - tid) + 1;
      const int c1 = hist[top], c0 = hist[top - 1];
      int x = c1 + c0;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int y = __shfl_up(x, o, 64);
        if (lane >= o) x += y;
      }
      if (lane == 63) wtot[wave] = x;
      __syncthreads();
      int above = x - c1 - c0;
      for (int v = 0; v < wave; ++v) above += wtot[v];
      if (above < rank && above + c1 >= rank) { s_bin = top; s_rank = rank - above; }
      else if (above + c1 < rank && above + c1 + c0 >= rank) { s_bin = top - 1; s_rank = rank - above - c1; }
      __syncthreads();
      prefix = (prefix << bits) | (uint32_t)s_bin;
      rank = s_rank;
    }
    thr = prefix;
  }
  // every wave's segment of the tokens: what it has above and at the threshold
  const int seg = ((n + kSelWaves - 1) / kSelWaves + 63) / 64 * 64;
  const int s0 = min(wave * seg, n), s1 = min(s0 + seg, n);
  int gt = 0, eq = 0;
  for (int i0 = s0; i0 < s1; i0 += 64) {
    const int i = i0 + lane;
    bool g = false, e = false;
    if (i < s1) {
      const uint32_t k = key_of(w[i]);
      const bool kept_anyway = i < lo || i >= hi;
      g = kept_anyway || (need > 0 && k > thr);
      e = !kept_anyway && need > 0 && k == thr;
    }
    gt += __popcll(__ballot(g));
    eq += __popcll(__ballot(e));
  }
  if (lane == 0) { wgt[wave] = gt; weq[wave] = eq; }
  __syncthreads();
  int dst = 0, eqs = 0;
  for (int v = 0; v < wave; ++v) {
    dst += wgt[v] + max(min(rank - eqs, weq[v]), 0);
    eqs += weq[v];
  }
  const uint64_t below = (1ull << lane) - 1;
  for (int i0 = s0; i0 < s1; i0 += 64) {
    const int i = i0 + lane;
    bool g = false, e = false;
    float x = 0.f;
    if (i < s1) {
      x = w[i];
      const uint32_t k = key_of(x);
      const bool kept_anyway = i < lo || i >= hi;
      g = kept_anyway || (need > 0 && k > thr);
      e = !kept_anyway && need > 0 && k == thr;
    }
    const uint64_t me = __ballot(e);
    const bool take = g || (e && eqs + __popcll(me & below) < rank);
    eqs += __popcll(me);
    const uint64_t mt = __ballot(take);
    if (take) {
      const int d = dst + __popcll(mt & below);
      kept[d] = i;
      nw[d] = x;
    }
    dst += __popcll(mt);
  }
  for (int i = a.budget + tid; i < a.w_tokens; i += kSelThreads) nw[i] = 0.f;
  if (h == 0 && tid == 0) a.new_lens[b] = a.budget;
}

__global__ __launch_bounds__(kMoveThreads) void paged_move_kernel(EvictArgs a) {
  constexpr int kLanes = kSlice / 16;  // a row
  const int h = blockIdx.y, b = blockIdx.z;
  const int side = blockIdx.x >= (uint32_t)a.slices, slice = blockIdx.x - side * a.slices;
  const PagedCache& pc = a.c;
  if (row_len(a, b) <= a.budget) return;
  const int32_t* kept = a.kept + ((int64_t)b * pc.kv_heads + h) * a.budget;
  if (kept[0] < 0) return;  // a row with a page that is not there
  const int32_t* tab = pc.table + b * pc.table_stride;
  uint8_t* const base = (side ? pc.v + h * pc.vsh : pc.k + h * pc.ksh) + slice * kSlice + (threadIdx.x % kLanes) * 16;
  const int64_t sp = side ? pc.vsp : pc.ksp, stt = side ? pc.vst : pc.kst;
  uint8_t* const sbase = side ? pc.vs + h * pc.vssh : pc.ks + h * pc.kssh;
  const int64_t ssp = side ? pc.vssp : pc.kssp;
  const int sb = a.scale_bytes;
  const bool scales = sb && slice == 0 && threadIdx.x % kLanes == 0;
  const int r0 = threadIdx.x / kLanes;

  u32x4 x[kMoveUnroll];
  u32x2 sc[kMoveUnroll];
  bool mv[kMoveUnroll];
  auto load = [&](int j0) {
#pragma unroll
    for (int u = 0; u < kMoveUnroll; ++u) {
      const int j = j0 + u * kMoveRows + r0;
      mv[u] = false;
      if (j < a.budget) {
        const int src = kept[j];
        if (src != j) {
          mv[u] = true;
          const int64_t page = tab[src >> pc.lg];
          const int slot = src & pc.page_mask;
          x[u] = *(const u32x4*)(base + page * sp + slot * stt);
          if (scales) {
            const uint8_t* s = sbase + page * ssp + slot * sb;
            if (sb == 8) sc[u] = *(const u32x2*)s;
            else if (sb == 4) sc[u][0] = *(const uint32_t*)s;
            else sc[u][0] = *(const uint16_t*)s;
          }
        }
      }
    }
  };
  load(0);
  for (int j0 = 0; j0 < a.budget; j0 += kMoveRows * kMoveUnroll) {
    // every load of the block has returned, in every wave, before a row of it is written
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    u32x4 y[kMoveUnroll];
    u32x2 sy[kMoveUnroll];
    bool my[kMoveUnroll];
#pragma unroll
    for (int u = 0; u < kMoveUnroll; ++u) { y[u] = x[u]; sy[u] = sc[u]; my[u] = mv[u]; }
    load(j0 + kMoveRows * kMoveUnroll);
#pragma unroll
    for (int u = 0; u < kMoveUnroll; ++u) {
      const int j = j0 + u * kMoveRows + r0;
      if (my[u]) {
        const int64_t page = tab[j >> pc.lg];
        const int slot = j & pc.page_mask;
        *(u32x4*)(base + page * sp + slot * stt) = y[u];
        if (scales) {
          uint8_t* s = sbase + page * ssp + slot * sb;
          if (sb == 8) *(u32x2*)s = sy[u];
          else if (sb == 4) *(uint32_t*)s = sy[u][0];
          else *(uint16_t*)s = (uint16_t)sy[u][0];
        }
      }
    }
  }
}

int evict(const kvq_paged_evict_params* p, hipStream_t st) {
  if (!p) return fail(KVQ_ERR_INVALID, "paged evict: NULL params");
  EvictArgs a{};
  int rc = paged_cache(p->cache, a.c);
  if (rc) return rc;
  const int B = a.c.batch, H = a.c.kv_heads;
  if (p->budget <= 0 || p->sinks < 0 || p->recent < 0 || (int64_t)p->sinks + p->recent > p->budget)
    return fail(KVQ_ERR_INVALID, "paged evict: budget must be positive and hold sinks + recent");
  if ((int64_t)p->w_tokens < (int64_t)p->cache.max_pages * p->cache.page_size)
    return fail(KVQ_ERR_INVALID, "paged evict: fewer weights than token slots");
  if (B > 65535 || H > 65535) return fail(KVQ_ERR_UNSUPPORTED, "paged evict: too many rows or heads");
  if (B == 0) return KVQ_OK;
  if (!p->context_lens || !p->weights || !p->new_lens || !p->kept || !p->new_weights)
    return fail(KVQ_ERR_INVALID, "paged evict: NULL pointer");
  a.lens = p->context_lens;
  a.w = p->weights; a.wsb = p->w_stride_b; a.wsh = p->w_stride_h;
  a.new_lens = p->new_lens; a.kept = p->kept; a.new_w = p->new_weights;
  a.w_tokens = p->w_tokens; a.budget = p->budget; a.sinks = p->sinks; a.recent = p->recent;
  const bool i8 = p->cache.format == KVQ_PAGED_INT8;
  a.slices = (i8 ? 128 : 256) / kSlice;
  a.scale_bytes = i8 ? 256 / p->cache.group_size : 0;
  hipLaunchKernelGGL(paged_select_kernel, dim3((unsigned)H, (unsigned)B), dim3(kSelThreads), 0, st, a);
  if ((rc = launched())) return rc;
  hipLaunchKernelGGL(paged_move_kernel, dim3((unsigned)(2 * a.slices), (unsigned)H, (unsigned)B), dim3(kMoveThreads), 0, st, a);
  return launched();
}

}  // namespace
}  // namespace kvq

extern "C" int kvq_paged_evict(const kvq_paged_evict_params* p, kvq_stream_t stream) {
  return kvq::guarded([&] { return kvq::evict(p, reinterpret_cast<hipStream_t>(stream)); });
}
