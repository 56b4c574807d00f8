// Eviction from a paged cache by accumulated weight (kvq_paged_evict), in two launches.
//
// paged_select_kernel: a work-group a (row, KV head); every wave has a segment of the tokens, with their
// weights in registers where the pages can hold 16384 to 32768 tokens a row.  The threshold, the need-th largest
// weight of the tokens that are not protected, by three passes of a radix select (11, 11 and 10 bits of a key
// that orders as the floats do) with LDS histograms; then every wave counts what it keeps of its segment, and
// writes it from the sum of the segments before it.
//
// paged_move_kernel: the kept rows to the front, in place and in order.  Row j's source lies at or behind
// j, so the rows of a block may be written once the whole block has been read: a work-group that has the
// same bytes of all rows (a slice of one side of one (row, head)) needs one barrier a block and nothing from
// the others.  Kept tokens are fetched two blocks ahead, their pages one, so that a block costs one latency.
//
// What bounds it, the kernels alone: the select is a chain of passes within a work-group (8 x 8 rows of 32768 tokens 27
// us, 1 x 2 of 640 8.9); the move is HBM (4096 kept of each, INT8: 37 us for 143 MB read and written), or a launch's
// latency where the budget is small (5 us).  Four rows a thread in flight: eight take 41 us, with fewer work-groups a CU.
#include "paged.h"

namespace kvq {
namespace {

constexpr int kBins = 2048;
constexpr int kMoveThreads = 512;
constexpr int kSlice = 64;                              // bytes of a row a work-group moves
constexpr int kMoveRows = kMoveThreads * 16 / kSlice;   // rows a load of all threads covers
constexpr int kMoveUnroll = 4;
constexpr int kSelKeys = 32;  // weights a lane keeps

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

// A token's key: larger key = larger weight, the zeros equal, NaN (1) below everything.  Tokens that stay
// anyway have the largest key of all, places that are no token 0: so the kept tokens are those of the `budget`
// largest keys.
constexpr uint32_t kStays = 0xFFFFFFFFu;
__device__ __forceinline__ uint32_t key_of(float x, int i, int lo, int hi, int n) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x + 0.f);  // -0 + 0 = 0
  uint32_t k = u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
  if (x != x) k = 1;
  if (i < lo || i >= hi) k = kStays;
  return i < n ? k : 0;
}

// Weights and keys of a wave's tokens [s0, s1), one of every 64 a lane: in registers (REG) or fetched each time.
template <bool REG>
struct Tokens {
  const float* w;
  int s0, s1, lo, hi, n;
  float x[REG ? kSelKeys : 1];
  uint32_t k[REG ? kSelKeys : 1];
  __device__ __forceinline__ float weight(int i) const { return i < s1 ? w[i] : 0.f; }
  __device__ __forceinline__ void load() {
    const int lane = threadIdx.x & 63;
    if constexpr (REG) {
#pragma unroll
      for (int j = 0; j < kSelKeys; ++j) x[j] = weight(s0 + 64 * j + lane);
#pragma unroll
      for (int j = 0; j < kSelKeys; ++j) k[j] = key_of(x[j], s0 + 64 * j + lane, lo, hi, s1);
    }
  }
  // f(first token of 64, weight, key) for every 64 tokens, all lanes together
  template <class F>
  __device__ __forceinline__ void each(F f) const {
    const int lane = threadIdx.x & 63;
    if constexpr (REG) {
#pragma unroll
      for (int j = 0; j < kSelKeys; ++j)
        if (s0 + 64 * j < s1) f(s0 + 64 * j, x[j], k[j]);
    } else {
      for (int i0 = s0; i0 < s1; i0 += 512) {
        float y[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = weight(i0 + 64 * j + lane);
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (i0 + 64 * j < s1) f(i0 + 64 * j, y[j], key_of(y[j], i0 + 64 * j + lane, lo, hi, s1));
      }
    }
  }
};

template <int THREADS, bool REG>
__global__ __launch_bounds__(THREADS) void paged_select_kernel(EvictArgs a) {
  constexpr int kWaves = THREADS / 64, kEach = kBins / THREADS;  // bins a thread
  __shared__ int hist[kBins];
  __shared__ int wtot[kWaves], wgt[kWaves], weq[kWaves];
  __shared__ int s_bin, s_rank;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int h = blockIdx.x, b = blockIdx.y;
  const int n = row_len(a, b);
  const float* w = a.w + b * a.wsb + h * a.wsh;
  const int64_t bh = (int64_t)b * a.c.kv_heads + h;
  int32_t* kept = a.kept + bh * a.budget;
  float* nw = a.new_w + bh * a.w_tokens;
  const int seg = ((n + kWaves - 1) / kWaves + 63) / 64 * 64, s0 = min(wave * seg, n);
  Tokens<REG> t{w, s0, min(s0 + seg, n), a.sinks, n - a.recent, n};
  bool bad = false;
  if (n > a.budget) {
    t.load();
    const int pages = (n + a.c.page_mask) >> a.c.lg;
    for (int i = tid; i < pages; i += THREADS)
      bad |= (uint32_t)a.c.table[b * a.c.table_stride + i] >= (uint32_t)a.c.num_pages;
  }
  const bool gone = __syncthreads_or(bad);
  if (n <= a.budget || gone) {  // everything stays
    for (int i = tid; i < a.w_tokens; i += THREADS) nw[i] = i < n ? w[i] : 0.f;
    for (int i = tid; i < a.budget; i += THREADS) kept[i] = i < n && !gone ? i : -1;
    if (h == 0 && tid == 0) a.new_lens[b] = n;
    return;
  }
  // the threshold: the budget-th largest key, and how many of those equal to it are kept
  uint32_t thr = 0;
  int rank = a.budget;  // among the keys that share the digits found
#pragma unroll
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
    const uint32_t mask = (1u << bits) - 1;
#pragma unroll
    for (int i = 0; i < kEach; ++i) hist[tid + i * THREADS] = 0;
    __syncthreads();
    t.each([&](int, float, uint32_t k) {
      if (pass == 0 ? k != 0 : (k >> (shift + bits)) == thr && k != 0) atomicAdd(&hist[(k >> shift) & mask], 1);
    });
    __syncthreads();
    // this thread's bins, from the top: what the threads before it have, by a sum over the work-group
    const int top = kBins - 1 - tid * kEach;
    int own = 0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) own += hist[top - i];
    int x = own;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int y = __shfl_up(x, o, 64);
      if (lane >= o) x += y;
    }
    if (lane == 63) wtot[wave] = x;
    __syncthreads();
    int above = x - own;
    for (int v = 0; v < wave; ++v) above += wtot[v];
    if (above < rank && above + own >= rank) {
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        const int c = hist[top - i];
        if (above < rank && above + c >= rank) { s_bin = top - i; s_rank = rank - above; }
        above += c;
      }
    }
    __syncthreads();
    thr = (thr << bits) | (uint32_t)s_bin;
    rank = s_rank;
  }
  // what every wave's segment has above and at the threshold
  int gt = 0, eq = 0;
  t.each([&](int, float, uint32_t k) {
    gt += __popcll(__ballot(k > thr));
    eq += __popcll(__ballot(k == thr));
  });
  if (lane == 0) { wgt[wave] = gt; weq[wave] = eq; }
  __syncthreads();
  int dst = 0, eqs = 0;
  for (int v = 0; v < wave; ++v) {
    dst += wgt[v] + max(min(rank - eqs, weq[v]), 0);
    eqs += weq[v];
  }
  t.each([&](int i, float x, uint32_t k) {
    const uint64_t me = __ballot(k == thr), mg = __ballot(k > thr);
    uint64_t take = mg;
    if (me) {  // the lowest of those equal to the threshold, as long as there is room
      const int before = eqs + __builtin_amdgcn_mbcnt_hi((uint32_t)(me >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)me, 0));
      take |= __ballot(k == thr && before < rank);
      eqs += __popcll(me);
    }
    if (take) {
      if (take >> lane & 1) {
        const int d = dst + __builtin_amdgcn_mbcnt_hi((uint32_t)(take >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)take, 0));
        kept[d] = i + lane;
        nw[d] = x;
      }
      dst += __popcll(take);
    }
  });
  for (int i = a.budget + tid; i < a.w_tokens; i += THREADS) nw[i] = 0.f;
  if (h == 0 && tid == 0) a.new_lens[b] = a.budget;
}

__global__ __launch_bounds__(kMoveThreads) void paged_move_kernel(EvictArgs a) {
  constexpr int kLanes = kSlice / 16, U = kMoveUnroll, kBlock = kMoveRows * U;
  // the slices of a (row, head) lie H * B work-groups apart: with 8 or a multiple, on one XCD, whose L2 has the
  // lines they share
  const int h = blockIdx.x, b = blockIdx.y;
  const int side = blockIdx.z >= (uint32_t)a.slices, slice = blockIdx.z - side * a.slices;
  const PagedCache& pc = a.c;
  const int n = row_len(a, b);
  if (n <= a.budget) return;
  const int32_t* kept = a.kept + ((int64_t)b * pc.kv_heads + h) * a.budget;
  if (kept[0] < 0) return;  // a row with a page that is not there
  const int32_t* tab = pc.table + b * pc.table_stride;
  uint8_t* const base = (side ? pc.v + h * pc.vsh : pc.k + h * pc.ksh) + slice * kSlice + (threadIdx.x % kLanes) * 16;
  const int64_t sp = side ? pc.vsp : pc.ksp, stt = side ? pc.vst : pc.kst;
  uint8_t* const sbase = side ? pc.vs + h * pc.vssh : pc.ks + h * pc.kssh;
  const int64_t ssp = side ? pc.vssp : pc.kssp;
  const int sb = a.scale_bytes;
  const bool scales = sb && slice == 0 && threadIdx.x % kLanes == 0;
  const int r0 = threadIdx.x / kLanes, last = a.budget - 1;

  // Block by block: kept tokens (bounded, whatever they are, by the row) of block i + 2, source and destination pages and rows of block i + 1
  int src2[U], src1[U], page1[U], to1[U];
  auto tokens = [&](int j0) {
#pragma unroll
    for (int u = 0; u < U; ++u) src2[u] = min(max(kept[min(j0 + u * kMoveRows + r0, last)], 0), n - 1);
  };
  auto pages = [&](int j0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      src1[u] = src2[u];
      page1[u] = tab[src1[u] >> pc.lg];
      to1[u] = tab[min(j0 + u * kMoveRows + r0, last) >> pc.lg];
    }
  };
  u32x4 x[U];
  u32x2 sc[U];
  int at[U], to[U];  // a row's source, -1: it stays; its destination's page
  auto rows = [&](int j0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = j0 + u * kMoveRows + r0;
      at[u] = j <= last && src1[u] != j ? src1[u] : -1;
      to[u] = to1[u];
      if (at[u] >= 0) {
        const int slot = at[u] & pc.page_mask;
        x[u] = *(const u32x4*)(base + page1[u] * sp + slot * stt);
        if (scales) {
          const uint8_t* s = sbase + page1[u] * ssp + slot * sb;
          if (sb == 8) sc[u] = *(const u32x2*)s;
          else if (sb == 4) sc[u][0] = *(const uint32_t*)s;
          else sc[u][0] = *(const uint16_t*)s;
        }
      }
    }
  };
  tokens(0);
  pages(0);
  tokens(kBlock);
  rows(0);
  pages(kBlock);
  tokens(2 * kBlock);
  for (int j0 = 0; j0 < a.budget; j0 += kBlock) {
    // every row of the block has arrived, in every wave, before one of it is written
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    u32x4 y[U];
    u32x2 sy[U];
    int where[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      y[u] = x[u];
      sy[u] = sc[u];
      where[u] = at[u] >= 0 ? to[u] : -1;
    }
    rows(j0 + kBlock);
    pages(j0 + 2 * kBlock);
    tokens(j0 + 3 * kBlock);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (where[u] >= 0) {
        const int64_t page = where[u];
        const int slot = (j0 + u * kMoveRows + r0) & pc.page_mask;
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

template <int THREADS, bool REG>
void select(const EvictArgs& a, hipStream_t st) {
  hipLaunchKernelGGL((paged_select_kernel<THREADS, REG>), dim3((unsigned)a.c.kv_heads, (unsigned)a.c.batch), dim3(THREADS), 0, st, a);
}

int evict(const kvq_paged_evict_params* p, hipStream_t st) {
  if (!p) return fail(KVQ_ERR_INVALID, "paged evict: NULL params");
  EvictArgs a{};
  int rc = paged_cache(p->cache, a.c);
  if (rc || (rc = paged_written(a.c))) return rc;
  const int B = a.c.batch, H = a.c.kv_heads;
  if (p->budget <= 0 || p->sinks < 0 || p->recent < 0 || (int64_t)p->sinks + p->recent > p->budget)
    return fail(KVQ_ERR_INVALID, "paged evict: budget must be positive and hold sinks + recent");
  if ((int64_t)p->w_tokens < (int64_t)p->cache.max_pages * p->cache.page_size)
    return fail(KVQ_ERR_INVALID, "paged evict: fewer weights than token slots");
  // places are counted on in 32 bits past the end by a work-group's share
  if (p->budget > (1 << 30) || p->w_tokens > (1 << 30)) return fail(KVQ_ERR_UNSUPPORTED, "paged evict: a budget or weights of more than 2^30 tokens");
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
  const int64_t cap = (int64_t)p->cache.max_pages * p->cache.page_size;
  // By the token slots of a row, us a call (its move is the same), 256 threads that fetch weights in every pass / 1024 that
  // do / 1024 that keep them in registers, which is a long straight line that an empty instruction cache pays for:
  //   1 row x 2 heads     512 12.1 / 12.5 / 19.3, 2048 15.0 / 15.3 / 20.7, 4096 21.4 / 17.7 / 23.3, 8192 35.0 / 23.5 / 27.5,
  //                       16384 61.6 / 37.8 / 38.0, 32768 115 / 66.4 / 58.5
  //   64 rows x 8 heads   512 23.7 / 26.5 / 43.6, 2048 45.7 / 49.5 / 64.1, 4096 91.7 / 90.1 / 105, 8192 219 / 212 / 224,
  //                       16384 483 / 464 / 470, 32768 965 / 929 / 926
  if (cap <= 2048) select<256, false>(a, st);
  else if (cap <= 512 * kSelKeys || cap > 1024 * kSelKeys) select<1024, false>(a, st);
  else select<1024, true>(a, st);
  if ((rc = launched())) return rc;
  hipLaunchKernelGGL(paged_move_kernel, dim3((unsigned)H, (unsigned)B, (unsigned)(2 * a.slices)), dim3(kMoveThreads), 0, st, a);
  return launched();
}

}  // namespace
}  // namespace kvq

extern "C" int kvq_paged_evict(const kvq_paged_evict_params* p, kvq_stream_t stream) {
  return kvq::guarded([&] { return kvq::evict(p, reinterpret_cast<hipStream_t>(stream)); });
}
