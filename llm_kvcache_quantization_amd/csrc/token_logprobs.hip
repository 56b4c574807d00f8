// Log probabilities of given tokens, entropy and the likeliest tokens of rows of logits (kvq_token_logprobs).
//
//   p = softmax(x / T),  log p_t = (x_t - m) / T - log l,  H = log l - sum (x - m) / T e^((x - m) / T) / l,
//   l = sum e^((x - m) / T)
//
// One pass over the logits: each thread keeps a running maximum m and the two sums in fp32.  What bounds it: HBM, and the
// vector units nearly as much (7 instructions a logit, one of them an exponential): 2047 rows of 152064 bf16 logits
// 105 us, 5.9 TB/s (12 us more with one instruction a logit more, and the likeliest by counting).  Few rows are split over
// work-groups, whose parts a second launch joins: 32 rows of 151936 with 20 of the likeliest 10 and 4.5 us, a chain of
// latencies (one row of 32000, in one launch, 8).
// Exponentials are the hardware's exp2, of an argument rounded as a difference and as a product: relative errors of 0.7 to
// 1.1e-7 (rows of 32000, one a call) and 0.8e-7 (2047 of 152064), where fp32 with the library's has 0.3 to 0.9e-7 and 0.8e-7.
//
// The likeliest: the pass leaves the maximum of every 32 logits that a lane takes (of 64 and more in long rows) in LDS.  The
// top-th largest of 64 groups' maxima is a bar that at least `top` logits reach; only the 32s that reach it are read
// again, and what reaches it in them, hardly more than `top` logits, is put in order by counting, for each, how many are
// above it.  A candidate is one whole number, the logit's order above the complement of the token's, so that no two
// are equal and the lower token wins among equal logits.  Rows that have too many candidates (masks that leave
// fewer than `top`, many equal logits) are gone through again with lists (pick).
#include <type_traits>

#include "kvq_logprobs.h"
#include "paged.h"

namespace kvq {
namespace {

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kVec = 4;                         // 16-byte vectors of a thread a step
constexpr int kTop = KVQ_LOGPROBS_MAX_TOP;
constexpr int kList = 128;                      // candidates of a wave's list
constexpr int kSlots = 16;                      // maxima that a thread leaves
constexpr int kBlocks = 128;                    // of them, those that are read again
constexpr int kKeys = kWaves * kList;           // candidates of a work-group
constexpr int kMaxParts = 64;                   // work-groups of a row
constexpr float kLowest = -3.4028234664e38f;

struct LpArgs {
  const uint8_t* logits;
  int64_t row_bytes;
  const void* tokens;
  float* logprobs;
  float* entropy;
  float* top_logprobs;
  int64_t* top_tokens;
  float4v* sums;     // [rows][parts] maximum, two sums
  uint64_t* keys;    // [rows][parts][top]
  int64_t rows;
  int32_t vocab, top, parts, tokens64;
  float c, inv;      // log2(e) / T, 1 / T
};

// A softmax in the making: the maximum of x, the sum of e = 2^((x - m) c), and that of (x - m) e.
struct Sums {
  float m, l, s;
  __device__ __forceinline__ void to(float m2, float c) {  // a maximum at or above m
    const float d = m - shift_of(m2), f = fast_exp2(d * c);
    s = f == 0.f ? 0.f : f * fmaf(d, l, s);  // d may be -Inf, or its product with l
    l *= f;
    m = m2;
  }
  __device__ __forceinline__ void add(Sums o, float c) {
    const float m2 = fmaxf(m, o.m);
    to(m2, c);
    o.to(m2, c);
    l += o.l;
    s += o.s;
  }
  // A logit at or below the maximum.  -Inf x 0 is no 0: where there may be such logits they are CLAMPed.
  template <bool CLAMP>
  __device__ __forceinline__ void add_logit(float x, float c) {
    const float d = x - shift_of(m), p = fast_exp2(d * c);
    l += p;
    s = fmaf(CLAMP ? fmaxf(d, kLowest) : d, p, s);
  }
  __device__ __forceinline__ void lanes(float c) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) add(Sums{__shfl_xor(m, o, 64), __shfl_xor(l, o, 64), __shfl_xor(s, o, 64)}, c);
  }
};

__device__ __forceinline__ uint32_t order_of(float x) {  // rising with x; 0 for NaN
  const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.f);  // -0 is 0
  return x != x ? 0u : b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ uint64_t key_of(float x, uint32_t token) { return (uint64_t)order_of(x) << 32 | (uint32_t)~token; }
__device__ __forceinline__ float logit_of(uint64_t key) {
  const uint32_t o = (uint32_t)(key >> 32);
  return o == 0 ? __builtin_nanf("") : __builtin_bit_cast(float, o & 0x80000000u ? o & 0x7FFFFFFFu : ~o);
}

__device__ __forceinline__ uint64_t read_lane(uint64_t x, int lane) {
  return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(x >> 32), lane) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)x, lane);
}

// The k-th largest of a wave's 64 numbers, bit by bit: counting those above each takes a work-group 1 us more.
__device__ __forceinline__ uint32_t kth_largest(uint32_t x, int k) {
  uint32_t found = 0;
#pragma unroll
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t t = found | 1u << bit;
    if (__popcll(__ballot(x >= t)) >= k) found = t;
  }
  return found;
}

typedef __attribute__((address_space(3))) uint64_t lds_u64;

// A wave's candidates where there are many: `count` of them in its list, of which the best `top` are kept.
struct List {
  lds_u64* key;    // [kList], this wave's
  uint64_t bar;    // no key at or below it is among the best
  float low;       // its logit: nothing below it needs a look
  int count, top;

  __device__ __forceinline__ void raise(uint64_t b) {
    if (b <= bar) return;
    bar = b;
    const float x = logit_of(b);
    low = x == x ? x : kNegInf;
  }
  // Sorts the list and keeps the best.
  __device__ __attribute__((noinline)) static int cut(lds_u64* key, int count, int top) {
    const int lane = threadIdx.x & 63;
    const uint64_t a = lane < count ? key[lane] : 0, b = lane + 64 < count ? key[lane + 64] : 0;
    int ra = 0, rb = 0;
    for (int i = 0; i < count; ++i) {
      const uint64_t k = key[i];
      ra += k > a;
      rb += k > b;
    }
    __builtin_amdgcn_wave_barrier();
    if (lane < count && ra < top) key[ra] = a;
    if (lane + 64 < count && rb < top) key[rb] = b;
    __builtin_amdgcn_wave_barrier();
    return min(count, top);
  }
  __device__ __forceinline__ void cut() {
    count = cut(key, count, top);
    if (count == top) raise(read_lane(key[top - 1], 0));
  }
  // One value a lane.
  __device__ __forceinline__ void offer(uint64_t k, bool valid) {
    const int lane = threadIdx.x & 63;
    uint64_t in = __ballot(valid && k > bar);
    if (!in) return;
    if (count + __popcll(in) > kList) {
      cut();
      in = __ballot(valid && k > bar);
    }
    if (valid && k > bar) key[count + __popcll(in & ((1ull << lane) - 1))] = k;
    count += __popcll(in);
    __builtin_amdgcn_wave_barrier();
  }
};

template <class T>
__device__ __forceinline__ float value_at(const uint8_t* p) {
  if constexpr (std::is_same<T, float>::value) return *(const float*)p;
  else return T::to_f(*(const uint16_t*)p);
}

// A logit's log p.
struct LogP {
  float m, inv, log_l;
  bool none;
  __device__ __forceinline__ LogP(const LpArgs& a, const Sums& f) : m(f.m), inv(a.inv), log_l(logf(f.l)), none(f.m == kNegInf) {}
  __device__ __forceinline__ float operator()(float x) const { return none ? __builtin_nanf("") : fmaf(x - m, inv, -log_l); }
};

// Writes a row's log p of its token and its entropy.  One thread.
template <class T>
__device__ __forceinline__ void finish(const LpArgs& a, int64_t row, const Sums& f) {
  const LogP log_p(a, f);
  const float nan = __builtin_nanf("");
  a.entropy[row] = log_p.none ? nan : fmaxf(log_p.log_l - a.inv * (f.s / f.l), 0.f) + 0.f * f.l;
  if (!a.tokens) return;
  const int64_t t = a.tokens64 ? ((const int64_t*)a.tokens)[row] : ((const int32_t*)a.tokens)[row];
  a.logprobs[row] = t >= 0 && t < a.vocab ? log_p(value_at<T>(a.logits + row * a.row_bytes + t * (std::is_same<T, float>::value ? 4 : 2))) : nan;
}

// Calls out(place, key) for the best `top` of n keys in LDS, place by place, by any thread of the work-group.  Many are
// thinned out first, into `few` (room for n), by the logit of the top-th largest of 64 groups' largest: 380 keys, of 19
// parts, counted as they are take the join 13 us, so 4.5; from 32, 64 or 128 keys on takes as long.
template <class F>
__device__ __forceinline__ void best_of(const lds_u64* key, int n, int top, lds_u64* few, int* count, F out) {
  if (n > 2 * 64) {
    const int lane = threadIdx.x & 63;
    uint64_t mine = 0;
    for (int i = lane; i < n; i += 64) mine = key[i] > mine ? key[i] : mine;
    const uint64_t bar = (uint64_t)kth_largest((uint32_t)(mine >> 32), top) << 32;
    if (threadIdx.x == 0) *count = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kThreads)
      if (key[i] >= bar) few[atomicAdd(count, 1)] = key[i];
    __syncthreads();
    key = few;
    n = *count;
  }
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const uint64_t mine = key[i];
    int above = 0;
#pragma unroll 8
    for (int j = 0; j < n; ++j) above += key[j] > mine;
    if (above < top) out(above, mine);
  }
}
__device__ __forceinline__ void put_top(const LpArgs& a, int64_t row, const LogP& log_p, int place, uint64_t key) {
  a.top_tokens[row * a.top + place] = (int64_t)(uint32_t)~(uint32_t)key;
  a.top_logprobs[row * a.top + place] = log_p(logit_of(key));
}

// A work-group's part of a row.
template <class T>
struct Part {
  static constexpr int E = std::is_same<T, float>::value ? 4 : 8, S = 16 / E;  // logits of a vector, bytes of one
  const uint8_t* x0;
  const u32x4* v;   // the row's whole vectors, from its first aligned logit on: begin .. end - 1 of them are the part's
  int head, begin, end;
  int first, rest;  // logits before the first vector and behind the last, where they are this part's
  __device__ __forceinline__ Part(const LpArgs& a, int64_t row, int part) {
    x0 = a.logits + row * a.row_bytes;
    head = min((int)(((0u - (uint32_t)(uintptr_t)x0) & 15u) / S), a.vocab);
    const int vectors = (a.vocab - head) / E;
    v = (const u32x4*)(x0 + head * S);
    begin = (int)((int64_t)vectors * part / a.parts);
    end = (int)((int64_t)vectors * (part + 1) / a.parts);
    first = part == 0 ? head : 0;
    rest = part == 0 ? a.vocab - head - vectors * E : 0;
  }
  // token i of the first + rest
  __device__ __forceinline__ int edge(const LpArgs& a, int i) const { return i < first ? i : a.vocab - rest + i - first; }
  static __device__ __forceinline__ float logit(const u32x4& w, int e) {
    const uint32_t bits = w[e * 4 / E];
    if constexpr (E == 4) return __builtin_bit_cast(float, bits);
    else return T::to_f((uint16_t)(bits >> (e & 1 ? 16 : 0)));
  }
};

// The part's best, by lists, whatever there is in it: a wave's `top` best at a time are what the next have to pass.
// Leaves each wave's in its list, count[wave] of them.
template <class T>
__device__ __attribute__((noinline)) void pick(const LpArgs* a, const Part<T>* p, lds_u64* keys, int* count) {
  constexpr int E = Part<T>::E;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  List list{keys + wave * kList, 0, kNegInf, 0, a->top};
  for (int at = p->begin + wave * 64; at < p->end; at += kThreads) {
    const int i = at + lane;
    const bool there = i < p->end;
    u32x4 w = {0, 0, 0, 0};
    if (there) w = p->v[i];
    for (int e = 0; e < E; ++e) {
      // element e of a vector in registers, e not a constant
      const uint32_t lo = E == 4 ? (e < 2 ? (e ? w[1] : w[0]) : e == 2 ? w[2] : w[3])
                                 : (e < 4 ? (e < 2 ? w[0] : w[1]) : e < 6 ? w[2] : w[3]);
      float x;
      if constexpr (E == 4) x = __builtin_bit_cast(float, lo);
      else x = T::to_f((uint16_t)(lo >> (e & 1 ? 16 : 0)));
      if (__any(there && !(x < list.low))) list.offer(key_of(x, p->head + i * E + e), there);
    }
  }
  if (wave == 0) {
    const int n = p->first + p->rest, token = p->edge(*a, lane);
    list.offer(lane < n ? key_of(value_at<T>(p->x0 + (int64_t)token * Part<T>::S), token) : 0, lane < n);
  }
  list.cut();
  if (lane == 0) count[wave] = list.count;
}

static_assert(sizeof(float) * kSlots * kThreads >= sizeof(uint64_t) * kKeys, "the keys that are thinned out lie where the maxima were");

// A part of a row a work-group.
template <class T, bool TOP>
__global__ __launch_bounds__(kThreads) void logprobs_kernel(LpArgs a) {
  using P = Part<T>;
  constexpr int E = P::E;
  __shared__ __attribute__((aligned(8))) float maxima[TOP ? kSlots : 1][kThreads];  // and room for kKeys keys
  __shared__ uint64_t keys[TOP ? kKeys : 1];
  __shared__ uint32_t blocks[TOP ? kBlocks : 1];
  __shared__ Sums sums[kWaves];
  __shared__ float group[TOP ? kThreads : 1];
  __shared__ int counts[kWaves], n_blocks, n_keys;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t row = blockIdx.x / (uint32_t)a.parts;
  const int part = (int)(blockIdx.x % (uint32_t)a.parts);
  const P p(a, row, part);
  // a thread's steps, and how many of them a maximum is of
  const int steps = (p.end - p.begin + kThreads * kVec - 1) / (kThreads * kVec), per = (steps + kSlots - 1) / kSlots;
  if (TOP && tid == 0) n_blocks = n_keys = 0;

  Sums f{kNegInf, 0.f, 0.f};
  float most = kNegInf, all = kNegInf;  // of the slot, of all
  bool clamp = false;
  auto step = [&](int at, bool whole) {
    u32x4 w[kVec];
#pragma unroll
    for (int u = 0; u < kVec; ++u) {
      const int i = at + 64 * u + lane;
      if (whole || i < p.end) w[u] = ld_stream<u32x4>(p.v + i);
    }
    float x[kVec][E], mx = kNegInf;
#pragma unroll
    for (int u = 0; u < kVec; ++u) {
      const bool there = whole || at + 64 * u + lane < p.end;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        x[u][e] = there ? P::logit(w[u], e) : kNegInf;
        mx = fmaxf(mx, x[u][e]);
      }
    }
    if (mx > f.m) f.to(mx, a.c);
    // a step's sums by themselves, a vector's apart: short chains, in time and in rounding
    auto sum = [&](auto clamp) {
      Sums g[2] = {{f.m, 0.f, 0.f}, {f.m, 0.f, 0.f}};
#pragma unroll
      for (int u = 0; u < kVec; ++u)
#pragma unroll
        for (int e = 0; e < E; ++e) g[u & 1].template add_logit<decltype(clamp)::value>(x[u][e], a.c);
      return Sums{f.m, g[0].l + g[1].l, g[0].s + g[1].s};
    };
    // The clamp is one of eight instructions, 115 us for 109 at 2047 rows of 152064: a wave takes it from the first step on
    // that has a -Inf (or no number).
    Sums g;
    if (whole && !clamp) {
      g = sum(std::false_type{});
      clamp = __any(g.s != g.s);
    }
    if (!whole || clamp) g = sum(std::true_type{});
    f.l += g.l;
    f.s += g.s;
    most = fmaxf(most, mx);
  };
  {
    int at = p.begin + wave * 64 * kVec;
    for (int i = 0, slot = 0; slot < kSlots && i < steps; ++slot) {
      for (int j = 0; j < per && i < steps; ++j, ++i, at += kThreads * kVec) {
        if (at + 64 * kVec <= p.end) step(at, true);
        else if (at < p.end) step(at, false);
      }
      if constexpr (TOP) maxima[slot][tid] = most;
      all = fmaxf(all, most);
      most = kNegInf;
    }
  }
  if (wave == 0 && p.first + p.rest > 0) {  // fewer than 16
    const bool there = lane < p.first + p.rest;
    const float x = there ? value_at<T>(p.x0 + (int64_t)p.edge(a, lane) * P::S) : kNegInf;
    if (x > f.m) f.to(x, a.c);
    f.add_logit<true>(x, a.c);
  }
  f.lanes(a.c);
  if (lane == 0) sums[wave] = f;
  if constexpr (TOP) group[tid] = all;
  __syncthreads();
  if (!TOP && wave) return;
  f = sums[0];
  for (int w = 1; w < kWaves; ++w) f.add(sums[w], a.c);
  if (tid == 0) {
    if (a.parts == 1) finish<T>(a, row, f);
    else a.sums[row * a.parts + part] = float4v{f.m, f.l, f.s, 0.f};
  }
  if constexpr (TOP) {
    // the bar: the top-th largest of 64 groups' maxima
    float mine = group[lane];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) mine = fmaxf(mine, group[64 * w + lane]);
    const float bar = logit_of((uint64_t)kth_largest(order_of(mine), a.top) << 32);
    for (int slot = 0; slot * per < steps; ++slot)
      if (maxima[slot][tid] >= bar) {
        const int i = atomicAdd(&n_blocks, 1);
        if (i < kBlocks) blocks[i] = (uint32_t)(slot << 16 | tid);
      }
    if (tid < p.first + p.rest) {
      const int token = p.edge(a, tid);
      const float x = value_at<T>(p.x0 + (int64_t)token * P::S);
      keys[atomicAdd(&n_keys, 1)] = key_of(x, token);
    }
    __syncthreads();
    const int nb = n_blocks;
    bool many = nb > kBlocks || bar == kNegInf;
    if (!many) {
      for (int i = tid; i < nb * per * kVec; i += kThreads) {
        const uint32_t b = blocks[i / (per * kVec)];
        const int j = i % (per * kVec), it = (int)(b >> 16) * per + j / kVec, t = (int)(b & 0xFFFF);
        const int at = p.begin + (it * kThreads + (t >> 6) * 64) * kVec + 64 * (j % kVec) + (t & 63);
        if (it >= steps || at >= p.end) continue;
        const u32x4 w = p.v[at];
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const float x = P::logit(w, e);
          if (x >= bar) {
            const int k = atomicAdd(&n_keys, 1);
            if (k < kKeys) keys[k] = key_of(x, p.head + at * E + e);
          }
        }
      }
      __syncthreads();
      many = n_keys > kKeys;
    }
    int n = n_keys;
    if (many) {
      const LpArgs args = a;
      const P mine2 = p;
      __syncthreads();
      pick<T>(&args, &mine2, (lds_u64*)keys, counts);
      __syncthreads();
      // the lists one behind the other: each wave moves its own, which ends before the next one's begins
      n = 0;
      for (int w = 0; w < kWaves; ++w) {
        const int c = counts[w];
        const uint64_t k = tid < c ? keys[w * kList + tid] : 0;
        __syncthreads();
        if (tid < c) keys[n + tid] = k;
        __syncthreads();
        n += c;
      }
    }
    if (a.parts == 1) {
      const LogP log_p(a, f);
      best_of((const lds_u64*)keys, n, a.top, (lds_u64*)&maxima[0][0], &n_blocks, [&](int place, uint64_t key) { put_top(a, row, log_p, place, key); });
    } else {
      uint64_t* const out = a.keys + (row * a.parts + part) * a.top;
      for (int i = n + tid; i < a.top; i += kThreads) out[i] = 0;  // below all keys
      best_of((const lds_u64*)keys, n, a.top, (lds_u64*)&maxima[0][0], &n_blocks, [&](int place, uint64_t key) { out[place] = key; });
    }
  }
}

// Joins the parts of a row: a work-group.
template <class T>
__global__ __launch_bounds__(kThreads) void logprobs_join_kernel(LpArgs a) {
  __shared__ uint64_t keys[kMaxParts * kTop], few[kMaxParts * kTop];
  __shared__ int count;
  const int tid = threadIdx.x, lane = tid & 63;
  const int64_t row = blockIdx.x;
  const int n = a.parts * a.top;
  for (int i = tid; i < n; i += kThreads) keys[i] = a.keys[row * n + i];
  Sums f{kNegInf, 0.f, 0.f};
  if (lane < a.parts) {
    const float4v x = a.sums[row * a.parts + lane];
    f = Sums{x[0], x[1], x[2]};
  }
  f.lanes(a.c);
  if (tid == 0) finish<T>(a, row, f);
  if (!a.top) return;
  __syncthreads();
  const LogP log_p(a, f);
  best_of((const lds_u64*)keys, n, a.top, (lds_u64*)few, &count, [&](int place, uint64_t key) { put_top(a, row, log_p, place, key); });
}

// ---------------------------------------------------------------- host

// Work-groups that fill the GPU, and rows from which on each has one.  Rows of 151936 bf16 logits with 5 of the likeliest, us in a
// graph: 128 over 512, 1024 and 2048 work-groups 17.3, 18.0, 22.8; 256 24.4, 23.6, 27.2, one each 29.4; 400 34.8 over 2048, one
// each 32.6; 768 51 and 44.
constexpr int kFill = 512;
constexpr int kMost = 384;
// Rows of so few steps have one too: a launch and its workspace less.  One row of 32000 fp16 logits, called one by one, 14.8
// us, split 18.3 (in a graph a split one is 2 us faster); of 5 and more steps both take as long.
constexpr int kSolo = 4;

// Work-groups of a row: as many as fill the GPU, none of less than a step.
int parts_of(const kvq_token_logprobs_params& p) {
  const int64_t step = (int64_t)kThreads * kVec * (p.logits_type == KVQ_LOGITS_F32 ? 4 : 8);
  int64_t parts = p.rows > 0 && p.rows < kMost ? (kFill + p.rows - 1) / p.rows : 1;
  const int64_t most = ((int64_t)p.vocab + step - 1) / step;
  if (parts > most) parts = most;
  if (most <= kSolo) parts = 1;
  if (parts > kMaxParts) parts = kMaxParts;
  return (int)(parts < 1 ? 1 : parts);
}

int64_t sums_bytes(const kvq_token_logprobs_params& p, int parts) { return 16 * p.rows * parts; }

int check(const kvq_token_logprobs_params* p) {
  if (!p) return fail(KVQ_ERR_INVALID, "token logprobs: NULL params");
  if (p->rows < 0 || p->vocab < 1) return fail(KVQ_ERR_INVALID, "token logprobs: rows must not be negative and vocab positive");
  if (p->logits_type < KVQ_LOGITS_F16 || p->logits_type > KVQ_LOGITS_F32) return fail(KVQ_ERR_INVALID, "token logprobs: unknown type");
  if (p->top < 0 || p->top > kTop || p->top > p->vocab) return fail(KVQ_ERR_INVALID, "token logprobs: top must be 0 to 32 and at most vocab");
  // hotter, the sum of (x - m) e passes fp32: x - m still has a weight up to 100 T, and there are 2^28 of them
  if (!(p->inv_temperature >= 0.999e-30f) || !(p->inv_temperature <= 1.001e30f))
    return fail(KVQ_ERR_INVALID, "token logprobs: inv_temperature must be 1e-30 to 1e30");
  if (p->vocab > (1 << 28)) return fail(KVQ_ERR_UNSUPPORTED, "token logprobs: more than 2^28 tokens");
  if (p->rows * parts_of(*p) >= (1 << 24)) return fail(KVQ_ERR_UNSUPPORTED, "token logprobs: too many rows");
  return KVQ_OK;
}

template <class T>
int launch(const LpArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)(a.rows * a.parts));
  if (a.top) hipLaunchKernelGGL((logprobs_kernel<T, true>), grid, dim3(kThreads), 0, st, a);
  else hipLaunchKernelGGL((logprobs_kernel<T, false>), grid, dim3(kThreads), 0, st, a);
  int rc = launched();
  if (rc || a.parts == 1) return rc;
  hipLaunchKernelGGL(logprobs_join_kernel<T>, dim3((unsigned)a.rows), dim3(kThreads), 0, st, a);
  return launched();
}

int logprobs(const kvq_token_logprobs_params* p, hipStream_t st) {
  const int rc = check(p);
  if (rc) return rc;
  if (p->rows == 0) return KVQ_OK;
  const int item = p->logits_type == KVQ_LOGITS_F32 ? 4 : 2;
  if (!p->logits || !p->entropy || (p->tokens && !p->logprobs) || (p->top && (!p->top_logprobs || !p->top_tokens)))
    return fail(KVQ_ERR_INVALID, "token logprobs: NULL pointer");
  if ((uintptr_t)p->logits % item) return fail(KVQ_ERR_INVALID, "token logprobs: logits must be aligned to their elements");
  LpArgs a{};
  a.parts = parts_of(*p);
  const int64_t sums = sums_bytes(*p, a.parts), bytes = a.parts > 1 ? sums + 8 * p->rows * a.parts * p->top : 0;
  if (bytes && (!p->workspace || p->workspace_bytes < bytes || (uintptr_t)p->workspace % 16))
    return fail(KVQ_ERR_INVALID, "token logprobs: workspace too small or not 16-byte aligned");
  a.logits = (const uint8_t*)p->logits;
  a.row_bytes = p->row_stride * item;
  a.tokens = p->tokens; a.tokens64 = p->tokens64;
  a.logprobs = p->logprobs; a.entropy = p->entropy;
  a.top_logprobs = p->top_logprobs; a.top_tokens = p->top_tokens;
  a.sums = (float4v*)p->workspace;
  a.keys = (uint64_t*)((uint8_t*)p->workspace + sums);
  a.rows = p->rows; a.vocab = p->vocab; a.top = p->top;
  a.inv = p->inv_temperature;
  a.c = a.inv * kLog2e;
  if (p->logits_type == KVQ_LOGITS_F16) return launch<TF16>(a, st);
  if (p->logits_type == KVQ_LOGITS_BF16) return launch<TB16>(a, st);
  return launch<float>(a, st);
}

}  // namespace
}  // namespace kvq

extern "C" int kvq_token_logprobs(const kvq_token_logprobs_params* p, kvq_stream_t stream) {
  return kvq::guarded([&] { return kvq::logprobs(p, reinterpret_cast<hipStream_t>(stream)); });
}

extern "C" int64_t kvq_token_logprobs_workspace_bytes(const kvq_token_logprobs_params* p) {
  if (kvq::guarded([&] { return kvq::check(p); })) return 0;
  const int parts = kvq::parts_of(*p);
  return parts > 1 ? kvq::sums_bytes(*p, parts) + 8 * p->rows * parts * p->top : 0;
}
