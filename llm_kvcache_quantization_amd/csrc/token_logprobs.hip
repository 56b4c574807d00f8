// Log probabilities of given tokens, entropy and the likeliest tokens of rows of logits (kvq_token_logprobs).
//
//   p = softmax(x / T),  log p_t = (x_t - m) / T - log l,  H = log l - sum (x - m) / T e^((x - m) / T) / l,
//   l = sum e^((x - m) / T)
//
// One pass over the logits: each thread keeps a running maximum m and the two sums in fp32.  What bounds it: HBM; few
// rows are split over work-groups, whose parts a second launch joins.
//
// The likeliest: a wave keeps a list of candidates of its own in LDS, and what all but its `top` best are below.  A
// vector is looked at only where its largest logit reaches that bar.  A candidate is one whole number, the
// logit's order above the complement of the token's, so that no two are equal and the lower token wins among equal
// logits; a list that is full is cut down to its best by counting, for each, how many are above it.  Sorted lists
// (of waves, then of work-groups) are joined by taking the largest of their heads, `top` times.
#include <type_traits>

#include "kvq_logprobs.h"
#include "paged.h"

namespace kvq {
namespace {

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kVec = 4;                         // 16-byte vectors of a thread a step
constexpr int kTop = KVQ_LOGPROBS_MAX_TOP;
constexpr int kList = 128;                      // candidates of a wave
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
  __device__ __forceinline__ void add_logit(float x, float c) {  // at or below the maximum
    const float d = x - shift_of(m), p = fast_exp2(d * c);
    l += p;
    s = fmaf(fmaxf(d, kLowest), p, s);  // -Inf x 0 would be no 0
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

typedef __attribute__((address_space(3))) uint64_t lds_u64;

// A wave's candidates: `count` of them in its list, of which the best `top` are kept.
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

// The k-th largest of the lanes' values: as many values as that are at or above it.
__device__ __forceinline__ float kth_of_lanes(float x, int k) {
  const int lane = threadIdx.x & 63;
  int above = 0;
#pragma unroll 8
  for (int i = 0; i < 64; ++i) {
    const float y = row_lane(x, i);
    above += y > x || (y == x && i < lane);
  }
  return row_lane(x, __builtin_ctzll(__ballot(above == k - 1)));
}

// The `top` largest keys of up to 64 sorted lists (lane p: list p of `have` keys); lane i < top has the i-th.
__device__ __forceinline__ uint64_t best_of(const lds_u64* list, int have, int top) {
  const int lane = threadIdx.x & 63;
  int at = 0;
  uint64_t head = have > 0 ? list[0] : 0, mine = 0;
  for (int i = 0; i < top; ++i) {
    uint64_t best = head;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      const uint64_t other = __shfl_xor((unsigned long long)best, o, 64);
      best = other > best ? other : best;
    }
    if (lane == i) mine = best;
    if (head == best) head = ++at < have ? list[at] : 0;  // no two keys are equal, but for the 0 of an empty list
  }
  return mine;
}

template <class T>
__device__ __forceinline__ float value_at(const uint8_t* p) {
  if constexpr (std::is_same<T, float>::value) return *(const float*)p;
  else return T::to_f(*(const uint16_t*)p);
}

// Writes a row's outputs from its sums and, in the lanes, its best keys.  One wave.
template <class T>
__device__ __forceinline__ void finish(const LpArgs& a, int64_t row, Sums f, uint64_t key) {
  const int lane = threadIdx.x & 63;
  const float log_l = logf(f.l), nan = __builtin_nanf("");
  const bool none = f.m == kNegInf;
  auto log_p = [&](float x) { return none ? nan : fmaf(x - f.m, a.inv, -log_l); };
  if (lane == 0) {
    a.entropy[row] = none ? nan : fmaxf(log_l - a.inv * (f.s / f.l), 0.f) + 0.f * f.l;
    if (a.tokens) {
      const int64_t t = a.tokens64 ? ((const int64_t*)a.tokens)[row] : ((const int32_t*)a.tokens)[row];
      a.logprobs[row] = t >= 0 && t < a.vocab
                            ? log_p(value_at<T>(a.logits + row * a.row_bytes + t * (std::is_same<T, float>::value ? 4 : 2))) : nan;
    }
  }
  if (lane < a.top) {
    a.top_tokens[row * a.top + lane] = (int64_t)(uint32_t)~(uint32_t)key;
    a.top_logprobs[row * a.top + lane] = log_p(logit_of(key));
  }
}

template <class T, bool TOP>
__global__ __launch_bounds__(kThreads) void logprobs_kernel(LpArgs a) {
  constexpr int E = std::is_same<T, float>::value ? 4 : 8, S = 16 / E;  // logits of a vector, bytes of one
  __shared__ uint64_t keys[TOP ? kWaves * kList : 1];
  __shared__ Sums sums[kWaves];
  __shared__ int counts[kWaves];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t parts = (uint32_t)a.parts;
  const int64_t row = blockIdx.x / parts;
  const int part = (int)(blockIdx.x % parts);
  const uint8_t* const x0 = a.logits + row * a.row_bytes;
  // the row's whole vectors, from its first aligned logit on, and this work-group's share of them
  const int head = min((int)(((0u - (uint32_t)(uintptr_t)x0) & 15u) / S), a.vocab), vectors = (a.vocab - head) / E;
  const u32x4* const v = (const u32x4*)(x0 + head * S);
  const int begin = (int)((int64_t)vectors * part / a.parts), end = (int)((int64_t)vectors * (part + 1) / a.parts);

  Sums f{kNegInf, 0.f, 0.f};
  List list{(lds_u64*)keys + (TOP ? wave * kList : 0), 0, kNegInf, 0, a.top};
  auto step = [&](int at, bool whole) {
    u32x4 w[kVec];
#pragma unroll
    for (int u = 0; u < kVec; ++u) {
      const int i = at + 64 * u + lane;
      if (whole || i < end) w[u] = ld_stream<u32x4>(v + i);
    }
    float x[kVec][E], top[kVec];
#pragma unroll
    for (int u = 0; u < kVec; ++u) {
      const bool there = whole || at + 64 * u + lane < end;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const uint32_t bits = w[u][e * 4 / E];
        if constexpr (E == 4) x[u][e] = __builtin_bit_cast(float, bits);
        else x[u][e] = T::to_f((uint16_t)(bits >> (e & 1 ? 16 : 0)));
        if (!there) x[u][e] = kNegInf;
      }
      top[u] = x[u][0];
#pragma unroll
      for (int e = 1; e < E; ++e) top[u] = fmaxf(top[u], x[u][e]);
    }
    float mx = top[0];
#pragma unroll
    for (int u = 1; u < kVec; ++u) mx = fmaxf(mx, top[u]);
    if (mx > f.m) f.to(mx, a.c);
#pragma unroll
    for (int u = 0; u < kVec; ++u)
#pragma unroll
      for (int e = 0; e < E; ++e) f.add_logit(x[u][e], a.c);
    if constexpr (TOP) {
      const bool first = list.bar == 0;
      if (first) list.low = fmaxf(list.low, kth_of_lanes(mx == mx ? mx : kNegInf, list.top));  // that many reach it
#pragma unroll
      for (int u = 0; u < kVec; ++u) {
        if (!__any(!(top[u] < list.low))) continue;
        const int i = at + 64 * u + lane;
        const bool there = whole || i < end;
#pragma unroll
        for (int e = 0; e < E; ++e) list.offer(key_of(x[u][e], head + i * E + e), there && !(x[u][e] < list.low));
      }
      if (first) list.cut();
    }
  };
  int at = begin + wave * 64 * kVec;
  for (; at + 64 * kVec <= end; at += kThreads * kVec) step(at, true);
  if (at < end) step(at, false);
  // the logits before the first vector and behind the last: fewer than 16
  if (part == 0 && wave == 0) {
    const int rest = a.vocab - head - vectors * E;
    const bool there = lane < head + rest;
    const int token = lane < head ? lane : a.vocab - rest + lane - head;
    const float x = there ? value_at<T>(x0 + token * S) : kNegInf;
    if (x > f.m) f.to(x, a.c);
    f.add_logit(x, a.c);
    if constexpr (TOP) list.offer(key_of(x, token), there);
  }

  // the lanes' sums, then the waves'
  f.lanes(a.c);
  if constexpr (TOP) list.cut();
  if (lane == 0) {
    sums[wave] = f;
    counts[wave] = list.count;
  }
  __syncthreads();
  if (wave) return;
  f = sums[0];
  for (int w = 1; w < kWaves; ++w) f.add(sums[w], a.c);
  uint64_t key = 0;
  if constexpr (TOP) key = best_of((lds_u64*)keys + (lane < kWaves ? lane : 0) * kList, lane < kWaves ? counts[lane] : 0, a.top);
  if (a.parts == 1) {
    finish<T>(a, row, f, key);
    return;
  }
  if (lane == 0) a.sums[row * a.parts + part] = float4v{f.m, f.l, f.s, 0.f};
  if (TOP && lane < a.top) a.keys[(row * a.parts + part) * a.top + lane] = key;
}

// Joins the parts of a row: a wave.
template <class T>
__global__ __launch_bounds__(64) void logprobs_join_kernel(LpArgs a) {
  __shared__ uint64_t keys[kMaxParts * kTop];
  const int lane = threadIdx.x;
  const int64_t row = blockIdx.x;
  Sums f{kNegInf, 0.f, 0.f};
  if (lane < a.parts) {
    const float4v x = a.sums[row * a.parts + lane];
    f = Sums{x[0], x[1], x[2]};
  }
  f.lanes(a.c);
  uint64_t key = 0;
  if (a.top) {
    for (int i = lane; i < a.parts * a.top; i += 64) keys[i] = a.keys[row * a.parts * a.top + i];
    __syncthreads();
    // a part of fewer logits ends its list with zeros, which are below all keys
    key = best_of((lds_u64*)keys + (lane < a.parts ? lane * a.top : 0), lane < a.parts ? a.top : 0, a.top);
  }
  finish<T>(a, row, f, key);
}

// ---------------------------------------------------------------- host

constexpr int kFill = 2048;  // work-groups that fill the GPU

// Work-groups of a row: as many as fill the GPU, none of less than a step.
int parts_of(const kvq_token_logprobs_params& p) {
  const int64_t step = (int64_t)kThreads * kVec * (p.logits_type == KVQ_LOGITS_F32 ? 4 : 8);
  int64_t parts = p.rows > 0 ? (kFill + p.rows - 1) / p.rows : 1;
  const int64_t most = ((int64_t)p.vocab + step - 1) / step;
  if (parts > most) parts = most;
  if (parts > kMaxParts) parts = kMaxParts;
  return (int)(parts < 1 ? 1 : parts);
}

int64_t sums_bytes(const kvq_token_logprobs_params& p, int parts) { return 16 * p.rows * parts; }

int check(const kvq_token_logprobs_params* p) {
  if (!p) return fail(KVQ_ERR_INVALID, "token logprobs: NULL params");
  if (p->rows < 0 || p->vocab < 1) return fail(KVQ_ERR_INVALID, "token logprobs: rows must not be negative and vocab positive");
  if (p->logits_type < KVQ_LOGITS_F16 || p->logits_type > KVQ_LOGITS_F32) return fail(KVQ_ERR_INVALID, "token logprobs: unknown type");
  if (p->top < 0 || p->top > kTop || p->top > p->vocab) return fail(KVQ_ERR_INVALID, "token logprobs: top must be 0 to 32 and at most vocab");
  if (!(p->inv_temperature > 0.f) || !(p->inv_temperature < 1e30f)) return fail(KVQ_ERR_INVALID, "token logprobs: inv_temperature must be positive and finite");
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
  hipLaunchKernelGGL(logprobs_join_kernel<T>, dim3((unsigned)a.rows), dim3(64), 0, st, a);
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
