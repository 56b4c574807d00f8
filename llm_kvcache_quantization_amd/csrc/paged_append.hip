// Append of K and V rows into pages, as they are or in INT8 (kvq_paged_append).
//
// 16 lanes take a token row of 128 values, 8 a lane: one 16-byte load, one store of 16 bytes (8 of
// codes), so that a wave instruction moves four whole rows.  The group's absmax is DPP steps within the
// 16 lanes.
//
// What bounds it: the launch for a step's rows (one token of 2 heads 2.3 us in the kernel); for prompts HBM and the
// chain length, page, row (4 padded prompts of up to 4095 tokens, 8 heads, bf16 to INT8 of groups of 32: 18.3 us a call,
// where a copy of their bytes takes 11.8; as they are 15.1, 5.0 TB/s, where a copy takes 15.4).
#include "paged.h"

#pragma clang fp contract(off)

namespace kvq {
namespace {

constexpr int kAppThreads = 256;
constexpr int kAppRows = kAppThreads / 16;  // rows a work-group takes at a time
constexpr int kAppTokens = 4 * kAppRows;    // tokens a work-group takes of a long prompt

struct AppSide {
  const uint8_t* x;
  int64_t sb, sh, ss;  // bytes
};
struct AppArgs {
  PagedCache c;
  AppSide side[2];
  const int32_t* write_pos;
  const int32_t* new_lens;
  int32_t seq_new;
  int64_t rows;  // batch * heads * seq_new
};

typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 h16x2 __attribute__((ext_vector_type(2)));

template <int CTRL>
__device__ __forceinline__ uint32_t dpp_max(uint32_t x) {
  return max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xf, 0xf, true));
}

// Codes of 8 values, and their group's scale: s = fp16(max(absmax, 1e-5) / 127), code = rint(fp16(x / s)) within
// +-127; zeros and a NaN scale for a group that is not all finite.
template <class T, int GS>
__device__ __forceinline__ u32x2 encode(const u32x4& w, half_t& sc) {
  // magnitudes order as their bits do, and those from Inf's on are not finite
  u16x2 t = __builtin_bit_cast(u16x2, w[0] & 0x7FFF7FFFu);
#pragma unroll
  for (int j = 1; j < 4; ++j) t = __builtin_elementwise_max(t, __builtin_bit_cast(u16x2, w[j] & 0x7FFF7FFFu));
  uint32_t top = max((uint32_t)t[0], (uint32_t)t[1]);
  // over the group's lanes: quad_perm [1,0,3,2] and [2,3,0,1], then half-row and row mirrors
  top = dpp_max<0xB1>(top);
  top = dpp_max<0x4E>(top);
  if (GS >= 64) top = dpp_max<0x141>(top);
  if (GS >= 128) top = dpp_max<0x140>(top);
  sc = (half_t)fminf(__fdiv_rn(fmaxf(T::to_f((uint16_t)top), 1e-5f), 127.0f), 65504.0f);
  const float sf = (float)sc, inv = __fdiv_rn(1.f, sf);
  uint32_t code[2] = {0, 0};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    h16x2 h;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      // x / s as the IEEE division has it, by one correction of x * (1 / s), which is within 2^-23: the remainder is
      // exact, the corrected value within 2^-46 before its rounding, and a quotient of two 11-bit significands
      // is no nearer than 2^-36 to a point between two floats.  (Where x is so small that the remainder underflows,
      // or x / s so large that fp16 has no room for it, the code is 0 or 127 all the same.)
      const float x = T::to_f((uint16_t)(w[j] >> 16 * k)), q = x * inv;
      h[k] = (_Float16)__builtin_fmaf(__builtin_fmaf(-q, sf, x), inv, q);
    }
    h = __builtin_elementwise_min(__builtin_elementwise_max(h, (h16x2){-127, -127}), (h16x2){127, 127});
#pragma unroll
    for (int k = 0; k < 2; ++k) code[j >> 1] |= (uint32_t)(uint8_t)(int8_t)__builtin_rintf16(h[k]) << (16 * (j & 1) + 8 * k);
  }
  if (top >= T::kInf) {
    code[0] = code[1] = 0;
    sc = __builtin_bit_cast(half_t, (uint16_t)0x7E00);
  }
  return u32x2{code[0], code[1]};
}

// The place of a row: its page (or none) and its slot.
struct AppPlace {
  int32_t page, slot;
  __device__ __forceinline__ AppPlace(const PagedCache& pc, uint32_t b, int64_t pos, bool there) {
    page = -1;
    if (there && pos >= 0 && pos < ((int64_t)pc.max_pages << pc.lg)) page = pc.table[b * pc.table_stride + (pos >> pc.lg)];
    slot = (int32_t)pos & pc.page_mask;
  }
};

template <class T, int GS>  // GS 0: rows as they are; else INT8 in groups of GS
__device__ __forceinline__ void put(const PagedCache& pc, int side, uint32_t h, const AppPlace& at, const u32x4& w, int c) {
  if ((uint32_t)at.page >= (uint32_t)pc.num_pages) return;
  uint8_t* dst = side ? pc.v + at.page * pc.vsp + h * pc.vsh + at.slot * pc.vst : pc.k + at.page * pc.ksp + h * pc.ksh + at.slot * pc.kst;
  if constexpr (GS == 0) {
    *(u32x4*)(dst + c * 16) = w;
  } else {
    half_t sc;
    *(u32x2*)(dst + c * 8) = encode<T, GS>(w, sc);
    constexpr int G = 128 / GS;
    if (c % (GS / 8) == 0) {
      uint8_t* so = side ? pc.vs + at.page * pc.vssp + h * pc.vssh : pc.ks + at.page * pc.kssp + h * pc.kssh;
      ((half_t*)so)[at.slot * G + c / (GS / 8)] = sc;
    }
  }
}

// Few new tokens a sequence: the rows of all sequences and heads in one line, a row per 16 lanes.
template <class T, int GS>
__global__ __launch_bounds__(kAppThreads) void paged_append_kernel(AppArgs a) {
  const int side = blockIdx.y, c = threadIdx.x & 15;
  const AppSide s = a.side[side];
  const PagedCache& pc = a.c;
  const int64_t step = (int64_t)gridDim.x * kAppRows;
  for (int64_t row = (int64_t)blockIdx.x * kAppRows + (threadIdx.x >> 4); row < a.rows; row += step) {
    const uint32_t i = (uint32_t)row % (uint32_t)a.seq_new, bh = (uint32_t)row / (uint32_t)a.seq_new;
    const uint32_t b = bh / (uint32_t)pc.kv_heads, h = bh % (uint32_t)pc.kv_heads;
    const int64_t pos = (int64_t)a.write_pos[b] + i;
    if (a.new_lens && (int32_t)i >= a.new_lens[b]) continue;
    const u32x4 w = *(const u32x4*)(s.x + b * s.sb + h * s.sh + i * s.ss + c * 16);
    put<T, GS>(pc, side, h, AppPlace(pc, b, pos, true), w, c);
  }
}

// kAppTokens and more: a work-group takes as many consecutive tokens of a sequence and head, four rows a thread with
// their loads side by side (the kernel alone on the prompts above 19.6 us; in one line 21.4; two or eight rows a thread
// 19.7 and 23.8).
template <class T, int GS>
__global__ __launch_bounds__(kAppThreads) void paged_append_long_kernel(AppArgs a) {
  constexpr int R = kAppTokens / kAppRows;
  const int side = blockIdx.y, c = threadIdx.x & 15;
  const AppSide s = a.side[side];
  const PagedCache& pc = a.c;
  const uint32_t chunks = (uint32_t)(a.seq_new + kAppTokens - 1) / kAppTokens, blocks = chunks * (uint32_t)(a.rows / a.seq_new);
  for (uint32_t at = blockIdx.x; at < blocks; at += gridDim.x) {
    const uint32_t i0 = at % chunks * kAppTokens, bh = at / chunks, b = bh / (uint32_t)pc.kv_heads, h = bh % (uint32_t)pc.kv_heads;
    const int32_t n = a.new_lens ? min(a.new_lens[b], a.seq_new) : a.seq_new;
    if ((int32_t)i0 >= n) continue;
    const int64_t pos0 = a.write_pos[b];
    const uint8_t* const x = s.x + b * s.sb + h * s.sh + c * 16;
    u32x4 w[R];
    int32_t i[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      i[r] = i0 + r * kAppRows + (threadIdx.x >> 4);
      w[r] = *(const u32x4*)(x + min(i[r], n - 1) * s.ss);
    }
    AppPlace place[R] = {{pc, b, pos0 + i[0], i[0] < n}, {pc, b, pos0 + i[1], i[1] < n}, {pc, b, pos0 + i[2], i[2] < n}, {pc, b, pos0 + i[3], i[3] < n}};
#pragma unroll
    for (int r = 0; r < R; ++r) put<T, GS>(pc, side, h, place[r], w[r], c);
  }
}

int append(const kvq_paged_append_params* p, hipStream_t st) {
  if (!p) return fail(KVQ_ERR_INVALID, "paged append: NULL params");
  AppArgs a{};
  int rc = paged_cache(p->cache, a.c);
  if (rc || (rc = paged_written(a.c))) return rc;
  if (p->seq_new < 0) return fail(KVQ_ERR_INVALID, "paged append: negative seq_new");
  // a row holds no more, and places of a work-group's share past the end stay in 32 bits
  if (p->seq_new > (1 << 30)) return fail(KVQ_ERR_UNSUPPORTED, "paged append: more than 2^30 new tokens");
  if (p->x_type != KVQ_PAGED_F16 && p->x_type != KVQ_PAGED_BF16) return fail(KVQ_ERR_INVALID, "paged append: unknown x_type");
  const int fmt = p->cache.format;
  if (fmt != KVQ_PAGED_INT8 && fmt != p->x_type) return fail(KVQ_ERR_INVALID, "paged append: the pages' type is another than the rows'");
  a.rows = (int64_t)a.c.batch * a.c.kv_heads * p->seq_new;
  if (a.rows == 0 || a.c.num_pages == 0 || a.c.max_pages == 0) return KVQ_OK;
  if (a.rows > (int64_t)1 << 31) return fail(KVQ_ERR_UNSUPPORTED, "paged append: too many rows");
  if (!p->k || !p->v || !p->write_pos) return fail(KVQ_ERR_INVALID, "paged append: NULL pointer");
  a.side[0] = AppSide{(const uint8_t*)p->k, 2 * p->k_stride_b, 2 * p->k_stride_h, 2 * p->k_stride_s};
  a.side[1] = AppSide{(const uint8_t*)p->v, 2 * p->v_stride_b, 2 * p->v_stride_h, 2 * p->v_stride_s};
  for (const AppSide& s : a.side)
    if (((uintptr_t)s.x | (uintptr_t)s.sb | (uintptr_t)s.sh | (uintptr_t)s.ss) % 16)
      return fail(KVQ_ERR_INVALID, "paged append: rows must be 16-byte aligned");
  a.write_pos = p->write_pos;
  a.new_lens = p->new_lens;
  a.seq_new = p->seq_new;
  const bool lng = a.seq_new >= kAppTokens;
  int64_t gx = lng ? a.rows / a.seq_new * ((a.seq_new + kAppTokens - 1) / kAppTokens) : (a.rows + kAppRows - 1) / kAppRows;
  if (gx > 65536) gx = 65536;
  const dim3 grid((unsigned)gx, 2), block(kAppThreads);
  const bool b16 = p->x_type == KVQ_PAGED_BF16;
  const int gs = fmt == KVQ_PAGED_INT8 ? p->cache.group_size : 0;
#define KVQ_APP(T, G)                                                            \
  if (lng) hipLaunchKernelGGL((paged_append_long_kernel<T, G>), grid, block, 0, st, a); \
  else hipLaunchKernelGGL((paged_append_kernel<T, G>), grid, block, 0, st, a)
  if (gs == 0) { KVQ_APP(TF16, 0); }  // a copy of 16-bit values, whatever they are
  else if (gs == 32) { if (b16) { KVQ_APP(TB16, 32); } else { KVQ_APP(TF16, 32); } }
  else if (gs == 64) { if (b16) { KVQ_APP(TB16, 64); } else { KVQ_APP(TF16, 64); } }
  else { if (b16) { KVQ_APP(TB16, 128); } else { KVQ_APP(TF16, 128); } }
#undef KVQ_APP
  return launched();
}

}  // namespace
}  // namespace kvq

extern "C" int kvq_paged_append(const kvq_paged_append_params* p, kvq_stream_t stream) {
  return kvq::guarded([&] { return kvq::append(p, reinterpret_cast<hipStream_t>(stream)); });
}
