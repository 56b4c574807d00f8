// Append of K and V rows into pages, as they are or in INT8 (kvq_paged_append).
//
// 16 lanes take a token row of 128 values, 8 a lane: one 16-byte load, one store of 16 bytes (8 of
// codes), so that a wave instruction moves four whole rows.  The group's absmax is DPP steps within the
// 16 lanes.  The division is the IEEE one (the framework's codes rest on its rounding).
//
// What bounds it: a launch for a step's rows, HBM for prompts.
#include "paged.h"

#pragma clang fp contract(off)

namespace kvq {
namespace {

constexpr int kAppThreads = 256;
constexpr int kAppRows = kAppThreads / 16;  // rows a work-group takes at a time

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

template <class T, int GS>  // GS 0: rows as they are; else INT8 in groups of GS
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
    if (pos < 0 || pos >= ((int64_t)pc.max_pages << pc.lg)) continue;
    const u32x4 w = *(const u32x4*)(s.x + b * s.sb + h * s.sh + i * s.ss + c * 16);
    const int32_t page = pc.table[b * pc.table_stride + (pos >> pc.lg)];
    if ((uint32_t)page >= (uint32_t)pc.num_pages) continue;
    const int32_t slot = (int32_t)pos & pc.page_mask;
    uint8_t* dst = side ? pc.v + page * pc.vsp + h * pc.vsh + slot * pc.vst : pc.k + page * pc.ksp + h * pc.ksh + slot * pc.kst;
    if constexpr (GS == 0) {
      *(u32x4*)(dst + c * 16) = w;
    } else {
      half_t sc;
      *(u32x2*)(dst + c * 8) = encode<T, GS>(w, sc);
      constexpr int G = 128 / GS;
      if (c % (GS / 8) == 0) {
        uint8_t* so = side ? pc.vs + page * pc.vssp + h * pc.vssh : pc.ks + page * pc.kssp + h * pc.kssh;
        ((half_t*)so)[slot * G + c / (GS / 8)] = sc;
      }
    }
  }
}

int append(const kvq_paged_append_params* p, hipStream_t st) {
  if (!p) return fail(KVQ_ERR_INVALID, "paged append: NULL params");
  AppArgs a{};
  const int rc = paged_cache(p->cache, a.c);
  if (rc) return rc;
  if (p->seq_new < 0) return fail(KVQ_ERR_INVALID, "paged append: negative seq_new");
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
  int64_t gx = (a.rows + kAppRows - 1) / kAppRows;
  if (gx > 65536) gx = 65536;
  const dim3 grid((unsigned)gx, 2), block(kAppThreads);
  const bool b16 = p->x_type == KVQ_PAGED_BF16;
  const int gs = fmt == KVQ_PAGED_INT8 ? p->cache.group_size : 0;
#define KVQ_APP(T, G) hipLaunchKernelGGL((paged_append_kernel<T, G>), grid, block, 0, st, a)
  if (gs == 0) KVQ_APP(TF16, 0);  // a copy of 16-bit values, whatever they are
  else if (gs == 32) { if (b16) KVQ_APP(TB16, 32); else KVQ_APP(TF16, 32); }
  else if (gs == 64) { if (b16) KVQ_APP(TB16, 64); else KVQ_APP(TF16, 64); }
  else { if (b16) KVQ_APP(TB16, 128); else KVQ_APP(TF16, 128); }
#undef KVQ_APP
  return launched();
}

}  // namespace
}  // namespace kvq

extern "C" int kvq_paged_append(const kvq_paged_append_params* p, kvq_stream_t stream) {
  return kvq::guarded([&] { return kvq::append(p, reinterpret_cast<hipStream_t>(stream)); });
}
