// Copies of pages, of the pools of all layers at once (kvq_copy_pages).
//
// What bounds it: the bytes, read once and written once (1000 pages of 64 KB in 8 pools, 524 MB each way: 189 us, 5.5 TB/s); a
// fork's few pages the launch (3 pages of 8 KB in 56 pools 3.4 us in a graph).  A work-group takes
// kChunk 16-byte pieces of one page of one pool, those that are copied counted through.  Up to kPools pools go into one
// launch, in its arguments.
#include "paged.h"
#include "kvq_shared.h"

namespace kvq {
namespace {

constexpr int kPools = 60;                  // of a launch: 48 bytes each, in 4 KB of arguments
constexpr int kThreads = 256;
constexpr int kPer = 8;                     // pieces a thread
constexpr int kChunk = kThreads * kPer;

// A pool's two sides.  Strides in pieces of 16 bytes.
struct CopyPool {
  const u32x4* from;
  u32x4* to;
  uint32_t fp, fh, ft, tp, th, tt;
  uint8_t lg_head;   // pieces of a head's slots, log2
  uint8_t lg_row;    // pieces of a row, log2; as lg_head where the slots lie one behind the other on both sides
  uint8_t lg_slot;   // bytes of a slot, log2
  uint8_t pad[5];
};

struct CopyArgs {
  const int32_t* src;
  const int32_t* dst;
  const int32_t* lens;
  uint32_t pairs, heads, from_pages, to_pages;
  int32_t page_size;
  CopyPool pool[kPools];
};

// STREAM: stores past the caches, for more than they hold.
template <bool STREAM>
__global__ __launch_bounds__(kThreads) void copy_pages_kernel(CopyArgs a) {
  const CopyPool& p = a.pool[blockIdx.z];
  const uint32_t pair = blockIdx.y;
  const uint32_t src = (uint32_t)a.src[pair], dst = (uint32_t)a.dst[pair];
  if (src >= a.from_pages || dst >= a.to_pages) return;  // a page that is not there
  const int n = a.lens ? min(max(a.lens[pair], 0), a.page_size) : a.page_size;
  const uint32_t bytes = (uint32_t)n << p.lg_slot;  // of a head
  const u32x4* const from = p.from + (uint64_t)src * p.fp;
  u32x4* const to = p.to + (uint64_t)dst * p.tp;
  // pieces of a head that are copied, and of all heads one behind the other
  const uint32_t pieces = (bytes + 15) / 16, count = a.heads * pieces;
  const float inv = 1.0f / (float)pieces;
  for (uint32_t v0 = blockIdx.x * kChunk; v0 < count; v0 += gridDim.x * kChunk) {
    u32x4 x[kPer];
    uint32_t head[kPer], w[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const uint32_t v = min(v0 + j * kThreads + threadIdx.x, count - 1);
      // v / pieces, below 2^12 heads: the quotient in fp32 is off by at most one
      uint32_t h = min((uint32_t)((float)v * inv), a.heads - 1);
      while (h * pieces > v) --h;
      while ((h + 1) * pieces <= v) ++h;
      head[j] = h;
      w[j] = v - h * pieces;
      const uint32_t row = w[j] >> p.lg_row, col = w[j] & ((1u << p.lg_row) - 1);
      x[j] = ld_stream<u32x4>(from + (uint64_t)h * p.fh + (uint64_t)row * p.ft + col);
    }
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      if (v0 + j * kThreads + threadIdx.x >= count) break;
      const uint32_t row = w[j] >> p.lg_row, col = w[j] & ((1u << p.lg_row) - 1), at = w[j] * 16;
      u32x4* const o = to + (uint64_t)head[j] * p.th + (uint64_t)row * p.tt + col;
      if (at + 16 <= bytes) {
        if constexpr (STREAM) __builtin_nontemporal_store(x[j], o);
        else *o = x[j];
      } else {  // slots of 2, 4 or 8 bytes may end inside a piece
        for (uint32_t b = 0; at + b < bytes; b += 2) ((uint16_t*)o)[b / 2] = (uint16_t)(x[j][b / 4] >> (b & 2 ? 16 : 0));
      }
    }
  }
}

// ---------------------------------------------------------------- host

bool side(const kvq_page_pool& s, int page_size, bool written, int pages, int heads) {
  const bool rows = s.row_bytes >= 16;
  if (!s.base || ((uintptr_t)s.base | (uintptr_t)s.stride_p | (uintptr_t)s.stride_h) % 16) return false;
  if (rows ? s.stride_t % 16 || s.stride_t < s.row_bytes : s.stride_t != s.row_bytes) return false;
  const int64_t top = (int64_t)16 << 31;  // strides are held in 31 bits of pieces
  if (s.stride_p < 0 || s.stride_h < 0 || s.stride_p >= top || s.stride_h >= top || s.stride_t >= top) return false;
  return !written || ((pages <= 1 || s.stride_p > 0) && (heads <= 1 || s.stride_h > 0));
}

int copy_pages(const kvq_copy_pages_params* p, hipStream_t st) {
  if (!p) return fail(KVQ_ERR_INVALID, "copy pages: NULL params");
  if (p->n_pools < 0 || p->pairs < 0 || p->heads <= 0 || p->from_pages < 0 || p->to_pages < 0)
    return fail(KVQ_ERR_INVALID, "copy pages: negative size");
  if (p->page_size < 16 || p->page_size > 256 || (p->page_size & (p->page_size - 1)))
    return fail(KVQ_ERR_INVALID, "copy pages: page_size must be 16, 32, 64, 128 or 256");
  if (p->heads > 4096) return fail(KVQ_ERR_UNSUPPORTED, "copy pages: too many heads");
  if (p->n_pools == 0 || p->pairs == 0 || p->from_pages == 0 || p->to_pages == 0) return KVQ_OK;
  if (!p->from || !p->to || !p->src || !p->dst) return fail(KVQ_ERR_INVALID, "copy pages: NULL pointer");
  for (int i = 0; i < p->n_pools; ++i) {
    const kvq_page_pool &f = p->from[i], &t = p->to[i];
    if (f.row_bytes < 2 || f.row_bytes > 1024 || (f.row_bytes & (f.row_bytes - 1)) || t.row_bytes != f.row_bytes)
      return fail(KVQ_ERR_INVALID, "copy pages: rows must have 2 to 1024 bytes, a power of two, alike on both sides");
    if (!side(f, p->page_size, false, p->from_pages, p->heads) || !side(t, p->page_size, true, p->to_pages, p->heads))
      return fail(KVQ_ERR_INVALID, "copy pages: pools must be 16-byte aligned, with strides that are too, rows of less than 16 "
                                   "bytes dense, and memory of their own where they are written");
  }
  const auto lg = [](int64_t x) { return (uint8_t)__builtin_ctzll((unsigned long long)x); };
  // 1000 pages of 64 KB in 8 pools, 524 MB: 189 us with stores past the caches, 199 without; a fork's few pages are read soon
  int64_t all = 0;
  for (int i = 0; i < p->n_pools; ++i) all += (int64_t)p->page_size * p->from[i].row_bytes * p->heads;
  const bool stream = !p->lens && all * p->pairs > ((int64_t)1 << 28);
  for (int i0 = 0; i0 < p->n_pools; i0 += kPools) {
    CopyArgs a{};
    const int n = p->n_pools - i0 < kPools ? p->n_pools - i0 : kPools;
    uint32_t chunks = 0;
    for (int i = 0; i < n; ++i) {
      const kvq_page_pool &f = p->from[i0 + i], &t = p->to[i0 + i];
      CopyPool& c = a.pool[i];
      c.from = (const u32x4*)f.base; c.to = (u32x4*)t.base;
      c.fp = (uint32_t)(f.stride_p / 16); c.fh = (uint32_t)(f.stride_h / 16); c.ft = (uint32_t)(f.stride_t / 16);
      c.tp = (uint32_t)(t.stride_p / 16); c.th = (uint32_t)(t.stride_h / 16); c.tt = (uint32_t)(t.stride_t / 16);
      c.lg_slot = lg(f.row_bytes);
      c.lg_head = lg((int64_t)p->page_size * f.row_bytes / 16);
      c.lg_row = f.stride_t == f.row_bytes && t.stride_t == t.row_bytes ? c.lg_head : lg(f.row_bytes / 16);
      const uint32_t all = (uint32_t)p->heads << c.lg_head, x = (all + kChunk - 1) / kChunk;  // at most 2^12 * 2^14
      chunks = x > chunks ? x : chunks;
    }
    // Parts of pages: a work-group a page where that is enough of them, or half of them find nothing to copy: 31 pairs of 48
    // pools of 64 KB, of which 19 of 64 slots, 16.4 us, so 13.9
    if (p->lens && (int64_t)n * p->pairs >= 1024) chunks = 1;
    a.heads = (uint32_t)p->heads; a.from_pages = (uint32_t)p->from_pages; a.to_pages = (uint32_t)p->to_pages;
    a.page_size = p->page_size;
    // at most 2^22 work-groups a launch (one pair has fewer): a grid of 2^32 threads is none
    uint32_t most = (1u << 22) / (chunks * (uint32_t)n);
    most = most < 1 ? 1 : most > 65535 ? 65535 : most;
    for (int j0 = 0; j0 < p->pairs; j0 += (int)most) {
      a.src = p->src + j0; a.dst = p->dst + j0; a.lens = p->lens ? p->lens + j0 : nullptr;
      a.pairs = (uint32_t)p->pairs - (uint32_t)j0 < most ? (uint32_t)p->pairs - (uint32_t)j0 : most;
      const dim3 grid(chunks, a.pairs, (unsigned)n);
      if (stream) hipLaunchKernelGGL(copy_pages_kernel<true>, grid, dim3(kThreads), 0, st, a);
      else hipLaunchKernelGGL(copy_pages_kernel<false>, grid, dim3(kThreads), 0, st, a);
      const int rc = launched();
      if (rc) return rc;
    }
  }
  return KVQ_OK;
}

}  // namespace
}  // namespace kvq

extern "C" int kvq_copy_pages(const kvq_copy_pages_params* p, kvq_stream_t stream) {
  return kvq::guarded([&] { return kvq::copy_pages(p, reinterpret_cast<hipStream_t>(stream)); });
}
