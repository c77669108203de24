// paged_attend.cu -- attention of drafted rows over a device-planned paged
// cache (paged.cu): packed row i of request s sees the request's seq_lens[s]
// cached positions and those of the request's new rows that its mask names
// (without masks: rows 0..i, the causal rule of decoder.rs:864).

#include <algorithm>

#include "wattn_common.cuh"
#include "wattn_internal.h"

namespace wattn {

namespace {

struct PagedAttendParams {
  const void *pool;
  int n_pages, n_layers, n_heads, page_rows, layer;
  const int *table;
  int64_t table_stride;
  int max_pages;
  const int *seq_lens, *row_start;
  int n_seqs;
  const int *row_mask;
  int mask_words;
  const void *q;
  void *o;
  int64_t q_rs, o_rs;
  int max_rows;
  float scale_log2;
  int *status;
};

// One warp per (row, head): two dims a lane, an online softmax over the keys
// one at a time.
template <typename T, typename OutT>
__global__ void paged_attend_simple_kernel(const PagedAttendParams p) {
  grid_dep_wait();  // (launched with programmatic serialisation)
  grid_dep_launch();
  const int lane = threadIdx.x & 31;
  const int r = blockIdx.x, head = blockIdx.y * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (head >= p.n_heads || r >= p.row_start[p.n_seqs]) return;
  int lo = 0, hi = p.n_seqs;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (p.row_start[mid] <= r) lo = mid; else hi = mid;
  }
  const int first = p.row_start[lo], n = p.row_start[lo + 1] - first, i = r - first;
  const int len = max(0, p.seq_lens[lo]);
  if (p.seq_lens[lo] < 0) report_error(p.status, WATTN_ERR_RANGE, 4 << 24);
  if (i < 0 || i >= n) return;
  const T *q = reinterpret_cast<const T *>(p.q) + (int64_t)r * p.q_rs + head * 64 + 2 * lane;
  const float q0 = to_f32(q[0]) * p.scale_log2, q1 = to_f32(q[1]) * p.scale_log2;
  const int64_t kv_off = (int64_t)p.n_heads * p.page_rows * 64;
  float m = -INFINITY, l = 0.f, o0 = 0.f, o1 = 0.f;
  int64_t end = (int64_t)len + n;
  if (end > (int64_t)p.max_pages * p.page_rows) {
    report_error(p.status, WATTN_ERR_RANGE, 4 << 24);
    end = (int64_t)p.max_pages * p.page_rows;
  }
  for (int64_t at = 0; at < end; ++at) {
    if (at >= len) {
      const int j = (int)(at - len);
      if (p.row_mask == nullptr) {
        if (j > i) break;
      } else if (j >= p.mask_words * 32 ||
                 !(p.row_mask[(int64_t)r * p.mask_words + (j >> 5)] >> (j & 31) & 1)) {
        continue;
      }
    }
    const int64_t pi = at / p.page_rows;
    const int page = pi < p.max_pages ? p.table[lo * p.table_stride + pi] : -1;
    if (page < 0 || page >= p.n_pages) {
      report_error(p.status, WATTN_ERR_RANGE, 4 << 24);
      continue;
    }
    const T *k = reinterpret_cast<const T *>(p.pool) +
                 ((int64_t)page * p.n_layers + p.layer) * 2 * kv_off +
                 ((int64_t)head * p.page_rows + at % p.page_rows) * 64 + 2 * lane;
    float x = fmaf(q0, to_f32(k[0]), q1 * to_f32(k[1]));
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
    const float mn = fmaxf(m, x);
    const float a = m == -INFINITY ? 0.f : ex2(m - mn);
    const float w = x == -INFINITY ? 0.f : ex2(x - mn);
    m = mn;
    l = fmaf(l, a, w);
    o0 = fmaf(o0, a, w * to_f32(k[kv_off]));
    o1 = fmaf(o1, a, w * to_f32(k[kv_off + 1]));
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  OutT *o = reinterpret_cast<OutT *>(p.o) + (int64_t)r * p.o_rs + head * 64 + 2 * lane;
  o[0] = from_f32<OutT>(o0 * inv);
  o[1] = from_f32<OutT>(o1 * inv);
}

template <typename T, typename OutT>
int launch_simple(const PagedAttendParams &p, cudaStream_t st) {
  launch_pdl(paged_attend_simple_kernel<T, OutT>, dim3(p.max_rows, (p.n_heads + 3) / 4), dim3(128),
             0, st, p);
  return check_launch("paged_attend");
}

}  // namespace
}  // namespace wattn

using namespace wattn;

extern "C" {

size_t wattn_paged_attend_workspace_bytes(int n_seqs, int max_rows, int n_heads) {
  if (n_seqs <= 0 || max_rows <= 0 || n_heads <= 0) return 0;
  return 0;
}

int wattn_paged_attend(const void *pool, int dtype, int n_pages, int n_layers, int n_heads,
                       int page_rows, int layer, const int *block_table, int64_t table_stride,
                       int max_pages, const int *seq_lens, const int *row_start, int n_seqs,
                       const int *row_mask, int mask_words, const void *q, int64_t q_row_stride,
                       void *o, int out_dtype, int64_t o_row_stride, int max_rows, float scale,
                       void *workspace, size_t workspace_bytes, void *stream) {
  clear_error();
  int rc = check_page_pool("paged_attend", pool, dtype, n_pages, n_layers, n_heads, page_rows);
  if (rc != WATTN_OK) return rc;
  if (layer < 0 || layer >= n_layers)
    return set_error(WATTN_ERR_RANGE, "paged_attend: layer %d out of range", layer);
  if (out_dtype != WATTN_F32 && out_dtype != dtype)
    return set_error(WATTN_ERR_INVALID, "paged_attend: out_dtype must be F32 or the pool's type");
  if (n_seqs < 0 || max_rows < 0 || max_pages <= 0 || table_stride < max_pages)
    return set_error(WATTN_ERR_INVALID, "paged_attend: invalid sizes");
  if (row_mask != nullptr && mask_words <= 0)
    return set_error(WATTN_ERR_INVALID, "paged_attend: mask_words must be positive");
  if (!(scale > 0.f) || scale > 3.0e38f)
    return set_error(WATTN_ERR_INVALID, "paged_attend: scale must be finite and positive");
  const int64_t w = (int64_t)n_heads * 64;
  if (q_row_stride < w || o_row_stride < w)
    return set_error(WATTN_ERR_INVALID, "paged_attend: row stride below width");
  if (n_seqs == 0 || max_rows == 0) return WATTN_OK;
  if (!block_table || !seq_lens || !row_start || !q || !o)
    return set_error(WATTN_ERR_INVALID, "paged_attend: NULL argument");
  if (((reinterpret_cast<uintptr_t>(block_table) | reinterpret_cast<uintptr_t>(seq_lens) |
        reinterpret_cast<uintptr_t>(row_start) | reinterpret_cast<uintptr_t>(row_mask)) & 3))
    return set_error(WATTN_ERR_INVALID, "paged_attend: integer arrays must be 4-byte aligned");
  if (((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(o)) & 15) ||
      (q_row_stride * elem_size(dtype)) % 16 || (o_row_stride * elem_size(out_dtype)) % 16)
    return set_error(WATTN_ERR_INVALID, "paged_attend: q and o must be 16-byte aligned with row "
                     "strides that are multiples of 16 bytes");
  (void)workspace;
  (void)workspace_bytes;
  PagedAttendParams p = {pool, n_pages, n_layers, n_heads, page_rows, layer, block_table,
                         table_stride, max_pages, seq_lens, row_start, n_seqs, row_mask,
                         mask_words, q, o, q_row_stride, o_row_stride, max_rows,
                         scale * 1.4426950408889634f, device_status_ptr()};
  if (p.status == nullptr) return WATTN_ERR_CUDA;
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == WATTN_F32) return launch_simple<float, float>(p, st);
  if (dtype == WATTN_F16)
    return out_dtype == WATTN_F32 ? launch_simple<__half, float>(p, st)
                                  : launch_simple<__half, __half>(p, st);
  return out_dtype == WATTN_F32 ? launch_simple<__nv_bfloat16, float>(p, st)
                                : launch_simple<__nv_bfloat16, __nv_bfloat16>(p, st);
}

}  // extern "C"
