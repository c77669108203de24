// paged.cu -- the device-planned paged cache: block tables and slot maps
// from request lengths, row writes through the slot map, and the acceptance
// of a verified draft tree. No counterpart in the reference, whose cache
// state lives on the host (DecoderKvCache, crates/whisper/src/decoder.rs:
// 131-264; kv_cache.cu here); with the state on the device a decode step has
// no host work of its own and one captured graph serves every length.
//
// The pool has the layout of kv_cache.cu: [page][layer][K|V][head]
// [page_rows][64]. A slot is page * page_rows + row in page. The attention
// over it is paged_attend.cu's.

#include <algorithm>

#include "wattn_common.cuh"
#include "wattn_internal.h"

namespace wattn {

namespace {

// ---------------------------------------------------------------- plan
struct PlanParams {
  const int *seq_lens, *n_new;
  int n_seqs, page_rows, n_pages;
  int *table;
  int64_t table_stride;
  int max_pages;
  int *n_held, *free_pages, *n_free;
  const int *parents;
  int *row_start, *row_pos, *row_slot, *row_mask;
  int mask_words, max_rows;
  int *status;
};

constexpr int kPlanThreads = 1024;

// What one request asks of the plan: new rows, pages taken and given back.
struct PlanSum {
  long long rows, take, give;
};
WATTN_DEVINL PlanSum operator+(const PlanSum &a, const PlanSum &b) {
  return {a.rows + b.rows, a.take + b.take, a.give + b.give};
}
WATTN_DEVINL PlanSum shfl_up(const PlanSum &x, int d) {
  return {__shfl_up_sync(0xffffffffu, x.rows, d), __shfl_up_sync(0xffffffffu, x.take, d),
          __shfl_up_sync(0xffffffffu, x.give, d)};
}

// Exclusive sums over the CTA's threads; `total` gets the sum of all.
WATTN_DEVINL PlanSum block_scan(PlanSum x, PlanSum *warp_sums, PlanSum &total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  PlanSum inc = x;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const PlanSum y = shfl_up(inc, d);
    if (lane >= d) inc = inc + y;
  }
  __syncthreads();  // the previous use of warp_sums is over
  if (lane == 31) warp_sums[warp] = inc;
  __syncthreads();
  if (warp == 0) {
    PlanSum w = warp_sums[lane];
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const PlanSum y = shfl_up(w, d);
      if (lane >= d) w = w + y;
    }
    warp_sums[lane] = w;
  }
  __syncthreads();
  total = warp_sums[kPlanThreads / 32 - 1];
  const PlanSum before = warp > 0 ? warp_sums[warp - 1] : PlanSum{0, 0, 0};
  return {inc.rows - x.rows + before.rows, inc.take - x.take + before.take,
          inc.give - x.give + before.give};
}

struct PlanSeq {
  int len, fresh, held;
  long long need;
};
WATTN_DEVINL PlanSeq plan_seq(const PlanParams &p, int s) {
  PlanSeq q = {0, 0, 0, 0};
  if (s < p.n_seqs) {
    q.len = p.seq_lens[s];
    q.fresh = p.n_new[s];
    q.held = p.n_held[s];
    q.need = ((long long)q.len + q.fresh + p.page_rows - 1) / p.page_rows;
  }
  return q;
}
WATTN_DEVINL PlanSum plan_sum(const PlanSeq &q) {
  return {q.fresh, max(0ll, q.need - q.held), max(0ll, q.held - q.need)};
}

// Lengths to row starts and pages, by one CTA. First the whole request is
// checked, so that a refused one changes nothing; then pages are given back
// to the stack, then taken from it. The g-th page given back (in the order
// of requests and of pages) lands where the g-th page taken comes from, so a
// plan that undoes another leaves the stack as it was.
__global__ void __launch_bounds__(kPlanThreads) plan_tables_kernel(const PlanParams p) {
  grid_dep_wait();  // (launched with programmatic serialisation)
  grid_dep_launch();
  __shared__ PlanSum warp_sums[32];
  __shared__ int s_bad;
  const int tid = threadIdx.x;
  if (tid == 0) s_bad = 0;
  __syncthreads();
  PlanSum total = {0, 0, 0};
  int bad = 0;  // bit 0: invalid, bit 1: out of range
  for (int s0 = 0; s0 < p.n_seqs; s0 += kPlanThreads) {
    const PlanSeq q = plan_seq(p, s0 + tid);
    if (q.len < 0 || q.fresh < 0 || q.held < 0 || q.held > p.max_pages) bad |= 1;
    if (q.need > p.max_pages || (p.row_mask != nullptr && q.fresh > p.mask_words * 32)) bad |= 2;
    PlanSum chunk;
    block_scan(plan_sum(q), warp_sums, chunk);
    total = total + chunk;
  }
  if (bad) atomicOr(&s_bad, bad);
  __syncthreads();
  const int n_free = *p.n_free;
  int status = WATTN_OK;
  if ((s_bad & 1) || n_free < 0 || n_free + total.give > p.n_pages) status = WATTN_ERR_INVALID;
  else if ((s_bad & 2) || total.rows > p.max_rows) status = WATTN_ERR_RANGE;
  else if (total.take > n_free + total.give) status = WATTN_ERR_NOMEM;
  if (status != WATTN_OK) {
    for (int s = tid; s <= p.n_seqs; s += kPlanThreads) p.row_start[s] = 0;
    if (tid == 0) *p.status = status;
    return;
  }
  const int top = n_free + (int)total.give;
  PlanSum base = {0, 0, 0}, chunk;
  for (int s0 = 0; s0 < p.n_seqs; s0 += kPlanThreads) {
    const int s = s0 + tid;
    const PlanSeq q = plan_seq(p, s);
    const PlanSum at = base + block_scan(plan_sum(q), warp_sums, chunk);
    base = base + chunk;
    if (s < p.n_seqs) {
      p.row_start[s] = (int)at.rows;
      int *row = p.table + s * p.table_stride;
      for (int i = (int)q.need; i < q.held; ++i) {
        p.free_pages[top - 1 - ((int)at.give + i - (int)q.need)] = row[i];
        row[i] = -1;
      }
    }
  }
  __syncthreads();  // the stack holds what was given back
  base = {0, 0, 0};
  for (int s0 = 0; s0 < p.n_seqs; s0 += kPlanThreads) {
    const int s = s0 + tid;
    const PlanSeq q = plan_seq(p, s);
    const PlanSum at = base + block_scan(plan_sum(q), warp_sums, chunk);
    base = base + chunk;
    if (s < p.n_seqs) {
      int *row = p.table + s * p.table_stride;
      for (int i = q.held; i < (int)q.need; ++i)
        row[i] = p.free_pages[top - 1 - ((int)at.take + i - q.held)];
      if (q.held != (int)q.need) p.n_held[s] = (int)q.need;
    }
  }
  if (tid == 0) {
    p.row_start[p.n_seqs] = (int)total.rows;
    *p.n_free = top - (int)total.take;
    *p.status = WATTN_OK;
  }
}

// The request that packed row r belongs to (row_start ascending, r below
// its last entry).
WATTN_DEVINL int seq_of_row(const int *row_start, int n_seqs, int r) {
  int lo = 0, hi = n_seqs;  // row_start[lo] <= r < row_start[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (row_start[mid] <= r) lo = mid; else hi = mid;
  }
  return lo;
}

// Position, slot and tree mask of each packed row; -1 (mask 0) behind the
// last one. A tree row's ancestors are found by walking its parents up; a
// row whose way up leaves [-1, child) is dead and gets position -1 and an
// empty mask.
__global__ void plan_rows_kernel(const PlanParams p) {
  grid_dep_wait();  // (launched with programmatic serialisation)
  grid_dep_launch();
  const int r = blockIdx.x * blockDim.x + threadIdx.x;
  if (r >= p.max_rows) return;
  int pos = -1, slot = -1;
  if (r < p.row_start[p.n_seqs]) {
    const int s = seq_of_row(p.row_start, p.n_seqs, r);
    const int first = p.row_start[s], t = r - first, at = p.seq_lens[s] + t;
    pos = at;
    if (p.parents != nullptr) {
      int depth = 0, j = t;
      for (;;) {
        const int up = p.parents[first + j];
        if (up == -1) break;
        if (up < -1 || up >= j) { depth = -1; break; }
        j = up;
        ++depth;
      }
      pos = depth < 0 ? -1 : p.seq_lens[s] + depth;
      for (int w = 0; w < p.mask_words; ++w) {
        uint32_t bits = 0;
        for (int i = t; depth >= 0 && i >= 0; i = p.parents[first + i])
          if ((i >> 5) == w) bits |= 1u << (i & 31);
        p.row_mask[(int64_t)r * p.mask_words + w] = (int)bits;
      }
    }
    const int page = p.table[s * p.table_stride + at / p.page_rows];
    if (page >= 0 && page < p.n_pages) slot = page * p.page_rows + at % p.page_rows;
  } else if (p.row_mask != nullptr) {
    for (int w = 0; w < p.mask_words; ++w) p.row_mask[(int64_t)r * p.mask_words + w] = 0;
  }
  p.row_pos[r] = pos;
  p.row_slot[r] = slot;
}

// ---------------------------------------------------------------- write
struct WriteParams {
  const int *row_slot;
  int n_slots, n_layers, n_heads, page_rows, layer;
  int64_t row_stride;
};

template <typename SrcT, typename DstT>
__global__ void paged_write_kernel(const SrcT *k_rows, const SrcT *v_rows, DstT *pool,
                                   const WriteParams p) {
  grid_dep_wait();  // (launched with programmatic serialisation)
  grid_dep_launch();
  const int r = blockIdx.x;
  const int slot = p.row_slot[r];
  if (slot < 0 || slot >= p.n_slots) return;
  const int page = slot / p.page_rows, row = slot % p.page_rows;
  const int64_t kv_off = (int64_t)p.n_heads * p.page_rows * 64;
  DstT *base = pool + ((int64_t)page * p.n_layers + p.layer) * 2 * kv_off + (int64_t)row * 64;
  for (int i = threadIdx.x; i < p.n_heads * 64; i += blockDim.x) {
    const int64_t dst = (int64_t)(i >> 6) * p.page_rows * 64 + (i & 63);
    base[dst] = from_f32<DstT>(to_f32(k_rows[(int64_t)r * p.row_stride + i]));
    base[kv_off + dst] = from_f32<DstT>(to_f32(v_rows[(int64_t)r * p.row_stride + i]));
  }
}

template <typename SrcT>
int launch_write_src(int dst_dt, const void *k, const void *v, void *pool, int n_rows,
                     const WriteParams &p, cudaStream_t st) {
  const SrcT *ks = (const SrcT *)k, *vs = (const SrcT *)v;
  if (dst_dt == WATTN_F32)
    launch_pdl(paged_write_kernel<SrcT, float>, dim3(n_rows), dim3(256), 0, st, ks, vs,
               (float *)pool, p);
  else if (dst_dt == WATTN_F16)
    launch_pdl(paged_write_kernel<SrcT, __half>, dim3(n_rows), dim3(256), 0, st, ks, vs,
               (__half *)pool, p);
  else
    launch_pdl(paged_write_kernel<SrcT, __nv_bfloat16>, dim3(n_rows), dim3(256), 0, st, ks, vs,
               (__nv_bfloat16 *)pool, p);
  return check_launch("paged_write");
}

// ---------------------------------------------------------------- accept
struct AcceptParams {
  const int *row_start;
  int n_seqs, max_rows;
  const int *parents, *row_slot, *tokens, *picked;
  int *seq_lens, *n_accepted, *path, *next_token;
  uint8_t *pool;
  int n_slots, page_rows, n_heads, n_layers;
  int row_bytes;  // 64 elements
};

// Rows of request s, within the row buffers whatever row_start holds.
WATTN_DEVINL int2 rows_of(const int *row_start, int s, int max_rows) {
  const int a = min(max(row_start[s], 0), max_rows);
  const int b = min(max(row_start[s + 1], a), max_rows);
  return make_int2(a, b - a);
}

// One warp per request walks from the root to the lowest child whose token
// is the one picked at its parent, until there is none.
__global__ void accept_walk_kernel(const AcceptParams p) {
  grid_dep_wait();  // (launched with programmatic serialisation)
  grid_dep_launch();
  const int lane = threadIdx.x & 31;
  const int warps = gridDim.x * (blockDim.x >> 5);
  const int warp = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  for (int s = warp; s < p.n_seqs; s += warps) {
    const int2 rw = rows_of(p.row_start, s, p.max_rows);
    const int a = rw.x, n = rw.y;
    int len = 0, cur = -1;
    if (n > 0 && (p.parents == nullptr || p.parents[a] == -1)) {
      cur = 0;
      if (lane == 0) p.path[a] = 0;
      len = 1;
      for (int c0 = 1; c0 < n;) {
        const int want = p.picked[a + cur];
        int found = -1;
        for (; c0 < n; c0 += 32) {
          const int c = c0 + lane;
          const bool hit = c < n && p.tokens[a + c] == want &&
                           (p.parents == nullptr ? c - 1 : p.parents[a + c]) == cur;
          const unsigned m = __ballot_sync(0xffffffffu, hit);
          if (m) {
            found = c0 + __ffs(m) - 1;
            break;
          }
        }
        if (found < 0) break;
        cur = found;
        if (lane == 0) p.path[a + len] = cur;
        ++len;
        c0 = found + 1;
      }
    }
    for (int j = len + lane; j < n; j += 32) p.path[a + j] = -1;
    if (lane == 0) {
      p.n_accepted[s] = len;
      p.next_token[s] = cur >= 0 ? p.picked[a + cur] : -1;
      p.seq_lens[s] += len;
    }
  }
  const int last = rows_of(p.row_start, p.n_seqs - 1, p.max_rows).x +
                   rows_of(p.row_start, p.n_seqs - 1, p.max_rows).y;
  for (int r = last + warp * 32 + lane; r < p.max_rows; r += warps * 32) p.path[r] = -1;
}

// Moves the accepted rows together, (request, layer) per CTA: each thread
// owns 16 bytes of a K or V head row and takes the path's rows in order.
// Path rows ascend and row j of the path lands at or before its own place,
// so no move overwrites a row that a later one reads.
__global__ void accept_move_kernel(const AcceptParams p) {
  grid_dep_wait();  // (launched with programmatic serialisation)
  grid_dep_launch();
  const int s = blockIdx.x, layer = blockIdx.y;
  const int a = rows_of(p.row_start, s, p.max_rows).x;
  const int n = p.n_accepted[s];
  const int chunks = p.row_bytes / 16, per_kv = p.n_heads * chunks;
  const int64_t page_bytes = (int64_t)p.n_layers * 2 * p.n_heads * p.page_rows * p.row_bytes;
  for (int i = threadIdx.x; i < 2 * per_kv; i += blockDim.x) {
    const int head = i / chunks % p.n_heads, kv = i / per_kv, c = i % chunks;
    uint8_t *base = p.pool + (((int64_t)layer * 2 + kv) * p.n_heads + head) * p.page_rows * p.row_bytes + c * 16;
    for (int j = 1; j < n; ++j) {
      const int from = p.path[a + j];
      if (from == j) continue;
      const int src = p.row_slot[a + from], dst = p.row_slot[a + j];
      if (src < 0 || src >= p.n_slots || dst < 0 || dst >= p.n_slots) continue;
      *reinterpret_cast<uint4 *>(base + dst / p.page_rows * page_bytes +
                                 (int64_t)(dst % p.page_rows) * p.row_bytes) =
          *reinterpret_cast<const uint4 *>(base + src / p.page_rows * page_bytes +
                                           (int64_t)(src % p.page_rows) * p.row_bytes);
    }
  }
}

bool int_aligned(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 3) == 0; }

}  // namespace

int check_page_pool(const char *what, const void *pool, int dtype, int n_pages, int n_layers,
                    int n_heads, int page_rows) {
  if (!valid_dtype(dtype)) return set_error(WATTN_ERR_INVALID, "%s: bad dtype %d", what, dtype);
  if (n_pages <= 0 || n_layers <= 0 || n_heads <= 0 || n_heads > 65535)
    return set_error(WATTN_ERR_INVALID, "%s: invalid pool sizes", what);
  if (page_rows <= 0 || page_rows % kPageRowsUnit != 0)
    return set_error(WATTN_ERR_INVALID, "%s: page_rows %d must be a positive multiple of %d", what,
                     page_rows, kPageRowsUnit);
  // (each factor is below 2^31; the products are taken one at a time)
  const int64_t lim = INT64_C(1) << 31;
  int64_t rows = (int64_t)n_pages * n_layers;
  if (rows < lim) rows *= 2 * n_heads;
  if (rows < lim) rows *= page_rows;
  if (rows >= lim) return set_error(WATTN_ERR_UNSUPPORTED, "%s: pool of 2^31 head rows or more", what);
  if (pool == nullptr || (reinterpret_cast<uintptr_t>(pool) & 15))
    return set_error(WATTN_ERR_INVALID, "%s: the pool must be a 16-byte aligned device pointer", what);
  return WATTN_OK;
}

}  // namespace wattn

using namespace wattn;

extern "C" {

int wattn_paged_plan(const int *seq_lens, const int *n_new, int n_seqs, int page_rows, int n_pages,
                     int *block_table, int64_t table_stride, int max_pages, int *n_held,
                     int *free_pages, int *n_free, const int *parents, int *row_start,
                     int *row_pos, int *row_slot, int *row_mask, int mask_words, int max_rows,
                     int *status, void *stream) {
  clear_error();
  if (n_seqs < 0 || max_rows < 0 || n_pages <= 0 || max_pages <= 0 || page_rows <= 0)
    return set_error(WATTN_ERR_INVALID, "paged_plan: invalid sizes");
  if ((int64_t)n_pages * page_rows >= (INT64_C(1) << 31))
    return set_error(WATTN_ERR_UNSUPPORTED, "paged_plan: pool of 2^31 slots or more");
  if (table_stride < max_pages)
    return set_error(WATTN_ERR_INVALID, "paged_plan: table_stride %lld < max_pages %d",
                     (long long)table_stride, max_pages);
  if ((parents == nullptr) != (row_mask == nullptr))
    return set_error(WATTN_ERR_INVALID, "paged_plan: parents and row_mask come together");
  if (row_mask != nullptr && mask_words <= 0)
    return set_error(WATTN_ERR_INVALID, "paged_plan: mask_words must be positive");
  if (!n_free || !free_pages || !row_start || !status ||
      (n_seqs > 0 && (!seq_lens || !n_new || !block_table || !n_held)) ||
      (max_rows > 0 && (!row_pos || !row_slot)))
    return set_error(WATTN_ERR_INVALID, "paged_plan: NULL argument");
  for (const void *p : {(const void *)seq_lens, (const void *)n_new, (const void *)block_table,
                        (const void *)n_held, (const void *)free_pages, (const void *)n_free,
                        (const void *)parents, (const void *)row_start, (const void *)row_pos,
                        (const void *)row_slot, (const void *)row_mask, (const void *)status})
    if (!int_aligned(p)) return set_error(WATTN_ERR_INVALID, "paged_plan: arrays must be 4-byte aligned");
  const PlanParams p = {seq_lens, n_new,   n_seqs,    page_rows, n_pages,  block_table, table_stride,
                        max_pages, n_held, free_pages, n_free,   parents,  row_start,   row_pos,
                        row_slot, row_mask, mask_words, max_rows, status};
  cudaStream_t st = (cudaStream_t)stream;
  launch_pdl(plan_tables_kernel, dim3(1), dim3(kPlanThreads), 0, st, p);
  int rc = check_launch("paged_plan");
  if (rc != WATTN_OK || max_rows == 0) return rc;
  launch_pdl(plan_rows_kernel, dim3((max_rows + 255) / 256), dim3(256), 0, st, p);
  return check_launch("paged_plan (rows)");
}

int wattn_paged_write(void *pool, int dtype, int n_pages, int n_layers, int n_heads, int page_rows,
                      int layer, const int *row_slot, int n_rows, const void *k_rows,
                      const void *v_rows, int src_dtype, int64_t row_stride, void *stream) {
  clear_error();
  int rc = check_page_pool("paged_write", pool, dtype, n_pages, n_layers, n_heads, page_rows);
  if (rc != WATTN_OK) return rc;
  if (layer < 0 || layer >= n_layers)
    return set_error(WATTN_ERR_RANGE, "paged_write: layer %d out of range", layer);
  if (!valid_dtype(src_dtype)) return set_error(WATTN_ERR_INVALID, "paged_write: bad dtype");
  if (n_rows < 0) return set_error(WATTN_ERR_INVALID, "paged_write: negative n_rows");
  if (row_stride < (int64_t)n_heads * 64)
    return set_error(WATTN_ERR_INVALID, "paged_write: row_stride %lld < width", (long long)row_stride);
  if (n_rows == 0) return WATTN_OK;
  if (!row_slot || !k_rows || !v_rows) return set_error(WATTN_ERR_INVALID, "paged_write: NULL argument");
  if (!int_aligned(row_slot) || !elem_aligned(k_rows, src_dtype) || !elem_aligned(v_rows, src_dtype))
    return set_error(WATTN_ERR_INVALID, "paged_write: arrays must be aligned to their element size");
  const WriteParams p = {row_slot, n_pages * page_rows, n_layers, n_heads, page_rows, layer, row_stride};
  cudaStream_t st = (cudaStream_t)stream;
  if (src_dtype == WATTN_F32) return launch_write_src<float>(dtype, k_rows, v_rows, pool, n_rows, p, st);
  if (src_dtype == WATTN_F16) return launch_write_src<__half>(dtype, k_rows, v_rows, pool, n_rows, p, st);
  return launch_write_src<__nv_bfloat16>(dtype, k_rows, v_rows, pool, n_rows, p, st);
}

int wattn_paged_accept(void *pool, int dtype, int n_pages, int n_layers, int n_heads, int page_rows,
                       const int *row_start, int n_seqs, int max_rows, const int *parents,
                       const int *row_slot, const int *tokens, const int *picked, int *seq_lens,
                       int *n_accepted, int *path, int *next_token, void *stream) {
  clear_error();
  int rc = check_page_pool("paged_accept", pool, dtype, n_pages, n_layers, n_heads, page_rows);
  if (rc != WATTN_OK) return rc;
  if (n_seqs < 0 || max_rows < 0 || n_layers > 65535)
    return set_error(WATTN_ERR_INVALID, "paged_accept: invalid sizes");
  if (n_seqs == 0) return WATTN_OK;
  if (!row_start || !seq_lens || !n_accepted || !next_token ||
      (max_rows > 0 && (!row_slot || !tokens || !picked || !path)))
    return set_error(WATTN_ERR_INVALID, "paged_accept: NULL argument");
  for (const void *q : {(const void *)row_start, (const void *)parents, (const void *)row_slot,
                        (const void *)tokens, (const void *)picked, (const void *)seq_lens,
                        (const void *)n_accepted, (const void *)path, (const void *)next_token})
    if (!int_aligned(q)) return set_error(WATTN_ERR_INVALID, "paged_accept: arrays must be 4-byte aligned");
  const AcceptParams p = {row_start, n_seqs,     max_rows, parents,    row_slot,
                          tokens,    picked,     seq_lens, n_accepted, path,
                          next_token, (uint8_t *)pool, n_pages * page_rows, page_rows, n_heads,
                          n_layers,  64 * elem_size(dtype)};
  cudaStream_t st = (cudaStream_t)stream;
  launch_pdl(accept_walk_kernel, dim3((n_seqs + 3) / 4), dim3(128), 0, st, p);
  if ((rc = check_launch("paged_accept")) != WATTN_OK) return rc;
  launch_pdl(accept_move_kernel, dim3(n_seqs, n_layers), dim3(256), 0, st, p);
  return check_launch("paged_accept (move)");
}

}  // extern "C"
