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
  bool rows_apart;
};

constexpr int kPlanThreads = 1024;
constexpr int kPlanCtas = 8;            // the portable cluster size
constexpr int kPlanSeqs = 2048;         // requests whose first rows and lengths a CTA keeps at hand
constexpr int kPlanParents = 16384;     // parents that a CTA keeps at hand
constexpr int kPlanRowsPerCta = 1024;   // rows (a request counts as 4) below which another CTA does not pay
constexpr int kPlanRowsApart = 16384;   // rows beyond which a launch of their own pays

// What one request asks of the plan: new rows, pages taken and given back.
struct PlanSum {
  long long rows, take, give;
};
WATTN_DEVINL PlanSum operator+(const PlanSum &a, const PlanSum &b) {
  return {a.rows + b.rows, a.take + b.take, a.give + b.give};
}
WATTN_DEVINL PlanSum operator-(const PlanSum &a, const PlanSum &b) {
  return {a.rows - b.rows, a.take - b.take, a.give - b.give};
}
WATTN_DEVINL PlanSum warp_scan(PlanSum x, int lane) {
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const PlanSum y = {__shfl_up_sync(0xffffffffu, x.rows, d), __shfl_up_sync(0xffffffffu, x.take, d),
                       __shfl_up_sync(0xffffffffu, x.give, d)};
    if (lane >= d) x = x + y;
  }
  return x;
}

// The last of n ascending numbers that is at most x (at[0] <= x): of a row,
// the request that it belongs to, given the requests' first rows.
WATTN_DEVINL int last_not_above(const int *at, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (at[mid] <= x) lo = mid; else hi = mid;
  }
  return lo;
}

struct PlanSmem {
  PlanSum warp_sums[32];
  PlanSum total;          // of this CTA's requests
  int bad;                // 1: invalid, 2: out of range
  int first[kPlanSeqs + 1], len[kPlanSeqs];
  int page_from[kPlanThreads], page_at[kPlanThreads];
  int parents[kPlanParents];
};

// Exclusive sums over the CTA's threads; `total` gets the sum of all.
WATTN_DEVINL PlanSum block_scan(PlanSum x, PlanSum *warp_sums, PlanSum &total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const PlanSum inc = warp_scan(x, lane);
  __syncthreads();  // the previous use of warp_sums is over
  if (lane == 31) warp_sums[warp] = inc;
  __syncthreads();
  if (warp == 0) warp_sums[lane] = warp_scan(warp_sums[lane], lane);
  __syncthreads();
  total = warp_sums[kPlanThreads / 32 - 1];
  return warp > 0 ? inc - x + warp_sums[warp - 1] : inc - x;
}

struct PlanSeq {
  int len, fresh, held;
  long long need;
};
WATTN_DEVINL PlanSeq plan_seq(const PlanParams &p, int s, int end) {
  PlanSeq q = {0, 0, 0, 0};
  if (s < end) {
    q.len = p.seq_lens[s];
    q.fresh = p.n_new[s];
    q.held = p.n_held[s];
    q.need = (long long)((uint32_t)q.len + (uint32_t)q.fresh + (long long)p.page_rows - 1) / p.page_rows;
  }
  return q;
}
WATTN_DEVINL PlanSum plan_sum(const PlanSeq &q) {
  return {q.fresh, max(0ll, q.need - q.held), max(0ll, q.held - q.need)};
}

WATTN_DEVINL void cluster_sync() {
  asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}
// A 4-byte word of another CTA's shared memory, at the place that `p` has in
// this one's.
WATTN_DEVINL uint32_t cluster_word(const void *p, int rank) {
  uint32_t at, v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
  return v;
}
WATTN_DEVINL long long cluster_word64(const long long *p, int rank) {
  const int *w = reinterpret_cast<const int *>(p);
  return (long long)cluster_word(w, rank) | (long long)cluster_word(w + 1, rank) << 32;
}

// Hands the pages [from, from + count) of each thread's request, all of the
// CTA's `total`, to its threads: f(i, t, rank) for page i of thread t's
// request, the rank-th in the order of threads and of pages (at: this
// thread's first rank).
template <typename F>
WATTN_DEVINL void each_page(PlanSmem &s, int from, int at, int total, F f) {
  if (total == 0) return;  // (the same for all threads)
  __syncthreads();
  s.page_from[threadIdx.x] = from;
  s.page_at[threadIdx.x] = at;
  __syncthreads();
  for (int g = threadIdx.x; g < total; g += kPlanThreads) {
    const int t = last_not_above(s.page_at, kPlanThreads, g);
    f(s.page_from[t] + g - s.page_at[t], t, g);
  }
}

// Position, slot and tree mask of packed row r, of request q whose rows
// begin at `first` and whose parents are at `up`.
WATTN_DEVINL void plan_row(const PlanParams &p, int r, int q, int first, int len, const int *up) {
  const int t = r - first, at = len + t;
  const int page = p.table[q * p.table_stride + at / p.page_rows];
  int pos = at;
  if (p.parents != nullptr) {
    // The ancestors, by walking up; a row whose way up leaves [-1, child)
    // is dead: position -1, empty mask.
    int depth = 0, j = t;
    for (;;) {
      const int u = up[j];
      if (u == -1) break;
      if (u < -1 || u >= j) { depth = -1; break; }
      j = u;
      ++depth;
    }
    pos = depth < 0 ? -1 : len + depth;
    // (parents descend: the words fill from the last to the first)
    int *mask = p.row_mask + (int64_t)r * p.mask_words;
    j = depth < 0 ? -1 : t;
    for (int w = p.mask_words - 1; w >= 0; --w) {
      uint32_t bits = 0;
      while (j >= 32 * w && j >= 0) {
        bits |= 1u << (j & 31);
        j = up[j];
      }
      mask[w] = (int)bits;
    }
  }
  p.row_pos[r] = pos;
  p.row_slot[r] = (unsigned)page < (unsigned)p.n_pages ? page * p.page_rows + at % p.page_rows : -1;
}
WATTN_DEVINL void plan_padding(const PlanParams &p, long long r) {
  p.row_pos[r] = p.row_slot[r] = -1;
  if (p.parents != nullptr)
    for (int w = 0; w < p.mask_words; ++w) p.row_mask[r * p.mask_words + w] = 0;
}

// The plan, by one cluster of up to eight CTAs (bound by latency: three
// dependent passes over the requests; 5.4 us for 320 requests of one row, 13 us
// for 2048 requests with 16,000 pages, of which 229,000 rows take 7 more in a
// launch of their own). Each CTA has a run of the requests.
// First all are checked, so that a refused plan changes nothing; then pages
// are given back to the stack, then taken from it, then the rows are filled
// in. The g-th page given back (in the order of requests and of pages) lands
// where the g-th page taken comes from, so a plan that undoes another leaves
// the stack as it was.
__global__ void __launch_bounds__(kPlanThreads) paged_plan_kernel(const PlanParams p) {
  extern __shared__ uint8_t plan_smem_raw[];
  PlanSmem &s = *reinterpret_cast<PlanSmem *>(plan_smem_raw);
  grid_dep_wait();  // (launched with programmatic serialisation)
  grid_dep_launch();
  const int tid = threadIdx.x, rank = blockIdx.x, ctas = gridDim.x;
  const int s0 = (int)((long long)p.n_seqs * rank / ctas);
  const int s1 = (int)((long long)p.n_seqs * (rank + 1) / ctas);
  if (tid == 0) s.bad = 0;
  const int n_free = *p.n_free;
  __syncthreads();
  // ---- sums and checks
  // (a CTA with no more requests than threads reads and adds them up once)
  const bool once = s1 - s0 <= kPlanThreads;
  PlanSum mine = {0, 0, 0};
  PlanSeq q = {0, 0, 0, 0};
  int bad = n_free < 0 ? 1 : 0;
  for (int b = s0; b < s1; b += kPlanThreads) {
    q = plan_seq(p, b + tid, s1);
    if ((q.len | q.fresh | q.held) < 0 || q.held > p.max_pages) bad |= 1;
    else if (q.need > p.max_pages || (p.row_mask != nullptr && q.fresh > (long long)p.mask_words * 32)) bad |= 2;
    mine = mine + plan_sum(q);
  }
  if (bad) atomicOr(&s.bad, bad);
  PlanSum sum;
  const PlanSum only = block_scan(mine, s.warp_sums, sum);
  if (tid == 0) s.total = sum;
  PlanSum before = {0, 0, 0}, total = sum;
  if (ctas > 1) {
    cluster_sync();
    total = {0, 0, 0};
    bad = 0;
    for (int r = 0; r < ctas; ++r) {
      const PlanSum t = {cluster_word64(&s.total.rows, r), cluster_word64(&s.total.take, r),
                         cluster_word64(&s.total.give, r)};
      if (r < rank) before = before + t;
      total = total + t;
      bad |= (int)cluster_word(&s.bad, r);
    }
    cluster_sync();  // all have read (also the stack's height)
  } else {
    __syncthreads();
    bad = s.bad;
  }
  int status = WATTN_OK;
  if ((bad & 1) || n_free + total.give > p.n_pages) status = WATTN_ERR_INVALID;
  else if ((bad & 2) || total.rows > p.max_rows) status = WATTN_ERR_RANGE;
  else if (total.take > n_free + total.give) status = WATTN_ERR_NOMEM;
  const bool ok = status == WATTN_OK;
  const int top = n_free + (int)total.give;
  const int row0 = ok ? (int)before.rows : 0;
  if (rank == ctas - 1 && tid == 0) {
    *p.status = status;
    p.row_start[p.n_seqs] = ok ? (int)total.rows : 0;
    if (ok) *p.n_free = top - (int)total.take;
  }
  // ---- pages given back
  PlanSum base = before, chunk = sum;
  for (int b = s0; b < s1; b += kPlanThreads) {
    const int i = b + tid;
    PlanSum in = only;  // sums before this thread's request, within the chunk
    if (!once) {
      q = plan_seq(p, i, s1);
      in = block_scan(plan_sum(q), s.warp_sums, chunk);
    }
    const int first = (int)(base.rows + in.rows);
    if (i < s1) p.row_start[i] = ok ? first : 0;
    if (i < s1 && i - s0 < kPlanSeqs) {
      s.first[i - s0] = first;
      s.len[i - s0] = q.len;
    }
    if (ok)
      each_page(s, (int)q.need, (int)in.give, (int)chunk.give, [&](int pi, int t, int g) {
        int *e = p.table + (b + t) * p.table_stride + pi;
        p.free_pages[top - 1 - ((int)base.give + g)] = *e;
        *e = -1;
      });
    base = base + chunk;
  }
  if (tid == 0 && s1 - s0 <= kPlanSeqs) s.first[s1 - s0] = (int)base.rows;
  if (ctas > 1) cluster_sync(); else __syncthreads();  // the stack holds what was given back
  // ---- pages taken
  if (ok) {
    base = before;
    for (int b = s0; b < s1; b += kPlanThreads) {
      const int i = b + tid;
      PlanSum in = only;
      if (!once) {
        q = plan_seq(p, i, s1);
        in = block_scan(plan_sum(q), s.warp_sums, chunk);
      }
      each_page(s, q.held, (int)in.take, (int)chunk.take, [&](int pi, int t, int g) {
        p.table[(b + t) * p.table_stride + pi] = p.free_pages[top - 1 - ((int)base.take + g)];
      });
      if (i < s1 && q.held != (int)q.need) p.n_held[i] = (int)q.need;
      base = base + chunk;
    }
  }
  // ---- rows: here, or (p.rows_apart) by a kernel of the whole GPU
  if (p.rows_apart) return;
  const int n_rows = ok ? (int)sum.rows : 0;
  const bool near = s1 - s0 <= kPlanSeqs;
  const bool near_parents = p.parents != nullptr && n_rows <= kPlanParents;
  if (near_parents)
    for (int i = tid; i < n_rows; i += kPlanThreads) s.parents[i] = p.parents[row0 + i];
  __syncthreads();  // the table has its new pages
  for (int i = tid; i < n_rows; i += kPlanThreads) {
    const int r = row0 + i;
    const int k = near ? last_not_above(s.first, s1 - s0, r) : last_not_above(p.row_start + s0, s1 - s0, r);
    const int first = near ? s.first[k] : p.row_start[s0 + k];
    plan_row(p, r, s0 + k, first, near ? s.len[k] : p.seq_lens[s0 + k],
             near_parents ? s.parents + (first - row0) : p.parents + first);
  }
  for (long long r = (ok ? total.rows : 0) + (long long)rank * kPlanThreads + tid; r < p.max_rows;
       r += (long long)ctas * kPlanThreads)
    plan_padding(p, r);
}

__global__ void __launch_bounds__(256) paged_plan_rows_kernel(const PlanParams p) {
  grid_dep_wait();  // (launched with programmatic serialisation)
  grid_dep_launch();
  const long long r = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  if (r >= p.max_rows) return;
  if (r >= p.row_start[p.n_seqs]) {
    plan_padding(p, r);
    return;
  }
  const int q = last_not_above(p.row_start, p.n_seqs, (int)r);
  const int first = p.row_start[q];
  plan_row(p, (int)r, q, first, p.seq_lens[q], p.parents + first);
}

// ---------------------------------------------------------------- write
struct WriteParams {
  const int *row_slot;
  int n_rows, n_slots, n_layers, n_heads, page_rows, layer;
  int64_t row_stride;
};

// One thread per 8 elements of a row's keys and of its values: 16 bytes of a
// 16-bit pool. VEC: the source rows are 16-byte aligned. Bound: HBM (64
// prompts of up to 224 rows x 1280, f32 into bf16, 121 MB: 20.3 us, 6.0 TB/s).
template <typename T> WATTN_DEVINL void load8(const T *src, float (&f)[8]) {
  if constexpr (sizeof(T) == 4) {
    const float4 a = reinterpret_cast<const float4 *>(src)[0];
    const float4 b = reinterpret_cast<const float4 *>(src)[1];
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
    f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
  } else {
    const uint4 w = *reinterpret_cast<const uint4 *>(src);
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 x = unpack2<T>(u[i]);
      f[2 * i] = x.x;
      f[2 * i + 1] = x.y;
    }
  }
}
template <typename T> WATTN_DEVINL void store8(T *dst, const float (&f)[8]) {
  if constexpr (sizeof(T) == 4) {
    reinterpret_cast<float4 *>(dst)[0] = make_float4(f[0], f[1], f[2], f[3]);
    reinterpret_cast<float4 *>(dst)[1] = make_float4(f[4], f[5], f[6], f[7]);
  } else {
    *reinterpret_cast<uint4 *>(dst) = make_uint4(pack2<T>(f[0], f[1]), pack2<T>(f[2], f[3]),
                                                 pack2<T>(f[4], f[5]), pack2<T>(f[6], f[7]));
  }
}

template <typename SrcT, typename DstT, bool VEC>
__global__ void __launch_bounds__(256)
    paged_write_kernel(const SrcT *k_rows, const SrcT *v_rows, DstT *pool, const WriteParams p) {
  grid_dep_wait();  // (launched with programmatic serialisation)
  grid_dep_launch();
  const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  const int chunks = p.n_heads * 8;
  const int r = (int)(i / chunks), c = (int)(i - (long long)r * chunks);
  if (r >= p.n_rows) return;
  const int slot = p.row_slot[r];
  const int64_t src = (int64_t)r * p.row_stride + c * 8;
  float k[8], v[8];
  if constexpr (VEC) {
    load8<SrcT>(k_rows + src, k);
    load8<SrcT>(v_rows + src, v);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      k[e] = to_f32(k_rows[src + e]);
      v[e] = to_f32(v_rows[src + e]);
    }
  }
  if ((unsigned)slot >= (unsigned)p.n_slots) return;
  const int page = slot / p.page_rows, row = slot - page * p.page_rows;
  const int64_t kv_off = (int64_t)p.n_heads * p.page_rows * 64;
  DstT *dst = pool + ((int64_t)page * p.n_layers + p.layer) * 2 * kv_off +
              ((int64_t)(c >> 3) * p.page_rows + row) * 64 + (c & 7) * 8;
  store8<DstT>(dst, k);
  store8<DstT>(dst + kv_off, v);
}

template <typename SrcT, typename DstT>
void launch_write(const SrcT *k, const SrcT *v, void *pool, const WriteParams &p, bool vec,
                  cudaStream_t st) {
  const dim3 grid((unsigned)(((long long)p.n_rows * p.n_heads * 8 + 255) / 256));
  if (vec)
    launch_pdl(paged_write_kernel<SrcT, DstT, true>, grid, dim3(256), 0, st, k, v, (DstT *)pool, p);
  else
    launch_pdl(paged_write_kernel<SrcT, DstT, false>, grid, dim3(256), 0, st, k, v, (DstT *)pool, p);
}

template <typename SrcT>
int launch_write_src(int dst_dt, const void *k, const void *v, void *pool, const WriteParams &p,
                     cudaStream_t st) {
  const SrcT *ks = (const SrcT *)k, *vs = (const SrcT *)v;
  const bool vec = ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) == 0 &&
                   (p.row_stride * (int64_t)sizeof(SrcT)) % 16 == 0;
  if (dst_dt == WATTN_F32) launch_write<SrcT, float>(ks, vs, pool, p, vec, st);
  else if (dst_dt == WATTN_F16) launch_write<SrcT, __half>(ks, vs, pool, p, vec, st);
  else launch_write<SrcT, __nv_bfloat16>(ks, vs, pool, p, vec, st);
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

constexpr int kAcceptThreads = 256;
constexpr int kAcceptCtas = 148 * 8;
constexpr int kAcceptNear = 1024;   // new rows of a request that a CTA keeps at hand
constexpr int kAcceptSteps = 256;   // accepted rows moved at a time
constexpr int kAcceptBatch = 8;     // rows whose loads a thread has in flight

struct AcceptSmem {
  int parents[kAcceptNear], tokens[kAcceptNear], picked[kAcceptNear];
  int path[kAcceptSteps];
  int64_t src[kAcceptSteps], dst[kAcceptSteps];  // byte offsets in the pool, -1: no move
  int len, steps, cur;
};

// Grid (request, slice of the columns). A column is 16 bytes of every row: of
// one layer's keys or values of one head. Every CTA walks its request's tree
// itself (it is a few hundred bytes) from the root to the lowest child whose
// token is the one picked at its parent, until there is none, and moves its
// columns of the accepted rows. Path rows ascend and row j of the path lands
// at or before its own place, so no store overwrites what a later load of
// the same column reads. Bound: latency for a few requests (6.4 us for one of
// 16 drafts), then HBM (32 requests of up to 64 drafts in 32 layers of 20
// heads, 25 MB moved: 11.9 us, the walk included).
__global__ void __launch_bounds__(kAcceptThreads) paged_accept_kernel(const AcceptParams p) {
  grid_dep_wait();  // (launched with programmatic serialisation)
  grid_dep_launch();
  __shared__ AcceptSmem s;
  const int tid = threadIdx.x, lane = tid & 31, q = blockIdx.x;
  const int2 rw = rows_of(p.row_start, q, p.max_rows);
  const int a = rw.x, n = rw.y;
  const bool writer = blockIdx.y == 0, near = n <= kAcceptNear;
  if (near) {
    for (int i = tid; i < n; i += kAcceptThreads) {
      s.parents[i] = p.parents != nullptr ? p.parents[a + i] : i - 1;
      s.tokens[i] = p.tokens[a + i];
      s.picked[i] = p.picked[a + i];
    }
  }
  __syncthreads();
  const int row_units = p.row_bytes / 16;
  const int64_t columns = (int64_t)p.n_layers * 2 * p.n_heads * row_units;
  const int64_t head_bytes = (int64_t)p.page_rows * p.row_bytes;
  const int64_t page_bytes = (int64_t)p.n_layers * 2 * p.n_heads * head_bytes;
  int cur = -1, next = 0, done = 0;  // (warp 0) last accepted row, next candidate; rows accepted
  for (;;) {
    if (tid < 32) {
      int steps = 0;
      if (cur < 0 && done == 0 && n > 0) {
        const int root = near ? s.parents[0] : p.parents != nullptr ? p.parents[a] : -1;
        if (root == -1) {
          cur = 0;
          next = 1;
          if (lane == 0) s.path[0] = 0;
          steps = 1;
        }
      }
      while (cur >= 0 && steps < kAcceptSteps && next < n) {
        const int want = near ? s.picked[cur] : p.picked[a + cur];
        int found = -1;
        for (; next < n; next += 32) {
          const int c = next + lane;
          bool hit = false;
          if (c < n)
            hit = near ? s.tokens[c] == want && s.parents[c] == cur
                       : p.tokens[a + c] == want &&
                             (p.parents != nullptr ? p.parents[a + c] : c - 1) == cur;
          const unsigned m = __ballot_sync(0xffffffffu, hit);
          if (m) {
            found = next + __ffs(m) - 1;
            break;
          }
        }
        if (found < 0) break;
        cur = found;
        next = found + 1;
        if (lane == 0) s.path[steps] = cur;
        ++steps;
      }
      if (lane == 0) {
        s.steps = steps;
        s.cur = cur;
      }
    }
    __syncthreads();
    const int steps = s.steps;
    for (int i = tid; i < steps; i += kAcceptThreads) {
      const int j = done + i, from = s.path[i];
      if (writer) p.path[a + j] = from;
      int64_t so = -1, to = -1;
      if (from != j) {
        const int src = p.row_slot[a + from], dst = p.row_slot[a + j];
        if ((unsigned)src < (unsigned)p.n_slots && (unsigned)dst < (unsigned)p.n_slots) {
          so = src / p.page_rows * page_bytes + (int64_t)(src % p.page_rows) * p.row_bytes;
          to = dst / p.page_rows * page_bytes + (int64_t)(dst % p.page_rows) * p.row_bytes;
        }
      }
      s.src[i] = so;
      s.dst[i] = to;
    }
    __syncthreads();
    for (int64_t c = (int64_t)blockIdx.y * kAcceptThreads + tid; c < columns;
         c += (int64_t)gridDim.y * kAcceptThreads) {
      uint8_t *col = p.pool + c / row_units * head_bytes + c % row_units * 16;
      for (int i = 0; i < steps; i += kAcceptBatch) {
        uint4 x[kAcceptBatch];
#pragma unroll
        for (int b = 0; b < kAcceptBatch; ++b)
          if (i + b < steps && s.src[i + b] >= 0) x[b] = *reinterpret_cast<const uint4 *>(col + s.src[i + b]);
#pragma unroll
        for (int b = 0; b < kAcceptBatch; ++b)
          if (i + b < steps && s.src[i + b] >= 0) *reinterpret_cast<uint4 *>(col + s.dst[i + b]) = x[b];
      }
    }
    done += steps;
    if (steps < kAcceptSteps) break;
    __syncthreads();  // the path's buffer is used again
  }
  if (!writer) return;
  for (int j = done + tid; j < n; j += kAcceptThreads) p.path[a + j] = -1;
  if (q == p.n_seqs - 1)  // padding behind the last request
    for (int r = a + n + tid; r < p.max_rows; r += kAcceptThreads) p.path[r] = -1;
  if (tid == 0) {
    p.n_accepted[q] = done;
    p.next_token[q] = s.cur >= 0 ? p.picked[a + s.cur] : -1;
    p.seq_lens[q] += done;
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
                        row_slot, row_mask, mask_words, max_rows, status, false};
  cudaStream_t st = (cudaStream_t)stream;
  constexpr int smem = (int)sizeof(PlanSmem);
  if (cudaFuncSetAttribute(paged_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) !=
      cudaSuccess)
    return check_launch("cudaFuncSetAttribute(paged_plan)");
  // Up to kPlanRowsApart rows the plan's own CTAs fill them in; more are
  // worth another launch (230,000 rows: 78 us by eight CTAs).
  PlanParams q = p;
  q.rows_apart = max_rows > kPlanRowsApart;
  const int64_t work = 4LL * n_seqs + (q.rows_apart ? max_rows / page_rows : (int64_t)max_rows);
  const unsigned grid = (unsigned)std::max<int64_t>(1, std::min<int64_t>(kPlanCtas, work / kPlanRowsPerCta));
  launch_pdl_cluster(paged_plan_kernel, dim3(grid), dim3(kPlanThreads), smem, st, grid, q);
  if (q.rows_apart) {
    int rc = check_launch("paged_plan");
    if (rc != WATTN_OK) return rc;
    launch_pdl(paged_plan_rows_kernel, dim3((unsigned)((max_rows + 255LL) / 256)), dim3(256), 0, st, q);
  }
  return check_launch("paged_plan");
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
  if ((int64_t)n_rows * n_heads * 8 >= (INT64_C(1) << 39))
    return set_error(WATTN_ERR_UNSUPPORTED, "paged_write: too many rows");
  if (n_rows == 0) return WATTN_OK;
  if (!row_slot || !k_rows || !v_rows) return set_error(WATTN_ERR_INVALID, "paged_write: NULL argument");
  if (!int_aligned(row_slot) || !elem_aligned(k_rows, src_dtype) || !elem_aligned(v_rows, src_dtype))
    return set_error(WATTN_ERR_INVALID, "paged_write: arrays must be aligned to their element size");
  const WriteParams p = {row_slot, n_rows, n_pages * page_rows, n_layers, n_heads, page_rows, layer, row_stride};
  cudaStream_t st = (cudaStream_t)stream;
  if (src_dtype == WATTN_F32) return launch_write_src<float>(dtype, k_rows, v_rows, pool, p, st);
  if (src_dtype == WATTN_F16) return launch_write_src<__half>(dtype, k_rows, v_rows, pool, p, st);
  return launch_write_src<__nv_bfloat16>(dtype, k_rows, v_rows, pool, p, st);
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
  // CTAs of each request: enough that all of them fill the GPU a few times
  // over, a column per thread at the most.
  const int64_t columns = (int64_t)n_layers * 2 * n_heads * (p.row_bytes / 16);
  const int64_t most = (columns + kAcceptThreads - 1) / kAcceptThreads;
  const unsigned slices = (unsigned)std::max<int64_t>(1, std::min<int64_t>(most, kAcceptCtas / n_seqs));
  launch_pdl(paged_accept_kernel, dim3(n_seqs, slices), dim3(kAcceptThreads), 0, st, p);
  return check_launch("paged_accept");
}

}  // extern "C"
