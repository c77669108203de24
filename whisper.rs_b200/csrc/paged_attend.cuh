// paged_attend.cuh -- what the attention kernels over a device-planned paged
// cache share (paged_attend.cu, paged_attend_wide.cu): which rows see what,
// how the work is shared out, and the walk over a share.
//
// An item is one (request, head, tile of rows), a stage some keys of it. Each
// kernel's configuration C gives kKeys of a stage, kRows of a row tile, kShares
// per CTA, kThreads that share the work out, and the units that a stage, a
// stage of more than 16 rows and an item besides its stages count for.
#pragma once

#include <limits.h>

#include "wattn_common.cuh"
#include "wattn_internal.h"

namespace wattn {

struct PagedAttendParams {
  const void *pool;
  int n_pages, n_layers, n_heads, page_rows, layer;
  const int *table;
  int64_t table_stride;
  int max_pages;
  const int *seq_lens, *row_start;
  int n_seqs;
  const int *row_mask;
  int mask_words, mask_bits;
  const void *q;
  void *o;
  int64_t q_rs, o_rs;
  int max_rows;
  float scale_log2;
  int cap;       // positions that the table can hold
  int box_rows;  // rows of a TMA box of whole stages
  float *part;   // partials of cut items
  int *count;    // finished CTAs of the item that each CTA starts and another ends
  int *taken;    // items taken from the queue
  int *status;
  int n_sm;
  bool choose;   // f16: the kernels' work decides which of the two does it
};

constexpr int kPaWarps = 4;      // narrow kernel: compute warps (one warpgroup), and as many load warps
constexpr int kPaThreads = 2 * kPaWarps * 32;
constexpr int kPaCtasPerSm = 2;
constexpr int kPaTail = 16;  // rows of a tail box: the pool's unit of page rows
constexpr int kPaMostKeys = 128;  // keys of a stage, at most
// f16 weights are taken relative to a running maximum that is lowered by this
// many powers of two: with the 2^8 that it may lag behind they reach 2^15, and
// what is lost below f16's least (a weight under 2^-25, or up to 2^-25 of one
// under 2^-14) is 2^-32 of the largest weight. Relative to the maximum itself it
// would be 2^-25, and 131072 keys of such weights 2^-8 of the output.
constexpr float kPaLower16 = 7.f;

// The narrow kernel's configuration (16-bit pools). A stage is 8 KB of keys and
// values. Units, measured: two tiles of 16 rows cost a quarter more than one, an
// item as much as three stages (with 2, 3 and 2 units trees of 64 rows over
// 32768 tokens take 82 us instead of 77).
struct PaShape {
  static constexpr int kShares = kPaWarps, kThreads = kPaThreads;
  // Items to a compute warp from which they are taken one by one (cached
  // lengths from 1 to 440, f16, taken / in equal shares: 200 requests of 12
  // heads 39.5 us / 35.4, 300 52.8 / 47.8, 400 53.0 / 60.6, 600 70.2 / 79.8, 320
  // of 20 heads 61.7 / 71.2, 2000 of 3 heads 65.5 / 72.3; 300 of 20 heads and 40
  // new rows 197 / 196).
  static constexpr int kQueueItems = 4;
  static constexpr int kStageUnits = 4, kWideUnits = 5, kItemUnits = 12;
  static constexpr int kMinUnits = 16;  // units of a share below which fewer warps work
};
struct PaNarrow16 : PaShape {
  static constexpr int kKeys = 32, kRows = 32;
};
// The wide kernel's.
struct PwShape {
  static constexpr int kKeys = kPaMostKeys, kRows = 128;
  static constexpr int kShares = 1, kThreads = kPaThreads;
  static constexpr int kStageUnits = 2, kWideUnits = 2, kItemUnits = 3;
  static constexpr int kMinUnits = 4;
};

// One request as the kernel sees it. One whose arrays are out of range has
// no rows here (and is reported).
struct PaSeq {
  int first, n;   // packed rows
  int len;        // cached positions, all seen
};

WATTN_DEVINL PaSeq pa_seq(const PagedAttendParams &p, int s, bool *bad) {
  const int a = p.row_start[s], b = p.row_start[s + 1], len = p.seq_lens[s];
  const bool ok = a >= 0 && b >= a && b <= p.max_rows && len >= 0 && len <= p.cap && b - a <= p.cap - len;
  if (bad != nullptr) *bad = !ok;
  return {a, ok ? b - a : 0, len};
}
// Positions that rows of tile rt may see.
template <typename C> WATTN_DEVINL int pa_end(const PagedAttendParams &p, const PaSeq &q, int rt) {
  return q.len + min(q.n, p.row_mask != nullptr ? p.mask_bits : C::kRows * (rt + 1));
}
template <typename C> WATTN_DEVINL int pa_stages(const PagedAttendParams &p, const PaSeq &q, int rt) {
  return (pa_end<C>(p, q, rt) + C::kKeys - 1) / C::kKeys;
}
// Units that a stage of row tile rt costs: two tiles of 16 rows cost more
// than one; C::kItemUnits are what an item costs besides its stages.
template <typename C> WATTN_DEVINL int pa_weight(const PaSeq &q, int rt) {
  return C::kRows > 16 && q.n - rt * C::kRows > 16 ? C::kWideUnits : C::kStageUnits;
}
template <typename C> WATTN_DEVINL int pa_units(const PagedAttendParams &p, const PaSeq &q, int rt) {
  return pa_stages<C>(p, q, rt) * pa_weight<C>(q, rt) + C::kItemUnits;
}
// Units of one head of a request: its full row tiles, then the last.
template <typename C> WATTN_DEVINL long long pa_head_units(const PagedAttendParams &p, const PaSeq &q) {
  if (q.n <= C::kRows) return q.n > 0 ? pa_units<C>(p, q, 0) : 0;
  const long long full = (q.n - 1) / C::kRows;
  long long stages = full * pa_stages<C>(p, q, 0);
  if (p.row_mask == nullptr) stages += full * (full - 1) / 2;  // one more from tile to tile
  return stages * pa_weight<C>(q, 0) + full * C::kItemUnits + pa_units<C>(p, q, (int)full);
}

// Whether a step (f16) is for the wide kernel: the narrow one's units are more
// than kPaWideRatio times the wide one's, and kPaWideUnits or more to each of
// its compute warps (below, the wide kernel's start of 20 us shows). Narrow /
// wide, us, trees of 128 rows unless said: 16 requests of 8 heads, 4096 cached
// 92 / 68, 64 rows 58 / 66, 100 rows 87 / 69, 160 rows 115 / 111, 256 rows
// 181 / 112; 16 of 16 heads, 2000 cached 101 / 83, 500 cached 47 / 46; 64 of 20
// heads, 300 cached 127 / 135, 384 cached 121 / 109; chains of 512 rows over
// 4000, 4 of 20 heads 208 / 146; 60 mixed requests of 20 heads, most with one
// row 150 / 273; one of one head, 1000 rows over 4000 26 / 39. Of 73 such points
// the rule takes the slower kernel by 9 % at most.
constexpr int kPaWideRatio = 33;
constexpr long long kPaWideUnits = 150;
constexpr int kPaWideCap = 512;  // positions of a table below which no point was the wide kernel's
struct PaChoice {
  long long narrow[kPaThreads / 32], wide[kPaThreads / 32];
};
WATTN_DEVINL bool pa_takes_wide(const PagedAttendParams &p, PaChoice &s) {
  long long narrow = 0, wide = 0;
  for (int i = threadIdx.x; i < p.n_seqs; i += kPaThreads) {
    const PaSeq q = pa_seq(p, i, nullptr);
    narrow += pa_head_units<PaNarrow16>(p, q);
    wide += pa_head_units<PwShape>(p, q);
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) {
    narrow += __shfl_xor_sync(0xffffffffu, narrow, d);
    wide += __shfl_xor_sync(0xffffffffu, wide, d);
  }
  if ((threadIdx.x & 31) == 0) {
    s.narrow[threadIdx.x >> 5] = narrow;
    s.wide[threadIdx.x >> 5] = wide;
  }
  __syncthreads();
  narrow = wide = 0;
#pragma unroll
  for (int w = 0; w < kPaThreads / 32; ++w) {
    narrow += s.narrow[w];
    wide += s.wide[w];
  }
  return narrow > kPaWideRatio * wide &&
         narrow * p.n_heads >= kPaWideUnits * p.n_sm * kPaCtasPerSm * kPaWarps;
}

// `total` units (below 2^31) in `parts` shares, in order: the first `more` of
// them have size + 1 units, the others size.
struct PaShares {
  int size, parts, more;
};
template <typename C> WATTN_DEVINL PaShares pa_shares(int total, int max_parts) {
  PaShares s;
  s.parts = max(1, min(max_parts, total / C::kMinUnits));
  // (whole CTAs: then a few items of one size are cut alike, and merged in one)
  if (s.parts > C::kShares) s.parts -= s.parts % C::kShares;
  s.size = total / s.parts;
  s.more = total - s.size * s.parts;
  return s;
}
WATTN_DEVINL int pa_share_begin(const PaShares &s, int c) { return c * s.size + min(c, s.more); }
// The share that unit u belongs to.
WATTN_DEVINL int pa_owner(const PaShares &s, int u) {
  const int big = s.more * (s.size + 1);
  return u < big ? u / (s.size + 1) : s.more + (u - big) / s.size;
}

// Where a share [lo, hi) begins: its first item (s, head, rt) starts at unit
// `at` <= lo.
struct PaStart {
  PaSeq q;
  int s, head, rt;
  int at, lo, hi;
};

// An item of a warp's share, as the loads announce it to the products.
struct PaItem {
  int row0, nr;      // packed rows of the tile
  int row;           // the tile's first row in the request
  int len, end;      // cached positions, positions that some row may see
  int head;
  int from, to, stages, weight;  // stages of this share, of the item; units of one
  int at;            // the item's first unit
};

// What finding the shares leaves behind (shared memory).
template <typename C> struct PaFind {
  int run_first[C::kShares], run_at[C::kShares];
  long long warp_sums[C::kThreads / 32];
  PaShares shares;
  int total;
  // Of a queue: (items and the units of the largest, of each warp's requests.)
  int warp_items[C::kThreads / 32], warp_most[C::kThreads / 32];
  // Whether the items are taken one by one; their number, that of the large
  // ones (over `small` units), and for each thread's run of requests the
  // large and the other items before its own.
  bool queue;
  int items, large, small;
  int run_large[C::kThreads], run_small[C::kThreads];
};

// The row tiles of a request, and the units of its largest item.
template <typename C> WATTN_DEVINL int pa_tiles(const PaSeq &q) { return (q.n + C::kRows - 1) / C::kRows; }
template <typename C> WATTN_DEVINL int pa_most(const PagedAttendParams &p, const PaSeq &q) {
  return q.n > 0 ? max(pa_units<C>(p, q, 0), pa_units<C>(p, q, pa_tiles<C>(q) - 1)) : 0;
}

// The shares. All threads of the CTA add up the units of a run of requests
// each; the sums are scanned, and for each share of the CTA the run that
// holds its first unit is noted. With QUEUE, many items of about the same size
// are left whole, for the warps to take one by one: those of more than half
// the largest's units first, so that short ones even out the end.
template <typename C, bool QUEUE = false> WATTN_DEVINL void pa_find_shares(const PagedAttendParams &p, PaFind<C> &s) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = (p.n_seqs + C::kThreads - 1) / C::kThreads;
  const int s0 = min(tid * per, p.n_seqs), s1 = min(s0 + per, p.n_seqs);
  long long mine = 0;
  int items = 0, most = 0;
#pragma unroll 4
  for (int i = s0; i < s1; ++i) {
    bool bad;
    const PaSeq q = pa_seq(p, i, &bad);
    if (bad) report_range(p.status, 4 << 24);
    mine += pa_head_units<C>(p, q) * p.n_heads;
    if constexpr (QUEUE) {
      items += pa_tiles<C>(q) * p.n_heads;
      most = max(most, pa_most<C>(p, q));
    }
  }
  if constexpr (QUEUE) {
    items = __reduce_add_sync(0xffffffffu, items);
    most = __reduce_max_sync(0xffffffffu, most);
    if (lane == 0) {
      s.warp_items[warp] = items;
      s.warp_most[warp] = most;
    }
  }
  long long inc = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const long long y = __shfl_up_sync(0xffffffffu, inc, d);
    if (lane >= d) inc += y;
  }
  if (lane == 31) s.warp_sums[warp] = inc;
  __syncthreads();
  long long before = inc - mine, total = 0;
#pragma unroll
  for (int w = 0; w < C::kThreads / 32; ++w) {
    if (w < warp) before += s.warp_sums[w];
    total += s.warp_sums[w];
  }
  if (total > INT_MAX) {  // more than a call may ask for
    if (tid == 0) report_range(p.status, 4 << 24);
    total = 0;
  }
  if constexpr (QUEUE) {
    items = most = 0;
#pragma unroll
    for (int w = 0; w < C::kThreads / 32; ++w) {
      items += s.warp_items[w];
      most = max(most, s.warp_most[w]);
    }
    const int parts = gridDim.x * C::kShares;
    // (the same for all CTAs)
    const bool queue = total > 0 && items >= C::kQueueItems * parts && most <= total / parts / 2;
    if (tid == 0) s.queue = queue;
    if (queue) {
      int large = 0, small = 0;
      for (int i = s0; i < s1; ++i) {
        const PaSeq q = pa_seq(p, i, nullptr);
        (pa_most<C>(p, q) > most / 2 ? large : small) += pa_tiles<C>(q) * p.n_heads;
      }
      int a = large, b = small;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, a, d), y = __shfl_up_sync(0xffffffffu, b, d);
        if (lane >= d) a += x, b += y;
      }
      __syncthreads();  // (warp_items has been read)
      if (lane == 31) {
        s.warp_items[warp] = a;
        s.warp_most[warp] = b;
      }
      __syncthreads();
      int la = 0, lb = 0, all = 0;
#pragma unroll
      for (int w = 0; w < C::kThreads / 32; ++w) {
        all += s.warp_items[w];
        if (w < warp) la += s.warp_items[w], lb += s.warp_most[w];
      }
      s.run_large[tid] = la + a - large;
      s.run_small[tid] = all + lb + b - small;
      if (tid == 0) {
        s.items = items;
        s.large = all;
        s.small = most / 2;
      }
      __syncthreads();
      return;
    }
  }
  const PaShares shares = pa_shares<C>((int)total, gridDim.x * C::kShares);
  if (tid == 0) {
    s.shares = shares;
    s.total = (int)total;
  }
  const int c0 = blockIdx.x * C::kShares;
#pragma unroll
  for (int k = 0; k < C::kShares; ++k) {
    const int lo = pa_share_begin(shares, c0 + k);
    if (c0 + k < shares.parts && before <= lo && lo < before + mine) {
      s.run_first[k] = s0;
      s.run_at[k] = (int)before;
    }
  }
  __syncthreads();
}

// Share blockIdx.x * C::kShares + k: walks to its first item.
template <typename C> WATTN_DEVINL PaStart pa_start(const PagedAttendParams &p, const PaFind<C> &s, int k) {
  PaStart w;
  w.lo = w.hi = 0;
  const int c = blockIdx.x * C::kShares + k;
  if (c >= s.shares.parts || s.total == 0) return w;
  w.lo = pa_share_begin(s.shares, c);
  w.hi = pa_share_begin(s.shares, c + 1);
  w.at = s.run_at[k];
  // (The walks end with the requests and row tiles even if another stream
  // changes the arrays meanwhile.)
  for (w.s = s.run_first[k];; ++w.s) {
    if (w.s >= p.n_seqs) {
      w.hi = w.lo;
      return w;
    }
    w.q = pa_seq(p, w.s, nullptr);
    const int u = (int)pa_head_units<C>(p, w.q);
    if (w.lo - w.at < (long long)u * p.n_heads) {
      w.head = (w.lo - w.at) / u;
      w.at += w.head * u;
      break;
    }
    w.at += u * p.n_heads;
  }
  for (w.rt = 0;; ++w.rt) {
    if (w.rt * C::kRows >= w.q.n) {
      w.hi = w.lo;
      return w;
    }
    const int u = pa_units<C>(p, w.q, w.rt);
    if (w.lo - w.at < u) break;
    w.at += u;
  }
  return w;
}

// Which of the 32 positions from seq_lens + off on row i sees, as bits: all
// of the cached ones (off < 0), then the row's mask, or the rows up to itself;
// `left` positions of them exist.
WATTN_DEVINL uint32_t pa_mask_word(const PagedAttendParams &p, int packed, int i, int w) {
  if (w < 0) return 0xffffffffu;
  if (p.row_mask == nullptr) {
    const int up = i + 1 - 32 * w;
    return up >= 32 ? 0xffffffffu : up <= 0 ? 0u : (1u << up) - 1u;
  }
  return w < p.mask_words ? (uint32_t)p.row_mask[(int64_t)packed * p.mask_words + w] : 0u;
}
WATTN_DEVINL uint32_t pa_visible(const PagedAttendParams &p, int packed, int i, int off, int left) {
  const int w = off >> 5;
  const uint32_t bits = __funnelshift_r(pa_mask_word(p, packed, i, w),
                                        pa_mask_word(p, packed, i, w + 1), off & 31);
  return left >= 32 ? bits : bits & ((1u << left) - 1u);
}

// A walk over a share.
struct PaLoads {
  PaStart w;
  int units, stages, weight;  // of the current item
  int t, to, end;        // its next stage, the share's last, its positions
  int page, in_page;     // table index and row of the next box
};

// The current item's stages that this share holds (a stage belongs to the
// share that holds its first unit), and where their keys are. False if none.
template <typename C> WATTN_DEVINL bool pa_enter(const PagedAttendParams &p, PaLoads &ld) {
  const PaStart &w = ld.w;
  ld.units = pa_units<C>(p, w.q, w.rt);
  ld.stages = pa_stages<C>(p, w.q, w.rt);
  ld.weight = pa_weight<C>(w.q, w.rt);
  const int d = w.lo - w.at, e = w.hi - w.at;
  ld.t = d <= 0 ? 0 : (d + ld.weight - 1) / ld.weight;
  ld.to = e >= ld.units ? ld.stages : min(ld.stages, (e + ld.weight - 1) / ld.weight);
  ld.end = pa_end<C>(p, w.q, w.rt);
  ld.page = ld.t * C::kKeys / p.page_rows;
  ld.in_page = ld.t * C::kKeys - ld.page * p.page_rows;
  return ld.t < ld.to;
}

// On to the next item of the share that has stages in it; false at the end.
// `fresh` is set on entering an item, `moved` on entering another request.
template <typename C>
WATTN_DEVINL bool pa_advance(const PagedAttendParams &p, PaLoads &ld, bool &fresh, bool &moved) {
  PaStart &w = ld.w;
  while (ld.t >= ld.to) {
    w.at += ld.units;
    if (w.at >= w.hi) return false;
    if (++w.rt * C::kRows >= w.q.n) {
      w.rt = 0;
      if (++w.head == p.n_heads) {
        w.head = 0;
        do {
          if (++w.s >= p.n_seqs) return false;
          w.q = pa_seq(p, w.s, nullptr);
        } while (w.q.n == 0);
        moved = true;
      }
    }
    fresh = pa_enter<C>(p, ld);
  }
  return true;
}

// Item k of those taken one by one, whole: the large ones in the order of
// requests, heads and row tiles, then the others. False if there is none (the
// arrays were changed meanwhile).
template <typename C>
WATTN_DEVINL bool pa_take(const PagedAttendParams &p, const PaFind<C> &s, PaLoads &ld, int k, int lane) {
  const bool large = k < s.large;
  const int *run = large ? s.run_large : s.run_small;
  int lo = 0, hi = C::kThreads;  // the last run with at most k items before it
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (run[mid] <= k) lo = mid; else hi = mid;
  }
  const int per = (p.n_seqs + C::kThreads - 1) / C::kThreads;
  PaStart &w = ld.w;
  int left = k - run[lo];
  for (int first = lo * per; first < p.n_seqs; first += 32) {
    // (32 requests at a time)
    int here = 0;
    if (first + lane < p.n_seqs) {
      const PaSeq q = pa_seq(p, first + lane, nullptr);
      if ((pa_most<C>(p, q) > s.small) == large) here = pa_tiles<C>(q) * p.n_heads;
    }
    int upto = here;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, upto, d);
      if (lane >= d) upto += x;
    }
    const unsigned over = __ballot_sync(0xffffffffu, upto > left);
    if (over != 0) {
      const int at = __ffs(over) - 1;
      left -= __shfl_sync(0xffffffffu, upto - here, at);
      w.s = first + at;
      w.q = pa_seq(p, w.s, nullptr);
      const int tiles = pa_tiles<C>(w.q);
      if (tiles == 0) return false;
      w.head = left / tiles;
      w.rt = left - w.head * tiles;
      w.at = w.lo = 0;
      w.hi = INT_MAX;
      return w.head < p.n_heads && pa_enter<C>(p, ld);
    }
    left -= __shfl_sync(0xffffffffu, upto, 31);
  }
  return false;
}

// The current item, as the loads announce it.
template <typename C>
WATTN_DEVINL PaItem pa_item_of(const PaLoads &ld) {
  const PaStart &w = ld.w;
  const int row = w.rt * C::kRows;
  PaItem it;
  it.row0 = w.q.first + row;
  it.nr = min(C::kRows, w.q.n - row);
  it.row = row;
  it.len = w.q.len;
  it.end = ld.end;
  it.head = w.head;
  it.from = ld.t;
  it.to = ld.to;
  it.stages = ld.stages;
  it.weight = ld.weight;
  it.at = w.at;
  return it;
}

// The kernel for many new rows a request (paged_attend_wide.cu), f16 pools.
int launch_paged_attend_wide(const PagedAttendParams &p, int out_dtype, cudaStream_t st);
size_t paged_attend_wide_workspace(int n_sm);

}  // namespace wattn
