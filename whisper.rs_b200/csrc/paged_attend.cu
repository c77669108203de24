// paged_attend.cu -- attention of drafted rows over a device-planned paged
// cache (paged.cu): packed row i of request s sees the request's seq_lens[s]
// cached positions and those of the request's new rows that its mask names
// (without masks: rows 0..i, the causal rule of decoder.rs:864).
//
// 16-bit pools: a persistent grid streams K and V once per tile of 64 rows.
// The unit of work is a 64-key sub-tile of one (request, head, row tile). The
// lengths are on the device, so every CTA adds up the requests' units itself
// and takes an equal share of them in order, wherever that cuts a row
// tile's keys (the parts of a cut one are merged by log-sum-exp, in order,
// by the CTA that finishes last: same inputs, same bits).

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
  int cap;       // positions that the table can hold
  int box_rows;  // rows of a TMA box of whole sub-tiles
  float *part;   // partials of cut items, two per CTA
  int *count;    // finished shares of the item that each CTA's share starts
  int *status;
};

// ---------------------------------------------------------------- shares of the work

constexpr int kPaSub = 64;        // keys of a sub-tile
constexpr int kPaTail = 16;       // rows of a tail box: the pool's unit of page rows
constexpr int kPaRows = 64;       // rows of a row tile
constexpr int kPaStages = 3;      // sub-tiles of the K/V ring: three CTAs to an SM
constexpr int kPaWarps = 4;       // compute warps; one more warp issues the loads
constexpr int kPaThreads = (kPaWarps + 1) * 32;
constexpr int kPaCtasPerSm = 3;
constexpr int kPaMinUnits = 4;    // units of a share below which fewer CTAs work
constexpr int kPaRedStride = 72;  // floats per row of the merge buffer: no bank met twice
constexpr int kPaPartStride = 68; // floats per row of a partial: acc[64], m, l

// One request as the kernel sees it, its arrays' values forced into range.
struct PaSeq {
  int first, n;   // packed rows
  int len;        // cached positions, all seen
  int end;        // positions that some row may see (without masks: of the last row tile)
  int row_tiles;
};

WATTN_DEVINL PaSeq pa_seq(const PagedAttendParams &p, int s, bool *bad) {
  PaSeq q;
  const int a = p.row_start[s], b = p.row_start[s + 1], len = p.seq_lens[s];
  q.first = min(max(a, 0), p.max_rows);
  q.n = min(max(b, q.first), p.max_rows) - q.first;
  q.len = min(max(len, 0), p.cap);
  const int vis = p.row_mask != nullptr ? (int)min((int64_t)q.n, (int64_t)p.mask_words * 32) : q.n;
  q.end = (int)min((int64_t)q.len + vis, (int64_t)p.cap);
  q.row_tiles = (q.n + kPaRows - 1) / kPaRows;
  if (bad != nullptr)
    *bad = a < 0 || b < a || b > p.max_rows || len < 0 || (int64_t)len + q.n > p.cap;
  return q;
}

// Positions that rows of tile rt may see.
WATTN_DEVINL int pa_end(const PagedAttendParams &p, const PaSeq &q, int rt) {
  return p.row_mask != nullptr
             ? q.end
             : (int)min((int64_t)q.len + min(q.n, kPaRows * (rt + 1)), (int64_t)q.end);
}
// Units of one row tile: its sub-tiles, and one for what an item costs besides.
WATTN_DEVINL int pa_units(const PagedAttendParams &p, const PaSeq &q, int rt) {
  return (pa_end(p, q, rt) + kPaSub - 1) / kPaSub + 1;
}
// Units of one head of a request.
WATTN_DEVINL long long pa_head_units(const PagedAttendParams &p, const PaSeq &q) {
  if (p.row_mask != nullptr) return (long long)q.row_tiles * pa_units(p, q, 0);
  long long u = 0;
  for (int rt = 0; rt < q.row_tiles; ++rt) u += pa_units(p, q, rt);
  return u;
}

// A walk over the items (request, head, row tile) of one CTA's share
// [lo, hi) of the units; `at` is the unit at which the current item starts.
struct PaWalk {
  PaSeq q;
  int s, head, rt, units;
  long long at, lo, hi;
};
WATTN_DEVINL bool pa_more(const PaWalk &w) { return w.at < w.hi; }
WATTN_DEVINL void pa_next(const PagedAttendParams &p, PaWalk &w) {
  w.at += w.units;
  if (w.at >= w.hi) return;
  if (++w.rt == w.q.row_tiles) {
    w.rt = 0;
    if (++w.head == p.n_heads) {
      w.head = 0;
      do w.q = pa_seq(p, ++w.s, nullptr); while (w.q.n == 0);
    }
  }
  w.units = pa_units(p, w.q, w.rt);
}
// The current item's sub-tiles of this share.
WATTN_DEVINL int pa_from(const PaWalk &w) { return (int)max(0ll, w.lo - w.at); }
WATTN_DEVINL int pa_to(const PaWalk &w) { return (int)min((long long)w.units - 1, w.hi - w.at); }

// The share that unit u belongs to, of `parts` shares of `total` units:
// share c is [c * total / parts, (c + 1) * total / parts).
WATTN_DEVINL int pa_owner(long long u, long long total, int parts) {
  return (int)(((u + 1) * parts - 1) / total);
}

struct PaShare {
  long long total;
  int parts;
};

// The CTA's share, found by all its threads: each adds up the units of a
// run of requests, the sums are scanned, and the thread whose run holds the
// share's first unit walks to the item that holds it.
WATTN_DEVINL void pa_find_share(const PagedAttendParams &p, PaWalk &walk, PaShare &share,
                                long long *warp_sums, PaWalk *s_walk) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = (p.n_seqs + kPaThreads - 1) / kPaThreads;
  const int s0 = min(tid * per, p.n_seqs), s1 = min(s0 + per, p.n_seqs);
  long long mine = 0;
  for (int s = s0; s < s1; ++s) {
    bool bad;
    const PaSeq q = pa_seq(p, s, &bad);
    if (bad) report_error(p.status, WATTN_ERR_RANGE, 4 << 24);
    mine += pa_head_units(p, q) * p.n_heads;
  }
  long long inc = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const long long y = __shfl_up_sync(0xffffffffu, inc, d);
    if (lane >= d) inc += y;
  }
  if (lane == 31) warp_sums[warp] = inc;
  __syncthreads();
  long long before = inc - mine, total = 0;
#pragma unroll
  for (int w = 0; w < kPaWarps + 1; ++w) {
    if (w < warp) before += warp_sums[w];
    total += warp_sums[w];
  }
  share.total = total;
  share.parts = (int)max(1ll, min((long long)gridDim.x, total / kPaMinUnits));
  const long long lo = blockIdx.x * total / share.parts;
  const long long hi = (int)blockIdx.x < share.parts ? (blockIdx.x + 1) * total / share.parts : lo;
  if (lo < hi && before <= lo && lo < before + mine) {
    PaWalk w;
    w.lo = lo;
    w.hi = hi;
    w.at = before;
    for (w.s = s0;; ++w.s) {
      w.q = pa_seq(p, w.s, nullptr);
      const long long u = pa_head_units(p, w.q);
      if (lo < w.at + u * p.n_heads) {
        w.head = (int)((lo - w.at) / u);
        w.at += w.head * u;
        break;
      }
      w.at += u * p.n_heads;
    }
    for (w.rt = 0;; ++w.rt) {
      w.units = pa_units(p, w.q, w.rt);
      if (lo < w.at + w.units) break;
      w.at += w.units;
    }
    *s_walk = w;
  }
  if (tid == 0 && lo >= hi) {
    s_walk->lo = s_walk->hi = s_walk->at = 0;
  }
  __syncthreads();
  walk = *s_walk;
}

// ---------------------------------------------------------------- 16-bit pools

template <typename T> struct PaType;
template <> struct PaType<__half> {
  static constexpr uint32_t kOne = 0x3c00u, kInf = 0x7c00u;
  static constexpr bool kResidual = false;  // f16 weights: 2^-11 each, within the 2e-3 bar
};
template <> struct PaType<__nv_bfloat16> {
  static constexpr uint32_t kOne = 0x3f80u, kInf = 0x7f80u;
  static constexpr bool kResidual = true;   // bf16's 2^-8 alone would not be: its rounding goes in too
};

struct PaSmem {
  uint8_t k[kPaStages][kPaSub * 128];
  uint8_t v[kPaStages][kPaSub * 128];
  float red[kPaWarps][16][kPaRedStride];
  float wm[kPaWarps][16], wl[kPaWarps][16];
  uint64_t kfull[kPaStages], vfull[kPaStages], empty[kPaStages];
  long long warp_sums[kPaWarps + 1];
  PaWalk walk;
  int abort, last;
};

template <typename T>
WATTN_DEVINL void pa_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (__is_same(T, __nv_bfloat16))
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
WATTN_DEVINL void pa_ldsm(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
WATTN_DEVINL void pa_ldsm_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
WATTN_DEVINL void pa_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }

// Which of the 32 positions from seq_lens + off on row i sees, as bits: all
// of the cached ones (off < 0), then the row's mask, or the rows up to itself.
WATTN_DEVINL uint32_t pa_mask_word(const PagedAttendParams &p, int packed, int i, int w) {
  if (w < 0) return 0xffffffffu;
  if (p.row_mask == nullptr) {
    const int up = i + 1 - 32 * w;
    return up >= 32 ? 0xffffffffu : up <= 0 ? 0u : (1u << up) - 1u;
  }
  return w < p.mask_words ? (uint32_t)p.row_mask[(int64_t)packed * p.mask_words + w] : 0u;
}
WATTN_DEVINL uint32_t pa_visible(const PagedAttendParams &p, int packed, int i, int off, int left) {
  if (left <= 0) return 0u;
  const int w = off >> 5;
  uint32_t bits = __funnelshift_r(pa_mask_word(p, packed, i, w), pa_mask_word(p, packed, i, w + 1),
                                  off & 31);
  return left >= 32 ? bits : bits & ((1u << left) - 1u);
}

// The two halves of a word that are infinite or NaN, as 0xffff each.
template <typename T> WATTN_DEVINL uint32_t pa_not_finite(uint32_t w) {
  constexpr uint32_t kInf2 = PaType<T>::kInf * 0x10001u;
  return __vcmpeq2(w & kInf2, kInf2);
}

// State of a warp's 16 query rows over an item: this lane's rows are g and g + 8.
struct PaAcc {
  float o[8][4];
  float m[2], l[2];
};

// One sub-tile's SL 16-key slices of this warp (slices kg, kg + 4 / SL, ...).
// few: at most 8 query rows in the tile of 16; its rows 8..15 then carry the
// weights' rounding residuals and cost no further products.
template <typename T, int SL>
WATTN_DEVINL void pa_sub_tile(const PagedAttendParams &p, const uint32_t (&qa)[4][4], PaAcc &a,
                              uint32_t ktile, uint32_t vtile, uint64_t *vbar, uint32_t ph,
                              volatile int *abort, int kg, bool few, int packed, int row, int n,
                              int off, int left, int lane) {
  constexpr int KG = kPaWarps / SL;
  const int g = lane >> 2, t4 = lane & 3;
  float sc[SL][2][4];
#pragma unroll
  for (int i = 0; i < SL; ++i) {
    const int j = kg + KG * i;
#pragma unroll
    for (int nb = 0; nb < 2; ++nb) {
      sc[i][nb][0] = sc[i][nb][1] = sc[i][nb][2] = sc[i][nb][3] = 0.f;
      const int key = j * 16 + nb * 8 + (lane & 7);
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        uint32_t r[4];
        pa_ldsm(ktile + key * 128 + (((4 * ks + (lane >> 3)) ^ (key & 7)) << 4), r);
        pa_mma<T>(sc[i][nb], qa[2 * ks], r[0], r[1]);
        pa_mma<T>(sc[i][nb], qa[2 * ks + 1], r[2], r[3]);
      }
    }
  }
  // off: first position of the sub-tile less seq_lens; left: positions of it
  // that any row may see.
  const bool drafts = off + kPaSub > 0;
  if (drafts || left < kPaSub) {
#pragma unroll
    for (int i = 0; i < SL; ++i) {
      const int j16 = (kg + KG * i) * 16;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t vis =
            row + 8 * h < n ? pa_visible(p, packed + 8 * h, row + 8 * h, off + j16, left - j16) : 0u;
#pragma unroll
        for (int nb = 0; nb < 2; ++nb)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            if (!(vis >> (nb * 8 + 2 * t4 + e) & 1u)) sc[i][nb][2 * h + e] = -INFINITY;
      }
    }
  }
  float mu[2] = {0.f, 0.f};
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if (few && h == 1) break;  // no rows there
    float mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < SL; ++i)
#pragma unroll
      for (int nb = 0; nb < 2; ++nb) mx = fmaxf(mx, fmaxf(sc[i][nb][2 * h], sc[i][nb][2 * h + 1]));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
    const float mc = mx * p.scale_log2;
    if (mc > a.m[h] + 8.0f) {  // rescale only when the running max grows by more than 2^8
      const float alpha = ex2(a.m[h] - mc);
      a.l[h] *= alpha;
#pragma unroll
      for (int db = 0; db < 8; ++db) {
        a.o[db][2 * h] *= alpha;
        a.o[db][2 * h + 1] *= alpha;
      }
      if (few)  // rows 8..15 hold the residuals of rows 0..7
#pragma unroll
        for (int db = 0; db < 8; ++db) {
          a.o[db][2] *= alpha;
          a.o[db][3] *= alpha;
        }
      a.m[h] = mc;
    }
    mu[h] = a.m[h] == -INFINITY ? 0.f : a.m[h];
  }
  mbar_wait(vbar, ph, abort, p.status, (4 << 24) | (2 << 16));
#pragma unroll
  for (int i = 0; i < SL; ++i) {
    const int j16 = (kg + KG * i) * 16;
    float pe[2][4];
#pragma unroll
    for (int nb = 0; nb < 2; ++nb)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        pe[nb][e] = ex2(fmaf(sc[i][nb][e], p.scale_log2, -mu[e >> 1]));
    uint32_t pa[4], pr[4];
#pragma unroll
    for (int nb = 0; nb < 2; ++nb) {
      a.l[0] += pe[nb][0] + pe[nb][1];
      pa[2 * nb] = pack2<T>(pe[nb][0], pe[nb][1]);
      const float2 r0 = unpack2<T>(pa[2 * nb]);
      const uint32_t lo = pack2<T>(pe[nb][0] - r0.x, pe[nb][1] - r0.y);
      if (few) {
        pa[2 * nb + 1] = lo;
      } else {
        a.l[1] += pe[nb][2] + pe[nb][3];
        pa[2 * nb + 1] = pack2<T>(pe[nb][2], pe[nb][3]);
        if constexpr (PaType<T>::kResidual) {
          const float2 r1 = unpack2<T>(pa[2 * nb + 1]);
          pr[2 * nb] = lo;
          pr[2 * nb + 1] = pack2<T>(pe[nb][2] - r1.x, pe[nb][3] - r1.y);
        }
      }
    }
    // Value rows behind the last position hold anything: zero for the product.
    const bool part = left - j16 < 16;
    uint32_t keep[2] = {0xffffffffu, 0xffffffffu};
    if (part) {
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const int k0 = j16 + b * 8 + 2 * t4;
        keep[b] = (k0 < left ? 0xffffu : 0u) | (k0 + 1 < left ? 0xffff0000u : 0u);
      }
    }
    const int key = j16 + ((lane >> 3) & 1) * 8 + (lane & 7);
    uint32_t vr[4][4];
    uint32_t odd = 0;
#pragma unroll
    for (int d2 = 0; d2 < 4; ++d2)
      pa_ldsm_t(vtile + key * 128 + (((d2 * 2 + (lane >> 4)) ^ (key & 7)) << 4), vr[d2]);
    if (part) {
#pragma unroll
      for (int d2 = 0; d2 < 4; ++d2)
#pragma unroll
        for (int e = 0; e < 4; ++e) vr[d2][e] &= keep[e & 1];
    }
    if (drafts) {
      // A draft's value that is infinite or NaN reaches the rows that see
      // it and, as 0 times it, would spoil those that do not.
#pragma unroll
      for (int d2 = 0; d2 < 4; ++d2)
#pragma unroll
        for (int e = 0; e < 4; ++e) odd |= pa_not_finite<T>(vr[d2][e]);
      if (__any_sync(0xffffffffu, odd != 0)) {
        uint32_t sees[4];
        constexpr uint32_t one = PaType<T>::kOne;
#pragma unroll
        for (int nb = 0; nb < 2; ++nb)
#pragma unroll
          for (int h = 0; h < 2; ++h)
            sees[2 * nb + h] = (sc[i][nb][2 * h] != -INFINITY ? one : 0u) |
                               (sc[i][nb][2 * h + 1] != -INFINITY ? one << 16 : 0u);
        if (few) sees[1] = sees[3] = 0u;
        constexpr uint32_t inf2 = PaType<T>::kInf * 0x10001u;
#pragma unroll
        for (int db = 0; db < 8; ++db) {
          uint32_t *v = &vr[db >> 1][(db & 1) * 2];
          // counts of +inf, -inf and NaN values that each row sees
          float np[4] = {0, 0, 0, 0}, nm[4] = {0, 0, 0, 0}, nn[4] = {0, 0, 0, 0};
          uint32_t up[2], down[2], nan[2];
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            up[b] = __vcmpeq2(v[b], inf2) & (one * 0x10001u);
            down[b] = __vcmpeq2(v[b], inf2 | 0x80008000u) & (one * 0x10001u);
            nan[b] = __vcmpgtu2(v[b] & 0x7fff7fffu, inf2) & (one * 0x10001u);
            v[b] &= ~pa_not_finite<T>(v[b]);
          }
          pa_mma<T>(np, sees, up[0], up[1]);
          pa_mma<T>(nm, sees, down[0], down[1]);
          pa_mma<T>(nn, sees, nan[0], nan[1]);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if (np[e] > 0.f) a.o[db][e] += INFINITY;
            if (nm[e] > 0.f) a.o[db][e] -= INFINITY;
            if (nn[e] > 0.f) a.o[db][e] = NAN;
          }
        }
      }
    }
#pragma unroll
    for (int db = 0; db < 8; ++db) {
      const uint32_t b0 = vr[db >> 1][(db & 1) * 2], b1 = vr[db >> 1][(db & 1) * 2 + 1];
      pa_mma<T>(a.o[db], pa, b0, b1);
      if constexpr (PaType<T>::kResidual)
        if (!few) pa_mma<T>(a.o[db], pr, b0, b1);
    }
  }
}

template <typename OutT>
WATTN_DEVINL void pa_store4(void *o, int64_t at, float4 x) {
  if constexpr (sizeof(OutT) == 4)
    *reinterpret_cast<float4 *>(reinterpret_cast<float *>(o) + at) = x;
  else
    *reinterpret_cast<uint2 *>(reinterpret_cast<OutT *>(o) + at) =
        make_uint2(pack2<OutT>(x.x, x.y), pack2<OutT>(x.z, x.w));
}

// The partial of share c for an item that share c0 starts.
WATTN_DEVINL float *pa_part(const PagedAttendParams &p, int c, int c0) {
  return p.part + ((int64_t)c * 2 + (c == c0 ? 1 : 0)) * kPaRows * kPaPartStride;
}

// An item's rows from the merged sums in `red`: stored, or, for an item cut
// by a share's end, left as a partial and merged with the others by the last
// of its shares to finish. KG warps share each tile of 16 rows.
template <typename OutT>
WATTN_DEVINL void pa_finish(const PagedAttendParams &p, PaSmem &s, const PaWalk &w,
                            const PaShare &share, int KG, int nr) {
  const int tid = threadIdx.x;
  const int row0 = w.q.first + w.rt * kPaRows;
  const int T = w.units - 1;
  const bool whole = pa_from(w) == 0 && pa_to(w) == T;
  const int c0 = pa_owner(w.at, share.total, share.parts);
  const int c1 = pa_owner(w.at + T - 1, share.total, share.parts);
  float *mine = whole ? nullptr : pa_part(p, blockIdx.x, c0);
  for (int i = tid; i < nr * 16; i += kPaWarps * 32) {
    const int r = i >> 4, d = (i & 15) * 4, w0 = (r >> 4) * KG;
    float M = -INFINITY, L = 0.f;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k = 0; k < KG; ++k) M = fmaxf(M, s.wm[w0 + k][r & 15]);
    for (int k = 0; k < KG; ++k) {
      const float4 y = *reinterpret_cast<const float4 *>(&s.red[w0 + k][r & 15][d]);
      x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
      L += s.wl[w0 + k][r & 15];
    }
    if (whole) {
      const float inv = L == 0.f ? 0.f : 1.f / L;
      pa_store4<OutT>(p.o, (int64_t)(row0 + r) * p.o_rs + w.head * 64 + d,
                      make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv));
    } else {
      *reinterpret_cast<float4 *>(mine + r * kPaPartStride + d) = x;
      if (d == 0) *reinterpret_cast<float2 *>(mine + r * kPaPartStride + 64) = make_float2(M, L);
    }
  }
  if (whole) return;
  pa_sync();
  if (tid == 0) {
    __threadfence();
    s.last = atomicAdd(&p.count[c0], 1) == c1 - c0;
    if (s.last) __threadfence();
  }
  pa_sync();
  if (!s.last) return;
  for (int i = tid; i < nr * 16; i += kPaWarps * 32) {
    const int r = i >> 4, d = (i & 15) * 4;
    float M = -INFINITY, L = 0.f;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int c = c0; c <= c1; ++c) M = fmaxf(M, __ldcg(pa_part(p, c, c0) + r * kPaPartStride + 64));
#pragma unroll 4
    for (int c = c0; c <= c1; ++c) {
      const float *q = pa_part(p, c, c0) + r * kPaPartStride;
      const float2 ml = __ldcg(reinterpret_cast<const float2 *>(q + 64));
      const float4 y = __ldcg(reinterpret_cast<const float4 *>(q + d));
      const float wt = ml.x == -INFINITY ? 0.f : ex2(ml.x - M);
      L = fmaf(wt, ml.y, L);
      x.x = fmaf(wt, y.x, x.x); x.y = fmaf(wt, y.y, x.y);
      x.z = fmaf(wt, y.z, x.z); x.w = fmaf(wt, y.w, x.w);
    }
    const float inv = L == 0.f ? 0.f : 1.f / L;
    pa_store4<OutT>(p.o, (int64_t)(row0 + r) * p.o_rs + w.head * 64 + d,
                    make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv));
  }
  if (tid == 0) p.count[c0] = 0;  // zeroed for the next call
}

// `map` has boxes of p.box_rows rows (64, 32 or 16: they lie in one page),
// `map_tail` boxes of 16.
template <typename T, typename OutT>
__global__ void __launch_bounds__(kPaThreads, kPaCtasPerSm)
    paged_attend_stream_kernel(const __grid_constant__ CUtensorMap map,
                               const __grid_constant__ CUtensorMap map_tail,
                               const PagedAttendParams p) {
  extern __shared__ uint8_t pa_smem_raw[];
  PaSmem &s = *reinterpret_cast<PaSmem *>(
      (reinterpret_cast<uintptr_t>(pa_smem_raw) + 1023) & ~uintptr_t(1023));
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int st = 0; st < kPaStages; ++st) {
      mbar_init(&s.kfull[st], 1);
      mbar_init(&s.vfull[st], 1);
      mbar_init(&s.empty[st], kPaWarps);
    }
    s.abort = 0;
    fence_barrier_init();
  }
  grid_dep_wait();  // (launched with programmatic serialisation)
  grid_dep_launch();
  PaWalk w;
  PaShare share;
  pa_find_share(p, w, share, s.warp_sums, &s.walk);
  volatile int *abort = &s.abort;
  uint32_t pos = 0;  // position in the ring

  if (warp == kPaWarps) {
    // ---- producer. Lane i holds table entry base + i of the request; a
    // request's heads follow each other, so the entries are mostly there.
    int have_s = -1, base = 0, entry = 0;
    for (; pa_more(w); pa_next(p, w)) {
      const int end = pa_end(p, w.q, w.rt);
      for (int t = pa_from(w); t < pa_to(w); ++t, ++pos) {
        const int stage = pos % kPaStages;
        const bool ok = mbar_wait(&s.empty[stage], ((pos / kPaStages) & 1) ^ 1, abort, p.status,
                                  (4 << 24) | (3 << 16) | ((pos & 0xff) << 8));
        if (!__all_sync(0xffffffffu, ok)) return;
        const int key = t * kPaSub, rows = min(kPaSub, end - key);
        const bool tail = rows < kPaSub;
        const int step = tail ? kPaTail : p.box_rows;
        const int boxes = (rows + step - 1) / step;
        if (lane == 0) {
          mbar_arrive_expect_tx(&s.kfull[stage], boxes * step * 128);
          mbar_arrive_expect_tx(&s.vfull[stage], boxes * step * 128);
        }
        for (int b = 0; b < boxes; ++b) {
          const int at = key + b * step;
          const int pi = at / p.page_rows;
          if (have_s != w.s || pi < base || pi >= base + 32) {
            have_s = w.s;
            base = pi;
            entry = base + lane < p.max_pages ? p.table[w.s * p.table_stride + base + lane] : 0;
          }
          int page = __shfl_sync(0xffffffffu, entry, pi - base);
          if (page < 0 || page >= p.n_pages) {
            if (lane == 0) report_error(p.status, WATTN_ERR_RANGE, (4 << 24) | (3 << 16));
            page = 0;
          }
          if (lane == 0) {
            const int rk = (((page * p.n_layers + p.layer) * 2) * p.n_heads + w.head) * p.page_rows +
                           at - pi * p.page_rows;
            const int rv = rk + p.n_heads * p.page_rows;
            const CUtensorMap *m = tail ? &map_tail : &map;
            tma_load_2d(s.k[stage] + b * step * 128, m, &s.kfull[stage], 0, rk);
            tma_load_2d(s.v[stage] + b * step * 128, m, &s.vfull[stage], 0, rv);
          }
        }
        __syncwarp();
      }
    }
    return;
  }

  // ---- compute warps
  const int g = lane >> 2, t4 = lane & 3;
  for (; pa_more(w); pa_next(p, w)) {
    const int from = pa_from(w), to = pa_to(w);
    if (from >= to) continue;
    const int nr = min(kPaRows, w.q.n - w.rt * kPaRows);
    // Warps to a tile of 16 rows: 4 up to 16 rows, 2 up to 32, else one.
    const int KG = nr <= 16 ? 4 : nr <= 32 ? 2 : 1;
    const int rg = warp / KG, kg = warp % KG;
    const int row = w.rt * kPaRows + rg * 16 + g, packed = w.q.first + row;
    const int here = nr - rg * 16;  // rows of this warp's tile (may be <= 0)
    const bool few = here <= 8;
    uint32_t qa[4][4];
    {
      const uint32_t *q0 = reinterpret_cast<const uint32_t *>(
          reinterpret_cast<const T *>(p.q) + (int64_t)packed * p.q_rs + w.head * 64);
      const uint32_t *q1 = reinterpret_cast<const uint32_t *>(
          reinterpret_cast<const T *>(p.q) + (int64_t)(packed + 8) * p.q_rs + w.head * 64);
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) {
        qa[ks][0] = g < here ? q0[ks * 8 + t4] : 0u;
        qa[ks][2] = g < here ? q0[ks * 8 + 4 + t4] : 0u;
        qa[ks][1] = g + 8 < here ? q1[ks * 8 + t4] : 0u;
        qa[ks][3] = g + 8 < here ? q1[ks * 8 + 4 + t4] : 0u;
      }
    }
    PaAcc a;
#pragma unroll
    for (int db = 0; db < 8; ++db) a.o[db][0] = a.o[db][1] = a.o[db][2] = a.o[db][3] = 0.f;
    a.m[0] = a.m[1] = -INFINITY;
    a.l[0] = a.l[1] = 0.f;
    const int end = pa_end(p, w.q, w.rt);
    for (int t = from; t < to; ++t, ++pos) {
      const int stage = pos % kPaStages;
      const uint32_t ph = (pos / kPaStages) & 1;
      // (a warp without rows waits too: it may not hand a stage back early)
      mbar_wait(&s.kfull[stage], ph, abort, p.status, (4 << 24) | (1 << 16) | ((pos & 0xff) << 8));
      if (here > 0) {
        const uint32_t kt = smem_u32(s.k[stage]), vt = smem_u32(s.v[stage]);
        const int off = t * kPaSub - w.q.len, left = end - t * kPaSub;
        if (KG == 4)
          pa_sub_tile<T, 1>(p, qa, a, kt, vt, &s.vfull[stage], ph, abort, kg, few, packed, row,
                            w.q.n, off, left, lane);
        else if (KG == 2)
          pa_sub_tile<T, 2>(p, qa, a, kt, vt, &s.vfull[stage], ph, abort, kg, few, packed, row,
                            w.q.n, off, left, lane);
        else
          pa_sub_tile<T, 4>(p, qa, a, kt, vt, &s.vfull[stage], ph, abort, kg, few, packed, row,
                            w.q.n, off, left, lane);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&s.empty[stage]);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      a.l[h] += __shfl_xor_sync(0xffffffffu, a.l[h], 1);
      a.l[h] += __shfl_xor_sync(0xffffffffu, a.l[h], 2);
    }
    if (few) {
#pragma unroll
      for (int db = 0; db < 8; ++db) {
        a.o[db][0] += a.o[db][2];
        a.o[db][1] += a.o[db][3];
      }
    }
    // ---- the KG warps of a tile of 16 rows merge (log-sum-exp)
    pa_sync();  // the previous item's sums have been read
    if (t4 == 0) {
      s.wm[warp][g] = a.m[0];
      s.wm[warp][g + 8] = a.m[1];
    }
    pa_sync();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (g + 8 * h >= here) continue;
      float M = -INFINITY;
      for (int k = 0; k < KG; ++k) M = fmaxf(M, s.wm[rg * KG + k][g + 8 * h]);
      const float wt = a.m[h] == -INFINITY ? 0.f : ex2(a.m[h] - M);
#pragma unroll
      for (int db = 0; db < 8; ++db)
        *reinterpret_cast<float2 *>(&s.red[warp][g + 8 * h][db * 8 + 2 * t4]) =
            make_float2(a.o[db][2 * h] * wt, a.o[db][2 * h + 1] * wt);
      if (t4 == 0) s.wl[warp][g + 8 * h] = a.l[h] * wt;
    }
    pa_sync();
    pa_finish<OutT>(p, s, w, share, KG, nr);
  }
}

int pa_grid() {
  static int sms[64] = {0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
  if (sms[dev] == 0) cudaDeviceGetAttribute(&sms[dev], cudaDevAttrMultiProcessorCount, dev);
  return sms[dev] * kPaCtasPerSm;
}

size_t pa_workspace(int grid) {
  return kCounterBytes + (size_t)grid * 2 * kPaRows * kPaPartStride * sizeof(float);
}

template <typename T, typename OutT>
int launch_stream(PagedAttendParams p, int dtype, cudaStream_t st) {
  const uint64_t rows = (uint64_t)p.n_pages * p.n_layers * 2 * p.n_heads * p.page_rows;
  p.box_rows = p.page_rows % 64 == 0 ? 64 : p.page_rows % 32 == 0 ? 32 : 16;
  const uint64_t dims[2] = {64, rows}, strides[1] = {128};
  const uint32_t box[2] = {64, (uint32_t)p.box_rows}, box_tail[2] = {64, kPaTail};
  CUtensorMap map, map_tail;
  int rc = encode_tmap(&map, tmap_dtype(dtype), 2, p.pool, dims, strides, box,
                       CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc == WATTN_OK)
    rc = encode_tmap(&map_tail, tmap_dtype(dtype), 2, p.pool, dims, strides, box_tail,
                     CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc != WATTN_OK) return rc;
  constexpr int smem = (int)sizeof(PaSmem) + 1024;
  auto kern = paged_attend_stream_kernel<T, OutT>;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
    return check_launch("cudaFuncSetAttribute(paged_attend)");
  launch_pdl(kern, dim3(pa_grid()), dim3(kPaThreads), smem, st, map, map_tail, p);
  return check_launch("paged_attend");
}

// ---------------------------------------------------------------- f32 pools

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
  return pa_workspace(pa_grid());
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
  PagedAttendParams p = {};
  p.pool = pool;
  p.n_pages = n_pages;
  p.n_layers = n_layers;
  p.n_heads = n_heads;
  p.page_rows = page_rows;
  p.layer = layer;
  p.table = block_table;
  p.table_stride = table_stride;
  p.max_pages = max_pages;
  p.seq_lens = seq_lens;
  p.row_start = row_start;
  p.n_seqs = n_seqs;
  p.row_mask = row_mask;
  p.mask_words = mask_words;
  p.q = q;
  p.o = o;
  p.q_rs = q_row_stride;
  p.o_rs = o_row_stride;
  p.max_rows = max_rows;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.cap = (int)std::min((int64_t)max_pages * page_rows, (int64_t)INT32_MAX - 2 * kPaSub);
  p.status = device_status_ptr();
  if (p.status == nullptr) return WATTN_ERR_CUDA;
  cudaStream_t st = (cudaStream_t)stream;
  const size_t need = pa_workspace(pa_grid());
  if (workspace == nullptr) {
    workspace = thread_workspace(need, st);
    if (workspace == nullptr) return set_error(WATTN_ERR_NOMEM, "paged_attend: workspace allocation failed");
  } else if (workspace_bytes < need) {
    return set_error(WATTN_ERR_INVALID, "paged_attend: workspace of %zu bytes, %zu needed",
                     workspace_bytes, need);
  } else if (reinterpret_cast<uintptr_t>(workspace) & 15) {
    return set_error(WATTN_ERR_INVALID, "paged_attend: the workspace must be 16-byte aligned");
  }
  p.count = reinterpret_cast<int *>(workspace);
  p.part = reinterpret_cast<float *>(reinterpret_cast<uint8_t *>(workspace) + kCounterBytes);
  if (dtype == WATTN_F32) return launch_simple<float, float>(p, st);
  if (dtype == WATTN_F16)
    return out_dtype == WATTN_F32 ? launch_stream<__half, float>(p, dtype, st)
                                  : launch_stream<__half, __half>(p, dtype, st);
  return out_dtype == WATTN_F32 ? launch_stream<__nv_bfloat16, float>(p, dtype, st)
                                : launch_stream<__nv_bfloat16, __nv_bfloat16>(p, dtype, st);
}

}  // extern "C"
