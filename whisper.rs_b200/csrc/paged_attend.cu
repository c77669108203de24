// paged_attend.cu -- attention of drafted rows over a device-planned paged
// cache (paged.cu): packed row i of request s sees the request's seq_lens[s]
// cached positions and those of the request's new rows that its mask names
// (without masks: rows 0..i, the causal rule of decoder.rs:864).
//
// 16-bit pools. Bound: HBM (each key's K and V, 256 bytes, meet up to 32
// query rows: 4 * 64 * 32 products on the tensor cores for 256 bytes). Every
// compute warp streams for itself: it has its own ring of three 32-key
// stages, which a load warp of its own fills by TMA through the block table,
// and multiplies with mma.sync; compute warps meet only when they are done.
// (A compute warp that issues its own loads spends 660 of 2400 cycles a stage
// on that.) An item is one (request, head, tile of up to 32 rows). The lengths
// are on the device, so each CTA adds up the requests' work itself and each
// compute warp takes an equal share of it, in order, wherever that cuts an
// item's keys. The parts of a cut item are merged by log-sum-exp in the order
// of the keys, by its CTA or, where it spans several, by the last of them:
// same inputs, same bits.
//
// Many small items (a step of 320 beams x 20 heads) are not cut but taken one
// by one from a counter: the warps of an SM share what it can read, so equal
// shares end unequally, and taken ones even that out. 370 MB of keys and
// values: bf16 70 us (5.3 TB/s); 320 beams over up to 440 tokens, f16: 61.7 us
// against 71.2 in equal shares.
//
// Elsewhere the chain of one stage bounds (scores, maximum, weights, products,
// with eight compute warps on an SM): 64 trees of up to 33 rows over up to 448
// tokens, 20 heads, f16 36 us (82 MB); 8 trees of up to 64 rows over up to
// 32768 tokens, 8 heads, bf16 76 us (238 MB); one tree of 16 rows 10.6 us, of
// which 3 are the launch. (Replayed graphs.)
#include <algorithm>

#include "paged_attend.cuh"

namespace wattn {

namespace {

// ---------------------------------------------------------------- shares of the work

constexpr int kPaStageBytes = 8192;  // keys, then values
constexpr int kPaStages = 3;      // stages of a warp's ring
// Registers per thread: what the block is launched with, then after the
// warpgroups' split (whose sum may not exceed twice the launch's).
constexpr int kPaRegs = 128, kPaComputeRegs = 216, kPaLoadRegs = 40;
static_assert(kPaComputeRegs + kPaLoadRegs <= 2 * kPaRegs, "a larger split never gets its registers");
// Whether a step of these sizes can be one for the wide kernel (pa_takes_wide):
// else only the narrow one is launched. What the requests hold is on the
// device; the buffers bound it.
inline bool pa_may_be_wide(const PagedAttendParams &p) {
  const int64_t tiles = (int64_t)p.max_rows / PaNarrow16::kRows + p.n_seqs;
  const int64_t stages = (p.cap + PaNarrow16::kKeys - 1) / PaNarrow16::kKeys;
  const int64_t units = tiles * (stages * PaNarrow16::kWideUnits + PaNarrow16::kItemUnits);
  return p.max_rows / p.n_seqs > PwShape::kRows - PaNarrow16::kRows && p.cap >= kPaWideCap &&
         units >= kPaWideUnits * p.n_sm * kPaCtasPerSm * kPaWarps / p.n_heads;
}
constexpr int kPaMergeAll = 8;    // CTAs beyond the first from which all warps merge an item
constexpr int kPaQueue = 8;       // items a warp may have loads for, and one more
constexpr int kPaTileFloats = 32 * 36;  // a partial's tile of 16 rows: 36 floats a lane
static_assert(kPaStages * kPaStageBytes >= kPaWarps * kPaTileFloats * 4, "a ring holds the warps' sums");

template <typename T> struct PaType;
template <> struct PaType<__half> : PaNarrow16 {
  static constexpr uint32_t kOne = 0x3c00u, kInf = 0x7c00u;
  // f16 weights of 9 rows or more: 2^-11 each, within the 2e-3 bar (with their
  // residuals one tree of 16 rows takes 12.9 us instead of 10.6, 64 of up to 33
  // 40.9 instead of 35.9).
  static constexpr bool kResidual = false;
  static constexpr float kLower = kPaLower16;
};
template <> struct PaType<__nv_bfloat16> : PaNarrow16 {
  static constexpr uint32_t kOne = 0x3f80u, kInf = 0x7f80u;
  static constexpr bool kResidual = true;   // bf16's 2^-8 alone would not be: its rounding goes in too
  static constexpr float kLower = 0.f;      // (f32's range)
};
template <> struct PaType<float> : PaShape {
  static constexpr int kKeys = 16, kRows = 16;
  // (8 / 16 units, 13 rows a request: 1 request of 6 heads over 448 tokens 12.2
  // us / 13.7, 4 of them 13.4 / 15.7, 16 of 8 heads over 224 tokens 13.9 / 16.4,
  // 1 of 8 heads over 4000 17.2 / 18.4; 4 units as 8, 32 up to 45 % longer.)
  static constexpr int kMinUnits = 8;
};
static_assert(PaType<__half>::kKeys <= kPaMostKeys && PaType<float>::kKeys <= kPaMostKeys, "see kPaMostKeys");

template <typename T>
struct PaSmem {
  uint8_t kv[kPaWarps][kPaStages][kPaStageBytes];
  uint64_t full[kPaWarps][kPaStages], empty[kPaWarps][kPaStages];
  PaItem queue[kPaWarps][kPaQueue];
  PaItem cut[kPaWarps][2];  // items cut by the share's begin and by its end (stages 0: none)
  PaFind<PaType<T>> find;
  PaChoice choice;
  int merge_first[2 * kPaWarps], merge_last[2 * kPaWarps];  // shares to merge, per cut item
  int final[2 * kPaWarps];  // this CTA merges the parts of them all
  int abort;
};

// ---------------------------------------------------------------- 16-bit pools

// (volatile: else the compiler computes the products of a branch not taken)
template <typename T>
WATTN_DEVINL void pa_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (__is_same(T, __nv_bfloat16))
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// The same with D = A B.
template <typename T>
WATTN_DEVINL void pa_mma0(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (__is_same(T, __nv_bfloat16))
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
// Four 8x8 matrices at addr + OFF; _t: transposed.
template <int OFF> WATTN_DEVINL void pa_ldsm(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4 + %5];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr), "n"(OFF)
               : "memory");
}
template <int OFF> WATTN_DEVINL void pa_ldsm_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4 + %5];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr), "n"(OFF)
               : "memory");
}

// The two halves of a word that are infinite or NaN, as 0xffff each.
template <typename T> WATTN_DEVINL uint32_t pa_not_finite(uint32_t w) {
  constexpr uint32_t kInf2 = PaType<T>::kInf * 0x10001u;
  return __vcmpeq2(w & kInf2, kInf2);
}

// x, or NaN in a half where that of w is infinite or NaN (x: two zeros of T).
template <typename T> WATTN_DEVINL uint32_t pa_nil(uint32_t w, uint32_t x) {
  if constexpr (__is_same(T, __nv_bfloat16))
    asm("fma.rn.bf16x2 %0, %1, %2, %0;" : "+r"(x) : "r"(w), "r"(0u));
  else
    asm("fma.rn.f16x2 %0, %1, %2, %0;" : "+r"(x) : "r"(w), "r"(0u));
  return x;
}
// The halves of a word holding keys k and k + 1 that lie before `left`.
WATTN_DEVINL uint32_t pa_keep(int k, int left) {
  return k + 1 < left ? 0xffffffffu : k < left ? 0xffffu : 0u;
}

template <typename OutT> WATTN_DEVINL void pa_store2(void *o, int64_t at, float x, float y) {
  if constexpr (sizeof(OutT) == 4)
    *reinterpret_cast<float2 *>(reinterpret_cast<float *>(o) + at) = make_float2(x, y);
  else
    *reinterpret_cast<uint32_t *>(reinterpret_cast<OutT *>(o) + at) = pack2<OutT>(x, y);
}
// A warp's 16 query rows over some keys: this lane's part of rows g and g + 8.
struct PaTile {
  float o[8][4];     // dims 8 db + 2 t4 and + 1 of row g, then of row g + 8
  float m[2], l[2];  // running max (less kLower); sum of this lane's weights
};

// Partials of cut items, in the lanes' layout: two slots per share (`starts`:
// the item that the share starts), behind them two per CTA.
WATTN_DEVINL float4 *pa_part(const PagedAttendParams &p, int slot, bool starts, int mt, int lane) {
  return reinterpret_cast<float4 *>(
             p.part + (((int64_t)slot * 2 + (starts ? 1 : 0)) * 2 + mt) * kPaTileFloats) + lane;
}
WATTN_DEVINL void pa_put(float4 *part, const PaTile &a) {
#pragma unroll
  for (int db = 0; db < 8; ++db) part[db * 32] = make_float4(a.o[db][0], a.o[db][1], a.o[db][2], a.o[db][3]);
  part[8 * 32] = make_float4(a.m[0], a.m[1], a.l[0], a.l[1]);
}
// Adds a partial to `a` (log-sum-exp). L2: it is other threads', in global memory.
template <bool L2 = true> WATTN_DEVINL void pa_add(PaTile &a, const float4 *part) {
  float4 x[9];
#pragma unroll
  for (int i = 0; i < 9; ++i) x[i] = L2 ? __ldcg(part + i * 32) : part[i * 32];
  float wa[2], wb[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const float mb = h ? x[8].y : x[8].x, lb = h ? x[8].w : x[8].z;
    const float m = fmaxf(a.m[h], mb);
    wa[h] = a.m[h] == -INFINITY ? 0.f : ex2(a.m[h] - m);
    wb[h] = mb == -INFINITY ? 0.f : ex2(mb - m);
    a.m[h] = m;
    a.l[h] = fmaf(a.l[h], wa[h], wb[h] * lb);
  }
#pragma unroll
  for (int db = 0; db < 8; ++db) {
    a.o[db][0] = fmaf(a.o[db][0], wa[0], wb[0] * x[db].x);
    a.o[db][1] = fmaf(a.o[db][1], wa[0], wb[0] * x[db].y);
    a.o[db][2] = fmaf(a.o[db][2], wa[1], wb[1] * x[db].z);
    a.o[db][3] = fmaf(a.o[db][3], wa[1], wb[1] * x[db].w);
  }
}
// The outputs of packed rows row0 + g and + 8 (nr rows exist), head h.
template <typename T, typename OutT>
WATTN_DEVINL void pa_output(const PagedAttendParams &p, const PaTile &a, int row0, int nr, int head,
                            int lane) {
  const int g = lane >> 2, t4 = lane & 3;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float sum = a.l[h];
    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
    if (g + 8 * h >= nr) continue;
    const float inv = sum == 0.f ? 0.f : __fdividef(1.f, sum);
    const int64_t at = (int64_t)(row0 + g + 8 * h) * p.o_rs + head * 64;
    if constexpr (sizeof(T) == 4) {  // (the f32 products' order of dims: pa_item)
      float *o = reinterpret_cast<float *>(p.o) + at + (t4 >> 1) * 32 + (t4 & 1) * 8;
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int c = 2 * h + e;
          *reinterpret_cast<float4 *>(o + j * 16 + e * 4) =
              make_float4(a.o[4 * j][c] * inv, a.o[4 * j + 1][c] * inv, a.o[4 * j + 2][c] * inv,
                          a.o[4 * j + 3][c] * inv);
        }
    } else {
#pragma unroll
      for (int db = 0; db < 8; ++db)
        pa_store2<OutT>(p.o, at + 2 * t4 + db * 8, a.o[db][2 * h] * inv, a.o[db][2 * h + 1] * inv);
    }
  }
}

// Announces the current item to the compute warp.
template <typename T>
WATTN_DEVINL void pa_announce(const PagedAttendParams &p, PaItem &to, const PaLoads &ld, int lane) {
  const PaItem it = pa_item_of<PaType<T>>(ld);
  if (lane == 0) to = it;
  if (lane < it.nr) {  // its query rows and masks will be wanted soon
    asm volatile("prefetch.global.L1 [%0];" ::"l"(reinterpret_cast<const T *>(p.q) +
                                                  (int64_t)(it.row0 + lane) * p.q_rs + it.head * 64));
    if (p.row_mask != nullptr)
      asm volatile("prefetch.global.L1 [%0];" ::"l"(p.row_mask +
                                                    (int64_t)(it.row0 + lane) * p.mask_words));
  }
}

// A load warp: fills the ring of compute warp k, stage by stage over its
// share's items, each announced before its first stage; an item without rows
// ends the share.
template <typename T, bool QUEUE>
WATTN_DEVINL void pa_load(const PagedAttendParams &p, PaSmem<T> &s, const CUtensorMap &map,
                          const CUtensorMap &map_tail, int k, int lane) {
  using C = PaType<T>;
  PaLoads ld;
  const bool queue = QUEUE && s.find.queue;
  if (!queue) ld.w = pa_start<C>(p, s.find, k);
  PaStart &w = ld.w;
  int base = INT_MIN / 2, entry = 0;  // lane i holds table entry base + i of the request
  int slot = 0;
  uint32_t phase = 1;  // (a wait for the phase before the first passes)
  uint32_t items = 0, issued = 0;
  bool fresh = false;  // an item not yet announced
  const bool some = !queue && w.lo < w.hi;
  if (some) fresh = pa_enter<C>(p, ld);
  bool first = true;
  if (queue) ld.t = ld.to = 0;
#pragma unroll 1
  for (;;) {
    bool moved = false;
    bool more = some && pa_advance<C>(p, ld, fresh, moved);
    if (queue) {
      more = ld.t < ld.to;
      while (!more) {
        const int warps = gridDim.x * kPaWarps;
        int i = blockIdx.x * kPaWarps + k;  // the first by the warp's place
        if (first) {
          first = false;
        } else {
          if (lane == 0) i = warps + atomicAdd(p.taken, 1);
          i = __shfl_sync(0xffffffffu, i, 0);
        }
        if (i >= s.find.items) {
          // The last warp to find nothing left sets the count back for the next call.
          if (lane == 0 && i == s.find.items + warps - 1) *p.taken = 0;
          break;
        }
        more = fresh = moved = pa_take<C>(p, s.find, ld, i, lane);
      }
    }
    if (moved) base = INT_MIN / 2;  // another request's table
    const bool ok = mbar_wait(&s.empty[k][slot], phase, &s.abort, p.status, (4 << 24) | (3 << 16));
    if (!__all_sync(0xffffffffu, ok)) {
      // winding down: the copies in flight land before the block leaves
      volatile int no_abort = 0;
      for (int st = 0; st < kPaStages; ++st)
        if (st < (int)min(issued, (uint32_t)kPaStages)) {
          const uint32_t c = issued - 1 - st;
          mbar_wait(&s.full[k][c % kPaStages], (c / kPaStages) & 1, &no_abort, p.status,
                    (4 << 24) | (4 << 16));
        }
      return;
    }
    uint64_t *bar = &s.full[k][slot];
    PaItem &it = s.queue[k][items % kPaQueue];
    if (!more) {
      if (lane == 0) {
        it.nr = 0;
        mbar_arrive(bar);
      }
      return;
    }
    if (fresh) {
      pa_announce<T>(p, it, ld, lane);
      ++items;
      fresh = false;
    }
    constexpr bool kF32 = sizeof(T) == 4;
    const int rows = ld.end - ld.t * PaType<T>::kKeys;
    const bool tail = rows < PaType<T>::kKeys;
    const int step = kF32 || tail ? kPaTail : p.box_rows;
    const int boxes = rows > step && step < PaType<T>::kKeys ? 2 : 1;  // a step is a stage, or half of one
#pragma unroll 1
    for (int b = 0; b < boxes; ++b) {
      if ((unsigned)(ld.page - base) >= 32u) {
        base = ld.page;
        entry = base + lane < p.max_pages ? p.table[w.s * p.table_stride + base + lane] : 0;
      }
      int page = __shfl_sync(0xffffffffu, entry, ld.page - base);
      if (lane == 0) {
        if (b == 0) mbar_arrive_expect_tx(bar, boxes * step * 4 * 32 * sizeof(T));  // (releases the announcement too)
        if ((unsigned)page >= (unsigned)p.n_pages) {
          report_range(p.status, (4 << 24) | (3 << 16));
          page = 0;
        }
        const int c1 = w.head * p.page_rows + ld.in_page, c3 = page * p.n_layers + p.layer;
        uint8_t *dst = s.kv[k][slot] + b * kPaTail * 128;
        if (kF32) {  // dims 0 to 31 of the keys and of the values, then the others
          tma_load_4d(dst, &map, bar, 0, c1, 0, c3);
          tma_load_4d(dst + kPaStageBytes / 2, &map, bar, 32, c1, 0, c3);
        } else if (step == PaType<T>::kKeys) {
          tma_load_4d(dst, &map, bar, 0, c1, 0, c3);  // the keys, and behind them the values
        } else {  // 16 rows of each
          tma_load_4d(dst, &map_tail, bar, 0, c1, 0, c3);
          tma_load_4d(dst + PaType<T>::kKeys * 128, &map_tail, bar, 0, c1, 1, c3);
        }
      }
      ld.in_page += step;
      if (ld.in_page >= p.page_rows) {
        ld.in_page = 0;
        ++ld.page;
      }
    }
    ++ld.t;
    ++issued;
    if (++slot == kPaStages) {
      slot = 0;
      phase ^= 1;
    }
    __syncwarp();
  }
}

// The products of one item's stages: MT tiles of 16 query rows against 32
// keys a stage. few (at most 8 rows): rows 8..15 of the tile carry the
// weights' rounding residuals and cost no further products, so f16 has them
// there too (4.8e-7 off instead of 3.3e-4, as in the host-planned decode). (One body for
// both MT is 14 % slower over single rows, its branches being predicated
// products; one more for few rows costs more instruction fetches than it saves.)
template <typename T, typename OutT, int MT>
WATTN_DEVINL void pa_item(const PagedAttendParams &p, PaSmem<T> &s, const PaItem &it, uint32_t &pos,
                          int warp, int lane) {
  const int g = lane >> 2, t4 = lane & 3;
  const bool few = MT == 1 && it.nr <= 8;
  uint32_t qa[MT][4][4];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = mt * 16 + h * 8 + g;
      const uint32_t *q = reinterpret_cast<const uint32_t *>(
          reinterpret_cast<const T *>(p.q) + (int64_t)(it.row0 + r) * p.q_rs + it.head * 64);
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) {
        qa[mt][ks][h] = r < it.nr ? q[ks * 8 + t4] : 0u;
        qa[mt][ks][2 + h] = r < it.nr ? q[ks * 8 + 4 + t4] : 0u;
      }
    }
  PaTile a[MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
    for (int db = 0; db < 8; ++db) a[mt].o[db][0] = a[mt].o[db][1] = a[mt].o[db][2] = a[mt].o[db][3] = 0.f;
    a[mt].m[0] = a[mt].m[1] = -INFINITY;
    a[mt].l[0] = a[mt].l[1] = 0.f;
  }
  // Lane offsets: keys in rows of 128 swizzled bytes, values transposed.
  const uint32_t koff = (lane & 7) * 128 + (((lane >> 3) ^ (lane & 7)) << 4);
  const uint32_t voff = ((lane >> 3) & 1) * 1024 + (lane & 7) * 128 + (((lane >> 4) ^ (lane & 7)) << 4);
#pragma unroll 1
  for (int t = it.from; t < it.to; ++t) {
    const int slot = pos & 3;
    mbar_wait(&s.full[warp][slot], pos >> 31, &s.abort, p.status,
              (4 << 24) | (1 << 16) | ((t & 0xff) << 8));
    pos = slot == kPaStages - 1 ? (pos & 0x80000000u) ^ 0x80000000u : pos + 1;
    const uint32_t ktile = smem_u32(s.kv[warp][slot]), vtile = ktile + PaType<T>::kKeys * 128;
    float sc[MT][4][4];
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      uint32_t r[4][4];
      const uint32_t at = ktile + (koff ^ (ks * 64));
      pa_ldsm<0>(at, r[0]);
      pa_ldsm<1024>(at, r[1]);
      pa_ldsm<2048>(at, r[2]);
      pa_ldsm<3 * 1024>(at, r[3]);
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int nb = 0; nb < 4; ++nb) {
            if (ks == 0 && half == 0)
              pa_mma0<T>(sc[mt][nb], qa[mt][0], r[nb][0], r[nb][1]);
            else
              pa_mma<T>(sc[mt][nb], qa[mt][2 * ks + half], r[nb][2 * half], r[nb][2 * half + 1]);
          }
    }
    const int off = t * PaType<T>::kKeys - it.len, left = it.end - t * PaType<T>::kKeys;
    const bool drafts = off + PaType<T>::kKeys > 0;       // the stage reaches past the cached positions
    const bool special = drafts || left < PaType<T>::kKeys;
    if (special) {
      // lane r finds what row r sees
      const uint32_t sees =
          lane < it.nr ? pa_visible(p, it.row0 + lane, it.row + lane, off, left) : 0u;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t vis = __shfl_sync(0xffffffffu, sees, mt * 16 + h * 8 + g) >> (2 * t4);
#pragma unroll
          for (int nb = 0; nb < 4; ++nb)
#pragma unroll
            for (int e = 0; e < 2; ++e)
              if (!(vis >> (nb * 8 + e) & 1u)) sc[mt][nb][2 * h + e] = -INFINITY;
        }
      }
    }
    float mu[MT][2], mc[MT][2];
    bool grows = false;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (h == 1 && few) break;
        float mx = -INFINITY;
#pragma unroll
        for (int nb = 0; nb < 4; ++nb) mx = fmax3(mx, sc[mt][nb][2 * h], sc[mt][nb][2 * h + 1]);
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        mc[mt][h] = fmaf(mx, p.scale_log2, -PaType<T>::kLower);
        grows |= mc[mt][h] > a[mt].m[h] + 8.0f;
      }
    }
    // (one branch for all rows: with four, trees of 64 rows over 32768 tokens take 5 % longer)
    if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (h == 1 && few) break;
          // rescale only when the running max grows by more than 2^8
          if (!(mc[mt][h] > a[mt].m[h] + 8.0f)) continue;
          const float alpha = ex2(a[mt].m[h] - mc[mt][h]);
          a[mt].l[h] *= alpha;
#pragma unroll
          for (int db = 0; db < 8; ++db) {
            a[mt].o[db][2 * h] *= alpha;
            a[mt].o[db][2 * h + 1] *= alpha;
            if (mt == 0 && h == 0 && few) {  // rows 8..15 hold the residuals of rows 0..7
              a[0].o[db][2] *= alpha;
              a[0].o[db][3] *= alpha;
            }
          }
          a[mt].m[h] = mc[mt][h];
        }
    }
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int h = 0; h < 2; ++h) mu[mt][h] = a[mt].m[h] == -INFINITY ? 0.f : a[mt].m[h];
    // Value rows behind the last position hold anything: zero for the
    // product. A draft's value that is infinite or NaN belongs to the rows
    // that see it and would, as 0 times it, spoil those that do not.
    bool odd = false;
    if (drafts) {
      uint32_t nil = 0;  // stays 0 while all is finite
#pragma unroll
      for (int sl = 0; sl < 2; ++sl) {
        const uint32_t keep0 = pa_keep(sl * 16 + 2 * t4, left), keep1 = pa_keep(sl * 16 + 8 + 2 * t4, left);
#pragma unroll
        for (int d2 = 0; d2 < 4; ++d2) {
          uint32_t vr[4];
          pa_ldsm_t<0>(vtile + sl * 2048 + (voff ^ (d2 * 32)), vr);
          nil = pa_nil<T>(vr[0] & keep0, nil);
          nil = pa_nil<T>(vr[1] & keep1, nil);
          nil = pa_nil<T>(vr[2] & keep0, nil);
          nil = pa_nil<T>(vr[3] & keep1, nil);
        }
      }
      odd = __any_sync(0xffffffffu, pa_not_finite<T>(nil) != 0);
    }
    if (__builtin_expect(odd, 0)) {
      constexpr uint32_t one2 = PaType<T>::kOne * 0x10001u, inf2 = PaType<T>::kInf * 0x10001u;
#pragma unroll
      for (int sl = 0; sl < 2; ++sl) {
        uint32_t sees[MT][4];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int nb = sl * 2 + (e >> 1), h = e & 1;
            sees[mt][e] = h && few
                              ? 0u
                              : ((sc[mt][nb][2 * h] != -INFINITY ? 0xffffu : 0u) |
                                 (sc[mt][nb][2 * h + 1] != -INFINITY ? 0xffff0000u : 0u)) & one2;
          }
#pragma unroll
        for (int d2 = 0; d2 < 4; ++d2) {
          uint32_t vr[4];
          pa_ldsm_t<0>(vtile + sl * 2048 + (voff ^ (d2 * 32)), vr);
#pragma unroll
          for (int e = 0; e < 4; ++e) vr[e] &= pa_keep(sl * 16 + (e & 1) * 8 + 2 * t4, left);
#pragma unroll
          for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
              // how many +inf, -inf and NaN values each row sees
              float np[4] = {0, 0, 0, 0}, nm[4] = {0, 0, 0, 0}, nn[4] = {0, 0, 0, 0};
              const uint32_t v0 = vr[2 * half], v1 = vr[2 * half + 1];
              pa_mma<T>(np, sees[mt], __vcmpeq2(v0, inf2) & one2, __vcmpeq2(v1, inf2) & one2);
              pa_mma<T>(nm, sees[mt], __vcmpeq2(v0, inf2 | 0x80008000u) & one2,
                        __vcmpeq2(v1, inf2 | 0x80008000u) & one2);
              pa_mma<T>(nn, sees[mt], __vcmpgtu2(v0 & 0x7fff7fffu, inf2) & one2,
                        __vcmpgtu2(v1 & 0x7fff7fffu, inf2) & one2);
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                float &x = a[mt].o[2 * d2 + half][e];
                if (np[e] > 0.f) x += INFINITY;
                if (nm[e] > 0.f) x -= INFINITY;
                if (nn[e] > 0.f) x = NAN;
              }
            }
        }
      }
    }
    // (Not unrolled: a third of the body is this loop's, and the warps of an SM
    // run three bodies: trees of up to 33 rows over 448 tokens 39 us against 43.)
#pragma unroll 1
    for (int sl = 0; sl < 2; ++sl) {
      uint32_t vr[4][4];
#pragma unroll
      for (int d2 = 0; d2 < 4; ++d2) pa_ldsm_t<0>(vtile + sl * 2048 + (voff ^ (d2 * 32)), vr[d2]);
      if (special) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint32_t keep = pa_keep(sl * 16 + e * 8 + 2 * t4, left);
#pragma unroll
          for (int d2 = 0; d2 < 4; ++d2) {
            vr[d2][e] &= keep;
            vr[d2][2 + e] &= keep;
          }
        }
        if (__builtin_expect(odd, 0)) {
#pragma unroll
          for (int d2 = 0; d2 < 4; ++d2)
#pragma unroll
            for (int e = 0; e < 4; ++e) vr[d2][e] &= ~pa_not_finite<T>(vr[d2][e]);
        }
      }
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        // (of a tile of few rows the residuals are rows 8..15)
        uint32_t pa[4], pr[4];
#pragma unroll
        for (int n2 = 0; n2 < 2; ++n2) {
          const float *x = sc[mt][n2];
          const float e0 = ex2(fmaf(x[0], p.scale_log2, -mu[mt][0]));
          const float e1 = ex2(fmaf(x[1], p.scale_log2, -mu[mt][0]));
          a[mt].l[0] += e0 + e1;
          pa[2 * n2] = pack2<T>(e0, e1);
          if (PaType<T>::kResidual || few) {
            const float2 r = unpack2<T>(pa[2 * n2]);
            pr[2 * n2] = pack2<T>(e0 - r.x, e1 - r.y);
          }
          if (few) {
            pa[2 * n2 + 1] = pr[2 * n2];
          } else {
            const float f0 = ex2(fmaf(x[2], p.scale_log2, -mu[mt][1]));
            const float f1 = ex2(fmaf(x[3], p.scale_log2, -mu[mt][1]));
            a[mt].l[1] += f0 + f1;
            pa[2 * n2 + 1] = pack2<T>(f0, f1);
            if (PaType<T>::kResidual) {
              const float2 r = unpack2<T>(pa[2 * n2 + 1]);
              pr[2 * n2 + 1] = pack2<T>(f0 - r.x, f1 - r.y);
            }
          }
        }
        // (a loop: as a condition it becomes products that are predicated off)
#pragma unroll 1
        for (int rep = 0; rep < (PaType<T>::kResidual && !few && MT == 1 ? 2 : 1); ++rep) {
#pragma unroll
          for (int db = 0; db < 8; ++db)
            pa_mma<T>(a[mt].o[db], pa, vr[db >> 1][(db & 1) * 2], vr[db >> 1][(db & 1) * 2 + 1]);
          if (PaType<T>::kResidual) {
#pragma unroll
            for (int e = 0; e < 4; ++e) pa[e] = pr[e];
          }
        }
        if (PaType<T>::kResidual && MT == 2) {
#pragma unroll
          for (int db = 0; db < 8; ++db)
            pa_mma<T>(a[mt].o[db], pr, vr[db >> 1][(db & 1) * 2], vr[db >> 1][(db & 1) * 2 + 1]);
        }
      }
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int e = 0; e < 8; ++e) sc[mt][e >> 2][e & 3] = sc[mt][2 + (e >> 2)][e & 3];
    }
    __syncwarp();  // every lane has read the stage
    if (lane == 0) mbar_arrive(&s.empty[warp][slot]);
  }
  if (few) {
#pragma unroll
    for (int db = 0; db < 8; ++db) {
      a[0].o[db][0] += a[0].o[db][2];
      a[0].o[db][1] += a[0].o[db][3];
    }
  }
  const bool whole = it.from == 0 && it.to == it.stages;
  const bool starts = it.from == 0;
  if (!whole && lane == 0) s.cut[warp][starts ? 1 : 0] = it;
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    if (whole)
      pa_output<T, OutT>(p, a[mt], it.row0 + mt * 16, it.nr - mt * 16, it.head, lane);
    else
      pa_put(pa_part(p, blockIdx.x * kPaWarps + warp, starts, mt, lane), a[mt]);
  }
}

// ---------------------------------------------------------------- f32 pools
//
// The same walk with 16-key stages and tiles of 16 rows on tf32 products,
// three for each: every operand enters as x = hi + lo, 11 significant bits
// each, and hi hi + hi lo + lo hi leaves out 2^-21 of each product at most.
WATTN_DEVINL void pa_mma_tf32(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
constexpr uint32_t kTf32 = 0xffffe000u;  // sign, exponent, 10 bits
// x to its nearest such (finite x stay finite; FAR: x may be near the largest).
template <bool FAR> WATTN_DEVINL uint32_t pa_tf32(float x) {
  const uint32_t u = __float_as_uint(x);
  if (!FAR) return (u + 0x1000u) & kTf32;
  return (min((u & 0x7fffffffu) + 0x1000u, 0x7f7fffffu) & kTf32) | (u & 0x80000000u);
}
// Queries, keys and weights are split to nearest, so that lo has either sign
// and what is left out of the products does not add up; values, of any size
// where they are masked, cut off and their lo to nearest. (Cut off throughout,
// scores and outputs come out too small: 1.1e-6 of the output against 5e-7.)
template <bool FAR> WATTN_DEVINL void pa_split(float x, uint32_t &hi, uint32_t &lo) {
  hi = pa_tf32<FAR>(x);
  lo = __float_as_uint(x - __uint_as_float(hi)) & kTf32;
}
WATTN_DEVINL void pa_split_value(float x, uint32_t &hi, uint32_t &lo) {
  hi = __float_as_uint(x) & kTf32;
  lo = pa_tf32<false>(x - __uint_as_float(hi));
}
WATTN_DEVINL float4 pa_lds(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

// The order of dims in the products is free as long as both operands share
// it, and chosen so that every lane reads 16 bytes and no bank meets twice:
// K: step (blk, j, pair) takes dims 32 blk + 8 t4 + 4 j + 2 pair (+ 1);
// V: column g of tile (j, e) is dim 32 (g >> 2) + 4 ((g & 3) + 4 j) + e.
WATTN_DEVINL void pa_item_f32(const PagedAttendParams &p, PaSmem<float> &s, const PaItem &it, uint32_t &pos,
                              int warp, int lane) {
  constexpr int kKeys = PaType<float>::kKeys;
  const int g = lane >> 2, t4 = lane & 3;
  uint32_t qh[8][4], ql[8][4];
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int c = 0; c < 4; ++c) {  // c = 2 blk + j
      const int r = h * 8 + g;
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
      if (r < it.nr)
        x = *reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(p.q) +
                                              (int64_t)(it.row0 + r) * p.q_rs + it.head * 64 +
                                              (c >> 1) * 32 + 8 * t4 + (c & 1) * 4);
      pa_split<true>(x.x, qh[2 * c][h], ql[2 * c][h]);
      pa_split<true>(x.y, qh[2 * c][2 + h], ql[2 * c][2 + h]);
      pa_split<true>(x.z, qh[2 * c + 1][h], ql[2 * c + 1][h]);
      pa_split<true>(x.w, qh[2 * c + 1][2 + h], ql[2 * c + 1][2 + h]);
    }
  PaTile a;
#pragma unroll
  for (int db = 0; db < 8; ++db) a.o[db][0] = a.o[db][1] = a.o[db][2] = a.o[db][3] = 0.f;
  a.m[0] = a.m[1] = -INFINITY;
  a.l[0] = a.l[1] = 0.f;
#pragma unroll 1
  for (int t = it.from; t < it.to; ++t) {
    const int slot = pos & 3;
    mbar_wait(&s.full[warp][slot], pos >> 31, &s.abort, p.status,
              (4 << 24) | (1 << 16) | ((t & 0xff) << 8));
    pos = slot == kPaStages - 1 ? (pos & 0x80000000u) ^ 0x80000000u : pos + 1;
    const uint32_t ktile = smem_u32(s.kv[warp][slot]), vtile = ktile + kKeys * 128;
    float sc[2][4], sx[2][4], sy[2][4];  // hi hi, hi lo, lo hi
#pragma unroll
    for (int nb = 0; nb < 2; ++nb)
#pragma unroll
      for (int e = 0; e < 4; ++e) sc[nb][e] = sx[nb][e] = sy[nb][e] = 0.f;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      float4 x[2];
#pragma unroll
      for (int nb = 0; nb < 2; ++nb)
        x[nb] = pa_lds(ktile + (c >> 1) * (kPaStageBytes / 2) + (nb * 8 + g) * 128 +
                       (((2 * t4 + (c & 1)) ^ g) << 4));
#pragma unroll
      for (int pair = 0; pair < 2; ++pair)
#pragma unroll
        for (int nb = 0; nb < 2; ++nb) {
          uint32_t h0, l0, h1, l1;
          pa_split<true>(pair ? x[nb].z : x[nb].x, h0, l0);
          pa_split<true>(pair ? x[nb].w : x[nb].y, h1, l1);
          pa_mma_tf32(sc[nb], qh[2 * c + pair], h0, h1);
          pa_mma_tf32(sx[nb], qh[2 * c + pair], l0, l1);
          pa_mma_tf32(sy[nb], ql[2 * c + pair], h0, h1);
        }
    }
#pragma unroll
    for (int nb = 0; nb < 2; ++nb)
#pragma unroll
      for (int e = 0; e < 4; ++e) sc[nb][e] += sx[nb][e] + sy[nb][e];
    const int off = t * kKeys - it.len, left = it.end - t * kKeys;
    const bool drafts = off + kKeys > 0;  // the stage reaches past the cached positions
    const bool special = drafts || left < kKeys;
    if (special) {
      const uint32_t sees =
          lane < it.nr ? pa_visible(p, it.row0 + lane, it.row + lane, off, left) : 0u;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t vis = __shfl_sync(0xffffffffu, sees, h * 8 + g) >> (2 * t4);
#pragma unroll
        for (int nb = 0; nb < 2; ++nb)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            if (!(vis >> (nb * 8 + e) & 1u)) sc[nb][2 * h + e] = -INFINITY;
      }
    }
    float mu[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float mx = fmax3(fmaxf(sc[0][2 * h], sc[0][2 * h + 1]), sc[1][2 * h], sc[1][2 * h + 1]);
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const float mc = mx * p.scale_log2;
      if (mc > a.m[h] + 8.0f) {
        const float alpha = ex2(a.m[h] - mc);
        a.l[h] *= alpha;
#pragma unroll
        for (int db = 0; db < 8; ++db) {
          a.o[db][2 * h] *= alpha;
          a.o[db][2 * h + 1] *= alpha;
        }
        a.m[h] = mc;
      }
      mu[h] = a.m[h] == -INFINITY ? 0.f : a.m[h];
    }
    // The stage's own sums: the tensor cores cut off what they add up, which
    // makes the outputs too small (one request of 32768 tokens: by 1.0e-6 of
    // their size, with sums of their own 4.2e-7).
    float o[8][4];
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
#pragma unroll
    for (int nb = 0; nb < 2; ++nb) {
      // two value rows, of keys 2 t4 and 2 t4 + 1, in column g of the 8 tiles
      float v[2][8];
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const int key = nb * 8 + 2 * t4 + b;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float4 x = pa_lds(vtile + (g >> 2) * (kPaStageBytes / 2) + key * 128 +
                                  ((((g & 3) + 4 * j) ^ (2 * t4 + b)) << 4));
          v[b][4 * j] = x.x;
          v[b][4 * j + 1] = x.y;
          v[b][4 * j + 2] = x.z;
          v[b][4 * j + 3] = x.w;
        }
        if (special && key >= left)  // behind the last position: anything
#pragma unroll
          for (int i = 0; i < 8; ++i) v[b][i] = 0.f;
      }
      if (drafts) {  // a draft's value that is not finite: only for the rows that see it
        float nil = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) nil = fmaf(v[0][i], 0.f, fmaf(v[1][i], 0.f, nil));
        if (__any_sync(0xffffffffu, nil != nil)) {
          const uint32_t one = __float_as_uint(1.f);
          uint32_t see[4];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            see[e] = sc[nb][2 * (e & 1) + (e >> 1)] != -INFINITY ? one : 0u;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            float np[4] = {0, 0, 0, 0}, nm[4] = {0, 0, 0, 0}, nn[4] = {0, 0, 0, 0};
            const float x = v[0][i], y = v[1][i];
            pa_mma_tf32(np, see, x == INFINITY ? one : 0u, y == INFINITY ? one : 0u);
            pa_mma_tf32(nm, see, x == -INFINITY ? one : 0u, y == -INFINITY ? one : 0u);
            pa_mma_tf32(nn, see, x != x ? one : 0u, y != y ? one : 0u);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              if (np[e] > 0.f) a.o[i][e] += INFINITY;
              if (nm[e] > 0.f) a.o[i][e] -= INFINITY;
              if (nn[e] > 0.f) a.o[i][e] = NAN;
            }
            if (!(fabsf(x) < INFINITY)) v[0][i] = 0.f;
            if (!(fabsf(y) < INFINITY)) v[1][i] = 0.f;
          }
        }
      }
      uint32_t ph[4], pl[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {  // row g + 8 (e & 1), key 2 t4 + (e >> 1)
        const float w = ex2(fmaf(sc[nb][2 * (e & 1) + (e >> 1)], p.scale_log2, -mu[e & 1]));
        a.l[e & 1] += w;
        pa_split<false>(w, ph[e], pl[e]);
      }
      uint32_t vh[2][8], vl[2][8];
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int i = 0; i < 8; ++i) pa_split_value(v[b][i], vh[b][i], vl[b][i]);
#pragma unroll
      for (int i = 0; i < 8; ++i) pa_mma_tf32(o[i], ph, vh[0][i], vh[1][i]);
#pragma unroll
      for (int i = 0; i < 8; ++i) pa_mma_tf32(o[i], ph, vl[0][i], vl[1][i]);
#pragma unroll
      for (int i = 0; i < 8; ++i) pa_mma_tf32(o[i], pl, vh[0][i], vh[1][i]);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) a.o[i][e] += o[i][e];
    __syncwarp();  // every lane has read the stage
    if (lane == 0) mbar_arrive(&s.empty[warp][slot]);
  }
  const bool starts = it.from == 0;
  if (starts && it.to == it.stages) {
    pa_output<float, float>(p, a, it.row0, it.nr, it.head, lane);
  } else {
    if (lane == 0) s.cut[warp][starts ? 1 : 0] = it;
    pa_put(pa_part(p, blockIdx.x * kPaWarps + warp, starts, 0, lane), a);
  }
}

// ---------------------------------------------------------------- kernel

// Barrier of the compute warps (the load warps have left by then).
WATTN_DEVINL void pa_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }

// Adds partials c0, c0 + step, ... up to c1 of a cut item, in order (`starts`:
// c0's is the one that starts it).
WATTN_DEVINL void pa_gather(const PagedAttendParams &p, PaTile &a, int c0, int c1, int step, bool starts,
                            int mt, int lane) {
#pragma unroll
  for (int db = 0; db < 8; ++db) a.o[db][0] = a.o[db][1] = a.o[db][2] = a.o[db][3] = 0.f;
  a.m[0] = a.m[1] = -INFINITY;
  a.l[0] = a.l[1] = 0.f;
#pragma unroll 2
  for (int c = c0; c <= c1; c += step) pa_add(a, pa_part(p, c, starts && c == c0, mt, lane));
}

// The items cut by the shares of this CTA's warps, after all of them are
// done: the CTA's parts of an item are merged, an item per warp, and where
// several CTAs have parts the last of them to arrive merges theirs. (A few
// by the same warp: with all warps trees of 33 rows over 448 tokens take 7 %
// longer; many with all: 81,000 cycles to 68,000 for one request of
// 32768 tokens, whose heads lie in 37 CTAs each.)
template <typename T, typename OutT>
WATTN_DEVINL void pa_finish(const PagedAttendParams &p, PaSmem<T> &s, int warp, int lane) {
  const int tid = threadIdx.x, cta0 = blockIdx.x * kPaWarps, ctas = gridDim.x * kPaWarps;
  pa_sync();
  if (tid < 2 * kPaWarps) {
    const PaItem &it = s.cut[tid >> 1][tid & 1];
    int w0 = 0, w1 = -1;
    bool fresh = it.stages > 0;  // (the same item may be listed by several warps)
    for (int i = 0; i < tid; ++i)
      if (s.cut[i >> 1][i & 1].stages > 0 && s.cut[i >> 1][i & 1].at == it.at) fresh = false;
    if (fresh) {
      w0 = pa_owner(s.find.shares, it.at);
      w1 = pa_owner(s.find.shares, it.at + (it.stages - 1) * it.weight);
    }
    s.merge_first[tid] = w0;
    s.merge_last[tid] = w1;
    s.final[tid] = 0;
  }
  pa_sync();
  int turn = 0;
  bool far = false;  // an item here lies in many CTAs
#pragma unroll 1
  for (int e = 0; e < 2 * kPaWarps; ++e) {
    const int w0 = s.merge_first[e], w1 = s.merge_last[e];
    far |= w1 / kPaWarps - w0 / kPaWarps >= kPaMergeAll;
    if (w1 < w0 || (turn++ & (kPaWarps - 1)) != warp) continue;
    const PaItem &it = s.cut[e >> 1][e & 1];
    const int first = max(w0, cta0), last = min(w1, cta0 + kPaWarps - 1);
    const bool alone = first == w0 && last == w1;
    const int tiles = it.nr > 16 ? 2 : 1;
#pragma unroll 1
    for (int mt = 0; mt < tiles; ++mt) {
      PaTile a;
      pa_gather(p, a, first, last, 1, first == w0, mt, lane);
      if (alone) pa_output<T, OutT>(p, a, it.row0 + mt * 16, it.nr - mt * 16, it.head, lane);
      else pa_put(pa_part(p, ctas + blockIdx.x, first == w0, mt, lane), a);
    }
    if (alone) continue;
    // Release: the warp's sync orders its lanes' partials before lane 0's
    // fence, and the fence orders them before the count.
    const int c0 = w0 / kPaWarps, c1 = w1 / kPaWarps;
    int mine = 0;
    __syncwarp();
    if (lane == 0) {
      __threadfence();
      mine = atomicAdd(&p.count[c0], 1) == c1 - c0;
      if (mine) {
        __threadfence();
        p.count[c0] = 0;  // zeroed for the next call
      }
    }
    if (!__shfl_sync(0xffffffffu, mine, 0)) continue;
    if (c1 - c0 >= kPaMergeAll) {
      if (lane == 0) s.final[e] = 1;
      continue;
    }
#pragma unroll 1
    for (int mt = 0; mt < tiles; ++mt) {
      PaTile a;
      pa_gather(p, a, ctas + c0, ctas + c1, 1, true, mt, lane);
      pa_output<T, OutT>(p, a, it.row0 + mt * 16, it.nr - mt * 16, it.head, lane);
    }
  }
  if (!far) return;  // (the same for all warps)
  pa_sync();
#pragma unroll 1
  for (int e = 0; e < 2 * kPaWarps; ++e) {
    if (s.final[e] == 0) continue;
    const PaItem &it = s.cut[e >> 1][e & 1];
    const int c0 = s.merge_first[e] / kPaWarps, c1 = s.merge_last[e] / kPaWarps;
    const int tiles = it.nr > 16 ? 2 : 1;
#pragma unroll 1
    for (int mt = 0; mt < tiles; ++mt) {
      // each warp every fourth CTA's, then the first warp the four sums (in
      // the ring, where no loads are under way any more)
      PaTile a;
      pa_gather(p, a, ctas + c0 + warp, ctas + c1, kPaWarps, warp == 0, mt, lane);
      float4 *sums = reinterpret_cast<float4 *>(s.kv[0][0]) + lane;
      if (warp > 0) pa_put(sums + warp * (kPaTileFloats / 4), a);
      pa_sync();
      if (warp == 0) {
        for (int w = 1; w < kPaWarps; ++w) pa_add<false>(a, sums + w * (kPaTileFloats / 4));
        pa_output<T, OutT>(p, a, it.row0 + mt * 16, it.nr - mt * 16, it.head, lane);
      }
      pa_sync();
    }
  }
}

// `map` has boxes of a stage's keys and values (used where pages hold whole
// stages), `map_tail` boxes of 16 rows of either.
template <typename T, typename OutT, bool QUEUE>
__global__ void __launch_bounds__(kPaThreads, kPaCtasPerSm)
    paged_attend_stream_kernel(const __grid_constant__ CUtensorMap map,
                               const __grid_constant__ CUtensorMap map_tail,
                               const PagedAttendParams p) {
  extern __shared__ uint8_t pa_smem_raw[];
  PaSmem<T> &s = *reinterpret_cast<PaSmem<T> *>(
      (reinterpret_cast<uintptr_t>(pa_smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (lane == 0 && warp < kPaWarps) {
    for (int st = 0; st < kPaStages; ++st) {
      mbar_init(&s.full[warp][st], 1);
      mbar_init(&s.empty[warp][st], 1);
    }
    s.cut[warp][0].stages = s.cut[warp][1].stages = 0;
    s.abort = 0;
    fence_barrier_init();
  }
  if (threadIdx.x == kPaWarps * 32) {
    tma_prefetch_desc(&map);
    tma_prefetch_desc(&map_tail);
  }
  grid_dep_wait();  // (launched with programmatic serialisation)
  grid_dep_launch();
  if constexpr (__is_same(T, __half))
    if (p.choose && pa_takes_wide(p, s.choice)) return;
  pa_find_shares<PaType<T>, QUEUE>(p, s.find);
  if (warp >= kPaWarps) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPaLoadRegs));
    pa_load<T, QUEUE>(p, s, map, map_tail, warp - kPaWarps, lane);
    return;
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kPaComputeRegs));
    uint32_t pos = 0;  // ring slot of the next stage, and in bit 31 its barrier's phase
#pragma unroll 1
    for (uint32_t i = 0;; ++i) {
      // The next stage's barrier covers the announcement of its item. A wait
      // may run out for some lanes only, and all of them stay or leave: they
      // vote, or such a lane ends the share for the others. (Which of the two
      // costs no registers: by vote, trees of 64 rows over 32768 tokens take
      // 5 % longer, by mark 320 single rows of f16 2 %.)
      uint64_t *const full = &s.full[warp][pos & 3];
      if constexpr (QUEUE) {
        if (!__all_sync(0xffffffffu, mbar_wait(full, pos >> 31, &s.abort, p.status, (4 << 24) | (2 << 16))))
          break;
      } else {
        if (!mbar_wait(full, pos >> 31, &s.abort, p.status, (4 << 24) | (2 << 16)))
          s.queue[warp][i % kPaQueue].nr = 0;
        __syncwarp();
      }
      const PaItem it = s.queue[warp][i % kPaQueue];
      if (it.nr == 0) break;
      if constexpr (sizeof(T) == 4) pa_item_f32(p, s, it, pos, warp, lane);
      else if (it.nr <= 16) pa_item<T, OutT, 1>(p, s, it, pos, warp, lane);
      else pa_item<T, OutT, 2>(p, s, it, pos, warp, lane);
    }
    __syncwarp();
    pa_finish<T, OutT>(p, s, warp, lane);
  }
}

// SMs of the current device.
int pa_sms() {
  static int sms[64] = {0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
  if (sms[dev] == 0) cudaDeviceGetAttribute(&sms[dev], cudaDevAttrMultiProcessorCount, dev);
  return sms[dev];
}

// Workspace of either kernel.
size_t pa_workspace(int n_sm) {
  const size_t narrow = kCounterBytes + (size_t)n_sm * kPaCtasPerSm * (kPaWarps + 1) * 4 * kPaTileFloats *
                                            sizeof(float);
  return std::max(narrow, paged_attend_wide_workspace(n_sm));
}

template <typename T, typename OutT, bool QUEUE>
int launch_stream_as(PagedAttendParams p, int dtype, cudaStream_t st) {
  // The pool as [page, layer][K|V][head, row][64]: one box holds a stage's
  // keys and its values; the tail map's boxes hold 16 rows of either.
  // f32: boxes of half the dims of a stage's 16 keys and values.
  const uint64_t kv_rows = (uint64_t)p.n_heads * p.page_rows, es = sizeof(T);
  p.box_rows = p.page_rows % PaType<T>::kKeys == 0 ? PaType<T>::kKeys : kPaTail;
  const uint64_t dims[4] = {64, kv_rows, 2, (uint64_t)p.n_pages * p.n_layers};
  const uint64_t strides[3] = {64 * es, kv_rows * 64 * es, kv_rows * 128 * es};
  const uint32_t width = 128 / sizeof(T);
  const uint32_t box[4] = {width, PaType<T>::kKeys, 2, 1}, box_tail[4] = {width, kPaTail, 1, 1};
  CUtensorMap map, map_tail;
  int rc = encode_tmap(&map_tail, tmap_dtype(dtype), 4, p.pool, dims, strides, box_tail,
                       CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc == WATTN_OK && p.box_rows == PaType<T>::kKeys)
    rc = encode_tmap(&map, tmap_dtype(dtype), 4, p.pool, dims, strides, box,
                     CU_TENSOR_MAP_SWIZZLE_128B);
  else
    map = map_tail;  // not used
  if (rc != WATTN_OK) return rc;
  constexpr int smem = (int)sizeof(PaSmem<T>) + 1024;
  auto kern = paged_attend_stream_kernel<T, OutT, QUEUE>;
  // Once per process and type: the warpgroups' register split counts on what
  // the kernel is launched with (with fewer it would wait for ever).
  static const int regs = [&] {
    cudaFuncAttributes a;
    return cudaFuncGetAttributes(&a, kern) == cudaSuccess ? a.numRegs : 0;
  }();
  if (regs != kPaRegs)
    return set_error(WATTN_ERR_CUDA, "paged_attend: built for %d registers a thread, not %d", kPaRegs, regs);
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
    return check_launch("cudaFuncSetAttribute(paged_attend)");
  launch_pdl(kern, dim3(p.n_sm * kPaCtasPerSm), dim3(kPaThreads), smem, st, map, map_tail, p);
  return check_launch("paged_attend");
}

template <typename T, typename OutT>
int launch_stream(const PagedAttendParams &p, int dtype, cudaStream_t st) {
  // (No more items than this.)
  const int64_t items = ((int64_t)p.max_rows / PaType<T>::kRows + p.n_seqs) * p.n_heads;
  const bool queue = items >= (int64_t)PaShape::kQueueItems * p.n_sm * kPaCtasPerSm * kPaWarps;
  return queue ? launch_stream_as<T, OutT, true>(p, dtype, st) : launch_stream_as<T, OutT, false>(p, dtype, st);
}

int launch_attend(const PagedAttendParams &p, int dtype, int out_dtype, cudaStream_t st) {
  if (dtype == WATTN_F32) return launch_stream<float, float>(p, dtype, st);
  if (dtype == WATTN_F16) {
    // The narrow kernel, or both, of which the one that is not for the step
    // leaves at once: 4 to 7 us. (320 single rows of 20 heads over up to 1000
    // tokens, in buffers for 128 rows each: 133 us, in buffers of their own 127;
    // in the wide kernel they would take 552.)
    PagedAttendParams q = p;
    q.choose = pa_may_be_wide(p);
    const int rc = out_dtype == WATTN_F32 ? launch_stream<__half, float>(q, dtype, st)
                                          : launch_stream<__half, __half>(q, dtype, st);
    return rc == WATTN_OK && q.choose ? launch_paged_attend_wide(q, out_dtype, st) : rc;
  }
  return out_dtype == WATTN_F32 ? launch_stream<__nv_bfloat16, float>(p, dtype, st)
                                : launch_stream<__nv_bfloat16, __nv_bfloat16>(p, dtype, st);
}

}  // namespace
}  // namespace wattn

using namespace wattn;

extern "C" {

size_t wattn_paged_attend_workspace_bytes(int n_seqs, int max_rows, int n_heads) {
  if (n_seqs <= 0 || max_rows <= 0 || n_heads <= 0) return 0;
  return pa_workspace(pa_sms());
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
  const float scale_log2 = scale * 1.4426950408889634f;  // (in the kernels' base: may be infinite where scale is not)
  if (!(scale > 0.f) || !(scale_log2 < INFINITY))
    return set_error(WATTN_ERR_INVALID, "paged_attend: scale must be positive and below 2.3e38");
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
  p.mask_bits = (int)std::min((int64_t)mask_words * 32, (int64_t)INT32_MAX);
  p.q = q;
  p.o = o;
  p.q_rs = q_row_stride;
  p.o_rs = o_row_stride;
  p.max_rows = max_rows;
  p.scale_log2 = scale_log2;
  // (positions rounded up to a stage of either kernel stay within 32 bits)
  p.cap = (int)std::min((int64_t)max_pages * page_rows, (int64_t)INT32_MAX - 2 * kPaMostKeys);
  p.status = device_status_ptr();
  if (p.status == nullptr) return WATTN_ERR_CUDA;
  cudaStream_t st = (cudaStream_t)stream;
  p.n_sm = pa_sms();
  const size_t need = pa_workspace(p.n_sm);
  void *own = nullptr;
  if (workspace == nullptr) {
    // A captured call gets a workspace of its graph's: the thread's may be in
    // use by another graph or call when this one is replayed, or be replaced.
    cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
    if (cudaStreamIsCapturing(st, &capture) != cudaSuccess) cudaGetLastError();
    if (capture == cudaStreamCaptureStatusActive) {
      if (cudaMallocAsync(&own, need, st) != cudaSuccess)
        return check_launch("paged_attend: a captured call's workspace");
      if (cudaMemsetAsync(own, 0, kCounterBytes, st) != cudaSuccess) {
        rc = check_launch("paged_attend: a captured call's workspace");
        cudaFreeAsync(own, st);
        return rc;
      }
      workspace = own;
    } else {
      workspace = thread_workspace(need, st);
    }
    if (workspace == nullptr) return set_error(WATTN_ERR_NOMEM, "paged_attend: workspace allocation failed");
  } else if (workspace_bytes < need) {
    return set_error(WATTN_ERR_INVALID, "paged_attend: workspace of %zu bytes, %zu needed",
                     workspace_bytes, need);
  } else if (reinterpret_cast<uintptr_t>(workspace) & 15) {
    return set_error(WATTN_ERR_INVALID, "paged_attend: the workspace must be 16-byte aligned");
  }
  p.count = reinterpret_cast<int *>(workspace);
  p.taken = p.count + kMaxSplitCounters - 1;
  p.part = reinterpret_cast<float *>(reinterpret_cast<uint8_t *>(workspace) + kCounterBytes);
  rc = launch_attend(p, dtype, out_dtype, st);
  if (own != nullptr && cudaFreeAsync(own, st) != cudaSuccess && rc == WATTN_OK)
    rc = check_launch("paged_attend: a captured call's workspace");
  return rc;
}

}  // extern "C"
