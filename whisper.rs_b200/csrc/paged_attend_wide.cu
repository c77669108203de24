// paged_attend_wide.cu -- attention of many new rows a request over a
// device-planned paged cache, on the tcgen05 tensor cores (f16 pools).
//
// The narrow kernel (paged_attend.cu) multiplies tiles of up to 32 rows with
// mma.sync and reads a request's keys once for each; here one tile takes 128
// rows, so that wide trees and the chunks of a long prompt read them once.
//
// One CTA per share, two CTAs on an SM (256 TMEM columns each): four softmax
// warps with a query row per thread, and a warpgroup that leaves them its
// registers, of which one warp loads (TMA through the block table, rings of
// two 128-key K tiles and three V tiles) and one issues the products. S = Q
// K^T lands in TMEM, the softmax writes the weights (f16: 2^-11 each, within
// the 2e-3 bar; small ones: kPaLower16) back to TMEM as the A operand of O += P
// V, and S of the next tile runs under the softmax of this one.
//
// bf16 pools stay with the narrow kernel: bf16 weights (2^-8 each) need their
// residuals in the product, here as a second set of 64 rows of the tile, and
// then it was no faster (64 rows 78 us against 81, 256 rows 232 against 227).
//
// Bound: the chain of one tile, about 4500 cycles a CTA (S 460 to wait for,
// scores and maximum 900, weights 1900 with the SFU shared by two CTAs, the
// last product 590, stores 670), not HBM (1424 a tile and SM).

#include <algorithm>

#include "paged_attend.cuh"

namespace wattn {

namespace {

constexpr int kPwKeys = PwShape::kKeys;  // keys of a stage
constexpr int kPwTile = kPwKeys * 128;
constexpr int kPwK = 2, kPwV = 3;  // ring depths
constexpr int kPwThreads = PwShape::kThreads;
constexpr int kPwLoadWarp = 4, kPwMmaWarp = 5;
// Registers per thread: at the launch, then after the warpgroups' split
// (whose sum may not exceed twice the launch's).
constexpr int kPwRegs = 128, kPwSoftmaxRegs = 216, kPwOtherRegs = 40;
static_assert(kPwSoftmaxRegs + kPwOtherRegs <= 2 * kPwRegs, "a larger split never gets its registers");
constexpr int kPwCtasPerSm = 2;
constexpr int kPwQueue = 2;        // items announced
// One pair of exponentials in so many runs on the FMA pipe instead of the SFU
// (7.5e-5 off at most, less than the weights' rounding to f16). The polynomial
// does not give NaN for NaN, nor 0 for -inf but 2^-126: rows with such scores
// are caught by their maximum, and 2^-126 is 0 in f16 and nothing in a sum that
// has a key.
constexpr int kPwFmaPairs = 4;
constexpr uint32_t kPwCols = 256;  // TMEM: S 128, P 64, O 64
constexpr int kPwPartFloats = 66 * 128;  // a partial: O [64][row], m, l

struct PwSmem {
  uint8_t q[kPwTile];
  uint8_t k[kPwK][kPwTile];
  uint8_t v[kPwV][kPwTile];
  uint64_t q_full, k_full[kPwK], k_empty[kPwK], v_full[kPwV], v_empty[kPwV];
  uint64_t s_full, s_free, p_full, o_done;
  uint64_t item_full[kPwQueue], item_empty[kPwQueue];
  uint64_t drain, done, meet;
  PaItem queue[kPwQueue];
  PaFind<PwShape> find;
  PaChoice choice;
  uint32_t odd[4];  // keys of a tile with values that are infinite or NaN
  uint32_t tmem;
  int abort, last;
};

#define PW_SITE(role, what) ((5 << 24) | ((role) << 16) | ((what) << 8))

// Barrier of the softmax warps, `count` (of such barriers so far) being the
// same in all of them. Bounded like all waits (a warp that gave up elsewhere
// does not come): false if it ran out.
WATTN_DEVINL bool pw_sync(const PagedAttendParams &p, PwSmem &s, uint32_t &count) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(&s.meet);
  return __all_sync(0xffffffffu, mbar_wait(&s.meet, count++ & 1, &s.abort, p.status, PW_SITE(2, 5)));
}

// ---------------------------------------------------------------- load warp

// Winding down after a wait that ran out: the copies in flight (of n_k and
// n_v tiles issued) land before the block leaves.
WATTN_DEVINL void pw_drain(const PagedAttendParams &p, PwSmem &s, uint32_t n_k, uint32_t n_v) {
  volatile int no_abort = 0;
  for (uint32_t c = n_k > kPwK ? n_k - kPwK : 0; c < n_k; ++c)
    mbar_wait(&s.k_full[c % kPwK], (c / kPwK) & 1, &no_abort, p.status, PW_SITE(0, 5));
  for (uint32_t c = n_v > kPwV ? n_v - kPwV : 0; c < n_v; ++c)
    mbar_wait(&s.v_full[c % kPwV], (c / kPwV) & 1, &no_abort, p.status, PW_SITE(0, 6));
}

WATTN_DEVINL void pw_load(const PagedAttendParams &p, PwSmem &s, const CUtensorMap &map,
                          const CUtensorMap &map_tail, int lane) {
  using C = PwShape;
  PaLoads ld;
  ld.w = pa_start<C>(p, s.find, 0);
  PaStart &w = ld.w;
  uint32_t n = 0, items = 0;  // stages and items so far
  bool fresh = false, moved = false;
  const bool some = w.lo < w.hi;
  if (some) fresh = pa_enter<C>(p, ld);
#pragma unroll 1
  for (;;) {
    const bool more = some && pa_advance<C>(p, ld, fresh, moved);
    if (fresh || !more) {
      const int slot = items % kPwQueue;
      if (!__all_sync(0xffffffffu, mbar_wait(&s.item_empty[slot], ((items / kPwQueue) & 1) ^ 1, &s.abort,
                                             p.status, PW_SITE(0, 0)))) {
        pw_drain(p, s, n, n);
        return;
      }
      PaItem it = pa_item_of<C>(ld);
      if (!more) it.nr = 0;  // the end
      if (lane == 0) {
        s.queue[slot] = it;
        mbar_arrive(&s.item_full[slot]);
      }
      for (int r = lane; r < it.nr; r += 32)  // its query rows will be wanted soon
        asm volatile("prefetch.global.L1 [%0];" ::"l"(reinterpret_cast<const __half *>(p.q) +
                                                      (int64_t)(it.row0 + r) * p.q_rs + it.head * 64));
      ++items;
      fresh = false;
      if (!more) return;
    }
    // Boxes of p.box_rows rows, or of 16 where the positions end; a lane each.
    const int rows = min(kPwKeys, ld.end - ld.t * kPwKeys);
    const int step = rows < kPwKeys ? kPaTail : p.box_rows;
    const int boxes = (rows + step - 1) / step;
    const CUtensorMap *m = rows < kPwKeys ? &map_tail : &map;
    int c1 = 0, c3 = 0;
    if (lane < boxes) {
      const int at = ld.t * kPwKeys + lane * step, pi = at / p.page_rows;
      int page = p.table[w.s * p.table_stride + pi];
      if ((unsigned)page >= (unsigned)p.n_pages) {
        report_range(p.status, PW_SITE(0, 1));
        page = 0;
      }
      c1 = w.head * p.page_rows + at - pi * p.page_rows;
      c3 = page * p.n_layers + p.layer;
    }
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      const int depth = kv ? kPwV : kPwK, slot = n % depth;
      uint64_t *full = kv ? &s.v_full[slot] : &s.k_full[slot];
      uint64_t *empty = kv ? &s.v_empty[slot] : &s.k_empty[slot];
      uint8_t *dst = kv ? s.v[slot] : s.k[slot];
      if (!__all_sync(0xffffffffu,
                      mbar_wait(empty, ((n / depth) & 1) ^ 1, &s.abort, p.status, PW_SITE(0, 2 + kv)))) {
        pw_drain(p, s, n + kv, n);
        return;
      }
      if (lane == 0) mbar_arrive_expect_tx(full, boxes * step * 128);
      __syncwarp();
      if (lane < boxes) {
        // (softmax threads may have written value rows of the tile that was here)
        if (kv) fence_proxy_async_smem();
        tma_load_4d(dst + lane * step * 128, m, full, 0, c1, kv, c3);
      }
      __syncwarp();
    }
    ++ld.t;
    ++n;
  }
}

// ---------------------------------------------------------------- product warp

WATTN_DEVINL void pw_products(const PagedAttendParams &p, PwSmem &s, uint32_t tmem) {
  constexpr uint32_t idesc_s = idesc_f16(0, 128, kPwKeys, 0, 0);  // Q and K K-major
  constexpr uint32_t idesc_o = idesc_f16(0, 128, 64, 0, 1);       // P from TMEM, V MN-major
  const uint64_t dq = smem_desc_sw128(smem_u32(s.q), 16, 1024);
  const uint64_t dk0 = smem_desc_sw128(smem_u32(s.k[0]), 16, 1024);
  const uint64_t dv0 = smem_desc_sw128(smem_u32(s.v[0]), 16384, 1024);
  const uint32_t d_s = tmem, d_p = tmem + 128, d_o = tmem + 192;
  uint32_t n_s = 0, n_p = 0;  // S and PV issued
  auto s_step = [&]() -> bool {
    const int slot = n_s % kPwK;
    if (!mbar_wait(&s.k_full[slot], (n_s / kPwK) & 1, &s.abort, p.status, PW_SITE(1, 0))) return false;
    // It overwrites the last S: the softmax must have read that.
    if (n_s > 0 && !mbar_wait(&s.s_free, (n_s - 1) & 1, &s.abort, p.status, PW_SITE(1, 1))) return false;
    tc_fence_after();
    const uint64_t dk = dk0 + (uint32_t)slot * (kPwTile >> 4);
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) umma_ss(d_s, dq + 2 * kk, dk + 2 * kk, idesc_s, kk > 0);
    umma_commit(&s.s_full);
    umma_commit(&s.k_empty[slot]);
    ++n_s;
    return true;
  };
  for (uint32_t i = 0;; ++i) {
    const int islot = i % kPwQueue;
    if (!mbar_wait(&s.item_full[islot], (i / kPwQueue) & 1, &s.abort, p.status, PW_SITE(1, 2))) break;
    const int nr = s.queue[islot].nr, n = s.queue[islot].to - s.queue[islot].from;
    mbar_arrive(&s.item_empty[islot]);
    if (nr == 0) break;
    if (!mbar_wait(&s.q_full, i & 1, &s.abort, p.status, PW_SITE(1, 3)) || !s_step()) break;
    bool ok = true;
    for (int j = 0; j < n && ok; ++j) {
      if (j + 1 < n && !s_step()) { ok = false; break; }
      const int slot = n_p % kPwV;
      ok = mbar_wait(&s.p_full, n_p & 1, &s.abort, p.status, PW_SITE(1, 4)) &&
           mbar_wait(&s.v_full[slot], (n_p / kPwV) & 1, &s.abort, p.status, PW_SITE(1, 5));
      if (!ok) break;
      tc_fence_after();
      const uint64_t dv = dv0 + (uint32_t)slot * (kPwTile >> 4);
#pragma unroll
      for (int kk = 0; kk < 8; ++kk)  // (O starts as zeros, written by the softmax)
        umma_ts(d_o, d_p + kk * 8, dv + 128 * kk, idesc_o, 1);
      umma_commit(&s.o_done);
      umma_commit(&s.v_empty[slot]);
      ++n_p;
    }
    if (!ok) break;
  }
  // Every product has completed before the columns are freed (a wait that
  // outlives a wind-down, but bounded).
  volatile int no_abort = 0;
  umma_commit(&s.drain);
  mbar_wait(&s.drain, 0, &no_abort, p.status, PW_SITE(1, 6));
}

// ---------------------------------------------------------------- softmax warps

template <typename OutT>
WATTN_DEVINL void pw_store_row(const PagedAttendParams &p, const float (&o)[64], float inv, int row,
                               int head) {
  const int64_t at = (int64_t)row * p.o_rs + head * 64;
#pragma unroll
  for (int c = 0; c < 64; c += 16 / sizeof(OutT)) {
    if constexpr (sizeof(OutT) == 4) {
      *reinterpret_cast<float4 *>(reinterpret_cast<float *>(p.o) + at + c) =
          make_float4(o[c] * inv, o[c + 1] * inv, o[c + 2] * inv, o[c + 3] * inv);
    } else {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = pack2<OutT>(o[c + 2 * i] * inv, o[c + 2 * i + 1] * inv);
      *reinterpret_cast<uint4 *>(reinterpret_cast<OutT *>(p.o) + at + c) =
          make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
}

WATTN_DEVINL float *pw_part(const PagedAttendParams &p, int c, bool starts) {
  return p.part + ((int64_t)c * 2 + (starts ? 1 : 0)) * kPwPartFloats;
}

// max(a, b, c), NaN if one of them is.
WATTN_DEVINL float pw_max3(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// Which of 32 positions row r of the item's tile sees (pa_visible).
WATTN_DEVINL uint32_t pw_visible(const PagedAttendParams &p, const PaItem &it, int r, int off, int left) {
  return left > 0 ? pa_visible(p, it.row0 + r, it.row + r, off, left) : 0u;
}

template <typename OutT>
WATTN_DEVINL void pw_softmax(const PagedAttendParams &p, PwSmem &s, uint32_t tmem, int tid) {
  const int wq = tid >> 5, lane = tid & 31;
  const int r = tid;  // row of the tile
  const uint32_t t_s = tmem + (uint32_t(wq * 32) << 16), t_p = t_s + 128, t_o = t_s + 192;
  uint32_t n = 0;      // tiles so far
  uint32_t met = 0;    // barriers of the softmax warps
#pragma unroll 1
  for (uint32_t i = 0;; ++i) {
    const int islot = i % kPwQueue;
    if (!__all_sync(0xffffffffu, mbar_wait(&s.item_full[islot], (i / kPwQueue) & 1, &s.abort, p.status,
                                           PW_SITE(2, 0))))
      return;
    const PaItem it = s.queue[islot];
    __syncwarp();
    if (lane == 0) mbar_arrive(&s.item_empty[islot]);
    if (it.nr == 0) return;
    const bool mine = r < it.nr;           // this thread has a row
    const bool warp_has = wq * 32 < it.nr;  // (one of) its warp has
    // ---- the query row, 128-byte swizzled, zeros behind the last; O = 0
    {
      const uint4 *src = reinterpret_cast<const uint4 *>(
          reinterpret_cast<const __half *>(p.q) + (int64_t)(it.row0 + r) * p.q_rs + it.head * 64);
#pragma unroll
      for (int c = 0; c < 8; ++c)
        *reinterpret_cast<uint4 *>(s.q + tid * 128 + ((c ^ (tid & 7)) << 4)) =
            mine ? src[c] : make_uint4(0, 0, 0, 0);
      fence_proxy_async_smem();
      uint32_t z[32];
#pragma unroll
      for (int e = 0; e < 32; ++e) z[e] = 0;
      __syncwarp();
      tmem_st32(t_o, z);
      tmem_st32(t_o + 32, z);
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(&s.q_full);
    }
    float m = -INFINITY, l = 0.f;  // running max (less kPaLower16), sum of the weights
#pragma unroll 1
    for (int t = it.from; t < it.to; ++t, ++n) {
      if (!__all_sync(0xffffffffu, mbar_wait(&s.s_full, n & 1, &s.abort, p.status, PW_SITE(2, 1)))) return;
      tc_fence_after();
      const int off = t * kPwKeys - it.len, left = it.end - t * kPwKeys;
      const bool drafts = off + kPwKeys > 0;  // the tile reaches past the cached positions
      const bool special = drafts || left < kPwKeys;
      float alpha = 1.f;
      bool rescale = false;
      uint32_t pk[64];  // the weights, packed: the scores are dead before P and O are touched
      if (!warp_has) {
        mbar_arrive(&s.s_free);
      } else {
        uint32_t sv[4][32];
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4) tmem_ld32(t_s + q4 * 32, sv[q4]);
        tmem_wait_ld();
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4) reg_fence(sv[q4]);
        tc_fence_before();
        mbar_arrive(&s.s_free);
        if (special) {
#pragma unroll
          for (int q4 = 0; q4 < 4; ++q4) {
            const uint32_t sees = mine ? pw_visible(p, it, r, off + 32 * q4, left - 32 * q4) : 0u;
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (!(sees >> e & 1u)) sv[q4][e] = __float_as_uint(-INFINITY);
          }
        }
        auto x = [&](int e) { return __uint_as_float(sv[e >> 5][e & 31]); };
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int e = 0; e < 128; e += 8)
#pragma unroll
          for (int a = 0; a < 4; ++a) mx[a] = pw_max3(mx[a], x(e + 2 * a), x(e + 2 * a + 1));
        const float top = pw_max3(pw_max3(mx[0], mx[1], mx[2]), mx[3], -INFINITY);
        const float mc = fmaf(top, p.scale_log2, -kPaLower16);
        const bool need = mc > m + 8.0f;  // rescale only when the running max grows by more than 2^8
        rescale = __any_sync(0xffffffffu, need) && t > it.from;
        if (need) {
          alpha = ex2(m - mc);
          l *= alpha;
          m = mc;
        }
        // A score that is NaN or +inf makes the row NaN (the polynomial below
        // would take it for a small weight).
        if (!(mc < INFINITY)) l = __int_as_float(0x7fffffff);
        const float mu = m == -INFINITY ? 0.f : m;
        const float2 c2 = make_float2(p.scale_log2, p.scale_log2), nmu2 = make_float2(-mu, -mu);
        float2 acc[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
        for (int e = 0; e < 64; ++e) {
          const float2 y = __ffma2_rn(make_float2(x(2 * e), x(2 * e + 1)), c2, nmu2);
          float2 w;
          if (e % kPwFmaPairs == kPwFmaPairs - 1) {
            w = exp2_fma2(y);
          } else {
            w.x = ex2(y.x);
            w.y = ex2(y.y);
          }
          acc[e & 1] = __fadd2_rn(acc[e & 1], w);
          pk[e] = pack2<__half>(w.x, w.y);
        }
        l += (acc[0].x + acc[0].y) + (acc[1].x + acc[1].y);
      }
      // The last product has read P and added to O: both may be written.
      if (n > 0 && !__all_sync(0xffffffffu, mbar_wait(&s.o_done, (n - 1) & 1, &s.abort, p.status, PW_SITE(2, 2))))
        return;
      tc_fence_after();
      if (rescale) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t o[32];
          tmem_ld32(t_o + 32 * h, o);
          tmem_wait_ld();
          reg_fence(o);
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
          tmem_st32(t_o + 32 * h, o);
        }
        if (special) tmem_wait_st();  // (below, O may be read back)
      }
      if (special) {
        // Thread k has value row k of the tile: one behind the last position
        // holds anything and becomes zeros; one of a draft with values that
        // are infinite or NaN belongs to the rows that see it (they add
        // these values themselves) and would, as 0 times it, spoil the others.
        const int vslot = n % kPwV;
        if (!__all_sync(0xffffffffu, mbar_wait(&s.v_full[vslot], (n / kPwV) & 1, &s.abort, p.status,
                                               PW_SITE(2, 3))))
          return;
        uint8_t *tile = s.v[vslot], *vrow = tile + tid * 128;
        constexpr uint32_t kInf2 = 0x7c007c00u;
        bool odd = false;
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          uint4 *at = reinterpret_cast<uint4 *>(vrow + (c << 4));
          if (tid >= left) {
            *at = make_uint4(0, 0, 0, 0);
          } else if (drafts) {
            const uint4 w = *at;
            odd |= (__vcmpeq2(w.x & kInf2, kInf2) | __vcmpeq2(w.y & kInf2, kInf2) |
                    __vcmpeq2(w.z & kInf2, kInf2) | __vcmpeq2(w.w & kInf2, kInf2)) != 0;
          }
        }
        const uint32_t flags = __ballot_sync(0xffffffffu, odd);
        if (lane == 0) s.odd[wq] = flags;
        if (!pw_sync(p, s, met)) return;
        if ((s.odd[0] | s.odd[1] | s.odd[2] | s.odd[3]) != 0) {
          if (warp_has) {
#pragma unroll 1
            for (int h = 0; h < 2; ++h) {
              uint32_t o[32];
              tmem_ld32(t_o + 32 * h, o);
              tmem_wait_ld();
              reg_fence(o);
              if (mine)
#pragma unroll 1
                for (int k = 0; k < kPwKeys; ++k) {
                  if (!(s.odd[k >> 5] >> (k & 31) & 1u)) continue;
                  if (!(pw_visible(p, it, r, off + (k & ~31), left - (k & ~31)) >> (k & 31) & 1u)) continue;
#pragma unroll
                  for (int e = 0; e < 32; ++e) {
                    const int d = h * 32 + e;
                    const float v = to_f32(*reinterpret_cast<const __half *>(
                        tile + k * 128 + (((d >> 3) ^ (k & 7)) << 4) + (d & 7) * 2));
                    if (!(fabsf(v) < INFINITY)) o[e] = __float_as_uint(__uint_as_float(o[e]) + v);
                  }
                }
              __syncwarp();
              tmem_st32(t_o + 32 * h, o);
            }
          }
          if (!pw_sync(p, s, met)) return;  // all have read the values
          if (odd) {
            uint32_t *w = reinterpret_cast<uint32_t *>(vrow);
            for (int e = 0; e < 32; ++e) w[e] &= ~__vcmpeq2(w[e] & kInf2, kInf2);
          }
        }
        fence_proxy_async_smem();
        if (!pw_sync(p, s, met)) return;  // (s.odd is used again; and the tile is clean for the product)
      }
      if (warp_has) {
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4) {
          uint32_t w[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) w[e] = pk[q4 * 16 + e];
          tmem_st16(t_p + q4 * 16, w);
        }
      }
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(&s.p_full);
    }
    // ---- the item's rows
    if (!__all_sync(0xffffffffu, mbar_wait(&s.o_done, (n - 1) & 1, &s.abort, p.status, PW_SITE(2, 4)))) return;
    tc_fence_after();
    float o[64];
    if (warp_has) {
      uint32_t u[2][32];
      tmem_ld32(t_o, u[0]);
      tmem_ld32(t_o + 32, u[1]);
      tmem_wait_ld();
      reg_fence(u[0]);
      reg_fence(u[1]);
#pragma unroll
      for (int e = 0; e < 64; ++e) o[e] = __uint_as_float(u[e >> 5][e & 31]);
    }
    const bool starts = it.from == 0;
    if (starts && it.to == it.stages) {
      if (mine)
        pw_store_row<OutT>(p, o, l == 0.f ? 0.f : __fdividef(1.f, l), it.row0 + r, it.head);
      continue;
    }
    // A cut item: this share's part, merged by the last of its shares.
    const int c0 = pa_owner(s.find.shares, it.at);
    const int c1 = pa_owner(s.find.shares, it.at + (it.stages - 1) * it.weight);
    if (mine) {
      float *part = pw_part(p, blockIdx.x, starts) + r;
#pragma unroll
      for (int e = 0; e < 64; ++e) part[e * 128] = o[e];
      part[64 * 128] = m;
      part[65 * 128] = l;
    }
    if (!pw_sync(p, s, met)) return;
    if (tid == 0) {
      // Release: the barrier orders the threads' partials before this
      // fence, and the fence orders them before the count.
      __threadfence();
      s.last = atomicAdd(&p.count[c0], 1) == c1 - c0;
      if (s.last) {
        __threadfence();
        p.count[c0] = 0;  // zeroed for the next call
      }
    }
    if (!pw_sync(p, s, met)) return;
    if (s.last && mine) {
      float M = -INFINITY, L = 0.f;
#pragma unroll
      for (int e = 0; e < 64; ++e) o[e] = 0.f;
#pragma unroll 1
      for (int c = c0; c <= c1; ++c) {
        const float *part = pw_part(p, c, c == c0) + r;
        const float mb = __ldcg(part + 64 * 128), lb = __ldcg(part + 65 * 128);
        const float mn = fmaxf(M, mb);
        const float wa = M == -INFINITY ? 0.f : ex2(M - mn), wb = mb == -INFINITY ? 0.f : ex2(mb - mn);
        M = mn;
        L = fmaf(L, wa, wb * lb);
#pragma unroll
        for (int e = 0; e < 64; ++e) o[e] = fmaf(o[e], wa, wb * __ldcg(part + e * 128));
      }
      pw_store_row<OutT>(p, o, L == 0.f ? 0.f : __fdividef(1.f, L), it.row0 + r, it.head);
    }
    if (!pw_sync(p, s, met)) return;  // s.last is used again
  }
}

// ---------------------------------------------------------------- kernel

template <typename OutT>
__global__ void __launch_bounds__(kPwThreads, kPwCtasPerSm)
    paged_attend_wide_kernel(const __grid_constant__ CUtensorMap map,
                             const __grid_constant__ CUtensorMap map_tail, const PagedAttendParams p) {
  extern __shared__ uint8_t pw_smem_raw[];
  PwSmem &s = *reinterpret_cast<PwSmem *>(
      (reinterpret_cast<uintptr_t>(pw_smem_raw) + 1023) & ~uintptr_t(1023));
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    mbar_init(&s.q_full, 128);
    for (int i = 0; i < kPwK; ++i) {
      mbar_init(&s.k_full[i], 1);
      mbar_init(&s.k_empty[i], 1);
    }
    for (int i = 0; i < kPwV; ++i) {
      mbar_init(&s.v_full[i], 1);
      mbar_init(&s.v_empty[i], 1);
    }
    mbar_init(&s.s_full, 1);
    mbar_init(&s.s_free, 128);
    mbar_init(&s.p_full, 128);
    mbar_init(&s.o_done, 1);
    for (int i = 0; i < kPwQueue; ++i) {
      mbar_init(&s.item_full[i], 1);
      mbar_init(&s.item_empty[i], 5);  // the product warp and four softmax warps
    }
    mbar_init(&s.drain, 1);
    mbar_init(&s.done, 128);
    mbar_init(&s.meet, 4);
    s.abort = 0;
    fence_barrier_init();
  }
  if (tid == kPwLoadWarp * 32) {
    tma_prefetch_desc(&map);
    tma_prefetch_desc(&map_tail);
  }
  if (warp == kPwMmaWarp) {
    __syncwarp();
    tmem_alloc(&s.tmem, kPwCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  grid_dep_wait();  // (launched with programmatic serialisation)
  grid_dep_launch();
  const uint32_t tmem = s.tmem;
  if (!pa_takes_wide(p, s.choice)) {
    if (warp == kPwMmaWarp) tmem_dealloc(tmem, kPwCols);
    return;
  }
  pa_find_shares<PwShape>(p, s.find);
  if (warp >= 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPwOtherRegs));
    if (warp == kPwLoadWarp) pw_load(p, s, map, map_tail, lane);
    if (warp == kPwMmaWarp) {
      if (lane == 0) pw_products(p, s, tmem);
      __syncwarp();
      // the softmax warps are done with the columns (bounded, like all waits)
      volatile int no_abort = 0;
      mbar_wait(&s.done, 0, &no_abort, p.status, PW_SITE(1, 7));
      __syncwarp();
      tc_fence_after();
      tmem_dealloc(tmem, kPwCols);
    }
    return;
  }
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kPwSoftmaxRegs));
  pw_softmax<OutT>(p, s, tmem, tid);
  tc_fence_before();
  mbar_arrive(&s.done);
}

template <typename OutT>
int launch_wide(PagedAttendParams p, cudaStream_t st) {
  // The pool as [page, layer][K|V][head, row][64]; boxes of rows within a page.
  const uint64_t kv_rows = (uint64_t)p.n_heads * p.page_rows;
  p.box_rows = p.page_rows % 128 == 0 ? 128 : p.page_rows % 64 == 0 ? 64 : p.page_rows % 32 == 0 ? 32 : kPaTail;
  const uint64_t dims[4] = {64, kv_rows, 2, (uint64_t)p.n_pages * p.n_layers};
  const uint64_t strides[3] = {128, kv_rows * 128, kv_rows * 256};
  const uint32_t box[4] = {64, (uint32_t)p.box_rows, 1, 1}, box_tail[4] = {64, kPaTail, 1, 1};
  CUtensorMap map, map_tail;
  int rc = encode_tmap(&map, tmap_dtype(WATTN_F16), 4, p.pool, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc == WATTN_OK)
    rc = encode_tmap(&map_tail, tmap_dtype(WATTN_F16), 4, p.pool, dims, strides, box_tail,
                     CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc != WATTN_OK) return rc;
  constexpr int smem = (int)sizeof(PwSmem) + 1024;
  auto kern = paged_attend_wide_kernel<OutT>;
  // Once per process and type: the warpgroups' register split counts on what
  // the kernel is launched with (with fewer it would wait for ever).
  static const int regs = [&] {
    cudaFuncAttributes a;
    return cudaFuncGetAttributes(&a, kern) == cudaSuccess ? a.numRegs : 0;
  }();
  if (regs != kPwRegs)
    return set_error(WATTN_ERR_CUDA, "paged_attend: built for %d registers a thread, not %d", kPwRegs, regs);
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
    return check_launch("cudaFuncSetAttribute(paged_attend_wide)");
  launch_pdl(kern, dim3(p.n_sm * kPwCtasPerSm), dim3(kPwThreads), smem, st, map, map_tail, p);
  return check_launch("paged_attend_wide");
}

}  // namespace

int launch_paged_attend_wide(const PagedAttendParams &p, int out_dtype, cudaStream_t st) {
  return out_dtype == WATTN_F32 ? launch_wide<float>(p, st) : launch_wide<__half>(p, st);
}

size_t paged_attend_wide_workspace(int n_sm) {
  return kCounterBytes + (size_t)n_sm * kPwCtasPerSm * 2 * kPwPartFloats * sizeof(float);
}

}  // namespace wattn
