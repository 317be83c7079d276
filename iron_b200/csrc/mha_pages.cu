// Attention of one query a sequence (a decode step) over a key/value cache that lies in pages of
// e4m3 codes, on warp MMAs; and the C entries of this and of the ragged form (mha_pages_tc.cu).
//
// Bound by the cache's bytes, so the kernel is built around keeping them coming: every warp has
// a ring of its own in shared memory that TMA fills (16 tokens of one page and head a box, the
// rows swizzled so that the fragment reads below meet no bank conflict), and no other warp to
// wait for until its run of tokens ends.  Scores are computed transposed, S^T = K Q^T (16 tokens x
// 8 query columns an MMA), and so is the output, O^T += V^T P^T, so a group of up to eight query
// heads fills the MMA's narrow side and the codes its wide one:
//   K fragment   lane (g, t) wants tokens g and g + 8, two adjacent elements a register.  Which
//                elements make up "k" is free as long as Q agrees: lane t takes a run of D / 4
//                consecutive codes of its tokens.
//   V fragment   lane (g, t) wants tokens 2t, 2t + 1, 2t + 8, 2t + 9 of "rows" d; it takes the
//                run of D / 8 codes at g * D / 8, and a byte permute pairs two tokens' codes.
//   P            the score fragment holds tokens by rows; movmatrix turns it into the B operand.
// Codes become halves exactly (one conversion a pair; the e4m3 form of the MMA, with Q as two
// codes an element, issued more instructions, not fewer: 398 a unit against 335).  Q goes to
// halves too: each row times a power of two that puts its largest element in [2^14, 2^15), so that
// elements down to 2^-31 of it keep all their bits.
// Scales join outside the products: a page's key scale multiplies its scores, and the logarithm of
// its value scale is added to them, so that what is exponentiated is a token's weight on the
// output, p * scale, under a running maximum of that weight (a maximum of p alone would let a
// heavy page with small p push the others below half's range); the softmax's denominator takes the
// weights over the scale again.  Weights are rounded to half (2^-11), held times 2^10, so
// those down to 2^-24 of the largest keep full precision; scores, maxima, sums and outputs are f32.
//
// Work is dealt out by the unit of 16 tokens: the units of all (sequence, KV head, column block)
// segments, end to end, are cut into equal runs, one a CTA, so ragged lengths leave no CTA idle.
// A CTA's four warps take a run's units in turn and merge in shared memory; a segment cut by a CTA
// boundary leaves partials in the workspace, which a second small launch folds in order.
//
// Over ragged rows (row_start) the kernel takes the sequences that bring one row and passes the others.
//
// Measured (32 heads over 8): 64 sequences of 2048, heads of 64: 32.4 us (135 MB, 4.2 TB/s, 64 % of a plain
// copy's rate); one of 120,001, heads of 128: 51.1 us (4.8 TB/s, 74 %); 128 of 3 to 8191, over 4, that hold
// 141 MB: 36.5 us (3.9 TB/s), 550 MB: 102 us (5.4 TB/s, 83 %); one of 500: 9.1 us.  A long call is bound by
// bytes; in a short one some 13,000 clocks go by before a CTA's first product (share, page ids, scales, copies),
// and each unit is a chain of conversions, products and exponentials (200 instructions at heads of 64, half
// of them on the integer pipe).
#include <type_traits>

#include "common.cuh"
#include "mma.cuh"
#include "pages.cuh"
#include "tc.cuh"

namespace iron {

constexpr int kPgWarps = 4;
constexpr int kPgThreads = kPgWarps * 32;
// CTAs an SM: what the registers of one or of two groups of eight columns allow without spilling.  (Two for
// one group: 64 x 2048 33.9 us for 31.9, 200 of 1 to 3000 76 for 67, one long sequence 48.8 for 50.8.)
constexpr int pg_ctas_per_sm(int nt) { return nt == 1 ? 3 : 2; }
constexpr int kPgCtas = kSMs * pg_ctas_per_sm(1);
constexpr int kPgUnit = 16;                 // tokens
constexpr int kPgStages = 2;                // of a warp's ring; a stage holds kGroup units
// Units a segment costs beside its own: its queries and the meeting of its warps.  128 sequences of 3 to
// 8191 that hold 141 MB with 8, 16, 24 and 40: 57, 41.7, 37.8 and 40.1 us; even lengths do not care.
constexpr int kPgSegCost = 24;
constexpr float kPgLift = 10.f;             // log2 of what probabilities are held times

// A sequence as the kernel sees it: its keys [lo, len), the first unit of 16 that holds one, and how
// many units a segment -- a KV head's group of columns -- has.  An empty one still has a unit:
// somebody must write its zeros.
struct PagesSeq {
  int len, lo, unit0, units, row;   // row: of q and of the outputs
};
__device__ __forceinline__ PagesSeq pages_seq(const PagesParams& p, int b) {
  PagesSeq s;
  s.len = seq_len(p, b);
  s.row = b;
  s.lo = p.window >= 0 ? max(0, s.len - 1 - p.window) : 0;
  s.unit0 = s.lo / kPgUnit;
  s.units = max(1, (s.len + kPgUnit - 1) / kPgUnit - s.unit0);
  if (p.row_start && seq_rows(p, b, s.row) != 1) s.units = 0;   // ragged rows: those of one row are this kernel's
  return s;
}

template <int D, int NT>
struct PgCfg {
  static constexpr int kCols = NT * 8;
  static constexpr int kPartial = kCols * D + 2 * kCols;   // floats of a partial: outputs, maxima, sums
  static constexpr int kGroup = D == 128 ? 2 : 4;          // units a warp takes at a time
  static constexpr int kHalf = kPgUnit * D;                // bytes of a unit's keys, and of its values
  static constexpr int kStage = kGroup * 2 * kHalf;        // 8 KB
  static constexpr int kParts = NT * D <= 64 ? 1 : NT * D / 64;   // steps (of 8 KB) the warps' outputs meet in
  static constexpr int kRing = 0;
  static constexpr int kMerge = kPgWarps * kPgStages * kStage;
  static constexpr int kBars = kMerge + kPgWarps * kCols * (D / kParts) * 4;
  static constexpr int kSmem = kBars + 128 + 1024;
};

// what a sequence's segments cost in units; `segs`: KV heads times groups of columns
__device__ __forceinline__ long long pages_cost(int segs, const PagesSeq& s) {
  return s.units ? (long long)segs * (s.units + kPgSegCost) : 0;
}

// units per CTA: an equal share, and two groups a warp at least
__device__ __forceinline__ long long pages_share(long long total, int ctas) {
  const long long even = div_ll(total + ctas - 1, ctas);
  return even < 2 * kPgWarps + kPgSegCost ? 2 * kPgWarps + kPgSegCost : even;
}

__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) {
  uint32_t r;
  asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(sel));
  return r;
}
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ void mma_f16_16816(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
      ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
      : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
  return v;
}

// One segment's piece of a CTA's share.
struct PagesPiece {
  int b, gh, col0, cols;        // sequence, KV head, first query head of its group, heads
  PagesSeq seq;
  int first, last;              // units of the segment
  long long end_at;             // where the segment ends in the dealt-out units
};

template <int D, int NT>
__global__ void __launch_bounds__(kPgThreads, pg_ctas_per_sm(NT))
mha_pages_kernel(const __grid_constant__ CUtensorMap map, const PagesParams p) {
  using Cfg = PgCfg<D, NT>;
  constexpr int COLS = Cfg::kCols, U = Cfg::kGroup;
  constexpr int KS = D / 16;                    // MMAs along d of a score
  constexpr int NB = 32 / U;                    // groups whose pages a warp's lanes look up at once
  extern __shared__ uint8_t pg_smem_raw[];
  __shared__ float s_m[kPgWarps][COLS], s_l[kPgWarps][COLS], s_w[kPgWarps][COLS];
  __shared__ int s_abort;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(pg_smem_raw) + 1023) & ~uintptr_t(1023));
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int hg = p.hg, page_mask = (1 << p.log_page) - 1;
  const int blocks = (hg + COLS - 1) / COLS, segs = p.G * blocks;
  float* s_o = reinterpret_cast<float*>(smem + Cfg::kMerge);   // [warp][column][D / kParts]
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Cfg::kBars) + warp * kPgStages;
  const uint32_t ring = smem_u32(smem + Cfg::kRing) + warp * kPgStages * Cfg::kStage;
  if (lane == 0) {
    for (int i = 0; i < kPgStages; ++i) mbar_init(bars + i, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (tid == 0) {
    s_abort = 0;
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map) : "memory");
  }

  __syncthreads();      // the abort flag is there
  volatile int* abort_flag = &s_abort;

  pdl_launch();
  pdl_wait();
  // Where this CTA's run of units begins: every warp looks at all sequences for itself, 32 at once, so
  // that none waits for another.
  auto seq_cost = [&](int b) { return b < p.B ? pages_cost(segs, pages_seq(p, b)) : 0ll; };
  long long total = 0;
  for (int b0 = 0; b0 < p.B; b0 += 32) total += seq_cost(b0 + lane);
#pragma unroll
  for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  const long long share = pages_share(total, p.ctas);
  const long long begin = (long long)blockIdx.x * share, end = min(begin + share, total);
  if (tid == 0) p.records[blockIdx.x].pieces = 0;   // until this CTA begins a segment that others go on with
  if (begin >= end) return;
  int seq_b = 0;
  long long seq_at = 0;         // where sequence seq_b begins in the dealt-out units
  for (;; seq_b += 32) {
    if (seq_b >= p.B) return;   // never, unless the lengths change under the call
    const long long own = seq_cost(seq_b + lane);
    long long upto = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, begin < seq_at + upto);
    if (hit) {
      seq_b += __ffs(hit) - 1;
      seq_at += __shfl_sync(0xffffffffu, upto - own, __ffs(hit) - 1);
      break;
    }
    seq_at += __shfl_sync(0xffffffffu, upto, 31);
  }
  PagesSeq seq = pages_seq(p, seq_b);

  // The piece of the share [at, end) that begins at `at`; false when nothing is left.  A segment's
  // units follow the kPgSegCost that it costs beside them, so a share may hold none of its own.
  auto next_piece = [&](long long& at, PagesPiece& x) {
    while (at < end) {
      for (long long w; at >= seq_at + (w = pages_cost(segs, seq));) {
        seq_at += w;
        if (++seq_b >= p.B) return false;   // never, unless the lengths change under the call
        seq = pages_seq(p, seq_b);
        while (seq.units == 0) {      // the next that has some, 32 at a look
          const unsigned some = __ballot_sync(0xffffffffu, seq_b + lane < p.B && pages_seq(p, seq_b + lane).units > 0);
          if (some) seq = pages_seq(p, seq_b += __ffs(some) - 1);
          else if ((seq_b += 32) >= p.B) return false;
        }
      }
      const int span = seq.units + kPgSegCost;
      const int seg = (int)div_ll(at - seq_at, span);
      const long long seg_at = seq_at + (long long)seg * span;
      const int lo = (int)(at - seg_at), hi = (int)(min(end, seg_at + span) - seg_at);
      at = seg_at + hi;
      x.first = max(lo - kPgSegCost, 0);
      x.last = max(hi - kPgSegCost, 0);
      if (x.first >= x.last) continue;
      x.b = seq_b;
      x.gh = blocks == 1 ? seg : seg / blocks;
      x.col0 = (seg - x.gh * blocks) * COLS;
      x.cols = min(COLS, hg - x.col0);
      x.seq = seq;
      x.end_at = seg_at + span;
      return true;
    }
    return false;
  };

  int filled = 0, drained = 0;   // groups of this warp so far: a group's stage and phase
  // lane l looks up unit l % U of group l / U of a batch of NB groups: the page ids two batches ahead, the
  // scales one, so that neither load is waited for in the run of the groups
  struct Batch { int entry; float2 scale; };
  auto look_up = [&](const PagesPiece& x, int k0) {
    const int u = x.first + ((k0 + lane / U) * kPgWarps + warp) * U + lane % U;
    int e = -1;
    if (u < x.last && x.seq.len > 0)
      e = p.tables[(long long)x.b * p.width + (((x.seq.unit0 + u) * kPgUnit) >> p.log_page)];
    return e >= 0 && e < p.P ? e : -1;
  };
  auto look_up_scales = [&](const PagesPiece& x, Batch& q) {
    q.scale = make_float2(1.f, 1.f);
    if (q.entry >= 0) q.scale = *reinterpret_cast<const float2*>(p.scales + ((long long)q.entry * p.G + x.gh) * 2);
  };
  // group k of the piece into the ring: lanes 0 .. U - 1 a unit each
  auto fill = [&](const PagesPiece& x, int entries, int k) {
    const int entry = __shfl_sync(0xffffffffu, entries, (k % NB) * U + (lane % U));
    const int u = x.first + (k * kPgWarps + warp) * U + lane;
    const bool on = lane < U && entry >= 0;
    const int n = __popc(__ballot_sync(0xffffffffu, on));
    const int stage = filled % kPgStages;
    if (lane == 0) mbar_expect_tx(bars + stage, n * 2 * Cfg::kHalf);
    __syncwarp();
    if (on) {
      const uint32_t dst = ring + stage * Cfg::kStage + lane * 2 * Cfg::kHalf, bar = smem_u32(bars + stage);
      const int off = ((x.seq.unit0 + u) * kPgUnit) & page_mask, block = entry * p.G + x.gh;
      tma_load_3d(dst, &map, 0, off, block, bar);
      tma_load_3d(dst + Cfg::kHalf, &map, 0, page_mask + 1 + off, block, bar);
    }
    ++filled;
  };
  auto groups_of = [&](const PagesPiece& x) {
    const int groups = (x.last - x.first + U - 1) / U;
    return (groups - warp + kPgWarps - 1) / kPgWarps;
  };

  long long at = begin;
  PagesPiece cur;
  Batch bat = {-1, make_float2(1.f, 1.f)}, bat_next = bat;
  int entry_after = -1;
  float key_scale = 1.f, log_v = 0.f, inv_v = 1.f;   // of `bat`
  auto use_scales = [&]() {
    key_scale = bat.scale.x;
    log_v = __log2f(bat.scale.y);
    inv_v = 1.f / bat.scale.y;
  };
  uint4 q_raw[NT][D / 32];      // this lane's share of the query of column 8 nt + g: a run of D / 4
  // the loads that a piece begins with, in the order in which others wait for them
  auto open_piece = [&]() {
    bat.entry = look_up(cur, 0);
    bat_next.entry = look_up(cur, NB);
    entry_after = look_up(cur, 2 * NB);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int c = nt * 8 + g;
      const __nv_bfloat16* src = p.q + ((long long)cur.seq.row * p.H + cur.gh * hg + cur.col0 + c) * D + t * (D / 4);
#pragma unroll
      for (int i = 0; i < D / 32; ++i) q_raw[nt][i] = c < cur.cols ? ld_cached(src + 8 * i) : make_uint4(0, 0, 0, 0);
    }
    look_up_scales(cur, bat);     // before the copies: behind everybody's they would come last
    const int n = groups_of(cur);
    for (int k = 0; k < kPgStages && k < n; ++k) fill(cur, bat.entry, k);
    look_up_scales(cur, bat_next);
  };
  bool have = next_piece(at, cur);
  bool ok = true;
  if (have) open_piece();
  while (have) {
    // ---- Q: this lane's share of column 8 nt + g, in halves under a power of two ----
    uint32_t qf[NT][KS][2];
    float colfac[NT][2];                        // of columns 8 nt + 2t and + 1
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float mx = 0.f;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        float f[8];
        unpack8(q_raw[nt][i], f);
#pragma unroll
        for (int j = 0; j < 8; ++j) mx = fmaxf(mx, fabsf(f[j]));
      }
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      // mx * up lies in [2^14, 2^15); zero, subnormal and non-finite rows keep finite factors
      const int e = min(max((int)(__float_as_uint(mx) >> 23), 15), 254);
      const float up = __uint_as_float((uint32_t)(268 - e) << 23);
      const float down = 1.0f / up;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        float f[8];
        unpack8(q_raw[nt][i], f);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          qf[nt][2 * i + j][0] = pack_half2(f[4 * j] * up, f[4 * j + 1] * up);
          qf[nt][2 * i + j][1] = pack_half2(f[4 * j + 2] * up, f[4 * j + 3] * up);
        }
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) colfac[nt][j] = __shfl_sync(0xffffffffu, down, (2 * t + j) * 4) * p.scale_log2;
    }

    float o[KS][NT][4], m_run[NT][2], l_run[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int j = 0; j < 2; ++j) { m_run[nt][j] = -INFINITY; l_run[nt][j] = 0.f; }
#pragma unroll
      for (int i = 0; i < KS; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[i][nt][j] = 0.f;
    }

    use_scales();
    const int groups = groups_of(cur);
    for (int k = 0; k < groups && ok; ++k) {
      const int stage = drained % kPgStages;
      ok = mbar_wait(bars + stage, (drained / kPgStages) & 1, abort_flag);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      ++drained;
      const uint32_t base = ring + stage * Cfg::kStage;
      const int src0 = (k % NB) * U, tok0 = (cur.seq.unit0 + cur.first + (k * kPgWarps + warp) * U) * kPgUnit;
      // Whether every unit of the group is there and its tokens are all keys.  The common case goes
      // without a branch, so that the units' chains of products interleave.
      const bool whole = __all_sync(0xffffffffu, __shfl_sync(0xffffffffu, bat.entry, src0 + lane % U) >= 0) &&
                         tok0 >= cur.seq.lo && tok0 + U * kPgUnit <= cur.seq.len;
      auto key = [&](int tok) { return tok >= cur.seq.lo && tok < cur.seq.len; };
      auto group = [&](auto is_whole) {
        constexpr bool kWhole = decltype(is_whole)::value;
        // ---- S^T = K Q^T ----
        float s[U][NT][4];
        uint32_t kf[U][2][D / 16];
#pragma unroll
        for (int i = 0; i < U; ++i) {
          const uint32_t kb = base + i * 2 * Cfg::kHalf;
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            if (D == 128) {
              const uint32_t row = kb + (g + 8 * r) * 128;
              const uint4 x = lds128(row + (((2 * t) ^ g) << 4)), y = lds128(row + (((2 * t + 1) ^ g) << 4));
              kf[i][r][0] = x.x; kf[i][r][1] = x.y; kf[i][r][2] = x.z; kf[i][r][3] = x.w;
              kf[i][r][D / 16 - 4] = y.x; kf[i][r][D / 16 - 3] = y.y; kf[i][r][D / 16 - 2] = y.z; kf[i][r][D / 16 - 1] = y.w;
            } else {
              const uint4 x = lds128(kb + (g + 8 * r) * 64 + ((t ^ ((g >> 1) & 3)) << 4));
              kf[i][r][0] = x.x; kf[i][r][1] = x.y; kf[i][r][2] = x.z; kf[i][r][3] = x.w;
            }
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) s[i][nt][0] = s[i][nt][1] = s[i][nt][2] = s[i][nt][3] = 0.f;
        }
#pragma unroll
        for (int c = 0; c < KS; ++c)
#pragma unroll
          for (int i = 0; i < U; ++i) {
            const uint32_t a[4] = {e4m3x2_to_half2(kf[i][0][c]), e4m3x2_to_half2(kf[i][1][c]),
                                   e4m3x2_hi_to_half2(kf[i][0][c]), e4m3x2_hi_to_half2(kf[i][1][c])};
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma_f16_16816(s[i][nt], a, qf[nt][c][0], qf[nt][c][1]);
          }
        // ---- scales, running maximum ----
        float m_new[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) m_new[nt][0] = m_run[nt][0], m_new[nt][1] = m_run[nt][1];
#pragma unroll
        for (int i = 0; i < U; ++i) {
          const float sk = __shfl_sync(0xffffffffu, key_scale, src0 + i), lv = __shfl_sync(0xffffffffu, log_v, src0 + i);
          bool seen[2] = {true, true};
          if (!kWhole) {
            const bool there = __shfl_sync(0xffffffffu, bat.entry, src0 + i) >= 0;
            seen[0] = there && key(tok0 + i * kPgUnit + g);
            seen[1] = there && key(tok0 + i * kPgUnit + g + 8);
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              s[i][nt][j] = seen[j >> 1] ? fmaf(s[i][nt][j], colfac[nt][j & 1] * sk, lv) : -INFINITY;
              m_new[nt][j & 1] = fmaxf(m_new[nt][j & 1], s[i][nt][j]);
            }
        }
        bool moved = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            float& m = m_new[nt][j];
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
            moved = moved || m != m_run[nt][j];
          }
        if (__any_sync(0xffffffffu, moved)) {   // seldom after the first groups
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const float corr = ex2(m_run[nt][j] - (m_new[nt][j] == -INFINITY ? 0.f : m_new[nt][j]));
              m_run[nt][j] = m_new[nt][j];
              l_run[nt][j] *= corr;
#pragma unroll
              for (int c = 0; c < KS; ++c) { o[c][nt][j] *= corr; o[c][nt][j + 2] *= corr; }
            }
        }
        // ---- weights and their sum; O^T += V^T P^T ----
        float zero[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float m = m_run[nt][j] == -INFINITY ? 0.f : m_run[nt][j], lifted = m - kPgLift;
            // past 2^27 the difference rounds to a lift of 16, which is past the largest half: none there
            zero[nt][j] = m - lifted > 15.f ? m : lifted;
          }
#pragma unroll
        for (int i = 0; i < U; ++i) {
          const float inv = __shfl_sync(0xffffffffu, inv_v, src0 + i);
          uint32_t pb[NT][2];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            float pr[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) pr[j] = ex2(s[i][nt][j] - zero[nt][j & 1]);
#pragma unroll
            for (int j = 0; j < 2; ++j) l_run[nt][j] = fmaf(pr[j] + pr[j + 2], inv, l_run[nt][j]);
            pb[nt][0] = movmatrix_trans(pack_half2(pr[0], pr[1]));
            pb[nt][1] = movmatrix_trans(pack_half2(pr[2], pr[3]));
          }
          uint32_t vf[4][D / 32];
          const uint32_t vb = base + i * 2 * Cfg::kHalf + Cfg::kHalf;
          const bool there = kWhole || __shfl_sync(0xffffffffu, bat.entry, src0 + i) >= 0;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int row = 2 * t + (r & 1) + (r >> 1) * 8;
            if (D == 128) {
              const uint4 x = lds128(vb + row * 128 + ((g ^ (row & 7)) << 4));
              vf[r][0] = x.x; vf[r][1] = x.y; vf[r][D / 32 - 2] = x.z; vf[r][D / 32 - 1] = x.w;
            } else {
              const uint2 x = lds64(vb + row * 64 + ((((g >> 1) ^ ((row >> 1) & 3)) << 4) | ((g & 1) << 3)));
              vf[r][0] = x.x; vf[r][1] = x.y;
            }
            // what lies where no key does (a page's tail, an absent page) may be NaN, and 0 x NaN is NaN
            if (!kWhole && !(there && key(tok0 + i * kPgUnit + row)))
#pragma unroll
              for (int w = 0; w < D / 32; ++w) vf[r][w] = 0;
          }
#pragma unroll
          for (int c = 0; c < KS; ++c) {
            const uint32_t sel = (c & 1) ? 0x7362u : 0x5140u;
            const uint32_t x = prmt(vf[0][c >> 1], vf[1][c >> 1], sel), y = prmt(vf[2][c >> 1], vf[3][c >> 1], sel);
            const uint32_t a[4] = {e4m3x2_to_half2(x), e4m3x2_hi_to_half2(x), e4m3x2_to_half2(y), e4m3x2_hi_to_half2(y)};
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma_f16_16816(o[c][nt], a, pb[nt][0], pb[nt][1]);
          }
        }
      };
      if (whole) group(std::true_type{}); else group(std::false_type{});
      // ---- the stage is read: the group kPgStages on takes it ----
      __syncwarp();
      const int kf_ = k + kPgStages;
      if (kf_ < groups) fill(cur, kf_ / NB == k / NB ? bat.entry : bat_next.entry, kf_);
      if ((k + 1) % NB == 0) {
        bat = bat_next;
        use_scales();
        bat_next.entry = entry_after;
        look_up_scales(cur, bat_next);
        entry_after = look_up(cur, k + 1 + 2 * NB);
      }
    }

    // the next piece's first groups come while this one's results meet
    const PagesPiece done = cur;
    have = ok && next_piece(at, cur);
    if (have) {
      open_piece();
    }

    // ---- the warps' results meet; a lane's sums are of its own tokens only ----
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float l = l_run[nt][j];
        l += __shfl_xor_sync(0xffffffffu, l, 4);
        l += __shfl_xor_sync(0xffffffffu, l, 8);
        l += __shfl_xor_sync(0xffffffffu, l, 16);
        if (g == 0) { s_m[warp][nt * 8 + 2 * t + j] = m_run[nt][j]; s_l[warp][nt * 8 + 2 * t + j] = l; }
      }
    __syncthreads();
    if (tid < COLS) {
      float m = -INFINITY, l = 0.f;
      for (int w = 0; w < kPgWarps; ++w) m = fmaxf(m, s_m[w][tid]);
      const float safe = m == -INFINITY ? 0.f : m;
      for (int w = 0; w < kPgWarps; ++w) {
        const float f = ex2(s_m[w][tid] - safe);
        s_w[w][tid] = f;
        l += s_l[w][tid] * f;
      }
      s_m[0][tid] = m; s_l[0][tid] = l;
    }
    const bool direct = done.first == 0 && done.last == done.seq.units;
    // a piece that begins before this CTA's share uses the CTA's first slot, one that goes on the second
    float* part = p.partial + ((long long)blockIdx.x * 2 + (done.first == 0 ? 1 : 0)) * Cfg::kPartial;
    // the outputs meet a part of d at a time: MMA c holds codes 2 c and 2 c + 1 of each lane
    // group's run of D / 8
    constexpr int kParts = Cfg::kParts, CP = KS / kParts, DP = D / kParts;
#pragma unroll
    for (int part_i = 0; part_i < kParts; ++part_i) {
      if (part_i) __syncthreads();
#pragma unroll
      for (int c = part_i * CP; c < (part_i + 1) * CP; ++c)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int col = nt * 8 + 2 * t + (j & 1);
            const int dd = g * (2 * CP) + 2 * (c - part_i * CP) + (j >> 1);   // of this part
            s_o[(warp * COLS + col) * DP + dd] = o[c][nt][j];
          }
      __syncthreads();
      for (int x = tid; x < done.cols * DP; x += kPgThreads) {
        const int col = x / DP, dd = x % DP;
        const int d = (dd / (2 * CP)) * (D / 8) + part_i * 2 * CP + dd % (2 * CP);
        float acc = 0.f;
#pragma unroll
        for (int w = 0; w < kPgWarps; ++w) acc += s_o[(w * COLS + col) * DP + dd] * s_w[w][col];
        if (direct) {
          const float l = s_l[0][col];
          // a row that sees nothing is zero; l is NaN where a score it sees is
          p.out[((long long)done.seq.row * p.H + done.gh * hg + done.col0 + col) * D + d] =
              __float2bfloat16_rn(l == 0.f ? 0.f : acc / l);
        } else {
          part[col * D + d] = acc;
        }
      }
    }
    if (!direct) {
      if (tid == 0 && done.first == 0) {
        PagesRecord r;
        r.pieces = (int)((done.end_at - 1) / share) - (int)blockIdx.x + 1;
        r.row0 = done.seq.row; r.head0 = done.gh * hg; r.col0 = done.col0;
        r.cols = done.cols;
        p.records[blockIdx.x] = r;
      }
      if (tid < done.cols) {
        part[COLS * D + tid] = s_m[0][tid];
        part[COLS * D + COLS + tid] = s_l[0][tid];
      }
    }
    __syncthreads();   // shared memory is the next piece's
    ok = ok && !*abort_flag;
    have = have && ok;
  }
  if (!ok) {
    // a wait gave up: give the copies in flight a millisecond, many times what one takes
    if (tid == 0 && p.status) *p.status = IRON_ERR_TIMEOUT;
    const unsigned long long t0 = global_ns();
    while (global_ns() - t0 < 1000000ull) {}
  }
}

// Folds the partials of a segment that several CTAs share, in the order of its keys.  One CTA for
// each main CTA, whose record says whether it begins such a segment, and column; the warps take the
// pieces in turn, a lane a stretch of d.
constexpr int kFoldWarps = 8;
constexpr int kFoldBatch = 4;    // pieces whose loads a warp has in flight at once
template <int D, int NT>
__global__ void __launch_bounds__(kFoldWarps * 32) mha_pages_fold_kernel(const PagesParams p) {
  using Cfg = PgCfg<D, NT>;
  constexpr int COLS = Cfg::kCols, PER = D / 32;
  __shared__ float s_o[kFoldWarps][D], s_m[kFoldWarps], s_l[kFoldWarps];
  pdl_launch();
  pdl_wait();
  const PagesRecord r = p.records[blockIdx.x];
  const int c = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (r.pieces <= 1 || c >= r.cols) return;
  float m = -INFINITY, l = 0.f, o[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) o[j] = 0.f;
  for (int i0 = warp; i0 < r.pieces; i0 += kFoldBatch * kFoldWarps) {
    float x[kFoldBatch][PER], mi[kFoldBatch], li[kFoldBatch];
#pragma unroll
    for (int k = 0; k < kFoldBatch; ++k) {
      const int i = min(i0 + k * kFoldWarps, r.pieces - 1);   // past the end: loaded again, not counted
      // the piece that begins the segment lies in its CTA's second slot, the others in the first
      const float* src = p.partial + ((long long)(blockIdx.x + i) * 2 + (i == 0 ? 1 : 0)) * Cfg::kPartial;
      mi[k] = src[COLS * D + c];
      li[k] = src[COLS * D + COLS + c];
      const float2* v = reinterpret_cast<const float2*>(src + c * D + lane * PER);
#pragma unroll
      for (int j = 0; j < PER / 2; ++j) { const float2 y = v[j]; x[k][2 * j] = y.x; x[k][2 * j + 1] = y.y; }
    }
#pragma unroll
    for (int k = 0; k < kFoldBatch; ++k) {
      if (i0 + k * kFoldWarps >= r.pieces) break;
      const float m_new = fmaxf(m, mi[k]), safe = m_new == -INFINITY ? 0.f : m_new;
      const float f = ex2(m - safe), fi = ex2(mi[k] - safe);
      m = m_new;
      l = l * f + li[k] * fi;
#pragma unroll
      for (int j = 0; j < PER; ++j) o[j] = o[j] * f + x[k][j] * fi;
    }
  }
#pragma unroll
  for (int j = 0; j < PER; ++j) s_o[warp][lane * PER + j] = o[j];
  if (lane == 0) { s_m[warp] = m; s_l[warp] = l; }
  __syncthreads();
  const int d = threadIdx.x, warps = min(kFoldWarps, r.pieces);
  if (d < D) {
    m = s_m[0];
    for (int w = 1; w < warps; ++w) m = fmaxf(m, s_m[w]);
    const float safe = m == -INFINITY ? 0.f : m;
    float acc = 0.f;
    l = 0.f;
    for (int w = 0; w < warps; ++w) {
      const float f = ex2(s_m[w] - safe);
      l += s_l[w] * f;
      acc += s_o[w][d] * f;
    }
    p.out[((long long)r.row0 * p.H + r.head0 + r.col0 + c) * D + d] = __float2bfloat16_rn(l == 0.f ? 0.f : acc / l);
  }
}

// What a call without a status word of its own reports to: one word a device, the library's.
__device__ int g_pages_status;
static int* pages_status_word() {
  static std::atomic<int*> known[64];
  const int dev = current_device();
  if (dev < 0) return nullptr;
  int* word = known[dev].load(std::memory_order_acquire);
  if (!word) {
    void* at = nullptr;
    if (cudaGetSymbolAddress(&at, g_pages_status) != cudaSuccess) return nullptr;
    word = (int*)at;
    known[dev].store(word, std::memory_order_release);
  }
  return word;
}

typedef CUresult (*PgEncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                               const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                               CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// (byte of a row, row of a (page, head)'s keys and values, page x head); boxes of 16 whole rows.
static bool pages_map(CUtensorMap* map, const PagesParams& p, int D) {
  static std::atomic<PgEncodeFn> known{nullptr};
  PgEncodeFn fn = known.load(std::memory_order_acquire);
  if (!fn) {
    void* sym = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &sym, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      return false;
    fn = reinterpret_cast<PgEncodeFn>(sym);
    known.store(fn, std::memory_order_release);
  }
  const cuuint64_t rows = (cuuint64_t)2 << p.log_page;
  const cuuint64_t dims[3] = {(cuuint64_t)D, rows, (cuuint64_t)p.P * p.G};
  const cuuint64_t strides[2] = {(cuuint64_t)D, (cuuint64_t)D * rows};
  const cuuint32_t box[3] = {(cuuint32_t)D, (cuuint32_t)kPgUnit, 1}, elem[3] = {1, 1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<uint8_t*>(p.pool), dims, strides, box, elem,
            CU_TENSOR_MAP_INTERLEAVE_NONE, D == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D, int NT>
static int launch_pages(PagesParams p, cudaStream_t stream) {
  p.ctas = kSMs * pg_ctas_per_sm(NT);
  CUtensorMap map;
  if (!pages_map(&map, p, D)) return IRON_ERR_UNSUPPORTED;
  constexpr int smem = PgCfg<D, NT>::kSmem;
  static DeviceOnce configured;
  if (!configured.done()) {
    if (cudaFuncSetAttribute(mha_pages_kernel<D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
      return IRON_ERR_LAUNCH;
    configured.mark();
  }
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(kPgThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  fill_pdl_attr(cfg, attr);
  cfg.gridDim = dim3(p.ctas);
  if (cudaLaunchKernelEx(&cfg, mha_pages_kernel<D, NT>, map, p) != cudaSuccess) return IRON_ERR_LAUNCH;
  cfg.gridDim = dim3(p.ctas, NT * 8 < p.hg ? NT * 8 : p.hg);
  cfg.blockDim = dim3(kFoldWarps * 32);
  cfg.dynamicSmemBytes = 0;
  return cudaLaunchKernelEx(&cfg, mha_pages_fold_kernel<D, NT>, p) == cudaSuccess ? IRON_OK : IRON_ERR_LAUNCH;
}

template <int D>
static int launch_pages_cols(const PagesParams& p, int cols, cudaStream_t stream) {
  // one group of eight columns where the heads of a KV head fit it (64 x 2048 with two: 41.9 us for 33.3, before the look-ups were moved ahead)
  return cols <= 8 ? launch_pages<D, 1>(p, stream) : launch_pages<D, 2>(p, stream);
}

static int launch_decode(const PagesParams& p, int D, cudaStream_t stream) {
  return D == 64 ? launch_pages_cols<64>(p, p.hg, stream) : launch_pages_cols<128>(p, p.hg, stream);
}

}  // namespace iron

using namespace iron;

extern "C" int* iron_mha_pages_status_word(void) { return pages_status_word(); }

extern "C" long long iron_mha_pages_workspace_bytes(int D, int prompt) {
  if (D != 64 && D != 128) return 0;
  const long long partial = 16ll * D + 32;
  return (prompt ? mha_pages_tc_workspace_bytes(D) : 0) +
         (long long)kPgCtas * (2 * partial * (long long)sizeof(float) + (long long)sizeof(PagesRecord));
}

static int pages_args(PagesParams& p, const void* q, const void* pool, const float* scales, int P, int page_size,
                      const int* tables, int width, const int* lengths, const int* row_start, int B, int rows, int H,
                      int G, int D, int causal, int window, float scale, void* workspace, long long workspace_bytes,
                      void* out) {
  const int log_page = log2_page(page_size);
  if (B < 0 || rows < 0 || H <= 0 || G <= 0 || H % G || (D != 64 && D != 128) || P <= 0 || width <= 0 || log_page < 0)
    return IRON_ERR_SHAPE;
  // indices of 16-token units, tokens and columns are 32-bit, with room for a tile's or an item's end
  constexpr long long kMost = 0x7fffffffll - 1023;
  if (G > 65535 || (long long)P * G * (page_size / 8) > kMost || (long long)P * page_size > kMost ||
      (long long)width * page_size > kMost || (long long)rows * H > kMost)
    return IRON_ERR_SHAPE;
  if (window >= 0 && !causal) return IRON_ERR_UNSUPPORTED;
  if (!(scale > 0.f)) return IRON_ERR_SHAPE;
  if (B == 0 || rows == 0) return 1;   // nothing to do
  if (!q || !pool || !scales || !tables || !lengths || !out || !workspace) return IRON_ERR_SHAPE;
  if (!aligned16(q) || !aligned16(pool) || !aligned16(out) || !aligned16(workspace) ||
      (reinterpret_cast<uintptr_t>(scales) & 7))
    return IRON_ERR_ALIGN;
  if (workspace_bytes < iron_mha_pages_workspace_bytes(D, row_start != nullptr)) return IRON_ERR_WORKSPACE;
  p.q = (const __nv_bfloat16*)q; p.pool = (const uint8_t*)pool; p.scales = scales; p.tables = tables;
  p.lengths = lengths; p.row_start = row_start; p.out = (__nv_bfloat16*)out;
  p.records = (PagesRecord*)((char*)workspace + (row_start ? mha_pages_tc_workspace_bytes(D) : 0));
  p.partial = (float*)(p.records + kPgCtas);
  p.B = B; p.H = H; p.G = G; p.hg = H / G; p.P = P; p.width = width; p.log_page = log_page; p.causal = causal;
  p.window = window < (long long)width * page_size ? window : -1;   // one that leaves nothing out is none: no difference wraps
  p.rows = rows;
  p.scale_log2 = scale * 1.4426950408889634f;
  return IRON_OK;
}

extern "C" int iron_mha_decode_pages_bf16(const void* q, const void* pool, const float* scales, int P, int page_size,
                                          const int* tables, int width, const int* lengths, int B, int H, int G, int D,
                                          int window, float scale, void* workspace, long long workspace_bytes, void* out,
                                          int* status, iron_stream_t stream) {
  PagesParams p = {};
  const int rc = pages_args(p, q, pool, scales, P, page_size, tables, width, lengths, nullptr, B, B, H, G, D, 1, window,
                            scale, workspace, workspace_bytes, out);
  if (rc) return rc == 1 ? IRON_OK : rc;
  p.status = status ? status : pages_status_word();
  return launch_decode(p, D, (cudaStream_t)stream);
}

extern "C" int iron_mha_prefill_pages_bf16(const void* q, const void* pool, const float* scales, int P, int page_size,
                                           const int* tables, int width, const int* lengths, const int* row_start, int B,
                                           int rows, int H, int G, int D, int causal, int window, float scale,
                                           void* workspace, long long workspace_bytes, void* out, int* status, iron_stream_t stream) {
  PagesParams p = {};
  const int rc = pages_args(p, q, pool, scales, P, page_size, tables, width, lengths, row_start, B, rows, H, G, D,
                            causal, window, scale, workspace, workspace_bytes, out);
  if (rc) return rc == 1 ? IRON_OK : rc;
  if (!row_start) return IRON_ERR_SHAPE;
  p.status = status ? status : pages_status_word();
  // A sequence of one row fills hg of the ragged kernel's 128 lanes, the decode kernel's eight columns
  // well.  32 heads over 8 of 128, pages of 64, without and with the split: 256 x 1 row on 300 tokens
  // 187 and 67 us, 64 x 1 on 3000 185 and 80, 16 x 1 on 300 27.6 and 21.5; where no sequence has one row
  // the decode kernel's launches are lost (8 x 64 rows on 1000: 43.0 and 49.2 us; 64 x 33: 118 and 123).
  // How many there are is known on the device alone, so: where there may be many, and where there
  // can be nothing else.  What the bound costs on either side of it: sixteen requests of one row each wait
  // 5 us longer than with the split, seventeen that bring more each some 5 us longer than without.
  p.split = B > 16 || rows == 1;
  if (rows > 1)
    if (const int bad = mha_pages_tc(p, D, workspace, (cudaStream_t)stream)) return bad;
  return p.split ? launch_decode(p, D, (cudaStream_t)stream) : IRON_OK;
}
