// Attention of ragged query rows over a key/value cache in pages of e4m3 codes, on tcgen05.
//
// A work item is a sequence, a KV head and up to 256 query columns -- (row, head of the group)
// pairs, so grouped heads fill the 128-row MMAs and share what is read -- against the keys any of
// them sees, in tiles of 128.  One persistent CTA an SM:
//   warps 8..11,  bring the codes: a tile's keys (8..11) and values (12..15) go from global memory,
//         12..15  page by page, the next tile's loads in flight, through registers, where codes
//                 become halves exactly, into the swizzled shared-memory operands
//   warps 16, 17  issue S = Q K^T and O += P V for the first and the second 128 columns, each on
//                 its own so that neither waits for the other's softmax
//   warps 0..3,   softmax of the first and the second 128 columns: a thread owns a column (one
//         4..7    lane of tensor memory) and has a step's 64 scores in registers at once; P takes
//                 half of their place in tensor memory as the second product's A operand
//   warp 18       walks the share's items and hands them to all through a ring
// A tile goes in two steps of 64 keys with a buffer of scores each, so that a step's exponentials are
// taken while the next one's scores are computed.  O stays in tensor memory; it is rescaled only when
// a row's maximum has grown by more than 2^8 over the one in use, which after the first tiles is seldom (the
// rescaling put off under a bounded slack is a published refinement of the online softmax).
//
// What the arithmetic is (scales, halves, weights) is the decode kernel's: Q as halves under a
// power of two a row, a page's key scale on its scores, the logarithm of its value scale added
// to them; P = p * value scale over the running maximum, in half, held times 2^6 so that with
// the 2^8 of slack it stays below half's 65504; weights down to 2^-20 of the maximum in use keep full
// precision.  Maxima, sums and outputs are f32.
//
// Items are dealt out by the tile: the tiles of all items, end to end, are cut into equal runs,
// one a CTA; an item that a boundary cuts leaves partials in the workspace, and a second small
// launch folds them in order.  Exponentials (16 a clock and SM) and MMAs both need 1024 clocks for
// 128 columns x 128 keys at D 128.
//
// Measured (32 heads over 8, a graph of ten calls at 1.965 GHz): 2048 causal rows, heads of 64: 61 us (280
// TFLOP/s); eight chunks of 61 to 1433 rows on 900 to 9001 tokens, heads of 128: 312 us (795 TFLOP/s), and 345 us
// (720 TFLOP/s) in a long run of calls, where the power cap holds the clock near 1.78 GHz; 16 x 7 rows on 4096:
// 73 us.  At its 96 registers a thread the kernel spills 12 (heads of 64) and 32 bytes (128).  What
// bounds the wide items is the softmax's chain: a step takes 2600 clocks of a half (290 until its scores are
// there, 560 for the maximum, 1250 for the weights, the rest handing over) where exponentials alone would
// take 1024, the exponentials' pipe is 41 % busy and the tensor pipe 41 %; registers allow no third
// group of warps to fill it.  Narrow items (few columns) wait for the converters, 5000 clocks a tile; a
// call has 12,000 to 14,000 clocks before its first tile and 4000 after an item's last.
//
// Every mbarrier wait is bounded; a wait that gives up sets the abort flag, every role unwinds,
// tensor memory is freed and the status word receives IRON_ERR_TIMEOUT.
#include "common.cuh"
#include "pages.cuh"
#include "tc.cuh"

namespace iron {

constexpr int kPtThreads = 640;
constexpr int kPtRows = 256;          // query columns of an item: two 128-row products
constexpr int kPtKeys = 128;          // keys of a tile
constexpr int kPtSub = 16384;         // a 128-row x 128-byte swizzled sub-tile
// What the tiles of one and of two 128-column halves cost, and an item beside its tiles: one half alone
// waits for its own chain of products and exponentials.  The eight ragged chunks with 2, 3, 4 for one half:
// 330, 311, 317 us; with 6, 12, 24 for an item: 345, 311, 317.
constexpr int kPtCostOne = 3, kPtCostTwo = 4, kPtItemCost = 12;
// A CTA's share is an item's own cost at least: 8 x 64 rows on 1000 tokens 43 us, with 36 51, with 72 73.
constexpr int kPtMinShare = 12;
constexpr float kPtLift = 6.f;        // log2 of what weights are held times
constexpr float kPtSlack = 8.f;       // log2 of how far the maximum in use may lag
constexpr float kPtFar = 4194304.f;   // 2^22: scores whose f32 steps reach the size of the lift and the slack
constexpr float kPtNone = -3.4028235e38f;   // the maximum in use of a row that has none
constexpr int kPtFoldWarps = 8;
constexpr int kPtSlots = 4;           // items looked up ahead
// Tiles whose scales are held.  Tile n's are written once the last scores of tile n - kStages are done, which the
// softmax's end with tile n - kStages - 1 precedes: kStages + 1 tiles may be wanted at once.
constexpr int kPtScales = 4;
constexpr int kPtPitch = 80;          // bytes between the rows a warp turns its outputs in: 16-byte pieces of 8 rows on 8 bank groups
constexpr int kPtRoles = 18;          // warps that read them

template <int D>
struct PtCfg {
  static constexpr int kChunks = D / 64;
  static constexpr int kTile = kChunks * kPtSub;
  static constexpr int kStages = D == 128 ? 2 : 3;
  static_assert(kPtScales >= kStages + 1, "the converters would write over scales that are still read");
  static constexpr int kQ = 0;
  static constexpr int kK = kQ + 2 * kTile;
  static constexpr int kV = kK + kStages * kTile;
  static constexpr int kScale = kV + kStages * kTile;      // a ring of tiles: [8 units] float4
  static constexpr int kItems = kScale + kPtScales * 8 * 16;   // a ring of items
  static constexpr int kOut = kItems + kPtSlots * 64;      // [8 warps] 32 rows x 64 bytes, kPtPitch apart
  static constexpr int kBars = kOut + 8 * 32 * kPtPitch;
  static constexpr int kSmem = kBars + 512 + 1024;
  static constexpr int kColS = 0;                          // 2 halves x 2 buffers x 64 columns (P: the last 32 of each)
  static constexpr int kColO = 256;                        // 2 x D columns
  static constexpr int kPartial = kPtRows * (D + 2);       // floats: outputs, maxima, sums
};

struct PtSeq {
  int len, row0, n, blocks;
};
__device__ __forceinline__ PtSeq pt_seq(const PagesParams& p, int b) {
  PtSeq s;
  s.len = seq_len(p, b);
  s.n = seq_rows(p, b, s.row0);
  if (p.split && s.n == 1) s.n = 0;    // the decode kernel's
  s.blocks = (s.n * p.hg + kPtRows - 1) / kPtRows;
  return s;
}

// An item: the columns, the keys that any and that every column sees, the tiles.
struct alignas(64) PtItem {
  int b, gh, col0, cols;             // no columns: the share's end
  int len, row0, past, whole;        // of the sequence; past: position of its first row; whole: no other CTA has tiles of it
  int any_lo, any_hi, all_lo, all_hi;
  int tile0, tiles;                  // first tile, and how many (at least one: somebody writes the zeros)
  int t_lo, t_hi;                    // this CTA's piece of them
};
__device__ __forceinline__ void pt_block(const PagesParams& p, const PtSeq& s, int j, PtItem& x) {
  x.col0 = j * kPtRows;
  x.cols = min(kPtRows, s.n * p.hg - x.col0);
  x.len = s.len; x.row0 = s.row0; x.past = s.len - s.n;
  const int first = x.past + x.col0 / p.hg, last = x.past + (x.col0 + x.cols - 1) / p.hg;
  x.any_lo = p.window >= 0 ? max(0, first - p.window) : 0;
  x.all_lo = p.window >= 0 ? last - p.window : 0;
  x.any_hi = p.causal ? max(0, min(s.len, last + 1)) : s.len;
  x.all_hi = p.causal ? max(0, min(s.len, first + 1)) : s.len;
  x.tile0 = x.any_lo / kPtKeys;
  x.tiles = max(1, (x.any_hi + kPtKeys - 1) / kPtKeys - x.tile0);
}
__device__ __forceinline__ int pt_tile_cost(const PtItem& x) { return x.cols > 128 ? kPtCostTwo : kPtCostOne; }
__device__ __forceinline__ int pt_cost(const PtItem& x) { return kPtItemCost + x.tiles * pt_tile_cost(x); }

__device__ __forceinline__ long long warp_sum_ll(long long v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// The items of [at, end) of the dealt-out cost, in order, as one warp walks them.
struct PtWalk {
  int b, g, j;
  long long at, end;       // where item (b, g, j) begins; the share's end
  long long begin, last_tile;   // last_tile: where the item's last tile begins
  PtSeq seq;
  __device__ __forceinline__ bool next(const PagesParams& p, PtItem& x) {
    while (at < end) {
      if (j >= seq.blocks) {
        j = 0;
        if (++g >= p.G) {
          g = 0;
          if (++b >= p.B) return false;   // never, unless the lengths change under the call
          seq = pt_seq(p, b);
          while (seq.blocks == 0) {
            // the next sequence with rows, 32 at a look
            const int lane = threadIdx.x & 31;
            const unsigned some = __ballot_sync(0xffffffffu, b + lane < p.B && pt_seq(p, b + lane).blocks > 0);
            if (some) seq = pt_seq(p, b += __ffs(some) - 1);
            else if ((b += 32) >= p.B) return false;
          }
        }
      }
      pt_block(p, seq, j, x);
      x.b = b; x.gh = g;
      const int cost = pt_cost(x), w = pt_tile_cost(x);
      // a tile belongs to the CTA whose share its cost begins in
      const long long lo = begin - at - kPtItemCost, hi = end - at - kPtItemCost;
      x.t_lo = (int)max(0ll, min((long long)x.tiles, (lo + w - 1) / w));
      x.t_hi = (int)max(0ll, min((long long)x.tiles, (hi + w - 1) / w));
      x.whole = x.t_lo == 0 && x.t_hi == x.tiles;
      last_tile = at + kPtItemCost + (long long)(x.tiles - 1) * w;
      at += cost;
      ++j;
      if (x.t_lo < x.t_hi) return true;
    }
    return false;
  }
};

__device__ __forceinline__ uint4 pt_lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
        "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
// Columns of this thread's row, waited for: the load and its wait are one, so that the registers
// are not touched in between.
__device__ __forceinline__ void tmem_ld16_now(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_ld64_now(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, "
      "%22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32, %33, %34, %35, %36, %37, %38, %39, %40, %41, "
      "%42, %43, %44, %45, %46, %47, %48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, "
      "%62, %63}, [%64];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]),
        "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]),
        "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]),
        "=r"(r[48]), "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]),
        "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_ld32_now(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, "
      "%22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// The second product: A in tensor memory (row = lane, two halves of K per 32-bit column).
__device__ __forceinline__ void tcgen05_mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                               uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// kind::f16 instruction descriptor: half x half -> f32, M 128, A K-major.
__host__ __device__ constexpr uint32_t pt_idesc(int n, bool b_n_major) {
  return (1u << 4) | ((b_n_major ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// Two f32 fused multiply-adds, and two sums, in one instruction each.
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float2 unpair(uint64_t x) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(x));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// A row's factor times a page's key scale; never zero, or a masked score, -inf, would become NaN.
__device__ __forceinline__ float score_factor(float row, uint32_t key_scale) {
  return fmaxf(row * __uint_as_float(key_scale), 1.17549435e-38f);
}
// Sixteen codes -> sixteen halves.
__device__ __forceinline__ void halves16(const uint4& c, uint4& lo, uint4& hi) {
  lo = make_uint4(e4m3x2_to_half2(c.x), e4m3x2_hi_to_half2(c.x), e4m3x2_to_half2(c.y), e4m3x2_hi_to_half2(c.y));
  hi = make_uint4(e4m3x2_to_half2(c.z), e4m3x2_hi_to_half2(c.z), e4m3x2_to_half2(c.w), e4m3x2_hi_to_half2(c.w));
}

template <int D>
__global__ void __launch_bounds__(kPtThreads, 1) mha_pages_tc_kernel(const PagesParams p) {
  using Cfg = PtCfg<D>;
  extern __shared__ uint8_t pt_smem_raw[];
  __shared__ long long s_sum[kPtThreads / 32];
  __shared__ int s_b, s_g, s_j, s_nan;
  __shared__ long long s_at;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(pt_smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Cfg::kBars);
  uint64_t* k_full = bars;                          // [kStages]
  uint64_t* k_empty = k_full + Cfg::kStages;
  uint64_t* v_full = k_empty + Cfg::kStages;
  uint64_t* v_empty = v_full + Cfg::kStages;
  uint64_t* q_full = v_empty + Cfg::kStages;        // [2] each: one a half of the columns
  uint64_t* s_full = q_full + 2;                    // [2][2]: of a half's two buffers
  uint64_t* p_full = s_full + 4;                    // [2][2]
  uint64_t* o_full = p_full + 4;                    // [2][2]: a step's product is done, by the buffer its P lay in
  uint64_t* o_free = o_full + 4;                    // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(o_free + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  uint64_t* item_full = o_free + 3;                 // [kPtSlots] each (behind the two words above)
  uint64_t* item_empty = item_full + kPtSlots;
  uint64_t* scale_full = item_empty + kPtSlots;     // [kPtScales]
  PtItem* items = reinterpret_cast<PtItem*>(smem + Cfg::kItems);
  constexpr int kWarps = kPtThreads / 32;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  // the barriers are set up by the warp that has no role, before and beside what the others look up
  if (tid == kPtThreads - 32) {
    for (int s = 0; s < Cfg::kStages; ++s) {
      mbar_init(k_full + s, 128); mbar_init(k_empty + s, 2); mbar_init(v_full + s, 128); mbar_init(v_empty + s, 2);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(q_full + i, 128);
      for (int k = 0; k < 2; ++k) {
        mbar_init(s_full + 2 * i + k, 1); mbar_init(p_full + 2 * i + k, 128); mbar_init(o_full + 2 * i + k, 1);
      }
      mbar_init(o_free + i, 128);
    }
    for (int s = 0; s < kPtSlots; ++s) { mbar_init(item_full + s, 1); mbar_init(item_empty + s, kPtRoles); }
    for (int s = 0; s < kPtScales; ++s) mbar_init(scale_full + s, 4);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  pdl_wait();
  // ---- where this CTA's share begins: a warp sums a stretch of the sequences, 32 at a look ----
  const int per_warp = (p.B + kWarps - 1) / kWarps;
  const int sb = min(warp * per_warp, p.B), se = min(sb + per_warp, p.B);
  auto seq_at = [&](int b) {
    PtSeq s = {};
    if (b < se) s = pt_seq(p, b);
    return s;
  };
  // every lane its sequence's cost of one KV head: one block is the lane's own to count, more are the warp's
  auto costs = [&](const PtSeq& s) {
    PtItem x;
    long long own = 0;
    if (s.blocks == 1) { pt_block(p, s, 0, x); own = pt_cost(x); }
    for (unsigned left = __ballot_sync(0xffffffffu, s.blocks > 1); left; left &= left - 1) {
      const int l = __ffs(left) - 1;
      PtSeq y = {};
      y.len = __shfl_sync(0xffffffffu, s.len, l);
      y.n = __shfl_sync(0xffffffffu, s.n, l);
      y.blocks = __shfl_sync(0xffffffffu, s.blocks, l);
      long long c = 0;
      for (int j = lane; j < y.blocks; j += 32) { pt_block(p, y, j, x); c += pt_cost(x); }
      c = warp_sum_ll(c);
      if (lane == l) own = c;
    }
    return own;
  };
  // sums over the lanes up to and with one's own
  auto upto_lane = [&](long long v) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += y;
    }
    return v;
  };
  long long mine = 0;
  for (int b0 = sb; b0 < se; b0 += 32) mine += costs(seq_at(b0 + lane));
  mine = warp_sum_ll(mine) * p.G;
  if (lane == 0) s_sum[warp] = mine;
  if (tid == 0) { s_nan = s_b = s_g = s_j = 0; s_at = 0; p.records[blockIdx.x].pieces = 0; }
  __syncthreads();
  const long long warp_sum = lane < kWarps ? s_sum[lane] : 0, upto_warp = upto_lane(warp_sum);
  const long long before = __shfl_sync(0xffffffffu, upto_warp - warp_sum, warp), total = __shfl_sync(0xffffffffu, upto_warp, 31);
  const long long share = max((long long)kPtMinShare, div_ll(total + gridDim.x - 1, gridDim.x));
  const long long begin = (long long)blockIdx.x * share, end = min(begin + share, total);
  if (begin >= end) return;
  if (begin >= before && begin < before + mine) {
    long long acc = before;
    for (int b0 = sb; b0 < se; b0 += 32) {
      PtSeq s = seq_at(b0 + lane);
      const long long own = costs(s), upto = upto_lane(own * p.G);
      const unsigned hit = __ballot_sync(0xffffffffu, begin < acc + upto);
      if (!hit) { acc += __shfl_sync(0xffffffffu, upto, 31); continue; }
      const int l = __ffs(hit) - 1;
      const long long one = __shfl_sync(0xffffffffu, own, l);
      acc += __shfl_sync(0xffffffffu, upto, l) - one * p.G;
      const int g = (int)(one >> 31 ? (begin - acc) / one : div_ll(begin - acc, (int)one));
      acc += one * g;
      s = pt_seq(p, b0 + l);
      for (int j0 = 0; j0 < s.blocks; j0 += 32) {
        PtItem x;
        int cost = 0;
        if (j0 + lane < s.blocks) { pt_block(p, s, j0 + lane, x); cost = pt_cost(x); }
        const long long so_far = upto_lane(cost);
        const unsigned in = __ballot_sync(0xffffffffu, cost > 0 && begin < acc + so_far);
        if (in) {
          if (lane == __ffs(in) - 1) { s_b = b0 + l; s_g = g; s_j = j0 + lane; s_at = acc + so_far - cost; }
          break;
        }
        acc += __shfl_sync(0xffffffffu, so_far, 31);
      }
      break;
    }
  }
  if (warp == 16) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem = *tmem_slot;
  // Successors may start only now: one that takes tensor memory before its own wait must not find a CTA
  // here that still asks for its columns, or each would wait for the other.
  pdl_launch();

  bool ok = true;
  // The next item, from the ring that warp 18 fills; `take` copies what the role needs of it.
  int slot = 0;
  uint32_t slot_phase = 0;
  auto next_item = [&](auto&& take) {
    ok = ok && mbar_wait(item_full + slot, slot_phase, abort_flag);
    ok = __all_sync(0xffffffffu, ok);
    if (!ok) return false;
    const PtItem& x = items[slot];
    const bool more = x.cols > 0;
    if (more) take(x);
    __syncwarp();
    if (lane == 0) mbar_arrive(item_empty + slot);
    if (++slot == kPtSlots) { slot = 0; slot_phase ^= 1; }
    return more;
  };

  // registers: 96 a thread at launch (5 x 96 = 480), dealt out anew: 2 x 128 + 2 x 80 + 64
  if (warp >= 16) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
    // ---------------- MMA issuers: the warp walks, an elected lane issues ----------------
    const int i = warp - 16;
    if (warp == 18) {
      // ---------------- the share's items, in order (warp 19 makes the group whole) ----------------
      PtWalk walk;
      walk.b = s_b; walk.g = s_g; walk.j = s_j; walk.at = s_at; walk.begin = begin; walk.end = end;
      walk.seq = pt_seq(p, walk.b);
      PtItem x;
      bool more = true;
      for (int n = 0; more; ++n) {
        more = walk.next(p, x);
        if (!more) x.cols = 0;
        const int at = n % kPtSlots;
        ok = mbar_wait_relaxed(item_empty + at, ((n / kPtSlots) & 1) ^ 1, abort_flag);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        if (lane == 0) {
          items[at] = x;
          if (more && !x.whole && x.t_lo == 0) {
            PagesRecord rec;
            rec.pieces = (int)div_ll(walk.last_tile, (int)min(share, 0x7fffffffll)) - (int)blockIdx.x + 1;
            rec.row0 = x.row0; rec.head0 = x.gh * p.hg; rec.col0 = x.col0;
            rec.cols = x.cols;
            p.records[blockIdx.x] = rec;
          }
          mbar_arrive(item_full + at);
        }
        __syncwarp();
      }
    }
    int cols = 0, n = 0;
    auto take = [&](const PtItem& x) { cols = x.cols; n = x.t_hi - x.t_lo; };
    constexpr uint32_t idesc_s = pt_idesc(64, false), idesc_o = pt_idesc(D, true);
    const uint64_t q_desc = make_desc(smem_u32(smem + Cfg::kQ + i * Cfg::kTile), 16, 1024);
    const uint64_t k_desc0 = make_desc(smem_u32(smem + Cfg::kK), 16, 1024);
    const uint64_t v_desc0 = make_desc(smem_u32(smem + Cfg::kV), kPtSub, 1024);
    const uint32_t s_col = tmem + Cfg::kColS + i * 128, o_col = tmem + Cfg::kColO + i * D;
    // A tile goes in two steps of 64 keys: while a step's exponentials are taken, the next one's
    // scores are computed into the other buffer.  t, t_s: steps of this half so far, and scores issued.
    int ks = 0, vs = 0, n_item = 0, t = 0, t_s = 0;
    uint32_t kp = 0, vp = 0;
    auto next_k = [&]() { if (++ks == Cfg::kStages) { ks = 0; kp ^= 1; } };
    auto next_v = [&]() { if (++vs == Cfg::kStages) { vs = 0; vp ^= 1; } };
    auto issue_s = [&]() {
      const int sub = t_s & 1;
      if (sub == 0 && !mbar_wait(k_full + ks, kp, abort_flag)) return false;
      __syncwarp();
      tcgen05_fence_after();
      if (elect_one()) {
        const uint64_t k_desc = k_desc0 + (uint64_t)((ks * Cfg::kTile + sub * 64 * 128) >> 4);
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint64_t off = (uint64_t)((k >> 2) * (kPtSub >> 4) + (k & 3) * 2);
          tcgen05_mma_bf16(s_col + sub * 64, q_desc + off, k_desc + off, idesc_s, k != 0);
        }
        if (sub) tcgen05_commit(k_empty + ks);
        tcgen05_commit(s_full + 2 * i + sub);
      }
      __syncwarp();
      if (sub) next_k();
      ++t_s;
      return true;
    };
    auto o_done = [&](int step) { return mbar_wait(o_full + 2 * i + (step & 1), (step >> 1) & 1, abort_flag); };
    while (i < 2 && next_item(take)) {
      if (cols <= i * 128) {
        // nothing for this half: the tiles are the other's alone
        for (int u = 0; u < n && ok; ++u) {
          ok = mbar_wait(k_full + ks, kp, abort_flag) && mbar_wait(v_full + vs, vp, abort_flag);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          if (lane == 0) {
            mbar_arrive(k_empty + ks);
            mbar_arrive(v_empty + vs);
          }
          next_k(); next_v();
        }
        continue;
      }
      // the softmax's threads have written Q; the last item's last product has read P
      ok = mbar_wait(q_full + i, n_item & 1, abort_flag) && (t == 0 || o_done(t - 1)) && issue_s() && issue_s();
      ok = __all_sync(0xffffffffu, ok);
      // the last item's outputs have been read
      if (ok && n_item > 0) ok = mbar_wait(o_free + i, (n_item - 1) & 1, abort_flag);
      ok = __all_sync(0xffffffffu, ok);
      ++n_item;
      for (int u = 0; u < 2 * n && ok; ++u, ++t) {
        const int sub = u & 1;
        ok = (sub || mbar_wait(v_full + vs, vp, abort_flag)) && mbar_wait(p_full + 2 * i + sub, (t >> 1) & 1, abort_flag);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tcgen05_fence_after();
        if (elect_one()) {
          const uint64_t v_desc = v_desc0 + (uint64_t)((vs * Cfg::kTile + sub * 64 * 128) >> 4);
#pragma unroll
          for (int k = 0; k < 4; ++k)
            tcgen05_mma_ts(o_col, s_col + sub * 64 + 32 + k * 8, v_desc + (uint64_t)((k * 16 * 128) >> 4), idesc_o,
                           u > 0 || k != 0);
          if (sub) tcgen05_commit(v_empty + vs);
          tcgen05_commit(o_full + 2 * i + sub);
        }
        __syncwarp();
        if (sub) next_v();
        if (u + 2 < 2 * n) {
          // the scores after the next take this step's place: the product that reads its P must be done
          ok = o_done(t) && issue_s();
          ok = __all_sync(0xffffffffu, ok);
        }
      }
    }
  } else if (warp >= 8) {
    // ---------------- converters: warps 8..11 the keys, 12..15 the values ----------------
    asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
    // A thread has a 16-code piece of some rows.  A load instruction takes whole rows; eight
    // lanes in a row, which store together, have four pieces of one sub-tile and two rows that
    // differ in the swizzle's lowest bit, so their 16-byte stores meet on no bank.
    constexpr int kPieces = D / 16, kRowsAtOnce = 32 / kPieces, kReps = 32 / kRowsAtOnce;
    const bool values = warp >= 12;
    const int w = warp & 3;
    const int piece = (lane & 3) + (D == 128 ? (lane >> 3 & 1) * 4 : 0);
    const int sub_row = (lane >> 2 & 1) + (D == 128 ? (lane >> 4) * 2 : (lane >> 3) * 2);
    uint64_t* full = values ? v_full : k_full;
    uint64_t* empty = values ? v_empty : k_empty;
    uint8_t* tiles = smem + (values ? Cfg::kV : Cfg::kK);
    // What is kept of a tile beside its codes, in few registers: the rows that some column sees
    // [lo, hi), whether some column does not see all of them, and where this lane's 16 keys begin in their
    // page (in sixteens).
    auto tile_word = [](int lo, int hi, bool partial, int off) { return lo | hi << 8 | (partial ? 1 << 16 : 0) | off << 17; };
    PtItem it;
    int t_at = 0;
    bool have_item = false;
    auto take = [&](const PtItem& x) { it = x; };
    int entry = -1, word = 0;      // of the next tile: this lane's page id, then its unit in the pool
    auto advance = [&]() {         // the next tile of the share; false at its end
      while (!have_item || t_at >= it.t_hi) {
        if (!next_item(take)) return false;
        have_item = true;
        t_at = it.t_lo;
      }
      const int key0 = (it.tile0 + t_at) * kPtKeys;
      const int key = key0 + 32 * w + 16 * (lane & 1);      // even lanes: the warp's first 16 keys
      entry = -1;
      if (key < it.any_hi) entry = p.tables[(long long)it.b * p.width + (key >> p.log_page)];
      word = tile_word(max(it.any_lo - key0, 0), min(max(it.any_hi - key0, 0), kPtKeys),
                       key0 < it.all_lo || key0 + kPtKeys > it.all_hi, (key & ((1 << p.log_page) - 1)) >> 4);
      ++t_at;
      return true;
    };
    uint4 codes[kReps];
    // byte offsets of this thread's two 16-byte chunks: the swizzle's rows repeat every eight
    const int at0 = (piece >> 2) * kPtSub + (32 * w + sub_row) * 128, chunk = 2 * (piece & 3);
    const uint8_t* my_codes = p.pool + sub_row * D + piece * 16;
    // A tile's page ids come as the index of a 16-token unit of one page, KV head and kind.
    auto load = [&]() {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int unit = __shfl_sync(0xffffffffu, entry, half);
        const uint8_t* base = my_codes + (long long)max(unit, 0) * (16 * D);
#pragma unroll
        for (int k = 0; k < kReps / 2; ++k)
          codes[half * (kReps / 2) + k] = unit >= 0 ? ld_stream(base + k * kRowsAtOnce * D) : make_uint4(0, 0, 0, 0);
      }
    };
    float2 scale = make_float2(1.f, 0.f);
    auto unit_of = [&]() {
      const bool there = entry >= 0 && entry < p.P;
      // an absent page: finite scores are -inf through the logarithm, its share of the sum nothing; an inverse of 0 marks it
      scale = make_float2(1.f, 0.f);
      if (!values && there && lane < 2)
        scale = *reinterpret_cast<const float2*>(p.scales + ((long long)entry * p.G + it.gh) * 2);
      entry = there ? (((entry * p.G + it.gh) * 2 + (values ? 1 : 0)) << (p.log_page - 4)) + (word >> 17) : -1;
    };
    auto store = [&](uint8_t* tile, int k, const uint4& c) {
      const int row7 = (k * kRowsAtOnce + sub_row) & 7;
      uint8_t* dst = tile + at0 + k * kRowsAtOnce * 128;
      uint4 lo, hi;
      halves16(c, lo, hi);
      *reinterpret_cast<uint4*>(dst + ((chunk ^ row7) << 4)) = lo;
      *reinterpret_cast<uint4*>(dst + (((chunk + 1) ^ row7) << 4)) = hi;
    };
    int now = 0;                // the word of the tile whose codes are held
    bool have = advance(), more = false;
    if (have) {
      unit_of();
      load();
      now = word;
      more = advance();         // its page ids are there by the time its loads begin
    }
    int s = 0, n_tile = 0;
    uint32_t ph = 0;
    while (have) {
      ok = mbar_wait_relaxed(empty + s, ph ^ 1, abort_flag, 64);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      if (values && (now >> 16 & 1)) {
        // values that no column sees count as zero; a NaN that some see is zero here and comes
        // back where it is seen when the outputs are written
#pragma unroll
        for (int k = 0; k < kReps; ++k) {
          const int row = 32 * w + k * kRowsAtOnce + sub_row;
          uint32_t* c = reinterpret_cast<uint32_t*>(&codes[k]);
          if (row < (now & 0xff) || row >= (now >> 8 & 0xff)) codes[k] = make_uint4(0, 0, 0, 0);
          if (nan_codes(c[0]) | nan_codes(c[1]) | nan_codes(c[2]) | nan_codes(c[3])) {
#pragma unroll
            for (int q = 0; q < 4; ++q) c[q] &= ~((nan_codes(c[q]) >> 7) * 0xffu);
            *reinterpret_cast<volatile int*>(&s_nan) = 1;
          }
        }
      }
      if (!values) {
        // the key scale, the logarithm of the value scale, its inverse: what the softmax asks for
        const int at = n_tile++ % kPtScales;
        if (lane < 2)
          reinterpret_cast<float4*>(smem + Cfg::kScale)[at * 8 + 2 * w + lane] =
              make_float4(scale.x, __log2f(scale.y), scale.y > 0.f ? __frcp_rn(scale.y) : 0.f, 0.f);
        __syncwarp();
        if (lane == 0) mbar_arrive(scale_full + at);
      }
      uint8_t* tile = tiles + s * Cfg::kTile;
#pragma unroll
      for (int k = 0; k < kReps; ++k) store(tile, k, codes[k]);
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      mbar_arrive(full + s);
      if (more) {
        unit_of();
        load();
      }
      if (++s == Cfg::kStages) { s = 0; ph ^= 1; }
      now = word;
      have = more;
      if (more) more = advance();
    }
  } else {
    // ---------------- softmax and output ----------------
    asm volatile("setmaxnreg.inc.sync.aligned.u32 128;");
    const int i = warp >> 2;                      // which 128 columns
    const int r = (warp & 3) * 32 + lane;
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t s_col = lanes + Cfg::kColS + i * 128, o_col = lanes + Cfg::kColO + i * D;
    uint8_t* q_row = smem + Cfg::kQ + i * Cfg::kTile + r * 128;
    int t = 0, n_tile = 0;                        // steps of this half, and tiles of the share, so far
    PtItem it;
    // what a thread keeps of its column
    struct Row { long long out_at; float factor; int hi_key, lo_key; bool live; } me;
    auto take = [&](const PtItem& x) { it = x; };
    // The next item with columns for this half, and its queries: halves under a power of two that
    // puts the row's largest in [2^14, 2^15).  The last item's scores have been computed, so Q's
    // place is free; its outputs may still be to come.
    auto open_item = [&]() {
      for (;;) {
        if (!next_item(take)) return false;
        if (it.cols > i * 128) break;
        n_tile += it.t_hi - it.t_lo;
      }
      const int c = it.col0 + i * 128 + r;        // column of the sequence and KV head
      const int row = c / p.hg, h = c - row * p.hg, pos = it.past + row;
      me.live = i * 128 + r < it.cols;
      me.hi_key = me.live ? (p.causal ? min(it.len, pos + 1) : it.len) : 0;
      me.lo_key = p.window >= 0 ? pos - p.window : 0;
      me.out_at = ((long long)(it.row0 + row) * p.H + it.gh * p.hg + h) * D;
      const uint4* src = reinterpret_cast<const uint4*>(p.q + me.out_at);
      uint4 raw[D / 8];
#pragma unroll
      for (int k = 0; k < D / 8; ++k) raw[k] = me.live ? ld_cached(src + k) : make_uint4(0, 0, 0, 0);
      // the largest magnitude, two elements at a time: bf16 magnitudes order as their bits do
      uint32_t top = 0;
#pragma unroll
      for (int k = 0; k < D / 8; ++k) {
        const uint32_t* w = reinterpret_cast<const uint32_t*>(&raw[k]);
#pragma unroll
        for (int q = 0; q < 4; ++q) top = __vmaxu2(top, w[q] & 0x7fff7fffu);
      }
      const float mx = __uint_as_float(max(top & 0xffffu, top >> 16) << 16);
      const int e = min(max((int)(__float_as_uint(mx) >> 23), 15), 254);
      const float up = __uint_as_float((uint32_t)(268 - e) << 23);
      me.factor = p.scale_log2 / up;
      // The logarithm of an absent page's scale masks finite scores, but a query that is not finite times the
      // page's zeros is NaN.  Where a row of this warp has one, the warp takes the careful way.
      if (__any_sync(0xffffffffu, mx == INFINITY || mx != mx)) it.all_hi = ~it.all_hi;
#pragma unroll
      for (int k = 0; k < D / 8; ++k) {
        float f[8];
        unpack8(raw[k], f);
        *reinterpret_cast<uint4*>(q_row + (k >> 3) * kPtSub + (((k & 7) ^ (r & 7)) << 4)) =
            make_uint4(pack_half2(f[0] * up, f[1] * up), pack_half2(f[2] * up, f[3] * up),
                       pack_half2(f[4] * up, f[5] * up), pack_half2(f[6] * up, f[7] * up));
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      mbar_arrive(q_full + i);
      return true;
    };
    // 64 bytes of each lane's row in: 16 bytes of rows 8 k + lane / 4 out, k = 0 .. 3.
    auto turn_rows = [&](uint32_t* o) {
      uint8_t* mine = smem + Cfg::kOut + warp * 32 * kPtPitch;
      __syncwarp();
#pragma unroll
      for (int k = 0; k < 4; ++k)
        *reinterpret_cast<uint4*>(mine + lane * kPtPitch + k * 16) = make_uint4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
      __syncwarp();
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint4 x = *reinterpret_cast<const uint4*>(mine + (8 * k + (lane >> 2)) * kPtPitch + (lane & 3) * 16);
        o[4 * k] = x.x; o[4 * k + 1] = x.y; o[4 * k + 2] = x.z; o[4 * k + 3] = x.w;
      }
    };
    bool have = open_item();
    while (have) {
      float factor = it.all_hi < 0 ? 1.f : me.factor;
      const int hi_key = me.hi_key, lo_key = me.lo_key;
      float base = kPtNone, l = 0.f;   // the maximum in use less the lift
      // The careful way, of a warp that has a query that is not finite or a score past kPtFar: no key counts as
      // seen by all (the bound is kept as its complement), so that every step passes the masks, where
      // absent pages (an inverse of 0) are masked too and scores are rounded before the maximum is taken
      // off; a fused product and difference would be off by the score's own rounding, 2^2 and far more.

      for (int u = 2 * it.t_lo; u < 2 * it.t_hi && ok; ++u, ++t) {
        const int sub = u & 1, buf = 2 * i + sub;
        const uint32_t col = s_col + sub * 64;
        const uint32_t sc_at = smem_u32(smem + Cfg::kScale) + (n_tile % kPtScales) * 128 + sub * 64;
        const int key0 = it.tile0 * kPtKeys + u * 64;
        ok = (sub || mbar_wait(scale_full + n_tile % kPtScales, (n_tile / kPtScales) & 1, abort_flag)) &&
             mbar_wait(s_full + buf, (t >> 1) & 1, abort_flag);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        if (sub) ++n_tile;
        tcgen05_fence_after();
        uint32_t v[64];
        tmem_ld64_now(col, v);
        // (key scale, log2 of the value scale, its inverse) of each 16 keys
        uint4 f[4] = {pt_lds128(sc_at), pt_lds128(sc_at + 16), pt_lds128(sc_at + 32), pt_lds128(sc_at + 48)};
        if (key0 < it.all_lo || key0 + 64 > it.all_hi) {
#pragma unroll
          for (int k = 0; k < 64; ++k)
            if (key0 + k >= hi_key || key0 + k < lo_key) v[k] = 0xff800000u;   // this column does not see the key
          if (__builtin_expect(it.all_hi < 0, 0)) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const float a = score_factor(me.factor, f[q].x);
#pragma unroll
              for (int k = 0; k < 16; ++k)
                v[16 * q + k] = f[q].z == 0 ? 0xff800000u : __float_as_uint(fmaf(__uint_as_float(v[16 * q + k]), a, __uint_as_float(f[q].y)));
              f[q].x = 0x3f800000u; f[q].y = 0;
            }
          }
        }
        // ---- the maximum ----
        float mx = -INFINITY;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          float top = fmaxf(__uint_as_float(v[16 * q]), __uint_as_float(v[16 * q + 1]));
#pragma unroll
          for (int k = 2; k < 16; k += 2) top = max3(top, __uint_as_float(v[16 * q + k]), __uint_as_float(v[16 * q + k + 1]));
          mx = fmaxf(mx, fmaf(top, score_factor(factor, f[q].x), __uint_as_float(f[q].y)));
        }
        if (__any_sync(0xffffffffu, mx - base > kPtLift + kPtSlack)) {
          const bool far = fabsf(mx) > kPtFar && mx != -INFINITY;
          if (it.all_hi >= 0 && __any_sync(0xffffffffu, far)) {   // this step once more: its scores still lie there
            it.all_hi = ~it.all_hi;
            factor = 1.f;
            --u; --t;
            if (sub) --n_tile;
            continue;
          }
          const float base_new = fmaxf(base, far ? mx : mx - kPtLift);   // a far one takes no lift: it would not come out whole
          const float corr = ex2(base - base_new);
          base = base_new;
          l *= corr;
          if (u > 2 * it.t_lo) {
            // once the last step's product is done the outputs lie still: this step's waits for P.
            // (These scores took the place of the step before's P: its product is done.)
            ok = mbar_wait(o_full + 2 * i + ((t - 1) & 1), ((t - 1) >> 1) & 1, abort_flag);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            tcgen05_fence_after();
#pragma unroll 1
            for (int q = 0; q < D / 16; ++q) {
              uint32_t o[16];
              tmem_ld16_now(o_col + q * 16, o);
#pragma unroll
              for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * corr);
              tmem_st16(o_col + q * 16, o);
            }
          }
        }
        // ---- weights and their sum: P over the scores' place ----
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          uint32_t out[16];
#pragma unroll
          for (int qq = 0; qq < 2; ++qq) {
            const int q = 2 * half + qq;
            const float a = score_factor(factor, f[q].x), b = __uint_as_float(f[q].y) - base;
            const uint64_t a2 = pair(a, a), b2 = pair(b, b);
            uint64_t sum[2] = {0, 0};
#pragma unroll
            for (int k = 0; k < 16; k += 2) {
              const float2 y = unpair(fma2(pair(__uint_as_float(v[16 * q + k]), __uint_as_float(v[16 * q + k + 1])), a2, b2));
              const float p0 = ex2(y.x), p1 = ex2(y.y);
              sum[(k >> 1) & 1] = add2(sum[(k >> 1) & 1], pair(p0, p1));
              out[qq * 8 + k / 2] = pack_half2(p0, p1);
            }
            const float2 total = unpair(add2(sum[0], sum[1]));
            l = fmaf(total.x + total.y, __uint_as_float(f[q].z), l);
          }
          tmem_st16(col + 32 + half * 16, out);
        }
        tmem_st_wait();
        tcgen05_fence_before();
        mbar_arrive(p_full + buf);
      }
      if (!ok) break;
      // ---- the next item's queries go first, then this one's results ----
      const PtItem done = it;
      const Row was = me;
      const int last = t - 1;
      have = open_item();
      ok = ok && mbar_wait(o_full + 2 * i + (last & 1), (last >> 1) & 1, abort_flag);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tcgen05_fence_after();
      float* part = p.partial + ((long long)blockIdx.x * 2 + (done.t_lo == 0 ? 1 : 0)) * Cfg::kPartial;
      const bool nans = *reinterpret_cast<volatile int*>(&s_nan) != 0;
      const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll 1
      for (int q = 0; q < D / 32; ++q) {
        uint32_t v[32];
        __syncwarp();
        tmem_ld32_now(o_col + q * 32, v);
        if (q == D / 32 - 1) {
          tcgen05_fence_before();
          mbar_arrive(o_free + i);     // the outputs are read: the next item's may come
        }
        if (nans && was.live) {
          // NaN codes of partial tiles were taken as zero: they are NaN to the rows that see them
          uint32_t hit = 0;
          const int from = max(was.lo_key, (done.tile0 + done.t_lo) * kPtKeys), to = min(was.hi_key, (done.tile0 + done.t_hi) * kPtKeys);
          for (int key = max(from, 0); key < to; ++key) {
            const int k0 = key / kPtKeys * kPtKeys;
            if (k0 >= done.all_lo && k0 + kPtKeys <= max(done.all_hi, ~done.all_hi)) { key = k0 + kPtKeys - 1; continue; }
            const int e = p.tables[(long long)done.b * p.width + (key >> p.log_page)];
            if (e < 0 || e >= p.P) continue;
            const long long block = ((long long)e * p.G + done.gh) * 2 + 1;
            const uint32_t* code = reinterpret_cast<const uint32_t*>(
                p.pool + ((block << p.log_page) + (key & ((1 << p.log_page) - 1))) * D + q * 32);
            for (int k = 0; k < 8; ++k) {
              const uint32_t b = nan_codes(code[k]) >> 7;
              hit |= ((b & 1) | (b >> 7 & 2) | (b >> 14 & 4) | (b >> 21 & 8)) << (4 * k);
            }
          }
#pragma unroll
          for (int k = 0; k < 32; ++k)
            if (hit >> k & 1) v[k] = 0x7fc00000u;
        }
        // A lane has 32 columns of its row; through shared memory four lanes have 64 bytes of one, so
        // that a store instruction writes eight rows' pieces instead of 32 rows'.
        if (done.whole) {
          uint32_t o[16];
#pragma unroll
          for (int k = 0; k < 16; ++k)
            o[k] = l == 0.f ? 0u : pack_bf16x2(__uint_as_float(v[2 * k]) * inv, __uint_as_float(v[2 * k + 1]) * inv);
          turn_rows(o);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const long long at = __shfl_sync(0xffffffffu, was.out_at, 8 * k + (lane >> 2));
            if (__shfl_sync(0xffffffffu, was.live ? 1 : 0, 8 * k + (lane >> 2)))
              *reinterpret_cast<uint4*>(p.out + at + q * 32 + (lane & 3) * 8) = make_uint4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
          }
        } else {
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            uint32_t* o = v + half * 16;
            turn_rows(o);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int row = (warp & 3) * 32 + 8 * k + (lane >> 2);
              if (i * 128 + row < done.cols)
                *reinterpret_cast<uint4*>(part + (i * 128 + row) * D + q * 32 + half * 16 + (lane & 3) * 4) =
                    make_uint4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
            }
          }
        }
      }
      if (was.live && !done.whole) {
        part[kPtRows * D + i * 128 + r] = base == kPtNone ? -INFINITY : base;
        part[kPtRows * D + kPtRows + i * 128 + r] = l;
      }
    }
  }

  if (*abort_flag) {
    // a wait gave up: give what is in flight a millisecond, many times what it takes
    const unsigned long long t0 = global_ns();
    while (global_ns() - t0 < 1000000ull) {}
  }
  tcgen05_fence_before();
  __syncthreads();
  if (tid == 0 && *abort_flag && p.status) *p.status = IRON_ERR_TIMEOUT;
  if (warp == 16) {
    tcgen05_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  }
}

// Folds the partials of an item that several CTAs share, in the order of its keys: one CTA for
// eight columns of each main CTA's record, a warp a column, a lane a stretch of d.
template <int D>
__global__ void __launch_bounds__(kPtFoldWarps * 32) mha_pages_tc_fold_kernel(const PagesParams p) {
  using Cfg = PtCfg<D>;
  constexpr int PER = D / 32, kBatch = 4;
  pdl_launch();
  pdl_wait();
  const PagesRecord r = p.records[blockIdx.x];
  const int lane = threadIdx.x & 31, c = blockIdx.y * kPtFoldWarps + (threadIdx.x >> 5);
  if (r.pieces <= 1 || c >= r.cols) return;
  float m = -INFINITY, l = 0.f, o[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) o[j] = 0.f;
  for (int i0 = 0; i0 < r.pieces; i0 += kBatch) {
    float x[kBatch][PER], mi[kBatch], li[kBatch];
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int i = min(i0 + k, r.pieces - 1);   // past the end: loaded again, not counted
      // the piece that begins the item lies in its CTA's second slot, the others in the first
      const float* src = p.partial + ((long long)(blockIdx.x + i) * 2 + (i == 0 ? 1 : 0)) * Cfg::kPartial;
      mi[k] = src[kPtRows * D + c];
      li[k] = src[kPtRows * D + kPtRows + c];
      const float2* v = reinterpret_cast<const float2*>(src + c * D + lane * PER);
#pragma unroll
      for (int j = 0; j < PER / 2; ++j) { const float2 y = v[j]; x[k][2 * j] = y.x; x[k][2 * j + 1] = y.y; }
    }
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      if (i0 + k >= r.pieces) break;
      const float m_new = fmaxf(m, mi[k]), safe = m_new == -INFINITY ? 0.f : m_new;
      const float f = ex2(m - safe), fi = ex2(mi[k] - safe);
      m = m_new;
      l = l * f + li[k] * fi;
#pragma unroll
      for (int j = 0; j < PER; ++j) o[j] = o[j] * f + x[k][j] * fi;
    }
  }
  const int row = (r.col0 + c) / p.hg, h = (r.col0 + c) - row * p.hg;
  __nv_bfloat16* dst = p.out + ((long long)(r.row0 + row) * p.H + r.head0 + h) * D + lane * PER;
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int j = 0; j < PER; j += 2)
    *reinterpret_cast<uint32_t*>(dst + j) = l == 0.f ? 0u : pack_bf16x2(o[j] * inv, o[j + 1] * inv);
}

long long mha_pages_tc_workspace_bytes(int D) {
  const long long partial = D == 64 ? PtCfg<64>::kPartial : PtCfg<128>::kPartial;
  return kSMs * ((long long)sizeof(PagesRecord) + 2 * partial * (long long)sizeof(float));
}

template <int D>
static int launch_pages_tc(PagesParams p, void* workspace, cudaStream_t stream) {
  p.records = (PagesRecord*)workspace;
  p.partial = (float*)(p.records + kSMs);
  static DeviceOnce configured;
  if (!configured.done()) {
    if (cudaFuncSetAttribute(mha_pages_tc_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, PtCfg<D>::kSmem) !=
        cudaSuccess)
      return IRON_ERR_LAUNCH;
    configured.mark();
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(kSMs);
  cfg.blockDim = dim3(kPtThreads);
  cfg.dynamicSmemBytes = PtCfg<D>::kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  fill_pdl_attr(cfg, attr);
  if (cudaLaunchKernelEx(&cfg, mha_pages_tc_kernel<D>, p) != cudaSuccess) return IRON_ERR_LAUNCH;
  const long long cols = (long long)p.rows * p.hg;
  cfg.gridDim = dim3(kSMs, (unsigned)(((cols < kPtRows ? cols : kPtRows) + kPtFoldWarps - 1) / kPtFoldWarps));
  cfg.blockDim = dim3(kPtFoldWarps * 32);
  cfg.dynamicSmemBytes = 0;
  return cudaLaunchKernelEx(&cfg, mha_pages_tc_fold_kernel<D>, p) == cudaSuccess ? IRON_OK : IRON_ERR_LAUNCH;
}

int mha_pages_tc(const PagesParams& p, int D, void* workspace, cudaStream_t stream) {
  return D == 64 ? launch_pages_tc<64>(p, workspace, stream) : launch_pages_tc<128>(p, workspace, stream);
}

}  // namespace iron
