// Attention over a key/value cache that lies in pages of e4m3 codes, on warp MMAs: one query a
// sequence (a decode step), or the few rows a sequence brings (a draft to verify, a short chunk).
//
// Bound by the cache's bytes, so the kernel is built around reading them once, in order, with
// no staging: a warp's loads ARE the operand fragments.  Scores are computed transposed,
// S^T = K Q^T (16 tokens x 8 query columns an MMA), and so is the output, O^T += V^T P^T, so a
// group of up to eight query heads fills the MMA's narrow side and the codes its wide one:
//   K fragment   lane (g, t) wants tokens g and g + 8, two adjacent elements a register.  Which
//                elements make up "k" is free as long as Q agrees: lane t takes a run of D / 4
//                consecutive codes of its tokens.
//   V fragment   lane (g, t) wants tokens 2t, 2t + 1, 2t + 8, 2t + 9 of "rows" d; it takes the
//                run of D / 8 codes at g * D / 8, and a byte permute pairs two tokens' codes.
//   P            the score fragment holds tokens by rows; movmatrix turns it into the B operand.
// Codes become halves exactly (one conversion a pair).  Q goes to halves too: each row times a
// power of two that puts its largest element in [2^14, 2^15), so that elements down to 2^-31 of it
// keep all their bits.  Scales join outside the products: a page's key scale multiplies its
// scores, and the logarithm of its value scale is added to them, so that what is exponentiated
// is a token's weight on the output, p * scale, under a running maximum of that weight (a maximum of p
// alone would let a heavy page with small p push the others below half's range); the softmax's
// denominator takes the weights over the scale again.  Weights are rounded to half (2^-11), held times
// 2^10, so those down to 2^-24 of the largest keep full precision; scores, maxima, sums and
// outputs are f32.
//
// Work is dealt out by the unit of 16 tokens: the units of all (sequence, KV head, column block)
// segments, end to end, are cut into equal runs, one a CTA, so ragged lengths leave no CTA idle.
// A CTA's four warps take a run's units in turn and merge in shared memory; a segment cut by a CTA
// boundary leaves partials in the workspace, which a second small launch folds in order.
#include "common.cuh"
#include "mma.cuh"
#include "pages.cuh"

namespace iron {

constexpr int kPgWarps = 4;
constexpr int kPgThreads = kPgWarps * 32;
constexpr int kPgCtasPerSm = 3;
constexpr int kPgCtas = kSMs * kPgCtasPerSm;
constexpr int kPgUnit = 16;                 // tokens
constexpr float kPgLift = 10.f;             // log2 of what probabilities are held times

struct PagesParams {
  const __nv_bfloat16* q;
  const uint8_t* pool;
  const float* scales;
  const int* tables;
  const int* lengths;
  const int* row_start;     // nullptr: one query a sequence
  __nv_bfloat16* out;
  float* partial;
  int B, H, G, P, width, log_page, causal, window, rows, ctas;
  float scale_log2;
};

// A sequence as the kernels see it: its keys, its query rows, and the units a segment spans.
struct PagesSeq {
  int len, row0, n, unit0;      // keys, first row, rows, first unit any row may see
  int segs, units;              // segments (KV heads x column blocks) and units each
};

template <int COLS>
__device__ __forceinline__ PagesSeq pages_seq(const PagesParams& p, int b) {
  PagesSeq s;
  s.len = max(0, (int)min((long long)p.lengths[b], (long long)p.width << p.log_page));
  if (p.row_start) {
    s.row0 = min(max(p.row_start[b], 0), p.rows);
    s.n = max(0, min(p.row_start[b + 1], p.rows) - s.row0);
  } else {
    s.row0 = b; s.n = 1;
  }
  const int first = p.window >= 0 ? max(0, s.len - s.n - p.window) : 0;
  s.unit0 = first / kPgUnit;
  const int hg = p.H / p.G;
  s.segs = p.G * (int)(((long long)s.n * hg + COLS - 1) / COLS);
  // an empty segment still has a unit: somebody must write its zeros
  s.units = max(1, (s.len + kPgUnit - 1) / kPgUnit - s.unit0);
  return s;
}

// floats of one partial: COLS x D outputs, then COLS maxima and COLS sums
template <int D, int NT>
struct PgCfg {
  static constexpr int kCols = NT * 8;
  static constexpr int kPartial = kCols * D + 2 * kCols;
};

// units per CTA: an equal share, and two a warp at least
__device__ __forceinline__ long long pages_share(long long total, int ctas) {
  const long long even = (total + ctas - 1) / ctas;
  return even < 2 * kPgWarps ? 2 * kPgWarps : even;
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
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// What a lane holds of one unit: K codes of two tokens, V codes of four.
template <int D>
struct PgUnit {
  uint32_t k[2][D / 16];    // D / 4 bytes of tokens g and g + 8
  uint32_t v[4][D / 32];    // D / 8 bytes of tokens 2t, 2t + 1, 2t + 8, 2t + 9
  float2 scale;             // keys, values; NaN-free: an absent page is masked as a whole
  bool present;
};

template <int D>
__device__ __forceinline__ void load_unit(PgUnit<D>& u, const PagesParams& p, int entry, int g_head, int off, int lane) {
  u.present = entry >= 0 && entry < p.P;
  const long long block = (long long)(u.present ? entry : 0) * p.G + g_head;
  const uint8_t* k = p.pool + ((block * 2) << p.log_page) * D + (long long)off * D;
  const uint8_t* v = k + ((long long)D << p.log_page);
  const int g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int c = 0; c < D / 64; ++c) {
      const uint4 x = ld_stream(k + (g + 8 * i) * D + t * (D / 4) + c * 16);
      u.k[i][4 * c] = x.x; u.k[i][4 * c + 1] = x.y; u.k[i][4 * c + 2] = x.z; u.k[i][4 * c + 3] = x.w;
    }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint8_t* src = v + (2 * t + (i & 1) + (i >> 1) * 8) * D + g * (D / 8);
    if (D == 128) {
      const uint4 x = ld_stream(src);
      u.v[i][0] = x.x; u.v[i][1] = x.y; u.v[i][D / 32 - 2] = x.z; u.v[i][D / 32 - 1] = x.w;
    } else {
      asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(u.v[i][0]), "=r"(u.v[i][1]) : "l"(src));
    }
  }
  u.scale = *reinterpret_cast<const float2*>(p.scales + block * 2);
}

// bit 7 of a byte set where the code is NaN (0x7f or 0xff)
__device__ __forceinline__ uint32_t nan_codes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

template <int D, int NT>
__global__ void __launch_bounds__(kPgThreads, kPgCtasPerSm) mha_pages_kernel(const PagesParams p) {
  using Cfg = PgCfg<D, NT>;
  constexpr int COLS = Cfg::kCols;
  constexpr int KS = D / 16;                    // MMAs along d of a score
  __shared__ float s_o[kPgWarps][COLS * D / 4];   // a quarter of d at a time
  __shared__ float s_m[kPgWarps][COLS], s_l[kPgWarps][COLS], s_w[kPgWarps][COLS];
  __shared__ long long s_scan[kPgThreads];
  __shared__ int s_b;
  __shared__ long long s_at;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int hg = p.H / p.G, page_mask = (1 << p.log_page) - 1;

  pdl_launch();
  pdl_wait();
  // where this CTA's run of units begins: every thread sums a stretch of the sequences
  const int per_thread = (p.B + kPgThreads - 1) / kPgThreads;
  const int sb = min(tid * per_thread, p.B), se = min(sb + per_thread, p.B);
  long long mine = 0;
  for (int b = sb; b < se; ++b) {
    const PagesSeq s = pages_seq<COLS>(p, b);
    mine += (long long)s.segs * s.units;
  }
  s_scan[tid] = mine;
  __syncthreads();
  long long before = 0, total = 0;
  for (int i = 0; i < kPgThreads; ++i) {
    const long long x = s_scan[i];
    if (i < tid) before += x;
    total += x;
  }
  const long long share = pages_share(total, p.ctas);
  long long at = (long long)blockIdx.x * share;
  const long long end = min(at + share, total);
  if (at >= end) return;
  if (at >= before && at < before + mine) {
    long long acc = before;
    for (int b = sb; b < se; ++b) {
      const PagesSeq s = pages_seq<COLS>(p, b);
      const long long w = (long long)s.segs * s.units;
      if (at < acc + w) { s_b = b; s_at = acc; break; }
      acc += w;
    }
  }
  __syncthreads();
  int b = s_b;
  long long seq_at = s_at;      // unit index where sequence b begins
  PagesSeq seq = pages_seq<COLS>(p, b);

  while (at < end) {
    while (at >= seq_at + (long long)seq.segs * seq.units) {
      seq_at += (long long)seq.segs * seq.units;
      seq = pages_seq<COLS>(p, ++b);
    }
    const int seg = (int)((at - seq_at) / seq.units);
    const long long seg_at = seq_at + (long long)seg * seq.units;
    const int u_lo = (int)(at - seg_at), u_hi = (int)(min(end, seg_at + seq.units) - seg_at);
    const int blocks = seq.segs / p.G;
    const int gh = seg / blocks, col0 = (seg % blocks) * COLS;
    const int cols = min(COLS, seq.n * hg - col0);
    const int past = seq.len - seq.n;           // position of the first row
    const int* table = p.tables + (long long)b * p.width;

    // ---- Q: this lane's share of column 8 nt + g, in halves under a power of two ----
    uint32_t qf[NT][KS][2];
    float colfac[NT][2];                        // of columns 8 nt + 2t and + 1
    int hi_key[NT][2], lo_key[NT][2];           // keys those columns see: [lo, hi)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int c = nt * 8 + g;
      const bool live = c < cols;
      const int row = live ? (col0 + c) / hg : 0, h = live ? (col0 + c) % hg : 0;
      const __nv_bfloat16* src = p.q + ((long long)(seq.row0 + row) * p.H + gh * hg + h) * D + t * (D / 4);
      uint4 raw[D / 32];
      float mx = 0.f;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        raw[i] = live ? ld_cached(src + 8 * i) : make_uint4(0, 0, 0, 0);
        float f[8];
        unpack8(raw[i], f);
#pragma unroll
        for (int j = 0; j < 8; ++j) mx = fmaxf(mx, fabsf(f[j]));
      }
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      // mx * up lies in [2^14, 2^15); zero, subnormal and non-finite rows keep finite factors
      const int e = min(max((int)(__float_as_uint(mx) >> 23), 1 + 14), 254);
      const float up = __uint_as_float((uint32_t)(127 + 14 + 127 - e > 254 ? 254 : 127 + 14 + 127 - e) << 23);
      const float down = 1.0f / up;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        float f[8];
        unpack8(raw[i], f);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          qf[nt][2 * i + j][0] = pack_half2(f[4 * j] * up, f[4 * j + 1] * up);
          qf[nt][2 * i + j][1] = pack_half2(f[4 * j + 2] * up, f[4 * j + 3] * up);
        }
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        colfac[nt][j] = __shfl_sync(0xffffffffu, down, (2 * t + j) * 4) * p.scale_log2;
        const int cc = nt * 8 + 2 * t + j;
        const int pos = past + (col0 + min(cc, cols - 1)) / hg;
        hi_key[nt][j] = cc < cols ? (p.causal ? min(seq.len, pos + 1) : seq.len) : 0;
        lo_key[nt][j] = p.window >= 0 ? pos - p.window : 0;
      }
    }
    // the keys every column sees, and any column sees
    int all_hi = seq.len, any_hi = seq.len, all_lo = 0, any_lo = 0;
    if (p.causal) {
      all_hi = min(seq.len, past + col0 / hg + 1);
      any_hi = min(seq.len, past + (col0 + cols - 1) / hg + 1);
    }
    if (p.window >= 0) {
      any_lo = past + col0 / hg - p.window;
      all_lo = past + (col0 + cols - 1) / hg - p.window;
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

    // units any column sees; the rest of the run is masked as a whole
    const int first = max(u_lo, max(any_lo, 0) / kPgUnit - seq.unit0);
    const int last = min(u_hi, (any_hi + kPgUnit - 1) / kPgUnit - seq.unit0);
    auto entry_of = [&](int u) {
      return u < last ? table[min(((seq.unit0 + u) * kPgUnit) >> p.log_page, p.width - 1)] : -1;
    };
    int u = first + warp;
    PgUnit<D> cur;
    int entry = entry_of(u);
    if (u < last) load_unit<D>(cur, p, entry, gh, ((seq.unit0 + u) * kPgUnit) & page_mask, lane);
    entry = entry_of(u + kPgWarps);
    for (; u < last; u += kPgWarps) {
      PgUnit<D> nxt;
      if (u + kPgWarps < last)
        load_unit<D>(nxt, p, entry, gh, ((seq.unit0 + u + kPgWarps) * kPgUnit) & page_mask, lane);
      entry = entry_of(u + 2 * kPgWarps);
      const int tok0 = (seq.unit0 + u) * kPgUnit;
      if (cur.present) {
        // ---- S^T = K Q^T ----
        float s[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
#pragma unroll
        for (int i = 0; i < KS; ++i) {
          const uint32_t a[4] = {e4m3x2_to_half2(cur.k[0][i]), e4m3x2_to_half2(cur.k[1][i]),
                                 e4m3x2_to_half2(cur.k[0][i] >> 16), e4m3x2_to_half2(cur.k[1][i] >> 16)};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma_f16_16816(s[nt], a, qf[nt][i][0], qf[nt][i][1]);
        }
        const bool whole = tok0 + kPgUnit <= all_hi && tok0 >= all_lo;
        const float log_v = __log2f(cur.scale.y), inv_v = 1.f / cur.scale.y;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            s[nt][j] = fmaf(s[nt][j], colfac[nt][j & 1] * cur.scale.x, log_v);
            if (!whole) {
              const int key = tok0 + g + (j >> 1) * 8;
              if (key >= hi_key[nt][j & 1] || key < lo_key[nt][j & 1]) s[nt][j] = -INFINITY;
            }
          }
        // ---- running maximum and sum ----
        uint32_t pb[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float pr[4];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            float m = fmaxf(s[nt][j], s[nt][j + 2]);
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
            const float m_new = fmaxf(m_run[nt][j], m);
            const float safe = m_new == -INFINITY ? 0.f : m_new;
            const float corr = ex2(m_run[nt][j] - safe);
            m_run[nt][j] = m_new;
            pr[j] = ex2(s[nt][j] - safe + kPgLift);
            pr[j + 2] = ex2(s[nt][j + 2] - safe + kPgLift);
            l_run[nt][j] = l_run[nt][j] * corr + (pr[j] + pr[j + 2]) * inv_v;
#pragma unroll
            for (int i = 0; i < KS; ++i) { o[i][nt][j] *= corr; o[i][nt][j + 2] *= corr; }
          }
          pb[nt][0] = movmatrix_trans(pack_half2(pr[0], pr[1]));
          pb[nt][1] = movmatrix_trans(pack_half2(pr[2], pr[3]));
        }
        // ---- a NaN value of a token some column does not see must not reach it through 0 x NaN ----
        if (!whole) {
          uint32_t bad = 0;
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int w = 0; w < D / 32; ++w) bad |= nan_codes(cur.v[i][w]);
          if (__any_sync(0xffffffffu, bad != 0)) {
            // NaN codes become zeros; where a column sees one, its output becomes NaN: the counts
            // of (NaN, seen) pairs are a product of the same shape
            uint32_t seen[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const int key = tok0 + g + h * 8;
                const bool s0 = key < hi_key[nt][0] && key >= lo_key[nt][0];
                const bool s1 = key < hi_key[nt][1] && key >= lo_key[nt][1];
                seen[nt][h] = movmatrix_trans((s0 ? 0x3c00u : 0u) | (s1 ? 0x3c000000u : 0u));
              }
#pragma unroll
            for (int i = 0; i < KS; ++i) {
              const int w = i >> 1, sh = 16 * (i & 1);
              uint32_t a[4];
#pragma unroll
              for (int r = 0; r < 4; ++r) {      // a0: byte 0 of tokens 0, 1; a1: byte 1; a2, a3: tokens 2, 3
                const uint32_t x = nan_codes(cur.v[(r >> 1) * 2][w]) >> (sh + 8 * (r & 1) + 7);
                const uint32_t y = nan_codes(cur.v[(r >> 1) * 2 + 1][w]) >> (sh + 8 * (r & 1) + 7);
                a[r] = ((x & 1u) ? 0x3c00u : 0u) | ((y & 1u) ? 0x3c000000u : 0u);
              }
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                float n[4] = {0.f, 0.f, 0.f, 0.f};
                mma_f16_16816(n, a, seen[nt][0], seen[nt][1]);
#pragma unroll
                for (int j = 0; j < 4; ++j)
                  if (n[j] > 0.f) o[i][nt][j] = __uint_as_float(0x7fc00000u);
              }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
              for (int w = 0; w < D / 32; ++w) cur.v[i][w] &= ~((nan_codes(cur.v[i][w]) >> 7) * 0xffu);
          }
        }
        // ---- O^T += V^T P^T ----
#pragma unroll
        for (int i = 0; i < KS; ++i) {
          const uint32_t sel = (i & 1) ? 0x7362u : 0x5140u;
          const uint32_t x = prmt(cur.v[0][i >> 1], cur.v[1][i >> 1], sel), y = prmt(cur.v[2][i >> 1], cur.v[3][i >> 1], sel);
          const uint32_t a[4] = {e4m3x2_to_half2(x), e4m3x2_to_half2(x >> 16), e4m3x2_to_half2(y), e4m3x2_to_half2(y >> 16)};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma_f16_16816(o[i][nt], a, pb[nt][0], pb[nt][1]);
        }
      }
      cur = nxt;
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
    const bool direct = u_lo == 0 && u_hi == seq.units;
    // a run that begins before this CTA's share uses the CTA's first slot, one that goes on the second
    float* part = p.partial + ((long long)blockIdx.x * 2 + (u_lo == 0 ? 1 : 0)) * Cfg::kPartial;
#pragma unroll
    for (int quarter = 0; quarter < 4; ++quarter) {
      __syncthreads();
      // rows of O^T in MMA i: codes 2 i and 2 i + 1 of each lane group's run of D / 8
#pragma unroll
      for (int i = quarter * KS / 4; i < (quarter + 1) * KS / 4; ++i)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int c = nt * 8 + 2 * t + (j & 1);
            const int dd = g * (D / 32) + 2 * (i - quarter * KS / 4) + (j >> 1);   // of this quarter
            s_o[warp][c * (D / 4) + dd] = o[i][nt][j];
          }
      __syncthreads();
      for (int x = tid; x < cols * (D / 4); x += kPgThreads) {
        const int c = x / (D / 4), dd = x % (D / 4);
        const int d = (dd / (D / 32)) * (D / 8) + quarter * (D / 32) + dd % (D / 32);
        float acc = 0.f;
#pragma unroll
        for (int w = 0; w < kPgWarps; ++w) acc += s_o[w][c * (D / 4) + dd] * s_w[w][c];
        if (direct) {
          const float l = s_l[0][c];
          const int row = (col0 + c) / hg, h = (col0 + c) % hg;
          // a row that sees nothing is zero; l is NaN where a score it sees is
          p.out[((long long)(seq.row0 + row) * p.H + gh * hg + h) * D + d] = __float2bfloat16_rn(l == 0.f ? 0.f : acc / l);
        } else {
          part[c * D + d] = acc;
        }
      }
    }
    if (!direct && tid < cols) {
      part[COLS * D + tid] = s_m[0][tid];
      part[COLS * D + COLS + tid] = s_l[0][tid];
    }
    __syncthreads();   // shared memory is the next run's
    at = seg_at + u_hi;
  }
}

// Folds the partials of cut segments, in the order of their keys.  One CTA a sequence (and a KV
// head); a segment that one CTA held whole was written by it.
template <int D, int NT>
__global__ void __launch_bounds__(kPgThreads) mha_pages_fold_kernel(const PagesParams p) {
  using Cfg = PgCfg<D, NT>;
  constexpr int COLS = Cfg::kCols;
  __shared__ long long s_sum[2 * kPgWarps];
  __shared__ float s_f[kPgCtas];
  pdl_launch();
  pdl_wait();
  const int b = blockIdx.x, gh = blockIdx.y, tid = threadIdx.x, hg = p.H / p.G;
  long long before = 0, total = 0;
  for (int i = tid; i < p.B; i += kPgThreads) {
    const PagesSeq s = pages_seq<COLS>(p, i);
    const long long w = (long long)s.segs * s.units;
    total += w;
    if (i < b) before += w;
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    before += __shfl_xor_sync(0xffffffffu, before, o);
    total += __shfl_xor_sync(0xffffffffu, total, o);
  }
  if ((tid & 31) == 0) { s_sum[2 * (tid >> 5)] = before; s_sum[2 * (tid >> 5) + 1] = total; }
  __syncthreads();
  before = total = 0;
  for (int w = 0; w < kPgWarps; ++w) { before += s_sum[2 * w]; total += s_sum[2 * w + 1]; }
  const PagesSeq seq = pages_seq<COLS>(p, b);
  const long long share = pages_share(total, p.ctas);
  const int blocks = seq.segs / p.G;
  for (int cb = 0; cb < blocks; ++cb) {
    const long long s0 = before + ((long long)gh * blocks + cb) * seq.units, s1 = s0 + seq.units;
    const int c_lo = (int)(s0 / share), c_hi = (int)((s1 - 1) / share), pieces = c_hi - c_lo + 1;
    if (pieces == 1) continue;
    const int col0 = cb * COLS, cols = min(COLS, seq.n * hg - col0);
    // the piece that begins the segment lies in its CTA's second slot, the others in the first
    auto slot_of = [&](int i) { return p.partial + ((long long)(c_lo + i) * 2 + (i == 0 ? 1 : 0)) * Cfg::kPartial; };
    for (int c = 0; c < cols; ++c) {
      __syncthreads();
      float m = -INFINITY;
      for (int i = 0; i < pieces; ++i) m = fmaxf(m, slot_of(i)[COLS * D + c]);
      const float safe = m == -INFINITY ? 0.f : m;
      for (int i = tid; i < pieces; i += kPgThreads) s_f[i] = ex2(slot_of(i)[COLS * D + c] - safe);
      __syncthreads();
      if (tid < D) {
        float l = 0.f, acc = 0.f;
        for (int i = 0; i < pieces; ++i) {
          l += slot_of(i)[COLS * D + COLS + c] * s_f[i];
          acc += slot_of(i)[c * D + tid] * s_f[i];
        }
        const int row = (col0 + c) / hg, h = (col0 + c) % hg;
        p.out[((long long)(seq.row0 + row) * p.H + gh * hg + h) * D + tid] = __float2bfloat16_rn(l == 0.f ? 0.f : acc / l);
      }
    }
  }
}

template <int D, int NT>
static int launch_pages(const PagesParams& p, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(kPgThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  fill_pdl_attr(cfg, attr);
  cfg.gridDim = dim3(p.ctas);
  if (cudaLaunchKernelEx(&cfg, mha_pages_kernel<D, NT>, p) != cudaSuccess) return IRON_ERR_LAUNCH;
  cfg.gridDim = dim3(p.B, p.G);
  return cudaLaunchKernelEx(&cfg, mha_pages_fold_kernel<D, NT>, p) == cudaSuccess ? IRON_OK : IRON_ERR_LAUNCH;
}

template <int D>
static int launch_pages_cols(const PagesParams& p, int cols, cudaStream_t stream) {
  return cols <= 8 ? launch_pages<D, 1>(p, stream) : launch_pages<D, 2>(p, stream);
}

}  // namespace iron

using namespace iron;

extern "C" long long iron_mha_pages_workspace_bytes(int D) {
  if (D != 64 && D != 128) return 0;
  const long long partial = 16ll * D + 32;
  return (long long)kPgCtas * 2 * partial * sizeof(float);
}

static int pages_args(PagesParams& p, const void* q, const void* pool, const float* scales, int P, int page_size,
                      const int* tables, int width, const int* lengths, const int* row_start, int B, int rows, int H,
                      int G, int D, int causal, int window, float scale, void* workspace, long long workspace_bytes,
                      void* out) {
  const int log_page = log2_page(page_size);
  if (B < 0 || rows < 0 || H <= 0 || G <= 0 || H % G || (D != 64 && D != 128) || P <= 0 || width <= 0 || log_page < 0)
    return IRON_ERR_SHAPE;
  if (G > 65535 || (long long)P * page_size > 0x7fffffffll || (long long)rows * H > 0x7fffffffll) return IRON_ERR_SHAPE;
  if ((long long)width * page_size > 0x7fffffffll) return IRON_ERR_SHAPE;
  if (window >= 0 && !causal) return IRON_ERR_UNSUPPORTED;
  if (!(scale > 0.f)) return IRON_ERR_SHAPE;
  if (B == 0 || rows == 0) return 1;   // nothing to do
  if (!q || !pool || !scales || !tables || !lengths || !out || !workspace) return IRON_ERR_SHAPE;
  if (!aligned16(q) || !aligned16(pool) || !aligned16(out) || !aligned16(workspace) ||
      (reinterpret_cast<uintptr_t>(scales) & 7))
    return IRON_ERR_ALIGN;
  if (workspace_bytes < iron_mha_pages_workspace_bytes(D)) return IRON_ERR_WORKSPACE;
  p.q = (const __nv_bfloat16*)q; p.pool = (const uint8_t*)pool; p.scales = scales; p.tables = tables;
  p.lengths = lengths; p.row_start = row_start; p.out = (__nv_bfloat16*)out; p.partial = (float*)workspace;
  p.B = B; p.H = H; p.G = G; p.P = P; p.width = width; p.log_page = log_page; p.causal = causal; p.window = window;
  p.rows = rows; p.ctas = kPgCtas;
  p.scale_log2 = scale * 1.4426950408889634f;
  return IRON_OK;
}

extern "C" int iron_mha_decode_pages_bf16(const void* q, const void* pool, const float* scales, int P, int page_size,
                                          const int* tables, int width, const int* lengths, int B, int H, int G, int D,
                                          int window, float scale, void* workspace, long long workspace_bytes, void* out,
                                          iron_stream_t stream) {
  PagesParams p = {};
  const int rc = pages_args(p, q, pool, scales, P, page_size, tables, width, lengths, nullptr, B, B, H, G, D, 1, window,
                            scale, workspace, workspace_bytes, out);
  if (rc) return rc == 1 ? IRON_OK : rc;
  return D == 64 ? launch_pages_cols<64>(p, H / G, (cudaStream_t)stream) : launch_pages_cols<128>(p, H / G, (cudaStream_t)stream);
}

extern "C" int iron_mha_prefill_pages_bf16(const void* q, const void* pool, const float* scales, int P, int page_size,
                                           const int* tables, int width, const int* lengths, const int* row_start, int B,
                                           int rows, int H, int G, int D, int causal, int window, float scale,
                                           void* workspace, long long workspace_bytes, void* out, iron_stream_t stream) {
  PagesParams p = {};
  const int rc = pages_args(p, q, pool, scales, P, page_size, tables, width, lengths, row_start, B, rows, H, G, D,
                            causal, window, scale, workspace, workspace_bytes, out);
  if (rc) return rc == 1 ? IRON_OK : rc;
  if (!row_start) return IRON_ERR_SHAPE;
  return D == 64 ? launch_pages<64, 2>(p, (cudaStream_t)stream) : launch_pages<128, 2>(p, (cudaStream_t)stream);
}
