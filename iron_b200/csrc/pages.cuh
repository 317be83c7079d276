// What the kernels of the paged 8-bit key/value cache share: the page sizes taken, the e4m3
// conversions, the power-of-two scale of a (page, KV head), and what the attention calls are given.
#pragma once
#include "common.cuh"

namespace iron {

constexpr int kMaxRequests = 8192;   // requests of one step (four words of shared memory each)

// log2 of a page size the kernels take (16, 32, 64, 128 or 256 tokens), else -1.
inline int log2_page(int page) {
  for (int k = 4; k <= 8; ++k)
    if (page == 1 << k) return k;
  return -1;
}

// Two floats -> two e4m3 codes (to nearest even; NaN stays NaN), the first in the low byte.
__device__ __forceinline__ uint32_t cvt_e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
// Two e4m3 codes -> two halves (exact).
__device__ __forceinline__ uint32_t e4m3x2_to_half2(uint32_t codes) {
  uint32_t r;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(r) : "r"(codes));
  return r;
}
// The same of a register's upper two codes: named as a half register, so that no shift is needed.
__device__ __forceinline__ uint32_t e4m3x2_hi_to_half2(uint32_t codes) {
  uint32_t r;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, hi;\n\t}" : "=r"(r) : "r"(codes));
  return r;
}
__device__ __forceinline__ float2 e4m3x2_to_float2(uint32_t codes) {
  const uint32_t h = e4m3x2_to_half2(codes);
  float2 f;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %2;\n\tcvt.f32.f16 %0, lo;\n\tcvt.f32.f16 %1, hi;\n\t}"
      : "=f"(f.x), "=f"(f.y)
      : "r"(h));
  return f;
}

// 2^e, e the smallest whole number with amax <= 448 * 2^e, and 2^-60 at least (an all-zero page).
// A float format rounds relative to the value, so a power of two costs no precision, and codes
// that a later, larger scale moves are exact but for underflow.  448 = 1.75 * 2^8: with
// amax = 1.f * 2^x, e = x - 8 where 1.f <= 1.75, else x - 7.
__device__ __forceinline__ float pow2_scale(float amax) {
  const uint32_t u = __float_as_uint(amax);
  int e = (int)(u >> 23) - 127 - ((u & 0x7fffffu) <= 0x600000u ? 8 : 7);
  e = max(e, -60);   // zero and subnormal magnitudes end here
  return __uint_as_float((uint32_t)(e + 127) << 23);
}

// A segment that several CTAs share, as the CTA that begins it leaves it for the fold.
struct PagesRecord {
  int pieces, row0, head0, col0, cols, pad[3];
};

struct PagesParams {
  const __nv_bfloat16* q;
  const uint8_t* pool;
  const float* scales;
  const int* tables;
  const int* lengths;
  const int* row_start;     // nullptr: one query a sequence, in order
  __nv_bfloat16* out;
  float* partial;
  PagesRecord* records;
  int B, H, G, hg, P, width, log_page, causal, window, rows, ctas;   // hg = H / G
  int split;                // sequences of one row are the decode kernel's, not the ragged one's
  float scale_log2;
  int* status;
};

// A sequence's tokens as far as its table goes, and the query rows it brings, inside the buffer.
__device__ __forceinline__ int seq_len(const PagesParams& p, int b) {
  return max(0, (int)min((long long)p.lengths[b], (long long)p.width << p.log_page));
}
__device__ __forceinline__ int seq_rows(const PagesParams& p, int b, int& row0) {
  row0 = min(max(p.row_start[b], 0), p.rows);
  return max(row0, min(p.row_start[b + 1], p.rows)) - row0;   // no difference that could wrap
}

// a / b for a >= 0, b > 0: the 64-bit division is a long routine, and seldom needed
__device__ __forceinline__ long long div_ll(long long a, int b) {
  return a >> 32 ? a / b : (long long)((uint32_t)a / (uint32_t)b);
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

// bit 7 of a byte set where the code is NaN (0x7f or 0xff)
__device__ __forceinline__ uint32_t nan_codes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

// The ragged form on tcgen05 (mha_pages_tc.cu).
long long mha_pages_tc_workspace_bytes(int D);
int mha_pages_tc(const PagesParams& p, int D, void* workspace, cudaStream_t stream);

}  // namespace iron
