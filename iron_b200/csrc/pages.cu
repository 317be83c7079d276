// The bookkeeping and the write of a key/value cache that lies in pages of 8-bit codes.
//
//   page_step      one serving step's bookkeeping: every request names how many rows it brings
//                  (or that it ended); requests in order take the pages they need from a ring
//                  of free page ids, ended ones give theirs back, and every new row learns
//                  its slot (page * page_size + offset) and its position.
//   rope_kv_pages  RoPE on a step's q and k; q goes out in bf16, k and v into their slots as
//                  e4m3 codes under one scale per (page, KV head, keys or values).
//
// The cache: pool (P, G, 2, page, D) e4m3 -- the keys and the values of one page and KV head are
// one run of memory -- and scales (P, G, 2) f32; a value is its code times its scale.
#include <cooperative_groups.h>

#include "common.cuh"
#include "pages.cuh"

namespace cg = cooperative_groups;

namespace iron {

// ---- page_step ----------------------------------------------------------------------------
// Three prefix sums over the requests (rows, pages taken, pages given back), then three flat
// loops over rows, taken pages and returned pages, each of which finds its request by binary
// search in shared memory, so one long prompt among many decode rows costs no more than its
// rows.  Every CTA of the (one) cluster computes the sums itself: the cluster meets once, after
// all of its reads of the lengths and the ring's header, so both may be updated in place.
// Bound by latency: the chain length -> sum -> search -> page id -> slot.  64 requests of a row each:
// 5.5 us; 509 requests with 16,384 rows: 8.5 us.
constexpr int kStepThreads = 1024;

// Inclusive sum over the block of two values at once; `total` gets the block's sums.
__device__ __forceinline__ longlong2 block_scan2(longlong2 v, longlong2* warp_sums, longlong2& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long x = __shfl_up_sync(0xffffffffu, v.x, o), y = __shfl_up_sync(0xffffffffu, v.y, o);
    if (lane >= o) { v.x += x; v.y += y; }
  }
  __syncthreads();   // warp_sums may still be read from an earlier call
  if (lane == 31) warp_sums[warp] = v;
  __syncthreads();
  longlong2 s = warp_sums[lane];   // 32 warps
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long x = __shfl_up_sync(0xffffffffu, s.x, o), y = __shfl_up_sync(0xffffffffu, s.y, o);
    if (lane >= o) { s.x += x; s.y += y; }
  }
  total.x = __shfl_sync(0xffffffffu, s.x, 31);
  total.y = __shfl_sync(0xffffffffu, s.y, 31);
  const int before = warp ? warp - 1 : 0;
  const long long bx = __shfl_sync(0xffffffffu, s.x, before), by = __shfl_sync(0xffffffffu, s.y, before);
  if (warp) { v.x += bx; v.y += by; }
  return v;
}

// The last b in [0, n) with first[b] <= x (first is sorted and first[0] <= x).
__device__ __forceinline__ int owner_of(const int* first, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first[mid] <= x) lo = mid; else hi = mid;
  }
  return lo;
}

__global__ void __launch_bounds__(kStepThreads) page_step_kernel(
    int* tables, int width, const int* lengths, const int* new_tokens, int B, int* pages, int P, const int* ring,
    int log_page, int rows, int* lengths_out, int* ring_out, int* slots, int* positions, int* row_start) {
  extern __shared__ int step_smem[];
  // per request: where its rows, its taken pages and its returned pages begin, and what it holds
  int* first_row = step_smem;
  int* first_taken = first_row + B;
  int* first_back = first_taken + B;
  int* length = first_back + B;      // tokens before the step; bit 31: the request was refused or ended
  __shared__ longlong2 warp_sums[32];
  __shared__ int s_used, s_refused;
  const int tid = threadIdx.x, ctas = gridDim.x;
  const int page = 1 << log_page;
  if (tid < 32) warp_sums[tid] = make_longlong2(0, 0);
  if (tid == 0) { s_used = 0; s_refused = 0; }
  pdl_wait();
  pdl_launch();
  const int head = P > 0 ? (int)(((long long)ring[0] % P + P) % P) : 0;
  const int count = max(0, min(ring[1], P));
  __syncthreads();

  long long rows_before = 0, taken_before = 0, back_before = 0;
  for (int b0 = 0; b0 < B; b0 += kStepThreads) {
    const int b = b0 + tid;
    const bool in = b < B;
    const int len = in ? max(lengths[b], 0) : 0;
    const int asked = in ? new_tokens[b] : 0;
    const bool ended = asked < 0;
    const int n = max(asked, 0);
    longlong2 total;
    const longlong2 r = block_scan2(make_longlong2(n, 0), warp_sums, total);
    const long long row_end = rows_before + r.x;
    rows_before += total.x;
    const int held = (int)min(((long long)len + page - 1) >> log_page, (long long)width);
    const long long want = ((long long)len + n + page - 1) >> log_page;
    const bool fits = in && !ended && want <= width && row_end <= rows;
    const int need = fits ? (int)(want - held) : 0;
    const int back = in && ended ? held : 0;
    const longlong2 t = block_scan2(make_longlong2(need, back), warp_sums, total);
    const long long taken_end = taken_before + t.x, back_end = back_before + t.y;
    taken_before += total.x;
    back_before += total.y;
    const bool served = fits && (need == 0 || taken_end <= count);
    if (in) {
      // sums past 2^31 belong to requests that are refused: clamped, they only end searches
      first_row[b] = (int)min(row_end - n, 0x7fffffffll);
      first_taken[b] = (int)min(taken_end - need, 0x7fffffffll);
      first_back[b] = (int)min(back_end - back, 0x7fffffffll);
      length[b] = len | (served ? 0 : (int)0x80000000);
      if (served && need) atomicMax(&s_used, (int)taken_end);
      if (!served && !ended) atomicAdd(&s_refused, 1);
    }
  }
  // every CTA has read what the step overwrites
  cg::this_cluster().sync();
  const int used = s_used;
  const int total_rows = (int)min(rows_before, 0x7fffffffll);
  const int given = (int)min(back_before, 0x7fffffffll);
  const int at = blockIdx.x * kStepThreads + tid, step = ctas * kStepThreads;

  for (int r = at; r < rows; r += step) {
    int slot = -1, pos = 0;
    if (r < total_rows) {
      const int b = owner_of(first_row, B, r);
      const int len = length[b];
      if (len >= 0) {
        pos = len + (r - first_row[b]);
        const int pi = pos >> log_page, held = (len + page - 1) >> log_page;
        const int entry = pi < held ? tables[(size_t)b * width + pi]
                                    : pages[(int)(((long long)head + first_taken[b] + (pi - held)) % P)];
        // an id that is no page's has no slots: decided before the product, which could wrap into the pool
        if ((unsigned)entry < (unsigned)P) slot = entry * page + (pos & (page - 1));
      }
    }
    slots[r] = slot;
    positions[r] = pos;
  }
  for (int t = at; t < used; t += step) {
    const int b = owner_of(first_taken, B, t);
    const int held = ((length[b] & 0x7fffffff) + page - 1) >> log_page;
    tables[(size_t)b * width + held + (t - first_taken[b])] = pages[(int)(((long long)head + t) % P)];
  }
  for (int t = at; t < given; t += step) {
    const int b = owner_of(first_back, B, t);
    pages[(int)(((long long)head + count + t) % P)] = tables[(size_t)b * width + (t - first_back[b])];
  }
  if (blockIdx.x == 0) {
    for (int b = tid; b < B; b += kStepThreads) {
      const int next = b + 1 < B ? first_row[b + 1] : total_rows;
      const int len = length[b];
      // an ended request holds nothing; a refused one keeps what it had
      const int asked_rows = next - first_row[b];
      row_start[b] = first_row[b];
      lengths_out[b] = len >= 0 ? len + asked_rows : (new_tokens[b] < 0 ? 0 : (len & 0x7fffffff));
    }
    if (tid == 0) {
      row_start[B] = total_rows;
      ring_out[0] = P > 0 ? (int)(((long long)head + used) % P) : 0;
      ring_out[1] = count - used + given;
      ring_out[2] = s_refused;
      ring_out[3] = total_rows;
    }
  }
}

// ---- rope_kv_pages --------------------------------------------------------------------------
// Bound by bytes: a row's qkv in, q in bf16 and k, v as codes out.  A page's scale needs the largest
// magnitude of all of a step's rows of that page before the first code, so the unit of work is a run -- the
// rows that go to one page -- of one head's keys or values: the CTA that finds its beginning in the slots
// takes all of it, a thread sixteen elements, held between the maximum and the conversion (at its bound of 64
// registers the kernel spills 88 bytes, 96 with heads of 128).
// Every run has one owner, so no atomics and one order.  q is the rest of the grid's.
// 2048 rows of a prompt, 32 heads over 8 of 128: 10.3 us (47 MB, 4.5 TB/s); 6111 ragged rows, over 4: 29.4 us
// (121 MB, 4.1 TB/s; issue slots 53 % used: conversions and the angles' table); 64 single rows 4.9 us.
constexpr int kWriteThreads = 256;
constexpr int kShortRun = 8;       // rows that one warp takes by itself
constexpr int kHeld = 1;           // 16-element pieces a thread holds in registers: two cost more in occupancy (11.1 us for 10.4)

struct WriteParams {
  const __nv_bfloat16* qkv;
  long long pitch;
  const __nv_bfloat16* angles;
  __nv_bfloat16* q_out;
  uint8_t* pool;
  float* scales;
  const int* slots;
  const int* positions;
  int rows, H, G, S, log_page;
  long long slots_max;      // P * page
  int chunk;                // rows a CTA of the k/v half looks at for the beginnings of page runs
  int kv_blocks;            // CTAs of the k/v half; the rest rotate q
};

// Sixteen elements of one head's row -- [i0, i0 + 8) and their partners half a head on -- turned by
// the row's angles when `turn`.  Products and sums are rounded one by one (no contraction), as
// the separate RoPE operator computes them.
template <int D>
__device__ __forceinline__ void load_turned(const WriteParams& p, int row, int head, int i0, bool turn, float* a, float* b) {
  const __nv_bfloat16* src = p.qkv + (long long)row * p.pitch + (long long)head * D;
  unpack8(ld_cached(src + i0), a);
  unpack8(ld_cached(src + D / 2 + i0), b);
  if (turn) {
    const int pos = max(0, min(p.positions[row], p.S - 1));
    const __nv_bfloat16* ar = p.angles + (size_t)pos * D;
    float cs[16];
    unpack8(ld_cached(ar + 2 * i0), cs);
    unpack8(ld_cached(ar + 2 * i0 + 8), cs + 8);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float c = cs[2 * j], s = cs[2 * j + 1];
      const float ya = __fsub_rn(__fmul_rn(a[j], c), __fmul_rn(b[j], s));
      const float yb = __fadd_rn(__fmul_rn(b[j], c), __fmul_rn(a[j], s));
      a[j] = ya; b[j] = yb;
    }
  }
}

// The largest finite magnitude of the sixteen: what is not finite is stored as e4m3's NaN and
// must not drive the page's scale.
__device__ __forceinline__ float finite_amax(const float* a, const float* b) {
  float m = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float x = fabsf(a[j]), y = fabsf(b[j]);
    if (x < INFINITY) m = fmaxf(m, x);
    if (y < INFINITY) m = fmaxf(m, y);
  }
  return m;
}
// x * 0 + x: x where x is finite, NaN otherwise (an infinity is no e4m3 value).
__device__ __forceinline__ uint32_t e4m3_pair(float x, float y, float inv) {
  return cvt_e4m3x2(fmaf(x, 0.f, x) * inv, fmaf(y, 0.f, y) * inv);
}
__device__ __forceinline__ uint2 e4m3_eight(const float* x, float inv) {
  return make_uint2(e4m3_pair(x[0], x[1], inv) | (e4m3_pair(x[2], x[3], inv) << 16),
                    e4m3_pair(x[4], x[5], inv) | (e4m3_pair(x[6], x[7], inv) << 16));
}

// Sixteen codes that lie under `old` brought under a larger scale.
__device__ __forceinline__ uint32_t rescale_word(uint32_t w, float ratio) {
  const float2 lo = e4m3x2_to_float2(w & 0xffffu), hi = e4m3x2_to_float2(w >> 16);
  return cvt_e4m3x2(lo.x * ratio, lo.y * ratio) | (cvt_e4m3x2(hi.x * ratio, hi.y * ratio) << 16);
}

// One run -- consecutive rows that go to consecutive slots of one page -- of one KV head's keys or
// values, by the `threads` threads that call this (a warp, or the CTA), `t` their index.  Every row
// takes D / 16 threads, a sixteen-element piece each; up to kHeld pieces a thread stay in registers
// between the maximum and the conversion, their loads all in flight at once; a longer run is read twice.
template <int D, bool kBlock>
__device__ __forceinline__ void write_run(const WriteParams& p, int row, int n, int slot, int g, int kind, int t,
                                          int threads, float* red) {
  constexpr int kPieces = D / 16;
  const int page = 1 << p.log_page, off = slot & (page - 1);
  const long long at = ((long long)(slot >> p.log_page) * p.G + g) * 2 + kind;
  uint8_t* base = p.pool + at * page * D;
  const float old = off ? p.scales[at] : 0.f;
  const int i0 = t % kPieces * 8, first = t / kPieces, rows_at_once = threads / kPieces;
  const int head = p.H + kind * p.G + g;
  const bool turn = kind == 0;

  float ka[kHeld][8], kb[kHeld][8];
  float m = 0.f;
#pragma unroll
  for (int k = 0; k < kHeld; ++k) {
    const int i = first + k * rows_at_once;
    if (i < n) load_turned<D>(p, row + i, head, i0, turn, ka[k], kb[k]);
  }
#pragma unroll
  for (int k = 0; k < kHeld; ++k)
    if (first + k * rows_at_once < n) m = fmaxf(m, finite_amax(ka[k], kb[k]));
  for (int i = first + kHeld * rows_at_once; i < n; i += rows_at_once) {
    float a[8], b[8];
    load_turned<D>(p, row + i, head, i0, turn, a, b);
    m = fmaxf(m, finite_amax(a, b));
  }
  m = warp_max(m);
  if (kBlock) {
    if ((t & 31) == 0) red[t >> 5] = m;
    __syncthreads();
    m = red[0];
    for (int w = 1; w < threads / 32; ++w) m = fmaxf(m, red[w]);
  }
  float scale = pow2_scale(m);
  if (off) {
    scale = fmaxf(scale, old);        // the page goes on: it keeps the larger scale
    if (scale != old) {
      // codes of earlier steps, 16 at a time; a ratio of powers of two is exact but for underflow
      const float ratio = old / scale;
      for (int i = t; i < off * kPieces; i += threads) {
        uint4* w = reinterpret_cast<uint4*>(base) + i;
        uint4 x = *w;
        x.x = rescale_word(x.x, ratio); x.y = rescale_word(x.y, ratio);
        x.z = rescale_word(x.z, ratio); x.w = rescale_word(x.w, ratio);
        *w = x;
      }
    }
  }
  if (kBlock) __syncthreads(); else __syncwarp();   // the old scale (and `red`) have been read
  if (t == 0) p.scales[at] = scale;
  const float inv = 1.0f / scale;
  uint8_t* dst = base + (size_t)off * D + i0;
#pragma unroll
  for (int k = 0; k < kHeld; ++k) {
    const int i = first + k * rows_at_once;
    if (i < n) {
      *reinterpret_cast<uint2*>(dst + (size_t)i * D) = e4m3_eight(ka[k], inv);
      *reinterpret_cast<uint2*>(dst + (size_t)i * D + D / 2) = e4m3_eight(kb[k], inv);
    }
  }
  for (int i = first + kHeld * rows_at_once; i < n; i += rows_at_once) {
    float a[8], b[8];
    load_turned<D>(p, row + i, head, i0, turn, a, b);
    *reinterpret_cast<uint2*>(dst + (size_t)i * D) = e4m3_eight(a, inv);
    *reinterpret_cast<uint2*>(dst + (size_t)i * D + D / 2) = e4m3_eight(b, inv);
  }
}

template <int D>
__global__ void __launch_bounds__(kWriteThreads, 4) rope_kv_pages_kernel(const WriteParams p) {
  __shared__ float red[kWriteThreads / 32];
  pdl_wait();
  pdl_launch();
  const int tid = threadIdx.x;
  if ((int)blockIdx.x >= p.kv_blocks) {
    // ---- q: rotated, rounded to bf16 ----
    constexpr int kPieces = D / 16;
    const long long total = (long long)p.rows * p.H * kPieces;
    for (long long i = (long long)(blockIdx.x - p.kv_blocks) * kWriteThreads + tid; i < total;
         i += (long long)(gridDim.x - p.kv_blocks) * kWriteThreads) {
      const int r = (int)div_ll(i, p.H * kPieces), of_row = (int)(i - (long long)r * (p.H * kPieces));
      const int piece = of_row % kPieces, h = of_row / kPieces;
      float a[8], b[8];
      load_turned<D>(p, r, h, piece * 8, true, a, b);
      __nv_bfloat16* dst = p.q_out + ((size_t)r * p.H + h) * D + piece * 8;
      *reinterpret_cast<uint4*>(dst) = pack8(a);
      *reinterpret_cast<uint4*>(dst + D / 2) = pack8(b);
    }
    return;
  }
  // ---- k and v: a CTA looks at some rows (32 at most, a lane each) for the beginnings of runs and
  // writes one KV head's keys or values of those ----
  const int which = blockIdx.x % (2 * p.G), g = which % p.G, kind = which / p.G;
  const int r0 = blockIdx.x / (2 * p.G) * p.chunk, r1 = min(r0 + p.chunk, p.rows);
  const int page = 1 << p.log_page, warp = tid >> 5, lane = tid & 31;
  auto slot_of = [&](int r) {
    const int s = r >= 0 && r < p.rows ? p.slots[r] : -1;
    return s < p.slots_max ? s : -1;
  };
  const int mine = r0 + lane < r1 ? slot_of(r0 + lane) : -1, before = slot_of(r0 + lane - 1);
  const bool goes_on = mine >= 0 && (mine & (page - 1)) != 0 && before == mine - 1;
  const unsigned on = __ballot_sync(0xffffffffu, goes_on);
  unsigned begin = __ballot_sync(0xffffffffu, mine >= 0 && !goes_on);
  // a short run is one warp's, in turn; a longer one is the whole CTA's
  for (int k = 0; begin; ++k) {
    const int l = __ffs(begin) - 1;
    begin &= begin - 1;
    const int slot = __shfl_sync(0xffffffffu, mine, l), most = page - (slot & (page - 1));
    int n = l == 31 ? 1 : __ffs(~(on >> (l + 1)));     // itself and the rows that go on
    n = min(n, most);
    if (r0 + l + n == r1 && n < most) {
      // it may go on behind the rows looked at
      for (bool more = true; more && n < most;) {
        const bool same = n + lane < most && slot_of(r0 + l + n + lane) == slot + n + lane;
        const unsigned m = __ballot_sync(0xffffffffu, same);
        more = m == 0xffffffffu;
        n += more ? 32 : __ffs(~m) - 1;
      }
    }
    if (n <= kShortRun) {
      if (k % (kWriteThreads / 32) == warp) write_run<D, false>(p, r0 + l, n, slot, g, kind, lane, 32, red);
    } else {
      __syncthreads();     // `red` is free
      write_run<D, true>(p, r0 + l, n, slot, g, kind, tid, kWriteThreads, red);
    }
  }
}

}  // namespace iron

using namespace iron;

extern "C" int iron_page_step_max_requests(void) { return kMaxRequests; }

extern "C" int iron_page_step(int* tables, int width, const int* lengths, const int* new_tokens, int B, int* pages,
                              int P, const int* ring, int page_size, int rows, int* lengths_out, int* ring_out,
                              int* slots, int* positions, int* row_start, iron_stream_t stream) {
  const int log_page = log2_page(page_size);
  if (B < 0 || B > kMaxRequests || width <= 0 || P <= 0 || rows < 0 || log_page < 0) return IRON_ERR_SHAPE;
  // slots and positions are 32-bit
  if ((long long)P * page_size > 0x7fffffffll || (long long)width * page_size > 0x7fffffffll) return IRON_ERR_SHAPE;
  if (!ring || !ring_out || !row_start || !pages) return IRON_ERR_SHAPE;
  if (B > 0 && (!tables || !lengths || !new_tokens || !lengths_out)) return IRON_ERR_SHAPE;
  if (rows > 0 && (!slots || !positions)) return IRON_ERR_SHAPE;
  const size_t smem = (size_t)4 * (B > 0 ? B : 1) * sizeof(int);
  static DeviceOnce configured;
  if (!configured.done()) {
    if (cudaFuncSetAttribute(page_step_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             4 * kMaxRequests * (int)sizeof(int)) != cudaSuccess)
      return IRON_ERR_LAUNCH;
    configured.mark();
  }
  cudaLaunchConfig_t cfg = {};
  // The flat loops are what a large step waits for (509 requests, 16,384 rows: 23.1 us with one CTA, 8.5
  // with eight); a small one is over before more CTAs would help (64 rows: 5.7 us with either).
  const int ctas = rows > 2 * kStepThreads || B > kStepThreads ? 8 : 1;
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(kStepThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = (cudaStream_t)stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ctas;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1 + pdl_attr_count();
  return cudaLaunchKernelEx(&cfg, page_step_kernel, tables, width, lengths, new_tokens, B, pages, P, ring, log_page, rows,
                            lengths_out, ring_out, slots, positions, row_start) == cudaSuccess
             ? IRON_OK
             : IRON_ERR_LAUNCH;
}

extern "C" int iron_rope_kv_pages_e4m3(const void* qkv, long long pitch, const void* angles, void* q_out, void* pool,
                                       float* scales, int P, int page_size, const int* slots, const int* positions,
                                       int rows, int H, int G, int D, int S, iron_stream_t stream) {
  const int log_page = log2_page(page_size);
  if (rows < 0 || H <= 0 || G <= 0 || (D != 64 && D != 128) || S <= 0 || P <= 0 || log_page < 0) return IRON_ERR_SHAPE;
  if ((long long)P * page_size > 0x7fffffffll) return IRON_ERR_SHAPE;
  if (pitch < (long long)(H + 2 * G) * D || (pitch & 7)) return IRON_ERR_SHAPE;
  // Rows a CTA looks at: a decode batch's rows are runs of one, a warp each, and want many CTAs; a
  // prompt's are runs of a page, and a CTA that finds none is in the way (2048 rows of a prompt, 32
  // heads over 8 of 128, pages of 64: 10.4 us with 32, 14.5 with 8; 64 single rows: 11.2 and 4.5 us).
  const int chunk = rows > 1024 ? 32 : kShortRun;
  const long long kv_blocks = ((long long)rows + chunk - 1) / chunk * 2 * G;
  if (kv_blocks > 0x3fffffffll) return IRON_ERR_SHAPE;
  if (rows == 0) return IRON_OK;
  if (!qkv || !angles || !q_out || !pool || !scales || !slots || !positions) return IRON_ERR_SHAPE;
  if (!aligned16(qkv) || !aligned16(angles) || !aligned16(q_out) || !aligned16(pool)) return IRON_ERR_ALIGN;
  WriteParams p = {};
  p.qkv = (const __nv_bfloat16*)qkv; p.pitch = pitch; p.angles = (const __nv_bfloat16*)angles;
  p.q_out = (__nv_bfloat16*)q_out; p.pool = (uint8_t*)pool; p.scales = scales; p.slots = slots;
  p.positions = positions; p.rows = rows; p.H = H; p.G = G; p.S = S; p.log_page = log_page;
  p.slots_max = (long long)P * page_size;
  p.chunk = chunk;
  p.kv_blocks = (int)kv_blocks;
  const long long q_items = (long long)rows * H * (D / 16);
  long long q_blocks = (q_items + kWriteThreads - 1) / kWriteThreads;
  q_blocks = q_blocks > 8 * kSMs ? 8 * kSMs : q_blocks;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(kv_blocks + q_blocks));
  cfg.blockDim = dim3(kWriteThreads);
  cfg.stream = (cudaStream_t)stream;
  cudaLaunchAttribute attr[1];
  fill_pdl_attr(cfg, attr);
  const cudaError_t e = D == 64 ? cudaLaunchKernelEx(&cfg, rope_kv_pages_kernel<64>, p)
                                : cudaLaunchKernelEx(&cfg, rope_kv_pages_kernel<128>, p);
  return e == cudaSuccess ? IRON_OK : IRON_ERR_LAUNCH;
}
