// kv4.hip — the 4-bit paged KV cache: page and slot planning, quantised
// appends, read-back and attention over the pages (glacier_hip_kv_plan_rows,
// glacier_hip_kv4_*, glacier_hip_paged_attention_kv4*). The page layout and
// the value of a code are stated in glacier_hip.h.
//
// Compiled with -ffp-contract=off; explicit fmaf() marks intended fusions.
#include <hip/hip_fp16.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>

#include "int4_ops.h"
#include "runtime.h"

namespace gk {
namespace {

constexpr int kPage = 16;       // positions of a page
constexpr int kMaxGroup = 8;    // query heads per KV head
constexpr int kMaxLanes = (int)GLACIER_HIP_KV_MAX_LANES;

struct Kv4 {  // the layer's view of a pool
  uint8_t *base;       // page 0, this layer
  size_t page_bytes;
  uint32_t page_count;
  int heads;           // KV heads
};

static __device__ __forceinline__ uint8_t *tile_of(const Kv4 &kv, uint32_t page, int head, int which,
                                                   int tile_bytes) {
  return kv.base + page * kv.page_bytes + (size_t)(2 * head + which) * tile_bytes;
}

// ---------------------------------------------------------------------------
// Planning. One workgroup, a lane a thread: two block-wide prefix sums (rows
// and new pages), then the new table entries. Few rows it writes too (a
// row's page is an old entry or one of the free pages it hands out, so no row
// waits for the table); many follow in a second launch. A launch is all that
// either costs: 64 lanes take 5.1 us with 64 rows and 6.6 us with 2048 where
// the second launch makes them 6.5 - 9.5 us; with 8192 rows it is 12.4 against 8.2.
// ---------------------------------------------------------------------------
constexpr uint32_t kPlanRows = 2048;  // rows that the planning workgroup writes itself
static __device__ __forceinline__ int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, true);  // row_shr 1, 2, 4, 8
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);  // lane 15 of rows 0, 2 onto 1, 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);  // lane 31 onto the upper half
  return v;
}

__global__ __launch_bounds__(kMaxLanes) void kv_plan_kernel(
    const int32_t *ctx, const int32_t *fresh, int lanes, int max_rows, int32_t *table,
    uint32_t max_pages, const int32_t *free_pages, uint32_t free_count, const int32_t *free_taken,
    int32_t *row_start, int32_t *ctx_after, int32_t *result, int64_t *slots, int32_t *row_lanes,
    int32_t *row_positions) {
  __shared__ int rows_of[kMaxLanes / 64], pages_of[kMaxLanes / 64];
  __shared__ int page_end[kMaxLanes], held_of[kMaxLanes], rows_end[kMaxLanes], after_of[kMaxLanes];
  const int t = threadIdx.x, w = t >> 6;
  const int c = t < lanes ? ctx[t] : 0;
  int n = t < lanes ? fresh[t] : 0;
  const int taken = *free_taken;
  const bool shape = c < 0 || n < 0 || n > max_rows;
  if (shape) n = 0;
  const uint32_t after = (uint32_t)max(c, 0) + (uint32_t)n;
  const bool full = after > (uint64_t)max_pages * kPage;
  const int held = (int)(((uint32_t)max(c, 0) + kPage - 1) / kPage);
  const int need = (int)((after + kPage - 1) / kPage) - held;
  int row_end = wave_scan(n), pg_end = wave_scan(need);
  if ((t & 63) == 63) {
    rows_of[w] = row_end;
    pages_of[w] = pg_end;
  }
  const int bad_shape = __syncthreads_or(shape), bad_full = __syncthreads_or(full);
  int rows = 0, pages = 0;
#pragma unroll
  for (int i = 0; i < kMaxLanes / 64; ++i) {
    if (i == w) {
      row_end += rows;
      pg_end += pages;
    }
    rows += rows_of[i];
    pages += pages_of[i];
  }
  const bool short_list =
      taken < 0 || (uint64_t)(uint32_t)taken + (uint32_t)pages > (uint64_t)free_count;
  const int status = bad_shape || rows > max_rows ? GLACIER_HIP_SHAPE_MISMATCH
                     : bad_full || short_list     ? GLACIER_HIP_CACHE_FULL
                                                  : GLACIER_HIP_OK;
  page_end[t] = pg_end;
  held_of[t] = held;
  rows_end[t] = row_end;
  after_of[t] = (int)after;
  __syncthreads();  // every read of ctx and free_taken is done: they may be outputs
  const bool good = status == GLACIER_HIP_OK;
  if (t < lanes) {
    row_start[t] = good ? row_end - n : 0;
    ctx_after[t] = good ? (int32_t)after : c;
  }
  if (t == 0) {
    row_start[lanes] = good ? rows : 0;
    result[0] = status;
    result[1] = good ? rows : 0;
    result[2] = good ? pages : 0;
    result[3] = taken + (good ? pages : 0);
  }
  auto past = [](const int *ends, int i) {  // the first lane that ends past i
    int lo = 0, hi = kMaxLanes - 1;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (ends[mid] > i) hi = mid;
      else lo = mid + 1;
    }
    return lo;
  };
  if (slots)
    for (int r = t; r < max_rows; r += kMaxLanes) {
      int64_t slot = -1;
      int lane = -1, pos = -1;
      if (good && r < rows) {
        lane = past(rows_end, r);
        pos = after_of[lane] - rows_end[lane] + r;
        const int p = pos / kPage - held_of[lane];
        const int page = p < 0 ? table[(size_t)lane * max_pages + pos / kPage]
                               : free_pages[taken + (lane ? page_end[lane - 1] : 0) + p];
        if (page >= 0) slot = (int64_t)page * kPage + pos % kPage;
      }
      slots[r] = slot;
      if (row_lanes) row_lanes[r] = lane;
      if (row_positions) row_positions[r] = pos;
    }
  if (!good) return;
  for (int p = t; p < pages; p += kMaxLanes) {
    const int lo = past(page_end, p), before = lo ? page_end[lo - 1] : 0;
    table[(size_t)lo * max_pages + held_of[lo] + (p - before)] = free_pages[taken + p];
  }
}

// Rows of a plan whose table, row_start and ctx_after are written.
__global__ __launch_bounds__(256) void kv_plan_rows_kernel(
    const int32_t *row_start, const int32_t *ctx_after, int lanes, int max_rows,
    const int32_t *table, uint32_t max_pages, int64_t *slots, int32_t *row_lanes,
    int32_t *row_positions) {
  const int r = blockIdx.x * 256 + threadIdx.x;
  if (r >= max_rows) return;
  int64_t slot = -1;
  int lane = -1, pos = -1;
  if (r < row_start[lanes]) {
    int lo = 0, hi = lanes - 1;  // the first lane whose rows end past r
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (row_start[mid + 1] > r) hi = mid;
      else lo = mid + 1;
    }
    lane = lo;
    pos = ctx_after[lane] - row_start[lane + 1] + r;
    const int page = table[(size_t)lane * max_pages + pos / kPage];
    if (page >= 0) slot = (int64_t)page * kPage + pos % kPage;
  }
  slots[r] = slot;
  if (row_lanes) row_lanes[r] = lane;
  if (row_positions) row_positions[r] = pos;
}

// ---------------------------------------------------------------------------
// Quantising rows into their slots, and reading them back
// ---------------------------------------------------------------------------
template <class T>
static __device__ __forceinline__ float widen(T v);
template <>
__device__ __forceinline__ float widen(float v) { return v; }
template <>
__device__ __forceinline__ float widen(__half v) { return __half2float(v); }
struct Bf16 {
  uint16_t bits;
};
template <>
__device__ __forceinline__ float widen(Bf16 v) { return __uint_as_float((uint32_t)v.bits << 16); }

template <int HD>
static __device__ __forceinline__ int step_byte(int P, int g) {
  return 8 * HD + 2 * ((P / 4) * (HD / 8) + g * 4 + P % 4);
}
template <int HD>
static __device__ __forceinline__ int low_byte(int which, int P, int g) {
  return which ? step_byte<HD>(P, g) + HD : 9 * HD + 2 * (P * (HD / 32) + g);
}

// Both kernels: a wave takes kRun rows of one KV head's K or V; neighbouring
// waves take the heads of the same rows.
template <int HD>
constexpr int kRun = 512 / HD;
struct StoreWave {
  int row, head, which;  // the first row
};
template <int HD>
static __device__ __forceinline__ StoreWave store_wave(int heads) {
  const int wave = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6)), unit = wave / heads;
  return {unit / 2 * kRun<HD>, wave - unit * heads, unit & 1};
}
// A slot's page and position; position < 0: none.
static __device__ __forceinline__ int place_of(const Kv4 &kv, const int64_t *slots, int r, int rows, uint32_t &page) {
  const uint64_t slot = r < rows ? (uint64_t)slots[r] : ~0ull;
  page = (uint32_t)(slot / kPage);
  return slot < (uint64_t)kv.page_count * kPage ? (int)(slot % kPage) : -1;
}

// The values' steps, minima and codes. A quotient (x - minimum) / step in f32
// is off by at most 2^-22 of itself (difference, reciprocal and product), 4e-6
// where it counts (up to 16): its nearest integer is certain unless it lies
// within 1e-5 of a half h + 1/2. Then the sign of (x - minimum) - (h + 1/2) step
// decides, which f32 holds exactly: the difference as a sum of two, the product
// (16 bits) taken off in one fma. (16-bit values hit such a tie in one group of
// sixty; in 64-bit arithmetic with a division the detour cost 4 of 19 us.)
struct Grid {
  __half step, low;
  float s, m, r;
};
// (The range over 15 is rounded as a division rounds it: the quotient's
// remainder is exact in one fma, and 1/15 has a single rounding; ranges too
// small for that become zero steps either way.)
static __device__ __forceinline__ Grid grid_of(float lo, float hi, bool bad) {
  constexpr float r15 = 1.0f / 15.0f;
  const float d = hi - lo, t = d * r15;
  float u = fmaf(fmaf(-t, 15.0f, d), r15, t);
  asm("" : "+v"(u));  // (rounded to 32 bits before it is to 16, not in one step)
  Grid q;
  q.step = bad ? __ushort_as_half(0x7E00) : __float2half_rn(u);
  q.low = bad ? __ushort_as_half(0x7E00) : __float2half_rn(lo);
  q.s = __half2float(q.step);
  q.m = __half2float(q.low);
  q.r = q.s > 0.0f ? __builtin_amdgcn_rcpf(q.s) : 0.0f;
  return q;
}
// Codes of four values from bit 0 on, and the largest distance from a nearest integer.
static __device__ __forceinline__ uint32_t codes_of(const float *x, const Grid &q, float &off) {
  float n[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float t = fminf(fmaxf((x[i] - q.m) * q.r, 0.0f), 15.0f);
    n[i] = rintf(t);
    off = fmaxf(off, fabsf(t - n[i]));
  }
  return (uint32_t)fmaf(fmaf(fmaf(n[3], 16.0f, n[2]), 16.0f, n[1]), 16.0f, n[0]);
}
static __device__ __forceinline__ uint32_t exact_code(float x, const Grid &q) {
  const float d = x - q.m, xx = d + q.m, rest = (x - xx) + ((xx - d) - q.m);
  const float t = fminf(fmaxf(d * q.r, 0.0f), 15.0f), h = floorf(t);
  if (fabsf(t - rintf(t)) <= 0.5f - 1e-5f) return (uint32_t)rintf(t);
  const float side = fmaf(-(h + 0.5f), q.s, d) + rest;
  return (uint32_t)h + (side > 0.0f || (side == 0.0f && ((int)h & 1)));
}
// Minimum and maximum, NaN where either value is, and over a quad of lanes.
static __device__ __forceinline__ float least(float a, float b) { return __builtin_elementwise_minimum(a, b); }
static __device__ __forceinline__ float most(float a, float b) { return __builtin_elementwise_maximum(a, b); }
static __device__ __forceinline__ void over_quad(float &lo, float &hi) {
  auto swap = [](float x, auto f) { return __int_as_float(f(__float_as_int(x))); };
  auto one = [](int x) { return __builtin_amdgcn_update_dpp(0, x, 0xB1, 0xF, 0xF, true); };
  auto two = [](int x) { return __builtin_amdgcn_update_dpp(0, x, 0x4E, 0xF, 0xF, true); };
  lo = least(lo, swap(lo, one));
  hi = most(hi, swap(hi, one));
  lo = least(lo, swap(lo, two));
  hi = most(hi, swap(hi, two));
}
// Nibble i of lane 8 (l / 8) + K's word, at bit AT of w.
template <int K, int AT>
static __device__ __forceinline__ void nibble_of(uint32_t &w, uint32_t word, int i) {
  w |= ((uint32_t)__builtin_amdgcn_ds_swizzle((int)word, K << 5 | 0x18) >> 4 * i & 15) << AT;
}
// Eight elements, as 16-byte loads where WIDE.
template <bool WIDE, class T>
static __device__ __forceinline__ void elements8(float (&f)[8], const T *x) {
  if constexpr (WIDE) {
    constexpr int N = 16 / sizeof(T);
    T e[8];
#pragma unroll
    for (int i = 0; i < 8; i += N) *(uint4 *)(e + i) = *(const uint4 *)(x + i);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = widen(e[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = widen(x[i]);
  }
}

// A thread quantises eight dims 8 q .. + 7 (q = l % (HD / 8)), a quad of lanes a
// group. K: its word of codes as it is. V: nibble j of eight threads' words, the
// dims 16 apart that a half word holds, by broadcasts inside eights of lanes.
// Few rows cost a launch (2.5 us of its 3.5); 16384 fp16 rows of 4 heads of 128
// (44 MB) take 17.2 us, four fifths of it issuing vector instructions (23 a
// value). Before: a group a thread, 64-bit divisions and byte stores 100 us; V as
// one thread per 4 dims 16 apart (no broadcasts, but reductions over 16 lanes) 26 us.
template <int HD, bool WIDE, class T>
__global__ __launch_bounds__(256) void kv4_append_kernel(Kv4 kv, const T *k, const T *v,
                                                         size_t k_stride, size_t v_stride,
                                                         const int64_t *slots, int rows) {
  constexpr int NG = HD / 32, NH = HD / 64;
  const StoreWave w = store_wave<HD>(kv.heads);
  if (w.row >= rows) return;
  const int l = threadIdx.x & 63, q = l % (HD / 8), g = q / 4, c = q % 4, r = w.row + l / (HD / 8);
  float f[8];
  elements8<WIDE>(f, (w.which ? v + (size_t)min(r, rows - 1) * v_stride : k + (size_t)min(r, rows - 1) * k_stride) +
                         w.head * HD + 8 * q);
  uint32_t page = 0;
  const int P = place_of(kv, slots, r, rows, page);
  float lo = least(f[0], f[1]), hi = most(f[0], f[1]);
#pragma unroll
  for (int i = 2; i < 8; i += 2) {
    lo = least(least(lo, f[i]), f[i + 1]);
    hi = most(most(hi, f[i]), f[i + 1]);
  }
  over_quad(lo, hi);
  const Grid grid = grid_of(lo, hi, !(hi <= 32768.0f && lo >= -32768.0f));
  float off = 0.0f;
  uint32_t word = codes_of(f, grid, off);
  word |= codes_of(f + 4, grid, off) << 16;
  if (__any(off > 0.5f - 1e-5f)) {
    word = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) word |= exact_code(f[i], grid) << 4 * i;
  }
  uint32_t half[2] = {0, 0};  // V: the half words of j = l % 8 and of j + 8
  if (w.which) {
    const int j = l & 7;
    nibble_of<0, 0>(half[0], word, j);
    nibble_of<2, 4>(half[0], word, j);
    nibble_of<4, 8>(half[0], word, j);
    nibble_of<6, 12>(half[0], word, j);
    nibble_of<1, 0>(half[1], word, j);
    nibble_of<3, 4>(half[1], word, j);
    nibble_of<5, 8>(half[1], word, j);
    nibble_of<7, 12>(half[1], word, j);
  }
  if (P < 0) return;
  uint8_t *tile = tile_of(kv, page, w.head, w.which, 10 * HD);
  if (w.which) {
    uint8_t *at = tile + (((P / 4 * 16 + (l & 7)) * 2 + P / 2 % 2) * NH + q / 8) * 4 + P % 2 * 2;
    *(uint16_t *)at = (uint16_t)half[0];
    *(uint16_t *)(at + 8 * 2 * NH * 4) = (uint16_t)half[1];
  } else {
    *(uint32_t *)(tile + P * (HD / 2) + (c * NG + g) * 4) = word;
  }
  if (c == 0) {
    *(__half *)(tile + step_byte<HD>(P, g)) = grid.step;
    *(__half *)(tile + low_byte<HD>(w.which, P, g)) = grid.low;
  }
}

template <int HD>
__global__ __launch_bounds__(256) void kv4_read_kernel(Kv4 kv, const int64_t *slots, int rows,
                                                       float *k, float *v) {
  constexpr int NG = HD / 32, NH = HD / 64;
  const StoreWave w = store_wave<HD>(kv.heads);
  const int l = threadIdx.x & 63;
  if (w.row >= rows) return;
  auto half_at = [](const uint8_t *p) { return __half2float(*(const __half *)p); };
  uint32_t page = 0;
  if (w.which == 0) {
    const int q = l % (HD / 8), g = q % NG, c = q / NG, r = w.row + l / (HD / 8);
    const int P = place_of(kv, slots, r, rows, page);
    if (P < 0) return;
    const uint8_t *tile = tile_of(kv, page, w.head, 0, 10 * HD);
    const uint32_t word = *(const uint32_t *)(tile + P * (HD / 2) + q * 4);
    const float step = half_at(tile + step_byte<HD>(P, g)), low = half_at(tile + low_byte<HD>(0, P, g));
    float4 *out = (float4 *)(k + ((size_t)r * kv.heads + w.head) * HD + 32 * g + 8 * c);
    auto value = [&](int i) { return (float)(word >> 4 * i & 15) * step + low; };
    out[0] = make_float4(value(0), value(1), value(2), value(3));
    out[1] = make_float4(value(4), value(5), value(6), value(7));
    return;
  }
  const int q = l % (HD / 4), h = q / 16, j = q % 16;
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int r = w.row + u * (256 / HD) + l / (HD / 4), P = place_of(kv, slots, r, rows, page);
    if (P < 0) continue;
    const uint8_t *tile = tile_of(kv, page, w.head, 1, 10 * HD);
    const uint32_t half =
        *(const uint16_t *)(tile + (((P / 4 * 16 + j) * 2 + P / 2 % 2) * NH + h) * 4 + P % 2 * 2);
    float *out = v + ((size_t)r * kv.heads + w.head) * HD + 64 * h + j;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      out[16 * e] = (float)(half >> 4 * e & 15) * half_at(tile + step_byte<HD>(P, 2 * h + e / 2)) +
                    half_at(tile + low_byte<HD>(1, P, 2 * h + e / 2));
  }
}

// ---------------------------------------------------------------------------
// Attention
// ---------------------------------------------------------------------------
struct AttnArgs {
  Kv4 kv;
  const float *q;
  const int32_t *table;
  size_t max_pages;
  const int32_t *row_start;  // null: lane i has row i alone
  const int32_t *ctx;
  int lanes, max_rows, num_heads, max_ctx;
  float *out;
};

// ---------------------------------------------------------------------------
// Decode attention
// ---------------------------------------------------------------------------
typedef float f4 __attribute__((ext_vector_type(4)));

constexpr int kWaves = 4;             // waves of a workgroup
constexpr int kRing = 2;              // pairs of pages a wave has on their way
constexpr int kUnit = 2 * kWaves * kPage;  // positions that a workgroup's waves take in one go, a pair of pages each
constexpr int kWhole = 4;             // units up to which a context stays one item
constexpr int kMaxSlots = 1024;       // workgroups that a batch is cut for, at most
constexpr float kSlack = 4.0f;        // log2 units a score may pass its reference before a rescale
constexpr float kShift = 11.0f;       // log2 of a weight at the reference
constexpr float kNoRef = -1e30f;      // the reference before the first score
constexpr int kMaxRecords = 2 * kMaxSlots + 2;  // 2 U / Q at most, U the batch's units (Q below)

static __device__ __forceinline__ v8h as_v8h(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  const v4u w = {a, b, c, d};
  return __builtin_bit_cast(v8h, w);
}

// Nibble N of both 16-bit halves of a word as halves (code - mid) * 2^-10, by
// one packed operation on the code's bits (code * 2^-24, or 16 times that).
// An MFMA takes the products of each eight k to 2^-24 of the largest, towards
// zero, and counts a subnormal operand as 2^-14 there: codes left at 2^-24
// cost 1e-5 of the output. V codes go around the middle of their range, 8:
// products of one sign would be cut by a bias that the minima's part does not
// take out again (1e-4 at 2048 positions); with K the query has both signs.
template <int N, bool kMid>
static __device__ __forceinline__ uint32_t code_pair(uint32_t w) {
  const v2h c = __builtin_bit_cast(v2h, w & (N ? 0x00F000F0u : 0x000F000Fu));
  const _Float16 k = N ? (_Float16)0x1p10f : (_Float16)0x1p14f, mid = (_Float16)-0x1p-7f;
  return __builtin_bit_cast(uint32_t, kMid ? __builtin_elementwise_fma(c, v2h{k, k}, v2h{mid, mid}) : c * v2h{k, k});
}

// Eight K codes of a word: nibbles 0, 4, 1, 5, 2, 6, 3, 7.
static __device__ __forceinline__ v8h codes8(uint32_t w) {
  const uint32_t u = w >> 8;
  return as_v8h(code_pair<0, false>(w), code_pair<1, false>(w), code_pair<0, false>(u), code_pair<1, false>(u));
}

// The value of lane N of each 16-lane row.
template <int N>
static __device__ __forceinline__ float row_lane(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x150 + N, 0xF, 0xF, true));
}

// What a wave requests of two pages for one KV head.
template <int HD>
struct Pair {
  static constexpr int NG = HD / 32;
  uint32_t kc[2][NG], vc[2][NG];        // codes
  uint32_t ks[2][2 * NG], vs[2][2 * NG];  // steps [g][4 positions]
  uint32_t km[2][NG / 2];               // minima of position j
  uint32_t vo[2][2], vm[2][2];          // steps and minima of group j (j = NG: a group of ones)
};

template <int N>
static __device__ __forceinline__ void load_words(uint32_t (&d)[N], const uint8_t *p) {
  if constexpr (N == 1) {
    d[0] = *(const uint32_t *)p;
  } else if constexpr (N == 2) {
    const uint2 v = *(const uint2 *)p;
    d[0] = v.x;
    d[1] = v.y;
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const uint4 v = *(const uint4 *)(p + 4 * i);
      d[i] = v.x;
      d[i + 1] = v.y;
      d[i + 2] = v.z;
      d[i + 3] = v.w;
    }
  }
}

// Pairs of pages come through LDS: a wave copies them straight there, kRing
// pairs ahead of the one it works on, each in loads of 16 bytes a lane, and
// reads its operands from its own ring. (Registers hold one pair more than
// the one in use at most, and the latency of a loaded memory takes three.)
// A slot: K codes of both pages in lane order, V codes, then each page's K
// steps, K minima, V steps, V minima.
template <int HD>
struct Slot {
  static constexpr int kCodes = 8 * HD, kMeta = 2 * HD;  // bytes of a tile's codes, steps and minima
  uint8_t kc[2][kCodes], vc[2][kCodes], meta[2][2 * kMeta];
  uint16_t one[8];  // four steps 0 and four minima 1: a group of ones
};
// Loads of a pair (each counts one in vmcnt).
template <int HD>
constexpr int kPairLoads = HD == 128 ? 5 : 3;

// 16 bytes a lane from p (+ off, p the wave's) to LDS base + 16 * lane (M0, which the compiler
// keeps nothing in). The compiler does not see these loads: with its own
// builtin every LDS read waits for all of them. arrive() waits for them, and
// no other wait gets shorter by them (vector memory operations complete in
// order).
static __device__ __forceinline__ void copy16(uint32_t base, const uint8_t *p, uint32_t off) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(base), "v"(off), "s"(p)
               : "memory");
}
static __device__ __forceinline__ void copy16(uint32_t base, const uint8_t *p) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(base), "v"(p)
               : "memory");
}
template <int N>
static __device__ __forceinline__ void arrive() {  // all but the last N vector memory operations
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

template <int HD>
static __device__ __forceinline__ void copy_pair(Slot<HD> *slot, const uint8_t *ta, const uint8_t *tb, int l) {
  constexpr int TILE = 10 * HD, kB = 64 * 16;  // bytes of a load
  const uint32_t at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)slot;
  // the slot's last reads are done
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  if constexpr (HD == 128) {
    const int kc = ((l & 15) * 4 + (l >> 4)) * 16;  // lane (c, j): chunk c of position j
    copy16(at, ta, kc);
    copy16(at + kB, tb, kc);
    copy16(at + 2 * kB, ta, TILE + l * 16);
    copy16(at + 3 * kB, tb, TILE + l * 16);
    const int m = l & 31;
    copy16(at + 4 * kB, (l < 32 ? ta : tb) + (m < 16 ? 8 * HD : TILE + 8 * HD) + (m & 15) * 16);
  } else {
    const uint8_t *t = l < 32 ? ta : tb;
    const int m = l & 31;
    copy16(at, t + m * 16);
    copy16(at + kB, t + TILE + m * 16);
    const int x = l & 15;
    if (l < 32) copy16(at + 2 * kB, (l < 16 ? ta : tb) + (x < 8 ? 8 * HD : TILE + 8 * HD) + (x & 7) * 16);
  }
}

template <int HD>
static __device__ __forceinline__ void read_keys(Pair<HD> &b, const Slot<HD> *s, int l) {
  constexpr int NG = HD / 32;
  const int c = l >> 4, j = l & 15;
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    load_words(b.kc[x], s->kc[x] + (HD == 128 ? l * 16 : j * 32 + c * 8));
    load_words(b.ks[x], s->meta[x] + c * (8 * NG));
    load_words(b.km[x], s->meta[x] + HD + j * (2 * NG));
  }
}

template <int HD>
static __device__ __forceinline__ void read_values(Pair<HD> &b, const Slot<HD> *s, int l) {
  constexpr int NG = HD / 32;
  const int c = l >> 4, j = l & 15;
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const uint8_t *t = s->meta[x] + 2 * HD;
    load_words(b.vc[x], s->vc[x] + l * (4 * NG));
    load_words(b.vs[x], t + c * (8 * NG));
    const uint8_t *one = (const uint8_t *)s->one, *o = t + c * (8 * NG) + min(j, NG - 1) * 8;
    load_words(b.vo[x], j == NG ? one : o);
    load_words(b.vm[x], j == NG ? one + 8 : o + HD);
  }
}

// Steps and minima of positions from n on (of 32) become zero: a stale page
// may hold anything there.
static __device__ __forceinline__ void masks_of(int left, uint32_t &lo, uint32_t &hi) {
  lo = left > 1 ? 0xFFFFFFFFu : left > 0 ? 0xFFFFu : 0u;
  hi = left > 3 ? 0xFFFFFFFFu : left > 2 ? 0xFFFFu : 0u;
}
template <int HD>
static __device__ __forceinline__ void cut_keys(Pair<HD> &b, int n, int l) {
  constexpr int NG = HD / 32;
  const int c = l >> 4, j = l & 15;
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    uint32_t lo, hi;
    masks_of(n - 16 * x - 4 * c, lo, hi);
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      b.ks[x][2 * g] &= lo;
      b.ks[x][2 * g + 1] &= hi;
    }
#pragma unroll
    for (int i = 0; i < NG / 2; ++i) b.km[x][i] = j < n - 16 * x ? b.km[x][i] : 0u;
  }
}
template <int HD>
static __device__ __forceinline__ void cut_values(Pair<HD> &b, int n, int l) {
  constexpr int NG = HD / 32;
  const int c = l >> 4;
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    uint32_t lo, hi;
    masks_of(n - 16 * x - 4 * c, lo, hi);
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      b.vs[x][2 * g] &= lo;
      b.vs[x][2 * g + 1] &= hi;
    }
    b.vo[x][0] &= lo;
    b.vo[x][1] &= hi;
    b.vm[x][0] &= lo;
    b.vm[x][1] &= hi;
  }
}

// The larger of each two halves (as integers: halves that are not negative).
static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
  typedef unsigned short u2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u2, a), __builtin_bit_cast(u2, b)));
}

static __device__ __forceinline__ float half_of(uint32_t w, int hi) {
  return (float)__builtin_bit_cast(v2h, w)[hi];
}

// fp16 of x and y, or with low = 1 of what that leaves of them. Both sides
// round the f32 value: the compiler would otherwise round the product that
// made it straight to fp16 on one of them, and where the two roundings differ
// the parts do not add up.
static __device__ __forceinline__ v2h half_parts(float x, float y, float low) {
  asm("" : "+v"(x), "+v"(y));
  uint32_t h = __builtin_bit_cast(uint32_t, v2h{(_Float16)x, (_Float16)y});
  asm("" : "+v"(h));  // one conversion for the two
  const v2h p = __builtin_bit_cast(v2h, h);
  return v2h{(_Float16)fmaf(-(float)p.x, low, x), (_Float16)fmaf(-(float)p.y, low, y)};
}

// A wave's running state for the query heads of one KV head. Lanes (c, j) =
// 16 c + j: columns j and j + 8 are one query head's fp16 high and low parts.
template <int HD>
struct Wave {
  v8h q[HD / 32];       // query operands, a group a step
  v8h qsum;             // and of the minima: sums of q over each group
  float mult;      // log2 units of a score's accumulator unit, a power of two
  f4 o[HD / 16];   // rows: heads (high, then low parts), columns: dims 16 e + j
  f4 om;           // the middles' part, columns: groups, then the sum of the weights
  float ref;       // log2 units of the head's reference score
  int e;           // V steps are below 2^e
  uint32_t bound;  // 2^e as two halves
};

// New reference of scores that passed the old one by kSlack, or a new bound
// of the V steps: what was summed so far follows. v: scores before mult.
template <int HD>
static __device__ __forceinline__ void raise(Wave<HD> &s, const float (&v)[8], const uint32_t (&steps)[2][2], int l) {
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = fmaxf(top, v[i] * s.mult);
  top = xor32_max(xor16_max(top));  // same in both columns of a head
  const float ref = top - s.ref > kSlack ? top : s.ref, f = exp2f(s.ref - ref);
  s.ref = ref;
  // steps that are no NaN, as integers in their order
  int big = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int a = (int)(steps[i >> 2][i >> 1 & 1] >> 16 * (i & 1) & 0x7FFFu);
    if (a < 0x7C00) big = max(big, a);
  }
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) big = max(big, __shfl_xor(big, m, 64));
  const int old = s.e;
  const int e = big >> 10 == 0 ? -14 : (big >> 10) - 14;  // below 2^e
  s.e = max(old, e);
  s.bound = (uint32_t)(s.e + 15) << 10;
  s.bound |= s.bound << 16;
  const float g = ldexpf(1.0f, old - s.e);
  const int c = l >> 4;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const float fr = __shfl(f, (4 * c + r) & 7, 64);
    s.om[r] *= fr;
#pragma unroll
    for (int e2 = 0; e2 < HD / 16; ++e2) s.o[e2][r] *= fr * g;
  }
}

// Scores of n positions (of 32) of a pair, in units that mult takes to log2:
// lane (c, j) has positions 4 c + r of both pages for column j.
template <int HD>
static __device__ __forceinline__ void scores(const Wave<HD> &s, Pair<HD> &b, int n, int l, float (&v)[8]) {
  constexpr int NG = HD / 32;
  const int c = l >> 4;
  if (n < 32) cut_keys(b, n, l);
  const f4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const v8h m = as_v8h(b.km[x][0], NG == 4 ? b.km[x][NG / 2 - 1] : 0u, 0u, 0u);
    f4 sc = __builtin_amdgcn_mfma_f32_16x16x32_f16(m, s.qsum, zero, 0, 0, 0);
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const f4 acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes8(b.kc[x][g]), s.q[g], zero, 0, 0, 0);
#pragma unroll
      for (int r = 0; r < 4; ++r)
        sc[r] = fmaf(half_of(b.ks[x][2 * g + (r >> 1)], r & 1), acc[r], sc[r]);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) v[4 * x + r] = sc[r] + row_xor8(sc[r]);  // high and low parts of the query
  }
  if (n < 32) {
    asm volatile("");  // (a branch, not selects in every pair)
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (16 * (i >> 2) + 4 * c + (i & 3) >= n) v[i] = -INFINITY;
  }
}

// Adds the pair's values with those scores to the state.
template <int HD>
static __device__ __forceinline__ void weigh(Wave<HD> &s, Pair<HD> &b, int n, int l, const float (&v)[8]) {
  constexpr int NG = HD / 32, NH = HD / 64;
  const int j = l & 15;
  if (n < 32) cut_values(b, n, l);
  const float top = fmaxf(fmaxf(fmaxf(fmaxf(v[0], v[1]), v[2]), fmaxf(fmaxf(v[3], v[4]), v[5])), fmaxf(v[6], v[7]));
  const bool over = max2(max2(max2(b.vo[0][0], b.vo[0][1]), max2(b.vo[1][0], b.vo[1][1])), s.bound) != s.bound;
  if (__any(fmaf(top, s.mult, -s.ref) > kSlack || over)) raise(s, v, b.vo, l);
  const float unit = ldexpf(1.0f, -s.e), low = j < 8 ? 0.0f : 1.0f;
  const float shift = kShift - s.ref;
  float p[8], pu[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    p[i] = __builtin_amdgcn_exp2f(fmaf(v[i], s.mult, shift));
    pu[i] = p[i] * unit;
  }
  auto part = [&](const float (&x)[8]) {
    v8h a;
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      const v2h h = half_parts(x[i], x[i + 1], low);
      a[i] = h.x;
      a[i + 1] = h.y;
    }
    return a;
  };
  v8h mid, rest;  // the middle of group j's range, code 8, in two parts
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    const uint32_t o = b.vo[i >> 2][(i & 3) >> 1], m = b.vm[i >> 2][(i & 3) >> 1];
    float y = fmaf(8.0f, half_of(o, 0), half_of(m, 0)), z = fmaf(8.0f, half_of(o, 1), half_of(m, 1));
    asm("" : "+v"(y), "+v"(z));
    uint32_t h = __builtin_bit_cast(uint32_t, v2h{(_Float16)y, (_Float16)z});
    asm("" : "+v"(h));
    const v2h p = __builtin_bit_cast(v2h, h);
    mid[i] = p.x;
    mid[i + 1] = p.y;
    rest[i] = (_Float16)(y - (float)p.x);
    rest[i + 1] = (_Float16)(z - (float)p.y);
  }
  const v8h pp = part(p);
  s.om = __builtin_amdgcn_mfma_f32_16x16x32_f16(pp, mid, s.om, 0, 0, 0);
  s.om = __builtin_amdgcn_mfma_f32_16x16x32_f16(pp, rest, s.om, 0, 0, 0);
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      x[i] = fmaf(half_of(b.vs[i >> 2][2 * g + ((i & 3) >> 1)], i & 1), pu[i], 0.0f);
    const v8h a = part(x);
    // blocks 2 g, 2 g + 1: nibbles 2 (g % 2), + 1 of the words of unit g / 2
    const int h = g >> 1, sh = 8 * (g & 1);
    const uint32_t w[4] = {b.vc[0][h] >> sh, b.vc[0][NH + h] >> sh, b.vc[1][h] >> sh,
                           b.vc[1][NH + h] >> sh};
    s.o[2 * g] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
        a, as_v8h(code_pair<0, true>(w[0]), code_pair<0, true>(w[1]), code_pair<0, true>(w[2]), code_pair<0, true>(w[3])),
        s.o[2 * g], 0, 0, 0);
    s.o[2 * g + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
        a, as_v8h(code_pair<1, true>(w[0]), code_pair<1, true>(w[1]), code_pair<1, true>(w[2]), code_pair<1, true>(w[3])),
        s.o[2 * g + 1], 0, 0, 0);
  }
}

// The query operands of one row's heads: q log2(e) / sqrt(HD) = 2^e q', the
// largest |q'| of a head in [2^13, 2^14), split into fp16 high and low parts.
// The waves of a workgroup split a group each and share them in LDS.
template <int HD>
struct QueryLds {
  v8h q[HD / 32][64];
  float sum[HD / 32][16];  // of the group, by column
};
template <int HD>
static __device__ __forceinline__ void load_query(Wave<HD> &s, QueryLds<HD> &lds, const float *q, int G,
                                                  int w, int l) {
  constexpr int NG = HD / 32;
  const int c = l >> 4, j = l & 15, head = j & 7;
  const float unit = 1.44269504088896341f / sqrtf((float)HD);
  float4 v[NG][2];
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    const float *p = q + (size_t)(head < G ? head : 0) * HD + 32 * g + 8 * c;
    v[g][0] = *(const float4 *)p;
    v[g][1] = *(const float4 *)(p + 4);
  }
  float top = 0.0f;
#pragma unroll
  for (int g = 0; g < NG; ++g)
#pragma unroll
    for (int i = 0; i < 2; ++i)
      top = fmaxf(fmaxf(fmaxf(fmaxf(top, fabsf(v[g][i].x)), fabsf(v[g][i].y)), fabsf(v[g][i].z)), fabsf(v[g][i].w));
  top = xor32_max(xor16_max(top)) * unit;
  // (a query below 2^-106 stays below 2^13)
  const int e = max(top > 0.0f ? __builtin_amdgcn_frexp_expf(top) - 14 : 0, -120);
  s.mult = ldexpf(1.0f, e + 10);
  const float scale = head < G ? ldexpf(1.0f, -e) : 0.0f, low = j < 8 ? 0.0f : 1.0f;
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    if (w % NG != g) continue;
    const float x[8] = {v[g][0].x, v[g][0].y, v[g][0].z, v[g][0].w, v[g][1].x, v[g][1].y, v[g][1].z, v[g][1].w};
    float y[8], sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      y[i] = x[i] * unit * scale;
      sum += y[i];
    }
    sum = xor32_add(xor16_add(sum)) * 0x1p-10f;  // (codes come times 2^-10)
    constexpr int order[8] = {0, 4, 1, 5, 2, 6, 3, 7};  // of codes8
    v8h o;
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      const v2h h = half_parts(y[order[i]], y[order[i + 1]], low);
      o[i] = h.x;
      o[i + 1] = h.y;
    }
    if (w < NG) {
      lds.q[g][l] = o;
      if (l < 16) lds.sum[g][l] = sum;
    }
  }
  __syncthreads();
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    s.q[g] = lds.q[g][l];
    const float sum = lds.sum[g][j];
    // high and low parts in the columns, what both leave in a second k-chunk
    const _Float16 sh = (_Float16)sum, sl = (_Float16)(sum - (float)sh);
    const float rest = (sum - (float)sh) - (float)sl;
    s.qsum[g] = (_Float16)(c == 0 ? (j < 8 ? (float)sh : (float)sl) : c == 1 && j < 8 ? rest : 0.0f);
  }
#pragma unroll
  for (int g = NG; g < 8; ++g) s.qsum[g] = (_Float16)0.0f;
}

struct WorkItem {
  int lane, head, ctx, chunk, chunks, start, most;  // lane < 0: none
};

// n / d rounded up, n < 2^24.
static __device__ __forceinline__ int ceil_div(int n, int d, float rd) {
  int q = (int)((float)n * rd);
  q += q * d < n;
  q -= (q - 1) * d >= n;
  return q;
}

// Item blockIdx.x of the list, by one wave (l its thread): a thread holds
// a.lanes / 64 lanes. lens: the lanes' lengths, 0 for those that do not hold.
static __device__ __forceinline__ WorkItem find_item(const AttnArgs &a, const int *lens, int slots, int l) {
  const int per = (a.lanes + 63) / 64, Hkv = a.kv.heads;
  auto pages_of = [&](int i) {
    const int at = l * per + i;
    return at < a.lanes ? (lens[at] + kUnit - 1) / kUnit : 0;
  };
  const int only = pages_of(0);
  int mine = only, live = only > 0;
  for (int i = 1; i < per; ++i) {
    const int p = pages_of(i);
    mine += p;
    live += p > 0;
  }
  const int pages_in = wave_scan(mine);
  const int total = __builtin_amdgcn_readlane(pages_in, 63) * Hkv;
  const int segments = __builtin_amdgcn_readlane(wave_scan(live), 63) * Hkv;
  auto chunks_of = [&](int q) {  // of the thread's lanes
    const float r = 1.0f / (float)q;
    int n = ceil_div(only, q, r);
    for (int i = 1; i < per; ++i) n += ceil_div(pages_of(i), q, r);
    return n;
  };
  const int room = max(slots - segments, slots / 2);
  int Q = max(1, (total + room - 1) / room);
  if (Q > 1 && segments < slots / 2) {
    // Q leaves slots items at most; try k / 4 of the way down to the mean
    const int full = Q, low = max(1, (total + slots - 1) / slots), step = (Q - low + 3) / 4;
#pragma unroll
    for (int k = 1; k < 4; ++k) {
      const int q = max(low, full - k * step);
      if (__builtin_amdgcn_readlane(wave_scan(chunks_of(q)), 63) * Hkv <= slots) Q = q;
    }
  }
  const int count = chunks_of(Q) * Hkv, last = wave_scan(count);
  const int item = blockIdx.x;
  WorkItem m{-1, 0, 0, 0, 0, 0, Q};
  const uint64_t past = __ballot(last > item);
  if (past == 0) return m;
  const int owner = __builtin_ctzll(past);
  // the owner's lanes, by every thread alike
  int at = __builtin_amdgcn_readlane(last - count, owner), pb = __builtin_amdgcn_readlane(pages_in - mine, owner);
  const float r = 1.0f / (float)Q;
  for (int i = 0; i < per; ++i) {
    const int lane = owner * per + i, n = lane < a.lanes ? lens[lane] : 0, p = (n + kUnit - 1) / kUnit;
    const int chunks = ceil_div(p, Q, r), k = item - at;
    if (k < chunks * Hkv) {
      const int head = k / chunks;
      m = {lane, head, n, k - head * chunks, chunks, pb * Hkv + head * p, Q};
      break;
    }
    at += chunks * Hkv;
    pb += p;
  }
  return m;
}

template <int HD>
struct DecodeLds {
  union {
    Slot<HD> ring[kWaves][kRing];
    float o[kWaves][kMaxGroup][HD];
    int lens[kMaxLanes];
  };
  float ref[kWaves][kMaxGroup], sum[kWaves][kMaxGroup], f[kWaves][kMaxGroup];
  QueryLds<HD> query;
  WorkItem item;
};

struct MergeItem {  // of a (lane, KV head): its chunks' records
  int start, units, chunks, half;
};
// First unit of chunk ch; a chunk's record is the place of its first unit in
// the batch divided by half the most units of a chunk.
static __device__ __forceinline__ int chunk_first(int ch, int units, int chunks) {
  return ch * (units / chunks) + min(ch, units % chunks);
}

// Work items: (lane, KV head, chunk of its units), a workgroup each; a unit is
// what its waves take in one go. Q, the most units of a chunk, comes from the
// batch's own lengths: the smallest of a few that leaves no more items than
// the device holds workgroups (`slots`), so that they all run at once and end
// together. (With more than slots / 2 contexts: 2 U / slots, U the batch's
// units.) The chunks of a context are of equal size
// to a unit, so where there are several they hold (Q + 1) / 2 units at least.
// (Chunks equal to a page instead, whose last round leaves waves idle, take a
// context of 32000 4 us more and 128 of 500 to 1500 1.2, the 32 below 1 less.)
//
// 32 contexts of 1 to 8192, 28 heads of 128 over 4 (89 MB of pages): 34.5 us
// with the merge, 31 without; the bytes take 13 at the rate of a large read.
// What bounds it is vector instructions, 1.4 us a pair of pages and SIMD:
// sixteen weights, their splits, and unpacking; 1.9 us find the item, 2.2 join
// the waves. One wave a (lane, query head) took 6479 us; the same products on
// pages loaded to registers instead of the LDS ring 48.5. Contexts of at most kWhole units are
// not cut, so that no merge follows: its launch costs 3 to 4 us, a unit 1.5.
template <int HD>
__global__ __launch_bounds__(64 * kWaves, HD == 128 ? 3 : 4) void kv4_decode_kernel(
    AttnArgs a, int slots, MergeItem *merge, float *records) {
  __shared__ __align__(16) DecodeLds<HD> s;
  const int t = threadIdx.x, l = t & 63, w = __builtin_amdgcn_readfirstlane(t >> 6);
  const int c = l >> 4, j = l & 15;
  const int Hkv = a.kv.heads, G = a.num_heads / Hkv;
  const float nan = __uint_as_float(0x7FC00000u);

  // a lane without positions, or with a length that does not hold
  if ((int)blockIdx.x < a.lanes) {
    const int n = a.ctx[blockIdx.x];
    if (n <= 0 || n > a.max_ctx) {
      for (int i = t; i < a.num_heads * HD; i += 64 * kWaves)
        a.out[(size_t)blockIdx.x * a.num_heads * HD + i] = n == 0 ? 0.0f : nan;
      if (merge)
        for (int i = t; i < Hkv; i += 64 * kWaves) merge[blockIdx.x * Hkv + i].chunks = 0;
    }
  }
  int lane, h, ctx, ch = 0, chunks = 1, start = 0, Q = 1;
  if (merge) {
    for (int i = t; i < a.lanes; i += 64 * kWaves) {
      const int n = a.ctx[i];
      s.lens[i] = n > 0 && n <= a.max_ctx ? n : 0;
    }
    __syncthreads();
    if (w == 0) {
      const WorkItem m = find_item(a, s.lens, slots, l);
      if (l == 0) s.item = m;
    }
    __syncthreads();
    lane = __builtin_amdgcn_readfirstlane(s.item.lane);
    if (lane < 0) return;
    h = __builtin_amdgcn_readfirstlane(s.item.head);
    ctx = __builtin_amdgcn_readfirstlane(s.item.ctx);
    ch = __builtin_amdgcn_readfirstlane(s.item.chunk);
    chunks = __builtin_amdgcn_readfirstlane(s.item.chunks);
    start = __builtin_amdgcn_readfirstlane(s.item.start);
    Q = __builtin_amdgcn_readfirstlane(s.item.most);
  } else {  // contexts are items
    lane = blockIdx.x / Hkv;
    if (lane >= a.lanes) return;
    h = blockIdx.x - lane * Hkv;
    ctx = a.ctx[lane];
    if (ctx <= 0 || ctx > a.max_ctx) return;
  }
  const int lane_pages = (ctx + kPage - 1) / kPage;
  const int units = (ctx + kUnit - 1) / kUnit, first_unit = chunk_first(ch, units, chunks), half = (Q + 1) / 2;
  const int first = first_unit * (kUnit / kPage);
  const int end = min(chunk_first(ch + 1, units, chunks) * (kUnit / kPage), lane_pages);
  if (merge && ch == 0 && t == 0) merge[lane * Hkv + h] = {start, units, chunks, half};

  Wave<HD> s_w;
#pragma unroll
  for (int e = 0; e < HD / 16; ++e) s_w.o[e] = f4{0.0f, 0.0f, 0.0f, 0.0f};
  s_w.om = f4{0.0f, 0.0f, 0.0f, 0.0f};
  s_w.ref = kNoRef;
  s_w.e = -14;
  s_w.bound = 1u << 10 | 1u << 26;
  load_query(s_w, s.query, a.q + ((size_t)lane * a.num_heads + h * G) * HD, G, w, l);

  if (l < kRing * 8) s.ring[w][l >> 3].one[l & 7] = (l & 7) < 4 ? 0 : 0x3C00;
  // a wave takes pairs of pages w, w + kWaves, ... of the chunk
  const int32_t *table = a.table + (size_t)lane * a.max_pages;
  const uint8_t *head_base = a.kv.base + (size_t)(2 * h) * (10 * HD);
  int bad = 0;
  const int stop = min(ctx, end * kPage);
  for (int p0 = first + 2 * w; p0 < end; p0 += 64 * kWaves) {
    // ids of the next 32 pairs, two lanes a pair (a page past the chunk: its first one)
    const int at = p0 + (l >> 1) * (2 * kWaves) + (l & 1);
    uint32_t id = (uint32_t)table[at < end ? at : first];
    if (id >= a.kv.page_count) {
      bad = 1;
      id = 0;
    }
    const int n = min(32, (end - p0 + 2 * kWaves - 1) / (2 * kWaves));  // pairs
    auto tile = [&](int i, int x) {
      return head_base + (size_t)(uint32_t)__builtin_amdgcn_readlane((int)id, 2 * i + x) * a.kv.page_bytes;
    };
    // (past the last pair it is requested again and not used)
    auto request = [&](int i) {
      const int k = min(i, n - 1);
      copy_pair(&s.ring[w][i % kRing], tile(k, 0), tile(k, 1), l);
    };
    for (int i = 0; i < kRing; ++i) request(i);
    for (int i = 0; i < n; ++i) {
      const int left = min(32, stop - (p0 + i * 2 * kWaves) * kPage);
      const Slot<HD> *slot = &s.ring[w][i % kRing];
      arrive<(kRing - 1) * kPairLoads<HD>>();
      Pair<HD> b;
      float x[8];
      read_keys(b, slot, l);
      scores(s_w, b, left, l, x);
      read_values(b, slot, l);
      weigh(s_w, b, left, l, x);
      request(i + kRing);
    }
  }
  arrive<0>();
  __syncthreads();  // the ring's room takes the waves' outputs

  // the waves' states, then their sums weighted by 2^(reference - the
  // largest). High and low parts are rows 4 c + r and 8 more, 32 lanes apart:
  // a swap of blocks e and e + HD / 32 leaves both parts of e in the lower
  // lanes, of the other in the upper ones.
  const float unit = ldexpf(1.0f, s_w.e + 10);
  float om[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) om[r] = xor32_add(s_w.om[r]);
#pragma unroll
  for (int e = 0; e < HD / 32; ++e)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const v2u x = __builtin_amdgcn_permlane32_swap(__float_as_uint(s_w.o[e][r]),
                                                     __float_as_uint(s_w.o[e + HD / 32][r]), false, false);
      const float m = l < 32 ? (e / 2 == 0 ? row_lane<0>(om[r]) : row_lane<1>(om[r]))
                      : HD == 64 ? row_lane<1>(om[r])
                                 : (e / 2 == 0 ? row_lane<2>(om[r]) : row_lane<3>(om[r]));
      s.o[w][4 * (c & 1) + r][16 * e + (l < 32 ? 0 : HD / 2) + j] =
          fmaf(__uint_as_float(x.x) + __uint_as_float(x.y), unit, m);
    }
  if (l < kMaxGroup) s.ref[w][l] = s_w.ref;
#pragma unroll
  for (int r = 0; r < 4; ++r)
    if (c < 2 && j == HD / 32) s.sum[w][4 * c + r] = om[r];
  bad = __syncthreads_or(bad);
  if (t < kMaxGroup) {
    float top = s.ref[0][t], L = 0.0f;
#pragma unroll
    for (int v = 1; v < kWaves; ++v) top = fmaxf(top, s.ref[v][t]);
#pragma unroll
    for (int v = 0; v < kWaves; ++v) {
      const float f = __builtin_amdgcn_exp2f(s.ref[v][t] - top);
      s.f[v][t] = f;
      L = fmaf(s.sum[v][t], f, L);
    }
    s.ref[0][t] = top;
    s.sum[0][t] = bad ? nan : L;
  }
  __syncthreads();
  float *rec = records + (size_t)((start + first_unit) / half) * (kMaxGroup * (HD + 2));
  for (int i = t; i < G * HD; i += 64 * kWaves) {
    const int g = i / HD, d = i % HD;
    const float L = s.sum[0][g];
    float O = 0.0f;
#pragma unroll
    for (int v = 0; v < kWaves; ++v) O = fmaf(s.o[v][g][d], s.f[v][g], O);
    if (chunks == 1) {
      a.out[((size_t)lane * a.num_heads + h * G + g) * HD + d] = O / L;
    } else {
      rec[g * (HD + 2) + 2 + d] = O;
      if (d == 0) {
        rec[g * (HD + 2)] = s.ref[0][g];
        rec[g * (HD + 2) + 1] = L;
      }
    }
  }
}

// The chunks of a (lane, query head) added up, weighted by 2^(reference - the
// largest): HD / 4 threads for each of 1024 / HD shares of the chunks, four
// chunks' loads on their way at a time; the shares meet in LDS, in a fixed
// order. 3.8 us, most of it a launch; with references, sums and records read one after
// the other 5.3, and 17.0 instead of 15.3 us for four lanes of 512 to 8192.
template <int HD>
__global__ __launch_bounds__(256) void kv4_merge_kernel(AttnArgs a, const MergeItem *merge,
                                                        const float *records) {
  constexpr int TPR = HD / 4, R = 256 / TPR, AT_ONCE = 4;
  __shared__ float4 o_s[R][TPR];
  __shared__ float2 stat[R];
  const int t = threadIdx.x, part = t / TPR, d = t % TPR * 4;
  const int lane = blockIdx.x / a.num_heads, qh = blockIdx.x % a.num_heads;
  const int G = a.num_heads / a.kv.heads, g = qh % G;
  const MergeItem m = merge[lane * a.kv.heads + qh / G];
  if (m.chunks <= 1) return;
  float top = kNoRef, sum = 0.0f;
  float4 o = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int i = part; i < m.chunks; i += AT_ONCE * R) {
    float2 rs[AT_ONCE], x[AT_ONCE], y[AT_ONCE];
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j) {
      const int at = (m.start + chunk_first(min(i + j * R, m.chunks - 1), m.units, m.chunks)) / m.half;
      const float *p = records + ((size_t)at * kMaxGroup + g) * (HD + 2);
      rs[j] = *(const float2 *)p;
      x[j] = *(const float2 *)(p + 2 + d);
      y[j] = *(const float2 *)(p + 4 + d);
    }
    float high = top;
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j)
      if (i + j * R < m.chunks) high = fmaxf(high, rs[j].x);
    const float f = __builtin_amdgcn_exp2f(top - high);
    top = high;
    sum *= f;
    o = {o.x * f, o.y * f, o.z * f, o.w * f};
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j)
      if (i + j * R < m.chunks) {
        const float e = __builtin_amdgcn_exp2f(rs[j].x - top);
        sum = fmaf(rs[j].y, e, sum);
        o = {fmaf(x[j].x, e, o.x), fmaf(x[j].y, e, o.y), fmaf(y[j].x, e, o.z), fmaf(y[j].y, e, o.w)};
      }
  }
  o_s[part][t % TPR] = o;
  if (d == 0) stat[part] = {top, sum};
  __syncthreads();
  if (t < HD) {
    float high = stat[0].x, v = 0.0f, total = 0.0f;
#pragma unroll
    for (int r = 1; r < R; ++r) high = fmaxf(high, stat[r].x);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const float e = __builtin_amdgcn_exp2f(stat[r].x - high);
      v = fmaf(((const float *)&o_s[r][t / 4])[t % 4], e, v);
      total = fmaf(stat[r].y, e, total);
    }
    a.out[((size_t)lane * a.num_heads + qh) * HD + t] = v / total;
  }
}

// ---------------------------------------------------------------------------
// Attention of row runs
// ---------------------------------------------------------------------------
// Columns are (row, query head of the KV head), a row's heads together, so a
// run of any length and any group size fills tiles of 32 columns a wave, 128
// a workgroup (a tile). The workgroup walks the keys 32 at a time: two pages'
// codes become values in LDS once for all columns, each as an fp16 high and
// low part (a value keeps 22 bits; the codes' steps do not fit the operands
// as they do with one row a head, whose weights take them). The pages come
// through an LDS ring, asked for three stages ahead by the waves in turn. V is
// unpacked between the products of the scores, the next stage's K between
// those of the output, so that vector instructions run beside the matrix
// ones; a barrier follows each:
//   scores  S^T = K . Q^T on v_mfma_f32_32x32x16_f16, high.high + high.low +
//           low.high; lane (h, col) ends with keys 8 (i / 4) + 4 h + i % 4
//           of its own column in register i,
//   softmax in registers, a column's reference in its two lanes; it follows
//           the scores only when one passes it by kSlack, so a stage takes
//           no cross-lane step,
//   output  O^T += V^T . P^T: the B operand is the lane's own registers (V's
//           keys are laid out in their order), so rescaling is lane-local.
// Long contexts of few columns are cut into chunks of stages (records, merged
// below) so that they spread over the device.
//
// A prompt of 2048 rows, 28 heads of 128 over 4: 131 us, 30 GFLOP, or 690
// TFLOP/s of the three fp16 products that make one (a large library product
// reaches 1343). A workgroup alone on a CU takes 2.05 us a stage, two 1.75 us a
// stage between them; the matrix unit is busy 41 % of that and vector
// instructions issue 54 %, and the two add up more than they overlap. 161 us
// with the unpacking apart from the products. Registers (256: outputs and both
// parts of the queries take 128) leave no third workgroup.
typedef float f16v __attribute__((ext_vector_type(16)));
constexpr int kTile = 128;        // columns of a workgroup
constexpr int kStage = 32;        // keys of a stage
// Stages of a chunk at least, and stages up to which contexts stay whole, so
// that no merge follows: at least 8, 4 and 2 stages a chunk take six drafting
// lanes 19.2, 15.3 and 15.0 us, 16 rows at the end of 1000 26.6, 20.0 and 17.1.
constexpr int kMinStages = 2, kWholeStages = 8;
constexpr int kRowsRing = 4;      // stages whose pages are in LDS or on their way
constexpr int kRowsSlots = 512;   // workgroups that a batch is cut for, at most
constexpr int kRowsRecords = kRowsSlots;  // chunks of cut tiles at most
constexpr size_t kRowsHeader = 16384;  // workspace: the cut tiles' count and places, then records

template <int HD>
struct RowsLds {
  // [step][high, low][lane] operands of K, [32 dims][16 keys][high, low][lane] of V
  uint8_t k[HD / 16][2][1024], v[HD / 32][2][2][1024];
  Slot<HD> ring[kRowsRing];  // the pages of the stages ahead
  int bad[kRowsRing];        // which of a slot's two pages lie outside the pool
  // keys whose V group is no number, by group, and whether there are any: of
  // this stage and the one before
  uint32_t odd[2][HD / 32 + 1];
  int item[8];
};

struct RowsItem {
  int lane, head, tile, chunk, chunks, record, split;  // lane < 0: none
};
struct RowsTile {  // a cut tile, for the merge
  int first, head, col, cols, chunks, record;  // its run's first row, its first column of the run's
};

static __device__ __forceinline__ float wave_scan_f(float v) {
  auto d = [](float x, auto f) { return x + __int_as_float(f(__float_as_int(x))); };
  v = d(v, [](int x) { return __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, true); });
  v = d(v, [](int x) { return __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, true); });
  v = d(v, [](int x) { return __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, true); });
  v = d(v, [](int x) { return __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, true); });
  v = d(v, [](int x) { return __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false); });
  return d(v, [](int x) { return __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false); });
}

// Rows of a lane (first, count; none where the run does not lie in the rows).
static __device__ __forceinline__ void run_of(const AttnArgs &a, int lane, int &first, int &n) {
  first = lane < a.lanes ? a.row_start[lane] : 0;
  const int end = lane < a.lanes ? a.row_start[lane + 1] : 0;
  n = first >= 0 && first < end && end <= a.max_rows ? end - first : 0;  // (no difference that wraps)
}

// Work items: (lane, tile, KV head, chunk), the tiles of a lane from its last
// on (the longest), by one wave; a thread holds lanes / 64 lanes. A lane's
// tiles are cut into as many chunks as its longest has shares Q of stages: the
// smallest Q of a few multiples of a slot's mean that leaves no more items
// than slots, or than the tiles and half the slots more. (A prompt that fills
// the device with whole tiles so stays whole: 2048 rows cut in two took 151 us
// instead of 133, 512 rows at the end of 4096 108 instead of 138.)
// The list is dealt in runs of 256 (a CU each), every other one backwards, so
// that CUs pair long items with short ones.
// runs: the lanes' rows and stages.
static __device__ __forceinline__ RowsItem find_rows_item(const AttnArgs &a, const int2 *runs, int slots, bool split,
                                                          int l, int *cut_tiles) {
  const int per = (a.lanes + 63) / 64, Hkv = a.kv.heads, G = a.num_heads / Hkv;
  auto tiles_of = [&](int i, int &stages, int &n) {
    const int at = l * per + i;
    const int2 r = at < a.lanes ? runs[at] : int2{0, 0};
    n = r.x;
    stages = r.y;
    return (n * G + kTile - 1) / kTile;
  };
  int n0, st0;
  const int tiles0 = tiles_of(0, st0, n0);
  int Q = 1 << 30;
  if (split) {
    float work = (float)tiles0 * ((float)st0 - 0.5f * (float)n0 / kStage);
    for (int i = 1; i < per; ++i) {
      int st, n;
      const int tiles = tiles_of(i, st, n);
      work += (float)tiles * ((float)st - 0.5f * (float)n / kStage);
    }
    work = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(wave_scan_f(work)), 63)) * (float)Hkv;
    auto items_of = [&](int q) {
      int items = tiles0 * max(1, (st0 + q - 1) / q);
      for (int i = 1; i < per; ++i) {
        int st, n;
        const int tiles = tiles_of(i, st, n);
        items += tiles * max(1, (st + q - 1) / q);
      }
      return __builtin_amdgcn_readlane(wave_scan(items), 63) * Hkv;
    };
    const int room = max(slots, items_of(Q) + slots / 2);
    for (int k = 4; k <= 16; k += 2) {  // quarters of the mean
      const int q = max(kMinStages, (int)fminf(work * (float)k / (4.0f * (float)slots), 1e9f) + 1);
      if (items_of(q) <= room) {
        Q = q;
        break;
      }
    }
  }
  int count = 0, cut = 0, cut_items = 0, rows = 0;
  for (int i = 0; i < per; ++i) {
    int st = st0, n = n0;
    const int tiles = i == 0 ? tiles0 : tiles_of(i, st, n), chunks = max(1, (st + Q - 1) / Q);
    rows += n;
    count += tiles * Hkv * chunks;
    if (chunks > 1) {
      cut += tiles * Hkv;
      cut_items += tiles * Hkv * chunks;
    }
  }
  const int last = wave_scan(count), cut_last = wave_scan(cut), rec_last = wave_scan(cut_items);
  // runs of more rows than there are (they overlap) have no items: the grid
  // holds those of max_rows rows
  const bool fits = __builtin_amdgcn_readlane(wave_scan(rows), 63) <= a.max_rows;
  const int all = fits ? __builtin_amdgcn_readlane(last, 63) : 0;
  *cut_tiles = fits ? __builtin_amdgcn_readlane(cut_last, 63) : 0;
  RowsItem m{-1, 0, 0, 0, 0, 0, 0};
  int item = blockIdx.x;
  if (item >= all) return m;
  const int run = item & ~255;
  if (item & 256) item = run + min(256, all - run) - 1 - (item - run);
  const int owner = __builtin_ctzll(__ballot(last > item));
  int at = __builtin_amdgcn_readlane(last - count, owner), tile_at = __builtin_amdgcn_readlane(cut_last - cut, owner);
  int rec_at = __builtin_amdgcn_readlane(rec_last - cut_items, owner);
  for (int i = 0; i < per; ++i) {
    const int lane = owner * per + i;
    const int2 run_here = lane < a.lanes ? runs[lane] : int2{0, 0};
    const int n = run_here.x, st = run_here.y;
    const int tiles = (n * G + kTile - 1) / kTile, chunks = max(1, (st + Q - 1) / Q), k = item - at;
    const int here = tiles * Hkv * chunks;
    if (k < here) {
      const int u = k / chunks;
      m = {lane, u % Hkv, tiles - 1 - u / Hkv, k - u * chunks, chunks, rec_at + k, tile_at + u};
      break;
    }
    at += here;
    if (chunks > 1) {
      tile_at += tiles * Hkv;
      rec_at += here;
    }
  }
  return m;
}

// What a thread turns into values of a stage: GPT = HD / 64 groups (those of
// half t / 128) of a K chunk (page, position, 8 dims c of a group) or of a V
// chunk (page, four positions c, column j).
template <int HD>
struct RawKeys {
  uint32_t code[HD / 64], step[HD / 64], low[HD / 64];
};
template <int HD>
struct RawValues {
  uint32_t code[2], step[HD / 32], low[HD / 32];
};

template <int HD>
static __device__ __forceinline__ RawKeys<HD> raw_keys(const Slot<HD> &s, int page, int part, int l) {
  constexpr int NG = HD / 32, GPT = HD / 64;
  const int c = l >> 4, j = l & 15, g0 = part * GPT;
  RawKeys<HD> r;
  load_words(r.code, s.kc[page] + (HD == 128 ? l * 16 : j * 32 + c * 8) + g0 * 4);
#pragma unroll
  for (int g = 0; g < GPT; ++g) {
    r.step[g] = *(const uint16_t *)(s.meta[page] + 2 * ((j >> 2) * (4 * NG) + (g0 + g) * 4 + (j & 3)));
    r.low[g] = *(const uint16_t *)(s.meta[page] + HD + 2 * (j * NG + g0 + g));
  }
  return r;
}
template <int HD>
static __device__ __forceinline__ RawValues<HD> raw_values(const Slot<HD> &s, int page, int part, int l) {
  constexpr int NG = HD / 32, GPT = HD / 64;
  const int c = l >> 4, g0 = part * GPT;
  RawValues<HD> r;
  // unit h = the half of a position pair's words
#pragma unroll
  for (int pr = 0; pr < 2; ++pr)
    r.code[pr] = *(const uint32_t *)(s.vc[page] + l * (4 * NG) + (pr * (HD / 64) + (HD == 128 ? part : 0)) * 4);
  load_words(r.step, s.meta[page] + 2 * HD + (c * NG + g0) * 8);
  load_words(r.low, s.meta[page] + 3 * HD + (c * NG + g0) * 8);
  return r;
}

// fp16 high and low parts of two values: the high one truncated, so that the
// rest is what a mask leaves, that one rounded.
static __device__ __forceinline__ void two_parts(float x, float y, uint32_t &high, uint32_t &low) {
  const float rx = x - __uint_as_float(__float_as_uint(x) & 0xFFFFE000u);
  const float ry = y - __uint_as_float(__float_as_uint(y) & 0xFFFFE000u);
  high = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(x, y));
  low = __builtin_bit_cast(uint32_t, v2h{(_Float16)rx, (_Float16)ry});
}

// The words become unknown to the compiler, which would move what both arms
// of a branch compute from them ahead of it, out of the matrix products' shadow.
template <int N>
static __device__ __forceinline__ void keep_here(uint32_t (&w)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+v"(w[i]));
}

// V positions past the context (left of the thread's four are inside), of no
// page or with no number become zeros; the last are noted for their groups,
// so that they reach the rows that see them and no others.
template <int HD>
static __device__ __forceinline__ void clean_values(uint32_t *notes, RawValues<HD> &r, int page, int part, int l,
                                                    int keys, bool bad) {
  constexpr int NG = HD / 32, GPT = HD / 64;
  const int c = l >> 4, left = keys - 16 * page - 4 * c;
  uint32_t most = 0;
#pragma unroll
  for (int i = 0; i < 2 * GPT; ++i) most = max2(most, max2(r.step[i] & 0x7FFF7FFFu, r.low[i] & 0x7FFF7FFFu));
  if (!__any(bad || left < 4 || max2(most, 0x7BFF7BFFu) != 0x7BFF7BFFu)) return;
#pragma unroll
  for (int g = 0; g < GPT; ++g)
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      const int i = 2 * g + (p >> 1), sh = 16 * (p & 1);
      const bool none = bad || p >= left;
      const bool nan = (r.step[i] >> sh & 0x7C00u) == 0x7C00u || (r.low[i] >> sh & 0x7C00u) == 0x7C00u;
      if (none || nan) {
        r.step[i] &= ~(0xFFFFu << sh);
        r.low[i] &= ~(0xFFFFu << sh);
      }
      if (nan && !none && (l & 15) == 0) {
        atomicOr(&notes[part * GPT + g], 1u << (16 * page + 4 * c + p));
        atomicOr(&notes[NG], 1u);
      }
    }
}

// The thread's K or V values as operands, a part at a time so that a few
// vector instructions can go between matrix products. K: two values of a
// group (part n of 4 GPT), the fourth two write the chunk.
template <int HD>
struct KeyChunk {
  uint32_t even, odd, hi[4], lo[4];
};
template <int HD>
static __device__ __forceinline__ void key_part(RowsLds<HD> &s, const RawKeys<HD> &r, KeyChunk<HD> &o, int n, int page,
                                                int part, int l, bool bad) {
  const int i = n >> 2, k = n & 3;
  if (k == 0) {
    o.even = r.code[i] & 0x0F0F0F0Fu;
    o.odd = r.code[i] >> 4 & 0x0F0F0F0Fu;
  }
  const float step = bad ? __uint_as_float(0x7FC00000u) : half_of(r.step[i], 0), low = half_of(r.low[i], 0);
  two_parts(fmaf((float)(o.even >> 8 * k & 0xFFu), step, low), fmaf((float)(o.odd >> 8 * k & 0xFFu), step, low),
            o.hi[k], o.lo[k]);
  if (k < 3) return;
  const int c = l >> 4, j = l & 15, at = (32 * (c & 1) + 16 * page + j) * 16, g = part * (HD / 64) + i;
  *(uint4 *)(s.k[2 * g + (c >> 1)][0] + at) = make_uint4(o.hi[0], o.hi[1], o.hi[2], o.hi[3]);
  *(uint4 *)(s.k[2 * g + (c >> 1)][1] + at) = make_uint4(o.lo[0], o.lo[1], o.lo[2], o.lo[3]);
}
// V: block b of 16 dims of a group, part n of 2 GPT.
template <int HD>
static __device__ __forceinline__ void value_part(RowsLds<HD> &s, const RawValues<HD> &r, int n, int page, int part,
                                                  int l) {
  const int i = n >> 1, b = n & 1, c = l >> 4, j = l & 15, g = part * (HD / 64) + i;
  // blocks 2 g, 2 g + 1: byte g % 2 of each position's half word
  float x[4];
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    const uint32_t w = r.code[p >> 1] >> (HD == 128 ? 8 * i : 8 * part);
    x[p] = fmaf((float)(w >> (16 * (p & 1) + 4 * b) & 15u), half_of(r.step[2 * i + (p >> 1)], p & 1),
                half_of(r.low[2 * i + (p >> 1)], p & 1));
  }
  uint32_t hi[2], lo[2];
  two_parts(x[0], x[1], hi[0], lo[0]);
  two_parts(x[2], x[3], hi[1], lo[1]);
  const int at = (32 * (c & 1) + 16 * b + j) * 16 + (c >> 1) * 8;
  *(uint2 *)(s.v[g][page][0] + at) = make_uint2(hi[0], hi[1]);
  *(uint2 *)(s.v[g][page][1] + at) = make_uint2(lo[0], lo[1]);
}
template <int HD>
static __device__ __forceinline__ void write_keys(RowsLds<HD> &s, const RawKeys<HD> &r, int page, int part, int l,
                                                  bool bad) {
  KeyChunk<HD> o;
#pragma unroll
  for (int n = 0; n < HD / 16; ++n) key_part(s, r, o, n, page, part, l, bad);
}
template <int HD>
static __device__ __forceinline__ void write_values(RowsLds<HD> &s, const RawValues<HD> &r, int page, int part, int l) {
#pragma unroll
  for (int n = 0; n < HD / 32; ++n) value_part(s, r, n, page, part, l);
}

template <int HD>
__global__ __launch_bounds__(256, 2) void kv4_rows_kernel(AttnArgs a, int slots, int split, int *header,
                                                       RowsTile *tiles, float *records) {
  constexpr int S = HD / 16, NG = HD / 32;
  __shared__ __align__(16) RowsLds<HD> s;
  const int t = threadIdx.x, l = t & 63, w = __builtin_amdgcn_readfirstlane(t >> 6);
  const int Hkv = a.kv.heads, G = a.num_heads / Hkv;
  const float nan = __uint_as_float(0x7FC00000u);
  static_assert(sizeof(s.k) >= kMaxLanes * sizeof(int2), "the lanes' runs lie where the keys come later");
  for (int i = t; i < a.lanes; i += 256) {
    int first, n;
    run_of(a, i, first, n);
    const int ctx = a.ctx[i];
    ((int2 *)s.k)[i] = {n, n > 0 && ctx >= n && ctx <= a.max_ctx ? (ctx + kStage - 1) / kStage : 0};
  }
  __syncthreads();
  if (w == 0) {
    int cut;
    const RowsItem m = find_rows_item(a, (const int2 *)s.k, slots, split, l, &cut);
    if (l == 0) {
      s.item[0] = m.lane;
      s.item[1] = m.head;
      s.item[2] = m.tile;
      s.item[3] = m.chunk;
      s.item[4] = m.chunks;
      s.item[5] = m.record;
      s.item[6] = m.split;
      if (blockIdx.x == 0 && split) header[0] = cut;
    }
  }
  if (t < 2 * (NG + 1)) s.odd[t / (NG + 1)][t % (NG + 1)] = 0;
  __syncthreads();
  const int lane = __builtin_amdgcn_readfirstlane(s.item[0]);
  if (lane < 0) return;
  const int h = __builtin_amdgcn_readfirstlane(s.item[1]), tile = __builtin_amdgcn_readfirstlane(s.item[2]);
  const int chunk = __builtin_amdgcn_readfirstlane(s.item[3]), chunks = __builtin_amdgcn_readfirstlane(s.item[4]);
  const int record = __builtin_amdgcn_readfirstlane(s.item[5]);
  int first, n;
  run_of(a, lane, first, n);
  first = __builtin_amdgcn_readfirstlane(first);
  n = __builtin_amdgcn_readfirstlane(n);
  const int ctx = __builtin_amdgcn_readfirstlane(a.ctx[lane]);
  const bool valid = ctx >= n && ctx <= a.max_ctx;
  const int half = l >> 5, cols = n * G;
  // this lane's column; past the run, the last one again (its output is not written)
  const int col = kTile * tile + 32 * w + (l & 31), colc = min(col, cols - 1);
  const int row = colc / G, head = h * G + colc - row * G;
  const int seen = ctx - n + row + 1;
  // the tile's stages, and this chunk's
  const int tile_row = (min(kTile * (tile + 1), cols) - 1) / G;
  const int all = valid ? (ctx - n + tile_row + 1 + kStage - 1) / kStage : 0;
  const int s0 = chunk_first(chunk, all, chunks), s1 = chunk_first(chunk + 1, all, chunks);
  if (split && chunks > 1 && chunk == 0 && t == 0)
    tiles[s.item[6]] = {first, h, kTile * tile, cols, chunks, record};

  // queries: q log2(e) / sqrt(HD) = 2^e q', the largest |q'| of a column in
  // [2^13, 2^14), as the B operand in two fp16 parts
  v8h qh[S], ql[S];
  float mult;
  {
    const float *q = a.q + ((size_t)(first + row) * a.num_heads + head) * HD + 8 * half;
    const float unit = 1.44269504088896341f / sqrtf((float)HD);
    float4 v[S][2];
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < S; ++i) {
      v[i][0] = *(const float4 *)(q + 16 * i);
      v[i][1] = *(const float4 *)(q + 16 * i + 4);
    }
#pragma unroll
    for (int i = 0; i < S; ++i)
#pragma unroll
      for (int k = 0; k < 2; ++k)
        top = fmaxf(fmaxf(fmaxf(fmaxf(top, fabsf(v[i][k].x)), fabsf(v[i][k].y)), fabsf(v[i][k].z)), fabsf(v[i][k].w));
    top = xor32_max(top) * unit;
    const int e = max(top > 0.0f ? __builtin_amdgcn_frexp_expf(top) - 14 : 0, -120);
    mult = ldexpf(1.0f, e);
    const float scale = ldexpf(1.0f, -e);
#pragma unroll
    for (int i = 0; i < S; ++i) {
      const float x[8] = {v[i][0].x, v[i][0].y, v[i][0].z, v[i][0].w, v[i][1].x, v[i][1].y, v[i][1].z, v[i][1].w};
      uint32_t hi[4], lo[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) two_parts(x[2 * k] * unit * scale, x[2 * k + 1] * unit * scale, hi[k], lo[k]);
      qh[i] = as_v8h(hi[0], hi[1], hi[2], hi[3]);
      ql[i] = as_v8h(lo[0], lo[1], lo[2], lo[3]);
    }
  }
  f16v o[NG];
#pragma unroll
  for (int g = 0; g < NG; ++g)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[g][i] = 0.0f;
  float ref = kNoRef, sum = 0.0f;
  int odd = 0;  // groups of this column with no number
  const bool wave_in = kTile * tile + 32 * w < cols;
  const int wave_first = __builtin_amdgcn_readfirstlane(seen);  // the fewest keys of the wave's columns

  const int32_t *table = a.table + (size_t)lane * a.max_pages;
  const int pages = (ctx + kPage - 1) / kPage;
  const uint8_t *head_base = a.kv.base + (size_t)(2 * h) * (10 * HD);
  const int page = w & 1, part = w >> 1;
  int id_base = -64;
  uint32_t ids = 0;
  // stage s0 + i into its slot, by wave i % kRowsRing
  auto request = [&](int i) {
    const int p = 2 * (s0 + i);
    if (p >= id_base + 64) {
      id_base = p;
      ids = (uint32_t)table[min(p + l, pages - 1)];
    }
    uint32_t id[2];
    int bad = 0;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      id[x] = (uint32_t)__builtin_amdgcn_readlane((int)ids, min(p + x, pages - 1) - id_base);
      if (id[x] >= a.kv.page_count) {
        bad |= 1 << x;
        id[x] = 0;
      }
    }
    if (l == 0) s.bad[i % kRowsRing] = bad;
    copy_pair(&s.ring[i % kRowsRing], head_base + id[0] * a.kv.page_bytes, head_base + id[1] * a.kv.page_bytes, l);
  };
  const int stages = s1 - s0;
  if (w < kRowsRing - 1 && w < stages) request(w);
  arrive<0>();
  __syncthreads();
  if (stages > 0) write_keys(s, raw_keys(s.ring[0], page, part, l), page, part, l, s.bad[0] >> page & 1);
  __syncthreads();
  for (int st = 0; st < stages; ++st) {
    const int key0 = (s0 + st) * kStage;
    if (w == (st + 3) % kRowsRing && st + 3 < stages) request(st + 3);
    // scores, and between the matrix products this stage's values
    RawValues<HD> rv = raw_values(s.ring[st % kRowsRing], page, part, l);
    if (t <= NG) s.odd[(st + 1) & 1][t] = 0;  // read before the last barrier, written after the next
    clean_values(s.odd[st & 1], rv, page, part, l, ctx - key0, s.bad[st % kRowsRing] >> page & 1);
    uint32_t ph[8], pl[8];
    if (wave_in) {
      keep_here(rv.code);
      f16v sc;
#pragma unroll
      for (int i = 0; i < 16; ++i) sc[i] = 0.0f;
      // (two sums in turn: a product that adds to the one before it waits for it)
      f16v sd;
#pragma unroll
      for (int i = 0; i < 16; ++i) sd[i] = 0.0f;
      v8h kh[4], kl[4];
      auto read_k = [&](int i) {
        kh[i & 3] = *(const v8h *)(s.k[i][0] + l * 16);
        kl[i & 3] = *(const v8h *)(s.k[i][1] + l * 16);
      };
      read_k(0);
      read_k(1);
      // the matrix products' wave first: the other workgroup's fills their gaps
      // (eight mixed lanes 61.7 -> 59.5 us)
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int i = 0; i < S; i += 2) {
        if (i + 2 < S) {
          read_k(i + 2);
          read_k(i + 3);
        }
        sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(kh[i & 3], ql[i], sc, 0, 0, 0);
        sd = __builtin_amdgcn_mfma_f32_32x32x16_f16(kh[i + 1 & 3], ql[i + 1], sd, 0, 0, 0);
        value_part(s, rv, i / 2, page, part, l);
        sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(kl[i & 3], qh[i], sc, 0, 0, 0);
        sd = __builtin_amdgcn_mfma_f32_32x32x16_f16(kl[i + 1 & 3], qh[i + 1], sd, 0, 0, 0);
        sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(kh[i & 3], qh[i], sc, 0, 0, 0);
        sd = __builtin_amdgcn_mfma_f32_32x32x16_f16(kh[i + 1 & 3], qh[i + 1], sd, 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
      }
      __builtin_amdgcn_s_setprio(0);
      sc += sd;
      if (key0 + kStage > wave_first) {
        asm volatile("");
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (key0 + 8 * (i >> 2) + 4 * half + (i & 3) >= seen) sc[i] = -INFINITY;
      }
      float top = sc[0];
#pragma unroll
      for (int i = 1; i < 15; i += 2) top = fmaxf(fmaxf(top, sc[i]), sc[i + 1]);
      top = fmaxf(top, sc[15]);
      if (__any(fmaf(top, mult, -ref) > kSlack)) {
        asm volatile("");
        const float high = xor32_max(top) * mult;
        const float above = high - ref > kSlack ? high : ref, f = exp2f(ref - above);
        ref = above;
        sum *= f;
#pragma unroll
        for (int g = 0; g < NG; ++g) o[g] *= f;
      }
      const float shift = kShift - ref;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        sc[i] = __builtin_amdgcn_exp2f(fmaf(sc[i], mult, shift));
        sum += sc[i];
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) two_parts(sc[2 * i], sc[2 * i + 1], ph[i], pl[i]);
    } else {
      write_values(s, rv, page, part, l);
    }
    if (w == (st + 1) % kRowsRing) arrive<0>();  // the next stage, asked for two and a half ago
    __syncthreads();
    // output, and between the matrix products the next stage's keys (past the
    // last one what the slot holds, which nothing reads)
    RawKeys<HD> rk = raw_keys(s.ring[(st + 1) % kRowsRing], page, part, l);
    const bool bad = s.bad[(st + 1) % kRowsRing] >> page & 1;
    if (wave_in) {
      keep_here(rk.code);
      KeyChunk<HD> kc;
      v8h vh[4], vl[4];
      auto read_v = [&](int i) {
        vh[i & 3] = *(const v8h *)(s.v[i % NG][i / NG][0] + l * 16);
        vl[i & 3] = *(const v8h *)(s.v[i % NG][i / NG][1] + l * 16);
      };
      read_v(0);
      read_v(1);
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int i = 0; i < 2 * NG; i += 2) {
        const int x = i / NG, g = i % NG;
        if (i + 2 < 2 * NG) {
          read_v(i + 2);
          read_v(i + 3);
        }
        const v8h bh = as_v8h(ph[4 * x], ph[4 * x + 1], ph[4 * x + 2], ph[4 * x + 3]);
        const v8h bl = as_v8h(pl[4 * x], pl[4 * x + 1], pl[4 * x + 2], pl[4 * x + 3]);
        o[g] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vh[i & 3], bl, o[g], 0, 0, 0);
        o[g + 1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vh[i + 1 & 3], bl, o[g + 1], 0, 0, 0);
        key_part(s, rk, kc, i, page, part, l, bad);
        o[g] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vl[i & 3], bh, o[g], 0, 0, 0);
        o[g + 1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vl[i + 1 & 3], bh, o[g + 1], 0, 0, 0);
        key_part(s, rk, kc, i + 1, page, part, l, bad);
        o[g] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vh[i & 3], bh, o[g], 0, 0, 0);
        o[g + 1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vh[i + 1 & 3], bh, o[g + 1], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
      }
      __builtin_amdgcn_s_setprio(0);
      if (__builtin_amdgcn_readfirstlane(s.odd[st & 1][NG])) {
        const int k = min(kStage, seen - key0);
        const uint32_t shown = k <= 0 ? 0u : k >= 32 ? 0xFFFFFFFFu : (1u << k) - 1;
#pragma unroll
        for (int g = 0; g < NG; ++g) odd |= (s.odd[st & 1][g] & shown) != 0 ? 1 << g : 0;
      }
    } else {
      write_keys(s, rk, page, part, l, bad);
    }
    __syncthreads();
  }
  sum = xor32_add(sum);
  if (col >= cols) return;
  if (chunks == 1) {
    const float inv = valid ? 1.0f / sum : nan;
    float *out = a.out + ((size_t)(first + row) * a.num_heads + head) * HD + 4 * half;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const float f = odd >> g & 1 ? nan : inv;
#pragma unroll
      for (int i = 0; i < 16; i += 4)
        *(float4 *)(out + 32 * g + 2 * i) = make_float4(o[g][i] * f, o[g][i + 1] * f, o[g][i + 2] * f, o[g][i + 3] * f);
    }
  } else {
    float *rec = records + (size_t)record * (kTile * (HD + 2));
    const int k = 32 * w + (l & 31);
    if (half == 0) {
      rec[2 * k] = ref;
      rec[2 * k + 1] = sum;
    }
    float *out = rec + 2 * kTile + k * HD + 4 * half;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const float f = odd >> g & 1 ? nan : 1.0f;
#pragma unroll
      for (int i = 0; i < 16; i += 4)
        *(float4 *)(out + 32 * g + 2 * i) = make_float4(o[g][i] * f, o[g][i + 1] * f, o[g][i + 2] * f, o[g][i + 3] * f);
    }
  }
}

// The chunks of cut tiles added up, weighted by 2^(reference - the largest):
// HD / 4 threads for a column (of many chunks: for one of kParts shares of
// them, which meet in LDS), four chunks' loads on their way at a time. The
// time is a chain of dependent loads: one thread for all chunks of a column,
// in two passes, took 17.5 us at 42 chunks where this takes 4.1.
constexpr int kParts = 4, kMergeGrid = 2048;
template <int HD>
__global__ __launch_bounds__(256) void kv4_rows_merge_kernel(AttnArgs a, const int *header, const RowsTile *tiles,
                                                             const float *records) {
  constexpr int TPC = HD / 4, SUBS = 256 / TPC;
  constexpr size_t REC = kTile * (HD + 2);
  __shared__ float4 acc[256];
  __shared__ float2 stat[256 / TPC];
  const int G = a.num_heads / a.kv.heads, cut = header[0], d = threadIdx.x % TPC * 4;
  for (int u = blockIdx.x; u < cut * (kTile / SUBS * kParts); u += gridDim.x) {
    const int unit = u / cut;
    const RowsTile m = tiles[u - unit * cut];
    // shares of a column's chunks, and this thread's column and share
    const int parts = m.chunks > 4 ? kParts : 1, part = threadIdx.x / TPC % parts;
    const int k0 = unit * (SUBS / parts), k = k0 + threadIdx.x / TPC / parts, col = m.col + k;
    if (k0 >= kTile || m.col + k0 >= m.cols) continue;  // (the whole workgroup)
    // past the run a record holds nothing: the last column again, not written
    const int kc = min(k, m.cols - 1 - m.col);
    const float *rec = records + m.record * REC;
    float top = kNoRef, sum = 0.0f;
    float4 o = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int i = part; i < m.chunks; i += 4 * parts) {
      float2 rs[4];
      float4 x[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float *p = rec + (size_t)min(i + j * parts, m.chunks - 1) * REC;
        rs[j] = *(const float2 *)(p + 2 * kc);
        x[j] = *(const float4 *)(p + 2 * kTile + kc * HD + d);
      }
      float high = top;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (i + j * parts < m.chunks) high = fmaxf(high, rs[j].x);
      const float f = __builtin_amdgcn_exp2f(top - high);
      top = high;
      sum *= f;
      o = {o.x * f, o.y * f, o.z * f, o.w * f};
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (i + j * parts < m.chunks) {
          const float g = __builtin_amdgcn_exp2f(rs[j].x - top);
          sum = fmaf(rs[j].y, g, sum);
          o = {fmaf(x[j].x, g, o.x), fmaf(x[j].y, g, o.y), fmaf(x[j].z, g, o.z), fmaf(x[j].w, g, o.w)};
        }
    }
    if (parts > 1) {
      acc[threadIdx.x] = o;
      if (d == 0) stat[threadIdx.x / TPC] = {top, sum};
      __syncthreads();
      if (part == 0)
#pragma unroll
        for (int j = 1; j < kParts; ++j) {
          const float2 rs = stat[threadIdx.x / TPC + j];
          const float4 x = acc[threadIdx.x + j * TPC];
          const float high = fmaxf(top, rs.x), f = __builtin_amdgcn_exp2f(top - high);
          const float g = __builtin_amdgcn_exp2f(rs.x - high);
          top = high;
          sum = fmaf(rs.y, g, sum * f);
          o = {fmaf(x.x, g, o.x * f), fmaf(x.y, g, o.y * f), fmaf(x.z, g, o.z * f), fmaf(x.w, g, o.w * f)};
        }
      __syncthreads();
    }
    if (part == 0 && k < kTile && col < m.cols) {
      const int row = col / G, head = m.head * G + col - row * G;
      *(float4 *)(a.out + ((size_t)(m.first + row) * a.num_heads + head) * HD + d) =
          make_float4(o.x / sum, o.y / sum, o.z / sum, o.w / sum);
    }
  }
}

}  // namespace
}  // namespace gk

// ---------------------------------------------------------------------------
// C ABI
// ---------------------------------------------------------------------------
namespace {

// The calling thread's device is the context's while a call launches.
struct DeviceScope {
  int before = -1;
  hipError_t err = hipSuccess;
  explicit DeviceScope(int device) {
    int now = 0;
    err = hipGetDevice(&now);
    if (err == hipSuccess && now != device) {
      err = hipSetDevice(device);
      if (err == hipSuccess) before = now;
    }
  }
  ~DeviceScope() {
    if (before >= 0) (void)hipSetDevice(before);
  }
};

bool aligned(const void *p, uintptr_t to) { return ((uintptr_t)p & (to - 1)) == 0; }

bool page_shape_ok(uint32_t num_layers, uint32_t num_kv_heads, uint32_t head_dim) {
  return (head_dim == 64 || head_dim == 128) && num_layers > 0 && num_kv_heads > 0 &&
         num_layers <= (1u << 16) && num_kv_heads <= (1u << 12);
}

int pool_view(const glacier_hip_kv4_pool_t *p, uint32_t layer, gk::Kv4 *out) {
  if (!p || !p->pages_dev || !aligned(p->pages_dev, 16)) return GLACIER_HIP_INVALID_ARGUMENT;
  if (!page_shape_ok(p->num_layers, p->num_kv_heads, p->head_dim) || p->page_count == 0 ||
      p->page_count > (1u << 31) || layer >= p->num_layers)
    return GLACIER_HIP_SHAPE_MISMATCH;
  out->page_bytes = glacier_hip_kv4_page_bytes(p->num_layers, p->num_kv_heads, p->head_dim);
  out->base = (uint8_t *)p->pages_dev + (size_t)layer * (out->page_bytes / p->num_layers);
  out->page_count = p->page_count;
  out->heads = (int)p->num_kv_heads;
  return GLACIER_HIP_OK;
}

size_t merge_bytes(uint32_t lanes, uint32_t heads) {
  return ((size_t)lanes * heads * sizeof(gk::MergeItem) + 255) & ~(size_t)255;
}

int attention(glacier_hip_context *ctx, const glacier_hip_kv4_pool_t *pool, uint32_t layer,
              const float *q, const int32_t *table, uint32_t max_pages, const int32_t *row_start,
              const int32_t *lens, uint32_t lanes, uint32_t max_rows, uint32_t num_heads,
              uint32_t max_ctx, float *out, void *ws, uint64_t ws_bytes, void *stream) {
  if (!ctx || !q || !table || !lens || !out || !ws || !aligned(q, 16) || !aligned(out, 16) ||
      !aligned(ws, 16))
    return GLACIER_HIP_INVALID_ARGUMENT;
  gk::AttnArgs a{};
  if (int rc = pool_view(pool, layer, &a.kv)) return rc;
  const uint64_t need = glacier_hip_kv4_attention_workspace_bytes(lanes, max_rows, num_heads,
                                                                  pool->num_kv_heads, pool->head_dim);
  if (need == 0 || ws_bytes < need || max_ctx == 0 || max_ctx > (1u << 26) ||
      max_ctx > (uint64_t)max_pages * gk::kPage ||
      (uint64_t)lanes * ((max_ctx + 15) / 16) * pool->num_kv_heads >= (1ull << 31))
    return GLACIER_HIP_SHAPE_MISMATCH;
  a.q = q;
  a.table = table;
  a.max_pages = max_pages;
  a.row_start = row_start;
  a.ctx = lens;
  a.lanes = (int)lanes;
  a.max_rows = (int)max_rows;
  a.num_heads = (int)num_heads;
  a.max_ctx = (int)max_ctx;
  a.out = out;
  GH_SUBMISSION(ctx);
  DeviceScope on(ctx->device);
  GH_CHECK(ctx, on.err);
  hipStream_t st = stream ? (hipStream_t)stream : ctx->stream;
  if (!row_start) {
    // a merge follows where a context may be more than one item
    const uint32_t units = (max_ctx + gk::kUnit - 1) / gk::kUnit;
    const bool split = units > (uint32_t)gk::kWhole;
    auto *merge = split ? (gk::MergeItem *)ws : nullptr;
    float *records = (float *)((char *)ws + merge_bytes(lanes, pool->num_kv_heads));
    const int slots = std::min(gk::kMaxSlots, ctx->props.multiProcessorCount * (pool->head_dim == 128 ? 3 : 4));
    // items at most: slots, or where there are many contexts one each and slots / 2 more
    const uint64_t heads = (uint64_t)lanes * a.kv.heads, each = split ? units : 1;
    const uint64_t most = heads <= (uint64_t)slots / 2 ? slots : heads + slots / 2;
    const uint32_t grid = (uint32_t)std::max<uint64_t>(lanes, std::min(heads * each, most));
    if (pool->head_dim == 128) {
      gk::kv4_decode_kernel<128><<<grid, 64 * gk::kWaves, 0, st>>>(a, slots, merge, records);
      if (split) gk::kv4_merge_kernel<128><<<lanes * num_heads, 256, 0, st>>>(a, merge, records);
    } else {
      gk::kv4_decode_kernel<64><<<grid, 64 * gk::kWaves, 0, st>>>(a, slots, merge, records);
      if (split) gk::kv4_merge_kernel<64><<<lanes * num_heads, 256, 0, st>>>(a, merge, records);
    }
    GH_CHECK(ctx, hipGetLastError());
    return GLACIER_HIP_OK;
  }
  // workgroups a CU holds
  const int slots = std::min(gk::kRowsSlots, ctx->props.multiProcessorCount * 2);
  const int split = (max_ctx + gk::kStage - 1) / gk::kStage > (uint32_t)gk::kWholeStages;
  const uint64_t tiles = (uint64_t)max_rows * (num_heads / a.kv.heads) / gk::kTile + lanes;
  // items at most. Chunks past the tiles' number are no more than slots less
  // the tiles or half the slots: those of cut tiles are slots at most.
  const uint32_t whole = (uint32_t)(tiles * a.kv.heads);
  const uint32_t grid = split ? std::max<uint32_t>(slots, whole + slots / 2) : whole;
  int *header = (int *)ws;
  auto *cut = (gk::RowsTile *)((char *)ws + 256);
  float *records = (float *)((char *)ws + gk::kRowsHeader);
  if (pool->head_dim == 128) {
    gk::kv4_rows_kernel<128><<<grid, 256, 0, st>>>(a, slots, split, header, cut, records);
    if (split) gk::kv4_rows_merge_kernel<128><<<gk::kMergeGrid, 256, 0, st>>>(a, header, cut, records);
  } else {
    gk::kv4_rows_kernel<64><<<grid, 256, 0, st>>>(a, slots, split, header, cut, records);
    if (split) gk::kv4_rows_merge_kernel<64><<<gk::kMergeGrid, 256, 0, st>>>(a, header, cut, records);
  }
  GH_CHECK(ctx, hipGetLastError());
  return GLACIER_HIP_OK;
}

// Workgroups of an append or a read: a wave for K and one for V per head and run of rows.
uint32_t store_grid(uint32_t rows, int heads, uint32_t hd) {
  const uint32_t run = 512 / hd;
  return ((rows + run - 1) / run * 2 * heads + 3) / 4;
}

template <class T>
void append_launch(const gk::Kv4 &kv, uint32_t hd, const void *k, const void *v, uint64_t ks,
                   uint64_t vs, const int64_t *slots, uint32_t rows, hipStream_t st) {
  const uint32_t grid = store_grid(rows, kv.heads, hd);
  // 16-byte loads where every row's elements allow them
  const bool wide = aligned(k, 16) && aligned(v, 16) && (ks | vs) * sizeof(T) % 16 == 0;
  auto launch = [&](auto *kernel) {
    kernel<<<grid, 256, 0, st>>>(kv, (const T *)k, (const T *)v, ks, vs, slots, (int)rows);
  };
  if (hd == 128) wide ? launch(gk::kv4_append_kernel<128, true, T>) : launch(gk::kv4_append_kernel<128, false, T>);
  else wide ? launch(gk::kv4_append_kernel<64, true, T>) : launch(gk::kv4_append_kernel<64, false, T>);
}

}  // namespace

extern "C" {

uint64_t glacier_hip_kv4_page_bytes(uint32_t num_layers, uint32_t num_kv_heads, uint32_t head_dim) {
  if (!page_shape_ok(num_layers, num_kv_heads, head_dim)) return 0;
  return 20ull * num_layers * num_kv_heads * head_dim;
}

int glacier_hip_kv_plan_rows(glacier_hip_context *ctx, const int32_t *ctx_lens_dev,
                             const int32_t *new_rows_dev, uint32_t lanes, uint32_t max_rows,
                             int32_t *page_table_dev, uint32_t max_pages,
                             const int32_t *free_pages_dev, uint32_t free_count,
                             const int32_t *free_taken_dev, int32_t *row_start_dev,
                             int32_t *ctx_after_dev, int64_t *slots_dev, int32_t *row_lanes_dev,
                             int32_t *row_positions_dev, int32_t *result_dev, void *stream) {
  if (!ctx || !ctx_lens_dev || !new_rows_dev || !page_table_dev || !free_taken_dev ||
      !row_start_dev || !ctx_after_dev || !slots_dev || !result_dev ||
      (!free_pages_dev && free_count))
    return GLACIER_HIP_INVALID_ARGUMENT;
  if (lanes == 0 || lanes > GLACIER_HIP_KV_MAX_LANES || max_rows == 0 ||
      max_rows > GLACIER_HIP_KV_MAX_ROWS || max_pages == 0 || max_pages > (1u << 26) ||
      (uint64_t)lanes * max_pages > (1ull << 31) || free_count > (1u << 30))
    return GLACIER_HIP_SHAPE_MISMATCH;
  GH_SUBMISSION(ctx);
  DeviceScope on(ctx->device);
  GH_CHECK(ctx, on.err);
  hipStream_t st = stream ? (hipStream_t)stream : ctx->stream;
  gk::kv_plan_kernel<<<1, gk::kMaxLanes, 0, st>>>(
      ctx_lens_dev, new_rows_dev, (int)lanes, (int)max_rows, page_table_dev, max_pages,
      free_pages_dev, free_count, free_taken_dev, row_start_dev, ctx_after_dev, result_dev,
      max_rows <= gk::kPlanRows ? slots_dev : nullptr, row_lanes_dev, row_positions_dev);
  GH_CHECK(ctx, hipGetLastError());
  if (max_rows <= gk::kPlanRows) return GLACIER_HIP_OK;
  gk::kv_plan_rows_kernel<<<(max_rows + 255) / 256, 256, 0, st>>>(
      row_start_dev, ctx_after_dev, (int)lanes, (int)max_rows, page_table_dev, max_pages, slots_dev,
      row_lanes_dev, row_positions_dev);
  GH_CHECK(ctx, hipGetLastError());
  return GLACIER_HIP_OK;
}

int glacier_hip_kv4_append(glacier_hip_context *ctx, const glacier_hip_kv4_pool_t *pool,
                           uint32_t layer, const void *k_dev, const void *v_dev, int kv_dtype,
                           uint64_t k_stride, uint64_t v_stride, const int64_t *slots_dev,
                           uint32_t rows, void *stream) {
  if (!ctx || !k_dev || !v_dev || !slots_dev) return GLACIER_HIP_INVALID_ARGUMENT;
  if (kv_dtype != GLACIER_HIP_F32 && kv_dtype != GLACIER_HIP_F16 && kv_dtype != GLACIER_HIP_BF16)
    return GLACIER_HIP_DTYPE_UNSUPPORTED;
  const uintptr_t size = kv_dtype == GLACIER_HIP_F32 ? 4 : 2;
  if (!aligned(k_dev, size) || !aligned(v_dev, size)) return GLACIER_HIP_INVALID_ARGUMENT;
  gk::Kv4 kv;
  if (int rc = pool_view(pool, layer, &kv)) return rc;
  const uint64_t width = (uint64_t)pool->num_kv_heads * pool->head_dim;
  if (rows == 0 || rows > GLACIER_HIP_KV_MAX_ROWS || k_stride < width || v_stride < width ||
      k_stride > (1ull << 32) || v_stride > (1ull << 32))
    return GLACIER_HIP_SHAPE_MISMATCH;
  GH_SUBMISSION(ctx);
  DeviceScope on(ctx->device);
  GH_CHECK(ctx, on.err);
  hipStream_t st = stream ? (hipStream_t)stream : ctx->stream;
  if (kv_dtype == GLACIER_HIP_F32)
    append_launch<float>(kv, pool->head_dim, k_dev, v_dev, k_stride, v_stride, slots_dev, rows, st);
  else if (kv_dtype == GLACIER_HIP_F16)
    append_launch<__half>(kv, pool->head_dim, k_dev, v_dev, k_stride, v_stride, slots_dev, rows, st);
  else
    append_launch<gk::Bf16>(kv, pool->head_dim, k_dev, v_dev, k_stride, v_stride, slots_dev, rows, st);
  GH_CHECK(ctx, hipGetLastError());
  return GLACIER_HIP_OK;
}

int glacier_hip_kv4_read(glacier_hip_context *ctx, const glacier_hip_kv4_pool_t *pool,
                         uint32_t layer, const int64_t *slots_dev, uint32_t rows, float *k_dev,
                         float *v_dev, void *stream) {
  if (!ctx || !slots_dev || !k_dev || !v_dev || !aligned(k_dev, 16) || !aligned(v_dev, 16))
    return GLACIER_HIP_INVALID_ARGUMENT;
  gk::Kv4 kv;
  if (int rc = pool_view(pool, layer, &kv)) return rc;
  if (rows == 0 || rows > GLACIER_HIP_KV_MAX_ROWS) return GLACIER_HIP_SHAPE_MISMATCH;
  GH_SUBMISSION(ctx);
  DeviceScope on(ctx->device);
  GH_CHECK(ctx, on.err);
  hipStream_t st = stream ? (hipStream_t)stream : ctx->stream;
  const uint32_t grid = store_grid(rows, kv.heads, pool->head_dim);
  if (pool->head_dim == 128) gk::kv4_read_kernel<128><<<grid, 256, 0, st>>>(kv, slots_dev, (int)rows, k_dev, v_dev);
  else gk::kv4_read_kernel<64><<<grid, 256, 0, st>>>(kv, slots_dev, (int)rows, k_dev, v_dev);
  GH_CHECK(ctx, hipGetLastError());
  return GLACIER_HIP_OK;
}

uint64_t glacier_hip_kv4_attention_workspace_bytes(uint32_t lanes, uint32_t max_rows,
                                                   uint32_t num_heads, uint32_t num_kv_heads,
                                                   uint32_t head_dim) {
  if (lanes == 0 || lanes > GLACIER_HIP_KV_MAX_LANES || max_rows == 0 ||
      max_rows > GLACIER_HIP_KV_MAX_ROWS || !page_shape_ok(1, num_kv_heads, head_dim) ||
      num_heads % num_kv_heads != 0 || num_heads / num_kv_heads == 0 ||
      num_heads / num_kv_heads > (uint32_t)gk::kMaxGroup)
    return 0;
  const uint64_t one = merge_bytes(lanes, num_kv_heads) +
                       (uint64_t)gk::kMaxRecords * gk::kMaxGroup * (head_dim + 2) * sizeof(float);
  const uint64_t runs = gk::kRowsHeader + (uint64_t)gk::kRowsRecords * gk::kTile * (head_dim + 2) * sizeof(float);
  return std::max(one, runs);
}

int glacier_hip_paged_attention_kv4(glacier_hip_context *ctx, const glacier_hip_kv4_pool_t *pool,
                                    uint32_t layer, const float *q_dev,
                                    const int32_t *page_table_dev, uint32_t max_pages_per_lane,
                                    const int32_t *ctx_lens_dev, uint32_t lanes,
                                    uint32_t num_heads, uint32_t max_ctx, float *out_dev,
                                    void *workspace_dev, uint64_t workspace_bytes, void *stream) {
  return attention(ctx, pool, layer, q_dev, page_table_dev, max_pages_per_lane, nullptr, ctx_lens_dev,
                   lanes, lanes, num_heads, max_ctx, out_dev, workspace_dev, workspace_bytes, stream);
}

int glacier_hip_paged_attention_kv4_rows(glacier_hip_context *ctx,
                                         const glacier_hip_kv4_pool_t *pool, uint32_t layer,
                                         const float *q_dev, const int32_t *page_table_dev,
                                         uint32_t max_pages_per_lane, const int32_t *row_start_dev,
                                         const int32_t *ctx_lens_dev, uint32_t lanes,
                                         uint32_t max_rows, uint32_t num_heads, uint32_t max_ctx,
                                         float *out_dev, void *workspace_dev,
                                         uint64_t workspace_bytes, void *stream) {
  if (!row_start_dev) return GLACIER_HIP_INVALID_ARGUMENT;
  return attention(ctx, pool, layer, q_dev, page_table_dev, max_pages_per_lane, row_start_dev,
                   ctx_lens_dev, lanes, max_rows, num_heads, max_ctx, out_dev, workspace_dev,
                   workspace_bytes, stream);
}

}  // extern "C"
