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
// and new pages), then the new table entries; the rows follow in a second
// launch once the table is whole.
// ---------------------------------------------------------------------------
static __device__ __forceinline__ int wave_scan(int v) {
  const int l = threadIdx.x & 63;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int u = __shfl_up(v, o, 64);
    if (l >= o) v += u;
  }
  return v;
}

__global__ __launch_bounds__(kMaxLanes) void kv_plan_kernel(
    const int32_t *ctx, const int32_t *fresh, int lanes, int max_rows, int32_t *table,
    uint32_t max_pages, const int32_t *free_pages, uint32_t free_count, const int32_t *free_taken,
    int32_t *row_start, int32_t *ctx_after, int32_t *result) {
  __shared__ int rows_of[kMaxLanes / 64], pages_of[kMaxLanes / 64];
  __shared__ int page_end[kMaxLanes], held_of[kMaxLanes];
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
  if (!good) return;
  for (int p = t; p < pages; p += kMaxLanes) {
    int lo = 0, hi = kMaxLanes - 1;  // the first lane whose pages end past p
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (page_end[mid] > p) hi = mid;
      else lo = mid + 1;
    }
    const int before = lo ? page_end[lo - 1] : 0;
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

// Byte of dim d of position P in a tile's codes, and whether it is the high nibble.
template <int HD>
static __device__ __forceinline__ int code_byte(int which, int P, int d, int &high) {
  constexpr int NG = HD / 32, NH = HD / 64;
  if (which == 0) {
    high = d & 1;
    return P * (HD / 2) + ((d % 32) / 8 * NG + d / 32) * 4 + d % 8 / 2;
  }
  const int e = d / 16;  // the value's block of 16 dims
  high = e & 1;
  return ((((P / 4) * 16 + d % 16) * 2 + P / 2 % 2) * NH + e / 4) * 4 + P % 2 * 2 + e % 4 / 2;
}
template <int HD>
static __device__ __forceinline__ int step_byte(int P, int g) {
  return 8 * HD + 2 * ((P / 4) * (HD / 8) + g * 4 + P % 4);
}
template <int HD>
static __device__ __forceinline__ int low_byte(int which, int P, int g) {
  return which ? step_byte<HD>(P, g) + HD : 9 * HD + 2 * (P * (HD / 32) + g);
}

// One thread a group of 32 dims of a row's K or V.
template <int HD, class T>
__global__ __launch_bounds__(256) void kv4_append_kernel(Kv4 kv, const T *k, const T *v,
                                                         size_t k_stride, size_t v_stride,
                                                         const int64_t *slots, int rows) {
  constexpr int NG = HD / 32;
  const int per_row = 2 * kv.heads * NG;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t r = i / per_row;
  if (r >= rows) return;
  const int j = (int)(i - r * per_row), g = j % NG, which = j / NG % 2, head = j / (2 * NG);
  const int64_t slot = slots[r];
  if (slot < 0 || slot / kPage >= (int64_t)kv.page_count) return;
  const T *x = (which ? v + r * v_stride : k + r * k_stride) + head * HD + g * 32;
  float lo = INFINITY, hi = -INFINITY;
  bool bad = false;
  for (int d = 0; d < 32; ++d) {
    const float f = widen(x[d]);
    bad |= !(fabsf(f) <= 32768.0f);
    lo = fminf(lo, f);
    hi = fmaxf(hi, f);
  }
  const __half step = bad ? __ushort_as_half(0x7E00) : __float2half_rn((hi - lo) / 15.0f);
  const __half low = bad ? __ushort_as_half(0x7E00) : __float2half_rn(lo);
  const int P = (int)(slot % kPage);
  uint8_t *tile = tile_of(kv, (uint32_t)(slot / kPage), head, which, 10 * HD);
  const double s = (double)__half2float(step), m = (double)__half2float(low);
  uint8_t code[32];
  for (int d = 0; d < 32; ++d)
    code[d] = s > 0.0 ? (uint8_t)fmin(fmax(rint(((double)widen(x[d]) - m) / s), 0.0), 15.0) : 0;
  for (int d = 0; d < 32; ++d) {
    int high;
    const int at = code_byte<HD>(which, P, g * 32 + d, high);
    if (!high) tile[at] = (uint8_t)(code[d] | code[d + (which ? 16 : 1)] << 4);
  }
  *(__half *)(tile + step_byte<HD>(P, g)) = step;
  *(__half *)(tile + low_byte<HD>(which, P, g)) = low;
}

template <int HD>
static __device__ __forceinline__ float kv4_value(const uint8_t *tile, int which, int P, int d) {
  int high;
  const int at = code_byte<HD>(which, P, d, high);
  const float c = (float)(tile[at] >> (4 * high) & 15);
  return c * __half2float(*(const __half *)(tile + step_byte<HD>(P, d / 32))) +
         __half2float(*(const __half *)(tile + low_byte<HD>(which, P, d / 32)));
}

template <int HD>
__global__ __launch_bounds__(256) void kv4_read_kernel(Kv4 kv, const int64_t *slots, int rows,
                                                       float *k, float *v) {
  const int width = kv.heads * HD;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t r = i / width;
  if (r >= rows) return;
  const int64_t slot = slots[r];
  if (slot < 0 || slot / kPage >= (int64_t)kv.page_count) return;
  const int d = (int)(i - r * width), head = d / HD, P = (int)(slot % kPage);
  const uint32_t page = (uint32_t)(slot / kPage);
  k[i] = kv4_value<HD>(tile_of(kv, page, head, 0, 10 * HD), 0, P, d % HD);
  v[i] = kv4_value<HD>(tile_of(kv, page, head, 1, 10 * HD), 1, P, d % HD);
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

// One workgroup a (row, KV head): 256 positions at a time, a thread scores
// each for the G query heads, then every thread adds up its dims.
template <int HD>
__global__ __launch_bounds__(256) void kv4_attn_kernel(AttnArgs a) {
  __shared__ float qs[kMaxGroup][HD], sc[kMaxGroup][256], top_s[kMaxGroup], keep_s[kMaxGroup],
      sum_s[kMaxGroup];
  const int t = threadIdx.x, r = blockIdx.x, h = blockIdx.y, G = a.num_heads / a.kv.heads;
  int lane = r, n = 1, first = r;
  if (a.row_start) {
    if (r >= a.row_start[a.lanes]) return;
    int lo = 0, hi = a.lanes - 1;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (a.row_start[mid + 1] > r) hi = mid;
      else lo = mid + 1;
    }
    lane = lo;
    first = a.row_start[lane];
    n = a.row_start[lane + 1] - first;
  }
  const int ctx = a.ctx[lane];
  bool bad = ctx < 0 || ctx > a.max_ctx || (a.row_start && n > ctx);
  const int seen = bad ? 0 : ctx - (first + n - 1 - r) * (a.row_start != nullptr);
  const float *q = a.q + ((size_t)r * a.num_heads + h * G) * HD;
  for (int i = t; i < G * HD; i += 256) qs[i / HD][i % HD] = q[i] / sqrtf((float)HD);
  if (t < kMaxGroup) {
    top_s[t] = -INFINITY;
    sum_s[t] = 0.0f;
  }
  constexpr int PER = kMaxGroup * HD / 256;
  float acc[PER] = {};
  const int32_t *pages = a.table + (size_t)lane * a.max_pages;
  for (int j0 = 0; j0 < seen; j0 += 256) {
    __syncthreads();
    const int j = j0 + t;
    for (int g = 0; g < G; ++g) sc[g][t] = -INFINITY;
    if (j < seen) {
      const uint32_t page = (uint32_t)pages[j / kPage];
      if (page >= a.kv.page_count) bad = true;
      else {
        const uint8_t *tile = tile_of(a.kv, page, h, 0, 10 * HD);
        float s[kMaxGroup] = {};
        for (int d = 0; d < HD; ++d) {
          const float x = kv4_value<HD>(tile, 0, j % kPage, d);
          for (int g = 0; g < G; ++g) s[g] = fmaf(qs[g][d], x, s[g]);
        }
        for (int g = 0; g < G; ++g) sc[g][t] = s[g];
      }
    }
    bad = __syncthreads_or(bad);
    if (bad) break;
    if (t < G) {
      float top = top_s[t], nan = 0.0f;
      for (int i = 0; i < 256; ++i) {
        top = fmaxf(top, sc[t][i]);
        nan += isnan(sc[t][i]) ? 1.0f : 0.0f;
      }
      if (nan > 0.0f) top = __uint_as_float(0x7FC00000u);
      float sum = 0.0f;
      for (int i = 0; i < 256; ++i) sum += sc[t][i] = expf(sc[t][i] - top);
      keep_s[t] = top_s[t] == -INFINITY ? 0.0f : expf(top_s[t] - top);
      sum_s[t] = sum_s[t] * keep_s[t] + sum;
      top_s[t] = top;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int g = (t + 256 * i) / HD, d = (t + 256 * i) % HD;
      if (g >= G) continue;
      float o = acc[i] * keep_s[g];
      for (int jj = 0; jj < min(256, seen - j0); ++jj) {
        const uint8_t *tile = tile_of(a.kv, (uint32_t)pages[(j0 + jj) / kPage], h, 1, 10 * HD);
        o = fmaf(sc[g][jj], kv4_value<HD>(tile, 1, jj % kPage, d), o);
      }
      acc[i] = o;
    }
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int g = (t + 256 * i) / HD, d = (t + 256 * i) % HD;
    if (g < G)
      a.out[((size_t)r * a.num_heads + h * G + g) * HD + d] =
          bad ? __uint_as_float(0x7FC00000u) : seen == 0 ? 0.0f : acc[i] / sum_s[g];
  }
}

// ---------------------------------------------------------------------------
// Decode attention
// ---------------------------------------------------------------------------
typedef float f4 __attribute__((ext_vector_type(4)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));

constexpr int kWaves = 4;             // waves of a workgroup
constexpr int kRing = 2;              // pairs of pages a wave has on their way
constexpr int kSplitPages = 2 * kWaves;   // fewest pages of a work item where a merge follows
constexpr int kWholePages = 8 * kWaves;   // pages up to which a context stays one item
constexpr int kMaxSlots = 1024;       // workgroups that a batch is cut for, at most
constexpr float kSlack = 4.0f;        // log2 units a score may pass its reference before a rescale
constexpr float kShift = 11.0f;       // log2 of a weight at the reference
constexpr float kNoRef = -1e30f;      // the reference before the first score
constexpr int kMaxRecords = 4 * kMaxSlots + 2;

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

static __device__ __forceinline__ int wave_scan_dpp(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, true);  // row_shr 1, 2, 4, 8
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);  // lane 15 of rows 0, 2 onto 1, 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);  // lane 31 onto the upper half
  return v;
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
  constexpr int TILE = 10 * HD;
  const uint32_t at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)slot;
  // the slot's last reads are done
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  if constexpr (HD == 128) {
    const int kc = ((l & 15) * 4 + (l >> 4)) * 16;  // lane (c, j): chunk c of position j
    copy16(at, ta, kc);
    copy16(at + 1024, tb, kc);
    copy16(at + 2048, ta, TILE + l * 16);
    copy16(at + 3072, tb, TILE + l * 16);
    const int m = l & 31;
    copy16(at + 4096, (l < 32 ? ta : tb) + (m < 16 ? 8 * HD : TILE + 8 * HD) + (m & 15) * 16);
  } else {
    const uint8_t *t = l < 32 ? ta : tb;
    const int m = l & 31;
    copy16(at, t + m * 16);
    copy16(at + 1024, t + TILE + m * 16);
    const int x = l & 15;
    if (l < 32) copy16(at + 2048, (l < 16 ? ta : tb) + (x < 8 ? 8 * HD : TILE + 8 * HD) + (x & 7) * 16);
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
template <int HD>
static __device__ __forceinline__ void load_query(Wave<HD> &s, const float *q, int G, int l) {
  constexpr int NG = HD / 32;
  const int c = l >> 4, j = l & 15, head = j & 7;
  const float unit = 1.44269504088896341f / sqrtf((float)HD);
  float v[NG][8];
  float top = 0.0f;
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    const float *p = q + (size_t)(head < G ? head : 0) * HD + 32 * g + 8 * c;
    const float4 a = *(const float4 *)p, b = *(const float4 *)(p + 4);
    const float w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      v[g][i] = head < G ? w[i] * unit : 0.0f;
      top = fmaxf(top, fabsf(v[g][i]));
    }
  }
  top = xor32_max(xor16_max(top));
  const int e = top > 0.0f ? __builtin_amdgcn_frexp_expf(top) - 14 : 0;
  s.mult = ldexpf(1.0f, e + 10);
  const float low = j < 8 ? 0.0f : 1.0f;
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      v[g][i] = ldexpf(v[g][i], -e);
      sum += v[g][i];
    }
    sum = xor32_add(xor16_add(sum)) * 0x1p-10f;  // (codes come times 2^-10)
    // high and low parts in the columns, what both leave in a second k-chunk
    const _Float16 sh = (_Float16)sum, sl = (_Float16)(sum - (float)sh);
    const float rest = (sum - (float)sh) - (float)sl;
    s.qsum[g] = (_Float16)(c == 0 ? (j < 8 ? (float)sh : (float)sl) : c == 1 && j < 8 ? rest : 0.0f);
    constexpr int order[8] = {0, 4, 1, 5, 2, 6, 3, 7};  // of codes8
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      const v2h h = half_parts(v[g][order[i]], v[g][order[i + 1]], low);
      s.q[g][i] = h.x;
      s.q[g][i + 1] = h.y;
    }
  }
#pragma unroll
  for (int g = NG; g < 8; ++g) s.qsum[g] = (_Float16)0.0f;
}

template <int HD>
struct DecodeLds {
  union {
    Slot<HD> ring[kWaves][kRing];
    float o[kWaves][kMaxGroup][HD];
  };
  float ref[kWaves][kMaxGroup], sum[kWaves][kMaxGroup];
  int scan[kWaves], live[kWaves], trial[3][kWaves], item[6];
};

struct MergeItem {  // of a (lane, KV head): its chunks' records
  int start, pages, chunks, half;
};
// First page of chunk ch, and its record: the place of its first page in the
// batch divided by half the most pages of a chunk.
static __device__ __forceinline__ int chunk_first(int ch, int pages, int chunks) {
  return ch * (pages / chunks) + min(ch, pages % chunks);
}

// Work items: (lane, KV head, chunk of its pages), a workgroup each. Q, the
// most pages of a chunk, comes from the batch's own lengths: the smallest of
// a few that leaves no more items than the device holds workgroups (`slots`),
// so that they all run at once and end together, `least` pages though. (With
// more than slots / 2 contexts: 2 U / slots, U the batch's pages.) The chunks
// of a context are of equal size to a page, so where there are several they
// hold Q / 2 pages at least.
template <int HD>
__global__ __launch_bounds__(64 * kWaves, HD == 128 ? 3 : 4) void kv4_decode_kernel(
    AttnArgs a, int least, int slots, MergeItem *merge, float *records) {
  __shared__ __align__(16) DecodeLds<HD> s;
  const int t = threadIdx.x, l = t & 63, w = __builtin_amdgcn_readfirstlane(t >> 6);
  const int c = l >> 4, j = l & 15;
  const int Hkv = a.kv.heads, G = a.num_heads / Hkv;
  const float nan = __uint_as_float(0x7FC00000u);

  // the lanes' pages: a thread holds `per` lanes
  const int per = (a.lanes + 64 * kWaves - 1) / (64 * kWaves);
  int pages[4], mine = 0, live = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int at = t * per + i;
    const int n = i < per && at < a.lanes ? a.ctx[at] : 0;
    pages[i] = n > 0 && n <= a.max_ctx ? (n + kPage - 1) / kPage : 0;
    mine += pages[i];
    live += pages[i] > 0;
  }
  const int pages_in = wave_scan_dpp(mine), live_in = wave_scan_dpp(live);
  if (l == 63) {
    s.scan[w] = pages_in;
    s.live[w] = live_in;
  }
  __syncthreads();
  int total = 0, pages_before = pages_in - mine, segments = 0;
#pragma unroll
  for (int i = 0; i < kWaves; ++i) {
    if (i < w) pages_before += s.scan[i];
    total += s.scan[i];
    segments += s.live[i];
  }
  total *= Hkv;
  segments *= Hkv;
  const int room = max(slots - segments, slots / 2);
  int Q = max(least, (total + room - 1) / room);
  if (Q > least && segments < slots / 2) {
    // Q leaves slots items at most; try Q - k / 4 of the way to the mean
    const int low = max(least, (total + slots - 1) / slots), step = (Q - low + 3) / 4;
    int n[3];
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      const int q = max(low, Q - (k + 1) * step);
      n[k] = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i < per) n[k] += (pages[i] + q - 1) / q;
      n[k] = wave_scan_dpp(n[k] * Hkv);
      if (l == 63) s.trial[k][w] = n[k];
    }
    __syncthreads();
    const int full = Q;
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      const int all = s.trial[k][0] + s.trial[k][1] + s.trial[k][2] + s.trial[k][3];
      if (all <= slots) Q = max(low, full - (k + 1) * step);
    }
  }
  Q = (Q + 1) & ~1;  // so that half of it is whole
  int items = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (i < per) items += (pages[i] + Q - 1) / Q * Hkv;
  const int items_in = wave_scan_dpp(items);
  __syncthreads();
  if (l == 63) s.scan[w] = items_in;
  __syncthreads();
  int all = 0, items_before = items_in - items;
#pragma unroll
  for (int i = 0; i < kWaves; ++i) {
    if (i < w) items_before += s.scan[i];
    all += s.scan[i];
  }

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
  const int item = blockIdx.x;
  if (item >= all) return;
  if (item >= items_before && item < items_before + items) {
    int at = items_before, pb = pages_before;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int chunks = (pages[i] + Q - 1) / Q, r = item - at;
      if (r >= 0 && r < chunks * Hkv) {
        s.item[0] = t * per + i;
        s.item[1] = r / chunks;
        s.item[2] = r % chunks;
        s.item[3] = chunks;
        s.item[4] = pages[i];
        s.item[5] = pb * Hkv + r / chunks * pages[i];
      }
      at += chunks * Hkv;
      pb += pages[i];
    }
  }
  __syncthreads();
  const int lane = __builtin_amdgcn_readfirstlane(s.item[0]), h = __builtin_amdgcn_readfirstlane(s.item[1]);
  const int ch = __builtin_amdgcn_readfirstlane(s.item[2]), chunks = __builtin_amdgcn_readfirstlane(s.item[3]);
  const int lane_pages = __builtin_amdgcn_readfirstlane(s.item[4]), start = __builtin_amdgcn_readfirstlane(s.item[5]);
  const int first = chunk_first(ch, lane_pages, chunks), end = chunk_first(ch + 1, lane_pages, chunks);
  const int ctx = __builtin_amdgcn_readfirstlane(a.ctx[lane]);
  if (merge && ch == 0 && t == 0) merge[lane * Hkv + h] = {start, lane_pages, chunks, Q / 2};

  Wave<HD> s_w;
#pragma unroll
  for (int e = 0; e < HD / 16; ++e) s_w.o[e] = f4{0.0f, 0.0f, 0.0f, 0.0f};
  s_w.om = f4{0.0f, 0.0f, 0.0f, 0.0f};
  s_w.ref = kNoRef;
  s_w.e = -14;
  s_w.bound = 1u << 10 | 1u << 26;
  load_query(s_w, a.q + ((size_t)lane * a.num_heads + h * G) * HD, G, l);

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

  // the waves' states, then their sums weighted by 2^(reference - the largest)
  const float unit = ldexpf(1.0f, s_w.e + 10);
  float om[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) om[r] = xor32_add(s_w.om[r]);
#pragma unroll
  for (int e = 0; e < HD / 16; ++e)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float m = e / 2 == 0 ? row_lane<0>(om[r]) : e / 2 == 1 ? row_lane<1>(om[r])
                      : e / 2 == 2 ? row_lane<2>(om[r]) : row_lane<3>(om[r]);
      const float v = fmaf(xor32_add(s_w.o[e][r]), unit, m);
      if (c < 2) s.o[w][4 * c + r][16 * e + j] = v;
    }
  if (l < kMaxGroup) s.ref[w][l] = s_w.ref;
#pragma unroll
  for (int r = 0; r < 4; ++r)
    if (c < 2 && j == HD / 32) s.sum[w][4 * c + r] = om[r];
  bad = __syncthreads_or(bad);
  float *rec = records + (size_t)((start + first) / (Q / 2)) * (kMaxGroup * (HD + 2));
  for (int i = t; i < G * HD; i += 64 * kWaves) {
    const int g = i / HD, d = i % HD;
    float top = s.ref[0][g];
#pragma unroll
    for (int v = 1; v < kWaves; ++v) top = fmaxf(top, s.ref[v][g]);
    float L = 0.0f, O = 0.0f;
#pragma unroll
    for (int v = 0; v < kWaves; ++v) {
      const float f = __builtin_amdgcn_exp2f(s.ref[v][g] - top);
      L = fmaf(s.sum[v][g], f, L);
      O = fmaf(s.o[v][g][d], f, O);
    }
    if (bad) L = nan;
    if (chunks == 1) {
      a.out[((size_t)lane * a.num_heads + h * G + g) * HD + d] = O / L;
    } else {
      rec[g * (HD + 2) + 2 + d] = O;
      if (d == 0) {
        rec[g * (HD + 2)] = top;
        rec[g * (HD + 2) + 1] = L;
      }
    }
  }
}

// The chunks of a (lane, query head) added up, weighted by 2^(reference - the
// largest): HD / 4 threads a record, in a fixed order.
template <int HD>
__global__ __launch_bounds__(256) void kv4_merge_kernel(AttnArgs a, const MergeItem *merge,
                                                        const float *records) {
  constexpr int TPR = HD / 4, R = 256 / TPR;  // threads a record, records at a time
  __shared__ float f_s[kMaxRecords];
  __shared__ float4 o_s[R][TPR];
  __shared__ float wave_s[2][4];
  const int t = threadIdx.x, l = t & 63, w = t >> 6;
  const int lane = blockIdx.x / a.num_heads, qh = blockIdx.x % a.num_heads;
  const int G = a.num_heads / a.kv.heads, g = qh % G;
  const MergeItem m = merge[lane * a.kv.heads + qh / G];
  if (m.chunks <= 1) return;
  auto rec = [&](int ch) {
    return records + ((size_t)((m.start + chunk_first(ch, m.pages, m.chunks)) / m.half) * kMaxGroup + g) * (HD + 2);
  };
  float top = -INFINITY;
  for (int ch = t; ch < m.chunks; ch += 256) {
    f_s[ch] = rec(ch)[0];
    top = fmaxf(top, f_s[ch]);
  }
  top = wave_max(top);
  if (l == 0) wave_s[0][w] = top;
  __syncthreads();
  top = fmaxf(fmaxf(wave_s[0][0], wave_s[0][1]), fmaxf(wave_s[0][2], wave_s[0][3]));
  float sum = 0.0f;
  for (int ch = t; ch < m.chunks; ch += 256) {
    const float f = __builtin_amdgcn_exp2f(f_s[ch] - top);
    f_s[ch] = f;
    sum = fmaf(rec(ch)[1], f, sum);
  }
  sum = wave_sum(sum);
  if (l == 0) wave_s[1][w] = sum;
  __syncthreads();
  sum = (wave_s[1][0] + wave_s[1][1]) + (wave_s[1][2] + wave_s[1][3]);
  const int rw = t / TPR, d = t % TPR * 4;
  float4 o = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int ch = rw; ch < m.chunks; ch += R) {
    const float *p = rec(ch) + 2 + d;
    const float f = f_s[ch];
    const float2 x = *(const float2 *)p, y = *(const float2 *)(p + 2);
    o.x = fmaf(x.x, f, o.x);
    o.y = fmaf(x.y, f, o.y);
    o.z = fmaf(y.x, f, o.z);
    o.w = fmaf(y.y, f, o.w);
  }
  o_s[rw][t % TPR] = o;
  __syncthreads();
  if (t < HD) {
    float v = 0.0f;
#pragma unroll
    for (int r = 0; r < R; ++r) v += ((const float *)&o_s[r][t / 4])[t % 4];
    a.out[((size_t)lane * a.num_heads + qh) * HD + t] = v / sum;
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
  if (need == 0 || ws_bytes < need || max_ctx == 0 || max_ctx > (1u << 30) ||
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
    const bool split = (max_ctx + gk::kPage - 1) / gk::kPage > (uint32_t)gk::kWholePages;
    const int least = split ? gk::kSplitPages : gk::kWholePages;
    auto *merge = split ? (gk::MergeItem *)ws : nullptr;
    float *records = (float *)((char *)ws + merge_bytes(lanes, pool->num_kv_heads));
    const int slots = std::min(gk::kMaxSlots, ctx->props.multiProcessorCount * (pool->head_dim == 128 ? 3 : 4));
    // items at most: slots, or where there are many contexts one each and slots / 2 more
    const uint64_t heads = (uint64_t)lanes * a.kv.heads, each = ((max_ctx + gk::kPage - 1) / gk::kPage + least - 1) / least;
    const uint64_t most = heads <= (uint64_t)slots / 2 ? slots : heads + slots / 2;
    const uint32_t grid = (uint32_t)std::max<uint64_t>(lanes, std::min(heads * each, most));
    if (pool->head_dim == 128) {
      gk::kv4_decode_kernel<128><<<grid, 64 * gk::kWaves, 0, st>>>(a, least, slots, merge, records);
      if (split) gk::kv4_merge_kernel<128><<<lanes * num_heads, 256, 0, st>>>(a, merge, records);
    } else {
      gk::kv4_decode_kernel<64><<<grid, 64 * gk::kWaves, 0, st>>>(a, least, slots, merge, records);
      if (split) gk::kv4_merge_kernel<64><<<lanes * num_heads, 256, 0, st>>>(a, merge, records);
    }
    GH_CHECK(ctx, hipGetLastError());
    return GLACIER_HIP_OK;
  }
  const dim3 grid(max_rows, pool->num_kv_heads);
  if (pool->head_dim == 128) gk::kv4_attn_kernel<128><<<grid, 256, 0, st>>>(a);
  else gk::kv4_attn_kernel<64><<<grid, 256, 0, st>>>(a);
  GH_CHECK(ctx, hipGetLastError());
  return GLACIER_HIP_OK;
}

template <class T>
void append_launch(const gk::Kv4 &kv, uint32_t hd, const void *k, const void *v, uint64_t ks,
                   uint64_t vs, const int64_t *slots, uint32_t rows, hipStream_t st) {
  const uint64_t threads = (uint64_t)rows * 2 * kv.heads * (hd / 32);
  const uint32_t grid = (uint32_t)((threads + 255) / 256);
  if (hd == 128)
    gk::kv4_append_kernel<128, T><<<grid, 256, 0, st>>>(kv, (const T *)k, (const T *)v, ks, vs, slots, (int)rows);
  else
    gk::kv4_append_kernel<64, T><<<grid, 256, 0, st>>>(kv, (const T *)k, (const T *)v, ks, vs, slots, (int)rows);
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
      free_pages_dev, free_count, free_taken_dev, row_start_dev, ctx_after_dev, result_dev);
  GH_CHECK(ctx, hipGetLastError());
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
  const uint64_t threads = (uint64_t)rows * pool->num_kv_heads * pool->head_dim;
  if ((threads + 255) / 256 > 0x7FFFFFFFull) return GLACIER_HIP_SHAPE_MISMATCH;
  const uint32_t grid = (uint32_t)((threads + 255) / 256);
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
  return merge_bytes(lanes, num_kv_heads) +
         (uint64_t)gk::kMaxRecords * gk::kMaxGroup * (head_dim + 2) * sizeof(float);
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
