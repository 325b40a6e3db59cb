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
      max_ctx > (uint64_t)max_pages * gk::kPage)
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
  return 256;
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
