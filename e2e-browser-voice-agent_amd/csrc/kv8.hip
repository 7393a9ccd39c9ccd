// kv8.hip -- the paged 8-bit K/V cache: plan, append, read and attention (include/q4hip.h, q4hip_kv8_*).
#include "kv8.h"

#include <algorithm>
#include <cmath>
#include <new>

#include "host.h"
#include "kv8_attend.h"
#include "kv8_plan.h"

namespace q4 {
namespace {

// Workgroups of attention that a step's pages are shared among: one for each CU.  (512: a prompt of 640 rows 24 us for 13.)
constexpr int kItemsAim = 256;
// Entries of a plan's lists (rows, the caller's tables) up to which one workgroup fills them, with the sums in shared memory (one
// launch against two: 200 sequences with tables, 6,400 entries, 9.0 us and 11.1; 48 with 2,171 rows 7.2 and 8.4) and in
// global memory (6,000 sequences 63 us and 38).
constexpr size_t kFillInPlan = 8192, kFillInPlanGlobal = 2048;
// Workgroups of attention at most; each takes every so-manieth tile or item.  (1,024: up to 9% more time, 512: up to 35%, as the
// tiles of a step differ in length.)
constexpr int64_t kMostWorkgroups = 8192;

// The quotient x / s rounded to fp32, from r = 1 / s rounded: one correction of x * r by its residual gives it
// (P. Markstein, IBM J. Res. Dev. 34(1), 1990) where the residual is exact, which |x / s| >= 1/4 and s >= 2^-100 make
// it; a smaller quotient has the code 0 either way.  Then rounded to the nearest even integer by the
// addition of 1.5 * 2^23, whose last byte becomes the code.
__device__ uint32_t code_bits(float x, float s, float r) {
  const float q0 = x * r, q = __builtin_fmaf(__builtin_fmaf(-q0, s, x), r, q0);
  return __float_as_uint(q + (12582912.0f + 128.0f));
}

// The same of any x: NaN 0, infinities the largest code.
__device__ uint32_t code_bits_any(float x, float s) {
  const float q = x != x || !(s > 0.0f) ? 0.0f : __builtin_fminf(__builtin_fmaxf(x / s, -127.0f), 127.0f);
  return __float_as_uint(q + (12582912.0f + 128.0f));
}

// The smallest k >= 0 with s * 2^k >= t (s, t > 0).
__device__ int doublings(float s, float t) {
  if (!(t > s)) return 0;
  const float ms = __builtin_amdgcn_frexp_mantf(s), mt = __builtin_amdgcn_frexp_mantf(t);
  return __builtin_amdgcn_frexp_expf(t) - __builtin_amdgcn_frexp_expf(s) + (mt > ms ? 1 : 0);
}

// RoPE of 4 columns and of those half a head later (kernels.c:337-345): cs holds their cosines and sines in turn.
__device__ inline void turn(float4& lo, float4& hi, const float4* cs) {
  const float4 a = cs[0], b = cs[1], x = lo, y = hi;
  lo = {x.x * a.x - y.x * a.y, x.y * a.z - y.y * a.w, x.z * b.x - y.z * b.y, x.w * b.z - y.w * b.w};
  hi = {y.x * a.x + x.x * a.y, y.y * a.z + x.y * a.w, y.z * b.x + x.z * b.y, y.w * b.z + x.w * b.w};
}

// A run of rows (blockIdx.x) of one kv head; K for blockIdx.z = 0, else V.  The rows pass through shared memory, where
// their 32-bit values are turned into the order of the codes; a thread forms 16 codes that lie together, so that they leave as
// 16 bytes; one barrier, as each wave's maximum and its check for infinities cross it together.
// Bytes bound it: 15,808 rows of 8 kv heads of 128 (bf16) take 24.4 us, 4.0 TB/s of rows in and codes out; a token's run
// is one chain of loads, 5.6 us.  A code needs the rounded quotient, which two fused operations give (code_bits), where the
// division's dozen instructions would bound the kernel.
// kWide: rows whose 16 bytes can be loaded at once.
// kRope: K is turned by its positions first, and q (blockIdx.z = 2: the heads that read this kv head) in place; a launch less in each
// layer of a batch's step (32 sequences at 1,024 positions, 28 layers, 2.66 -> 2.61 ms).
template <int HD, class T, bool kWide, bool kRope>
__global__ __launch_bounds__(2 * HD) void k_kv8_append(Kv8View v, int layer, const T* __restrict__ k, const T* __restrict__ val,
                                                     int64_t k_stride, int64_t v_stride, int rows, int g0, Kv8Rope rope) {
  __shared__ float tile[kKv8Block][HD + 1];
  __shared__ float most[HD / 32];
  __shared__ int odd[HD / 32];                 // of a wave's values, whether one is not finite
  const int g = g0 + blockIdx.y, tid = threadIdx.x, lane = tid & 63;
  const bool is_v = blockIdx.z == 1;
  const Kv8Head head = *v.head;
  const Kv8Run run = v.runs[blockIdx.x];       // on its way together with the head: the grid is no larger than the list
  if (head.rows > rows) {                      // replayed on a larger plan than it was launched for
    if (tid == 0) v.head->status = KV8_STALE;
    return;
  }
  if ((int)blockIdx.x >= head.runs) return;
  const int m = run.m, f = run.slot % kKv8Block;
  if constexpr (kRope)
    if (blockIdx.z == 2) {
      const int G = v.H / v.KVH;
      for (int i = tid; i < m * G * (HD / 8); i += 2 * HD) {
        const int r = i / (G * (HD / 8)), e = i - r * (G * (HD / 8)), c = e % (HD / 8) * 4;
        float4* const p = (float4*)(rope.q + (run.t + r) * rope.q_stride + (g * G + e / (HD / 8)) * HD + c);
        float4 lo = p[0], hi = p[HD / 8];
        turn(lo, hi, (const float4*)(rope.table + (size_t)rope.pos[run.t + r] * HD + 2 * c));
        p[0] = lo;
        p[HD / 8] = hi;
      }
      return;
    }
  const int64_t ld = is_v ? v_stride : k_stride;
  const T* x = (is_v ? val : k) + (int64_t)run.t * ld + (int)blockIdx.y * HD;
  const size_t block = ((size_t)layer * v.pages + run.slot / kKv8Block) * v.KVH + g;
  float* const scale = (float*)(v.scales + block) + (is_v ? 1 : 0);
  uint4* const codes = (uint4*)(v.codes + (block * 2 + (is_v ? 1 : 0)) * (kKv8Block * HD));
  const bool whole = m == kKv8Block;
  const float before = *scale;
  uint4 w = {};
  if (!whole) w = codes[tid];
  float a = 0.0f;
  bool strange = false;
  auto take = [&](int r, int c, float y) {
    tile[f + r][c] = y;
    const float z = __builtin_fabsf(y);
    if (z < __builtin_inff()) a = __builtin_fmaxf(a, z);
    else strange = true;
  };
  if (kRope && !is_v) {
    for (int i = tid; i < m * (HD / 8); i += 2 * HD) {
      const int r = i / (HD / 8), c = i % (HD / 8) * 4;
      const float4* const p = (const float4*)(x + r * ld + c);
      float4 lo = p[0], hi = p[HD / 8];
      turn(lo, hi, (const float4*)(rope.table + (size_t)rope.pos[run.t + r] * HD + 2 * c));
      const float *const y0 = (const float*)&lo, *const y1 = (const float*)&hi;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        take(r, c + j, y0[j]);
        take(r, c + HD / 2 + j, y1[j]);
      }
    }
  } else if constexpr (kWide) {
    constexpr int kVec = 16 / sizeof(T), kCols = HD / kVec;
    for (int i = tid; i < m * kCols; i += 2 * HD) {
      const int r = i / kCols, c = i % kCols * kVec;
      struct alignas(16) Vec { T y[kVec]; };
      const Vec z = *(const Vec*)(x + r * ld + c);
#pragma unroll
      for (int j = 0; j < kVec; j++) take(r, c + j, (float)z.y[j]);
    }
  } else {
    for (int i = tid; i < m * HD; i += 2 * HD) take(i / HD, i % HD, (float)x[i / HD * ld + i % HD]);
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) a = __builtin_fmaxf(a, __shfl_xor(a, d));
  const bool any_strange = __builtin_amdgcn_ballot_w64(strange) != 0;
  if (lane == 0) { most[tid >> 6] = a; odd[tid >> 6] = any_strange; }
  __syncthreads();
  int any_odd = 0;
  a = 0.0f;
#pragma unroll
  for (int i = 0; i < HD / 32; i++) {
    a = __builtin_fmaxf(a, most[i]);
    any_odd |= odd[i];
  }
  const float old = f ? before : 0.0f, t127 = a / 127.0f, need = t127 < kKv8MinScale ? 0.0f : t127;
  const int twice = old > 0.0f ? doublings(old, need) : 0;
  const float s = old > 0.0f ? __builtin_ldexpf(old, twice) : need;
  const bool any = any_odd || !(s > 0.0f);
  const float r = any ? 0.0f : 1.0f / s;
  const int q = tid >> 6;
  uint32_t* const words = (uint32_t*)&w;
  bool changed = whole;
#pragma unroll
  for (int j = 0; j < 16; j += 4) {
    // four codes: columns of a position of K, positions of a column of V, one after the other
    int tok, col;
    if (is_v) {
      tok = ((j >> 2) & 1) * 16 + (lane >> 4) * 4;
      col = (2 * q + (j >> 3)) * 16 + (lane & 15);
    } else {
      tok = q / (HD / 64) * 16 + (lane & 15);
      col = (2 * (q % (HD / 64)) + (j >> 3)) * 32 + (lane >> 4) * 8 + (j & 7);
    }
    const int dt = is_v ? 1 : 0, dc = 1 - dt;
    if (whole && !any) {
      uint32_t c[4];
#pragma unroll
      for (int b = 0; b < 4; b++) c[b] = code_bits(tile[tok + b * dt][col + b * dc], s, r);
      const uint32_t lo = __builtin_amdgcn_perm(c[1], c[0], 0x0c0c0400u), hi = __builtin_amdgcn_perm(c[3], c[2], 0x04000c0cu);
      words[j >> 2] = lo | hi;
      continue;
    }
    for (int b = 0; b < 4; b++) {
      const int tk = tok + b * dt, sh = 8 * b;
      uint32_t c;
      if (tk >= f && tk < f + m) {
        const float y = tile[tk][col + b * dc];
        c = any ? code_bits_any(y, s) : code_bits(y, s, r);
      } else if (tk < f && twice) {
        const int before_code = (int)(words[j >> 2] >> sh & 255) - 128;
        c = (uint32_t)((int)__builtin_rintf(__builtin_ldexpf((float)before_code, -twice)) + 128);
      } else {
        continue;
      }
      words[j >> 2] = (words[j >> 2] & ~(255u << sh)) | (c & 255u) << sh;
      changed = true;
    }
  }
  if (changed) codes[tid] = w;
  if (tid == 0 && s != before) *scale = s;      // every thread has read the old one before the barriers
}

// The values that the cache stands for at n pairs of a sequence and a position; 0 where it holds none.  A thread
// forms 4 columns of K and V of one kv head.  The fp32 rows that it writes bound it: 15,950 positions of 8 heads of 128 in
// 35 us, 4.7 TB/s with the codes.
template <int HD>
__global__ __launch_bounds__(256) void k_kv8_read(Kv8View v, int layer, const int* __restrict__ seq, const int* __restrict__ pos,
                                                  int n, float* __restrict__ k, float* __restrict__ val) {
  constexpr int kCols = HD / 4, kRows = 256 / kCols;
  const int g = blockIdx.y, d = threadIdx.x % kCols * 4;
  for (int i = blockIdx.x * kRows + threadIdx.x / kCols; i < n; i += gridDim.x * kRows) {
    const int b = seq[i], p = pos[i];
    float a[4] = {}, c[4] = {};
    if (b >= 0 && b < v.B && p >= 0 && p < v.lens[b]) {
      const int t = p % kKv8Block;
      const size_t block = ((size_t)layer * v.pages + v.table[(size_t)b * v.W + p / kKv8Block]) * v.KVH + g;
      const uint8_t* codes = v.codes + block * 2 * (kKv8Block * HD);
      const float2 s = v.scales[block];
      const uint32_t kw = *(const uint32_t*)(codes + kv8_k_byte(HD, t, d));
#pragma unroll
      for (int j = 0; j < 4; j++) {
        a[j] = s.x * (float)((int)(kw >> 8 * j & 255) - 128);
        c[j] = s.y * (float)((int)codes[kKv8Block * HD + kv8_v_byte(t, d + j)] - 128);
      }
    }
    const size_t at = ((size_t)i * v.KVH + g) * HD + d;
#pragma unroll
    for (int j = 0; j < 4; j++) { k[at + j] = a[j]; val[at + j] = c[j]; }
  }
}

// The free pages in the order in which they are taken, and a table without pages.
__global__ __launch_bounds__(256) void k_kv8_reset(Kv8View v) {
  const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
  if (i < (size_t)v.B * v.W) v.table[i] = -1;
  if (i < (size_t)v.pages) v.stack[i] = v.pages - 1 - (int)i;
  if (i <= (size_t)v.B) {
    v.starts[i] = 0;
    if (i < (size_t)v.B) { v.held[i] = 0; v.base[i] = 0; v.lens[i] = 0; }
  }
  if (i == 0) *v.head = Kv8Head{KV8_OK, 0, v.pages, 0, 0, 0, 1};
}

// At most so many tiles have `rows` rows: of full ones, and of a last one of each sequence.
size_t tiles_bound(const Kv8View& v, int rows) {
  return (size_t)((int64_t)rows * (v.H / v.KVH) / kKv8TileRows + std::min(v.B, rows / (v.unit_rows + 1)) + 1);
}

int elem_size(int type) { return type == Q4HIP_TYPE_F32 ? 4 : 2; }

// Whether 16 bytes of any row can be loaded at once.
bool aligned16(const void* p, int64_t stride, int type) {
  return ((uintptr_t)p | (uintptr_t)(stride * elem_size(type))) % 16 == 0;
}

int check_layer(const q4hip_kv8* kv, int layer, int type) {
  if (layer < 0 || layer >= kv->v.layers) return fail(Q4HIP_EINVAL, "layer %d of %d", layer, kv->v.layers);
  if (type != Q4HIP_TYPE_F32 && type != Q4HIP_TYPE_F16 && type != Q4HIP_TYPE_BF16)
    return fail(Q4HIP_ETYPE, "type %d: expected F32, F16 or BF16", type);
  return Q4HIP_OK;
}

// `rows` rows of `width` elements, `stride` elements apart.
int check_rows(const q4hip_kv8* kv, const void* p, int rows, int width, int64_t stride, int type, const char* what) {
  const int es = elem_size(type);
  if ((uintptr_t)p % es) return fail(Q4HIP_EINVAL, "%s: not aligned to its type", what);
  if (stride < width) return fail(Q4HIP_EINVAL, "%s: rows of %d values, %lld apart", what, width, (long long)stride);
  if (stride > ((int64_t)1 << 31)) return fail(Q4HIP_EINVAL, "%s: rows %lld values apart", what, (long long)stride);
  return check_device_span(p, ((size_t)(rows - 1) * stride + width) * es, kv->device, what);
}

// Rows that one call reads and another buffer's that it writes must not share a byte.  Neighbouring columns of the same
// rows may: where the strides differ, the whole spans count.
int check_apart(const void* p, int64_t p_stride, const void* out, int64_t out_stride, int rows, int width, int type) {
  const int es = elem_size(type);
  const uintptr_t a = (uintptr_t)p, b = (uintptr_t)out, w = (uintptr_t)width * es;
  const uintptr_t a_end = a + (uintptr_t)(rows - 1) * p_stride * es + w, b_end = b + (uintptr_t)(rows - 1) * out_stride * es + w;
  if (a_end <= b || b_end <= a) return Q4HIP_OK;
  if (p_stride == out_stride) {
    const uintptr_t s = (uintptr_t)p_stride * es, d = b >= a ? (b - a) % s : (s - (a - b) % s) % s;
    if (d >= w && s - d >= w) return Q4HIP_OK;
  }
  return fail(Q4HIP_EINVAL, "q and out overlap");
}

// int32 arrays of n elements; NULL or an empty one is not looked at.
int check_ints(const q4hip_kv8* kv, const void* p, size_t n, const char* what) {
  if (!p || !n) return Q4HIP_OK;
  if ((uintptr_t)p % 4) return fail(Q4HIP_EINVAL, "%s: not aligned to its type", what);
  return check_device_span(p, n * 4, kv->device, what);
}

int plan_error(const q4hip_kv8* kv, int status) {
  switch (status) {
    case KV8_OK: return Q4HIP_OK;
    case KV8_BAD_LENGTH: return fail(Q4HIP_EINVAL, "plan: a negative length");
    case KV8_TOO_LONG: return fail(Q4HIP_ECONTEXT, "plan: a sequence longer than %d positions", kv->v.max_len);
    case KV8_STALE:
      return fail(Q4HIP_ESTATE, "append or attend replayed on a plan of more rows than they were captured for");
    case KV8_ROWS: return fail(Q4HIP_EINVAL, "plan: more rows than it was called for");
    default: return fail(Q4HIP_ECONTEXT, "plan: more than the pool's %d pages", kv->v.pages);
  }
}

// The capture that `s` is in, 0 for none.
int capture_of(hipStream_t s, unsigned long long* id) {
  hipStreamCaptureStatus st;
  HIPCHK(hipStreamGetCaptureInfo(s, &st, id));
  if (st == hipStreamCaptureStatusNone) *id = 0;
  return Q4HIP_OK;
}

// Rows of the plan that a call on `s` follows: the one captured before it in the same capture, else the last one outside of any.
int rows_on(const q4hip_kv8* kv, hipStream_t s, int* rows) {
  unsigned long long id;
  const int rc = capture_of(s, &id);
  *rows = id && id == kv->capture ? kv->capture_rows : kv->rows;
  return rc;
}

int read_head(q4hip_kv8* kv, hipStream_t s) {
  HIPCHK(hipMemcpyAsync(kv->pin, kv->v.head, sizeof(Kv8Head), hipMemcpyDeviceToHost, s));
  HIPCHK(hipStreamSynchronize(s));
  return Q4HIP_OK;
}

template <class F>
void by_type(int type, F f) {
  if (type == Q4HIP_TYPE_F32) f(float());
  else if (type == Q4HIP_TYPE_F16) f(_Float16());
  else f(__bf16());
}

}  // namespace

void kv8_launch_plan(q4hip_kv8* kv, hipStream_t s, const int* have, const int* add, int rows, int* starts, int* positions, int* slots,
                     int* tables) {
  const Kv8View& v = kv->v;
  // What the lists hold in all: in the same launch if the one workgroup is through with it in a few rounds, which takes less
  // than a second launch does.
  const size_t items = rows + std::min<size_t>(kKv8MoreItems * v.items_aim, rows ? (size_t)v.pages * rows / kKv8MinPart : 0);
  const size_t entries = std::max<size_t>(items, tables ? (size_t)v.B * v.W : 0);
  const bool shared = v.B <= kPlanShared, fill = entries <= (shared ? kFillInPlan : kFillInPlanGlobal);
  if (shared) {
    const int threads = v.B <= 512 && (!fill || entries <= 2048) ? 512 : kPlanThreads;
    k_kv8_plan<true><<<1, threads, 0, s>>>(v, have, add, rows, starts, positions, slots, tables, fill);
  } else {
    k_kv8_plan<false><<<1, kPlanThreads, 0, s>>>(v, have, add, rows, starts, positions, slots, tables, fill);
  }
  if (!fill) k_kv8_fill<<<(unsigned)std::min<size_t>((entries + 255) / 256, 1024), 256, 0, s>>>(v, positions, slots, tables);
}

namespace {

// runs of a sequence: its rows over 32, and two at its ends
unsigned runs_bound(const Kv8View& v, int rows) {
  return (unsigned)std::min<int64_t>(rows, rows / kKv8Block + 2 * (int64_t)std::min(v.B, rows));
}

}  // namespace

void kv8_launch_append(q4hip_kv8* kv, hipStream_t s, int layer, const void* k, const void* v, int type, int64_t k_stride,
                       int64_t v_stride, int g0, int heads, int rows) {
  const Kv8View& w = kv->v;
  if (!rows) return;
  const dim3 grid(runs_bound(w, rows), (unsigned)heads, 2);
  const bool wide = aligned16(k, k_stride, type) && aligned16(v, v_stride, type);
  by_type(type, [&](auto zero) {
    using T = decltype(zero);
    auto* fn = w.HD == 64 ? (wide ? k_kv8_append<64, T, true, false> : k_kv8_append<64, T, false, false>)
                          : (wide ? k_kv8_append<128, T, true, false> : k_kv8_append<128, T, false, false>);
    fn<<<grid, 2 * w.HD, 0, s>>>(w, layer, (const T*)k, (const T*)v, k_stride, v_stride, rows, g0, Kv8Rope{});
  });
}

void kv8_launch_append_rope(q4hip_kv8* kv, hipStream_t s, int layer, float* qkv, int64_t stride, const float* table, const int* pos,
                            int rows) {
  const Kv8View& w = kv->v;
  if (!rows) return;
  const float *const k = qkv + w.H * w.HD, *const v = k + w.KVH * w.HD;
  auto* fn = w.HD == 64 ? k_kv8_append<64, float, true, true> : k_kv8_append<128, float, true, true>;
  fn<<<dim3(runs_bound(w, rows), (unsigned)w.KVH, 3), 2 * w.HD, 0, s>>>(w, layer, k, v, stride, stride, rows, 0,
                                                                  Kv8Rope{table, pos, qkv, stride});
}

void kv8_launch_attend(q4hip_kv8* kv, hipStream_t s, int layer, const void* q, void* out, int type, int64_t q_stride,
                       int64_t out_stride, float scale, int rows) {
  const Kv8View& w = kv->v;
  if (!rows) return;
  // the softmax's exponentials are powers of two
  const float log2_scale = (float)((scale == 0.0f ? 1.0 / std::sqrt((double)w.HD) : (double)scale) * 1.4426950408889634);
  const int units = (int)std::min<int64_t>(rows, rows / w.unit_rows + (int64_t)std::min(w.B, rows));
  const int64_t items = units + std::min<int64_t>(kKv8MoreItems * w.items_aim, (int64_t)units * (w.pages / kKv8MinPart));
  const bool wide = aligned16(q, q_stride, type) && aligned16(out, out_stride, type);
  const bool few = rows <= w.unit_rows;    // neither wide units nor tiles
  const int64_t work = items * w.KVH * w.row_tiles + (few ? 0 : (int64_t)tiles_bound(w, rows) * w.KVH);
  const unsigned grid = (unsigned)std::min<int64_t>(work, kMostWorkgroups);
  by_type(type, [&](auto zero) {
    using T = decltype(zero);
    auto* fn = w.HD == 64 ? (few ? k_kv8_attend<64, T, 0> : k_kv8_attend<64, T, 2>)
                          : (few ? k_kv8_attend<128, T, 0> : k_kv8_attend<128, T, 2>);
    fn<<<grid, 256, 0, s>>>(w, layer, (const T*)q, (T*)out, q_stride, out_stride, log2_scale, rows, wide);
  });
}

void kv8_launch_read(q4hip_kv8* kv, hipStream_t s, int layer, const int* seq, const int* pos, int n, float* k, float* v) {
  const Kv8View& w = kv->v;
  const int per = 1024 / w.HD;                 // rows of a workgroup
  const dim3 grid((unsigned)std::min((n + per - 1) / per, 16384), (unsigned)w.KVH);
  if (w.HD == 64) k_kv8_read<64><<<grid, 256, 0, s>>>(w, layer, seq, pos, n, k, v);
  else k_kv8_read<128><<<grid, 256, 0, s>>>(w, layer, seq, pos, n, k, v);
}

}  // namespace q4

using namespace q4;

extern "C" {

void q4hip_kv8_destroy(q4hip_kv8* kv) {
  if (!kv) return;
  (void)hipSetDevice(kv->device);
  if (kv->stream) (void)hipStreamSynchronize(kv->stream);
  Kv8View& v = kv->v;
  void* bufs[] = {v.codes, v.scales, v.table, v.held, v.stack, v.head, v.base, v.lens, v.starts, v.free_at, v.take_at,
                  v.run_at, v.item_at, v.part_at, v.tile_at, v.runs, v.items, v.tiles, v.part_o, v.part_ml, v.arrived};
  for (void* p : bufs) if (p) (void)hipFree(p);
  if (kv->pin) (void)hipHostFree(kv->pin);
  if (kv->stream) (void)hipStreamDestroy(kv->stream);
  delete kv;
}

int q4hip_kv8_create(q4hip_kv8** out, int layers, int heads, int kv_heads, int head_dim, int seqs, int max_len, int pages,
                     int max_rows, int device) {
  if (!out) return fail(Q4HIP_EINVAL, "null argument");
  *out = nullptr;
  if (layers <= 0 || heads <= 0 || kv_heads <= 0 || seqs <= 0 || max_len <= 0 || pages <= 0 || max_rows <= 0)
    return fail(Q4HIP_EINVAL, "bad configuration");
  if (heads % kv_heads) return fail(Q4HIP_EINVAL, "heads must be a multiple of kv_heads");
  if (head_dim != 64 && head_dim != 128) return fail(Q4HIP_EINVAL, "head_dim %d unsupported (64 or 128)", head_dim);
  if (heads > 65535 || layers > 65535) return fail(Q4HIP_EINVAL, "bad configuration");
  if (heads / kv_heads > 1024) return fail(Q4HIP_EINVAL, "more than 1024 heads to a kv head");
  if (pages > INT32_MAX / kKv8Block) return fail(Q4HIP_EINVAL, "%d pages: at most %d", pages, INT32_MAX / kKv8Block);
  if (max_len > INT32_MAX - kKv8Block) return fail(Q4HIP_EINVAL, "sequences of %d positions", max_len);
  int ndev = 0;
  HIPCHK(hipGetDeviceCount(&ndev));
  if (device < 0 || device >= ndev) return fail(Q4HIP_EINVAL, "device %d of %d", device, ndev);
  HIPCHK(hipSetDevice(device));
  q4hip_kv8* kv = new (std::nothrow) q4hip_kv8();
  if (!kv) return fail(Q4HIP_EHIP, "out of host memory");
  kv->device = device;
  kv->max_rows = max_rows;
  Kv8View& v = kv->v;
  v.layers = layers; v.H = heads; v.KVH = kv_heads; v.HD = head_dim;
  v.B = seqs; v.W = (max_len + kKv8Block - 1) / kKv8Block; v.pages = pages; v.max_len = max_len;
  const int G = heads / kv_heads;
  if ((int64_t)max_rows * G * G > UINT32_MAX) {
    delete kv;
    return fail(Q4HIP_EINVAL, "plans of %d rows with %d heads to a kv head: at most %u", max_rows, G, UINT32_MAX / (G * G));
  }
  v.g_magic = G == 1 ? 0 : (uint32_t)((((uint64_t)1 << 32) + G - 1) / G);
  v.unit_rows = std::max(1, 16 / G);
  v.wide_rows = std::max(1, 32 / G);
  v.row_tiles = (std::min(v.unit_rows, max_rows) * G + 15) / 16;
  v.items_aim = std::max(1, kItemsAim / (kv_heads * v.row_tiles));
  v.aim_inverse = std::nextafter(1.0 / v.items_aim, 2.0);
  const size_t blocks = (size_t)layers * pages * kv_heads, bytes = blocks * 2 * kKv8Block * head_dim;
  hipError_t e = hipStreamCreateWithFlags(&kv->stream, hipStreamNonBlocking);
  auto al = [&](auto** p, size_t n) { if (e == hipSuccess) e = hipMalloc((void**)p, n * sizeof(**p)); };
  al(&v.codes, bytes);
  al(&v.scales, blocks);
  al(&v.table, (size_t)seqs * v.W);
  al(&v.held, seqs);
  al(&v.stack, pages);
  al(&v.head, 1);
  al(&v.base, seqs);
  al(&v.lens, seqs);
  for (int** p : {&v.starts, &v.free_at, &v.take_at, &v.run_at, &v.item_at, &v.part_at, &v.tile_at}) al(p, (size_t)seqs + 1);
  al(&v.runs, max_rows);
  const size_t most_items = (size_t)kKv8MoreItems * v.items_aim;      // beyond one for each unit
  al(&v.items, max_rows + most_items);
  al(&v.tiles, tiles_bound(v, max_rows));
  // units in several parts: each has more pages than a part, so that the last one's part at most doubles them
  const size_t parts = 2 * most_items * kv_heads * v.row_tiles;
  al(&v.part_o, parts * 32 * head_dim);
  al(&v.part_ml, parts * 32);
  al(&v.arrived, parts);
  if (e == hipSuccess) e = hipHostMalloc((void**)&kv->pin, sizeof(Kv8Head), hipHostMallocDefault);
  if (e == hipSuccess) e = hipMemsetAsync(v.codes, 128, bytes, kv->stream);
  if (e == hipSuccess) e = hipMemsetAsync(v.scales, 0, blocks * sizeof(float2), kv->stream);
  if (e == hipSuccess) e = hipMemsetAsync(v.arrived, 0, parts * sizeof(int), kv->stream);
  if (e == hipSuccess) {
    const size_t n = std::max({(size_t)seqs * v.W, (size_t)pages, (size_t)seqs + 1});
    k_kv8_reset<<<(unsigned)((n + 255) / 256), 256, 0, kv->stream>>>(v);
    e = hipGetLastError();
  }
  if (e == hipSuccess) e = hipStreamSynchronize(kv->stream);
  if (e != hipSuccess) {
    const int rc = fail(Q4HIP_EHIP, "8-bit cache of %d pages: %s", pages, hipGetErrorString(e));
    q4hip_kv8_destroy(kv);
    return rc;
  }
  *out = kv;
  return Q4HIP_OK;
}

int q4hip_kv8_plan(q4hip_kv8* kv, const int* have, const int* add, int rows, int* starts, int* positions, int* slots,
                   int* tables, void* stream) {
  if (!kv || !have || !add) return fail(Q4HIP_EINVAL, "null argument");
  if (rows < 0 || rows > kv->max_rows) return fail(Q4HIP_EINVAL, "%d rows: a plan holds up to %d", rows, kv->max_rows);
  const Kv8View& v = kv->v;
  HIPCHK(hipSetDevice(kv->device));
  const struct { const void* p; size_t n; const char* what; } spans[] = {
      {have, (size_t)v.B, "have"}, {add, (size_t)v.B, "add"}, {starts, (size_t)v.B + 1, "starts"},
      {positions, (size_t)rows, "positions"}, {slots, (size_t)rows, "slots"}, {tables, (size_t)v.B * v.W, "tables"}};
  for (const auto& a : spans) {
    const int rc = check_ints(kv, a.p, a.n, a.what);
    if (rc) return rc;
  }
  hipStream_t s = stream ? (hipStream_t)stream : kv->stream;
  unsigned long long id;
  int rc = capture_of(s, &id);
  if (rc) return rc;
  kv8_launch_plan(kv, s, have, add, rows, starts, positions, slots, tables);
  HIPCHK(hipGetLastError());
  if (id) {
    kv->capture = id;
    kv->capture_rows = rows;
  } else {
    kv->rows = rows;
  }
  if (stream) return Q4HIP_OK;
  rc = read_head(kv, s);
  return rc ? rc : plan_error(kv, kv->pin->status);
}

int q4hip_kv8_status(q4hip_kv8* kv, void* stream, int* rows, int* free_pages) {
  if (!kv) return fail(Q4HIP_EINVAL, "null argument");
  HIPCHK(hipSetDevice(kv->device));
  const int rc = read_head(kv, stream ? (hipStream_t)stream : kv->stream);
  if (rc) return rc;
  if (rows) *rows = kv->pin->rows;
  if (free_pages) *free_pages = kv->pin->free_pages;
  return plan_error(kv, kv->pin->status);
}

int q4hip_kv8_append(q4hip_kv8* kv, int layer, const void* k, const void* v, int type, int64_t k_stride, int64_t v_stride,
                     void* stream) {
  if (!kv || !k || !v) return fail(Q4HIP_EINVAL, "null argument");
  int rc = check_layer(kv, layer, type);
  if (rc) return rc;
  HIPCHK(hipSetDevice(kv->device));
  hipStream_t s = stream ? (hipStream_t)stream : kv->stream;
  int rows;
  rc = rows_on(kv, s, &rows);
  if (rc || !rows) return rc;
  const Kv8View& w = kv->v;
  rc = check_rows(kv, k, rows, w.KVH * w.HD, k_stride, type, "k");
  if (!rc) rc = check_rows(kv, v, rows, w.KVH * w.HD, v_stride, type, "v");
  if (rc) return rc;
  kv8_launch_append(kv, s, layer, k, v, type, k_stride, v_stride, 0, w.KVH, rows);
  HIPCHK(hipGetLastError());
  if (!stream) HIPCHK(hipStreamSynchronize(s));
  return Q4HIP_OK;
}

int q4hip_kv8_read(q4hip_kv8* kv, int layer, const int* seq, const int* pos, int n, float* k, float* v, void* stream) {
  if (!kv || !seq || !pos || !k || !v) return fail(Q4HIP_EINVAL, "null argument");
  int rc = check_layer(kv, layer, Q4HIP_TYPE_F32);
  if (rc) return rc;
  if (n < 0) return fail(Q4HIP_EINVAL, "%d positions", n);
  if (!n) return Q4HIP_OK;
  HIPCHK(hipSetDevice(kv->device));
  const Kv8View& w = kv->v;
  const size_t row = (size_t)w.KVH * w.HD;
  rc = check_ints(kv, seq, n, "seq");
  if (!rc) rc = check_ints(kv, pos, n, "pos");
  if (!rc) rc = check_rows(kv, k, n, (int)row, row, Q4HIP_TYPE_F32, "k");
  if (!rc) rc = check_rows(kv, v, n, (int)row, row, Q4HIP_TYPE_F32, "v");
  if (rc) return rc;
  hipStream_t s = stream ? (hipStream_t)stream : kv->stream;
  kv8_launch_read(kv, s, layer, seq, pos, n, k, v);
  HIPCHK(hipGetLastError());
  if (!stream) HIPCHK(hipStreamSynchronize(s));
  return Q4HIP_OK;
}

int q4hip_kv8_attend(q4hip_kv8* kv, int layer, const void* q, void* out, int type, int64_t q_stride, int64_t out_stride,
                     float scale, void* stream) {
  if (!kv || !q || !out) return fail(Q4HIP_EINVAL, "null argument");
  int rc = check_layer(kv, layer, type);
  if (rc) return rc;
  if (!std::isfinite(scale) || scale < 0.0f) return fail(Q4HIP_EINVAL, "scale %g", (double)scale);
  HIPCHK(hipSetDevice(kv->device));
  hipStream_t s = stream ? (hipStream_t)stream : kv->stream;
  int rows;
  rc = rows_on(kv, s, &rows);
  if (rc || !rows) return rc;
  const Kv8View& w = kv->v;
  rc = check_rows(kv, q, rows, w.H * w.HD, q_stride, type, "q");
  if (!rc) rc = check_rows(kv, out, rows, w.H * w.HD, out_stride, type, "out");
  if (!rc) rc = check_apart(q, q_stride, out, out_stride, rows, w.H * w.HD, type);
  if (rc) return rc;
  kv8_launch_attend(kv, s, layer, q, out, type, q_stride, out_stride, scale, rows);
  HIPCHK(hipGetLastError());
  if (!stream) HIPCHK(hipStreamSynchronize(s));
  return Q4HIP_OK;
}

}  // extern "C"
