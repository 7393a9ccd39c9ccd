// kv8.hip -- the paged 8-bit K/V cache: plan, append, read and attention (include/q4hip.h, q4hip_kv8_*).
#include "kv8.h"

#include <algorithm>
#include <cmath>
#include <cstdlib>
#include <new>

#include "host.h"
#include "kv8_attend.h"
#include "kv8_fork.h"
#include "kv8_joint.h"
#include "kv8_plan.h"
#include "rows.h"

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

// Workgroups of attention with joints: two for each CU, as many as its registers hold.
constexpr int kJointWorkgroups = 512;
// Workgroups that add a step's joints up, at most; without any they cost 2 us.
constexpr int64_t kGatherWorkgroups = 2048;
// Workgroups of a fork's copies at most.
constexpr int64_t kForkGrid = 4096;

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
__global__ __launch_bounds__(256) void k_kv8_reset(Kv8View v, Kv8ForkView f) {
  const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
  if (i < (size_t)v.B * v.W) v.table[i] = -1;
  if (i < (size_t)v.pages) {
    v.stack[i] = v.pages - 1 - (int)i;
    if (f.fork) {
      v.count()[i] = 0;
      v.first()[i] = INT32_MAX;
    }
  }
  if (i <= (size_t)v.B) {
    v.starts[i] = 0;
    if (i < (size_t)v.B) { v.held[i] = 0; v.base[i] = 0; v.lens[i] = 0; }
  }
  if (i == 0) {
    *v.head = Kv8Head{KV8_OK, 0, v.pages, 0, 0, 0, 1, 0, 0, 0, 0};
    if (f.fork) *f.fork = Kv8Fork{};
  }
}

// At most so many tiles have `rows` rows: of full ones, and of a last one of each sequence.
size_t tiles_bound(const Kv8View& v, int rows) {
  return (size_t)((int64_t)rows * (v.H / v.KVH) / kKv8TileRows + std::min(v.B, rows / (v.unit_rows + 1)) + 1);
}

int check_layer(const q4hip_kv8* kv, int layer, int type) {
  if (layer < 0 || layer >= kv->v.layers) return fail(Q4HIP_EINVAL, "layer %d of %d", layer, kv->v.layers);
  return check_type(type);
}

int plan_error(const q4hip_kv8* kv, int status) {
  switch (status) {
    case KV8_OK: return Q4HIP_OK;
    case KV8_BAD_LENGTH: return fail(Q4HIP_EINVAL, "plan or fork: a negative length");
    case KV8_TOO_LONG: return fail(Q4HIP_ECONTEXT, "plan: a sequence longer than %d positions", kv->v.max_len);
    case KV8_STALE:
      return fail(Q4HIP_ESTATE, "append or attend replayed on a plan of more rows than they were captured for");
    case KV8_ROWS: return fail(Q4HIP_EINVAL, "plan: more rows than it was called for");
    case KV8_SHARED:
      return fail(Q4HIP_EINVAL, "plan: rows into a page that another sequence holds, too: cut the sequence back by a fork first");
    case KV8_FORK_SOURCE: return fail(Q4HIP_EINVAL, "fork: a sequence that there is not, or more positions than it holds");
    case KV8_FORK_PAGES: return fail(Q4HIP_ECONTEXT, "fork: more than the pool's %d pages", kv->v.pages);
    case KV8_ENTRIES:
      return fail(Q4HIP_ECONTEXT, "plan or fork: sequences of more than %d pages in all while some share any", kKv8Entries);
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
int rows_on(q4hip_kv8* kv, hipStream_t s, int* rows) {
  unsigned long long id;
  const int rc = capture_of(s, &id);
  kv->capturing = !rc && id;
  *rows = id && id == kv->capture ? kv->capture_rows : kv->rows;
  return rc;
}

// Whether a step's units may be joined, if the plan finds that it is worth it (no length is known here): then there is a launch more, which
// costs 2.5 us where it is not.  Steps of few rows, which are mostly short, are not.  One by one and together, us: 4 answers of 14 heads
// (2 x 64) behind 300 positions 6.2 and 12.0, behind 32,000 12.9 and 13.9; 12 of 20 heads (20 x 64) behind 300 6.4 and 10.5, behind 2,000
// 11.5 and 11.4, but behind 16,000 50 and 16; 4 of 32 heads (8 x 128) behind 300 7.2 and 12.0, behind 16,000 20 and 15.
bool joined(const q4hip_kv8* kv, int rows) {
  const int G = kv->v.H / kv->v.KVH;
  const bool shared = kv->forked && (!kv->unshared || kv->capturing || kv->fork_captured);
  return shared && kv->j.most && rows > 1 && ((int64_t)rows * G > 32 || (int64_t)rows * kv->v.H >= 256 || !kv->j.saves);
}

int read_head(q4hip_kv8* kv, hipStream_t s) {
  HIPCHK(hipMemcpyAsync(kv->pin, kv->v.head, sizeof(Kv8Head), hipMemcpyDeviceToHost, s));
  HIPCHK(hipStreamSynchronize(s));
  if (!kv->pin->shared) kv->unshared = true;
  return Q4HIP_OK;
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
  if (!joined(kv, rows)) return;
  if (shared) k_kv8_joints<true><<<1, kJointThreads, 0, s>>>(v, kv->j, nullptr);
  else k_kv8_joints<false><<<1, kJointThreads, 0, s>>>(v, kv->j, kv->joint_scratch);
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
  const bool joint = joined(kv, rows);
  const int64_t work = items * w.KVH * w.row_tiles + (few ? 0 : (int64_t)tiles_bound(w, rows) * w.KVH);
  const unsigned grid = (unsigned)std::min<int64_t>(work, kMostWorkgroups);
  by_type(type, [&](auto zero) {
    using T = decltype(zero);
    if (joint) {
      auto* fn = w.HD == 64 ? k_kv8_attend_joint<64, T> : k_kv8_attend_joint<128, T>;
      fn<<<(unsigned)std::min<int64_t>(work + (int64_t)std::min(units, kv->j.most) * w.KVH, kv->j.workgroups), 256, 0, s>>>(
          w, kv->j, layer, (const T*)q, (T*)out, q_stride, out_stride, log2_scale, rows, wide);
      // rows of joints, or less
      const int64_t most = std::min<int64_t>(32 * (int64_t)kv->j.most, (int64_t)rows * (w.H / w.KVH) + 31 * (rows / 2));
      auto* sum = w.HD == 64 ? k_kv8_gather<64, T> : k_kv8_gather<128, T>;
      sum<<<(unsigned)std::min<int64_t>(most * w.KVH, kGatherWorkgroups), 256, 0, s>>>(w, kv->j, (T*)out, out_stride, rows, wide);
      return;
    }
    auto* fn = w.HD == 64 ? (few ? k_kv8_attend<64, T, 0> : k_kv8_attend<64, T, 2>)
                          : (few ? k_kv8_attend<128, T, 0> : k_kv8_attend<128, T, 2>);
    fn<<<grid, 256, 0, s>>>(w, layer, (const T*)q, (T*)out, q_stride, out_stride, log2_scale, rows, wide);
  });
}

namespace {

void launch_fork(q4hip_kv8* kv, hipStream_t s, const int* from, const int* keep, int* tables) {
  const Kv8View& v = kv->v;
  kv->forked = true;
  kv->unshared = false;
  const unsigned chunks = (unsigned)((v.pages + kKv8Chunk - 1) / kKv8Chunk), all = (unsigned)kForkGrid;
  const size_t entries = (size_t)v.B * v.W;
  if (v.B <= kPlanShared && v.pages <= kForkPages && entries + kForkEach * v.B <= (size_t)kForkEntries) {
    k_kv8_fork_small<<<1, kPlanThreads, 0, s>>>(v, kv->f, from, keep, tables);
  } else {
    k_kv8_fork_count<<<dim3((unsigned)std::min((v.W + kForkThreads - 1) / kForkThreads, 64), (unsigned)std::min(v.B, 65535)), kForkThreads,
                       0, s>>>(v, kv->f, from, keep);
    k_kv8_fork_weigh<<<chunks + 1, kKv8Chunk, 0, s>>>(v, kv->f, keep);
    k_kv8_fork_commit<<<std::max(chunks, (unsigned)std::min<size_t>((entries + kKv8Chunk - 1) / kKv8Chunk, 512)), kKv8Chunk, 0, s>>>(
        v, kv->f, keep, tables);
  }
  k_kv8_fork_copy<<<(unsigned)std::min<int64_t>((int64_t)v.B * v.layers * v.KVH, all), kForkThreads, 0, s>>>(v, kv->f, keep, tables);
}

}  // namespace

void kv8_launch_read(q4hip_kv8* kv, hipStream_t s, int layer, const int* seq, const int* pos, int n, float* k, float* v) {
  const Kv8View& w = kv->v;
  const int per = 1024 / w.HD;                 // rows of a workgroup
  const dim3 grid((unsigned)std::min((n + per - 1) / per, 16384), (unsigned)w.KVH);
  if (w.HD == 64) k_kv8_read<64><<<grid, 256, 0, s>>>(w, layer, seq, pos, n, k, v);
  else k_kv8_read<128><<<grid, 256, 0, s>>>(w, layer, seq, pos, n, k, v);
}

int kv8_create(q4hip_kv8** out, int layers, int heads, int kv_heads, int head_dim, int seqs, int max_len, int pages, int max_rows,
               int device, bool forks) {
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
  al(&v.stack, (size_t)(forks ? 4 : 1) * pages);
  if (forks) {
    al(&kv->f.next, (size_t)seqs * v.W);
    al(&kv->f.copies, seqs);
    al(&kv->f.chunk, (pages + kKv8Chunk - 1) / kKv8Chunk);
    al(&kv->f.fork, 1);
  }
  al(&v.head, 1);
  al(&v.base, seqs);
  al(&v.lens, seqs);
  for (int** p : {&v.starts, &v.free_at, &v.take_at, &v.run_at, &v.item_at, &v.part_at, &v.tile_at}) al(p, (size_t)seqs + 1);
  al(&v.runs, max_rows);
  const size_t most_items = (size_t)kKv8MoreItems * v.items_aim;      // beyond one for each unit
  al(&v.items, max_rows + most_items);
  al(&v.tiles, tiles_bound(v, max_rows));
  if (forks && seqs > 1 && G <= 16) {
    // the rows of groups of two and more, in whole joints
    kv->j.most = (int)std::min<int64_t>(((int64_t)seqs * v.unit_rows * G + 31) / 32 + seqs / 2, kKv8Joints);
    al(&kv->j.items, max_rows + most_items + kv->j.most);
    al(&kv->j.joints, kv->j.most);
    al(&kv->j.rows, (size_t)32 * kv->j.most);
    kv->j.workgroups = kJointWorkgroups;
    const char* saves = getenv("Q4HIP_KV8_JOINT_SAVES");
    kv->j.saves = saves ? atoi(saves) : kKv8JointSaves;
    al(&kv->j.queue, 1);
    if (e == hipSuccess) e = hipMemsetAsync(kv->j.queue, 0, sizeof(int), kv->stream);
    if (seqs > kPlanShared) al(&kv->joint_scratch, (size_t)kJointArrays * seqs);
  }
  // units in several parts: each has more pages than a part, so that the last one's part at most doubles them
  const size_t parts = (2 * most_items + 2 * (size_t)kv->j.most) * kv_heads * v.row_tiles;
  al(&v.part_o, parts * 32 * head_dim);
  al(&v.part_ml, parts * 32);
  al(&v.arrived, parts);
  if (e == hipSuccess) e = hipHostMalloc((void**)&kv->pin, sizeof(Kv8Head), hipHostMallocDefault);
  if (e == hipSuccess) e = hipMemsetAsync(v.codes, 128, bytes, kv->stream);
  if (e == hipSuccess) e = hipMemsetAsync(v.scales, 0, blocks * sizeof(float2), kv->stream);
  if (e == hipSuccess) e = hipMemsetAsync(v.arrived, 0, parts * sizeof(int), kv->stream);
  if (e == hipSuccess) {
    const size_t n = std::max({(size_t)seqs * v.W, (size_t)pages, (size_t)seqs + 1});
    k_kv8_reset<<<(unsigned)((n + 255) / 256), 256, 0, kv->stream>>>(v, kv->f);
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

}  // namespace q4

using namespace q4;

extern "C" {

void q4hip_kv8_destroy(q4hip_kv8* kv) {
  if (!kv) return;
  (void)hipSetDevice(kv->device);
  if (kv->stream) (void)hipStreamSynchronize(kv->stream);
  Kv8View& v = kv->v;
  void* bufs[] = {v.codes, v.scales, v.table, v.held, v.stack, v.head, v.base, v.lens, v.starts, v.free_at, v.take_at,
                  kv->f.next, kv->f.copies, kv->f.chunk, kv->f.fork, v.run_at, v.item_at, v.part_at, v.tile_at, v.runs, v.items, v.tiles, v.part_o, v.part_ml, v.arrived,
                  kv->j.items, kv->j.joints, kv->j.rows, kv->j.queue, kv->joint_scratch};
  for (void* p : bufs) if (p) (void)hipFree(p);
  if (kv->pin) (void)hipHostFree(kv->pin);
  if (kv->stream) (void)hipStreamDestroy(kv->stream);
  delete kv;
}

int q4hip_kv8_create(q4hip_kv8** out, int layers, int heads, int kv_heads, int head_dim, int seqs, int max_len, int pages,
                     int max_rows, int device) {
  return kv8_create(out, layers, heads, kv_heads, head_dim, seqs, max_len, pages, max_rows, device, true);
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
    const int rc = check_ints(kv->device, a.p, a.n, a.what);
    if (rc) return rc;
  }
  hipStream_t s = stream ? (hipStream_t)stream : kv->stream;
  unsigned long long id;
  int rc = capture_of(s, &id);
  if (rc) return rc;
  kv->capturing = id != 0;
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

int q4hip_kv8_fork(q4hip_kv8* kv, const int* from, const int* keep, int* tables, void* stream) {
  if (!kv || !from || !keep) return fail(Q4HIP_EINVAL, "null argument");
  const Kv8View& v = kv->v;
  HIPCHK(hipSetDevice(kv->device));
  int rc = check_ints(kv->device, from, v.B, "from");
  if (!rc) rc = check_ints(kv->device, keep, v.B, "keep");
  if (!rc) rc = check_ints(kv->device, tables, (size_t)v.B * v.W, "tables");
  const size_t n = (size_t)v.B * 4;
  if (!rc && tables && (overlap(tables, n * v.W, from, n) || overlap(tables, n * v.W, keep, n)))
    rc = fail(Q4HIP_EINVAL, "tables overlaps from or keep");
  if (rc) return rc;
  hipStream_t s = stream ? (hipStream_t)stream : kv->stream;
  unsigned long long id;
  rc = capture_of(s, &id);
  if (rc) return rc;
  launch_fork(kv, s, from, keep, tables);
  HIPCHK(hipGetLastError());
  // the step is over: nothing is left to append or attend
  if (id) {
    kv->fork_captured = true;
    kv->capture = id;
    kv->capture_rows = 0;
  } else {
    kv->rows = 0;
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

int q4hip_kv8_shared(q4hip_kv8* kv, void* stream, int* shared, int* joints) {
  if (!kv) return fail(Q4HIP_EINVAL, "null argument");
  HIPCHK(hipSetDevice(kv->device));
  const int rc = read_head(kv, stream ? (hipStream_t)stream : kv->stream);
  if (rc) return rc;
  if (shared) *shared = kv->pin->shared != 0;
  if (joints) *joints = kv->pin->joints;
  return Q4HIP_OK;
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
  rc = check_rows(kv->device, k, rows, w.KVH * w.HD, k_stride, type, "k");
  if (!rc) rc = check_rows(kv->device, v, rows, w.KVH * w.HD, v_stride, type, "v");
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
  rc = check_ints(kv->device, seq, n, "seq");
  if (!rc) rc = check_ints(kv->device, pos, n, "pos");
  if (!rc) rc = check_rows(kv->device, k, n, (int)row, row, Q4HIP_TYPE_F32, "k");
  if (!rc) rc = check_rows(kv->device, v, n, (int)row, row, Q4HIP_TYPE_F32, "v");
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
  rc = check_rows(kv->device, q, rows, w.H * w.HD, q_stride, type, "q");
  if (!rc) rc = check_rows(kv->device, out, rows, w.H * w.HD, out_stride, type, "out");
  if (!rc) rc = check_apart(q, q_stride, out, out_stride, rows, w.H * w.HD, type, "q and out");
  if (rc) return rc;
  kv8_launch_attend(kv, s, layer, q, out, type, q_stride, out_stride, scale, rows);
  HIPCHK(hipGetLastError());
  if (!stream) HIPCHK(hipStreamSynchronize(s));
  return Q4HIP_OK;
}

}  // extern "C"
