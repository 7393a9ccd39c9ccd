// rope.hip -- rotary positions of rows of heads (include/q4hip.h, q4hip_rope_*).
//
// A pair (x, y) of a row at position p becomes a (x cos t - y sin t, y cos t + x sin t), t = p f.  A far position times a
// frequency needs more than fp32 holds (at p = 10^6 its last bit is 0.06 rad), and a table of cosines for every position
// would be read beside the rows.  So a frequency is held as a part of a turn in 2^-64 (as a whole number): p f mod 2^64 is the
// angle without its full turns, exactly but for the frequency's own rounding (2^-65 p turns, whatever the frequency).  Its upper 32
// bits go into sine and cosine, cut off there: the nearest quarter of a turn by the upper two, the rest, within an eighth, as an fp32
// number by the power series.
//
// Bytes bound it: 8,192 rows of 40 heads of 128 (bf16), 168 MB read and written, take 36.0 us, 4.67 TB/s (a 1 GiB copy moves 5.18).
// A workgroup takes `each` rows: its threads form the cosines and sines of these in shared memory, once for all heads, while
// the first 16 bytes of each thread are on their way; then every thread takes 16 bytes (halves: and those rot / 2 columns later) at a time.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <new>

#include "rows.h"

struct q4hip_rope {
  int device = 0, head_dim = 0, rot = 0, pairs = 0;
  float amplitude = 1.0f;
  uint64_t* turns = nullptr;   // [rot / 2] of a turn in 2^-64
  hipStream_t stream = nullptr;
};

namespace q4 {
namespace {

constexpr int kRopeThreads = 256;
// Rows of a workgroup at most.
constexpr int kRopeRows = 4;

// Sine and cosine of a part of a turn in 2^-32.
__device__ inline float2 cos_sin(uint32_t turn) {
  const uint32_t quarter = (turn + 0x20000000u) >> 30;
  const float r = (float)(int32_t)(turn - (quarter << 30)) * 1.4629180792671596e-9f;       // 2 pi / 2^32: within pi / 4
  const float z = r * r;
  // power series: the first terms left out are under 2e-9 and 2e-10 within pi / 4
  float s = __builtin_fmaf(z, 2.7557319e-6f, -1.9841270e-4f);
  s = __builtin_fmaf(s, z, 8.3333333e-3f);
  s = __builtin_fmaf(s, z, -0.16666667f);
  s = __builtin_fmaf(s * z, r, r);
  float c = __builtin_fmaf(z, -2.7557319e-7f, 2.4801587e-5f);
  c = __builtin_fmaf(c, z, -1.3888889e-3f);
  c = __builtin_fmaf(c, z, 4.1666667e-2f);
  c = __builtin_fmaf(c, z, -0.5f);
  c = __builtin_fmaf(c, z, 1.0f);
  const float a = quarter & 1 ? s : c, b = quarter & 1 ? c : s;
  return {(quarter + 1) & 2 ? -a : a, quarter & 2 ? -b : b};
}

struct RopeShape {
  const uint64_t* turns;
  float amplitude;
  int heads, head_dim, rot;
  int chunks, turned;          // pieces of a head that a thread takes at once; those that are turned
  uint32_t by_chunks, by_heads;   // 2^32 / chunks and heads rounded up: i / chunks = i * by_chunks >> 32 while i * chunks < 2^32
};

__device__ inline uint32_t div_by(uint32_t i, uint32_t magic) { return magic ? __umulhi(i, magic) : i; }

// kPairs: x and y side by side, else rot / 2 columns apart.  V: columns that are loaded at once, 16 bytes or one.
template <class T, bool kPairs, int V>
__global__ __launch_bounds__(kRopeThreads) void k_rope_rows(RopeShape sh, const T* x, T* y, int64_t x_stride, int64_t y_stride,
                                                            const int* __restrict__ pos, int rows, const int* __restrict__ count,
                                                            int first, int each) {
  extern __shared__ float2 cs[];             // [each][rot / 2]
  constexpr int W = kPairs && V == 1 ? 2 : V;      // columns of a turned piece (halves: of each of its two)
  struct alignas(V > 1 ? 16 : sizeof(T)) Vec { T e[W]; };
  const int tid = threadIdx.x, half = sh.rot / 2;
  const int row0 = first + blockIdx.x * each;
  if (count) rows = min(rows, *count);
  const int n = min(each, rows - row0);
  if (n <= 0) return;
  const uint32_t all = (uint32_t)n * sh.heads * sh.chunks;
  // piece i: of row i / (heads * chunks), of head ..
  Vec a, b;
  const T* from;
  T* to;
  int pair, kind;                            // of cs; 0 turned, 1 as it is
  auto load = [&](uint32_t i) {
    const uint32_t hr = div_by(i, sh.by_chunks), r = div_by(hr, sh.by_heads);
    const int c = (int)(i - hr * sh.chunks), head = (int)(hr - r * sh.heads);
    const int at = c < sh.turned ? c * W : sh.rot + (c - sh.turned) * V;
    from = x + (int64_t)(row0 + (int)r) * x_stride + head * sh.head_dim + at;
    to = y + (int64_t)(row0 + (int)r) * y_stride + head * sh.head_dim + at;
    kind = c >= sh.turned;
    pair = (int)r * half + (kPairs ? at / 2 : at);
    if (kind && W != V) {
      a.e[0] = *from;
    } else {
      a = *(const Vec*)from;
      if (!kPairs && !kind) b = *(const Vec*)(from + half);
    }
  };
  if ((uint32_t)tid < all) load(tid);
  for (int i = tid; i < n * half; i += kRopeThreads) {
    const int r = i / half;
    const uint64_t turn = (uint64_t)(int64_t)pos[row0 + r] * sh.turns[i - r * half];
    float2 w = cos_sin((uint32_t)(turn >> 32));
    w.x *= sh.amplitude;
    w.y *= sh.amplitude;
    cs[i] = w;
  }
  __syncthreads();
  for (uint32_t i = tid; i < all;) {
    if (!kind) {
      if constexpr (kPairs) {
#pragma unroll
        for (int j = 0; j < W; j += 2) {
          const float2 w = cs[pair + j / 2];
          const float u = (float)a.e[j], v = (float)a.e[j + 1];
          a.e[j] = (T)__builtin_fmaf(u, w.x, -(v * w.y));
          a.e[j + 1] = (T)__builtin_fmaf(v, w.x, u * w.y);
        }
      } else {
#pragma unroll
        for (int j = 0; j < W; j++) {
          const float2 w = cs[pair + j];
          const float u = (float)a.e[j], v = (float)b.e[j];
          a.e[j] = (T)__builtin_fmaf(u, w.x, -(v * w.y));
          b.e[j] = (T)__builtin_fmaf(v, w.x, u * w.y);
        }
        *(Vec*)(to + half) = b;
      }
    }
    if (kind && W != V) *to = a.e[0];
    else *(Vec*)to = a;
    i += kRopeThreads;
    if (i < all) load(i);
  }
}

// 1 / (2 pi), 64 bits a word: as many as the largest double's part of a turn is formed of.
constexpr uint64_t kTurns[] = {
    0x28be60db9391054a, 0x7f09d5f47d4d3770, 0x36d8a5664f10e410, 0x7f9458eaf7aef158, 0x6dc91b8e909374b8, 0x01924bba82746487,
    0x3f877ac72c4a69cf, 0xba208d7d4baed121, 0x3a671c09ad17df90, 0x4e64758e60d4ce7d, 0x272117e2ef7e4a0e, 0xc7fe25fff7816603,
    0xfbcbc462d6829b47, 0xdb4d9fb3c9f2c26d, 0xd3d18fd9a797fa8b, 0x5d49eeb1faf97c5e, 0xcf41ce7de294a4ba, 0x9afed7ec47e35742};

// f radians without their full turns, in 2^-64 of a turn, rounded.  |f| = m 2^e, m of 53 bits: of 2^e / (2 pi) the full turns are left
// out, which m only multiplies, and 128 bits behind the point are taken, so that what is cut off is under 2^-75.
uint64_t turns_of(double f) {
  int e;
  const uint64_t m = (uint64_t)std::ldexp(std::frexp(std::fabs(f), &e), 53);
  e -= 53;
  auto bits = [](int at) -> uint64_t {       // 64 of 1 / (2 pi) from the one worth 2^-(at + 1)
    if (at < 0) return at > -64 ? kTurns[0] >> -at : 0;
    const int w = at / 64, s = at % 64;
    return s ? kTurns[w] << s | kTurns[w + 1] >> (64 - s) : kTurns[w];
  };
  const unsigned __int128 p = (unsigned __int128)bits(e + 64) * m + ((unsigned __int128)(bits(e) * m) << 64);
  const uint64_t t = (uint64_t)(p >> 64) + ((uint64_t)p >> 63);
  return f < 0.0 ? -t : t;
}

uint32_t magic_of(int d) { return d == 1 ? 0 : (uint32_t)((((uint64_t)1 << 32) + d - 1) / d); }

}  // namespace
}  // namespace q4

using namespace q4;

extern "C" {

int q4hip_rope_frequencies(int rot, double theta, int scaling, double factor, double original, double low, double high, double* freq,
                           float* amplitude) {
  if (!freq || !amplitude) return fail(Q4HIP_EINVAL, "null argument");
  if (rot < 2 || rot % 2 || rot > Q4HIP_ROPE_MAX_DIM) return fail(Q4HIP_EINVAL, "rot %d: an even number up to %d", rot, Q4HIP_ROPE_MAX_DIM);
  if (!(theta > 1.0) || !std::isfinite(theta)) return fail(Q4HIP_EINVAL, "theta %g", theta);
  if (scaling < Q4HIP_ROPE_PLAIN || scaling > Q4HIP_ROPE_YARN) return fail(Q4HIP_EINVAL, "scaling %d", scaling);
  if (scaling != Q4HIP_ROPE_PLAIN && (!(factor >= 1.0) || !std::isfinite(factor))) return fail(Q4HIP_EINVAL, "factor %g", factor);
  if (scaling >= Q4HIP_ROPE_BANDS && (!(original > 0.0) || !(low > 0.0) || !(high > low) || !std::isfinite(original) || !std::isfinite(high)))
    return fail(Q4HIP_EINVAL, "original %g, bounds %g and %g", original, low, high);
  constexpr double kTurn = 6.283185307179586477;
  *amplitude = 1.0f;
  double first = 0.0, last = 0.0;            // pairs between which YaRN's share falls
  if (scaling == Q4HIP_ROPE_YARN) {
    auto pair_of = [&](double turns) { return rot * std::log(original / (kTurn * turns)) / (2.0 * std::log(theta)); };
    first = std::max(std::floor(pair_of(high)), 0.0);
    last = std::min(std::ceil(pair_of(low)), rot - 1.0);
    *amplitude = factor > 1.0 ? (float)(0.1 * std::log(factor) + 1.0) : 1.0f;
  }
  for (int i = 0; i < rot / 2; i++) {
    const double f = std::pow(theta, -2.0 * i / rot);
    double share = 1.0;                      // of the frequency as it is, beside the stretched one
    if (scaling == Q4HIP_ROPE_LINEAR) share = 0.0;
    if (scaling == Q4HIP_ROPE_BANDS) share = std::min(std::max((original * f / kTurn - low) / (high - low), 0.0), 1.0);
    if (scaling == Q4HIP_ROPE_YARN) share = 1.0 - std::min(std::max((i - first) / std::max(last - first, 0.001), 0.0), 1.0);
    freq[i] = scaling == Q4HIP_ROPE_PLAIN ? f : f / factor * (1.0 - share) + f * share;
  }
  return Q4HIP_OK;
}

void q4hip_rope_destroy(q4hip_rope* r) {
  if (!r) return;
  (void)hipSetDevice(r->device);
  if (r->stream) (void)hipStreamSynchronize(r->stream);
  if (r->turns) (void)hipFree(r->turns);
  if (r->stream) (void)hipStreamDestroy(r->stream);
  delete r;
}

int q4hip_rope_create(q4hip_rope** out, int head_dim, int rot, int order, const double* freq, float amplitude, int device) {
  if (!out || !freq) return fail(Q4HIP_EINVAL, "null argument");
  *out = nullptr;
  if (head_dim < 2 || head_dim > Q4HIP_ROPE_MAX_DIM) return fail(Q4HIP_EINVAL, "head_dim %d: 2 to %d", head_dim, Q4HIP_ROPE_MAX_DIM);
  if (rot < 2 || rot % 2 || rot > head_dim) return fail(Q4HIP_EINVAL, "rot %d: an even number up to head_dim", rot);
  if (order != Q4HIP_ROPE_HALVES && order != Q4HIP_ROPE_PAIRS) return fail(Q4HIP_EINVAL, "order %d", order);
  if (!std::isfinite(amplitude)) return fail(Q4HIP_EINVAL, "amplitude %g", (double)amplitude);
  for (int i = 0; i < rot / 2; i++)
    if (!std::isfinite(freq[i])) return fail(Q4HIP_EINVAL, "frequency %d: %g", i, freq[i]);
  int ndev = 0;
  HIPCHK(hipGetDeviceCount(&ndev));
  if (device < 0 || device >= ndev) return fail(Q4HIP_EINVAL, "device %d of %d", device, ndev);
  HIPCHK(hipSetDevice(device));
  q4hip_rope* r = new (std::nothrow) q4hip_rope();
  if (!r) return fail(Q4HIP_EHIP, "out of host memory");
  r->device = device;
  r->head_dim = head_dim;
  r->rot = rot;
  r->pairs = order == Q4HIP_ROPE_PAIRS;
  r->amplitude = amplitude;
  uint64_t turns[Q4HIP_ROPE_MAX_DIM / 2];
  for (int i = 0; i < rot / 2; i++) turns[i] = turns_of(freq[i]);
  hipError_t e = hipStreamCreateWithFlags(&r->stream, hipStreamNonBlocking);
  if (e == hipSuccess) e = hipMalloc(&r->turns, (size_t)rot / 2 * sizeof(uint64_t));
  if (e == hipSuccess) e = hipMemcpy(r->turns, turns, (size_t)rot / 2 * sizeof(uint64_t), hipMemcpyHostToDevice);
  if (e != hipSuccess) {
    const int rc = fail(Q4HIP_EHIP, "rotary positions: %s", hipGetErrorString(e));
    q4hip_rope_destroy(r);
    return rc;
  }
  *out = r;
  return Q4HIP_OK;
}

int q4hip_rope_run(q4hip_rope* r, const void* x, void* y, int heads, int type, int64_t x_stride, int64_t y_stride, const int* pos,
                   int rows, const int* count, void* stream) {
  if (!r || !x || !y || !pos) return fail(Q4HIP_EINVAL, "null argument");
  int rc = check_type(type);
  if (rc) return rc;
  // so that the quotients of k_rope_rows hold: each * heads * chunks^2 and each * heads^2 stay below 2^32
  if (heads <= 0 || heads > 16384 || (int64_t)heads * r->head_dim > 1 << 20)
    return fail(Q4HIP_EINVAL, "%d heads of %d columns: up to 16384, and 2^20 columns", heads, r->head_dim);
  if (rows < 0) return fail(Q4HIP_EINVAL, "%d rows", rows);
  if (!rows) return Q4HIP_OK;
  HIPCHK(hipSetDevice(r->device));
  const int64_t width = (int64_t)heads * r->head_dim;
  rc = check_rows(r->device, x, rows, width, x_stride, type, "x");
  const bool in_place = x == y && x_stride == y_stride;
  if (!rc && !in_place) rc = check_rows(r->device, y, rows, width, y_stride, type, "y");
  if (!rc && !in_place) rc = check_apart(x, x_stride, y, y_stride, rows, width, type, "x and y");
  if (!rc) rc = check_ints(r->device, pos, rows, "pos");
  if (!rc) rc = check_ints(r->device, count, 1, "count");
  if (rc) return rc;
  const size_t span = ((size_t)(rows - 1) * y_stride + width) * elem_size(type);
  if (overlap(y, span, pos, (size_t)rows * 4) || (count && overlap(y, span, count, 4)))
    return fail(Q4HIP_EINVAL, "y overlaps pos or count");
  hipStream_t s = stream ? (hipStream_t)stream : r->stream;
  const int vec = 16 / elem_size(type), half = r->rot / 2;
  const bool wide = aligned16(x, x_stride, type) && aligned16(y, y_stride, type) && r->head_dim % vec == 0 &&
                    (r->pairs ? r->rot : half) % vec == 0;
  const int V = wide ? vec : 1, W = r->pairs ? std::max(V, 2) : V;
  RopeShape sh;
  sh.turns = r->turns;
  sh.amplitude = r->amplitude;
  sh.heads = heads;
  sh.head_dim = r->head_dim;
  sh.rot = r->rot;
  sh.turned = (r->pairs ? r->rot : half) / W;
  sh.chunks = sh.turned + (in_place ? 0 : (r->head_dim - r->rot) / V);
  sh.by_chunks = magic_of(sh.chunks);
  sh.by_heads = magic_of(heads);
  const int each = std::max(1, std::min(kRopeRows, rows / 1024));
  const int64_t most = (int64_t)kMostThreads / kRopeThreads * each;      // rows of a launch
  by_type(type, [&](auto zero) {
    using T = decltype(zero);
    constexpr int kVec = 16 / sizeof(T);
    auto* fn = r->pairs ? (wide ? k_rope_rows<T, true, kVec> : k_rope_rows<T, true, 1>)
                        : (wide ? k_rope_rows<T, false, kVec> : k_rope_rows<T, false, 1>);
    for (int64_t first = 0; first < rows; first += most) {
      const unsigned grid = (unsigned)((std::min(most, rows - first) + each - 1) / each);
      fn<<<grid, kRopeThreads, (size_t)each * half * sizeof(float2), s>>>(sh, (const T*)x, (T*)y, x_stride, y_stride, pos, rows, count,
                                                                         (int)first, each);
    }
  });
  HIPCHK(hipGetLastError());
  if (!stream) HIPCHK(hipStreamSynchronize(s));
  return Q4HIP_OK;
}

}  // extern "C"
