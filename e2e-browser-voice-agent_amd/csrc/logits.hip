// logits.hip -- penalties, biases and masks on rows of logits, and the best token of each (include/q4hip.h, q4hip_logits_*).
//
// A workgroup takes a piece of a row: a block of threads with N tokens of each in registers.  How often the row's history
// has each of these is counted in shared memory (whole numbers: any order of the additions gives the same), then the biases' last
// entries are found there the same way, over the counts, and a thread looks up its own tokens.  So a row's logits are read and written
// once, no counts of the whole vocabulary lie in memory, and one launch does all of it; the history is read once for every piece, from the
// L2.  The best token: the largest of (value, lowest token first) as whole numbers of 64 bits, joined over the pieces by an
// atomic maximum, which the row's last piece reads and clears.
//
// What bounds it.  One row of 151,936 fp32 logits: the launch and a chain of loads, 6.0 us.  256 rows (fp32) with 2,000 to 16,000 tokens
// of history: bytes, 311 MB in 82.0 us, 3.8 TB/s, beside 19 passes over each history.  64 rows (bf16) with up to 4,000 tokens and 40
// biases: 25.3 us, of which 14 are left without lists: 1,216 workgroups, where 1,024 fit, with up to four barriers each.
// Not kept: looking nothing up in pieces that no entry falls into (256 rows 97 us: nearly all have one).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <new>

#include "rows.h"

struct q4hip_logits {
  int device = 0, vocab = 0, max_rows = 0;
  unsigned long long* best = nullptr;   // [max_rows] 0 between calls
  int* arrived = nullptr;               // [max_rows] pieces that are done, 0 between calls
  hipStream_t stream = nullptr;
};

namespace q4 {
namespace {

// Tokens of a piece: large ones where the rows fill the GPU, as every piece reads the whole history.  (64 rows in small pieces 45 us, in
// 256 * 16 tokens 27.5, in 256 * 32 27.8; 256 rows in 256 * 16 106, in 256 * 32 112.)
constexpr int kSmallThreads = 256, kSmallEach = 8, kLargeThreads = 512, kLargeEach = 16;
constexpr int kLargeFrom = 512;         // large pieces from which on they are taken

// Entries of a list at most: counts and the biases' numbers share a word.
constexpr int kMostEntries = 1 << 30;

// x as a whole number in the order of the values, -0 as +0.
__device__ inline uint32_t order_of(float x) {
  const uint32_t u = __float_as_uint(x + 0.0f);
  return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}

struct LogitsCall {
  const q4hip_logits_row* rows;
  const int* history;
  const q4hip_logits_bias* biases;
  const uint32_t* mask;
  int64_t history_n, biases_n, mask_rows;
  int vocab, pieces, words;
  int64_t x_stride, y_stride;
  int* best;
  unsigned long long* top;
  int* arrived;
};

// V: neighbouring tokens that are loaded at once, 16 bytes or one.
template <class T, int V, int kThreads, int N>
__global__ __launch_bounds__(kThreads) void k_logits(LogitsCall c, const T* x, T* y) {
  constexpr int kPiece = kThreads * N, kSteps = N / V;
  __shared__ __attribute__((aligned(16))) int table[kPiece];
  __shared__ unsigned long long tops[kThreads / 64];
  struct alignas(V > 1 ? 16 : sizeof(T)) Vec { T e[V]; };
  const int tid = threadIdx.x, piece = blockIdx.x % c.pieces, row = blockIdx.x / c.pieces;
  const int first = piece * kPiece, n = min(kPiece, c.vocab - first);
  const q4hip_logits_row p = c.rows[row];
  const T* const from = x + (int64_t)row * c.x_stride + first;
  T* const to = y + (int64_t)row * c.y_stride + first;
  // thread's tokens: V from (step * kThreads + tid) * V on
  float value[N];
#pragma unroll
  for (int s = 0; s < kSteps; s++) {
    const int at = (s * kThreads + tid) * V;
    if (at + V <= n) {
      const Vec w = *(const Vec*)(from + at);
#pragma unroll
      for (int k = 0; k < V; k++) value[s * V + k] = (float)w.e[k];
    } else {
#pragma unroll
      for (int k = 0; k < V; k++) value[s * V + k] = at + k < n ? (float)from[at + k] : -__builtin_inff();
    }
  }
  // entries [begin, end) of a list of `all`, none where they are not in order
  auto bounds = [](int64_t begin, int64_t end, int64_t all, int64_t& lo, int64_t& hi) {
    lo = begin < 0 ? 0 : begin;
    hi = end > all ? all : end;
  };
  // f(entry, place in the piece) of a list's entries that are of the piece; four loads on their way at once
  auto scan = [&](int64_t lo, int64_t hi, auto token, auto f) {
    for (int64_t i = lo + tid; i < hi; i += 4 * kThreads) {
      uint32_t at[4];
#pragma unroll
      for (int u = 0; u < 4; u++) at[u] = (uint32_t)token(min(i + u * kThreads, hi - 1)) - (uint32_t)first;
#pragma unroll
      for (int u = 0; u < 4; u++)
        if (at[u] < (uint32_t)n && i + u * kThreads < hi) f(i + u * kThreads, at[u]);
    }
    __syncthreads();
  };
  // of the lists behind, what is waited for: the mask's words, and the first biases of each thread, on their way at once with the history
  const uint32_t* const mask = p.mask >= 0 && p.mask < c.mask_rows ? c.mask + (int64_t)p.mask * c.words : nullptr;
  uint32_t bits[kSteps];
#pragma unroll
  for (int s = 0; s < kSteps; s++) {
    const int at = (s * kThreads + tid) * V;
    bits[s] = mask && at < n ? mask[(first + at) >> 5] : ~0u;
  }
  auto entry = [&](int s, int k) { return table[(s * kThreads + tid) * V + k]; };
  int64_t lo, hi, bias_lo, bias_hi;
  bounds(p.history_begin, p.history_end, c.history_n, lo, hi);
  bounds(p.bias_begin, p.bias_end, c.biases_n, bias_lo, bias_hi);
  q4hip_logits_bias bias{-1, 0.0f};            // the thread's first
  if (bias_lo + tid < bias_hi) bias = c.biases[bias_lo + tid];
  if (lo < hi || bias_lo < bias_hi) {
    for (int i = tid; i < kPiece / 4; i += kThreads) ((int4*)table)[i] = int4{0, 0, 0, 0};
    __syncthreads();
  }
  if (lo < hi) {
    scan(lo, hi, [&](int64_t i) { return c.history[i]; }, [&](int64_t, uint32_t at) { atomicAdd(&table[at], 1); });
#pragma unroll
    for (int s = 0; s < kSteps; s++)
#pragma unroll
      for (int k = 0; k < V; k++) {
        const int times = entry(s, k);
        float& v = value[s * V + k];
        if (times) {
          const float t = p.frequency * (float)times;
          v = v > 0.0f ? v / p.repetition : v * p.repetition;
          v = v - (t + p.presence);
        }
      }
    if (bias_lo < bias_hi) __syncthreads();
  }
  if (bias_lo < bias_hi) {
    // over the counts: any bias' number is larger than these
    const uint32_t at = (uint32_t)bias.token - (uint32_t)first;
    if (at < (uint32_t)n) atomicMax(&table[at], kMostEntries + tid);
    scan(bias_lo + kThreads, bias_hi, [&](int64_t i) { return c.biases[i].token; },
         [&](int64_t i, uint32_t at) { atomicMax(&table[at], kMostEntries + (int)(i - bias_lo)); });
#pragma unroll
    for (int s = 0; s < kSteps; s++)
#pragma unroll
      for (int k = 0; k < V; k++) {
        const int e = entry(s, k);
        if (e >= kMostEntries) value[s * V + k] += c.biases[bias_lo + e - kMostEntries].value;
      }
  }
  float most = -__builtin_inff();            // of the thread's values, the first of the largest, and its place
  int where = 0;
#pragma unroll
  for (int s = 0; s < kSteps; s++) {
    const int at = (s * kThreads + tid) * V;
    const uint32_t own = bits[s] >> ((first + at) & 31);
#pragma unroll
    for (int k = 0; k < V; k++) {
      float& v = value[s * V + k];
      v = own >> k & 1 ? v : -__builtin_inff();
      if (v > most) { most = v; where = at + k; }
    }
  }
  auto store = [&] {
#pragma unroll
    for (int s = 0; s < kSteps; s++) {
      const int at = (s * kThreads + tid) * V;
      Vec w;
#pragma unroll
      for (int k = 0; k < V; k++) w.e[k] = (T)value[s * V + k];
      if (at + V <= n) {
        *(Vec*)(to + at) = w;
      } else {
#pragma unroll
        for (int k = 0; k < V; k++)
          if (at + k < n) to[at + k] = w.e[k];
      }
    }
  };
  if (!c.best) {
    store();
    return;
  }
  unsigned long long top = most > -__builtin_inff() ? (unsigned long long)order_of(most) << 32 | (uint32_t)~(first + where) : 0;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const unsigned long long other = __shfl_xor(top, d);
    top = other > top ? other : top;
  }
  if ((tid & 63) == 0) tops[tid >> 6] = top;
  __syncthreads();
  unsigned long long before = 0;
  if (tid == 0) {
#pragma unroll
    for (int i = 1; i < kThreads / 64; i++) top = tops[i] > top ? tops[i] : top;
    if (c.pieces > 1) before = __hip_atomic_fetch_max(c.top + row, top, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  store();                                   // the maximum is on its way meanwhile
  if (tid) return;
  if (c.pieces > 1) {
    // the maximum is in memory before the arrival: its value before has come back
    int one = 1;
    asm volatile("" : "+v"(one) : "v"(before));
    if (__hip_atomic_fetch_add(c.arrived + row, one, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) != c.pieces - 1) return;
    top = __hip_atomic_exchange(c.top + row, 0ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __hip_atomic_store(c.arrived + row, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  c.best[row] = top ? (int)~(uint32_t)top : -1;
}

}  // namespace
}  // namespace q4

using namespace q4;

extern "C" {

void q4hip_logits_destroy(q4hip_logits* lg) {
  if (!lg) return;
  (void)hipSetDevice(lg->device);
  if (lg->stream) (void)hipStreamSynchronize(lg->stream);
  if (lg->best) (void)hipFree(lg->best);
  if (lg->arrived) (void)hipFree(lg->arrived);
  if (lg->stream) (void)hipStreamDestroy(lg->stream);
  delete lg;
}

int q4hip_logits_create(q4hip_logits** out, int vocab, int max_rows, int device) {
  if (!out) return fail(Q4HIP_EINVAL, "null argument");
  *out = nullptr;
  if (vocab <= 0 || vocab > 1 << 30) return fail(Q4HIP_EINVAL, "a vocabulary of %d", vocab);
  if (max_rows <= 0 || max_rows > 1 << 20) return fail(Q4HIP_EINVAL, "%d rows: up to 2^20", max_rows);
  const int64_t pieces = ((int64_t)vocab + kLargeThreads * kLargeEach - 1) / (kLargeThreads * kLargeEach);
  if (pieces * max_rows > INT32_MAX / 8) return fail(Q4HIP_EINVAL, "%d rows of a vocabulary of %d", max_rows, vocab);
  int ndev = 0;
  HIPCHK(hipGetDeviceCount(&ndev));
  if (device < 0 || device >= ndev) return fail(Q4HIP_EINVAL, "device %d of %d", device, ndev);
  HIPCHK(hipSetDevice(device));
  q4hip_logits* lg = new (std::nothrow) q4hip_logits();
  if (!lg) return fail(Q4HIP_EHIP, "out of host memory");
  lg->device = device;
  lg->vocab = vocab;
  lg->max_rows = max_rows;
  hipError_t e = hipStreamCreateWithFlags(&lg->stream, hipStreamNonBlocking);
  if (e == hipSuccess) e = hipMalloc(&lg->best, (size_t)max_rows * sizeof(*lg->best));
  if (e == hipSuccess) e = hipMalloc(&lg->arrived, (size_t)max_rows * sizeof(int));
  if (e == hipSuccess) e = hipMemsetAsync(lg->best, 0, (size_t)max_rows * sizeof(*lg->best), lg->stream);
  if (e == hipSuccess) e = hipMemsetAsync(lg->arrived, 0, (size_t)max_rows * sizeof(int), lg->stream);
  if (e == hipSuccess) e = hipStreamSynchronize(lg->stream);
  if (e != hipSuccess) {
    const int rc = fail(Q4HIP_EHIP, "logits of %d rows: %s", max_rows, hipGetErrorString(e));
    q4hip_logits_destroy(lg);
    return rc;
  }
  *out = lg;
  return Q4HIP_OK;
}

int q4hip_logits_run(q4hip_logits* lg, const void* x, void* y, int type, int64_t x_stride, int64_t y_stride, int rows,
                     const q4hip_logits_row* params, const int* history, int64_t history_n, const q4hip_logits_bias* biases,
                     int64_t biases_n, const uint32_t* mask, int mask_rows, int* best, void* stream) {
  if (!lg || !x || !y || !params) return fail(Q4HIP_EINVAL, "null argument");
  int rc = check_type(type);
  if (rc) return rc;
  if (rows < 0 || rows > lg->max_rows) return fail(Q4HIP_EINVAL, "%d rows: up to %d", rows, lg->max_rows);
  if (history_n < 0 || biases_n < 0 || mask_rows < 0 || (history_n && !history) || (biases_n && !biases) || (mask_rows && !mask))
    return fail(Q4HIP_EINVAL, "%lld tokens of history, %lld biases, %d masks", (long long)history_n, (long long)biases_n, mask_rows);
  if (history_n >= kMostEntries || biases_n >= kMostEntries) return fail(Q4HIP_EINVAL, "lists of less than 2^30 entries");
  if (!rows) return Q4HIP_OK;
  HIPCHK(hipSetDevice(lg->device));
  const int V = lg->vocab, words = (V + 31) / 32;
  const bool in_place = x == y && x_stride == y_stride;
  rc = check_rows(lg->device, x, rows, V, x_stride, type, "x");
  if (!rc && !in_place) rc = check_rows(lg->device, y, rows, V, y_stride, type, "y");
  if (!rc && !in_place) rc = check_apart(x, x_stride, y, y_stride, rows, V, type, "x and y");
  const size_t span = ((size_t)(rows - 1) * y_stride + V) * elem_size(type);
  const struct { const void* p; size_t n; const char* what; } lists[] = {
      {params, (size_t)rows * 8, "params"}, {history, (size_t)history_n, "history"}, {biases, (size_t)biases_n * 2, "biases"},
      {mask, (size_t)mask_rows * words, "mask"}};
  for (const auto& a : lists) {
    if (!rc) rc = check_ints(lg->device, a.p, a.n, a.what);
    if (!rc && (overlap(y, span, a.p, a.n * 4) || (best && overlap(best, (size_t)rows * 4, a.p, a.n * 4))))
      rc = fail(Q4HIP_EINVAL, "y or best overlaps %s", a.what);
  }
  if (!rc) rc = check_ints(lg->device, best, rows, "best");
  if (rc) return rc;
  const size_t x_span = ((size_t)(rows - 1) * x_stride + V) * elem_size(type);
  if (best && (overlap(best, (size_t)rows * 4, y, span) || overlap(best, (size_t)rows * 4, x, x_span)))
    return fail(Q4HIP_EINVAL, "best overlaps x or y");
  hipStream_t s = stream ? (hipStream_t)stream : lg->stream;
  const int large = kLargeThreads * kLargeEach, small = kSmallThreads * kSmallEach;
  const bool in_large = (int64_t)rows * ((V + large - 1) / large) >= kLargeFrom;
  const int size = in_large ? large : small, pieces = (V + size - 1) / size;
  const int threads = in_large ? kLargeThreads : kSmallThreads;
  const bool wide = aligned16(x, x_stride, type) && aligned16(y, y_stride, type);
  const int most = std::max(1, (int)(kMostThreads / threads / pieces));      // rows of a launch
  by_type(type, [&](auto zero) {
    using T = decltype(zero);
    constexpr int kVec = 16 / sizeof(T);
    auto* fn = in_large ? (wide ? k_logits<T, kVec, kLargeThreads, kLargeEach> : k_logits<T, 1, kLargeThreads, kLargeEach>)
                        : (wide ? k_logits<T, kVec, kSmallThreads, kSmallEach> : k_logits<T, 1, kSmallThreads, kSmallEach>);
    for (int64_t r = 0; r < rows; r += most) {
      const LogitsCall c{params + r, history, biases, mask, history_n, biases_n, mask_rows, V, pieces, words, x_stride, y_stride,
                         best ? best + r : nullptr, lg->best + r, lg->arrived + r};
      fn<<<(unsigned)(std::min<int64_t>(most, rows - r) * pieces), threads, 0, s>>>(c, (const T*)x + r * x_stride, (T*)y + r * y_stride);
    }
  });
  HIPCHK(hipGetLastError());
  if (!stream) HIPCHK(hipStreamSynchronize(s));
  return Q4HIP_OK;
}

}  // extern "C"
