// kv8_attend.h -- attention over the paged 8-bit cache, on the matrix cores.
//
// For 16 rows r (a row: a position's q of one head; the heads of a kv head are rows of the same keys) and a page:
//   S^T = K q^T      16 positions x 16 rows a tile: the operand's positions are the codes as they lie in the cache
//   w   = 2^(S c + v - m)      c: K scale, attention scale, log2 e; v: log2 of the page's V scale; m: the row's
//                    largest such sum so far, less 14
//   O^T = V^T w      16 columns x 16 rows a tile, over the 32 positions of a page
//   l   = sum w 2^(m - v - r)
//                    r: the row's largest score in powers of two, less 14 and at most 1 more, so that m - r is a whole number
// The scale of V goes into the exponent, so that the weights that the matrix cores take in fp16 are relative to the
// row's largest contribution and no page needs a product of its own.  The tile of scores leaves the matrix cores
// with the positions where the second product wants them (kv8.h: the order of V), so no weight changes lanes.
// l has a reference of its own, as the V scales of a sequence's pages may lie 2^221 apart: relative to 2^m, the probabilities of
// zeros (which count as kKv8MinScale) would pass fp32 after 16,384 positions, or vanish beside a large V.  A part of a
// sequence travels as its own average of V, which fp32 holds, with l and r.
//
// w is the sum of two fp16 numbers, 22 bits, and is multiplied twice.  One number, off by up to 2^-11, adds an error of the
// size of fp16 outputs' own rounding where many positions count alike: 3,900 fp16 rows behind 4,000 positions 3.0e-4,
// with two 2.07e-4, which is the rounding alone (bf16 rows behind 60,000 1.69e-3 and 1.67e-3).
// V's codes become fp16 by a byte permute (0x6400 | u = 1024 + u, u = code + 128) and one packed subtraction, exactly.  The
// permute alone gives u * 2^-24, whose 128 the weights' sum could take back.  But the matrix instruction keeps no more of a
// product than the largest summand's 24 bits (32 products of 2^-25 leave 1 as it is), and what is left of sums
// of positive products after that is not exact enough: a token over 131,072 positions, columns of different size, was off by
// 2.7e-4 so (2.8e-4 where they were taken back at every page), 2.2e-4 now, the rounding alone.
// fp32 rows (kTwo) hold q, too, as the sum of two fp16 numbers; v is a whole number there and the scale's rest a factor
// of w, so that 2^-v is exact.
// 16-bit rows hold q as given.  K's codes are u * 2^-24 for them, and the product's first addend takes the 128 from the scores: the
// same outputs' errors as with exact codes in all of the cases above, and 775 us against 821 for the 8,192 rows below, 79 and
// 91 for a step of 4 prompts and 44 tokens (20 kv heads of 64; 32 tokens at 1,024 positions, though, 23 and 19).  l is the sum of the
// fp16 weights, a product with a row of ones.  (Not of a faint page, whose V scale is under 2^-12 of an earlier one's, 2^-40 for
// fp32 rows: its weights may be too small where its probabilities are not.)
//
// What bounds it.  One token of a short text: the launch and one chain of loads (5.8 us at 300 positions).  Many tokens: the
// cache's bytes, 1.12 GB in 216 us, 5.2 TB/s (64 sequences of up to 16,000 positions, 8 kv heads of 128 columns); a 1 GiB copy
// moves 5.15.  Prompts: the vector instructions that turn codes into fp16 (96 of some 220 for a page and 32 rows), split the
// weights (24), form the exponentials (16, at a quarter of the rate) and find the largest, 68% of the issue slots, beside matrix
// instructions that are busy 51% of the time: 8,192 bf16 rows, 32 heads of 128, in 772 us, 712 TFLOP/s; a large bf16 product
// reaches 1,221.
// Not kept, while weights were one fp16 number: raised priority around the matrix instructions (0 to 8% slower); a page's scores
// formed beside the weights of the page before (fp16 head_dim 64 5% faster, head_dim 128 out of registers and 2% slower, fp32 7%
// slower).
#pragma once
#include "kv8.h"

namespace q4 {

using kv8_h2 = _Float16 __attribute__((ext_vector_type(2)));
using kv8_f2 = float __attribute__((ext_vector_type(2)));
using kv8_h8 = _Float16 __attribute__((ext_vector_type(8)));
using kv8_f4 = float __attribute__((ext_vector_type(4)));

constexpr float kKv8Lowest = -3.402823466e38f;

// 8 codes (two words) as fp16: u = code + 128 as u * 2^-24, or exactly code.
template <bool kExact>
__device__ inline kv8_h8 kv8_halves(uint32_t lo, uint32_t hi) {
  constexpr uint32_t kHigh = kExact ? 0x64646464u : 0u;
  union { kv8_h2 h[4]; kv8_h8 v; } u;
  u.h[0] = __builtin_bit_cast(kv8_h2, __builtin_amdgcn_perm(kHigh, lo, kExact ? 0x04010400u : 0x0c010c00u));
  u.h[1] = __builtin_bit_cast(kv8_h2, __builtin_amdgcn_perm(kHigh, lo, kExact ? 0x04030402u : 0x0c030c02u));
  u.h[2] = __builtin_bit_cast(kv8_h2, __builtin_amdgcn_perm(kHigh, hi, kExact ? 0x04010400u : 0x0c010c00u));
  u.h[3] = __builtin_bit_cast(kv8_h2, __builtin_amdgcn_perm(kHigh, hi, kExact ? 0x04030402u : 0x0c030c02u));
  if constexpr (kExact) {
    const kv8_h2 off = {(_Float16)-1152.0f, (_Float16)-1152.0f};
    for (auto& h : u.h) h += off;
  }
  return u.v;
}

__device__ inline float kv8_max_quarters(float x) {      // over lanes l, l ^ 16, l ^ 32, l ^ 48
  x = __builtin_fmaxf(x, __shfl_xor(x, 16));
  return __builtin_fmaxf(x, __shfl_xor(x, 32));
}
__device__ inline float kv8_sum_quarters(float x) {
  x += __shfl_xor(x, 16);
  return x + __shfl_xor(x, 32);
}

// Parts of a unit travel between workgroups, whose XCDs have L2 caches of their own: 8-byte accesses of agent scope,
// which neither cache keeps.  A fence would write back and drop a whole L2 (30 us in a batch of 32 sequences).
using kv8_word = unsigned long long;
__device__ inline void kv8_send(float* p, float a, float b) {
  const kv8_word w = (kv8_word)__float_as_uint(b) << 32 | __float_as_uint(a);
  __hip_atomic_store((kv8_word*)p, w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ inline float2 kv8_receive(const float* p) {
  const kv8_word w = __hip_atomic_load((const kv8_word*)p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  return {__uint_as_float((uint32_t)w), __uint_as_float((uint32_t)(w >> 32))};
}

__device__ inline int kv8_div_g(const Kv8View& v, int r) { return v.g_magic ? (int)__umulhi((uint32_t)r, v.g_magic) : r; }

// 4 neighbouring values of a row; wide: its 16 bytes can be stored at once.
template <class T>
__device__ __forceinline__ void kv8_put4(T* p, bool wide, const kv8_f4& x) {
  union { uint64_t w[sizeof(T) / 2]; T y[4]; } u;
#pragma unroll
  for (int i = 0; i < 4; i++) u.y[i] = (T)x[i];
  if (wide) {
    if constexpr (sizeof(T) == 4) *(uint4*)p = *(const uint4*)&u;
    else *(uint64_t*)p = u.w[0];
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++) p[i] = u.y[i];
  }
}

// A page's codes in the registers of a wave.
template <int HD>
struct Kv8Codes {
  uint4 k[HD / 32], v[HD / 32];
  __device__ void load_k(const uint8_t* page, int lane) {
    const uint4* p = (const uint4*)page + lane;
#pragma unroll
    for (int i = 0; i < HD / 32; i++) k[i] = p[i * 64];
  }
  __device__ void load_v(const uint8_t* page, int lane) {
    const uint4* p = (const uint4*)page + lane;
#pragma unroll
    for (int i = 0; i < HD / 32; i++) v[i] = p[(HD / 32 + i) * 64];
  }
};

// What the softmax needs of a page's scales.
struct Kv8Scale {
  float k, v, iv, mant;      // K scale; v, 2^-v; the V scale over 2^v
};
template <bool kTwo>
__device__ inline Kv8Scale kv8_scale(float2 s) {
  const float vs = s.y > 0.0f ? s.y : kKv8MinScale;          // codes of 0: any scale will do
  if constexpr (kTwo) {
    const int e = __builtin_amdgcn_frexp_expf(vs) - 1;
    return {s.x, (float)e, __builtin_ldexpf(1.0f, -e), __builtin_ldexpf(vs, -e)};
  } else {
    const float v = __builtin_amdgcn_logf(vs);
    return {s.x, v, __builtin_amdgcn_exp2f(-v), 1.0f};
  }
}

// 16 N rows of a wave.  Lane l: rows l % 16 of each 16, quarter l / 16 of every contraction.
template <int HD, bool kTwo, int N>
struct Kv8Rows {
  kv8_h8 q[N][kTwo ? 2 : 1][HD / 32];
  kv8_f4 o[N][HD / 16];
  kv8_f4 first[kTwo ? 1 : N];                     // what the 128 add to the scores, negative
  float m[N], l[N], c[N];                         // c: attention scale, log2 e and the power of two that q was divided by
  float high[N];                                  // the largest score, less 14
  int d[N];                                       // m - r

  // The rows at row[t]; wide: 16 bytes of a row can be loaded at once.  All loads before any use: they wait for one another
  // otherwise.
  template <class T>
  __device__ __forceinline__ void init(const T* const (&row)[N], int quarter, bool wide, float scale) {
    union Raw { uint4 w[sizeof(T) / 2]; T y[8]; } raw[N][HD / 32];
    if (wide) {
#pragma unroll
      for (int t = 0; t < N; t++)
#pragma unroll
        for (int s = 0; s < HD / 32; s++)
#pragma unroll
          for (int i = 0; i < (int)sizeof(T) / 2; i++) raw[t][s].w[i] = ((const uint4*)(row[t] + s * 32 + quarter * 8))[i];
    } else {
#pragma unroll
      for (int t = 0; t < N; t++)
#pragma unroll
        for (int s = 0; s < HD / 32; s++)
#pragma unroll
          for (int i = 0; i < 8; i++) raw[t][s].y[i] = row[t][s * 32 + quarter * 8 + i];
    }
#pragma unroll
    for (int t = 0; t < N; t++) {
      float x[HD / 32][8];
#pragma unroll
      for (int s = 0; s < HD / 32; s++)
#pragma unroll
        for (int i = 0; i < 8; i++) x[s][i] = (float)raw[t][s].y[i];
      init_row(t, x, scale);
    }
  }

  __device__ __forceinline__ void init_row(int t, const float (&x)[HD / 32][8], float scale) {
    float most = 0.0f;
#pragma unroll
    for (int s = 0; s < HD / 32; s++)
#pragma unroll
      for (int i = 0; i < 8; i++) most = __builtin_fmaxf(most, __builtin_fabsf(x[s][i]));
    most = kv8_max_quarters(most);
    const int e = 14 - __builtin_amdgcn_frexp_expf(most);      // the largest value becomes 2^13 .. 2^14
    float all = 0.0f;
#pragma unroll
    for (int s = 0; s < HD / 32; s++)
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const float y = __builtin_ldexpf(x[s][i], e);
        const _Float16 hi = (_Float16)y;
        q[t][0][s][i] = hi;
        if constexpr (kTwo) q[t][1][s][i] = (_Float16)(y - (float)hi);
        else all += (float)hi;
      }
    // finite also for q of 2^119 and more, as the product with a page's K scale of 0 is 0
    c[t] = __builtin_fminf(__builtin_ldexpf(scale, -e + (kTwo ? 0 : 24)), -kKv8Lowest);
    if constexpr (!kTwo) {
      all = kv8_sum_quarters(all) * -0x1p-17f;                  // 128 * 2^-24
      first[t] = kv8_f4{all, all, all, all};
    }
    m[t] = kKv8Lowest;
    l[t] = 0.0f;
    high[t] = kKv8Lowest;
    d[t] = 0;
#pragma unroll
    for (auto& x : o[t]) x = kv8_f4{0.0f, 0.0f, 0.0f, 0.0f};
  }

  __device__ __forceinline__ void scores(const Kv8Codes<HD>& w, kv8_f4 (&s)[N][2]) const {
#pragma unroll
    for (int t = 0; t < N; t++)
#pragma unroll
      for (int h = 0; h < 2; h++) {
        if constexpr (kTwo) s[t][h] = kv8_f4{0.0f, 0.0f, 0.0f, 0.0f};
        else s[t][h] = first[t];
      }
#pragma unroll
    for (int p = 0; p < HD / 32; p++)       // the 2 N sums in turn, as each addition waits for the one before
#pragma unroll
      for (int part = 0; part < (kTwo ? 2 : 1); part++)
#pragma unroll
        for (int h = 0; h < 2; h++) {
          const uint4 a = w.k[h * (HD / 64) + p / 2];
          const kv8_h8 x = p % 2 ? kv8_halves<kTwo>(a.z, a.w) : kv8_halves<kTwo>(a.x, a.y);
#pragma unroll
          for (int t = 0; t < N; t++) s[t][h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, q[t][part][p], s[t][h], 0, 0, 0);
        }
  }

  // Scores of positions that a row does not look at.  (ks of at least 2^-60, as 0 would make them NaN: it changes no
  // exponent by more than 2^-25.)
  __device__ __forceinline__ void mask(kv8_f4 (&s)[N][2], float (&ks)[N], int quarter, const int (&seen)[N]) const {
#pragma unroll
    for (int t = 0; t < N; t++) {
      ks[t] = __builtin_fmaxf(ks[t], 0x1p-60f);
#pragma unroll
      for (int i = 0; i < 8; i++)
        if ((i >> 2) * 16 + quarter * 4 + (i & 3) >= seen[t]) s[t][i >> 2][i & 3] = -__builtin_inff();
    }
  }

  // m becomes m2, after scores of up to `most`.
  __device__ __forceinline__ void move(int t, float m2, float most) {
    high[t] = __builtin_fmaxf(high[t], most - 14.0f);
    const int d2 = (int)__builtin_floorf(__builtin_fminf(__builtin_fmaxf(m2 - high[t], -256.0f), 256.0f));
    l[t] *= __builtin_amdgcn_exp2f((m[t] - m2) + (float)(d2 - d[t]));
    m[t] = m2;
    d[t] = d2;
  }

  // One page from its scores: the number of its positions that this lane's rows look at (masked: not all rows look at
  // all 32); faint: its share of l is formed of its scores alone.
  __device__ __forceinline__ void page(kv8_f4 (&s)[N][2], const Kv8Codes<HD>& w, Kv8Scale sc, int quarter, bool masked,
                                       const int (&seen)[N], bool faint) {
    float ks[N], most[N];
#pragma unroll
    for (int t = 0; t < N; t++) ks[t] = sc.k * c[t];
    // the branches that few pages take lie behind the loop (8,192 fp32 rows 284 us, within it 287)
    if (__builtin_expect(masked, 0)) mask(s, ks, quarter, seen);
    bool up = false;
#pragma unroll
    for (int t = 0; t < N; t++) {
      most[t] = s[t][0][0];
#pragma unroll
      for (int i = 1; i < 8; i++) most[t] = __builtin_fmaxf(most[t], s[t][i >> 2][i & 3]);
      most[t] = __builtin_fmaf(most[t], ks[t], sc.v);
      // weights of up to 2^14, or 2^15.5 before m is moved again
      up = up || most[t] - (kTwo ? 14.0f : 15.5f) > m[t];
    }
    if (__builtin_expect(__builtin_amdgcn_ballot_w64(up) != 0, 0))
#pragma unroll
      for (int t = 0; t < N; t++) {
        const float x = kv8_max_quarters(most[t]), m2 = __builtin_fmaxf(x - 14.0f, m[t]), f = __builtin_amdgcn_exp2f(m[t] - m2);
        move(t, m2, x - sc.v);
#pragma unroll
        for (auto& y : o[t]) y *= f;
      }
    if (__builtin_expect(faint, 0))
#pragma unroll
      for (int t = 0; t < N; t++) {
        move(t, m[t], kv8_max_quarters(most[t]) - sc.v);
        float all = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; i++) all += __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][i >> 2][i & 3], ks[t], (float)d[t] - m[t]));
        l[t] += kTwo ? all : kv8_sum_quarters(all);
      }
    const float l_scale = faint ? 0.0f : sc.iv;
    float minus = -1.0f;
    asm("" : "+s"(minus));        // not known to the compiler: the difference below stays one fused operation that rounds to fp16
    kv8_h8 hi[N], lo[N];
#pragma unroll
    for (int t = 0; t < N; t++) {
      const float v = sc.v - m[t];
      float all = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        kv8_f2 y;
#pragma unroll
        for (int k = 0; k < 2; k++) y[k] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][i >> 2][(i & 3) + k], ks[t], v));
        if constexpr (kTwo) {
          all += y[0];
          all += y[1];
          y *= sc.mant;
          asm("" : "+v"(y));      // rounded to fp32 here: else one of its two uses takes the product rounded to fp16 at once
        }
        kv8_h2 h = __builtin_convertvector(y, kv8_h2);
        asm("" : "+v"(h));        // both by one conversion, not again one by one
#pragma unroll
        for (int k = 0; k < 2; k++) {
          hi[t][i + k] = h[k];
          lo[t][i + k] = (_Float16)__builtin_fmaf((float)h[k], minus, y[k]);
        }
      }
      if constexpr (!kTwo) {
        const kv8_h8 ones = {1, 1, 1, 1, 1, 1, 1, 1};
        kv8_f4 r = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, hi[t], kv8_f4{0.0f, 0.0f, 0.0f, 0.0f}, 0, 0, 0);
        r = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, lo[t], r, 0, 0, 0);
        all = r[0];
      }
      l[t] = __builtin_fmaf(all, __builtin_ldexpf(l_scale, d[t]), l[t]);
    }
#pragma unroll
    for (int p = 0; p < HD / 32; p++) {
      const kv8_h8 a0 = kv8_halves<true>(w.v[p].x, w.v[p].y), a1 = kv8_halves<true>(w.v[p].z, w.v[p].w);
#pragma unroll
      for (int t = 0; t < N; t++) {
        o[t][2 * p] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a0, hi[t], o[t][2 * p], 0, 0, 0);
        o[t][2 * p + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a1, hi[t], o[t][2 * p + 1], 0, 0, 0);
        o[t][2 * p] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a0, lo[t], o[t][2 * p], 0, 0, 0);
        o[t][2 * p + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a1, lo[t], o[t][2 * p + 1], 0, 0, 0);
      }
    }
  }

  // The pages seen: l becomes the sum of all quarters.
  __device__ void finish(int t) {
    if constexpr (kTwo) l[t] = kv8_sum_quarters(l[t]);
  }
  __device__ float reference(int t) const { return m[t] - (float)d[t]; }

  // Pages first, first + step, ... (count of them) of a sequence's table, whose first row of this wave lies at
  // position `from`; lane's row t looks at positions up to last[t].  A page's K is loaded when the scores of the page
  // before are formed, its V when that page's are used up.
  __device__ __forceinline__ void run(const Kv8View& v, int layer, int g, const int* table, int first, int step, int count, int from,
                                      const int (&last)[N]) {
    const int lane = threadIdx.x & 63, quarter = lane >> 4;
    const size_t page_bytes = (size_t)2 * kKv8Block * HD;
    float top = kKv8Lowest;
    for (int j0 = 0; j0 < count; j0 += 64) {
      // lane j holds the place and the scales of the j-th of the next 64 pages
      const int n = min(64, count - j0);
      size_t at = 0;
      Kv8Scale sc = {};
      if (lane < n) {
        at = ((size_t)layer * v.pages + table[first + step * (j0 + lane)]) * v.KVH + g;
        sc = kv8_scale<kTwo>(v.scales[at]);
      }
      const uint32_t at_lo = (uint32_t)at, at_hi = (uint32_t)(at >> 32);
      auto page_at = [&](int j) {
        const size_t b = ((size_t)__builtin_amdgcn_readlane((int)at_hi, j) << 32) | (uint32_t)__builtin_amdgcn_readlane((int)at_lo, j);
        return v.codes + b * page_bytes;
      };
      auto lane_of = [](float x, int j) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), j)); };
      Kv8Codes<HD> w;
      w.load_k(page_at(0), lane);
      w.load_v(page_at(0), lane);
      for (int j = 0; j < n; j++) {
        const uint8_t* const next = page_at(min(j + 1, n - 1));
        kv8_f4 s[N][2];
        scores(w, s);
        w.load_k(next, lane);
        const Kv8Scale y = {lane_of(sc.k, j), lane_of(sc.v, j), lane_of(sc.iv, j), kTwo ? lane_of(sc.mant, j) : 1.0f};
        const int p0 = (first + step * (j0 + j)) * kKv8Block;
        int seen[N];
#pragma unroll
        for (int t = 0; t < N; t++) seen[t] = last[t] + 1 - p0;
        page(s, w, y, quarter, p0 + kKv8Block - 1 > from, seen, y.v < top - (kTwo ? 40.0f : 12.0f));
        w.load_v(next, lane);
        top = __builtin_fmaxf(top, y.v);
      }
    }
  }
};

// 4 columns of a row of the average of `parts` parts at `slot`, `slot + step`, ...: o; l relative to 2^m.
template <int HD>
__device__ inline void kv8_join(const Kv8View& v, size_t slot, size_t step, int parts, int row, int d, kv8_f4& o, float& m, float& l) {
  const float* const ml = (const float*)(v.part_ml + slot * 32 + row);
  const float* const po = v.part_o + (slot * 32 + row) * HD + d;
  m = kKv8Lowest;
  l = 0.0f;
  o = kv8_f4{0.0f, 0.0f, 0.0f, 0.0f};
  for (int k0 = 0; k0 < parts; k0 += 8) {         // 8 parts on their way at once
    float2 a[8], x[8][2];
    float m2 = m;
#pragma unroll
    for (int k = 0; k < 8; k++) {
      const size_t at = (size_t)min(k0 + k, parts - 1) * step * 32;
      a[k] = kv8_receive(ml + at * 2);
      x[k][0] = kv8_receive(po + at * HD);
      x[k][1] = kv8_receive(po + at * HD + 2);
    }
#pragma unroll
    for (int k = 0; k < 8; k++) m2 = __builtin_fmaxf(m2, a[k].x);
    const float l0 = l * __builtin_amdgcn_exp2f(m - m2);
    l = l0;
    m = m2;
#pragma unroll
    for (int k = 0; k < 8; k++) {
      a[k].y *= k0 + k < parts ? __builtin_amdgcn_exp2f(a[k].x - m) : 0.0f;
      l += a[k].y;
    }
    const float il = l == 0.0f ? 0.0f : 1.0f / l;
    o *= l0 * il;
#pragma unroll
    for (int k = 0; k < 8; k++) {
      const float f = a[k].y * il;
      o[0] = __builtin_fmaf(x[k][0].x, f, o[0]);
      o[1] = __builtin_fmaf(x[k][0].y, f, o[1]);
      o[2] = __builtin_fmaf(x[k][1].x, f, o[2]);
      o[3] = __builtin_fmaf(x[k][1].y, f, o[3]);
    }
  }
}

template <int HD>
__device__ inline void kv8_send_part(const Kv8View& v, size_t slot, int row, int d, kv8_f4 o, float m, float l) {
  float* const p = v.part_o + (slot * 32 + row) * HD + d;
  kv8_send(p, o[0], o[1]);
  kv8_send(p + 2, o[2], o[3]);
  if (d == 0) kv8_send((float*)(v.part_ml + slot * 32 + row), m, l);
}

// The same for the launch behind this one, which no other XCD's access needs to get past a cache for.
template <int HD>
__device__ inline void kv8_keep_part(const Kv8View& v, size_t slot, int row, int d, kv8_f4 o, float m, float l) {
  *(kv8_f4*)(v.part_o + (slot * 32 + row) * HD + d) = o;
  if (d == 0) v.part_ml[slot * 32 + row] = {m, l};
}

template <int HD>
struct Kv8Shared {
  float o[4][16][HD + 4];
  float m[4][16], r[4][16], l[4][16];
  int last;
};

// Whether this workgroup is the last of `count` to arrive at *counter, with what it sent in memory before.
template <class S>
__device__ inline bool kv8_last(S& sh, int* counter, int count) {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0) {
    sh.last = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == count - 1;
    if (sh.last) __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);   // for the next launch
  }
  __syncthreads();
  return sh.last != 0;
}

// An item of the plan and 16 N of its unit's rows of a kv head (y).  Waves share the pages and not the rows, as a token has
// few rows and the loads of four waves are in flight at once; 131,072 positions of one sequence, in parts, 14.5 us.
// The four waves take every fourth page each and add up their sums in shared memory, 16 rows at a time.  A unit in
// several parts: the last workgroup of each 16 parts to be done adds those up, and the last of these the sums of 16, always
// in the order of the parts.
// kJoint: the item may be of a joint.  Then its sums stay in the workspace, for kv8_gather.
template <int HD, class T, int N, bool kJoint>
__device__ __forceinline__ void kv8_item(const Kv8View& v, const Kv8JointView& jv, const Kv8Item& it, Kv8Shared<HD>& sh, int layer,
                                         const T* q, T* out, int64_t q_stride, int64_t out_stride, float scale, bool wide, int y) {
  constexpr bool kTwo = sizeof(T) == 4;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = lane & 15, quarter = lane >> 4, G = v.H / v.KVH;
  const int g = y / v.row_tiles, r0 = (y % v.row_tiles) * (16 * N);
  const bool joint = kJoint && it.joint, common = joint && it.joint > 0;
  const int rows = min(16 * N, common ? it.n : it.n * G - r0);                  // of this tile
  if (rows <= 0) return;
  Kv8Rows<HD, kTwo, N> w;
  int row_last[N];
  const T* row[N];
#pragma unroll
  for (int t = 0; t < N; t++) {
    const int r = r0 + min(t * 16 + n, rows - 1), tok = kv8_div_g(v, r);      // rows behind the end: as the last one, not written
    if (common) {
      const Kv8JointRow* const jr = jv.rows + (size_t)(it.joint - 1) * 32 + r;
      row[t] = q + (int64_t)jr->t * q_stride + (g * G + jr->h) * HD;
      row_last[t] = INT32_MAX - 1;             // all of the pages
      continue;
    }
    row[t] = q + (int64_t)(it.t + tok) * q_stride + (g * G + r - tok * G) * HD;
    row_last[t] = it.pos + tok;
  }
  w.init(row, quarter, wide, scale);
  w.run(v, layer, g, v.table + (size_t)it.seq * v.W, it.page0 + wave, 4, (it.pages - wave + 3) >> 2, common ? INT32_MAX : it.pos,
        row_last);
  const int ys = v.KVH * v.row_tiles;
  const size_t slot = (size_t)max(it.slot, 0) * ys + y;         // of the unit's first part
  auto write = [&](int row, int d, const kv8_f4& o) {
    const int r = r0 + row, tok = kv8_div_g(v, r);
    kv8_put4(out + (int64_t)(it.t + tok) * out_stride + (g * G + r - tok * G) * HD + d, wide, o);
  };
#pragma unroll
  for (int t = 0; t < N; t++) {
    w.finish(t);
    __syncthreads();                         // the shared sums before have been read
    if (quarter == 0) { sh.m[wave][n] = w.m[t]; sh.r[wave][n] = w.reference(t); sh.l[wave][n] = w.l[t]; }
#pragma unroll
    for (int d = 0; d < HD / 16; d++) *(kv8_f4*)&sh.o[wave][n][d * 16 + quarter * 4] = w.o[t][d];
    __syncthreads();
    for (int e = tid; e < min(16, rows - t * 16) * (HD / 4); e += 256) {
      const int row = e / (HD / 4), d = e % (HD / 4) * 4;
      const float r = __builtin_fmaxf(__builtin_fmaxf(sh.r[0][row], sh.r[1][row]), __builtin_fmaxf(sh.r[2][row], sh.r[3][row]));
      float l = 0.0f;
      for (int k = 0; k < 4; k++) l = __builtin_fmaf(sh.l[k][row], __builtin_amdgcn_exp2f(sh.r[k][row] - r), l);
      const float il = l == 0.0f ? 0.0f : 1.0f / l;
      kv8_f4 o = {0.0f, 0.0f, 0.0f, 0.0f};
      for (int k = 0; k < 4; k++) {
        const float f = __builtin_amdgcn_exp2f(sh.m[k][row] - r);          // f * il may be too small
        const kv8_f4 x = *(const kv8_f4*)&sh.o[k][row][d];
        for (int c = 0; c < 4; c++) o[c] = __builtin_fmaf(x[c] * il, f, o[c]);
      }
      if (joint && !common && it.parts == 1) {
        const int at = it.row + t * 16 + row;
        kv8_keep_part<HD>(v, (size_t)(jv.most + (at >> 5)) * ys + y, at & 31, d, o, r, l);
      } else if (joint) {
        kv8_keep_part<HD>(v, slot + (size_t)it.part * ys, t * 16 + row, d, o, r, l);
      } else if (it.parts == 1) write(t * 16 + row, d, o);
      else kv8_send_part<HD>(v, slot + (size_t)it.part * ys, t * 16 + row, d, o, r, l);
    }
  }
  if (it.parts > 1 && !joint) {
    const int first = it.part & ~15, mine = min(16, it.parts - first), sixteens = (it.parts + 15) >> 4;
    const size_t own = slot + (size_t)first * ys;
    if (kv8_last(sh, v.arrived + own, mine)) {
      for (int e = tid; e < rows * (HD / 4); e += 256) {
        const int row = e / (HD / 4), d = e % (HD / 4) * 4;
        kv8_f4 o;
        float m, l;
        kv8_join<HD>(v, own, ys, mine, row, d, o, m, l);
        if (sixteens == 1) write(row, d, o);
        else kv8_send_part<HD>(v, own, row, d, o, m, l);        // over the first part: a row's threads are of one wave
      }
      if (sixteens > 1 && kv8_last(sh, v.arrived + slot + ys, sixteens))      // counted at the second part
        for (int e = tid; e < rows * (HD / 4); e += 256) {
          const int row = e / (HD / 4), d = e % (HD / 4) * 4;
          kv8_f4 o;
          float m, l;
          kv8_join<HD>(v, slot, (size_t)16 * ys, sixteens, row, d, o, m, l);
          write(row, d, o);
        }
    }
  }
}

// Many rows: 64 N neighbouring rows of a sequence and kv head (row r: position r / G of the step, head r % G), 16 N of each
// wave, which passes over all the pages that they look at.  So a page is fetched once for 128 rows, and from the L2 by each
// wave: no shared memory, no barrier.  (32 rows of a wave rather than 16: the codes' fp16 forms serve both.)
template <int HD, class T, int N>
__device__ __forceinline__ void kv8_tile(const Kv8View& v, int layer, const T* q, T* out, int64_t q_stride, int64_t out_stride,
                                         float scale, bool wide, int tile, int g) {
  constexpr bool kTwo = sizeof(T) == 4;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, quarter = lane >> 4, G = v.H / v.KVH;
  const Kv8Tile it = v.tiles[tile];
  const int r0 = it.tile * kKv8TileRows + wave * (16 * N), end = it.n * G;
  if (r0 >= end) return;
  Kv8Rows<HD, kTwo, N> w;
  int last[N];
  const T* row[N];
#pragma unroll
  for (int t = 0; t < N; t++) {
    const int r = min(r0 + t * 16 + n, end - 1), tok = kv8_div_g(v, r);      // rows behind the end: as the last one, not written
    last[t] = it.pos + tok;
    row[t] = q + (int64_t)(it.t + tok) * q_stride + (g * G + r - tok * G) * HD;
  }
  w.init(row, quarter, wide, scale);
  const int from = it.pos + kv8_div_g(v, r0), to = it.pos + kv8_div_g(v, min(r0 + 16 * N, end) - 1);
  w.run(v, layer, g, v.table + (size_t)it.seq * v.W, 0, 1, to / kKv8Block + 1, from, last);
#pragma unroll
  for (int t = 0; t < N; t++) {
    w.finish(t);
    const int r = r0 + t * 16 + n, tok = kv8_div_g(v, r);
    if (r >= end) continue;
    T* const p = out + (int64_t)(it.t + tok) * out_stride + (g * G + r - tok * G) * HD + quarter * 4;
    const float il = w.l[t] == 0.0f ? 0.0f : 1.0f / w.l[t], f = __builtin_ldexpf(1.0f, w.d[t]);
#pragma unroll
    for (int d = 0; d < HD / 16; d++) kv8_put4(p + d * 16, wide, w.o[t][d] * il * f);
  }
}

// A step's tiles, the longest first, then its items.  The kv heads are neighbours in the grid, so that the tiles of one
// meet on the same XCDs and find its pages in their L2.
template <int HD, class T, int N>
__global__ __launch_bounds__(256, 2) void k_kv8_attend(Kv8View v, int layer, const T* __restrict__ q, T* __restrict__ out,
                                                    int64_t q_stride, int64_t out_stride, float scale, int rows, bool wide) {
  __shared__ Kv8Shared<HD> sh;
  const int ys = v.KVH * v.row_tiles;
  const Kv8Head head = *v.head;
  Kv8Item it;
  if constexpr (N == 0) it = v.items[blockIdx.x / ys];      // on its way together with the head: the grid is no larger than the list
  if (head.rows > rows) {                      // replayed on a larger plan than it was launched for
    if (threadIdx.x == 0) v.head->status = KV8_STALE;
    return;
  }
  const int tiles = N ? head.tiles * v.KVH : 0, all = tiles + head.items * ys;
  for (int i = blockIdx.x; i < all; i += gridDim.x) {
    if constexpr (N > 0)
      if (i < tiles) {
        kv8_tile<HD, T, N>(v, layer, q, out, q_stride, out_stride, scale, wide, i / v.KVH, i % v.KVH);
        continue;
      }
    const int k = i - tiles, y = k % ys;
    if (N > 0 || i != (int)blockIdx.x) it = v.items[k / ys];
    if constexpr (N > 0)
      if (it.wide) {
        kv8_item<HD, T, N, false>(v, {}, it, sh, layer, q, out, q_stride, out_stride, scale, wide, y);
        continue;
      }
    kv8_item<HD, T, 1, false>(v, {}, it, sh, layer, q, out, q_stride, out_stride, scale, wide, y);
  }
}

// The same from the list with joints, if the plan has made one.  Its items differ in length by a factor of ten, and a grid's
// workgroups go to the 4 shader engines of an XCD one after the other, whatever these still hold: 512 items of joints beside as many
// short ones ran on half of the CUs.  So as many workgroups as fit stay, and draw an item when they are done with one.  (Drawn a turn
// ahead, an item waits for its workgroup's long one beside idle ones.)
template <int HD, class T>
__global__ __launch_bounds__(256, 2) void k_kv8_attend_joint(Kv8View v, Kv8JointView jv, int layer, const T* __restrict__ q,
                                                          T* __restrict__ out, int64_t q_stride, int64_t out_stride, float scale,
                                                          int rows, bool wide) {
  __shared__ Kv8Shared<HD> sh;
  __shared__ int drawn;
  const int ys = v.KVH * v.row_tiles, tid = threadIdx.x;
  const Kv8Head head = *v.head;
  if (head.rows > rows) {
    if (tid == 0) v.head->status = KV8_STALE;
    return;
  }
  const Kv8Item* const items = head.joint_items ? jv.items : v.items;
  const int tiles = head.tiles * v.KVH, all = tiles + (head.joint_items ? head.joint_items : head.items) * ys;
  for (int i = blockIdx.x; i < all;) {
    if (i < tiles) {
      kv8_tile<HD, T, 2>(v, layer, q, out, q_stride, out_stride, scale, wide, i / v.KVH, i % v.KVH);
    } else {
      const int k = i - tiles;
      const Kv8Item it = items[k / ys];
      if (it.wide) kv8_item<HD, T, 2, true>(v, jv, it, sh, layer, q, out, q_stride, out_stride, scale, wide, k % ys);
      else kv8_item<HD, T, 1, true>(v, jv, it, sh, layer, q, out, q_stride, out_stride, scale, wide, k % ys);
    }
    if (all <= (int)gridDim.x) return;
    __syncthreads();                           // everybody has read `drawn`
    if (tid == 0) drawn = gridDim.x + __hip_atomic_fetch_add(jv.queue, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    i = __builtin_amdgcn_readfirstlane(drawn);
  }
}

// The rows of joints: threads of a row take 4 columns each, of every so-manieth part of its joint and its unit, so that each has about
// four to load; what they have is added up in shared memory.
// (The last workgroup to be done could, too, as it does for units: but it alone then reads up to 128 parts of 32 rows.  8 sequences
// behind 131,072 positions: 41.3 us so, 26.2 in a launch of its own.)
template <int HD, class T>
__global__ __launch_bounds__(256) void k_kv8_gather(Kv8View v, Kv8JointView jv, T* __restrict__ out, int64_t out_stride, int rows,
                                                    bool wide) {
  constexpr int kCols = HD / 4, kGroups = 256 / kCols;
  __shared__ kv8_f4 so[kGroups][kCols];
  __shared__ float2 sml[kGroups];
  const Kv8Head head = *v.head;
  if (head.rows > rows) return;
  int slices = 1;
  while (slices < kGroups && 4 * slices < head.most_parts) slices *= 2;
  if (blockIdx.x == 0 && threadIdx.x == 0) *jv.queue = 0;
  const int tid = threadIdx.x, col = tid % kCols, mine = tid / kCols, group = mine % slices, d = col * 4, G = v.H / v.KVH, ys = v.KVH;
  const int each = kGroups / slices, all = head.joints * 32 * ys;
  for (int i0 = blockIdx.x * each; i0 < all; i0 += gridDim.x * each) {
    const int i = min(i0 + mine / slices, all - 1), at = i / ys, y = i - at * ys;
    const Kv8JointRow r = jv.rows[at];
    const Kv8Joint j = jv.joints[at >> 5];
    const int parts = r.t < 0 ? 0 : j.parts + r.parts;
    float m = kKv8Lowest, l = 0.0f;
    kv8_f4 o = {0.0f, 0.0f, 0.0f, 0.0f};       // an average, as in kv8_join
    for (int k0 = group; k0 < parts; k0 += 4 * slices) {
      float2 a[4];
      kv8_f4 x[4];
      float m2 = m;
#pragma unroll
      for (int k = 0; k < 4; k++) {
        const int p = min(k0 + k * slices, parts - 1);
        const bool common = p < j.parts;
        const size_t e = ((size_t)(common ? j.slot + p : r.slot + p - j.parts) * ys + y) * 32 + (common ? at & 31 : r.row);
        a[k] = v.part_ml[e];
        x[k] = *(const kv8_f4*)(v.part_o + e * HD + d);
      }
#pragma unroll
      for (int k = 0; k < 4; k++) {
        if (k0 + k * slices >= parts) a[k] = {kKv8Lowest, 0.0f};
        m2 = __builtin_fmaxf(m2, a[k].x);
      }
      const float l0 = l * __builtin_amdgcn_exp2f(m - m2);
      m = m2;
      l = l0;
#pragma unroll
      for (int k = 0; k < 4; k++) {
        a[k].y *= __builtin_amdgcn_exp2f(a[k].x - m);
        l += a[k].y;
      }
      const float il = l == 0.0f ? 0.0f : 1.0f / l;
      o *= l0 * il;
#pragma unroll
      for (int k = 0; k < 4; k++)
        for (int c = 0; c < 4; c++) o[c] = __builtin_fmaf(x[k][c], a[k].y * il, o[c]);
    }
    if (slices > 1) {
      __syncthreads();                         // the rows before have been read
      so[mine][col] = o;
      if (col == 0) sml[mine] = {m, l};
      __syncthreads();
    }
    if (group || !parts) continue;
    if (slices > 1) {
      const int used = min(parts, slices);
      for (int k = 0; k < used; k++) m = __builtin_fmaxf(m, sml[mine + k].x);
      l = 0.0f;
      o = kv8_f4{0.0f, 0.0f, 0.0f, 0.0f};
      for (int k = 0; k < used; k++) l = __builtin_fmaf(sml[mine + k].y, __builtin_amdgcn_exp2f(sml[mine + k].x - m), l);
      const float il = l == 0.0f ? 0.0f : 1.0f / l;
      for (int k = 0; k < used; k++) {
        const float f = sml[mine + k].y * il * __builtin_amdgcn_exp2f(sml[mine + k].x - m);
        const kv8_f4 x = so[mine + k][col];
        for (int c = 0; c < 4; c++) o[c] = __builtin_fmaf(x[c], f, o[c]);
      }
    }
    kv8_put4(out + (int64_t)r.t * out_stride + (y * G + r.h) * HD + d, wide, o);
  }
}

}  // namespace q4
