// kv8_attend.h -- attention of a few rows over the paged 8-bit cache, on the matrix cores.
//
// For the rows r of a unit (16 / G neighbouring rows of a sequence and the G heads of a kv head) and its pages:
//   S^T = K q^T      16 positions x 16 rows a tile: the operand's positions are the codes as they lie in the cache
//   w   = 2^(S c + v - m)      c: K scale, attention scale, log2 e; v: exponent of the page's V scale; m: the row's
//                    largest such sum so far, less 14
//   O^T = V^T w      16 columns x 16 rows a tile, over the 32 positions of a page
//   l   = sum w 2^-v
// The scale of V goes into the exponent, so that the weights that the matrix cores take in fp16 are relative to the
// row's largest contribution and no page needs a product of its own.  The tile of scores leaves the matrix cores
// with the positions where the second product wants them (kv8.h: the order of V), so no weight changes lanes.
// Codes become fp16 by a byte permute (0x6400 | u = 1024 + u) and one packed subtraction: exact.  fp32 rows hold
// q and w as sums of two fp16 numbers and multiply twice; 16-bit rows as one.
#pragma once
#include "kv8.h"

namespace q4 {

using kv8_h2 = _Float16 __attribute__((ext_vector_type(2)));
using kv8_h8 = _Float16 __attribute__((ext_vector_type(8)));
using kv8_f4 = float __attribute__((ext_vector_type(4)));

constexpr float kKv8Lowest = -3.402823466e38f;

// 8 codes (two words) as the exact fp16 values code - 128.
__device__ inline kv8_h8 kv8_halves(uint32_t lo, uint32_t hi) {
  const kv8_h2 off = {(_Float16)-1152.0f, (_Float16)-1152.0f};
  union { kv8_h2 h[4]; kv8_h8 v; } u;
  u.h[0] = __builtin_bit_cast(kv8_h2, __builtin_amdgcn_perm(0x64646464u, lo, 0x04010400u)) + off;
  u.h[1] = __builtin_bit_cast(kv8_h2, __builtin_amdgcn_perm(0x64646464u, lo, 0x04030402u)) + off;
  u.h[2] = __builtin_bit_cast(kv8_h2, __builtin_amdgcn_perm(0x64646464u, hi, 0x04010400u)) + off;
  u.h[3] = __builtin_bit_cast(kv8_h2, __builtin_amdgcn_perm(0x64646464u, hi, 0x04030402u)) + off;
  return u.v;
}

__device__ inline float kv8_max_quarters(float x) {      // over lanes l, l ^ 16, l ^ 32, l ^ 48
  x = __builtin_fmaxf(x, __shfl_xor(x, 16));
  return __builtin_fmaxf(x, __shfl_xor(x, 32));
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

// A page's codes in the registers of a wave.
template <int HD>
struct Kv8Codes {
  uint4 k[HD / 32], v[HD / 32];
  __device__ void load(const uint8_t* page, int lane) {
    const uint4* p = (const uint4*)page + lane;
    for (int i = 0; i < HD / 32; i++) k[i] = p[i * 64];
    for (int i = 0; i < HD / 32; i++) v[i] = p[(HD / 32 + i) * 64];
  }
};

// Lane l: row l % 16 of the unit, quarter l / 16 of every contraction.
template <int HD, bool kTwo>
struct Kv8Rows {
  kv8_h8 q[kTwo ? 2 : 1][HD / 32];
  kv8_f4 o[HD / 16];
  float m, l, c;      // c: attention scale, log2 e and the power of two that q was divided by

  template <class T>
  __device__ void init(const T* row, int quarter, bool valid, float scale) {
    float x[HD / 32][8], most = 0.0f;
    for (int s = 0; s < HD / 32; s++)
      for (int i = 0; i < 8; i++) {
        x[s][i] = valid ? (float)row[s * 32 + quarter * 8 + i] : 0.0f;
        most = __builtin_fmaxf(most, __builtin_fabsf(x[s][i]));
      }
    most = kv8_max_quarters(most);
    const int e = 14 - __builtin_amdgcn_frexp_expf(most);      // the largest value becomes 2^13 .. 2^14
    for (int s = 0; s < HD / 32; s++)
      for (int i = 0; i < 8; i++) {
        const float y = __builtin_ldexpf(x[s][i], e);
        const _Float16 hi = (_Float16)y;
        q[0][s][i] = hi;
        if constexpr (kTwo) q[1][s][i] = (_Float16)(y - (float)hi);
      }
    c = __builtin_ldexpf(scale, -e);
    m = kKv8Lowest;
    l = 0.0f;
    for (auto& t : o) t = kv8_f4{0.0f, 0.0f, 0.0f, 0.0f};
  }

  // One page: its codes and scales (k, v), and the number of its positions that this lane's row looks at
  // (masked: some lane's row does not look at all 32).
  __device__ void page(const Kv8Codes<HD>& w, float k_scale, float v_scale, int quarter, bool masked, int seen) {
    kv8_f4 s[2] = {};
    for (int t = 0; t < 2; t++)
      for (int p = 0; p < HD / 64; p++) {
        const uint4 a = w.k[t * (HD / 64) + p];
        const kv8_h8 a0 = kv8_halves(a.x, a.y), a1 = kv8_halves(a.z, a.w);
        s[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a0, q[0][2 * p], s[t], 0, 0, 0);
        s[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a1, q[0][2 * p + 1], s[t], 0, 0, 0);
        if constexpr (kTwo) {
          s[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a0, q[1][2 * p], s[t], 0, 0, 0);
          s[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a1, q[1][2 * p + 1], s[t], 0, 0, 0);
        }
      }
    // v_scale = mant * 2^v with mant in [1, 2)
    const float vs = v_scale > 0.0f ? v_scale : kKv8MinScale;
    const int ve = __builtin_amdgcn_frexp_expf(vs) - 1;
    const float v = (float)ve, mant = __builtin_ldexpf(vs, -ve), ks = k_scale * c;
    float x[8], most = kKv8Lowest;
    for (int i = 0; i < 8; i++) {
      x[i] = __builtin_fmaf(s[i >> 2][i & 3], ks, v);
      if (masked && (i >> 2) * 16 + quarter * 4 + (i & 3) >= seen) x[i] = -__builtin_inff();
      most = __builtin_fmaxf(most, x[i]);
    }
    if (__builtin_amdgcn_ballot_w64(most - 14.0f > m) != 0) {      // rare but for the first pages
      const float m2 = __builtin_fmaxf(kv8_max_quarters(most) - 14.0f, m), f = __builtin_amdgcn_exp2f(m - m2);
      m = m2;
      l *= f;
      for (auto& t : o) t *= f;
    }
    float sum = 0.0f;
    kv8_h8 hi, lo;
    for (int i = 0; i < 8; i++) {
      const float e = __builtin_amdgcn_exp2f(x[i] - m);
      sum += e;
      float y = e * mant;
      if constexpr (kTwo) asm("" : "+v"(y));      // rounded to fp32 here: else one of its two uses takes the product rounded to fp16 at once
      hi[i] = (_Float16)y;
      if constexpr (kTwo) lo[i] = (_Float16)(y - (float)hi[i]);
    }
    l = __builtin_fmaf(sum, __builtin_ldexpf(1.0f, -ve), l);
    for (int p = 0; p < HD / 32; p++) {
      const kv8_h8 a0 = kv8_halves(w.v[p].x, w.v[p].y), a1 = kv8_halves(w.v[p].z, w.v[p].w);
      o[2 * p] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a0, hi, o[2 * p], 0, 0, 0);
      o[2 * p + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a1, hi, o[2 * p + 1], 0, 0, 0);
      if constexpr (kTwo) {
        o[2 * p] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a0, lo, o[2 * p], 0, 0, 0);
        o[2 * p + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a1, lo, o[2 * p + 1], 0, 0, 0);
      }
    }
  }
};

// A workgroup takes items of the plan, its four waves every fourth page each, and adds up their sums in shared
// memory.  Of a unit in several parts, the workgroup that is done last adds up the parts, in their order.
template <int HD, class T>
__global__ __launch_bounds__(256) void k_kv8_attend(Kv8View v, int layer, const T* __restrict__ q, T* __restrict__ out,
                                                    int64_t q_stride, int64_t out_stride, float scale, int rows) {
  constexpr bool kTwo = sizeof(T) == 4;
  constexpr int kLd = HD + 4;
  __shared__ float so[4][16][kLd];
  __shared__ float sm[4][16], sl[4][16];
  __shared__ int last;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = lane & 15, quarter = lane >> 4, G = v.H / v.KVH;
  const int g = blockIdx.y / v.row_tiles, r0 = (blockIdx.y % v.row_tiles) * 16;
  if (v.head->rows > rows) {                   // replayed on a larger plan than it was launched for
    if (tid == 0) v.head->status = KV8_STALE;
    return;
  }
  const size_t page_bytes = (size_t)2 * kKv8Block * HD;
  for (int i = blockIdx.x; i < v.head->items; i += gridDim.x) {
    const Kv8Item it = v.items[i];
    const int r = r0 + n, tok = r / G, h = r % G;
    const bool valid = r < it.n * G;
    Kv8Rows<HD, kTwo> w;
    w.init(q + (int64_t)(it.t + (valid ? tok : 0)) * q_stride + (g * G + (valid ? h : 0)) * HD, quarter, valid, scale);
    const int row_pos = it.pos + (valid ? tok : it.n - 1);      // the last position that this lane's row looks at
    const int* const table = v.table + (size_t)it.seq * v.W + it.page0;
    const int mine = (it.pages - wave + 3) >> 2;                // this wave's pages: wave, wave + 4, ...
    for (int j0 = 0; j0 < mine; j0 += 64) {
      // lane j holds the address and the scales of the j-th of the next 64 pages
      const int count = min(64, mine - j0);
      size_t at = 0;
      float2 sc = {0.0f, 0.0f};
      if (lane < count) {
        at = ((size_t)layer * v.pages + table[wave + 4 * (j0 + lane)]) * v.KVH + g;
        sc = v.scales[at];
      }
      const uint32_t at_lo = (uint32_t)at, at_hi = (uint32_t)(at >> 32);
      auto page_at = [&](int j) {
        const size_t b = ((size_t)__builtin_amdgcn_readlane((int)at_hi, j) << 32) | (uint32_t)__builtin_amdgcn_readlane((int)at_lo, j);
        return v.codes + b * page_bytes;
      };
      Kv8Codes<HD> buf[2];
      buf[0].load(page_at(0), lane);
      auto step = [&](int j, Kv8Codes<HD>& now, Kv8Codes<HD>& next) {
        if (j + 1 < count) next.load(page_at(j + 1), lane);
        const float ks = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(sc.x), j));
        const float vs = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(sc.y), j));
        const int p0 = (it.page0 + wave + 4 * (j0 + j)) * kKv8Block;
        w.page(now, ks, vs, quarter, p0 + kKv8Block - 1 > it.pos, row_pos + 1 - p0);
      };
      for (int j = 0; j < count; j += 2) {
        step(j, buf[0], buf[1]);
        if (j + 1 < count) step(j + 1, buf[1], buf[0]);
      }
    }
    w.l += __shfl_xor(w.l, 16);
    w.l += __shfl_xor(w.l, 32);
    if (quarter == 0) { sm[wave][n] = w.m; sl[wave][n] = w.l; }
    for (int d = 0; d < HD / 16; d++) *(kv8_f4*)&so[wave][n][d * 16 + quarter * 4] = w.o[d];
    __syncthreads();
    const size_t slot = (size_t)max(it.slot, 0) * gridDim.y + blockIdx.y;
    auto write = [&](int row, int d, kv8_f4 o, float l) {
      const int tk = (r0 + row) / G, hh = (r0 + row) % G;
      if (r0 + row >= it.n * G) return;
      T* p = out + (int64_t)(it.t + tk) * out_stride + (g * G + hh) * HD + d;
      for (int k = 0; k < 4; k++) p[k] = (T)(l == 0.0f ? 0.0f : o[k] / l);
    };
    for (int e = tid; e < 4 * HD; e += 256) {
      const int row = e / (HD / 4), d = e % (HD / 4) * 4;
      const float m = __builtin_fmaxf(__builtin_fmaxf(sm[0][row], sm[1][row]), __builtin_fmaxf(sm[2][row], sm[3][row]));
      kv8_f4 o = {0.0f, 0.0f, 0.0f, 0.0f};
      float l = 0.0f;
      for (int k = 0; k < 4; k++) {
        const float f = __builtin_amdgcn_exp2f(sm[k][row] - m);
        l = __builtin_fmaf(sl[k][row], f, l);
        const kv8_f4 x = *(const kv8_f4*)&so[k][row][d];
        for (int c = 0; c < 4; c++) o[c] = __builtin_fmaf(x[c], f, o[c]);
      }
      if (it.parts == 1) {
        write(row, d, o, l);
      } else {
        const size_t s = slot + (size_t)it.part * gridDim.y;
        if (r0 + row >= it.n * G) continue;
        float* const p = v.part_o + (s * 16 + row) * HD + d;
        kv8_send(p, o[0], o[1]);
        kv8_send(p + 2, o[2], o[3]);
        if (d == 0) kv8_send((float*)(v.part_ml + s * 16 + row), m, l);
      }
    }
    if (it.parts > 1) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");      // the part has arrived in memory before it is counted
      __syncthreads();
      if (tid == 0) {
        last = __hip_atomic_fetch_add(v.arrived + slot, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == it.parts - 1;
        if (last) __hip_atomic_store(v.arrived + slot, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);   // for the next launch
      }
      __syncthreads();
      if (last) {
        const size_t next = (size_t)gridDim.y * 16;          // from a part's rows to the next part's
        for (int e = tid; e < 4 * HD; e += 256) {
          const int row = e / (HD / 4), d = e % (HD / 4) * 4;
          if (r0 + row >= it.n * G) continue;
          const float* const ml = (const float*)(v.part_ml + slot * 16 + row);
          const float* const po = v.part_o + (slot * 16 + row) * HD + d;
          float m = kKv8Lowest, l = 0.0f;
          kv8_f4 o = {0.0f, 0.0f, 0.0f, 0.0f};
          for (int k0 = 0; k0 < it.parts; k0 += 8) {         // 8 parts on their way at once
            float2 a[8], x[8][2];
            float m2 = m;
#pragma unroll
            for (int k = 0; k < 8; k++) {
              const size_t at = (size_t)min(k0 + k, it.parts - 1) * next;
              a[k] = kv8_receive(ml + at * 2);
              x[k][0] = kv8_receive(po + at * HD);
              x[k][1] = kv8_receive(po + at * HD + 2);
            }
#pragma unroll
            for (int k = 0; k < 8; k++) m2 = __builtin_fmaxf(m2, a[k].x);
            const float f0 = __builtin_amdgcn_exp2f(m - m2);
            l *= f0;
            o *= f0;
            m = m2;
#pragma unroll
            for (int k = 0; k < 8; k++) {
              const float f = k0 + k < it.parts ? __builtin_amdgcn_exp2f(a[k].x - m) : 0.0f;
              l = __builtin_fmaf(a[k].y, f, l);
              o[0] = __builtin_fmaf(x[k][0].x, f, o[0]);
              o[1] = __builtin_fmaf(x[k][0].y, f, o[1]);
              o[2] = __builtin_fmaf(x[k][1].x, f, o[2]);
              o[3] = __builtin_fmaf(x[k][1].y, f, o[3]);
            }
          }
          write(row, d, o, l);
        }
      }
    }
    __syncthreads();                           // the shared sums have been read
  }
}

}  // namespace q4
