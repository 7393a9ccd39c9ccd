// kv8_plan.h -- a step's pages, rows and work lists from request lengths, on the GPU.
//
// One workgroup sums over the sequences (pages given back and taken, rows, runs, items); whoever then wants
// the i-th page, row, run or item finds its sequence by bisection of those sums.  So no thread walks through a
// long sequence alone, and the lists can be spread over the GPU where there is much of them.
// Nothing but latency bounds it: a chain of loads, sums and bisections.  With up to kPlanShared sequences
// the sums stay in shared memory (32 sequences 13.2 -> 7.1 us a launch).
#pragma once
#include "kv8.h"

namespace q4 {

constexpr int kPlanThreads = 1024;
constexpr int kPlanShared = 1024;

__device__ inline int kv8_pages(int n) { return (n + kKv8Block - 1) / kKv8Block; }

// Inclusive sums of N numbers over the workgroup's threads; total[] receives the sums of all.
template <int N>
__device__ void wg_scan(int (&x)[N], int (&total)[N], int (*part)[N]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1)
#pragma unroll
    for (int k = 0; k < N; k++) {
      const int u = __shfl_up(x[k], d);
      if (lane >= d) x[k] += u;
    }
  __syncthreads();                       // `part` of the sums before has been read
  if (lane == 63)
#pragma unroll
    for (int k = 0; k < N; k++) part[wave][k] = x[k];
  __syncthreads();
#pragma unroll
  for (int k = 0; k < N; k++) total[k] = 0;
  for (int w = 0; w < waves; w++)
#pragma unroll
    for (int k = 0; k < N; k++) {
      const int p = part[w][k];
      if (w < wave) x[k] += p;
      total[k] += p;
    }
}

// The last sequence b with at[b] <= i.
__device__ inline int find(const int* at, int B, int i) {
  int lo = 0, hi = B;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (at[mid] <= i) lo = mid; else hi = mid;
  }
  return lo;
}

// Rows of the units of a sequence that adds `add` rows, units, tiles, and the parts of a unit.
__device__ inline int kv8_unit_rows(const Kv8View& v, int add) { return add > v.unit_rows ? v.wide_rows : v.unit_rows; }
__device__ inline int kv8_units(const Kv8View& v, int add) {
  const int r = kv8_unit_rows(v, add);
  return (add + r - 1) / r;
}
__device__ inline int kv8_tiles(const Kv8View& v, int add) {
  return add > v.unit_rows ? (int)(((int64_t)add * (v.H / v.KVH) + kKv8TileRows - 1) / kKv8TileRows) : 0;
}
__device__ inline int kv8_parts(int pages, int parts_of) { return pages <= kKv8Whole ? 1 : (pages + parts_of - 1) / parts_of; }

// What is known of the sequences, in shared or global memory: [B] positions before and after the step and pages
// held so far; sums over the sequences before.
struct Kv8Sums {
  int *base, *lens, *held, *free_at, *take_at, *starts, *run_at, *item_at, *part_at, *tile_at;
};
__device__ inline Kv8Sums kv8_sums(const Kv8View& v) {
  return {v.base, v.lens, v.held, v.free_at, v.take_at, v.starts, v.run_at, v.item_at, v.part_at, v.tile_at};
}

// Entries first, first + stride, ... of everything that a step's kernels read: runs, items; the caller's copies.
__device__ __forceinline__ void kv8_fill(const Kv8View& v, const Kv8Sums& s, const Kv8Head& h, int first, int stride, int* pos_out,
                                         int* slot_out, int* tables_out) {
  if (pos_out || slot_out)
    for (int t = first; t < h.rows; t += stride) {
      const int b = find(s.starts, v.B, t), p = s.base[b] + t - s.starts[b];
      if (pos_out) pos_out[t] = p;
      if (slot_out) slot_out[t] = v.table[(size_t)b * v.W + p / kKv8Block] * kKv8Block + p % kKv8Block;
    }
  for (int i = first; i < h.runs; i += stride) {
    const int b = find(s.run_at, v.B, i), have = s.base[b], page = have / kKv8Block + i - s.run_at[b];
    const int p0 = max(have, page * kKv8Block), p1 = min(s.lens[b], (page + 1) * kKv8Block);
    v.runs[i] = {s.starts[b] + p0 - have, v.table[(size_t)b * v.W + page] * kKv8Block + p0 % kKv8Block, p1 - p0, 0};
  }
  for (int i = first; i < h.items; i += stride) {
    const int b = find(s.item_at, v.B, i), have = s.base[b], add = s.lens[b] - have;
    const int parts = kv8_parts(kv8_pages(s.lens[b]), h.parts_of), k = i - s.item_at[b];
    const int unit = parts == 1 ? k : k / parts, part = k - unit * parts, rows = kv8_unit_rows(v, add);
    Kv8Item e{};
    e.seq = b;
    e.t = s.starts[b] + unit * rows;
    e.n = min(rows, add - unit * rows);
    e.pos = have + unit * rows;
    e.wide = add > v.unit_rows;
    const int pages = kv8_pages(e.pos + e.n), each = parts == 1 ? pages : (pages + parts - 1) / parts;
    e.page0 = min(part * each, pages);
    e.pages = min(each, pages - e.page0);
    e.part = part;
    e.parts = parts;
    e.slot = parts > 1 ? s.part_at[b] + unit * parts : -1;
    v.items[i] = e;
  }
  for (int i = first; i < h.tiles; i += stride) {
    const int b = find(s.tile_at, v.B, i), have = s.base[b], add = s.lens[b] - have;
    // the longest first
    v.tiles[i] = {b, s.starts[b], add, have, kv8_tiles(v, add) - 1 - (i - s.tile_at[b]), {}};
  }
  if (tables_out) {
    const size_t n = (size_t)v.B * v.W;
    for (size_t i = first; i < n; i += stride) tables_out[i] = v.table[i];
  }
}

// Pages and sums of a step from have[b] and add[b].  Pages beyond a sequence's need go back to the stack in
// the order of the sequences, then they are taken from its top in that order.  `fill`: the lists, too.
// kShared: v.B <= kPlanShared and one thread a sequence.
template <bool kShared>
__global__ __launch_bounds__(kPlanThreads) void k_kv8_plan(Kv8View v, const int* __restrict__ have,
                                                           const int* __restrict__ add, int rows, int* __restrict__ starts_out,
                                                           int* __restrict__ pos_out, int* __restrict__ slot_out,
                                                           int* __restrict__ tables_out, bool fill) {
  __shared__ int part[kPlanThreads / 64][7];
  __shared__ unsigned long long sums[kPlanThreads / 64][5];
  __shared__ int worsts[kPlanThreads / 64];
  __shared__ int store[kShared ? 10 : 1][kShared ? kPlanShared : 1];
  const int tid = threadIdx.x, threads = blockDim.x;
  Kv8Sums s = kv8_sums(v);
  if constexpr (kShared) s = {store[0], store[1], store[2], store[3], store[4], store[5], store[6], store[7], store[8], store[9]};
  Kv8Head head = *v.head;
  unsigned long long x_sum[5] = {};            // rows, pages, pages of all units and of those outside tiles, tiles and
                                               // units outside
  int worst = KV8_OK, mine[3] = {};
  for (int b = tid; b < v.B; b += threads) {
    const int h = have[b], a = add[b], had = kShared ? v.held[b] : 0;
    if (h < 0 || a < 0) worst = max(worst, (int)KV8_BAD_LENGTH);
    else if ((long long)h + a > v.max_len) worst = max(worst, (int)KV8_TOO_LONG);
    else {
      const int need = kv8_pages(h + a);
      const unsigned long long w = (unsigned long long)kv8_units(v, a) * need;
      x_sum[0] += a;
      x_sum[1] += need;
      x_sum[2] += w;
      x_sum[3] += a > v.unit_rows ? 0 : w;
      x_sum[4] += a > v.unit_rows ? kv8_tiles(v, a) : a > 0;
    }
    if constexpr (kShared) { mine[0] = h; mine[1] = a; mine[2] = had; }
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
#pragma unroll
    for (int k = 0; k < 5; k++) x_sum[k] += __shfl_xor(x_sum[k], d);
    worst = max(worst, __shfl_xor(worst, d));
  }
  if ((tid & 63) == 0) {
#pragma unroll
    for (int k = 0; k < 5; k++) sums[tid >> 6][k] = x_sum[k];
    worsts[tid >> 6] = worst;
  }
  __syncthreads();
  unsigned long long adds = 0, needs = 0, work = 0, work_few = 0, tiles = 0;
  int bad = KV8_OK;
  for (int w = 0; w < threads >> 6; w++) {
    adds += sums[w][0];
    needs += sums[w][1];
    work += sums[w][2];
    work_few += sums[w][3];
    tiles += sums[w][4];
    bad = max(bad, worsts[w]);
  }
  const int free0 = head.free_pages;
  head.status = bad ? bad : adds > (unsigned long long)rows ? KV8_ROWS : needs > (unsigned long long)v.pages ? KV8_PAGES : KV8_OK;
  if (head.status) {
    head.rows = head.runs = head.items = head.tiles = 0;
    for (int b = tid; b <= v.B; b += threads) {
      v.starts[b] = 0;
      if (starts_out) starts_out[b] = 0;
    }
    if (tid == 0) *v.head = head;
    if (fill) kv8_fill(v, s, head, tid, threads, nullptr, nullptr, tables_out);
    return;
  }
  // a unit's pages are shared where there are too few units to fill the GPU
  const bool in_tiles = tiles * v.KVH >= kKv8MinTiles;
  if (in_tiles) work = work_few;
  const unsigned long long share = work + v.items_aim - 1;
  const int each = share < 0x100000000ull ? (int)((uint32_t)share / (uint32_t)v.items_aim) : (int)(share / v.items_aim);
  head.parts_of = max(max(kKv8MinPart, (each + kKv8MoreItems - 1) / kKv8MoreItems), min(each, kKv8MaxPart));
  int sum[7] = {};
  for (int b0 = 0; b0 < v.B; b0 += threads) {
    const int b = b0 + tid;
    int x[7] = {}, own[7] = {}, total[7];
    if (b < v.B) {
      const int h = kShared ? mine[0] : have[b], a = kShared ? mine[1] : add[b], had = kShared ? mine[2] : v.held[b];
      const int need = kv8_pages(h + a), nt = in_tiles ? kv8_tiles(v, a) : 0;
      const int u = nt ? 0 : kv8_units(v, a), parts = kv8_parts(need, head.parts_of);
      v.base[b] = h;
      v.lens[b] = h + a;
      if constexpr (kShared) {
        s.base[b] = h;
        s.lens[b] = h + a;
        s.held[b] = had;
        v.held[b] = need;
      }
      own[0] = max(had - need, 0);
      own[1] = max(need - had, 0);
      own[2] = a;
      own[3] = a ? need - h / kKv8Block : 0;
      own[4] = u * parts;
      own[5] = parts > 1 ? u * parts : 0;
      own[6] = nt;
    }
#pragma unroll
    for (int k = 0; k < 7; k++) x[k] = own[k];
    wg_scan<7>(x, total, part);
#pragma unroll
    for (int k = 0; k < 7; k++) {
      x[k] += sum[k] - own[k];
      sum[k] += total[k];
    }
    if (b < v.B) {
      s.free_at[b] = x[0];
      s.take_at[b] = x[1];
      s.starts[b] = x[2];
      s.run_at[b] = x[3];
      s.item_at[b] = x[4];
      s.part_at[b] = x[5];
      s.tile_at[b] = x[6];
      if (starts_out) starts_out[b] = x[2];
      if (kShared && !fill) { v.starts[b] = x[2]; v.run_at[b] = x[3]; v.item_at[b] = x[4]; v.part_at[b] = x[5]; v.tile_at[b] = x[6]; }
    }
  }
  head.rows = sum[2];
  head.free_pages = free0 + sum[0] - sum[1];
  head.runs = sum[3];
  head.items = sum[4];
  head.tiles = sum[6];
  if (tid == 0) {
    if (starts_out) starts_out[v.B] = sum[2];
    *v.head = head;
  }
  __syncthreads();
  if (sum[0]) {
    for (int i = tid; i < sum[0]; i += threads) {
      const int b = find(s.free_at, v.B, i);
      int* e = v.table + (size_t)b * v.W + kv8_pages(s.lens[b]) + i - s.free_at[b];
      v.stack[free0 + i] = *e;
      *e = -1;
    }
    __syncthreads();
  }
  if (sum[1]) {
    const int top = free0 + sum[0];
    for (int i = tid; i < sum[1]; i += threads) {
      const int b = find(s.take_at, v.B, i);
      v.table[(size_t)b * v.W + s.held[b] + i - s.take_at[b]] = v.stack[top - 1 - i];
    }
    __syncthreads();
  }
  if constexpr (!kShared)
    for (int b = tid; b < v.B; b += threads) v.held[b] = kv8_pages(s.lens[b]);
  if (fill) kv8_fill(v, s, head, tid, threads, pos_out, slot_out, tables_out);
}

__global__ __launch_bounds__(256) void k_kv8_fill(Kv8View v, int* __restrict__ pos_out, int* __restrict__ slot_out,
                                                  int* __restrict__ tables_out) {
  kv8_fill(v, kv8_sums(v), *v.head, blockIdx.x * 256 + threadIdx.x, gridDim.x * 256, pos_out, slot_out, tables_out);
}

}  // namespace q4
