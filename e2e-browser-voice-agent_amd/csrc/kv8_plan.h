// kv8_plan.h -- a step's pages, rows and work lists from request lengths, on the GPU.
//
// One workgroup sums over the sequences (pages given back and taken, rows, runs, items, tiles); whoever then
// wants the i-th page, row, run or item finds its sequence by bisection of those sums.  So no thread walks through a
// long sequence alone, and the lists can be spread over the GPU where there is much of them.
// Nothing but latency bounds it: a chain of loads, sums and bisections, and the fetches of code that runs once.  So
// the code is short (a thread forms its sequence's numbers, then a wave takes each sum), sums over a wave stay in
// registers, those over up to kPlanShared sequences in shared memory, and all lists are filled in one loop.  (Which of the ten
// arrays a wave takes is chosen as it runs: the compiler keeps their addresses in 88 bytes of scratch memory a lane, and
// reaches the arrays by flat accesses.)  A launch with
// all of the caller's arrays: 32 sequences 6.6 us, 48 with 2,171 rows 9.8, 1,024 with 15,454 rows 15.6 (two launches); with
// every sum unrolled through shared memory 7.7, 15.8 and 24.
#pragma once
#include <type_traits>

#include "kv8.h"

namespace q4 {

constexpr int kPlanThreads = 1024;
constexpr int kPlanShared = 1024;
constexpr int kScanAtOnce = 4;      // chunks of 64 sequences (8: the same; 1 where there is one)

__device__ inline int kv8_pages(int n) { return (n + kKv8Block - 1) / kKv8Block; }

// Inclusive sums over a wave, in registers.
template <int kCtrl, int kRows>
__device__ __forceinline__ uint32_t kv8_lane_below(uint32_t x) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, kCtrl, kRows, 0xf, false);
}
__device__ __forceinline__ uint32_t kv8_wave_sums(uint32_t x) {
  x += kv8_lane_below<0x111, 0xf>(x);       // from 1, 2, 4, 8 lanes below in a row of 16
  x += kv8_lane_below<0x112, 0xf>(x);
  x += kv8_lane_below<0x114, 0xf>(x);
  x += kv8_lane_below<0x118, 0xf>(x);
  x += kv8_lane_below<0x142, 0xa>(x);       // from lanes 15 and 47, into the rows above
  x += kv8_lane_below<0x143, 0xc>(x);       // from lane 31
  return x;
}
// The sum over a wave.
__device__ __forceinline__ uint64_t kv8_wave_sum(uint64_t x) {
  // 22 bits of each lane at a time: no sum of 64 passes 32 bits
  uint64_t all = 0;
#pragma unroll 1
  for (int i = 0; i < 66; i += 22)
    all += (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)kv8_wave_sums((uint32_t)(x >> i) & 0x3fffff), 63) << i;
  return all;
}

// Sums over the threads before, and over all; `store` is shared memory.  All of kPlanThreads threads call it.
template <int K>
__device__ inline void kv8_block_scan(uint32_t (&x)[K], uint32_t (&all)[K], uint32_t (*store)[kPlanThreads / 64]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t before[K];
#pragma unroll
  for (int k = 0; k < K; k++) {
    const uint32_t y = kv8_wave_sums(x[k]);
    if (lane == 63) store[k][wave] = y;
    before[k] = y - x[k];
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < K; k++) {
    all[k] = 0;
    for (int w = 0; w < kPlanThreads / 64; w++) {
      const uint32_t y = store[k][w];
      before[k] += w < wave ? y : 0;
      all[k] += y;
    }
    x[k] = before[k];
  }
  __syncthreads();
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
  return (int)(((uint32_t)add + r - 1) / (uint32_t)r);
}
__device__ inline int kv8_tiles(const Kv8View& v, int add) {
  return add > v.unit_rows ? (int)(((int64_t)add * (v.H / v.KVH) + kKv8TileRows - 1) / kKv8TileRows) : 0;
}
__device__ inline int kv8_parts(int pages, int parts_of) {
  return pages <= kKv8Whole ? 1 : (int)((uint32_t)(pages + parts_of - 1) / (uint32_t)parts_of);
}

// What is known of the sequences, in shared or global memory: [B] positions before and after the step and pages
// held so far; sums over the sequences before.
struct Kv8Sums {
  int *base, *lens, *held, *free_at, *take_at, *starts, *run_at, *item_at, *part_at, *tile_at;
};
__device__ inline Kv8Sums kv8_sums(const Kv8View& v) {
  return {v.base, v.lens, v.held, v.free_at, v.take_at, v.starts, v.run_at, v.item_at, v.part_at, v.tile_at};
}

// Entries first, first + stride, ... of everything that a step's kernels read: runs, items, tiles; the caller's copies.
// All of them in one loop, so that no kind waits for another.
__device__ __forceinline__ void kv8_fill(const Kv8View& v, const Kv8Sums& s, const Kv8Head& h, int first, int stride, int* pos_out,
                                         int* slot_out, int* tables_out) {
  if (tables_out) {
    const size_t n = (size_t)v.B * v.W;
    for (size_t i = first; i < n; i += stride) tables_out[i] = v.table[i];
  }
  const int64_t rows_end = pos_out || slot_out ? h.rows : 0, runs_end = rows_end + h.runs, items_end = runs_end + h.items,
                end = items_end + h.tiles;
  for (int64_t j = first; j < end; j += stride) {
    const int kind = j < rows_end ? 0 : j < runs_end ? 1 : j < items_end ? 2 : 3;
    const int i = (int)(j - (kind == 0 ? 0 : kind == 1 ? rows_end : kind == 2 ? runs_end : items_end));
    const int* const at = kind == 0 ? s.starts : kind == 1 ? s.run_at : kind == 2 ? s.item_at : s.tile_at;
    const int b = find(at, v.B, i), k = i - at[b], have = s.base[b], len = s.lens[b], add = len - have, t = s.starts[b];
    const int* const table = v.table + (size_t)b * v.W;
    if (kind < 2) {
      const int page = kind ? have / kKv8Block + k : (have + k) / kKv8Block;
      const int p0 = kind ? max(have, page * kKv8Block) : have + k;
      const int slot = table[page] * kKv8Block + p0 % kKv8Block;
      if (kind) {
        v.runs[i] = {t + p0 - have, slot, min(len, (page + 1) * kKv8Block) - p0, 0};
      } else {
        if (pos_out) pos_out[i] = p0;
        if (slot_out) slot_out[i] = slot;
      }
    } else if (kind == 2) {
      const int parts = kv8_parts(kv8_pages(len), h.parts_of), rows = kv8_unit_rows(v, add);
      const int unit = parts == 1 ? k : (int)((uint32_t)k / (uint32_t)parts), part = k - unit * parts;
      Kv8Item e{};
      e.seq = b;
      e.t = t + unit * rows;
      e.n = min(rows, add - unit * rows);
      e.pos = have + unit * rows;
      e.wide = add > v.unit_rows;
      const int pages = kv8_pages(e.pos + e.n), each = parts == 1 ? pages : (int)((uint32_t)(pages + parts - 1) / (uint32_t)parts);
      e.page0 = min(part * each, pages);
      e.pages = min(each, pages - e.page0);
      e.part = part;
      e.parts = parts;
      e.slot = parts > 1 ? s.part_at[b] + unit * parts : -1;
      v.items[i] = e;
    } else {
      v.tiles[i] = {b, t, add, have, kv8_tiles(v, add) - 1 - k, {}};        // the longest first
    }
  }
}

// Which pages a step gives back while some belong to several sequences: those that all of their holders give up, at the place of
// the first of them.  Entry i of the `gone` ones (sequences in order, their pages in order; at[b] counts those before) is in first()
// and count() until kv8_shared_done().
// One workgroup goes over them, three times and with a bisection each: 6 to 12 ns an entry.  Half of 128 sequences behind 14,500 positions
// end in 0.27 ms, half of 1,024 behind 8,000 in 0.76, half of 64 behind 131,072 in 1.05; a plan by which none ends takes 9 to 14 us.
// Both are calls, with what they need by value: within the kernel they cost every plan 0.25 us of 6.0, so 0.1.
struct Kv8Gone {
  int *table, *refs, *count, *first;
  const int* at;
  int B, W, gone;
};
__device__ inline int kv8_peek(const int* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

// Pages given back, or less than 0 where the step's rows would lie in a page that others keep (-KV8_SHARED) or take more than there
// are free (-KV8_PAGES).
__device__ __attribute__((noinline)) int kv8_shared_gone(Kv8Gone g, const int* have, const int* add, const int* held, int most) {
  const int tid = threadIdx.x, threads = blockDim.x;
  auto page_of = [&](int i) {
    const int b = find(g.at, g.B, i);
    return g.table[(size_t)b * g.W + (kv8_pages(have[b] + add[b]) + i - g.at[b])];
  };
  for (int i = tid; i < g.gone; i += threads) {
    const int page = page_of(i);
    atomicAdd(g.count + page, 1);
    atomicMin(g.first + page, i);
  }
  __syncthreads();
  int n = 0;
  for (int i = tid; i < (g.gone + threads - 1) / threads * threads; i += threads) {
    bool mine = false;
    if (i < g.gone) {
      const int page = page_of(i);
      mine = kv8_peek(g.first + page) == i && kv8_peek(g.count + page) == g.refs[page];
    }
    n += __syncthreads_count(mine);
  }
  bool others = false;
  for (int b = tid; b < g.B; b += threads) {
    const int end = min(held[b], kv8_pages(have[b] + add[b]));
    for (int j = add[b] ? have[b] / kKv8Block : end; j < end; j++) {
      const int page = g.table[(size_t)b * g.W + j];
      others |= g.refs[page] - kv8_peek(g.count + page) > 1;
    }
  }
  const int status = __syncthreads_or(others) ? KV8_SHARED : most < -n ? KV8_PAGES : KV8_OK;
  if (!status) return n;
  for (int i = tid; i < g.gone; i += threads) {
    const int page = page_of(i);
    g.count[page] = 0;
    g.first[page] = INT32_MAX;
  }
  return -status;
}

// Gives the pages back: onto the stack from `top` on.  lens: positions after the step.
__device__ __attribute__((noinline)) void kv8_shared_done(Kv8Gone g, const int* lens, int* top) {
  const int tid = threadIdx.x, threads = blockDim.x, lane = tid & 63, waves = threads >> 6;
  __shared__ int counts[kPlanThreads / 64];
  auto place = [&](int i) {
    const int b = find(g.at, g.B, i);
    return g.table + (size_t)b * g.W + kv8_pages(lens[b]) + i - g.at[b];
  };
  for (int i0 = 0; i0 < g.gone; i0 += threads) {
    const int i = i0 + tid, page = i < g.gone ? *place(i) : 0;
    const bool mine = i < g.gone && kv8_peek(g.first + page) == i && kv8_peek(g.count + page) == g.refs[page];
    const uint64_t ballot = __builtin_amdgcn_ballot_w64(mine);
    if (lane == 0) counts[tid >> 6] = __builtin_popcountll(ballot);
    __syncthreads();
    for (int w = 0; w < waves; w++) {
      if (w == tid >> 6 && mine) top[__builtin_popcountll(ballot & ((1ull << lane) - 1))] = page;
      top += counts[w];
    }
    __syncthreads();
  }
  for (int i = tid; i < g.gone; i += threads) {
    int* const e = place(i);
    const int page = *e;
    *e = -1;
    if (kv8_peek(g.first + page) == i) {       // nobody else's, before and after
      g.refs[page] -= kv8_peek(g.count + page);
      g.count[page] = 0;
      __hip_atomic_store(g.first + page, INT32_MAX, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
  }
  __syncthreads();
}

// Pages and sums of a step from have[b] and add[b].  Pages beyond a sequence's need go back to the stack in
// the order of the sequences, then they are taken from its top in that order.  `fill`: the lists, too.
// kShared: v.B <= kPlanShared and blockDim.x.
template <bool kShared>
__global__ __launch_bounds__(kPlanThreads) void k_kv8_plan(Kv8View v, const int* __restrict__ have,
                                                           const int* __restrict__ add, int rows, int* __restrict__ starts_out,
                                                           int* __restrict__ pos_out, int* __restrict__ slot_out,
                                                           int* __restrict__ tables_out, bool fill) {
  // of each thread's sequences: rows, pages, pages of all units and of those outside tiles, tiles and units outside; bad lengths
  __shared__ uint64_t share[6][kPlanThreads];
  __shared__ uint64_t sums[6];                 // of all
  __shared__ int total[7];                     // of free_at .. tile_at
  __shared__ int store[kShared ? 10 : 1][kShared ? kPlanShared : 1];
  const int tid = threadIdx.x, threads = blockDim.x, lane = tid & 63, waves = threads >> 6;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  Kv8Sums s = kv8_sums(v);
  if constexpr (kShared) s = {store[0], store[1], store[2], store[3], store[4], store[5], store[6], store[7], store[8], store[9]};
  Kv8Head head = *v.head;
  uint64_t mine[6] = {};
  for (int b = tid; b < v.B; b += threads) {
    const int h = have[b], a = add[b], had = v.held[b];
    const bool bad = (h | a) < 0, longer = !bad && (uint32_t)h + (uint32_t)a > (uint32_t)v.max_len;
    mine[5] += bad ? 1 : longer ? (uint64_t)1 << 32 : 0;
    if (bad || longer) continue;               // and no sum is looked at
    const int need = kv8_pages(h + a);
    const uint64_t pages = (uint64_t)kv8_units(v, a) * need;
    const bool many = a > v.unit_rows;
    mine[0] += a;
    mine[1] += need;
    mine[2] += pages;
    mine[3] += many ? 0 : pages;
    mine[4] += many ? kv8_tiles(v, a) : a > 0;
    if constexpr (kShared) { s.base[b] = h; s.lens[b] = a; s.held[b] = had; }
    s.free_at[b] = max(had - need, 0);
    s.take_at[b] = max(need - had, 0);
    s.starts[b] = a;
    s.run_at[b] = a ? need - h / kKv8Block : 0;
  }
  const int busy = min((v.B + 63) & ~63, threads);       // threads with a sequence, whole waves
#pragma unroll
  for (int k = 0; k < 6; k++)
    if (tid < busy) share[k][tid] = mine[k];
  __syncthreads();

  // sums over the sequences before, in place, by a wave
  auto scan64 = [&](auto chunks, int kind) {
    constexpr int U = decltype(chunks)::value;      // 64 sequences each, on their way together
    int* const at = kind == 0 ? s.free_at : kind == 1 ? s.take_at : kind == 2 ? s.starts : kind == 3 ? s.run_at : kind == 4 ? s.item_at
                    : kind == 5 ? s.part_at : s.tile_at;
    uint32_t before = 0;
    for (int b0 = 0; b0 < v.B; b0 += 64 * U) {
      uint32_t x[U], y[U];
#pragma unroll
      for (int u = 0; u < U; u++) {
        const int b = b0 + u * 64 + lane;
        x[u] = (uint32_t)at[min(b, v.B - 1)];
        if (b >= v.B) x[u] = 0;
      }
#pragma unroll
      for (int u = 0; u < U; u++) y[u] = kv8_wave_sums(x[u]);
#pragma unroll
      for (int u = 0; u < U; u++) {
        const int b = b0 + u * 64 + lane;
        if (b < v.B) at[b] = (int)(before + y[u] - x[u]);
        before += (uint32_t)__builtin_amdgcn_readlane((int)y[u], 63);
      }
    }
    if (lane == 0) total[kind] = (int)before;
  };
  auto scan = [&](int kind) {
    if (v.B <= 64) scan64(std::integral_constant<int, 1>(), kind);
    else scan64(std::integral_constant<int, kScanAtOnce>(), kind);
  };
  for (int k = wave; k < 10; k += waves) {     // a wave takes a sum at a time
    if (k < 4) {
      scan(k);
    } else {
      uint64_t x = 0;
      for (int i = lane; i < busy; i += 64) x += share[k - 4][i];
      x = kv8_wave_sum(x);
      if (lane == 0) sums[k - 4] = x;
    }
  }
  __syncthreads();
  const int free0 = head.free_pages;
  const uint64_t bad = sums[5];
  head.joint_items = head.joints = 0;
  head.status = bad >> 32 ? KV8_TOO_LONG : bad ? KV8_BAD_LENGTH : sums[0] > (uint64_t)rows ? KV8_ROWS
                : sums[1] <= (uint64_t)(head.shared ? kKv8Entries : v.pages) ? KV8_OK
                : head.shared ? KV8_ENTRIES : KV8_PAGES;
  int freed = total[0];
  if (__builtin_expect(head.shared && !head.status, 0)) {
    freed = kv8_shared_gone({v.table, v.refs(), v.count(), v.first(), s.free_at, v.B, v.W, total[0]}, kShared ? s.base : have,
                            kShared ? s.lens : add, s.held, free0 - total[1]);
    if (freed < 0) head.status = -freed;
  }
  if (head.status) {
    head.rows = head.runs = head.items = head.tiles = 0;
    if (starts_out)
      for (int b = tid; b <= v.B; b += threads) starts_out[b] = 0;
    if (tid == 0) *v.head = head;
    if (fill) kv8_fill(v, s, head, tid, threads, nullptr, nullptr, tables_out);
    return;
  }
  // a unit's pages are shared where there are too few units to fill the GPU
  const bool in_tiles = sums[4] * v.KVH >= kKv8MinTiles;
  const double pages_each = (double)(sums[in_tiles ? 3 : 2] + v.items_aim - 1) * v.aim_inverse;
  const int each = (int)__builtin_fmin(pages_each, 1073741824.0);
  head.parts_of = max(max(kKv8MinPart, (each + kKv8MoreItems - 1) / kKv8MoreItems), min(each, kKv8MaxPart));
  for (int b = tid; b < v.B; b += threads) {
    const int h = kShared ? s.base[b] : have[b], a = kShared ? s.lens[b] : add[b];
    const int tiles = in_tiles ? kv8_tiles(v, a) : 0, parts = kv8_parts(kv8_pages(h + a), head.parts_of);
    const int items = tiles ? 0 : kv8_units(v, a) * parts;
    s.item_at[b] = items;
    s.part_at[b] = parts > 1 ? items : 0;
    s.tile_at[b] = tiles;
    if constexpr (kShared) s.lens[b] = h + a;
    else v.base[b] = h;
    v.lens[b] = h + a;
  }
  __syncthreads();
  for (int k = 4 + wave; k < 7; k += waves) scan(k);
  __syncthreads();
  head.rows = total[2];
  head.free_pages = free0 + freed - total[1];
  const bool shared = head.shared;
  head.shared = shared && sums[1] > (uint64_t)(v.pages - head.free_pages);
  head.runs = total[3];
  head.items = total[4];
  head.tiles = total[6];
  for (int b = tid; b < v.B; b += threads) {
    if constexpr (kShared) v.held[b] = kv8_pages(s.lens[b]);
    if (starts_out) starts_out[b] = s.starts[b];
    if (kShared && (!fill || shared)) v.base[b] = s.base[b];       // shared: for k_kv8_joints
    if (kShared && !fill) {
      v.starts[b] = s.starts[b];
      v.run_at[b] = s.run_at[b];
      v.item_at[b] = s.item_at[b];
      v.part_at[b] = s.part_at[b];
      v.tile_at[b] = s.tile_at[b];
    }
  }
  if (tid == 0) {
    if (starts_out) starts_out[v.B] = head.rows;
    *v.head = head;
  }
  __syncthreads();
  if (__builtin_expect(shared, 0)) {
    kv8_shared_done({v.table, v.refs(), v.count(), v.first(), s.free_at, v.B, v.W, total[0]}, s.lens, v.stack + free0);
  } else if (total[0]) {
    for (int i = tid; i < total[0]; i += threads) {
      const int b = find(s.free_at, v.B, i);
      int* e = v.table + (size_t)b * v.W + kv8_pages(s.lens[b]) + i - s.free_at[b];
      v.stack[free0 + i] = *e;
      *e = -1;
    }
    __syncthreads();
  }
  if (total[1]) {
    const int top = free0 + freed;
    for (int i = tid; i < total[1]; i += threads) {
      const int b = find(s.take_at, v.B, i), page = v.stack[top - 1 - i];
      v.table[(size_t)b * v.W + s.held[b] + i - s.take_at[b]] = page;
      if (shared) v.refs()[page] = 1;
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
