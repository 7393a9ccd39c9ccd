// kv8_plan.h -- a step's pages, rows and work lists from request lengths, on the GPU.
//
// One workgroup sums over the sequences (pages given back and taken, rows, runs, items); whoever then wants
// the i-th page, row, run or item finds its sequence by bisection of those sums.  So no thread walks through a
// long sequence alone, and the second part is spread over the GPU where there is much of it.
#pragma once
#include "kv8.h"

namespace q4 {

constexpr int kPlanThreads = 1024;

__device__ inline int kv8_pages(int n) { return (n + kKv8Block - 1) / kKv8Block; }

// Inclusive sums of N numbers over the workgroup's threads; total[] receives the sums of all.
template <int N>
__device__ void wg_scan(int (&x)[N], int (&total)[N], int (*part)[N]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int d = 1; d < 64; d <<= 1)
    for (int k = 0; k < N; k++) {
      const int u = __shfl_up(x[k], d);
      if (lane >= d) x[k] += u;
    }
  __syncthreads();                       // `part` of the sums before has been read
  if (lane == 63)
    for (int k = 0; k < N; k++) part[wave][k] = x[k];
  __syncthreads();
  for (int k = 0; k < N; k++) total[k] = 0;
  for (int w = 0; w < kPlanThreads / 64; w++)
    for (int k = 0; k < N; k++) {
      if (w < wave) x[k] += part[w][k];
      total[k] += part[w][k];
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

// Units of sequence b's rows, and the parts of each.
__device__ inline int kv8_units(const Kv8View& v, int add) { return (add + v.unit_rows - 1) / v.unit_rows; }
__device__ inline int kv8_parts(int pages, int parts_of) { return (pages + parts_of - 1) / parts_of; }

// Entries i, i + stride, ... of everything that a step's kernels read: rows, runs, items; the caller's copies.
__device__ inline void kv8_fill(const Kv8View& v, const Kv8Head& h, int first, int stride, int* pos_out, int* slot_out,
                                int* tables_out) {
  for (int t = first; t < h.rows && (pos_out || slot_out); t += stride) {
    const int b = find(v.starts, v.B, t), p = v.base[b] + t - v.starts[b];
    const int s = v.table[(size_t)b * v.W + p / kKv8Block] * kKv8Block + p % kKv8Block;
    if (pos_out) pos_out[t] = p;
    if (slot_out) slot_out[t] = s;
  }
  for (int i = first; i < h.runs; i += stride) {
    const int b = find(v.run_at, v.B, i), have = v.base[b], page = have / kKv8Block + i - v.run_at[b];
    const int p0 = max(have, page * kKv8Block), p1 = min(v.lens[b], (page + 1) * kKv8Block);
    v.runs[i] = {v.starts[b] + p0 - have, v.table[(size_t)b * v.W + page] * kKv8Block + p0 % kKv8Block, p1 - p0, 0};
  }
  for (int i = first; i < h.items; i += stride) {
    const int b = find(v.item_at, v.B, i), have = v.base[b], add = v.lens[b] - have;
    const int parts = kv8_parts(kv8_pages(v.lens[b]), h.parts_of);
    const int unit = (i - v.item_at[b]) / parts, part = (i - v.item_at[b]) % parts;
    Kv8Item e{};
    e.seq = b;
    e.t = v.starts[b] + unit * v.unit_rows;
    e.n = min(v.unit_rows, add - unit * v.unit_rows);
    e.pos = have + unit * v.unit_rows;
    const int pages = kv8_pages(e.pos + e.n), each = (pages + parts - 1) / parts;
    e.page0 = min(part * each, pages);
    e.pages = min(each, pages - e.page0);
    e.part = part;
    e.parts = parts;
    e.slot = parts > 1 ? v.part_at[b] + unit * parts : -1;
    v.items[i] = e;
  }
  if (tables_out) {
    const size_t n = (size_t)v.B * v.W;
    for (size_t i = first; i < n; i += stride) tables_out[i] = v.table[i];
  }
}

// Pages and sums of a step from have[b] and add[b].  Pages beyond a sequence's need go back to the stack in
// the order of the sequences, then they are taken from its top in that order.  `fill`: the lists, too.
__global__ __launch_bounds__(kPlanThreads) void k_kv8_plan(Kv8View v, const int* __restrict__ have,
                                                           const int* __restrict__ add, int rows, int* __restrict__ starts_out,
                                                           int* __restrict__ pos_out, int* __restrict__ slot_out,
                                                           int* __restrict__ tables_out, bool fill) {
  __shared__ int part[kPlanThreads / 64][4];
  __shared__ unsigned long long sums[kPlanThreads / 64][3];
  __shared__ int worsts[kPlanThreads / 64];
  const int tid = threadIdx.x;
  unsigned long long a_sum = 0, n_sum = 0, w_sum = 0;
  int worst = KV8_OK;
  for (int b = tid; b < v.B; b += kPlanThreads) {
    const int h = have[b], a = add[b];
    if (h < 0 || a < 0) worst = max(worst, (int)KV8_BAD_LENGTH);
    else if ((long long)h + a > v.max_len) worst = max(worst, (int)KV8_TOO_LONG);
    else {
      const int need = kv8_pages(h + a);
      a_sum += a;
      n_sum += need;
      w_sum += (unsigned long long)kv8_units(v, a) * need;
    }
  }
  for (int d = 1; d < 64; d <<= 1) {
    a_sum += __shfl_xor(a_sum, d);
    n_sum += __shfl_xor(n_sum, d);
    w_sum += __shfl_xor(w_sum, d);
    worst = max(worst, __shfl_xor(worst, d));
  }
  if ((tid & 63) == 0) {
    sums[tid >> 6][0] = a_sum;
    sums[tid >> 6][1] = n_sum;
    sums[tid >> 6][2] = w_sum;
    worsts[tid >> 6] = worst;
  }
  __syncthreads();
  unsigned long long adds = 0, needs = 0, work = 0;
  int bad = KV8_OK;
  for (int w = 0; w < kPlanThreads / 64; w++) {
    adds += sums[w][0];
    needs += sums[w][1];
    work += sums[w][2];
    bad = max(bad, worsts[w]);
  }
  Kv8Head head = *v.head;
  const int free0 = head.free_pages;
  head.status = bad ? bad : adds > (unsigned long long)rows ? KV8_ROWS : needs > (unsigned long long)v.pages ? KV8_PAGES : KV8_OK;
  if (head.status) {
    head.rows = head.runs = head.items = 0;
    for (int b = tid; b <= v.B; b += kPlanThreads) {
      v.starts[b] = 0;
      if (starts_out) starts_out[b] = 0;
    }
    if (tid == 0) *v.head = head;
    if (fill) kv8_fill(v, head, tid, kPlanThreads, nullptr, nullptr, tables_out);
    return;
  }
  // a unit's pages are shared where there are too few units to fill the GPU
  head.parts_of = (int)max((unsigned long long)kKv8MinPart, (work + v.items_aim - 1) / v.items_aim);
  int sum[4] = {}, more[2] = {};
  for (int b0 = 0; b0 < v.B; b0 += kPlanThreads) {
    const int b = b0 + tid;
    int x[4] = {}, y[2] = {}, total[4], total2[2];
    int own[4] = {}, own2[2] = {};
    if (b < v.B) {
      const int h = have[b], a = add[b], need = kv8_pages(h + a), had = v.held[b], u = kv8_units(v, a);
      const int parts = kv8_parts(need, head.parts_of);
      v.base[b] = h;
      v.lens[b] = h + a;
      own[0] = max(had - need, 0);
      own[1] = max(need - had, 0);
      own[2] = a;
      own[3] = a ? need - h / kKv8Block : 0;
      own2[0] = u * parts;
      own2[1] = parts > 1 ? u * parts : 0;
    }
    for (int k = 0; k < 4; k++) x[k] = own[k];
    for (int k = 0; k < 2; k++) y[k] = own2[k];
    wg_scan<4>(x, total, part);
    wg_scan<2>(y, total2, (int(*)[2])part);
    if (b < v.B) {
      v.free_at[b] = sum[0] + x[0] - own[0];
      v.take_at[b] = sum[1] + x[1] - own[1];
      v.starts[b] = sum[2] + x[2] - own[2];
      if (starts_out) starts_out[b] = sum[2] + x[2] - own[2];
      v.run_at[b] = sum[3] + x[3] - own[3];
      v.item_at[b] = more[0] + y[0] - own2[0];
      v.part_at[b] = more[1] + y[1] - own2[1];
    }
    for (int k = 0; k < 4; k++) sum[k] += total[k];
    for (int k = 0; k < 2; k++) more[k] += total2[k];
  }
  __syncthreads();
  for (int i = tid; i < sum[0]; i += kPlanThreads) {
    const int b = find(v.free_at, v.B, i);
    int* e = v.table + (size_t)b * v.W + kv8_pages(v.lens[b]) + i - v.free_at[b];
    v.stack[free0 + i] = *e;
    *e = -1;
  }
  __syncthreads();
  const int top = free0 + sum[0];
  for (int i = tid; i < sum[1]; i += kPlanThreads) {
    const int b = find(v.take_at, v.B, i);
    v.table[(size_t)b * v.W + v.held[b] + i - v.take_at[b]] = v.stack[top - 1 - i];
  }
  __syncthreads();
  for (int b = tid; b < v.B; b += kPlanThreads) v.held[b] = kv8_pages(v.lens[b]);
  head.rows = sum[2];
  head.free_pages = top - sum[1];
  head.runs = sum[3];
  head.items = more[0];
  if (tid == 0) {
    v.starts[v.B] = sum[2];
    if (starts_out) starts_out[v.B] = sum[2];
    *v.head = head;
  }
  if (fill) kv8_fill(v, head, tid, kPlanThreads, pos_out, slot_out, tables_out);
}

__global__ __launch_bounds__(256) void k_kv8_fill(Kv8View v, int* __restrict__ pos_out, int* __restrict__ slot_out,
                                                  int* __restrict__ tables_out) {
  kv8_fill(v, *v.head, blockIdx.x * 256 + threadIdx.x, gridDim.x * 256, pos_out, slot_out, tables_out);
}

}  // namespace q4
