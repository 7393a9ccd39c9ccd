// kv8_fork.h -- sequences that become the beginnings of others: pages shared, last pages copied, pages given back.
//
// All sequences change at once, from the tables as they were: `next` holds the tables that come of it.  How many sequences hold a page
// afterwards is counted page by page, so that no order of the work shows in what comes of it; the free pages are then those that
// nobody holds, and lie on the stack in the order of their numbers.  A last page that is not whole, which its sequence goes on writing
// to, belongs to one alone: v.first() finds who keeps it (-1: nobody, as it is another one's whole page).
// Four launches, each of which needs what all workgroups of the one before have written:
//   count   next tables, holders of a page, the first whose last page it is
//   weigh   free pages of each kKv8Chunk; who needs a copy (one workgroup, in the order of the sequences)
//   commit  tables, holders, the stack; nothing, where the arguments or the pages do not do
//   copy    the last pages' codes and scales, in every layer
// Of a small cache, the first three are one launch of one workgroup.
#pragma once
#include "kv8_plan.h"

namespace q4 {

constexpr int kForkThreads = 256;

__global__ __launch_bounds__(kForkThreads) void k_kv8_fork_count(Kv8View v, Kv8ForkView f, const int* __restrict__ from, const int* __restrict__ keep) {
  for (int b = blockIdx.y; b < v.B; b += gridDim.y) {
    const int n = keep[b];
    if (n == 0) continue;
    const int source = from[b];
    if (n < 0 || source < 0 || source >= v.B || n > v.lens[source]) {
      if (blockIdx.x == 0 && threadIdx.x == 0) atomicMax(&f.fork->bad, n < 0 ? (int)KV8_BAD_LENGTH : (int)KV8_FORK_SOURCE);
      continue;
    }
    const int need = kv8_pages(n);
    for (int j = blockIdx.x * kForkThreads + threadIdx.x; j < need; j += gridDim.x * kForkThreads) {
      const int page = v.table[(size_t)source * v.W + j];
      f.next[(size_t)b * v.W + j] = page;
      atomicAdd(v.count() + page, 1);
      atomicMin(v.first() + page, j < n / kKv8Block ? -1 : b);
    }
  }
}

// The sum over a workgroup, for all of its threads; `store`: one for each wave.
__device__ inline int kv8_block_sum(int x, int* store) {
  const int tid = threadIdx.x, waves = blockDim.x >> 6;
  x = (int)kv8_wave_sums((uint32_t)x);
  __syncthreads();
  if ((tid & 63) == 63) store[tid >> 6] = x;
  __syncthreads();
  x = 0;
  for (int w = 0; w < waves; w++) x += store[w];
  return x;
}

__global__ __launch_bounds__(kKv8Chunk) void k_kv8_fork_weigh(Kv8View v, Kv8ForkView f, const int* __restrict__ keep) {
  __shared__ int store[kKv8Chunk / 64];
  __shared__ uint64_t all;
  const int tid = threadIdx.x, lane = tid & 63;
  if (blockIdx.x) {                            // a chunk of pages
    const int c = blockIdx.x - 1;
    const int64_t page = (int64_t)c * kKv8Chunk + tid;
    const int n = kv8_block_sum(page < v.pages && kv8_peek(v.count() + page) == 0, store);
    if (tid == 0) f.chunk[c] = n;
    return;
  }
  const int bad = kv8_peek(&f.fork->bad);
  if (tid == 0) all = 0;
  __syncthreads();
  int copies = 0;
  uint64_t entries = 0;
  for (int b0 = 0; b0 < v.B && !bad; b0 += kKv8Chunk) {
    const int b = b0 + tid, n = b < v.B ? keep[b] : 0;
    int page = 0;
    bool copy = false;
    if (n % kKv8Block) {
      page = f.next[(size_t)b * v.W + n / kKv8Block];
      copy = kv8_peek(v.first() + page) != b;
    }
    entries += kv8_pages(n);
    const uint64_t ballot = __builtin_amdgcn_ballot_w64(copy);
    __syncthreads();
    if (lane == 0) store[tid >> 6] = __builtin_popcountll(ballot);
    __syncthreads();
    for (int w = 0; w < kKv8Chunk / 64; w++) {
      if (w == tid >> 6 && copy) {
        f.copies[copies + __builtin_popcountll(ballot & ((1ull << lane) - 1))] = {b, page};
        atomicSub(v.count() + page, 1);          // others hold it, still
      }
      copies += store[w];
    }
  }
  entries = kv8_wave_sum(entries);
  if (lane == 0) atomicAdd((unsigned long long*)&all, (unsigned long long)entries);
  __syncthreads();
  if (tid == 0) *f.fork = {0, bad, copies, all};
}

// Workgroup c: pages of chunk c, and its share of the tables.
__global__ __launch_bounds__(kKv8Chunk) void k_kv8_fork_commit(Kv8View v, Kv8ForkView f, const int* __restrict__ keep, int* __restrict__ tables_out) {
  __shared__ int store[kKv8Chunk / 64];
  const int tid = threadIdx.x, lane = tid & 63, chunks = (v.pages + kKv8Chunk - 1) / kKv8Chunk, c = blockIdx.x;
  const Kv8Fork w = *f.fork;
  int before = 0, free = 0;
  for (int i = tid; i < chunks; i += kKv8Chunk) {
    const int n = f.chunk[i];
    free += n;
    before += i < c ? n : 0;
  }
  free = kv8_block_sum(free, store);
  before = kv8_block_sum(before, store);
  const int status = w.status ? w.status : w.copies > free ? (int)KV8_FORK_PAGES
                     : w.entries > (uint64_t)kKv8Entries ? (int)KV8_ENTRIES : (int)KV8_OK;
  if (c < chunks) {
    const int64_t page = (int64_t)c * kKv8Chunk + tid;
    const int count = page < v.pages ? v.count()[page] : 1;
    const uint64_t ballot = __builtin_amdgcn_ballot_w64(count == 0);
    __syncthreads();
    if (lane == 0) store[tid >> 6] = __builtin_popcountll(ballot);
    __syncthreads();
    for (int i = 0; i < tid >> 6; i++) before += store[i];
    if (page < v.pages) {
      if (!status) {
        const int at = free - 1 - (before + __builtin_popcountll(ballot & ((1ull << lane) - 1)));
        if (count == 0) v.stack[at] = (int)page;
        // the pages on top become copies
        v.refs()[page] = count ? count : at >= free - w.copies;
      }
      v.count()[page] = 0;
      v.first()[page] = INT32_MAX;
    }
  }
  // (a last page that is copied gets its place from the copies' launch)
  const size_t n = (size_t)v.B * v.W;
  for (size_t i = (size_t)c * kKv8Chunk + tid; i < n; i += (size_t)gridDim.x * kKv8Chunk) {
    const int b = (int)(i / v.W), j = (int)(i - (size_t)b * v.W);
    if (!status) v.table[i] = j < kv8_pages(keep[b]) ? f.next[i] : -1;
    if (tables_out) tables_out[i] = v.table[i];
  }
  for (int64_t b = (int64_t)c * kKv8Chunk + tid; b < v.B && !status; b += (int64_t)gridDim.x * kKv8Chunk) {
    v.base[b] = v.lens[b] = keep[b];
    v.held[b] = kv8_pages(keep[b]);
  }
  if (c == 0 && tid == 0) {
    Kv8Head h = *v.head;
    h.status = status;
    h.rows = h.runs = h.items = h.tiles = h.joint_items = h.joints = 0;
    if (!status) {
      h.free_pages = free - w.copies;
      h.shared = w.entries > (uint64_t)(v.pages - h.free_pages);
    }
    *v.head = h;
  }
}

// Up to this many pages, and entries of all tables with kForkEach more for each sequence, one workgroup counts, weighs and commits: two
// launches less, but what many do at once one after the other.  By one and by many, a call with its copies, us: 4 sequences of 11 entries
// 7.3 and 16.1, of 1,000 13.7 and 15.9, of 2,048 17.0 and 15.8; 64 of 64 11.9 and 16.4, of 128 17.7 and 16.9; 256 of 8 14.4 and 18.0,
// of 16 20.0 and 17.5; 1,000 of 4 30.1 and 25.0.
constexpr int kForkPages = 4 * kPlanThreads, kForkEntries = 6144, kForkEach = 16;

// v.B <= kPlanShared.  A thread has a sequence, and four pages.
__global__ __launch_bounds__(kPlanThreads) void k_kv8_fork_small(Kv8View v, Kv8ForkView f, const int* __restrict__ from,
                                                                 const int* __restrict__ keep, int* __restrict__ tables_out) {
  __shared__ int kept[kPlanShared], source[kPlanShared];
  __shared__ uint32_t store[3][kPlanThreads / 64];
  const int tid = threadIdx.x, n = tid < v.B ? keep[tid] : 0;
  bool other = false;
  if (tid < v.B) {
    const int a = n ? from[tid] : 0;
    other = n > 0 && (a < 0 || a >= v.B || n > v.lens[a < 0 || a >= v.B ? 0 : a]);
    kept[tid] = n;
    source[tid] = a;
  }
  const int bad = __syncthreads_or(other) ? (int)KV8_FORK_SOURCE : __syncthreads_or(n < 0) ? (int)KV8_BAD_LENGTH : (int)KV8_OK;
  const int entries = v.B * v.W;
  for (int i = tid; i < entries && !bad; i += kPlanThreads) {
    const int b = i / v.W, j = i - b * v.W;
    if (j >= kv8_pages(kept[b])) continue;
    const int page = v.table[(size_t)source[b] * v.W + j];
    f.next[i] = page;
    atomicAdd(v.count() + page, 1);
    atomicMin(v.first() + page, j < kept[b] / kKv8Block ? -1 : b);
  }
  __syncthreads();
  int last = 0;
  bool copy = false;
  if (!bad && n % kKv8Block) {
    last = f.next[(size_t)tid * v.W + n / kKv8Block];
    copy = kv8_peek(v.first() + last) != tid;
    if (copy) atomicSub(v.count() + last, 1);            // others hold it, still
  }
  __syncthreads();
  int count[4];
  uint32_t x[3] = {copy, 0, bad ? 0 : (uint32_t)kv8_pages(n)}, all[3];
#pragma unroll
  for (int k = 0; k < 4; k++) {
    count[k] = 4 * tid + k < v.pages ? kv8_peek(v.count() + 4 * tid + k) : 1;
    x[1] += count[k] == 0;
  }
  kv8_block_scan(x, all, store);
  const int copies = (int)all[0], free = (int)all[1];
  const int status = bad ? bad : copies > free ? (int)KV8_FORK_PAGES : (int)KV8_OK;
  if (copy) f.copies[x[0]] = {tid, last};
#pragma unroll
  for (int k = 0; k < 4; k++) {
    const int page = 4 * tid + k;
    if (page >= v.pages) break;
    if (!status) {
      if (!count[k]) v.stack[free - 1 - (int)x[1]] = page;
      v.refs()[page] = count[k] ? count[k] : (int)x[1] < copies;      // the first free ones become copies
    }
    x[1] += count[k] == 0;
    v.count()[page] = 0;
    v.first()[page] = INT32_MAX;
  }
  for (int i = tid; i < entries; i += kPlanThreads) {
    const int b = i / v.W, j = i - b * v.W;
    if (!status) v.table[i] = j < kv8_pages(kept[b]) ? f.next[i] : -1;
    if (tables_out) tables_out[i] = v.table[i];
  }
  if (!status && tid < v.B) {
    v.base[tid] = v.lens[tid] = n;
    v.held[tid] = kv8_pages(n);
  }
  if (tid == 0) {
    *f.fork = {0, status, copies, all[2]};
    Kv8Head h = *v.head;
    h.status = status;
    h.rows = h.runs = h.items = h.tiles = h.joint_items = h.joints = 0;
    if (!status) {
      h.free_pages = free - copies;
      h.shared = all[2] > (uint32_t)(v.pages - h.free_pages);
    }
    *v.head = h;
  }
}

// A kv head of a copied page in a layer, one after the other.
__global__ __launch_bounds__(kForkThreads) void k_kv8_fork_copy(Kv8View v, Kv8ForkView f, const int* __restrict__ keep, int* __restrict__ tables_out) {
  const int tid = threadIdx.x;
  if (v.head->status) return;
  const int copies = f.fork->copies, free = v.head->free_pages;
  const int units = 4 * v.HD, per = v.layers * v.KVH;              // 16 bytes of K and V of a page and kv head
  for (int64_t i = blockIdx.x; i < (int64_t)copies * per; i += gridDim.x) {
    const int k = (int)(i / per), e = (int)(i - (int64_t)k * per), layer = e / v.KVH, g = e - layer * v.KVH;
    const int2 from = f.copies[k];
    const int to = v.stack[free + copies - 1 - k];
    const size_t a = ((size_t)layer * v.pages + from.y) * v.KVH + g, b = ((size_t)layer * v.pages + to) * v.KVH + g;
    const uint4* const x = (const uint4*)v.codes + a * units;
    uint4* const y = (uint4*)v.codes + b * units;
    for (int u = tid; u < units; u += kForkThreads) y[u] = x[u];
    if (tid == 0) {
      v.scales[b] = v.scales[a];
      if (e == 0) {
        const size_t at = (size_t)from.x * v.W + keep[from.x] / kKv8Block;
        v.table[at] = to;
        if (tables_out) tables_out[at] = to;
      }
    }
  }
}

}  // namespace q4
