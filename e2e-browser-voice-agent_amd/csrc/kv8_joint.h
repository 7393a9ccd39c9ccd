// kv8_joint.h -- the lists of a step whose sequences begin with the same pages: one pass over these for all of them.
//
// Sequences that share pages share them from the first one on, as they come of forks: if two tables have the same page at one place, they
// have the same pages before it.  So a group is the units (sequences that add up to a unit's rows) with the same first page, and
// what they have in common with the first of them is found by search and not by comparing.  The group's rows of attention, unit
// after unit, are joints of 32 (kv8.h).  Their pages, like a long unit's, may be shared among workgroups.
// One workgroup does it in one launch behind the plan, once for all layers (32 sequences 14 us, 128 with joints in 256 parts 25); the
// members' order is the sequences', whatever the atomics' order was.  Where nothing is shared, or too little, there is no such list, and
// attention takes the plan's.
#pragma once
#include "kv8_plan.h"

namespace q4 {

constexpr int kJointThreads = kPlanThreads;
// A group has at least so many pages in common.
constexpr int kJointPages = 8;

constexpr int kJointArrays = 11;

// kShared: v.B <= kPlanShared, and the arrays are in shared memory, else in `scratch`, [kJointArrays][B].
template <bool kShared>
__global__ __launch_bounds__(kJointThreads) void k_kv8_joints(Kv8View v, Kv8JointView jv, int* scratch) {
  __shared__ int room[kShared ? kJointArrays : 1][kShared ? kPlanShared : 1];
  __shared__ uint32_t store[4][kPlanThreads / 64];
  __shared__ int4 chunk[kJointThreads / 4], added[kJointThreads / 4];
  __shared__ unsigned long long pages_all;
  __shared__ int joints_all, most_parts, most_own;      // parts of a group's pages, of a member's own
  __shared__ unsigned long long saved;                  // pages that the groups' members need not pass over by themselves
  const Kv8Head head = *v.head;
  if (!head.shared || !head.rows) return;
  const int tid = threadIdx.x, lane = tid & 63, G = v.H / v.KVH, B = v.B;
  auto array = [&](int k) { return kShared ? room[kShared ? k : 0] : scratch + (size_t)k * B; };
  // of a sequence: the first one of its group, -1 for none; rows of the members before; its first row of the step
  int *const lead = array(0), *const before_of = array(1), *const start = array(2);
  // of a group, at its first sequence: pages in common, members, their rows; joints of the groups before
  int *const common = array(3), *const count = array(4), *const total = array(5), *const joint_at = array(6);
  // (what atomics have written in global memory lies in the L2)
  auto in = [](const int* p) { return kShared ? *p : kv8_peek(p); };
  // sums over the sequences before: items and slots of joints, of units
  int *const common_at = array(7), *const common_slot = array(8), *const item_at = array(9), *const slot_at = array(10);
  // the step's lengths as the plan has taken them: the caller's arrays may be those that it has written to since
  auto have = [&](int b) { return v.base[b]; };
  auto add = [&](int b) { return v.lens[b] - v.base[b]; };
  auto page0 = [&](int b) { return v.table[(size_t)b * v.W]; };
  // what a sequence that adds a unit may have in common with others: pages before its rows
  auto mine = [&](int b) { return add(b) > 0 && add(b) <= v.unit_rows ? have(b) / kKv8Block : 0; };
  for (int b = tid; b < B; b += kJointThreads)
    if (mine(b) >= kJointPages) atomicMin(v.first() + page0(b), b);
  __syncthreads();
  for (int b = tid; b < B; b += kJointThreads) {
    const int n = mine(b);
    lead[b] = n >= kJointPages ? kv8_peek(v.first() + page0(b)) : -1;
    common[b] = n;
    count[b] = total[b] = 0;
  }
  if (tid == 0) pages_all = saved = joints_all = most_parts = most_own = 0;
  __syncthreads();
  for (int b = tid; b < B; b += kJointThreads)
    if (lead[b] == b) v.first()[page0(b)] = INT32_MAX;
  // pages in common with the group's first: 16 lanes try as many places of what is left at once
  for (int b = tid >> 4; b < B; b += kJointThreads / 16) {
    const int a = lead[b];
    if (a < 0 || a == b) continue;
    const int *const x = v.table + (size_t)a * v.W, *const y = v.table + (size_t)b * v.W;
    int lo = 1, hi = min(mine(a), mine(b));
    while (lo < hi) {
      const int step = (hi - lo + 15) >> 4, at = lo + ((lane & 15) + 1) * step - 1;
      const bool same = at < hi && x[at] == y[at];
      const int n = __builtin_ctz(~(uint32_t)(__builtin_amdgcn_ballot_w64(same) >> (lane & 48) & 0xffff));
      hi = min(hi, lo + (n + 1) * step - 1);
      lo += n * step;
    }
    if ((lane & 15) == 0) atomicMin(&common[a], lo);
  }
  // members in the order of the sequences, 1,024 at a time
  for (int b0 = 0; b0 < B; b0 += kJointThreads) {
    const int b = b0 + tid, a = b < B ? lead[b] : -1, n = a >= 0 ? add(b) : 0;
    ((int*)chunk)[tid] = a;
    ((int*)added)[tid] = n;
    __syncthreads();
    int before = 0;
    if (a >= 0) {
      before = in(total + a);
      for (int i = 0; 4 * i < tid; i++) {
        const int4 c = chunk[i], m = added[i];
        before += (c.x == a ? m.x : 0) + (c.y == a && 4 * i + 1 < tid ? m.y : 0) + (c.z == a && 4 * i + 2 < tid ? m.z : 0) +
                  (c.w == a && 4 * i + 3 < tid ? m.w : 0);
      }
    }
    __syncthreads();
    if (b < B) before_of[b] = before;
    if (a >= 0) {
      atomicAdd(&count[a], 1);
      atomicAdd(&total[a], n);
    }
    __syncthreads();
  }
  // groups
  auto joints_of = [&](int b) {
    if (b >= B || lead[b] != b || in(count + b) < 2 || in(common + b) < kJointPages) return 0;
    return (int)(((int64_t)in(total + b) * G + 31) / 32);
  };
  uint32_t sum[2] = {};
  for (int b0 = 0; b0 < B; b0 += kJointThreads) {
    const int b = b0 + tid, n = joints_of(b);
    uint32_t x[2] = {b < B ? (uint32_t)add(b) : 0, (uint32_t)n}, all[2];
    kv8_block_scan(x, all, store);
    if (b < B) {
      start[b] = (int)(sum[0] + x[0]);
      joint_at[b] = (int)(sum[1] + x[1]);
      // groups that there is no room for stay as they are, and so do those behind them
      if (!n || joint_at[b] + n > jv.most) count[b] = 0;
      else {
        atomicMax(&joints_all, joint_at[b] + n);
        atomicAdd(&saved, (unsigned long long)(in(count + b) - n) * in(common + b));
      }
    }
#pragma unroll
    for (int k = 0; k < 2; k++) sum[k] += all[k];
  }
  __syncthreads();
  if (!joints_all) return;
  // pages that a sequence's units do not look at themselves
  auto skipped = [&](int b) { return lead[b] >= 0 && in(count + lead[b]) ? in(common + lead[b]) : 0; };
  const bool in_tiles = head.tiles > 0;
  auto units_of = [&](int b) { return in_tiles && kv8_tiles(v, add(b)) ? 0 : kv8_units(v, add(b)); };
  uint64_t pages = 0;
  for (int b = tid; b < B; b += kJointThreads) {
    pages += (uint64_t)units_of(b) * (kv8_pages(v.lens[b]) - skipped(b));
    if (in(count + b)) pages += (uint64_t)joints_of(b) * in(common + b);
  }
  pages = kv8_wave_sum(pages);
  if (lane == 0) atomicAdd(&pages_all, (unsigned long long)pages);
  __syncthreads();
  const int each = (int)__builtin_fmin((double)(pages_all + v.items_aim - 1) * v.aim_inverse, 1073741824.0);
  const int parts_of = max(max(kKv8MinPart, (each + kKv8MoreItems - 1) / kKv8MoreItems), min(each, kKv8MaxPart));
  uint32_t at[4] = {};
  for (int b0 = 0; b0 < B; b0 += kJointThreads) {
    const int b = b0 + tid;
    uint32_t x[4] = {}, all[4];
    if (b < B) {
      if (in(count + b)) {
        const int parts = kv8_parts(in(common + b), parts_of);
        x[0] = joints_of(b) * parts;
        x[1] = parts > 1 ? x[0] : 0;
        atomicMax(&most_parts, parts);
      }
      const int parts = kv8_parts(kv8_pages(v.lens[b]) - skipped(b), parts_of);
      if (skipped(b)) atomicMax(&most_own, parts);
      x[2] = units_of(b) * parts;
      x[3] = parts > 1 ? x[2] : 0;
    }
    kv8_block_scan(x, all, store);
    if (b < B) {
      common_at[b] = (int)(at[0] + x[0]);
      common_slot[b] = (int)(at[1] + x[1]);
      item_at[b] = (int)(at[2] + x[2]);
      slot_at[b] = (int)(at[3] + x[3]);
    }
#pragma unroll
    for (int k = 0; k < 4; k++) at[k] += all[k];
  }
  __syncthreads();
  const int slots = 2 * jv.most, commons = (int)at[0], items = (int)(at[0] + at[2]);
  // worth it? (kv8.h)
  const int64_t rounds = ((int64_t)items * v.KVH - 1) / jv.workgroups - ((int64_t)head.items * v.KVH - 1) / jv.workgroups;
  if (jv.saves && (int64_t)saved * v.KVH * v.HD < 128 * (jv.saves + kKv8JointRound * rounds)) return;
  for (int b = tid; b < B; b += kJointThreads) {
    const int a = lead[b];
    if (a < 0 || !in(count + a)) continue;
    const int n = add(b) * G, row0 = joint_at[a] * 32 + before_of[b] * G;
    const int parts = kv8_parts(kv8_pages(v.lens[b]) - skipped(b), parts_of), slot = slots + (int)at[1] + slot_at[b];
    for (int i = 0; i < n; i++) {
      const int r = row0 + i, tok = kv8_div_g(v, i);
      jv.rows[r] = {start[b] + tok, i - tok * G, parts > 1 ? slot : jv.most + (r >> 5), parts, parts > 1 ? i : r & 31, {}};
    }
    if (a == b) {
      const int joints = joints_of(b), parts = kv8_parts(in(common + b), parts_of);
      for (int j = 0; j < joints; j++)
        jv.joints[joint_at[b] + j] = {parts > 1 ? slots + common_slot[b] + j * parts : joint_at[b] + j, parts};
      for (int r = in(total + b) * G; r < joints * 32; r++) jv.rows[joint_at[b] * 32 + r].t = -1;
    }
  }
  // The joints' items, which compute and are the longest, come first; and if not all of the list fits on the GPU, the units', which
  // load, in turn with them until there are no more of one kind.  `turn`: items after which an XCD's turn comes again; a run of one
  // kind goes over its 4 shader engines, too, which take workgroups one after the other, whatever these still hold (in turn XCD by
  // XCD, 512 items of joints ran on half of the CUs).
  int turn = 8;
  while (turn > 1 && turn / 2 * v.KVH % 8 == 0) turn /= 2;
  const int run = 4 * turn, pairs = (int64_t)items * v.KVH > jv.workgroups ? min(commons, items - commons) / run : 0;
  for (int n = tid; n < items; n += kJointThreads) {
    Kv8Item e{};
    const int at_run = n / run;
    bool is_common;
    int i;                                     // the number of its kind
    if (at_run < 2 * pairs) {
      is_common = at_run % 2 == 0;
      i = n - (at_run + 1) / 2 * run;
    } else {
      i = n - pairs * run;
      is_common = i < commons;
      if (!is_common) i += pairs * run - commons;
    }
    if (is_common) {
      const int b = find(common_at, B, i), k = i - common_at[b], joints = joints_of(b), parts = kv8_parts(in(common + b), parts_of);
      // `turn` parts of each one in turn: the group's joints meet on the same XCD over the same pages
      const int block = k / (turn * joints), width = min(turn, parts - block * turn), rest = k - block * turn * joints;
      const int joint = rest / width, pages_in = in(common + b), per = (pages_in + parts - 1) / parts;
      e.seq = b;
      e.part = block * turn + rest % width;
      e.parts = parts;
      e.n = min(32, in(total + b) * G - joint * 32);
      e.wide = e.n > 16;
      e.page0 = min(e.part * per, pages_in);
      e.pages = min(per, pages_in - e.page0);
      e.slot = parts > 1 ? slots + common_slot[b] + joint * parts : joint_at[b] + joint;
      e.joint = joint_at[b] + joint + 1;
    } else {
      const int b = find(item_at, B, i), k = i - item_at[b], h = have(b), more = add(b), skip = skipped(b);
      const int parts = kv8_parts(kv8_pages(h + more) - skip, parts_of), rows = kv8_unit_rows(v, more), u = k / parts;
      e.seq = b;
      e.part = k - u * parts;
      e.parts = parts;
      e.t = start[b] + u * rows;
      e.n = min(rows, more - u * rows);
      e.pos = h + u * rows;
      e.wide = more > v.unit_rows;
      const int all = kv8_pages(e.pos + e.n) - skip, per = (all + parts - 1) / parts;
      e.page0 = min(e.part * per, all);
      e.pages = min(per, all - e.page0);
      e.page0 += skip;
      e.slot = parts > 1 ? slots + (int)at[1] + slot_at[b] + u * parts : -1;
      if (skip) {
        e.joint = -1;
        e.row = joint_at[lead[b]] * 32 + before_of[b] * G;
      }
    }
    jv.items[n] = e;
  }
  if (tid == 0) {
    v.head->joint_items = items;
    v.head->joints = joints_all;
    v.head->most_parts = most_parts + most_own;
  }
}

}  // namespace q4
