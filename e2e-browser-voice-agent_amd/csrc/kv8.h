// kv8.h -- the paged K/V cache in 8 bits: its layout, and what the other translation units launch of it.
//
// A page holds kKv8Block = 32 positions of one sequence in one layer.  Per (layer, page, kv head) there
// are 32 x HD codes of K, then as many of V, and one fp32 scale for each: a value is scale * code, the
// code in -127..127 held as code + 128 in a byte.  Which 16 bytes a lane loads at once is laid out as the
// matrix cores take them (v_mfma_f32_16x16x32_f16: lane l holds row l % 16 and the 8 values of quarter
// l / 16 of the contraction):
//   K  byte of (position t, column d): the rows of the operand are 16 positions, the contraction 32
//      columns; one 16-byte load holds a lane's 8 columns of two contractions, 64 columns apart by halves
//   V  the rows are 16 columns, the contraction the 32 positions of the page in the order in which the
//      scores of 16 x 16 tiles lie in the lanes (quarter g: 4g..4g+3, then 16+4g..16+4g+3); one load holds a
//      lane's 8 positions of two neighbouring tiles of columns
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace q4 {

constexpr int kKv8Block = 32;
// A unit of more than kKv8Whole pages is shared among several workgroups, in parts of at least kKv8MinPart pages and, while
// that leaves no more than kKv8MoreItems times the items aimed at, at most kKv8MaxPart.  One token (14 heads, 2 kv heads of
// 64 columns): 300 positions whole 6.0 us, in parts 7.4; 1,000 positions whole 8.7, in parts of 8 pages 7.6.  64
// sequences of up to 16,000 positions: parts of at most 128 pages 225 us, as long as the aim asks 245.
constexpr int kKv8Whole = 16, kKv8MinPart = 8, kKv8MaxPart = 128, kKv8MoreItems = 4;
constexpr int kKv8TileRows = 128;
// Sequences are attended to together where that saves passes over so many pages of a kv head, of 128 columns (one of 64 has half the
// bytes), and kKv8JointRound more for each further round of workgroups that its items take.  Of 2,588 random steps (2 to 256 sequences of 7
// layouts behind 260 to 16,000 positions, with up to 1,000 of their own) that is 1.0% slower than the better way in each; the pages alone,
// 5,500 of them, 1.5%, never 36%, always 6%.  Together and one by one, us: 64 sequences (32 heads of 8 x 128), each with up to 40 positions of
// its own and so in a round more, behind 900 (9,400 pages saved) 20.3 and 16.9, 1,600 (22,400) 23.5 and 25.3, 4,000 (56,000) 29.7
// and 49.6; with up to 500 of their own, in no round more, behind 700 21.3 and 21.2, 900 21.3 and 23.0; 64 (16 heads of 8 x 64), a round
// more, behind 1,200 (17,800 of half the bytes) 16.7 and 14.8, 2,400 (36,000) 17.9 and 21.2; 16 (20 of 20 x 64) behind 300 (2,700) 10.8
// and 11.0, 700 (6,300) 10.9 and 12.7.
constexpr int kKv8JointSaves = 3000, kKv8JointRound = 8000;
// Joints of a step at most, which is 8,192 rows of attention of a kv head: two slots of 128 * head_dim bytes a kv head for each.
constexpr int kKv8Joints = 256;
constexpr int kKv8Chunk = 1024;     // pages whose free ones a workgroup of fork counts
// Pages of all tables at most while some belong to several sequences, each counted for each: so plan's sums over the sequences fit 32
// bits, where the pool's pages do not bound them.
constexpr int kKv8Entries = 1 << 30;
// Sequences that add more than one unit are taken in tiles where these and the units of the others are work for
// kKv8MinTiles workgroups; else in units, whose pages can be shared.  Tiles and units, us: 2,048 rows of 14 heads (fp32)
// 57 and 42, 8,192 rows 283 and 370; of 32 heads (bf16) 83 and 84, 773 and 860; of 8 heads of one kv head (bf16) 65 and 32, 262
// and 237; a step of 4 prompts and 44 tokens, 20 kv heads, 78 and 87.
constexpr int kKv8MinTiles = 640;
constexpr float kKv8MinScale = 0x1p-100f;     // a smaller scale is 0, and so are the values

__host__ __device__ constexpr int kv8_k_byte(int HD, int t, int d) {
  const int lane = ((d >> 3) & 3) * 16 + (t & 15);
  return (((t >> 4) * (HD / 64) + (d >> 6)) * 64 + lane) * 16 + ((d >> 5) & 1) * 8 + (d & 7);
}
__host__ __device__ constexpr int kv8_v_byte(int t, int d) {
  const int lane = ((t >> 2) & 3) * 16 + (d & 15);
  return ((d >> 5) * 64 + lane) * 16 + ((d >> 4) & 1) * 8 + (t >> 4) * 4 + (t & 3);
}

// What a plan says of itself.
struct Kv8Head {
  int status;      // KV8_*
  int rows;        // rows of the plan, 0 when it failed
  int free_pages;
  int runs, items, tiles;
  int parts_of;    // pages from which on a unit's pages are shared among several items, and in parts of how many
  int shared;      // whether any page belongs to several sequences (else refs() means nothing)
  int joint_items, joints; // items of the list with joints and joints, 0 where there is no such list
  int most_parts;  // of a row in a joint
};
enum { KV8_OK, KV8_BAD_LENGTH, KV8_TOO_LONG, KV8_ROWS, KV8_PAGES, KV8_STALE, KV8_SHARED, KV8_FORK_SOURCE, KV8_FORK_PAGES, KV8_ENTRIES };

// What the launches of a fork tell one another.
struct Kv8Fork {
  int bad;         // an argument that cannot be, 0 between calls
  int status, copies;
  uint64_t entries;    // of all tables, afterwards
};

// A run: rows t.. that lie in one page from `slot` on, m of them.
struct Kv8Run {
  int t, slot, m, unused;
};

// Attention's work.  A unit is up to 16 / G neighbouring rows of a sequence (G query heads to a kv head; one row
// where G > 16), so that they fill 16 rows of a matrix core, or up to 32 / G of one that adds more than 16 / G; an
// item is one of the `parts` that share a unit's pages.
struct Kv8Item {
  int seq, t, n;         // sequence, first row, rows
  int pos;               // position of the first row
  int page0, pages;      // of the sequence's table
  int part, slot;        // slot: of the unit's first part in the workspace, -1 for a unit in one part
  int parts, wide;
  // of a list with joints: the joint (counted from 1) of an item over a joint's pages, whose n are its rows of attention; -1
  // for a unit with rows in joints, the first of which is `row`; 0 for any other
  int joint, row;
};

// A joint: up to 32 rows of attention, neighbours among the rows of units whose sequences begin with the same pages.  One pass over those
// pages serves them all; a row is the sum of that and of its unit's pass over the pages behind.
struct Kv8Joint {
  int slot, parts;       // where its sums lie in the workspace
};
struct Kv8JointRow {
  int t, h;              // the row of the step (-1: none), the head of the kv head's
  int slot, parts, row;  // where its unit's sums lie
  int unused[3];
};

// A tile: kKv8TileRows rows of attention (positions x G) of a sequence with many rows.
struct Kv8Tile {
  int seq, t, n;         // sequence, its first row, its rows
  int pos;               // position of the first row
  int tile, unused[3];
};

// RoPE beside an append: the table ([positions][head_dim] cosines and sines in turn), the rows' positions, their q.
struct Kv8Rope {
  const float* table;
  const int* pos;
  float* q;
  int64_t q_stride;
};

// The device side of a cache.
struct Kv8View {
  uint8_t* codes;      // [layers][pages][kv_heads][K, V][32 * HD]
  float2* scales;      // [layers][pages][kv_heads] of K, V
  int* table;          // [seqs][blocks] pages, -1 past those a sequence holds
  int* held;           // [seqs] pages of a sequence
  int* stack;          // [4][pages]: free pages, the next one to take last; refs(), count(), first() (of a cache that forks)
  Kv8Head* head;
  int *base, *lens;    // [seqs] positions before and after the step
  int* starts;         // [seqs + 1] first row of a sequence in the step
  int *free_at, *take_at, *run_at, *item_at, *part_at, *tile_at;   // [seqs + 1] sums over the sequences before: pages
                       // given back and taken, runs, items, slots in the workspace, tiles
  Kv8Run* runs;
  Kv8Item* items;
  Kv8Tile* tiles;
  float* part_o;       // [slots][kv_heads * row tiles][32][HD] averages of V of a part
  float2* part_ml;     // [slots][kv_heads * row tiles][32] reference exponent, sum of the probabilities relative to it
  int* arrived;        // [slots][kv_heads * row tiles] parts of a unit that are done (at its first slot)
  int layers, H, KVH, HD, B, W, pages, max_len;
  uint32_t g_magic;    // 2^32 / G rounded up (0 for G = 1): r / G = r * g_magic >> 32 while r * G < 2^32
  int unit_rows, wide_rows;       // rows of a unit
  int row_tiles;       // of a unit: 16 rows (32 of a wide one, which has no more of them)
  int items_aim;       // items that fill the GPU
  double aim_inverse;  // 1 / items_aim, not rounded down
  // Behind the stack and not pointers of their own: every launch takes this struct along, and 56 more bytes cost 0.2 us.
  __device__ int* refs() const { return stack + pages; }                 // sequences that hold a page, while any page has several
  __device__ int* count() const { return stack + 2 * (size_t)pages; }    // scratch of plan and fork, 0 between calls
  __device__ int* first() const { return stack + 3 * (size_t)pages; }    // alike, INT_MAX between calls
};

// The lists with joints, which a step of a cache with shared pages has beside its own.
struct Kv8JointView {
  Kv8Item* items;
  Kv8Joint* joints;    // [most]
  Kv8JointRow* rows;   // [most][32]
  int workgroups;      // of attention
  int saves;           // as kKv8JointSaves; 0: joints whatever they save
  int* queue;          // items of attention that have been drawn, 0 between launches
  int most;            // joints of a step.  The workspace's slots 0..most-1 are of joints in one part, rows of units in one part lie
                       // in the slots most..2 most-1 (32 each, as in the joints), other slots begin behind them
};

// The scratch memory of a fork.
struct Kv8ForkView {
  int* next;           // [seqs][blocks] the tables afterwards
  int2* copies;        // [seqs] a sequence whose last page is copied, and the page
  int* chunk;          // [pages / kKv8Chunk] free pages
  Kv8Fork* fork;
};

}  // namespace q4

struct q4hip_kv8 {
  q4::Kv8View v{};
  q4::Kv8ForkView f{};
  q4::Kv8JointView j{};
  int* joint_scratch = nullptr;
  // Whether pages may be shared, so that a plan makes lists with joints, too: there was a fork, and no call that waits has found since that
  // none is.  A graph may be replayed after other forks, and fork at any time itself.
  bool forked = false, unshared = false, fork_captured = false;
  bool capturing = false;      // the call on its way
  int device = 0, max_rows = 0;
  int rows = 0;                // rows the last plan was called for, outside of captures
  unsigned long long capture = 0;   // the last capture of a plan, and the rows of that
  int capture_rows = 0;
  hipStream_t stream = nullptr;
  q4::Kv8Head* pin = nullptr;  // pinned copy of v.head
};

namespace q4 {

// q4hip_kv8_create; a cache that is never forked (forks false) has no memory for that.
int kv8_create(q4hip_kv8** out, int layers, int heads, int kv_heads, int head_dim, int seqs, int max_len, int pages, int max_rows,
               int device, bool forks);

// The operators' launches without the checks of their arguments (include/q4hip.h); q and out, k and v of `type`; rows: of the plan.
void kv8_launch_plan(q4hip_kv8* kv, hipStream_t s, const int* have, const int* add, int rows, int* starts, int* positions, int* slots,
                     int* tables);
// heads [g0, g0 + heads) of the cache from heads 0.. of the rows
void kv8_launch_append(q4hip_kv8* kv, hipStream_t s, int layer, const void* k, const void* v, int type, int64_t k_stride,
                       int64_t v_stride, int g0, int heads, int rows);
// Rows of q|k|v that begin at multiples of 16 bytes: q turned in place, k and v into the cache, k turned on its way.
void kv8_launch_append_rope(q4hip_kv8* kv, hipStream_t s, int layer, float* qkv, int64_t stride, const float* table, const int* pos,
                            int rows);
void kv8_launch_attend(q4hip_kv8* kv, hipStream_t s, int layer, const void* q, void* out, int type, int64_t q_stride,
                       int64_t out_stride, float scale, int rows);
void kv8_launch_read(q4hip_kv8* kv, hipStream_t s, int layer, const int* seq, const int* pos, int n, float* k, float* v);

}  // namespace q4
