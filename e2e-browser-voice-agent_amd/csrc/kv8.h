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
};
enum { KV8_OK, KV8_BAD_LENGTH, KV8_TOO_LONG, KV8_ROWS, KV8_PAGES, KV8_STALE };

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
  int parts, wide, unused[2];
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
  int* stack;          // [pages] free pages, the next one to take last
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
};

}  // namespace q4

struct q4hip_kv8 {
  q4::Kv8View v{};
  int device = 0, max_rows = 0;
  int rows = 0;                // rows the last plan was called for, outside of captures
  unsigned long long capture = 0;   // the last capture of a plan, and the rows of that
  int capture_rows = 0;
  hipStream_t stream = nullptr;
  q4::Kv8Head* pin = nullptr;  // pinned copy of v.head
};

namespace q4 {

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
