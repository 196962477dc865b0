// Low-rank adapters beside a shared projection: the host plan of a batch and
// the device kernels' launchers.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include <vector>

namespace laya {

// An adapter's rank is cut into chunks of 16 columns (one K step of an f16
// MMA, 32 bytes a row), the last one filled up with zeros.  In a bank, chunk c
// of slot s is chunk s * chunks_per_slot + c of
//   A [chunk][16][in_pad]   (in_pad: in rounded up to 64)
//   B [chunk][out_pad][16]  (out_pad: out rounded up to 256; a row's two 8-element
//                            halves placed by lora_at)
constexpr int kLoraChunk = 16;
// Rows of a block: the GEMM's row tile.
constexpr int kLoraBlock = 256;

// Where element j of row r of an MMA operand of 16 columns lies: the 32-byte
// swizzle of a K-major operand, which swaps a row's halves in every second
// group of four rows.  Kept in memory, so that a tile is one contiguous copy:
// the copy unit works by rows, and rows of 128 bytes are a fourth as many as rows
// of 32 through a swizzling tensor map (16384 rows, 1024 -> 5248, ranks to 128, with
// u as one operand an entry: 165.5 us, this way 161.7).
#ifdef __CUDACC__
__host__ __device__
#endif
constexpr int lora_at(int r, int j) { return r * kLoraChunk + ((((j >> 3) ^ (r >> 2)) & 1) << 3) + (j & 7); }

inline int lora_chunks(int rank) { return (rank + kLoraChunk - 1) / kLoraChunk; }

// The adapters each block of 256 rows needs.  Entry e in [off[b], off[b + 1])
// is one chunk of one adapter that some row of block b has; a slot's chunks
// are consecutive entries, slots in order of first use.  row_entry[m]: the
// first entry of row m's adapter, or -1.  u, the rank-space vectors scale *
// (x A^T), is [entries][values, remainders][256 rows][16], halves placed by
// lora_at, zero for rows of other adapters.
//
// u passes between the two products as two values of the 16-bit type, a value
// and what rounding it left: 2^-22 of u is lost in f16 and 2^-16 in bf16, far
// inside the rounding of y.  One f16 alone would lose 2^-11 of the adapter's part
// beside the 2^-11 of y's own rounding.  An f16 ends at 2^-24, so of values below
// 2^-3 up to 2^-25 is lost, which f16's range costs y too; and u must stay below
// 65504, f16's largest.
struct LoraLayout {
  int rows = 0;
  std::vector<int> off;
  std::vector<int2> chunk;      // (slot, chunk of the slot)
  std::vector<int> row_entry;   // [rows]
};
// Throws OpError; chunks_of(slot) is the slot's chunk count, 0 if it is empty.
LoraLayout lora_layout(const int32_t* rows, const int32_t* slot, int n, const std::vector<int>& chunks_of);

// An adapter's host matrices (a [rank, in], b [out, rank], `type` LAYA_F16,
// LAYA_BF16 or LAYA_F32) as the bank's chunks in the 16-bit type: [chunk][16][in_pad]
// and [chunk][out_pad][16] (lora_at), zeros past rank, in and out.  Output row n of b goes
// to row row_of[n] (empty: n).  Throws OpError on a value that is not finite in
// the 16-bit type.
std::vector<uint16_t> lora_pack_a(const void* a, int type, int rank, int in, int in_pad, bool bf16);
std::vector<uint16_t> lora_pack_b(const void* b, int type, int rank, int out, int out_pad, bool bf16,
                                  const std::vector<int>& row_of);

// 16-column operands of u that an entry has, and its elements.
constexpr int kLoraParts = 2;
constexpr size_t kLoraEntryElems = static_cast<size_t>(kLoraBlock) * kLoraChunk * kLoraParts;

// The work of the rank-space product: item i computes entries
// entry[item.y .. item.y + item.z) for rows [128 item.x, 128 item.x + 128).
// Only entries some row of those 128 has are listed.
constexpr int kLoraItemRows = 128;
constexpr int kLoraMaxGroup = 8;  // entries per item
struct LoraItems {
  int group = 1;            // most entries of an item: 1, 2, 4 or 8
  std::vector<int4> item;
  std::vector<int> entry;
};
LoraItems lora_items(const LoraLayout& L, int num_sms);
// CTAs, one an SM, that are taken to run at once in clusters of this size: a
// cluster lies within a group of SMs that its size need not divide (33 clusters of
// 4 do; 16 of 8 were no faster than 16 of 4).
inline int lora_cluster_room(int cluster, int num_sms) {
  return cluster <= 2 ? num_sms : cluster <= 4 ? num_sms * 9 / 10 : num_sms * 2 / 3;
}
// K parts of the rank-space product of `rows` rows: 1, 2, 4 or 8, as many as
// one 128-row item a block leaves SMs for.
int lora_splits(int rows, int num_sms);

// Timeout test: the launch's loads first wait on a barrier that nothing completes,
// or its exchange in the cluster expects bytes that nobody sends, for
// wait_limit_ns.
enum LoraStuck : int { kLoraStuckNone = 0, kLoraStuckLoads = 1, kLoraStuckExchange = 2 };

struct LoraShrinkArgs {
  const int4* item;
  const int* item_entry;
  const int* item_chunk;  // the entries' chunks in the bank, same order
  int items, group;
  const int* row_entry;   // [rows]
  const int* entry_chunk; // [entries]: chunk in the bank
  const float* scale;     // per slot
  void* u;
  int rows, num_kb;       // num_kb: in / 64, rounded up
  int chunks_per_slot;
  bool bf16;
  int* err;
  int stuck;  // see LoraStuck
  unsigned long long wait_limit_ns;
};
// u entries of every row with an adapter.
// x: box 64 x 128, A (make_tmap_pitched, [chunks * 16, in_pad]): box 64 x 16.
// Both launches of u pass grid_dep_wait() before grid_dep_trigger(), so a GEMM
// behind them may start early.
cudaError_t launch_lora_shrink(const CUtensorMap& x, const CUtensorMap& a_map, const LoraShrinkArgs& a, int num_sms,
                               cudaStream_t s);

// The same for few (row, chunk) pairs: pair p is (row, entry, chunk in the
// bank, slot).
struct LoraPairsArgs {
  const int4* pair;
  int pairs;
  const void* x;          // pitch ldx, 16-byte aligned
  long long ldx;
  const void* a;          // the bank's A
  const float* scale;
  void* u;
  int in, in_pad;
  bool bf16;
};
cudaError_t launch_lora_pairs(const LoraPairsArgs& a, cudaStream_t s);

// The projection of few rows: lora_small.cu.  Row tiles of xrows (a multiple
// of 16), tiles of `width` output columns.  `fused`: it computes u too, for at
// most kLoraMaxGroup entries a row tile; otherwise u comes from the launch before
// it (early), and row tile t reads list[off[t]] .. list[off[t + 1] - 1], the
// (entry, its chunk in the bank) some row of it has.
// Maps: x [rows, in] box 64 x xrows, W box 64 x width, u box xrows, B box
// width, A box 64 x 16.
constexpr int kLoraSmallTile = 128;   // most rows a tile
constexpr int kLoraSmallTiles = 40;   // most row tiles with entries
struct LoraSmallPlan {
  bool use = false, fused = false;
  int xrows = 0, width = 0;
  int entries = 0;                                     // of the fullest tile
  std::vector<int> off;                                // not fused: each tile's part
  std::vector<int2> list;                              // of the list
  int tile_entries[kLoraSmallTiles] = {};              // fused: of each row tile,
  int chunk[kLoraSmallTiles][kLoraMaxGroup] = {};      // and their chunks in the bank
};
// Whether and how the rows of L go through lora_small.cu.
LoraSmallPlan lora_small_plan(const LoraLayout& L, int out, int chunks_per_slot, int num_sms);

struct LoraSmallArgs {
  const int* off;
  const int2* list;
  const int* entry_chunk;
  const int* row_entry;
  const float* scale;
  int entries;                                    // as in LoraSmallPlan
  int xrows, width;
  int tile_entries[kLoraSmallTiles];
  int chunk[kLoraSmallTiles][kLoraMaxGroup];
  int chunks_per_slot;
  int b_rows;
  const float* bias;
  void* y;
  long long ldy;
  int rows, out, num_kb;
  bool bf16;
  int early;              // see GemmExt; not with fused
  int* err;
  int stuck;              // see LoraStuck
  unsigned long long wait_limit_ns;
};
cudaError_t launch_lora_small(const CUtensorMap& x, const CUtensorMap& w, const CUtensorMap& u, const CUtensorMap& b,
                              const CUtensorMap& a_map, const LoraSmallArgs& a, bool fused, int num_sms, cudaStream_t s);

}  // namespace laya
