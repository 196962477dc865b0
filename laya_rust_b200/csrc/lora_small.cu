// The adapter projection for few rows: y = x W^T + bias + u B^T.
//
// With few rows the product is a stream of W: what counts is how many SMs read
// it at once and how short the chain behind the loads is.  So W takes the M
// side of the MMA (128 output columns a tile) and a tile of 16..128 rows of x
// the N side (no padding beyond 16), and K is cut over a cluster of up to 8
// CTAs, each with a few k-blocks that are all in flight together: 3072 outputs
// are 24 tiles x 8 parts.  The adapter entries are dealt out over the cluster
// the same way.  D is transposed (TMEM lane = output column, TMEM column =
// row), so a CTA leaves its f32 sums in shared memory as [row][128 columns].
// Each CTA owns a share of the rows: the others send it their sums of those rows
// with one bulk copy each (shared memory to shared memory; plain stores or loads
// through the cluster measured 4 us for 16 KB), and it adds them in rank order
// and stores 16 bytes a thread.
//
// With at most 8 entries a row tile (FUSED) the same launch computes u as well:
// the A rows of the entries ride along the K loop against the same x.  Joint, they
// share the M side with W: a tile is then 128 - 16 entries output columns, and D's
// last lanes are rank space.  Apart, they are a second M = 128 operand with an
// accumulator of its own.  The cluster adds the rank-space sums first, and each
// CTA turns the entries it owns into 16-bit operands of the adapter step in its
// own shared memory.  Every cluster repeats u for its rows (16 rows of A per entry
// from L2), which costs less than a launch of its own.
//
// With more entries u comes from the launch before, and a row tile goes through
// the list of the entries some row of it has (256 rows with an adapter each, 1024
// -> 3072: 22.5 us, by the GEMM 46; through all of the block's 256 entries it took
// 2.4 times as long).  Measured otherwise: one row, 1024 -> 3072, rank 16: 5.8 us;
// 179 rows, 2624 -> 1024, rank 32: 9.4 us; 48 rows with an adapter each: 10.5 us.
#include <cuda_bf16.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "common.cuh"
#include "kernels.h"
#include "lora.h"

namespace laya {

namespace {

constexpr int kCols = 128;                    // output columns of a tile
constexpr int kWBytes = kCols * 64 * 2;       // W operand of a k-block
constexpr int kBBytes = kCols * 32;           // one entry's B operand
constexpr int kABytes = kLoraChunk * 64 * 2;  // one entry's A operand of a k-block
constexpr int kMaxStages = 8;
constexpr int kThreads = 128;
constexpr int kMaxRows = kLoraSmallTile;      // rows a tile
constexpr int kPartLd = kCols + 4;            // floats a row of the f32 parts
constexpr int kPartULd = kLoraChunk + 4;      // and of the rank-space parts
constexpr size_t kSmemLimit = 232448 - 2048;  // dynamic, beside the static barriers and tables

struct SmallMaps {
  CUtensorMap x, w, u, b, a;
};

// What the launch decides.
struct SmallShape {
  int stages;
  int own;     // FUSED: most entries a CTA owns
  int ring_bytes;
};

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// The address in CTA `rank`'s shared memory that `p` has in this CTA's.
__device__ __forceinline__ uint32_t map_to_rank(const void* p, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
  return r;
}
// Copies `bytes` (a multiple of 16) to shared memory of CTA `rank`, at the
// address `dst` has there, counted on that CTA's `bar`.
__device__ __forceinline__ void bulk_to_rank(const void* dst, uint64_t* bar, const void* src, uint32_t bytes, uint32_t rank) {
  asm volatile("cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   map_to_rank(dst, rank)),
               "r"(smem_u32(src)), "r"(bytes), "r"(map_to_rank(bar, rank))
               : "memory");
}

// Eight consecutive floats of every CTA's part, added in rank order: this CTA's
// own at `own`, those it was sent `step` floats apart from `in` (rank c at place
// c, or c - 1 past its own rank).
template <int SPLITS>
__device__ __forceinline__ void sum_parts(const float* own, const float* in, int step, int rank, float (&v)[8]) {
#pragma unroll
  for (int c = 0; c < SPLITS; ++c) {
    const float* p = c == rank ? own : in + (c < rank ? c : c - 1) * step;
    const float4 s = *reinterpret_cast<const float4*>(p), t = *reinterpret_cast<const float4*>(p + 4);
    if (c == 0) {
      v[0] = s.x, v[1] = s.y, v[2] = s.z, v[3] = s.w;
      v[4] = t.x, v[5] = t.y, v[6] = t.z, v[7] = t.w;
    } else {
      v[0] += s.x, v[1] += s.y, v[2] += s.z, v[3] += s.w;
      v[4] += t.x, v[5] += t.y, v[6] += t.z, v[7] += t.w;
    }
  }
}

template <class T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
  } else {
    __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
  }
}

template <class T, int SPLITS, bool FUSED>
__global__ void __launch_bounds__(kThreads)
    lora_small_kernel(const __grid_constant__ SmallMaps maps, const __grid_constant__ LoraSmallArgs a, const SmallShape sh) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t full[kMaxStages], empty[kMaxStages], done, b_full, done2, in_full, in_u_full, stuck_bar;
  __shared__ int row_slot[kMaxRows];
  __shared__ float row_scale[kMaxRows];
  __shared__ uint32_t tmem_holder;
  __shared__ int abort_word;
  volatile int* abort_flag = &abort_word;
  uint8_t* smem = smem_raw + (((smem_u32(smem_raw) + 1023u) & ~1023u) - smem_u32(smem_raw));
  const int warp = threadIdx.x >> 5;
  const int rank = SPLITS > 1 ? static_cast<int>(cluster_rank()) : 0;
  const int width = a.width;                  // output columns of a tile
  const bool joint = FUSED && width < kCols;  // A rows beside W's
  // apart, a whole tile of 128 rows in one CTA: x takes the M side against the
  // entries' A rows (N = 16 entries), so only their rows are read, and a thread
  // finds its row's rank values in its own TMEM lane
  const bool by_row = SPLITS == 1 && FUSED && !joint && a.xrows == kCols;
  const int n0 = static_cast<int>(blockIdx.x) / SPLITS * width;
  const int xrows = a.xrows, m0 = static_cast<int>(blockIdx.y) * xrows;
  // FUSED: this row tile's entries
  const int* const chunk = a.chunk[FUSED ? blockIdx.y : 0];
  const int entries = FUSED ? a.tile_entries[blockIdx.y] : 0;
  const int rows = min(xrows, a.rows - m0);
  constexpr int kParts = kLoraParts;      // operands of u an entry has
  constexpr int kPerStage = 4 / kParts;   // entries a stage
  const int x_bytes = xrows * 128, u_bytes = xrows * 32;
  // a stage: [W | A, joint] [x] [A, apart], room for the fullest tile's entries
  const int stage_bytes = kWBytes + x_bytes + (FUSED && !joint ? a.entries * kABytes : 0);
  const int load_bytes = width * 128 + x_bytes + (FUSED ? entries * kABytes : 0);
  const int kb0 = rank * a.num_kb / SPLITS, kb1 = (rank + 1) * a.num_kb / SPLITS;
  int e0 = rank * entries / SPLITS, e1 = (rank + 1) * entries / SPLITS;
  // else: this CTA's part of the tile's list, read by each role once it has
  // something else to wait for
  auto find_entries = [&] {
    if (FUSED || a.entries == 0) return;
    const int first = __ldg(a.off + blockIdx.y), n = __ldg(a.off + blockIdx.y + 1) - first;
    e0 = first + rank * n / SPLITS;
    e1 = first + (rank + 1) * n / SPLITS;
  };
  const int need_cols = FUSED && !joint ? 2 * xrows : xrows;
  const uint32_t tmem_cols = need_cols <= 32 ? 32 : need_cols <= 64 ? 64 : need_cols <= 128 ? 128 : 256;
  // A cluster: [owned B operands | owned u operands] [ring] [part] [parts sent
  // here] [rank-space part] [parts sent here], the parts apart from the ring,
  // which this CTA may still be using when another one's sums arrive.  One CTA
  // alone: [owned B operands] [ring], and over the idle ring first [rank-space
  // part] [u operands], then [part].
  // Every operand of the ring starts on the 1024 bytes of its swizzle's period: an
  // owned B operand is 4096 bytes and a pair of u's is xrows * 64, xrows and width
  // are multiples of 16.
  const int u_entry = xrows * kPartULd;
  const int own_rows = xrows / SPLITS;                            // rows rank * own_rows ..
  uint8_t* own_b = smem;
  uint8_t* own_u = own_b + sh.own * kBBytes;
  uint8_t* ring = SPLITS > 1 ? own_u + sh.own * kParts * u_bytes : own_u;
  if (SPLITS == 1) own_u = ring + a.entries * u_entry * 4;
  float* part = reinterpret_cast<float*>(SPLITS > 1 ? ring + sh.ring_bytes : ring);   // [xrows][kPartLd]
  float* part_in = part + xrows * kPartLd;                                            // [SPLITS - 1][own_rows][kPartLd]
  float* part_u = SPLITS > 1 ? part_in + (SPLITS - 1) * own_rows * kPartLd : part;    // [entries][xrows][kPartULd]
  float* part_u_in = part_u + a.entries * u_entry;                // [SPLITS - 1][e1 - e0][xrows][kPartULd]
  if (threadIdx.x == 0) {
    for (int s = 0; s < sh.stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(&done, 1);
    mbar_init(&b_full, 1);
    mbar_init(&done2, 1);
    mbar_init(&in_full, 1);
    mbar_init(&in_u_full, 1);
    mbar_init(&stuck_bar, 1);
    tma_prefetch_desc(&maps.w);
    tma_prefetch_desc(&maps.x);
    if (FUSED) tma_prefetch_desc(&maps.a);
    tma_prefetch_desc(&maps.b);
    if (!FUSED) tma_prefetch_desc(&maps.u);
    abort_word = 0;
    fence_mbar_init();
    if (SPLITS > 1) {
      const int extra = a.stuck == kLoraStuckExchange ? 16 : 0;
      mbar_arrive_expect_tx(&in_full, (SPLITS - 1) * own_rows * kPartLd * 4 + extra);
      if (FUSED && e0 < e1) mbar_arrive_expect_tx(&in_u_full, (SPLITS - 1) * (e1 - e0) * u_entry * 4 + extra);
    }
  }
  if (warp == 1) {
    tmem_alloc(&tmem_holder, tmem_cols);
    tmem_relinquish();
  }
  __syncwarp();
  if (SPLITS > 1) cluster_arrive();  // this CTA's shared memory exists
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_holder, tmem_u = joint ? tmem : tmem + xrows;
  if (!a.early) grid_dep_wait();
  grid_dep_trigger();

  const uint32_t idesc = std::is_same<T, __nv_bfloat16>::value ? umma_idesc_bf16(kCols, xrows) : umma_idesc_f16(kCols, xrows);
  const uint32_t idesc_u = std::is_same<T, __nv_bfloat16>::value ? umma_idesc_bf16(kCols, kLoraChunk * entries)
                                                                  : umma_idesc_f16(kCols, kLoraChunk * entries);
  if (warp == 0) {
    if (elect_one()) {
      bool ok = true;
      int stage = 0;
      uint32_t phase = 0;
      auto next = [&]() {
        if (++stage == sh.stages) {
          stage = 0;
          phase ^= 1u;
        }
      };
      if (a.stuck == kLoraStuckLoads)
        ok = mbar_wait_bounded(&stuck_bar, 0, a.err, kErrLoraWait, abort_flag, a.wait_limit_ns);
      for (int kb = kb0; kb < kb1 && ok; ++kb) {
        ok = mbar_wait_bounded(&empty[stage], phase ^ 1u, a.err, kErrLoraWait, abort_flag);
        if (!ok) break;
        uint8_t* sw = ring + stage * stage_bytes;
        mbar_arrive_expect_tx(&full[stage], load_bytes);
        tma_load_2d(sw, &maps.w, kb * 64, n0, &full[stage]);
        tma_load_2d(sw + kWBytes, &maps.x, kb * 64, m0, &full[stage]);
        if constexpr (FUSED) {
#pragma unroll
          for (int i = 0; i < kLoraMaxGroup; ++i)
            if (i < entries)
              tma_load_2d((joint ? sw + width * 128 : sw + kWBytes + x_bytes) + i * kABytes, &maps.a, kb * 64,
                          chunk[i] * kLoraChunk, &full[stage]);
        }
        next();
      }
      find_entries();
      if constexpr (FUSED) {
        if (e0 < e1 && ok) {
          mbar_arrive_expect_tx(&b_full, (e1 - e0) * width * 32);
#pragma unroll
          for (int i = 0; i < kLoraMaxGroup; ++i)
            if (i >= e0 && i < e1) tma_load_2d(own_b + (i - e0) * kBBytes, &maps.b, 0, (chunk[i] * a.b_rows + n0) / 4, &b_full);
        }
      } else if (e0 < e1 && ok) {
        // B operands do not wait for u: those of the stages that are free now go
        // ahead of it
        auto load_b = [&](int st, int e, int n) {
          uint8_t* sb = ring + st * stage_bytes;
          mbar_arrive_expect_tx(&full[st], n * (kBBytes + kParts * u_bytes));
          int c[kPerStage];
#pragma unroll
          for (int i = 0; i < kPerStage; ++i) c[i] = i < n ? __ldg(&a.list[e + i].y) : 0;
#pragma unroll
          for (int i = 0; i < kPerStage; ++i)
            if (i < n) tma_load_2d(sb + i * kBBytes, &maps.b, 0, (c[i] * a.b_rows + n0) / 4, &full[st]);
        };
        // of the next stage
        int ent[kPerStage];
        auto find_u = [&](int e) {
#pragma unroll
          for (int i = 0; i < kPerStage; ++i) ent[i] = e + i < e1 ? __ldg(&a.list[e + i].x) : 0;
        };
        auto load_u = [&](int st, int n) {
#pragma unroll
          for (int i = 0; i < kPerStage; ++i) {
            if (i >= n) break;
            uint8_t* su = ring + st * stage_bytes + kWBytes + i * kParts * u_bytes;
            const int y = ent[i] * kParts * kLoraBlock + m0 % kLoraBlock;
            tma_load_2d(su, &maps.u, 0, y / 4, &full[st]);
            tma_load_2d(su + u_bytes, &maps.u, 0, (y + kLoraBlock) / 4, &full[st]);
          }
        };
        int ahead = e0, st = stage;
        uint32_t ph = phase;
        for (int i = 0; i < sh.stages && ahead < e1 && mbar_try_wait(&empty[st], ph ^ 1u); ++i) {
          load_b(st, ahead, min(kPerStage, e1 - ahead));
          ahead += kPerStage;
          if (++st == sh.stages) {
            st = 0;
            ph ^= 1u;
          }
        }
        find_u(e0);
        grid_dep_wait();  // u is complete
        for (int e = e0; e < e1; e += kPerStage) {
          const int n = min(kPerStage, e1 - e);
          if (e >= ahead) {
            ok = mbar_wait_bounded(&empty[stage], phase ^ 1u, a.err, kErrLoraWait, abort_flag);
            if (!ok) break;
            load_b(stage, e, n);
          }
          load_u(stage, n);
          find_u(e + kPerStage);
          next();
        }
      }
      if (!ok || *abort_flag) wait_for_copies();
    }
    __syncwarp();
  } else if (warp == 1) {
    if (elect_one()) {
      find_entries();
      bool ok = true;
      int stage = 0;
      uint32_t phase = 0;
      auto next = [&]() {
        umma_commit(&empty[stage]);
        if (++stage == sh.stages) {
          stage = 0;
          phase ^= 1u;
        }
      };
      for (int kb = kb0; kb < kb1; ++kb) {
        ok = mbar_wait_bounded(&full[stage], phase, a.err, kErrLoraWait, abort_flag);
        if (!ok) break;
        tc_fence_after();
        const uint32_t w_addr = smem_u32(ring + stage * stage_bytes), x_addr = w_addr + kWBytes;
#pragma unroll
        for (int k = 0; k < 4; ++k)
          umma_f16(tmem, umma_desc_sw128(w_addr + k * 32), umma_desc_sw128(x_addr + k * 32), idesc,
                   (kb != kb0 || k != 0) ? 1u : 0u);
        if (by_row && entries > 0) {
#pragma unroll
          for (int k = 0; k < 4; ++k)
            umma_f16(tmem_u, umma_desc_sw128(x_addr + k * 32), umma_desc_sw128(x_addr + x_bytes + k * 32), idesc_u,
                     (kb != kb0 || k != 0) ? 1u : 0u);
        } else if (FUSED && !joint && entries > 0) {
          // 128 rows from the A operand on: past the entries' they are whatever
          // follows in shared memory, and their sums are never read
#pragma unroll
          for (int k = 0; k < 4; ++k)
            umma_f16(tmem_u, umma_desc_sw128(x_addr + x_bytes + k * 32), umma_desc_sw128(x_addr + k * 32), idesc,
                     (kb != kb0 || k != 0) ? 1u : 0u);
        }
        next();
      }
      if constexpr (!FUSED) {
        for (int e = e0; e < e1 && ok; e += kPerStage) {
          ok = mbar_wait_bounded(&full[stage], phase, a.err, kErrLoraWait, abort_flag);
          if (!ok) break;
          tc_fence_after();
          const uint32_t b_addr = smem_u32(ring + stage * stage_bytes);
          for (int i = 0; i < min(kPerStage, e1 - e); ++i) {
            const uint64_t db = umma_desc_sw32(b_addr + i * kBBytes);
            const uint32_t su = b_addr + kWBytes + i * kParts * u_bytes;
            umma_f16(tmem, db, umma_desc_sw32(su), idesc, 1u);
            umma_f16(tmem, db, umma_desc_sw32(su + u_bytes), idesc, 1u);
          }
          next();
        }
      }
      umma_commit(&done);
    }
    __syncwarp();
  } else if (!FUSED) {
    // the list, into this SM's L1 before warp 0 asks for it
    find_entries();
    for (int e = e0 + 16 * (static_cast<int>(threadIdx.x) - 64); e < e1; e += 16 * 64) {
      int v;
      asm volatile("ld.global.nc.b32 %0, [%1];" : "=r"(v) : "l"(&a.list[e]));
    }
  } else {
    // whose adapter each row has, while the other warps load and multiply
    for (int m = static_cast<int>(threadIdx.x) - 64; m < xrows; m += 64) {
      const int re = m < rows ? __ldg(a.row_entry + m0 + m) : -1;
      const int slot = re >= 0 ? __ldg(a.entry_chunk + re) / a.chunks_per_slot : -1;
      row_slot[m] = slot;
      row_scale[m] = slot >= 0 ? __ldg(a.scale + slot) : 0.0f;
    }
  }
  const uint32_t lane_base = static_cast<uint32_t>(warp * 32) << 16;
  bool ok = mbar_wait_bounded(&done, 0, a.err, kErrLoraWait, nullptr) && !*abort_flag;
  ok = __syncthreads_and(ok);
  tc_fence_after();
  if (SPLITS > 1) cluster_wait();  // every CTA of the cluster has started
  if constexpr (FUSED) {
    if (by_row) {
      const int m = threadIdx.x, slot_of_row = row_slot[m];
      const float scale = row_scale[m];
      for (int e = 0; e < entries; ++e) {
        uint32_t v[16];
        tmem_ld_32x32b_x16(tmem_u + lane_base + e * kLoraChunk, v);
        tmem_ld_wait();
        const bool mine = slot_of_row == chunk[e] / a.chunks_per_slot;
        uint8_t* op = own_u + e * kParts * u_bytes;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t hi[4] = {0, 0, 0, 0}, lo[4] = {0, 0, 0, 0};
          if (mine) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              lora_split<T>(__uint_as_float(v[8 * h + 2 * j]) * scale, __uint_as_float(v[8 * h + 2 * j + 1]) * scale, hi[j], lo[j]);
          }
          const int at = 2 * lora_at(m, 8 * h);
          *reinterpret_cast<uint4*>(op + at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
          *reinterpret_cast<uint4*>(op + u_bytes + at) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        }
        __syncwarp();  // the next load takes a whole warp
      }
    }
    // lane = row of A, from the first rank-space lane on
    const int lane0 = joint ? width : 0, ar = static_cast<int>(threadIdx.x) - lane0;
    if (!by_row && warp * 32 + 31 >= lane0 && warp * 32 < lane0 + entries * kLoraChunk) {
      float* dst = part_u + (ar / kLoraChunk) * u_entry + ar % kLoraChunk;
      for (int m = 0; m < rows; m += 16) {
        uint32_t v[16];
        tmem_ld_32x32b_x16(tmem_u + lane_base + m, v);
        tmem_ld_wait();
        if (ar >= 0 && ar < entries * kLoraChunk) {
#pragma unroll
          for (int j = 0; j < 16; ++j) dst[(m + j) * kPartULd] = __uint_as_float(v[j]);
        }
        __syncwarp();
      }
    }
    fence_proxy_async_smem();
    __syncthreads();
    if (SPLITS > 1) {
      // each owner's entries, to the owner
      const int to = static_cast<int>(threadIdx.x);
      if (to < SPLITS && to != rank) {
        const int f0 = to * entries / SPLITS, f1 = (to + 1) * entries / SPLITS;
        if (f0 < f1)
          bulk_to_rank(part_u_in + (rank < to ? rank : rank - 1) * (f1 - f0) * u_entry, &in_u_full, part_u + f0 * u_entry,
                       (f1 - f0) * u_entry * 4, to);
      }
      if (e0 < e1 && !mbar_wait_bounded(&in_u_full, 0, a.err, kErrLoraWait, nullptr, a.wait_limit_ns)) {
        ok = false;
        wait_for_copies();
      }
    }
    for (int e = e0; e < e1 && !by_row; ++e) {
      const int slot = chunk[e] / a.chunks_per_slot;
      uint8_t* hi_op = own_u + (e - e0) * kParts * u_bytes;
      // thread: half (8 of 16 rank values) of a row
      for (int i = threadIdx.x; i < 2 * xrows; i += kThreads) {
        const int m = i >> 1, h = i & 1;
        uint32_t hi[4] = {0, 0, 0, 0}, lo[4] = {0, 0, 0, 0};
        if (row_slot[m] == slot) {
          float v[8];
          sum_parts<SPLITS>(part_u + e * u_entry + m * kPartULd + 8 * h,
                            part_u_in + (e - e0) * u_entry + m * kPartULd + 8 * h, (e1 - e0) * u_entry, rank, v);
          const float scale = row_scale[m];
#pragma unroll
          for (int j = 0; j < 4; ++j) lora_split<T>(v[2 * j] * scale, v[2 * j + 1] * scale, hi[j], lo[j]);
        }
        const int at = 2 * lora_at(m, 8 * h);
        *reinterpret_cast<uint4*>(hi_op + at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        *reinterpret_cast<uint4*>(hi_op + u_bytes + at) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
      }
    }
    tc_fence_before();
    fence_proxy_async_smem();
    // each thread waited for the rank-space sums by itself: where one of them gave
    // up, all skip the adapter step (elect_one needs its whole warp)
    ok = __syncthreads_and(ok);
    if (e0 < e1 && ok) {
      if (warp == 1 && elect_one()) {
        if (mbar_wait_bounded(&b_full, 0, a.err, kErrLoraWait, abort_flag)) {
          tc_fence_after();
          for (int i = 0; i < e1 - e0; ++i) {
            const uint64_t db = umma_desc_sw32(smem_u32(own_b + i * kBBytes));
            const uint32_t su = smem_u32(own_u + i * kParts * u_bytes);
            umma_f16(tmem, db, umma_desc_sw32(su), idesc, 1u);
            umma_f16(tmem, db, umma_desc_sw32(su + u_bytes), idesc, 1u);
          }
        }
        umma_commit(&done2);
      }
      ok = mbar_wait_bounded(&done2, 0, a.err, kErrLoraWait, nullptr) && !*abort_flag;
    }
    ok = __syncthreads_and(ok);
    tc_fence_after();
  }
  // thread = output column
  for (int m = 0; m < rows; m += 16) {
    uint32_t v[16];
    tmem_ld_32x32b_x16(tmem + lane_base + m, v);
    tmem_ld_wait();
#pragma unroll
    for (int j = 0; j < 16; ++j) part[(m + j) * kPartLd + threadIdx.x] = __uint_as_float(v[j]);
  }
  tc_fence_before();
  fence_proxy_async_smem();
  __syncthreads();
  if (SPLITS > 1) {
    // each owner's rows, to the owner
    const int to = static_cast<int>(threadIdx.x);
    if (to < SPLITS && to != rank)
      bulk_to_rank(part_in + (rank < to ? rank : rank - 1) * own_rows * kPartLd, &in_full, part + to * own_rows * kPartLd,
                   own_rows * kPartLd * 4, to);
    if (!mbar_wait_bounded(&in_full, 0, a.err, kErrLoraWait, nullptr, a.wait_limit_ns)) {
      ok = false;
      wait_for_copies();
    }
    __syncwarp();
    cluster_arrive();  // what this CTA was sent has landed
  }
  // the owned rows: 16 threads a row, 8 columns each
  const int col = n0 + static_cast<int>(threadIdx.x & 15) * 8;
  // columns of this thread that exist (the tile's, then the output's)
  const int left = static_cast<int>(threadIdx.x & 15) * 8 < width ? a.out - col : 0;
  for (int i = static_cast<int>(threadIdx.x >> 4); i < own_rows && left > 0 && ok; i += 8) {
    const int m = rank * own_rows + i;
    if (m >= rows) break;
    float v[8];
    sum_parts<SPLITS>(part + m * kPartLd + (threadIdx.x & 15) * 8, part_in + i * kPartLd + (threadIdx.x & 15) * 8,
                      own_rows * kPartLd, rank, v);
    if (a.bias) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < left) v[j] += __ldg(a.bias + col + j);
    }
    uint32_t o[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = pack2<T>(v[2 * j], v[2 * j + 1]);
    uint16_t* dst = static_cast<uint16_t*>(a.y) + static_cast<size_t>(m0 + m) * a.ldy + col;
    if (left >= 8) {
      *reinterpret_cast<uint4*>(dst) = make_uint4(o[0], o[1], o[2], o[3]);
    } else {
#pragma unroll
      for (int j = 0; j < 7; ++j)
        if (j < left) dst[j] = static_cast<uint16_t>(o[j / 2] >> (16 * (j & 1)));
    }
  }
  __syncwarp();
  if constexpr (!FUSED) grid_dep_wait();  // this grid does not complete before the one that computes u
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, tmem_cols);
  }
  __syncwarp();
  if (SPLITS > 1) cluster_wait();  // no CTA leaves while a copy may still read its part
}

template <class T, int SPLITS, bool FUSED>
cudaError_t launch(const SmallMaps& maps, const LoraSmallArgs& a, const SmallShape& sh, size_t smem, cudaStream_t s) {
  static std::atomic<bool> configured[64] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  if (!configured[dev]) {
    e = cudaFuncSetAttribute(lora_small_kernel<T, SPLITS, FUSED>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             static_cast<int>(kSmemLimit));
    if (e != cudaSuccess) return e;
    configured[dev] = true;
  }
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = SPLITS;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  const dim3 grid((a.out + a.width - 1) / a.width * SPLITS, (a.rows + a.xrows - 1) / a.xrows);
  return launch_pdl(lora_small_kernel<T, SPLITS, FUSED>, grid, dim3(kThreads), smem, s, attr, 1, maps, a, sh);
}

template <class T, bool FUSED>
cudaError_t launch_splits(int splits, const SmallMaps& maps, const LoraSmallArgs& a, const SmallShape& sh, size_t smem,
                          cudaStream_t s) {
  switch (splits) {
    case 1: return launch<T, 1, FUSED>(maps, a, sh, smem, s);
    case 2: return launch<T, 2, FUSED>(maps, a, sh, smem, s);
    case 4: return launch<T, 4, FUSED>(maps, a, sh, smem, s);
    default: return launch<T, 8, FUSED>(maps, a, sh, smem, s);
  }
}

}  // namespace

LoraSmallPlan lora_small_plan(const LoraLayout& L, int out, int chunks_per_slot, int num_sms) {
  const int rows = L.rows;
  LoraSmallPlan best;
  if (rows < 1) return best;
  const bool one_block = rows <= kLoraBlock, any = !L.chunk.empty();
  // row tiles of at most 64, of equal size within one block, or of 128
  const int tiles64 = (rows + 63) / 64;
  const int even = one_block ? ((rows + tiles64 - 1) / tiles64 + 15) / 16 * 16 : 64;
  for (int xrows : {even, kLoraSmallTile}) {
    const int tiles = (rows + xrows - 1) / xrows;
    if (tiles > kLoraSmallTiles || (xrows > even && rows <= even)) continue;
    // without adapters the GEMM has no launch before it, and beats tiles of 128
    // (1357 rows, 1000 -> 1536: 9.3 and 10.3 us; with one adapter 14.2 and 11.5)
    if (!any && !one_block && xrows > even) continue;
    LoraSmallPlan p;
    p.use = true;
    p.xrows = xrows;
    // the chunks some row of each tile has
    bool fits = true;
    for (int m = 0; m < rows && fits; ++m) {
      const int e0 = L.row_entry[m];
      if (e0 < 0) continue;
      int* const chunk = p.chunk[m / xrows];
      int& n = p.tile_entries[m / xrows];
      for (int e = e0; e < static_cast<int>(L.chunk.size()) && (e == e0 || L.chunk[e].y > 0); ++e) {
        const int c = L.chunk[e].x * chunks_per_slot + L.chunk[e].y;
        if (std::find(chunk, chunk + n, c) != chunk + n) continue;
        if (n == kLoraMaxGroup) {
          fits = false;
          break;
        }
        chunk[n++] = c;
      }
    }
    p.fused = any && fits;
    const int most = *std::max_element(p.tile_entries, p.tile_entries + tiles);
    p.entries = most;
    if (any && !fits) {
      std::vector<int> seen(L.chunk.size(), -1);
      for (int t = 0; t < tiles; ++t) {
        p.off.push_back(static_cast<int>(p.list.size()));
        for (int m = t * xrows; m < std::min(rows, (t + 1) * xrows); ++m) {
          const int e0 = L.row_entry[m];
          if (e0 < 0 || seen[e0] == t) continue;
          seen[e0] = t;
          for (int e = e0; e < static_cast<int>(L.chunk.size()) && (e == e0 || L.chunk[e].y > 0); ++e)
            p.list.push_back(make_int2(e, L.chunk[e].x * chunks_per_slot + L.chunk[e].y));
        }
        p.entries = std::max(p.entries, static_cast<int>(p.list.size()) - p.off.back());
      }
      p.off.push_back(static_cast<int>(p.list.size()));
    }
    // joint pays where the K loop carries many rows (256 rows, 1024 -> 3072, one
    // entry: 8.8 us, apart 10.2 us); with few, more tiles cost what a second
    // operand does (1 row: 5.1 us either way)
    for (int width : {kCols - most * kLoraChunk, kCols}) {
      if (width < kCols && !(p.fused && most <= 4 && rows > 32)) continue;
      p.width = width;
      // every CTA on an SM of its own; failing that, within one block of rows,
      // the smaller tiles in rounds (beyond it the GEMM is faster: 1000 rows of 100
      // adapters, 1024 -> 3072, 21 us and, in two rounds, 26; in one round: 768 rows
      // with an adapter each, 2624 -> 1024, 66 us by the GEMM, 36 here)
      if ((out + width - 1) / width * tiles <= num_sms) return p;
      if (one_block && !best.use) best = p;
    }
  }
  return best;
}

cudaError_t launch_lora_small(const CUtensorMap& x, const CUtensorMap& w, const CUtensorMap& u, const CUtensorMap& b,
                              const CUtensorMap& a_map, const LoraSmallArgs& a, bool fused, int num_sms, cudaStream_t s) {
  if (a.rows <= 0) return cudaSuccess;
  const int row_tiles = a.xrows > 0 ? (a.rows + a.xrows - 1) / a.xrows : 0;
  if (a.num_kb < 1 || a.xrows < 16 || a.xrows > kLoraSmallTile || a.xrows % 16 || a.width < 16 || a.width > kCols ||
      (fused && (a.entries < 1 || a.entries > kLoraMaxGroup || row_tiles > kLoraSmallTiles)) ||
      (!fused && a.entries > 0 && (!a.off || !a.list)))
    return cudaErrorInvalidValue;
  SmallShape sh{};
  const bool apart = fused && a.width == kCols;
  const int tiles = (a.out + a.width - 1) / a.width * row_tiles;
  // K parts: as many as still run at once (64 rows with one adapter, 1024 -> 3072: 4
  // parts, 7.1 us; 8 parts, in two rounds, 14 us); tiles of 16 rows leave room
  // for two CTAs an SM (1 row: 4 parts 5.4 us, 8 parts 5.2 us)
  int splits = 1;
  while (splits < 8 && 2 * splits <= a.num_kb &&
         2 * splits * tiles <= (a.xrows <= 16 ? 2 : 1) * lora_cluster_room(2 * splits, num_sms))
    splits *= 2;
  constexpr int per_stage = 4 / kLoraParts;
  const int stage_bytes = kWBytes + a.xrows * 128 + (apart ? a.entries * kABytes : 0);
  const size_t rank_part = fused ? sizeof(float) * a.xrows * kPartULd : 0;   // of one entry
  const size_t u_ops = static_cast<size_t>(kLoraParts) * a.xrows * 32;       // of one entry
  // A CTA waits for its cluster, so no CTA may be left waiting for TMEM that a
  // waiting one holds: shared memory in proportion to the TMEM columns (456 of
  // an SM's 233472 bytes a column, of its 512) keeps the columns of the CTAs
  // on an SM, of this kernel and the other clustered ones, within 512.
  const int need = apart ? 2 * a.xrows : a.xrows;
  const int cols = need <= 32 ? 32 : need <= 64 ? 64 : need <= 128 ? 128 : 256;
  size_t smem = 0;
  for (;; splits /= 2) {
    sh.own = fused ? (a.entries + splits - 1) / splits : 0;
    const int steps = (a.num_kb + splits - 1) / splits +
                      (fused ? 0 : ((a.entries + splits - 1) / splits + per_stage - 1) / per_stage);
    // what lies behind the ring (a cluster), or over it (one CTA)
    const size_t parts = splits > 1 ? sizeof(float) * kPartLd * (a.xrows + (splits - 1) * (a.xrows / splits)) +
                                          rank_part * (a.entries + (splits - 1) * sh.own)
                                    : 0;
    const size_t over =
        splits > 1 ? 0 : std::max(sizeof(float) * kPartLd * a.xrows, (rank_part + (fused ? u_ops : 0)) * a.entries);
    // apart: the last stage's A operand is read as 128 rows, so 16 KB must follow
    const size_t fixed = 1024 + static_cast<size_t>(sh.own) * (kBBytes + (splits > 1 ? u_ops : 0)) +
                         std::max<size_t>(parts, apart ? 128 * 128 : 0);
    const int room = fixed < kSmemLimit ? static_cast<int>((kSmemLimit - fixed) / stage_bytes) : 0;
    sh.stages = std::min(std::min(kMaxStages, steps), room);
    sh.ring_bytes = sh.stages * stage_bytes;
    smem = std::max(fixed + std::max(static_cast<size_t>(sh.ring_bytes), over), static_cast<size_t>(cols) * 456 - 1024);
    if (sh.stages >= std::min(2, steps) && smem <= kSmemLimit) break;
    if (splits == 1) return cudaErrorInvalidValue;
  }
  const SmallMaps maps{x, w, u, b, a_map};
  if (a.bf16)
    return fused ? launch_splits<__nv_bfloat16, true>(splits, maps, a, sh, smem, s)
                 : launch_splits<__nv_bfloat16, false>(splits, maps, a, sh, smem, s);
  return fused ? launch_splits<__half, true>(splits, maps, a, sh, smem, s)
               : launch_splits<__half, false>(splits, maps, a, sh, smem, s);
}

}  // namespace laya
