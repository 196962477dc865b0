// The adapter projection for few rows (at most 256): y = x W^T + bias + u B^T.
//
// With few rows the product is a stream of W: what counts is how many SMs read
// it at once and how short the chain behind the loads is.  So W takes the M
// side of the MMA (128 output columns a tile) and the rows of x the N side
// (16..256, no padding beyond 16), and K is cut over a cluster of up to 8 CTAs,
// each with a few k-blocks that are all in flight together: 3072 outputs are
// 24 tiles x 8 parts.  The adapter entries are dealt out over the cluster the
// same way.  D is transposed (TMEM lane = output column, TMEM column = row), so
// a CTA writes its f32 part to shared memory as [row][128 columns]; the CTAs
// then each add a share of the rows over the cluster in rank order
// (distributed shared memory) and store them 16 bytes a thread.
//
// Measured (one B200, whole call as a graph, L2 cold): see lora_use_small.
#include <cuda_bf16.h>

#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "kernels.h"
#include "lora.h"

namespace laya {

namespace {

constexpr int kCols = 128;                    // output columns of a tile
constexpr int kWBytes = kCols * 64 * 2;       // W operand of a k-block
constexpr int kBBytes = kCols * 32;           // one entry's B operand
constexpr int kMaxStages = 8;
constexpr int kThreads = 128;
constexpr int kPartLd = kCols + 4;            // floats a row of the f32 part
constexpr size_t kSmemLimit = 232448;

struct SmallMaps {
  CUtensorMap x, w, u, b;
};

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float4 ld_cluster_f4(const float* p, uint32_t rank) {
  uint32_t r;
  float4 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(r)
               : "memory");
  return v;
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

template <class T>
__global__ void __launch_bounds__(kThreads)
    lora_small_kernel(const __grid_constant__ SmallMaps maps, const LoraSmallArgs a, const int splits, const int stages) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t full[kMaxStages], empty[kMaxStages], done;
  __shared__ uint32_t tmem_holder;
  __shared__ int abort_word;
  volatile int* abort_flag = &abort_word;
  uint8_t* smem = smem_raw + (((smem_u32(smem_raw) + 1023u) & ~1023u) - smem_u32(smem_raw));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = static_cast<int>(cluster_rank());
  const int n0 = static_cast<int>(blockIdx.x) / splits * kCols;
  const int xrows = (a.rows + 15) & ~15;              // N of the MMA
  const int x_bytes = xrows * 128, u_bytes = xrows * 32;
  const int stage_bytes = kWBytes + ((x_bytes + 1023) & ~1023);
  const int kb0 = rank * a.num_kb / splits, kb1 = (rank + 1) * a.num_kb / splits;
  const int e0 = rank * a.entries / splits, e1 = (rank + 1) * a.entries / splits;
  const uint32_t tmem_cols = xrows <= 32 ? 32 : xrows <= 64 ? 64 : xrows <= 128 ? 128 : 256;

  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(&done, 1);
    abort_word = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(&tmem_holder, tmem_cols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_holder;
  if (!a.early) grid_dep_wait();
  grid_dep_trigger();

  if (warp == 0) {
    if (lane == 0) {
      bool ok = true;
      int stage = 0;
      uint32_t phase = 0;
      auto next = [&]() {
        if (++stage == stages) {
          stage = 0;
          phase ^= 1u;
        }
      };
      for (int kb = kb0; kb < kb1 && ok; ++kb) {
        ok = mbar_wait_bounded(&empty[stage], phase ^ 1u, a.err, kErrLoraWait, abort_flag);
        if (!ok) break;
        uint8_t* sw = smem + stage * stage_bytes;
        mbar_arrive_expect_tx(&full[stage], kWBytes + x_bytes);
        tma_load_2d(sw, &maps.w, kb * 64, n0, &full[stage]);
        tma_load_2d(sw + kWBytes, &maps.x, kb * 64, 0, &full[stage]);
        next();
      }
      if (e0 < e1 && ok) {
        int chunk = __ldg(a.entry_chunk + e0);
        grid_dep_wait();  // u is complete
        for (int e = e0; e < e1; e += 2) {
          const int n = min(2, e1 - e);
          ok = mbar_wait_bounded(&empty[stage], phase ^ 1u, a.err, kErrLoraWait, abort_flag);
          if (!ok) break;
          uint8_t* sb = smem + stage * stage_bytes;
          mbar_arrive_expect_tx(&full[stage], n * (kBBytes + 2 * u_bytes));
          for (int i = 0; i < n; ++i) {
            uint8_t* su = sb + kWBytes + i * 2 * u_bytes;
            tma_load_2d(sb + i * kBBytes, &maps.b, 0, chunk * a.b_rows + n0, &full[stage]);
            tma_load_2d(su, &maps.u, 0, (e + i) * kLoraBlock, &full[stage]);
            tma_load_2d(su + u_bytes, &maps.u, 16, (e + i) * kLoraBlock, &full[stage]);
            if (e + i + 1 < e1) chunk = __ldg(a.entry_chunk + e + i + 1);
          }
          next();
        }
      }
      if (!ok || *abort_flag) {
        // loads in flight land before the CTA leaves
        const unsigned long long t0 = global_ns();
        while (global_ns() - t0 < 2000000ull) __nanosleep(1000);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t idesc =
          std::is_same<T, __nv_bfloat16>::value ? umma_idesc_bf16(kCols, xrows) : umma_idesc_f16(kCols, xrows);
      bool ok = true;
      int stage = 0;
      uint32_t phase = 0;
      auto next = [&]() {
        umma_commit(&empty[stage]);
        if (++stage == stages) {
          stage = 0;
          phase ^= 1u;
        }
      };
      for (int kb = kb0; kb < kb1 && ok; ++kb) {
        ok = mbar_wait_bounded(&full[stage], phase, a.err, kErrLoraWait, abort_flag);
        if (!ok) break;
        tc_fence_after();
        const uint32_t w_addr = smem_u32(smem + stage * stage_bytes), x_addr = w_addr + kWBytes;
#pragma unroll
        for (int k = 0; k < 4; ++k)
          umma_f16(tmem, umma_desc_sw128(w_addr + k * 32), umma_desc_sw128(x_addr + k * 32), idesc,
                   (kb != kb0 || k != 0) ? 1u : 0u);
        next();
      }
      for (int e = e0; e < e1 && ok; e += 2) {
        ok = mbar_wait_bounded(&full[stage], phase, a.err, kErrLoraWait, abort_flag);
        if (!ok) break;
        tc_fence_after();
        const uint32_t b_addr = smem_u32(smem + stage * stage_bytes);
        for (int i = 0; i < min(2, e1 - e); ++i) {
          const uint64_t db = umma_desc_sw32(b_addr + i * kBBytes);
          const uint32_t su = b_addr + kWBytes + i * 2 * u_bytes;
          umma_f16(tmem, db, umma_desc_sw32(su), idesc, 1u);
          umma_f16(tmem, db, umma_desc_sw32(su + u_bytes), idesc, 1u);
        }
        next();
      }
      umma_commit(&done);
    }
    __syncwarp();
  }
  // this CTA's f32 part to shared memory (the ring is idle: every stage was
  // consumed): thread = output column, 16 rows at a time
  float* part = reinterpret_cast<float*>(smem);
  bool ok = mbar_wait_bounded(&done, 0, a.err, kErrLoraWait, nullptr) && !*abort_flag;
  ok = __syncthreads_and(ok);
  tc_fence_after();
  if (ok) {
    for (int m = 0; m < xrows; m += 16) {
      uint32_t v[16];
      tmem_ld_32x32b_x16(tmem + (static_cast<uint32_t>(warp * 32) << 16) + m, v);
      tmem_ld_wait();
#pragma unroll
      for (int j = 0; j < 16; ++j) part[(m + j) * kPartLd + threadIdx.x] = __uint_as_float(v[j]);
    }
  }
  tc_fence_before();
  if (splits > 1)
    cluster_sync();
  else
    __syncthreads();
  // rows rank, rank + splits, ...: 16 threads a row, 8 columns each
  const int col = n0 + static_cast<int>(threadIdx.x & 15) * 8;
  const int left = a.out - col;  // columns of this thread that exist
  for (int m = rank + static_cast<int>(threadIdx.x >> 4) * splits; m < a.rows && left > 0 && ok; m += 8 * splits) {
    const float* p = part + m * kPartLd + (threadIdx.x & 15) * 8;
    float4 s = ld_cluster_f4(p, 0), t = ld_cluster_f4(p + 4, 0);
    for (int c = 1; c < splits; ++c) {
      const float4 s1 = ld_cluster_f4(p, c), t1 = ld_cluster_f4(p + 4, c);
      s.x += s1.x, s.y += s1.y, s.z += s1.z, s.w += s1.w;
      t.x += t1.x, t.y += t1.y, t.z += t1.z, t.w += t1.w;
    }
    float v[8] = {s.x, s.y, s.z, s.w, t.x, t.y, t.z, t.w};
    if (a.bias) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < left) v[j] += __ldg(a.bias + col + j);
    }
    uint32_t o[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = pack2<T>(v[2 * j], v[2 * j + 1]);
    uint16_t* dst = static_cast<uint16_t*>(a.y) + static_cast<size_t>(m) * a.ldy + col;
    if (left >= 8) {
      *reinterpret_cast<uint4*>(dst) = make_uint4(o[0], o[1], o[2], o[3]);
    } else {
#pragma unroll
      for (int j = 0; j < 7; ++j)
        if (j < left) dst[j] = static_cast<uint16_t>(o[j / 2] >> (16 * (j & 1)));
    }
  }
  grid_dep_wait();  // this grid does not complete before the one that computes u
  if (splits > 1)
    cluster_sync();  // no CTA leaves while another may still read its part
  else
    __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, tmem_cols);
  }
}

template <class T>
cudaError_t launch(const SmallMaps& maps, const LoraSmallArgs& a, int splits, int stages, size_t smem, cudaStream_t s) {
  static bool configured[64] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  if (!configured[dev]) {
    e = cudaFuncSetAttribute(lora_small_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             static_cast<int>(kSmemLimit - 1024));
    if (e != cudaSuccess) return e;
    configured[dev] = true;
  }
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = splits;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  const dim3 grid((a.out + kCols - 1) / kCols * splits);
  return launch_pdl(lora_small_kernel<T>, grid, dim3(kThreads), smem, s, attr, 1, maps, a, splits, stages);
}

}  // namespace

cudaError_t launch_lora_small(const CUtensorMap& x, const CUtensorMap& w, const CUtensorMap& u, const CUtensorMap& b,
                              const LoraSmallArgs& a, int num_sms, cudaStream_t s) {
  if (a.rows <= 0) return cudaSuccess;
  if (a.rows > kLoraBlock || a.num_kb < 1) return cudaErrorInvalidValue;
  const int tiles = (a.out + kCols - 1) / kCols, xrows = (a.rows + 15) / 16 * 16;
  int splits = 1;
  while (splits < 8 && 2 * splits <= a.num_kb && tiles * splits < num_sms) splits *= 2;
  const int stage_bytes = kWBytes + (xrows * 128 + 1023) / 1024 * 1024;
  const int steps = (a.num_kb + splits - 1) / splits + ((a.entries + splits - 1) / splits + 1) / 2;
  const int room = static_cast<int>((kSmemLimit - 4096) / stage_bytes);
  const int stages = std::max(1, std::min(std::min(kMaxStages, steps), room));
  // A CTA waits for its cluster, so no CTA may be left waiting for TMEM that a
  // waiting one holds: shared memory in proportion to the TMEM columns (456 of
  // an SM's 233472 bytes a column, of its 512) keeps the columns of the CTAs
  // on an SM, of this kernel and the other clustered ones, within 512.
  const int cols = xrows <= 32 ? 32 : xrows <= 64 ? 64 : xrows <= 128 ? 128 : 256;
  const size_t smem = std::max(1024 + std::max(static_cast<size_t>(stages) * stage_bytes, sizeof(float) * xrows * kPartLd),
                               static_cast<size_t>(cols) * 456 - 1024);
  const SmallMaps maps{x, w, u, b};
  return a.bf16 ? launch<__nv_bfloat16>(maps, a, splits, stages, smem, s)
                : launch<__half>(maps, a, splits, stages, smem, s);
}

}  // namespace laya
