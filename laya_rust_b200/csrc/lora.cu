// A projection shared by many requests, each segment of rows with its own
// low-rank adapter or none (laya_lora_*):
//
//   y[m] = x[m] W^T + bias + s_a (x[m] A_a^T) B_a^T
//
// Two launches.  The first computes u = s_a (x A_a^T) in rank space, in f32, and
// rounds it to the 16-bit operands of the second product (lora.h says how).
// The second computes x W^T + u B^T in one f32 accumulator and rounds once: the
// tcgen05 GEMM of gemm.cu, whose K loop goes on over the adapters of its row block
// (GemmExt).  It is launched with programmatic serialization and waits for u only
// before its adapter steps.  A CTA of either fills an SM's shared memory, so its
// K loop starts beside the first launch only on the SMs that one leaves idle, and
// on the others as its CTAs end.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstring>
#include <memory>
#include <mutex>
#include <type_traits>
#include <utility>

#include "common.cuh"
#include "kernels.h"
#include "lora.h"
#include "ops_common.h"

namespace laya {

namespace {

template <class T>
struct Num;
template <>
struct Num<__half> {
  static __device__ __forceinline__ float up(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half down(float v) { return __float2half_rn(v); }
};
template <>
struct Num<__nv_bfloat16> {
  static __device__ __forceinline__ float up(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __nv_bfloat16 down(float v) { return __float2bfloat16_rn(v); }
};

// Elements from a value in u to its remainder.
constexpr int kRemainder = kLoraBlock * kLoraChunk;

template <class T>
__device__ __forceinline__ T* u_entry(void* u, int entry) {
  return static_cast<T*>(u) + static_cast<size_t>(entry) * kLoraEntryElems;
}
// Rank values j, j + 1 (j even) of a row of the batch into an entry.
template <class T>
__device__ __forceinline__ void store_u2(T* entry, int row, int j, float a, float b) {
  uint32_t hi, lo;
  lora_split<T>(a, b, hi, lo);
  T* d = entry + lora_at(row % kLoraBlock, j);
  *reinterpret_cast<uint32_t*>(d) = hi;
  *reinterpret_cast<uint32_t*>(d + kRemainder) = lo;
}
// All 16, as 16-byte stores.
template <class T>
__device__ __forceinline__ void store_u16(T* entry, int row, const float (&v)[16]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) lora_split<T>(v[8 * h + 2 * j], v[8 * h + 2 * j + 1], hi[j], lo[j]);
    T* d = entry + lora_at(row % kLoraBlock, 8 * h);
    *reinterpret_cast<uint4*>(d) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
    *reinterpret_cast<uint4*>(d + kRemainder) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
  }
}

constexpr int kXBytes = kLoraItemRows * 64 * 2;   // x operand of a k-block: 16 KB
constexpr int kABytes = kLoraChunk * 64 * 2;      // one entry's A operand: 2 KB
constexpr int kRingBytes = 192 * 1024;
constexpr int kMaxStages = 8;
constexpr size_t kShrinkSmem = 1024 + kRingBytes;

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t map_to_rank(const void* p, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ void bulk_to_rank(const void* dst, uint64_t* bar, const void* src, uint32_t bytes, uint32_t rank) {
  asm volatile("cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   map_to_rank(dst, rank)),
               "r"(smem_u32(src)), "r"(bytes), "r"(map_to_rank(bar, rank))
               : "memory");
}

// u = scale (x A^T) for one item: 128 rows against up to 8 entries (M = 128,
// N = 16 entries), K cut over the CTAs of a cluster.  Per CTA: warp 0 loads
// (TMA ring of x and A k-blocks), warp 1 issues the MMAs, warps 2 and 3 look up
// the rows' adapters.  Then a thread has its row's sums in TMEM: alone it stores
// them; in a cluster each CTA owns a share of the rows, the others send it
// their sums with one bulk copy each, and it adds them in rank order.
// Bound by the latency of its chain (loads, MMA, exchange): about 5 us for 9872
// rows, 1024 inputs, 16 adapters of rank 16, where x alone is 3 us of HBM.
template <class T, int SPLITS>
__global__ void __launch_bounds__(128, 1)
    lora_shrink_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmA,
                       const LoraShrinkArgs a) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t full[kMaxStages], empty[kMaxStages], done, in_full, stuck_bar;
  __shared__ uint32_t tmem_holder;
  __shared__ int abort_word;
  __shared__ int row_slot[kLoraItemRows];
  __shared__ float row_scale[kLoraItemRows];
  __shared__ int item_entry[kLoraMaxGroup], item_slot[kLoraMaxGroup];
  volatile int* abort_flag = &abort_word;
  uint8_t* smem = smem_raw + (((smem_u32(smem_raw) + 1023u) & ~1023u) - smem_u32(smem_raw));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = SPLITS > 1 ? static_cast<int>(cluster_rank()) : 0;
  const int4 item = __ldg(a.item + blockIdx.x / SPLITS);
  const int n = item.z;
  const int stage_bytes = kXBytes + a.group * kABytes;
  // the sums, apart from the ring: [128][ld] and, sent here, [SPLITS - 1][own rows][ld]
  const int ld = 16 * a.group + 4, own_rows = kLoraItemRows / SPLITS;
  const int part_bytes = SPLITS > 1 ? 2 * kLoraItemRows * ld * 4 : 0;
  const int stages = min(kMaxStages, (kRingBytes - part_bytes) / stage_bytes);
  float* part = reinterpret_cast<float*>(smem + kRingBytes - part_bytes);
  float* part_in = part + kLoraItemRows * ld;
  const int kb0 = rank * a.num_kb / SPLITS, kb1 = (rank + 1) * a.num_kb / SPLITS;
  const uint32_t tmem_cols = a.group <= 2 ? 32 : 16 * a.group;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kMaxStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(&done, 1);
    mbar_init(&in_full, 1);
    mbar_init(&stuck_bar, 1);
    abort_word = 0;
    fence_mbar_init();
    if (SPLITS > 1)
      mbar_arrive_expect_tx(&in_full, (SPLITS - 1) * own_rows * ld * 4 + (a.stuck == kLoraStuckExchange ? 16 : 0));
    tma_prefetch_desc(&tmX);
    tma_prefetch_desc(&tmA);
  }
  if (warp == 1) {
    tmem_alloc(&tmem_holder, tmem_cols);
    tmem_relinquish();
  }
  // lane i of warp 0 holds entry i's row of A
  const int a_row = warp == 0 && lane < n ? __ldg(a.item_chunk + item.y + lane) * kLoraChunk : 0;
  __syncwarp();
  if (SPLITS > 1) cluster_arrive();  // this CTA's shared memory exists
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_holder;
  // everything above reads only the plan
  grid_dep_wait();
  grid_dep_trigger();

  if (warp == 0) {
    int a_rows[kLoraMaxGroup];
#pragma unroll
    for (int i = 0; i < kLoraMaxGroup; ++i) a_rows[i] = __shfl_sync(0xffffffffu, a_row, i);
    if (elect_one()) {
      bool ok = true;
      int stage = 0;
      uint32_t phase = 0;
      if (a.stuck == kLoraStuckLoads)
        ok = mbar_wait_bounded(&stuck_bar, 0, a.err, kErrLoraWait, abort_flag, a.wait_limit_ns);
      for (int kb = kb0; kb < kb1 && ok; ++kb) {
        ok = mbar_wait_bounded(&empty[stage], phase ^ 1u, a.err, kErrLoraWait, abort_flag);
        if (!ok) break;
        uint8_t* sx = smem + stage * stage_bytes;
        mbar_arrive_expect_tx(&full[stage], kXBytes + n * kABytes);
        tma_load_2d(sx, &tmX, kb * 64, item.x * kLoraItemRows, &full[stage]);
#pragma unroll
        for (int i = 0; i < kLoraMaxGroup; ++i)
          if (i < n) tma_load_2d(sx + kXBytes + i * kABytes, &tmA, kb * 64, a_rows[i], &full[stage]);
        if (++stage == stages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      if (!ok || *abort_flag) wait_for_copies();
    }
    __syncwarp();
  } else if (warp == 1) {
    if (elect_one()) {
      const uint32_t idesc = std::is_same<T, __nv_bfloat16>::value ? umma_idesc_bf16(kLoraItemRows, 16 * n)
                                                                    : umma_idesc_f16(kLoraItemRows, 16 * n);
      int stage = 0;
      uint32_t phase = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait_bounded(&full[stage], phase, a.err, kErrLoraWait, abort_flag)) break;
        tc_fence_after();
        const uint32_t x_addr = smem_u32(smem + stage * stage_bytes), a_addr = x_addr + kXBytes;
#pragma unroll
        for (int k = 0; k < 4; ++k)
          umma_f16(tmem, umma_desc_sw128(x_addr + k * 32), umma_desc_sw128(a_addr + k * 32), idesc,
                   (kb != kb0 || k != 0) ? 1u : 0u);
        umma_commit(&empty[stage]);
        if (++stage == stages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      umma_commit(&done);
    }
    __syncwarp();
  } else {
    for (int r = static_cast<int>(threadIdx.x) - 64; r < kLoraItemRows; r += 64) {
      const int row = item.x * kLoraItemRows + r;
      const int e0 = row < a.rows ? __ldg(a.row_entry + row) : -1;
      const int slot = e0 >= 0 ? __ldg(a.entry_chunk + e0) / a.chunks_per_slot : -1;
      row_slot[r] = slot;
      row_scale[r] = slot >= 0 ? __ldg(a.scale + slot) : 0.0f;
    }
    const int i = static_cast<int>(threadIdx.x) - 64;
    if (i < n) {
      item_entry[i] = __ldg(a.item_entry + item.y + i);
      item_slot[i] = __ldg(a.item_chunk + item.y + i) / a.chunks_per_slot;
    }
  }
  bool ok = mbar_wait_bounded(&done, 0, a.err, kErrLoraWait, nullptr) && !*abort_flag;
  ok = __syncthreads_and(ok);
  tc_fence_after();
  const uint32_t lane_base = static_cast<uint32_t>(warp * 32) << 16;
  if constexpr (SPLITS == 1) {
    const int r = threadIdx.x;
    const int slot = ok ? row_slot[r] : -1;
    const float scale = row_scale[r];
    for (int i = 0; i < n; ++i) {
      uint32_t v[16];
      tmem_ld_32x32b_x16(tmem + lane_base + i * 16, v);
      tmem_ld_wait();
      if (item_slot[i] == slot) {
        float f[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) f[j] = __uint_as_float(v[j]) * scale;
        store_u16<T>(u_entry<T>(a.u, item_entry[i]), item.x * kLoraItemRows + r, f);
      }
      __syncwarp();  // the next load takes a whole warp
    }
    tc_fence_before();
    __syncthreads();
  } else {
    cluster_wait();  // every CTA of the cluster has started
    for (int i = 0; i < n; ++i) {
      uint32_t v[16];
      tmem_ld_32x32b_x16(tmem + lane_base + i * 16, v);
      tmem_ld_wait();
      uint4* dst = reinterpret_cast<uint4*>(part + threadIdx.x * ld + i * 16);
#pragma unroll
      for (int j = 0; j < 4; ++j) dst[j] = make_uint4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
    }
    tc_fence_before();
    fence_proxy_async_smem();
    __syncthreads();
    const int to = static_cast<int>(threadIdx.x);
    if (to < SPLITS && to != rank)
      bulk_to_rank(part_in + (rank < to ? rank : rank - 1) * own_rows * ld, &in_full, part + to * own_rows * ld,
                   own_rows * ld * 4, to);
    if (!mbar_wait_bounded(&in_full, 0, a.err, kErrLoraWait, nullptr, a.wait_limit_ns)) {
      ok = false;
      wait_for_copies();
    }
    __syncwarp();
    cluster_arrive();  // what this CTA was sent has landed
    // SPLITS threads a row, each every SPLITS-th entry
    const int q = static_cast<int>(threadIdx.x) / SPLITS, r = rank * own_rows + q;
    const int slot = ok ? row_slot[r] : -1;
    for (int i = static_cast<int>(threadIdx.x) % SPLITS; i < n && slot >= 0; i += SPLITS) {
      if (item_slot[i] != slot) continue;
      float f[16];
#pragma unroll
      for (int c = 0; c < SPLITS; ++c) {
        const float* p = (c == rank ? part + r * ld : part_in + ((c < rank ? c : c - 1) * own_rows + q) * ld) + i * 16;
#pragma unroll
        for (int j = 0; j < 16; ++j) f[j] = c == 0 ? p[j] : f[j] + p[j];
      }
#pragma unroll
      for (int j = 0; j < 16; ++j) f[j] *= row_scale[r];
      store_u16<T>(u_entry<T>(a.u, item_entry[i]), item.x * kLoraItemRows + r, f);
    }
    __syncwarp();
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, tmem_cols);
  }
  __syncwarp();
  if (SPLITS > 1) cluster_wait();  // no CTA leaves while a copy may still read its part
}

// u = scale (x A^T) for one (row, chunk) pair a block: a warp takes two of the
// chunk's 16 rows of A over all of K, so no sum leaves its warp.  A is read once
// a pair, 32 bytes an input and pair from HBM or L2 (48 rows with an adapter each,
// 1024 inputs, with the projection behind it: 10.5 us, by items 13.4).
template <class T>
__global__ void __launch_bounds__(256) lora_pairs_kernel(const LoraPairsArgs a) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int4 p = __ldg(a.pair + blockIdx.x);
  grid_dep_wait();
  grid_dep_trigger();
  const float scale = __ldg(a.scale + p.w);
  const T* x = static_cast<const T*>(a.x) + p.x * a.ldx;
  const T* A0 = static_cast<const T*>(a.a) + (static_cast<size_t>(p.z) * kLoraChunk + 2 * warp) * a.in_pad;
  const T* A1 = A0 + a.in_pad;
  float s0 = 0.0f, s1 = 0.0f;
  const int whole = a.in & ~7;  // the rest of a row of x may hold anything
#pragma unroll 4
  for (int k = 8 * lane; k < whole; k += 256) {
    const uint4 xv = *reinterpret_cast<const uint4*>(x + k);
    const uint4 av = __ldg(reinterpret_cast<const uint4*>(A0 + k)), bv = __ldg(reinterpret_cast<const uint4*>(A1 + k));
    const T* xe = reinterpret_cast<const T*>(&xv);
    const T* ae = reinterpret_cast<const T*>(&av);
    const T* be = reinterpret_cast<const T*>(&bv);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float v = Num<T>::up(xe[j]);
      s0 += v * Num<T>::up(ae[j]);
      s1 += v * Num<T>::up(be[j]);
    }
  }
  if (lane < a.in - whole) {
    const float v = Num<T>::up(x[whole + lane]);
    s0 += v * Num<T>::up(A0[whole + lane]);
    s1 += v * Num<T>::up(A1[whole + lane]);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    s0 += __shfl_xor_sync(0xffffffffu, s0, o);
    s1 += __shfl_xor_sync(0xffffffffu, s1, o);
  }
  if (lane == 0) {
    store_u2<T>(u_entry<T>(a.u, p.y), p.x, 2 * warp, s0 * scale, s1 * scale);
  }
}

template <class T, int SPLITS>
cudaError_t launch_shrink(const CUtensorMap& x, const CUtensorMap& a_map, const LoraShrinkArgs& a, cudaStream_t s) {
  static std::atomic<bool> configured[64] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  if (!configured[dev]) {
    e = cudaFuncSetAttribute(lora_shrink_kernel<T, SPLITS>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             static_cast<int>(kShrinkSmem));
    if (e != cudaSuccess) return e;
    configured[dev] = true;
  }
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = SPLITS;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  return launch_pdl(lora_shrink_kernel<T, SPLITS>, dim3(a.items * SPLITS), dim3(128), kShrinkSmem, s, attr, 1, x, a_map, a);
}

template <class T>
cudaError_t launch_shrink(int splits, const CUtensorMap& x, const CUtensorMap& a_map, const LoraShrinkArgs& a,
                          cudaStream_t s) {
  switch (splits) {
    case 1: return launch_shrink<T, 1>(x, a_map, a, s);
    case 2: return launch_shrink<T, 2>(x, a_map, a, s);
    case 4: return launch_shrink<T, 4>(x, a_map, a, s);
    default: return launch_shrink<T, 8>(x, a_map, a, s);
  }
}

}  // namespace

cudaError_t launch_lora_shrink(const CUtensorMap& x, const CUtensorMap& a_map, const LoraShrinkArgs& a, int num_sms,
                               cudaStream_t s) {
  if (a.items <= 0) return cudaSuccess;
  if (a.num_kb < 1 || a.group < 1 || a.group > kLoraMaxGroup) return cudaErrorInvalidValue;
  // by the rows and K alone: a row's sums keep their order whatever adapters
  // the other rows have
  int splits = lora_splits(a.rows, num_sms);
  while (splits > 1 && 2 * splits > a.num_kb) splits /= 2;
  return a.bf16 ? launch_shrink<__nv_bfloat16>(splits, x, a_map, a, s) : launch_shrink<__half>(splits, x, a_map, a, s);
}

cudaError_t launch_lora_pairs(const LoraPairsArgs& a, cudaStream_t s) {
  if (a.pairs <= 0) return cudaSuccess;
  auto* kernel = a.bf16 ? &lora_pairs_kernel<__nv_bfloat16> : &lora_pairs_kernel<__half>;
  return launch_pdl(kernel, dim3(a.pairs), dim3(256), 0, s, nullptr, 0, a);
}

// As many parts as keep every item on an SM (3034 rows, 1024 -> 3072, 16 adapters:
// 4 parts 24.5 us, 8 parts 34; 10387 rows: 1 part 63 us, 2 parts 75).
int lora_splits(int rows, int num_sms) {
  const int halves = (rows + kLoraItemRows - 1) / kLoraItemRows;
  int splits = 1;
  while (splits < 8 && 2 * splits * halves <= lora_cluster_room(2 * splits, num_sms)) splits *= 2;
  return splits;
}

LoraItems lora_items(const LoraLayout& L, int num_sms) {
  // the entries of each 128 rows, by the order of their first row
  LoraItems it;
  const int halves = (L.rows + kLoraItemRows - 1) / kLoraItemRows;
  std::vector<std::vector<int>> need(halves);
  for (int h = 0; h < halves; ++h) {
    std::vector<int>& v = need[h];
    int last = -1;
    for (int m = h * kLoraItemRows; m < std::min(L.rows, (h + 1) * kLoraItemRows); ++m) {
      const int e0 = L.row_entry[m];
      if (e0 < 0 || e0 == last) continue;
      last = e0;
      if (std::find(v.begin(), v.end(), e0) != v.end()) continue;
      for (int e = e0; e < static_cast<int>(L.chunk.size()) && (e == e0 || L.chunk[e].y > 0); ++e) v.push_back(e);
    }
  }
  // the smallest group whose items still run at once (10387 rows of 16 adapters,
  // 1024 -> 3072, in all: groups of 1 entry 67 us, of 2 as chosen here 63; 3034
  // rows: 1 or 2 28.6 us, 4 as chosen 24.6, 8 27.7)
  const size_t most = num_sms / lora_splits(L.rows, num_sms);
  for (it.group = 1;; it.group *= 2) {
    size_t items = 0;
    for (const auto& v : need) items += (v.size() + it.group - 1) / it.group;
    if (items <= most || it.group == kLoraMaxGroup) break;
  }
  for (int h = 0; h < halves; ++h)
    for (size_t i = 0; i < need[h].size(); i += it.group) {
      const int n = static_cast<int>(std::min<size_t>(it.group, need[h].size() - i));
      it.item.push_back(make_int4(h, static_cast<int>(it.entry.size()), n, 0));
      it.entry.insert(it.entry.end(), need[h].begin() + i, need[h].begin() + i + n);
    }
  return it;
}

namespace {

float bits_f32(uint32_t u) {
  float f;
  memcpy(&f, &u, 4);
  return f;
}
uint32_t f32_bits(float f) {
  uint32_t u;
  memcpy(&u, &f, 4);
  return u;
}

float host_f32(const void* p, int type, size_t i) {
  if (type == LAYA_F32) return static_cast<const float*>(p)[i];
  const uint16_t v = static_cast<const uint16_t*>(p)[i];
  if (type == LAYA_BF16) return bits_f32(static_cast<uint32_t>(v) << 16);
  __half_raw r;
  r.x = v;
  return __half2float(__half(r));
}

// Nearest value of the 16-bit type, ties to even; false if it is not finite.
bool host_bf16(float f, uint16_t* out) {
  const uint32_t u = f32_bits(f);
  const uint32_t r = u + 0x7fffu + ((u >> 16) & 1u);
  *out = static_cast<uint16_t>(r >> 16);
  return (u & 0x7f800000u) != 0x7f800000u && (r & 0x7f800000u) != 0x7f800000u;
}
bool host_f16(float f, uint16_t* out) {
  const uint32_t u = f32_bits(f), sign = (u >> 16) & 0x8000u, mag = u & 0x7fffffffu;
  if (mag >= 0x477ff000u) return false;  // rounds to 65536 or more, or is not finite
  uint32_t h;
  if (mag < 0x38800000u)  // below 2^-14: the sum with 1/2 rounds at 2^-24, f16's last place there
    h = f32_bits(bits_f32(mag) + 0.5f) - 0x3f000000u;
  else
    h = (mag - 0x38000000u + 0x0fffu + ((mag >> 13) & 1u)) >> 13;
  *out = static_cast<uint16_t>(sign | h);
  return true;
}
uint16_t host_round(const void* p, int type, size_t i, bool bf16) {
  // the type's own values pass through when they are finite
  uint16_t h;
  const float f = host_f32(p, type, i);
  op_require(bf16 ? host_bf16(f, &h) : host_f16(f, &h), "adapter: a value is not finite in the projection's type");
  return h;
}

}  // namespace

std::vector<uint16_t> lora_pack_a(const void* a, int type, int rank, int in, int in_pad, bool bf16) {
  std::vector<uint16_t> v(static_cast<size_t>(lora_chunks(rank)) * kLoraChunk * in_pad);
  for (int r = 0; r < rank; ++r)
    for (int c = 0; c < in; ++c)
      v[static_cast<size_t>(r) * in_pad + c] = host_round(a, type, static_cast<size_t>(r) * in + c, bf16);
  return v;
}

std::vector<uint16_t> lora_pack_b(const void* b, int type, int rank, int out, int out_pad, bool bf16,
                                  const std::vector<int>& row_of) {
  std::vector<uint16_t> v(static_cast<size_t>(lora_chunks(rank)) * out_pad * kLoraChunk);
  for (int n = 0; n < out; ++n) {
    const int row = row_of.empty() ? n : row_of[n];
    for (int r = 0; r < rank; ++r)
      v[static_cast<size_t>(r / kLoraChunk) * out_pad * kLoraChunk + lora_at(row, r % kLoraChunk)] =
          host_round(b, type, static_cast<size_t>(n) * rank + r, bf16);
  }
  return v;
}

LoraLayout lora_layout(const int32_t* rows, const int32_t* slot, int n, const std::vector<int>& chunks_of) {
  op_require(n >= 0 && (n == 0 || (rows && slot)), "lora plan: null segments");
  LoraLayout L;
  int64_t total = 0;
  const int slots = static_cast<int>(chunks_of.size());
  for (int i = 0; i < n; ++i) {
    op_require(rows[i] >= 0, "lora plan: a segment has a negative number of rows");
    op_require(slot[i] == LAYA_LORA_NONE || (slot[i] >= 0 && slot[i] < slots), "lora plan: slot out of range");
    op_require(rows[i] == 0 || slot[i] < 0 || chunks_of[slot[i]] > 0, "lora plan: a segment's slot is empty");
    total += rows[i];
    op_require(total <= LAYA_LORA_MAX_ROWS, "lora plan: too many rows");
  }
  L.rows = static_cast<int>(total);
  L.row_entry.resize(total);
  L.off.push_back(0);
  std::vector<int> first(slots, -1), used;  // a slot's first entry in the current block
  int seg = 0, left = n > 0 ? rows[0] : 0;
  for (int m = 0; m < L.rows; ++m) {
    while (left == 0) left = rows[++seg];
    --left;
    const int s = slot[seg];
    if (s < 0) {
      L.row_entry[m] = -1;
    } else {
      if (first[s] < 0) {
        first[s] = static_cast<int>(L.chunk.size());
        used.push_back(s);
        for (int c = 0; c < chunks_of[s]; ++c) L.chunk.push_back(make_int2(s, c));
        op_require(L.chunk.size() < (size_t{1} << 21), "lora plan: too many adapters in one batch");
      }
      L.row_entry[m] = first[s];
    }
    if ((m + 1) % kLoraBlock == 0 || m + 1 == L.rows) {
      L.off.push_back(static_cast<int>(L.chunk.size()));
      for (int u : used) first[u] = -1;
      used.clear();
    }
  }
  return L;
}

namespace {

struct Buf {
  void* p = nullptr;
  ~Buf() {
    if (p) cudaFree(p);
  }
  void alloc(size_t bytes, const char* what) { op_check(cudaMalloc(&p, bytes ? bytes : 256), what); }
  template <class T>
  T* as() const {
    return static_cast<T*>(p);
  }
};

struct Slot {
  int rank = 0;     // 0: empty
};

// The adapters of one projection on one device.
struct Bank {
  int device = 0, num_sms = 0;
  bool bf16 = false;
  int in = 0, out = 0, in_pad = 0, out_pad = 0, slots = 0, max_rank = 0, cps = 0;
  const void* w = nullptr;
  long long ldw = 0;
  const float* bias = nullptr;
  // Held while an adapter is replaced and while a run is checked and enqueued: a
  // run that another thread enqueues comes before or after the whole of it.
  mutable std::mutex lock;
  std::vector<Slot> slot;
  Buf a, b, scale;
  CUtensorMap a_map;
  CUtensorMap b_map[2];  // B for 256- and 128-column tiles
  cudaStream_t stream = nullptr;  // uploads
  ~Bank() {
    int prev = -1;
    cudaGetDevice(&prev);
    cudaSetDevice(device);
    if (stream) cudaStreamDestroy(stream);
    for (Buf* x : {&a, &b, &scale}) {
      if (x->p) cudaFree(x->p);
      x->p = nullptr;
    }
    if (prev >= 0) cudaSetDevice(prev);
  }
  std::vector<int> chunks_of() const {
    std::vector<int> c(slot.size());
    for (size_t i = 0; i < slot.size(); ++i) c[i] = lora_chunks(slot[i].rank);
    return c;
  }
};

struct Plan {
  std::shared_ptr<Bank> bank;
  LoraLayout lay;
  std::vector<std::pair<int, int>> used;  // (slot, chunks)
  Buf dev, u;
  int stuck_kind = -1;  // laya_lora_test_timeout_next
  unsigned long long stuck_limit_ns = 0;
  LoraSmallPlan small;  // use: lora_small.cu, not the GEMM
  int items = 0, group = 0;
  const int4* d_item = nullptr;
  const int* d_item_entry = nullptr;
  const int* d_item_chunk = nullptr;
  const int4* d_pair = nullptr;
  const int* d_soff = nullptr;
  const int2* d_list = nullptr;
  int pairs = 0;  // > 0: the rank-space product goes by pairs, not items
  const int* d_row_entry = nullptr;
  const int* d_entry_chunk = nullptr;
  const int* d_off = nullptr;
  int* d_err = nullptr;
  CUtensorMap u_map;
  ~Plan() {
    int prev = -1;
    cudaGetDevice(&prev);
    if (bank) cudaSetDevice(bank->device);
    for (Buf* x : {&dev, &u}) {
      if (x->p) cudaFree(x->p);
      x->p = nullptr;
    }
    if (prev >= 0) cudaSetDevice(prev);
  }
};

// The rank-space product by (row, chunk) pairs, a block each that reads 16 rows of
// A, or by items of 128 rows?  Pairs while they are few, or few of them share
// an adapter's chunk: 256 rows with an adapter each, 1024 -> 3072: 22.5 us, by items
// 38; 2048 rows in turn with 256 adapters 100 and 159 us; 128 segments of 8 rows, 16
// adapters, 18 and 26 us; but 64 segments of 16 rows, 64 adapters of rank 64, 2624
// -> 1024 (4096 pairs of 256 chunks): 53 and 41 us.
bool lora_by_pairs(size_t pairs, size_t entries) { return pairs <= 1024 || pairs <= 8 * entries; }

constexpr uint64_t kMaxStuckNs = 2000000000;  // laya_lora_test_timeout_next

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

}  // namespace
}  // namespace laya

using namespace laya;

struct laya_lora {
  std::shared_ptr<Bank> bank;
};
struct laya_lora_plan {
  Plan p;
};

extern "C" {

int laya_lora_create(int device, int type, int64_t in, int64_t out, const void* w, int64_t ldw, const float* bias,
                     int slots, int max_rank, laya_lora** lora) {
  return op_guard([&] {
    op_require(lora, "lora_create: null argument");
    *lora = nullptr;
    op_require(w, "lora_create: null weight");
    op_require(type == LAYA_F16 || type == LAYA_BF16, "lora_create: type must be LAYA_F16 or LAYA_BF16");
    op_require(in >= 1 && in <= (1 << 20) && out >= 1 && out <= (1 << 20), "lora_create: in and out must be 1..2^20");
    op_require(ldw >= in && ldw <= (int64_t{1} << 30), "lora_create: ldw is smaller than in");
    op_require(aligned16(w) && ldw % 8 == 0, "lora_create: W and its pitch must be multiples of 16 bytes");
    op_require(reinterpret_cast<uintptr_t>(bias) % 4 == 0, "lora_create: bias is not aligned");
    op_require(slots >= 1 && slots <= LAYA_LORA_MAX_SLOTS, "lora_create: slots must be 1..LAYA_LORA_MAX_SLOTS");
    op_require(max_rank >= 1 && max_rank <= LAYA_LORA_MAX_RANK, "lora_create: max_rank must be 1..LAYA_LORA_MAX_RANK");
    const int64_t in_pad = (in + 63) / 64 * 64, out_pad = (out + 255) / 256 * 256;
    const int64_t chunks = static_cast<int64_t>(slots) * lora_chunks(max_rank);
    // the kernels address chunks through 32-bit TMA row coordinates
    op_require(chunks * out_pad < (int64_t{1} << 31), "lora_create: slots * max_rank * out is too large");
    DeviceScope scope(device);
    require_device_ptr(w, device, "lora_create: W");
    if (bias) require_device_ptr(bias, device, "lora_create: bias");
    auto k = std::make_shared<Bank>();
    k->device = device;
    int major = 0;
    op_check(cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, device), "device query");
    if (major != 10) throw OpError(LAYA_E_CUDA, "lora_create: this build targets sm_100a (B200)");
    op_check(cudaDeviceGetAttribute(&k->num_sms, cudaDevAttrMultiProcessorCount, device), "device query");
    k->bf16 = type == LAYA_BF16;
    k->in = static_cast<int>(in);
    k->out = static_cast<int>(out);
    k->in_pad = static_cast<int>(in_pad);
    k->out_pad = static_cast<int>(out_pad);
    k->slots = slots;
    k->max_rank = max_rank;
    k->cps = lora_chunks(max_rank);
    k->w = w;
    k->ldw = ldw;
    k->bias = bias;
    k->slot.resize(slots);
    op_check(cudaStreamCreateWithFlags(&k->stream, cudaStreamNonBlocking), "lora stream");
    k->a.alloc(chunks * kLoraChunk * in_pad * 2, "lora adapters");
    k->b.alloc(chunks * kLoraChunk * out_pad * 2, "lora adapters");
    k->scale.alloc(sizeof(float) * slots, "lora scales");
    op_check(cudaMemsetAsync(k->a.p, 0, chunks * kLoraChunk * in_pad * 2, k->stream), "lora clear");
    op_check(cudaMemsetAsync(k->b.p, 0, chunks * kLoraChunk * out_pad * 2, k->stream), "lora clear");
    op_check(cudaMemsetAsync(k->scale.p, 0, sizeof(float) * slots, k->stream), "lora clear");
    op_check(cudaStreamSynchronize(k->stream), "lora clear");
    if (make_tmap_pitched(&k->a_map, k->a.p, k->bf16, chunks * kLoraChunk, in_pad, in_pad, kLoraChunk) ||
        make_tmap_lora(&k->b_map[0], k->b.p, k->bf16, chunks * out_pad, kGemmBBoxRows) ||
        make_tmap_lora(&k->b_map[1], k->b.p, k->bf16, chunks * out_pad, kGemmBBoxRowsNarrow))
      throw OpError(LAYA_E_CUDA, "lora_create: tensor map encode failed");
    *lora = new laya_lora{k};
  });
}

int laya_lora_set(laya_lora* lora, int slot, int rank, const void* a, const void* b, int host_type, float scale) {
  return op_guard([&] {
    op_require(lora && a && b, "lora_set: null argument");
    Bank& k = *lora->bank;
    op_require(slot >= 0 && slot < k.slots, "lora_set: slot out of range");
    op_require(rank >= 1 && rank <= k.max_rank, "lora_set: rank must be 1..max_rank");
    op_require(host_type == LAYA_F16 || host_type == LAYA_BF16 || host_type == LAYA_F32, "lora_set: unknown type");
    op_require(std::isfinite(scale), "lora_set: scale is not finite");
    const std::vector<uint16_t> ha = lora_pack_a(a, host_type, rank, k.in, k.in_pad, k.bf16);
    const std::vector<uint16_t> hb = lora_pack_b(b, host_type, rank, k.out, k.out_pad, k.bf16, {});
    const std::lock_guard<std::mutex> held(k.lock);
    DeviceScope scope(k.device);
    // runs already queued on the caller's streams may still read the slot
    op_check(cudaDeviceSynchronize(), "lora_set");
    const size_t na = static_cast<size_t>(k.cps) * kLoraChunk * k.in_pad, nb = static_cast<size_t>(k.cps) * kLoraChunk * k.out_pad;
    uint16_t* da = k.a.as<uint16_t>() + na * slot;
    uint16_t* db = k.b.as<uint16_t>() + nb * slot;
    op_check(cudaMemcpyAsync(da, ha.data(), ha.size() * 2, cudaMemcpyHostToDevice, k.stream), "lora upload");
    op_check(cudaMemcpyAsync(db, hb.data(), hb.size() * 2, cudaMemcpyHostToDevice, k.stream), "lora upload");
    // chunks an earlier, larger rank used
    op_check(cudaMemsetAsync(da + ha.size(), 0, (na - ha.size()) * 2, k.stream), "lora upload");
    op_check(cudaMemsetAsync(db + hb.size(), 0, (nb - hb.size()) * 2, k.stream), "lora upload");
    op_check(cudaMemcpyAsync(k.scale.as<float>() + slot, &scale, 4, cudaMemcpyHostToDevice, k.stream), "lora upload");
    op_check(cudaStreamSynchronize(k.stream), "lora upload");
    k.slot[slot].rank = rank;
  });
}

int laya_lora_clear(laya_lora* lora, int slot) {
  return op_guard([&] {
    op_require(lora, "lora_clear: null argument");
    op_require(slot >= 0 && slot < lora->bank->slots, "lora_clear: slot out of range");
    const std::lock_guard<std::mutex> held(lora->bank->lock);
    lora->bank->slot[slot].rank = 0;
  });
}

void laya_lora_destroy(laya_lora* lora) { delete lora; }

int laya_lora_plan_create(laya_lora* lora, const int32_t* rows, const int32_t* slot, int n, laya_lora_plan** plan) {
  return op_guard([&] {
    op_require(lora && plan, "lora_plan_create: null argument");
    *plan = nullptr;
    auto p = std::make_unique<laya_lora_plan>();
    Plan& q = p->p;
    q.bank = lora->bank;
    const Bank& k = *q.bank;
    std::vector<int> chunks;
    {
      const std::lock_guard<std::mutex> held(k.lock);
      chunks = k.chunks_of();
    }
    q.lay = lora_layout(rows, slot, n, chunks);
    const LoraLayout& L = q.lay;
    std::vector<int> entry_chunk;
    for (const int2& c : L.chunk) {
      entry_chunk.push_back(c.x * k.cps + c.y);
      if (c.y == 0) q.used.emplace_back(c.x, chunks[c.x]);
    }
    std::sort(q.used.begin(), q.used.end());
    q.used.erase(std::unique(q.used.begin(), q.used.end()), q.used.end());
    DeviceScope scope(k.device);
    q.small = lora_small_plan(L, k.out, k.cps, k.num_sms);
    // u apart from the projection: few (row, chunk) pairs one block each, else
    // items of 128 rows
    const bool u_apart = !q.small.fused;
    std::vector<int4> pair;
    for (int m = 0; u_apart && m < L.rows && lora_by_pairs(pair.size(), L.chunk.size()); ++m) {
      const int e0 = L.row_entry[m];
      if (e0 < 0) continue;
      for (int e = e0; e < static_cast<int>(L.chunk.size()) && (e == e0 || L.chunk[e].y > 0); ++e)
        pair.push_back(make_int4(m, e, entry_chunk[e], L.chunk[e].x));
    }
    LoraItems it;
    if (!u_apart) {
    } else if (lora_by_pairs(pair.size(), L.chunk.size())) {
      q.pairs = static_cast<int>(pair.size());
    } else {
      pair.clear();
      it = lora_items(L, k.num_sms);
    }
    std::vector<int> item_chunk;
    for (int e : it.entry) item_chunk.push_back(entry_chunk[e]);
    q.items = static_cast<int>(it.item.size());
    q.group = it.group;
    // [error word | off | row entries | entry chunks | items | their entries |
    // their chunks | pairs | row tiles' lists], each 256-byte aligned
    auto up = [](size_t v) { return (v + 63) / 64 * 64; };
    const size_t o_off = 64, o_row = o_off + up(L.off.size()), o_ent = o_row + up(L.row_entry.size());
    const size_t o_item = o_ent + up(entry_chunk.size()), o_ie = o_item + up(4 * it.item.size());
    const size_t o_ic = o_ie + up(it.entry.size()), o_pair = o_ic + up(item_chunk.size());
    const size_t o_soff = o_pair + up(4 * pair.size()), o_list = o_soff + up(q.small.off.size());
    std::vector<int> h(o_list + up(2 * q.small.list.size()));
    std::copy(q.small.off.begin(), q.small.off.end(), h.begin() + o_soff);
    if (!q.small.list.empty()) memcpy(h.data() + o_list, q.small.list.data(), q.small.list.size() * sizeof(int2));
    if (!pair.empty()) memcpy(h.data() + o_pair, pair.data(), pair.size() * sizeof(int4));
    std::copy(item_chunk.begin(), item_chunk.end(), h.begin() + o_ic);
    if (!it.item.empty()) memcpy(h.data() + o_item, it.item.data(), it.item.size() * sizeof(int4));
    std::copy(it.entry.begin(), it.entry.end(), h.begin() + o_ie);
    std::copy(L.off.begin(), L.off.end(), h.begin() + o_off);
    std::copy(L.row_entry.begin(), L.row_entry.end(), h.begin() + o_row);
    std::copy(entry_chunk.begin(), entry_chunk.end(), h.begin() + o_ent);
    q.dev.alloc(h.size() * 4, "lora plan");
    const size_t entries = std::max<size_t>(1, L.chunk.size());
    q.u.alloc(entries * kLoraEntryElems * 2, "lora workspace");
    if (make_tmap_lora(&q.u_map, q.u.p, k.bf16, entries * kLoraBlock * kLoraParts,
                       q.small.use ? q.small.xrows : kGemmABoxRows))
      throw OpError(LAYA_E_CUDA, "lora_plan_create: tensor map encode failed");
    op_check(cudaMemcpyAsync(q.dev.p, h.data(), h.size() * 4, cudaMemcpyHostToDevice, k.stream), "lora plan upload");
    // rows of other adapters are zero in an entry, and stay zero: every run
    // writes the same rows of each entry
    op_check(cudaMemsetAsync(q.u.p, 0, entries * kLoraEntryElems * 2, k.stream), "lora workspace clear");
    op_check(cudaStreamSynchronize(k.stream), "lora plan upload");
    q.d_err = q.dev.as<int>();
    q.d_off = q.dev.as<int>() + o_off;
    q.d_row_entry = q.dev.as<int>() + o_row;
    q.d_entry_chunk = q.dev.as<int>() + o_ent;
    q.d_item = reinterpret_cast<const int4*>(q.dev.as<int>() + o_item);
    q.d_item_entry = q.dev.as<int>() + o_ie;
    q.d_item_chunk = q.dev.as<int>() + o_ic;
    q.d_pair = reinterpret_cast<const int4*>(q.dev.as<int>() + o_pair);
    q.d_soff = q.dev.as<int>() + o_soff;
    q.d_list = reinterpret_cast<const int2*>(q.dev.as<int>() + o_list);
    *plan = p.release();
  });
}

int laya_lora_run(laya_lora* lora, laya_lora_plan* plan, const void* x, int64_t ldx, void* y, int64_t ldy,
                  void* stream) {
  return op_guard([&] {
    op_require(lora && plan, "lora_run: null argument");
    Plan& q = plan->p;
    const Bank& k = *q.bank;
    op_require(lora->bank == q.bank, "lora_run: the plan belongs to another projection");
    if (q.lay.rows == 0) return;
    op_require(x && y, "lora_run: null buffer");
    constexpr int64_t kMaxPitch = int64_t{1} << 30;
    op_require(ldx >= k.in && ldx <= kMaxPitch, "lora_run: ldx is smaller than in");
    op_require(ldy >= k.out && ldy <= kMaxPitch, "lora_run: ldy is smaller than out");
    op_require(aligned16(x) && aligned16(y) && ldx % 8 == 0 && ldy % 8 == 0,
               "lora_run: x, y and their pitches must be multiples of 16 bytes");
    op_require(x != y, "lora_run: x and y must be apart");
    const std::lock_guard<std::mutex> held(k.lock);
    for (const auto& u : q.used)
      if (lora_chunks(k.slot[u.first].rank) != u.second)
        throw OpError(LAYA_E_STATE, "lora_run: an adapter of the plan was cleared or changed its rank; make a new plan");
    DeviceScope scope(k.device);
    require_device_ptr(x, k.device, "lora_run: x");
    require_device_ptr(y, k.device, "lora_run: y");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int stuck = std::exchange(q.stuck_kind, -1);
    const uint32_t xbox = q.small.use ? q.small.xrows : kGemmABoxRows;
    CUtensorMap mx, mw, my;
    if (make_tmap_pitched(&mx, x, k.bf16, q.lay.rows, k.in, ldx, xbox))
      throw OpError(LAYA_E_CUDA, "lora_run: tensor map encode failed");
    if (q.pairs > 0) {
      LoraPairsArgs s{};
      s.pair = q.d_pair;
      s.pairs = q.pairs;
      s.x = x;
      s.ldx = ldx;
      s.a = k.a.p;
      s.scale = k.scale.as<float>();
      s.u = q.u.p;
      s.in = k.in;
      s.in_pad = k.in_pad;
      s.bf16 = k.bf16;
      op_check(launch_lora_pairs(s, st), "lora launch");
    } else if (q.items > 0) {
      CUtensorMap mxi = mx;
      if (xbox != kLoraItemRows && make_tmap_pitched(&mxi, x, k.bf16, q.lay.rows, k.in, ldx, kLoraItemRows))
        throw OpError(LAYA_E_CUDA, "lora_run: tensor map encode failed");
      LoraShrinkArgs s{};
      s.item = q.d_item;
      s.item_entry = q.d_item_entry;
      s.item_chunk = q.d_item_chunk;
      s.items = q.items;
      s.group = q.group;
      s.row_entry = q.d_row_entry;
      s.entry_chunk = q.d_entry_chunk;
      s.scale = k.scale.as<float>();
      s.u = q.u.p;
      s.rows = q.lay.rows;
      s.num_kb = k.in_pad / 64;
      s.chunks_per_slot = k.cps;
      s.bf16 = k.bf16;
      s.err = q.d_err;
      s.stuck = stuck == 0 ? kLoraStuckLoads : stuck == 2 ? kLoraStuckExchange : kLoraStuckNone;
      s.wait_limit_ns = s.stuck ? q.stuck_limit_ns : 0;
      op_check(launch_lora_shrink(mxi, k.a_map, s, k.num_sms, st), "lora launch");
    }
    // x W^T and u B^T in one accumulator
    const bool early = q.pairs > 0 || q.items > 0;
    if (q.small.use) {
      const int width = q.small.width;
      CUtensorMap mb;
      if (make_tmap_pitched(&mw, k.w, k.bf16, k.out, k.in, k.ldw, width) ||
          make_tmap_lora(&mb, k.b.p, k.bf16, static_cast<uint64_t>(k.slots) * k.cps * k.out_pad, width))
        throw OpError(LAYA_E_CUDA, "lora_run: tensor map encode failed");
      LoraSmallArgs g{};
      g.off = q.d_soff;
      g.list = q.d_list;
      g.entry_chunk = q.d_entry_chunk;
      g.row_entry = q.d_row_entry;
      g.scale = k.scale.as<float>();
      g.entries = q.small.entries;
      g.xrows = q.small.xrows;
      g.width = width;
      memcpy(g.tile_entries, q.small.tile_entries, sizeof g.tile_entries);
      memcpy(g.chunk, q.small.chunk, sizeof g.chunk);
      g.chunks_per_slot = k.cps;
      g.b_rows = k.out_pad;
      g.bias = k.bias;
      g.y = y;
      g.ldy = ldy;
      g.rows = q.lay.rows;
      g.out = k.out;
      g.num_kb = k.in_pad / 64;
      g.bf16 = k.bf16;
      g.early = early;
      g.err = q.d_err;
      g.stuck = stuck == 1 ? kLoraStuckLoads : stuck == 2 ? kLoraStuckExchange : kLoraStuckNone;
      g.wait_limit_ns = g.stuck ? q.stuck_limit_ns : 0;
      op_check(launch_lora_small(mx, mw, q.u_map, mb, k.a_map, g, q.small.fused, k.num_sms, st), "lora launch");
      return;
    }
    // 256 x 128 tiles where 256 x 256 ones would fill at most half the
    // clusters, as in the engine (600 rows, 1024 -> 1024, 2 adapters: 10.2 us and,
    // wide, 11.8; 1300 rows -> 3072: 16.6 and, wide, 15.9)
    const int tiles = (q.lay.rows + kGemmBM - 1) / kGemmBM * (k.out_pad / kGemmBN);
    const bool narrow = tiles * 2 <= k.num_sms / 2;
    const int bn = narrow ? kGemmBNNarrow : kGemmBN;
    CUtensorMap mw_half;
    if (make_tmap_pitched(&mw, k.w, k.bf16, k.out, k.in, k.ldw, bn / 2) ||
        make_tmap_pitched(&mw_half, k.w, k.bf16, k.out, k.in, k.ldw, kGemmBBoxRowsNarrow) ||
        make_tmap_pitched(&my, y, k.bf16, q.lay.rows, std::max(k.out & ~7, 8), ldy, kGemmOutBoxRows))
      throw OpError(LAYA_E_CUDA, "lora_run: tensor map encode failed");
    GemmArgs g{};
    g.M = q.lay.rows;
    g.N = (k.out + bn - 1) / bn * bn;
    g.K = k.in_pad;
    g.err = q.d_err;
    g.out = y;
    g.ldo = static_cast<int>(ldy);
    g.bias = k.bias;
    g.n_valid = k.out;
    g.stuck = stuck == 1;
    g.wait_limit_ns = g.stuck ? q.stuck_limit_ns : 0;
    const GemmExt ext{&q.u_map, &k.b_map[narrow], &mw_half, &k.b_map[1], q.d_off, q.d_entry_chunk, k.out_pad, early};
    op_check(launch_gemm(k.bf16 ? kEpiPlainBf16 : kEpiPlainF16, GemmMaps{&mx, &mw, &my}, g, k.num_sms, st, bn, &ext),
             "lora launch");
  });
}

int laya_lora_status(laya_lora_plan* plan) {
  return op_guard([&] {
    op_require(plan, "lora_status: null argument");
    const Plan& q = plan->p;
    DeviceScope scope(q.bank->device);
    op_check(cudaDeviceSynchronize(), "lora_status");
    int err = 0;
    op_check(cudaMemcpy(&err, q.d_err, sizeof(int), cudaMemcpyDeviceToHost), "lora_status");
    if (err != 0) {
      op_check(cudaMemset(q.d_err, 0, sizeof(int)), "lora_status");
      op_check(cudaDeviceSynchronize(), "lora_status");
      throw OpError(LAYA_E_DEVICE_TIMEOUT, "lora_run: a device-side wait expired (code " + std::to_string(err) + ")");
    }
  });
}

int laya_lora_test_timeout_next(laya_lora_plan* plan, int kind, uint64_t limit_ns) {
  return op_guard([&] {
    op_require(plan, "lora_test_timeout_next: null argument");
    Plan& q = plan->p;
    op_require(kind >= 0 && kind <= 2 && limit_ns > 0 && limit_ns <= kMaxStuckNs,
               "lora_test_timeout_next: kind must be 0..2 and 0 < limit_ns <= 2e9");
    const std::lock_guard<std::mutex> held(q.bank->lock);
    op_require(kind != 0 || q.items > 0, "lora_test_timeout_next: the plan has no launch of that kind");
    q.stuck_kind = kind;
    q.stuck_limit_ns = limit_ns;
  });
}

void laya_lora_plan_destroy(laya_lora_plan* plan) { delete plan; }

int laya_lora_layout(const int32_t* rows, const int32_t* slot, int n, const int32_t* ranks, int slots,
                     int64_t* blocks, int64_t* entries, int32_t* off, int64_t cap_blocks, int32_t* chunks,
                     int64_t cap_entries) {
  return op_guard([&] {
    op_require(blocks && entries && (ranks || slots == 0) && slots >= 0, "lora_layout: null argument");
    std::vector<int> c(slots);
    for (int i = 0; i < slots; ++i) {
      op_require(ranks[i] >= 0 && ranks[i] <= LAYA_LORA_MAX_RANK, "lora_layout: rank out of range");
      c[i] = lora_chunks(ranks[i]);
    }
    const LoraLayout L = lora_layout(rows, slot, n, c);
    *blocks = static_cast<int64_t>(L.off.size()) - 1;
    *entries = static_cast<int64_t>(L.chunk.size());
    if (off) {
      op_require(cap_blocks >= *blocks, "lora_layout: block capacity too small");
      std::copy(L.off.begin(), L.off.end(), off);
    }
    if (chunks) {
      op_require(cap_entries >= *entries, "lora_layout: entry capacity too small");
      for (size_t i = 0; i < L.chunk.size(); ++i) {
        chunks[2 * i] = L.chunk[i].x;
        chunks[2 * i + 1] = L.chunk[i].y;
      }
    }
  });
}

}  // extern "C"
