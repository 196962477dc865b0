// A projection shared by many requests, each segment of rows with its own
// low-rank adapter or none (laya_lora_*):
//
//   y[m] = x[m] W^T + bias + s_a (x[m] A_a^T) B_a^T
//
// Two launches.  The first computes u = s_a (x A_a^T) in rank space, f32, and
// leaves it as a pair of 16-bit values (value and remainder, together 16 bits
// more than one), so the second product's operands are 16-bit and the pair's
// rounding stays far below that of y.  The second computes x W^T + u B^T in one f32
// accumulator and rounds once: the tcgen05 GEMM of gemm.cu, whose K loop goes on
// over the adapters of its row block (GemmExt).
//
// u, simple form: one warp per row.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>
#include <cstring>
#include <memory>

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

// v as a 16-bit value and the 16-bit remainder; a value that is not finite has
// remainder 0 (inf - inf would be NaN).
template <class T>
__device__ __forceinline__ void split_value(float v, T& hi, T& lo) {
  hi = Num<T>::down(v);
  const float h = Num<T>::up(hi);
  lo = Num<T>::down(isfinite(h) ? v - h : 0.0f);
}

template <class T>
__global__ void __launch_bounds__(256) lora_shrink_rows(const LoraShrinkArgs a) {
  const int row = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (row >= a.rows) return;
  const int e0 = a.row_entry[row];
  if (e0 < 0) return;
  const int slot = a.entry_chunk[e0] / a.chunks_per_slot;
  const float scale = a.scale[slot];
  const T* x = static_cast<const T*>(a.x) + row * a.ldx;
  for (int c = 0; c < a.nchunks[slot]; ++c) {
    const T* A = static_cast<const T*>(a.a) + static_cast<size_t>(a.entry_chunk[e0 + c]) * kLoraChunk * a.in_pad;
    float acc[kLoraChunk] = {};
    for (int k = lane; k < a.in; k += 32) {
      const float v = Num<T>::up(x[k]);
#pragma unroll
      for (int j = 0; j < kLoraChunk; ++j) acc[j] += v * Num<T>::up(A[static_cast<size_t>(j) * a.in_pad + k]);
    }
    T* u = static_cast<T*>(a.u) + (e0 + c) * kLoraEntryElems + static_cast<size_t>(row % kLoraBlock) * 2 * kLoraChunk;
#pragma unroll
    for (int j = 0; j < kLoraChunk; ++j) {
      float v = acc[j];
      for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
      if (lane == 0) split_value<T>(v * scale, u[j], u[kLoraChunk + j]);
    }
  }
}

}  // namespace

cudaError_t launch_lora_shrink(const LoraShrinkArgs& a, cudaStream_t s) {
  if (a.rows <= 0) return cudaSuccess;
  const int grid = (a.rows + 7) / 8;
  if (a.bf16)
    lora_shrink_rows<__nv_bfloat16><<<grid, 256, 0, s>>>(a);
  else
    lora_shrink_rows<__half><<<grid, 256, 0, s>>>(a);
  return cudaGetLastError();
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
        op_require(L.chunk.size() < (size_t{1} << 22), "lora plan: too many adapters in one batch");
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
  std::vector<Slot> slot;
  Buf a, b, scale, nchunks;
  CUtensorMap b_map[2];  // B for 256- and 128-column tiles
  cudaStream_t stream = nullptr;  // uploads
  ~Bank() {
    int prev = -1;
    cudaGetDevice(&prev);
    cudaSetDevice(device);
    if (stream) cudaStreamDestroy(stream);
    for (Buf* x : {&a, &b, &scale, &nchunks}) {
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

float load_host(const void* p, int type, size_t i) {
  if (type == LAYA_F32) return static_cast<const float*>(p)[i];
  const uint16_t v = static_cast<const uint16_t*>(p)[i];
  if (type == LAYA_BF16) {
    const uint32_t u = static_cast<uint32_t>(v) << 16;
    float f;
    memcpy(&f, &u, 4);
    return f;
  }
  __half_raw r;
  r.x = v;
  return __half2float(__half(r));
}

uint16_t store_host(float v, bool bf16) {
  uint16_t b;
  if (bf16) {
    const __nv_bfloat16 h = __float2bfloat16_rn(v);
    op_require(std::isfinite(__bfloat162float(h)), "lora_set: a value is not finite in the projection's type");
    memcpy(&b, &h, 2);
  } else {
    const __half h = __float2half_rn(v);
    op_require(std::isfinite(__half2float(h)), "lora_set: a value is not finite in the projection's type");
    memcpy(&b, &h, 2);
  }
  return b;
}

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
    k->nchunks.alloc(sizeof(int) * slots, "lora ranks");
    op_check(cudaMemsetAsync(k->a.p, 0, chunks * kLoraChunk * in_pad * 2, k->stream), "lora clear");
    op_check(cudaMemsetAsync(k->b.p, 0, chunks * kLoraChunk * out_pad * 2, k->stream), "lora clear");
    op_check(cudaMemsetAsync(k->scale.p, 0, sizeof(float) * slots, k->stream), "lora clear");
    op_check(cudaMemsetAsync(k->nchunks.p, 0, sizeof(int) * slots, k->stream), "lora clear");
    op_check(cudaStreamSynchronize(k->stream), "lora clear");
    if (make_tmap_lora(&k->b_map[0], k->b.p, k->bf16, chunks * out_pad, kLoraChunk, kGemmBBoxRows) ||
        make_tmap_lora(&k->b_map[1], k->b.p, k->bf16, chunks * out_pad, kLoraChunk, kGemmBBoxRowsNarrow))
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
    // the slot's chunks, zero past the rank
    std::vector<uint16_t> ha(static_cast<size_t>(k.cps) * kLoraChunk * k.in_pad), hb(static_cast<size_t>(k.cps) * kLoraChunk * k.out_pad);
    for (int r = 0; r < rank; ++r)
      for (int c = 0; c < k.in; ++c)
        ha[static_cast<size_t>(r) * k.in_pad + c] = store_host(load_host(a, host_type, static_cast<size_t>(r) * k.in + c), k.bf16);
    for (int n = 0; n < k.out; ++n)
      for (int r = 0; r < rank; ++r)
        hb[(static_cast<size_t>(r / kLoraChunk) * k.out_pad + n) * kLoraChunk + r % kLoraChunk] =
            store_host(load_host(b, host_type, static_cast<size_t>(n) * rank + r), k.bf16);
    DeviceScope scope(k.device);
    const int nc = lora_chunks(rank);
    // runs already queued on the caller's streams may still read the slot
    op_check(cudaDeviceSynchronize(), "lora_set");
    op_check(cudaMemcpyAsync(k.a.as<uint16_t>() + ha.size() * slot, ha.data(), ha.size() * 2, cudaMemcpyHostToDevice, k.stream), "lora upload");
    op_check(cudaMemcpyAsync(k.b.as<uint16_t>() + hb.size() * slot, hb.data(), hb.size() * 2, cudaMemcpyHostToDevice, k.stream), "lora upload");
    op_check(cudaMemcpyAsync(k.scale.as<float>() + slot, &scale, 4, cudaMemcpyHostToDevice, k.stream), "lora upload");
    op_check(cudaMemcpyAsync(k.nchunks.as<int>() + slot, &nc, 4, cudaMemcpyHostToDevice, k.stream), "lora upload");
    op_check(cudaStreamSynchronize(k.stream), "lora upload");
    k.slot[slot].rank = rank;
  });
}

int laya_lora_clear(laya_lora* lora, int slot) {
  return op_guard([&] {
    op_require(lora, "lora_clear: null argument");
    op_require(slot >= 0 && slot < lora->bank->slots, "lora_clear: slot out of range");
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
    const std::vector<int> chunks = k.chunks_of();
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
    // [error word | off | row entries | entry chunks], each 256-byte aligned
    auto up = [](size_t v) { return (v + 63) / 64 * 64; };
    const size_t o_off = 64, o_row = o_off + up(L.off.size()), o_ent = o_row + up(L.row_entry.size());
    std::vector<int> h(o_ent + up(entry_chunk.size()));
    std::copy(L.off.begin(), L.off.end(), h.begin() + o_off);
    std::copy(L.row_entry.begin(), L.row_entry.end(), h.begin() + o_row);
    std::copy(entry_chunk.begin(), entry_chunk.end(), h.begin() + o_ent);
    q.dev.alloc(h.size() * 4, "lora plan");
    const size_t entries = std::max<size_t>(1, L.chunk.size());
    q.u.alloc(entries * kLoraEntryElems * 2, "lora workspace");
    if (make_tmap_lora(&q.u_map, q.u.p, k.bf16, entries * kLoraBlock, 2 * kLoraChunk, kGemmABoxRows))
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
    *plan = p.release();
  });
}

int laya_lora_run(laya_lora* lora, laya_lora_plan* plan, const void* x, int64_t ldx, void* y, int64_t ldy,
                  void* stream) {
  return op_guard([&] {
    op_require(lora && plan, "lora_run: null argument");
    const Plan& q = plan->p;
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
    for (const auto& u : q.used)
      if (lora_chunks(k.slot[u.first].rank) != u.second)
        throw OpError(LAYA_E_STATE, "lora_run: an adapter of the plan was cleared or changed its rank; make a new plan");
    DeviceScope scope(k.device);
    require_device_ptr(x, k.device, "lora_run: x");
    require_device_ptr(y, k.device, "lora_run: y");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    LoraShrinkArgs s{};
    s.x = x;
    s.ldx = ldx;
    s.a = k.a.p;
    s.row_entry = q.d_row_entry;
    s.entry_chunk = q.d_entry_chunk;
    s.scale = k.scale.as<float>();
    s.u = q.u.p;
    s.rows = q.lay.rows;
    s.in = k.in;
    s.in_pad = k.in_pad;
    s.chunks_per_slot = k.cps;
    s.nchunks = k.nchunks.as<int>();
    s.bf16 = k.bf16;
    if (!q.used.empty()) op_check(launch_lora_shrink(s, st), "lora launch");
    // x W^T and u B^T in one accumulator.  256 x 128 tiles where 256 x 256 ones
    // would fill at most half the clusters, as in the engine.
    const int tiles = (q.lay.rows + kGemmBM - 1) / kGemmBM * (k.out_pad / kGemmBN);
    const bool narrow = tiles * 2 <= k.num_sms / 2;
    const int bn = narrow ? kGemmBNNarrow : kGemmBN;
    CUtensorMap mx, mw, my;
    if (make_tmap_pitched(&mx, x, k.bf16, q.lay.rows, k.in, ldx, kGemmABoxRows) ||
        make_tmap_pitched(&mw, k.w, k.bf16, k.out, k.in, k.ldw, bn / 2) ||
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
    const GemmExt ext{&q.u_map, &k.b_map[narrow], q.d_off, q.d_entry_chunk, k.out_pad};
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
