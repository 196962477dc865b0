// Rotary positions on [tokens, heads, dim] views (laya_rope) and the cos/sin
// tables of stretched frequencies the engine's Wqkv epilogue reads.
//
// A pair (a, b) of a head turns by the angle p f_j: (a c - b s, b c + a s).
// Angles: p f_j needs more than 32 bits once p is large (at p = 2^20 an f32
// product is off by up to 0.06 radian), so a frequency is kept as a 64-bit
// fixed-point fraction of a turn per position.  The integer product p F drops
// whole turns by itself (mod 2^64), is off by at most |p| 2^-65 of a turn from
// F's rounding, and its top 32 bits (rounded) are the angle to 2^-33 of a turn.  Those
// split into the nearest quadrant and a remainder of at most 1/8 turn, exact
// as an integer, so the f32 sine and cosine see a reduced argument whose
// conversion rounds relative to itself.
//
// Bound by memory: every element is read and written once.  A block takes a few
// tokens and all their heads (up to 256 units of two 16-byte pieces times 4 heads),
// so a sine and cosine is computed once for all heads and passed through shared
// memory, and all of a thread's loads are issued before it needs an angle.
// Measured: 65536 tokens x 40 heads x 128, bf16: 206 us, 6.5 TB/s, the rate of a
// plain copy; 9872 x 32 x 64, f16: 15.0 us, 5.4 TB/s (4.2 tiles a block: ramp and
// tail); 3001 x 15 x 80 with 20 rotated, f32: 6.9 us, 4.2 TB/s; 1 token: 1.7 us.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <type_traits>
#include <vector>

#include "common.cuh"
#include "ops_common.h"
#include "rope.h"

#include <cuda_bf16.h>

namespace laya {

namespace {

constexpr int kMaxPairs = LAYA_ROPE_MAX_DIM / 2;
constexpr int kMaxTensors = 4;
constexpr double kMaxFreq = 1048576.0;  // radians per position; keeps rope_turns' remainder in 64 bits

struct RopeTensorArg {
  const void* x;
  void* out;
  long long x_token, x_head, out_token, out_head;
  int heads;
  int group0;  // first head group of this tensor (heads_per_thread heads each)
};

struct RopeArgs {
  RopeTensorArg t[kMaxTensors];
  int count;
  int dim, rot;
  int heads_per_thread, groups;       // groups: of heads, over all tensors
  int block_tokens, block_groups;
  long long tokens;
  const int* pos;
  long long pos0;
  float mscale, sign;
  uint64_t turns[kMaxPairs];
};

// (cos, sin) of position p times the fixed-point frequency `turns`.
__device__ __forceinline__ void rope_angle(uint64_t turns, long long p, float& c, float& s) {
  const uint64_t t = turns * static_cast<uint64_t>(p);
  const uint32_t v = static_cast<uint32_t>((t + 0x80000000ull) >> 32);  // angle in 2^-32 turns
  const uint32_t quad = (v + 0x20000000u) >> 30;
  const float r = static_cast<float>(static_cast<int32_t>(v - (quad << 30))) * 4.656612873077393e-10f;  // 2^-31: half turns
  float rs, rc;
  sincospif(r, &rs, &rc);
  // angle = quad quarter turns + r
  const float a = (quad & 1u) ? rs : rc, b = (quad & 1u) ? rc : rs;
  c = (quad == 1u || quad == 2u) ? -a : a;
  s = (quad & 2u) ? -b : b;
}

template <class T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32(float v) { return __float2bfloat16_rn(v); }

// V elements moved as one access of sizeof(T) * V bytes: 32-bit words, or one
// 16-bit element.
template <class T, int V>
struct alignas(sizeof(T) * V) Vec {
  using Word = std::conditional_t<(sizeof(T) * V >= 4), uint32_t, T>;
  static constexpr int kWords = sizeof(T) * V >= 4 ? sizeof(T) * V / 4 : 1;
  Word w[kWords];
};

// The two elements of a word, and back (one rounding each).
template <class T>
__device__ __forceinline__ float2 unpack(uint32_t w);
template <>
__device__ __forceinline__ float2 unpack<__half>(uint32_t w) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <>
__device__ __forceinline__ float2 unpack<__nv_bfloat16>(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <class T>
__device__ __forceinline__ uint32_t pack(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack<__half>(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

constexpr int kThreads = 256;
static_assert(kMaxPairs <= kThreads, "a head's units, of two elements at least, fit a block");
constexpr int kMaxHeads = 4;  // heads a thread turns, all loaded before the first is turned
// Blocks an SM.  Pieces of 16 bytes need 128 registers a thread to have a tile's
// loads in flight together (65536 tokens x 40 heads x 128, bf16: 2 blocks 207 us, 3
// blocks 217 us), but not in the half layout with dims to copy, whose two kinds
// of unit overlap better in 3 blocks (rot 64 of the same: 251 and 221 us); smaller
// pieces need more threads (9872 x 15 x 37, rot 36, f16: 13.2 and 10.9 us).
template <class T, int VEC, bool HALF, bool COPY>
constexpr int kBlocks = sizeof(T) * VEC == 16 && !(HALF && COPY) ? 2 : 3;

// (a c - b s, b c + a s), a pair of pairs an instruction (packed f32 pairs, each
// rounded as the scalar operation).
__device__ __forceinline__ void turn2(uint64_t a, uint64_t b, uint64_t c, uint64_t s, float (&x)[2], float (&y)[2]) {
  f2_get(f2_sub(f2_mul(a, c), f2_mul(b, s)), x[0], x[1]);
  f2_get(f2_fma(a, s, f2_mul(b, c)), y[0], y[1]);
}

// Turns the pairs across two pieces (half layout): pair j is (p[j], q[j]).
template <class T, int VEC>
__device__ __forceinline__ void turn_across(Vec<T, VEC>& p, Vec<T, VEC>& q, const float (&c)[VEC], const float (&s)[VEC]) {
  if constexpr (VEC == 1) {
    const T* pe = reinterpret_cast<const T*>(p.w);
    const T* qe = reinterpret_cast<const T*>(q.w);
    const float v0 = to_f32(*pe), v1 = to_f32(*qe);
    *reinterpret_cast<T*>(p.w) = from_f32<T>(v0 * c[0] - v1 * s[0]);
    *reinterpret_cast<T*>(q.w) = from_f32<T>(v1 * c[0] + v0 * s[0]);
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int j = 0; j < VEC; j += 2) {
      float x[2], y[2];
      turn2(f2(__uint_as_float(p.w[j]), __uint_as_float(p.w[j + 1])), f2(__uint_as_float(q.w[j]), __uint_as_float(q.w[j + 1])),
            f2(c[j], c[j + 1]), f2(s[j], s[j + 1]), x, y);
      p.w[j] = __float_as_uint(x[0]);
      p.w[j + 1] = __float_as_uint(x[1]);
      q.w[j] = __float_as_uint(y[0]);
      q.w[j + 1] = __float_as_uint(y[1]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < VEC / 2; ++j) {
      const float2 a = unpack<T>(p.w[j]), b = unpack<T>(q.w[j]);
      float x[2], y[2];
      turn2(f2(a.x, a.y), f2(b.x, b.y), f2(c[2 * j], c[2 * j + 1]), f2(s[2 * j], s[2 * j + 1]), x, y);
      p.w[j] = pack<T>(x[0], x[1]);
      q.w[j] = pack<T>(y[0], y[1]);
    }
  }
}

// Turns the neighbours within one piece (interleaved layout).
template <class T, int VEC>
__device__ __forceinline__ void turn_within(Vec<T, VEC>& p, const float (&c)[VEC / 2], const float (&s)[VEC / 2]) {
#pragma unroll
  for (int j = 0; j < VEC / 2; ++j) {
    float2 v;
    if constexpr (sizeof(T) == 4)
      v = make_float2(__uint_as_float(p.w[2 * j]), __uint_as_float(p.w[2 * j + 1]));
    else
      v = unpack<T>(p.w[j]);
    const float x = v.x * c[j] - v.y * s[j], y = v.y * c[j] + v.x * s[j];
    if constexpr (sizeof(T) == 4) {
      p.w[2 * j] = __float_as_uint(x);
      p.w[2 * j + 1] = __float_as_uint(y);
    } else {
      p.w[j] = pack<T>(x, y);
    }
  }
}

// A block turns tiles of a.block_tokens tokens by a.block_groups groups of
// heads, one tile after another; a thread keeps its place in the tile (unit,
// then group, then token), so its index arithmetic is done once.  The angles of
// the next tile go to the other half of the shared buffer while this tile's
// loads are in flight.  A unit is two pieces of VEC elements: a piece and what it
// turns with, two pieces of neighbouring pairs, or (COPY: rot < dim) two to copy.
// rot / 2 (half) or rot (interleaved), dim - rot, every stride and address are
// multiples of VEC.
template <class T, int VEC, bool HALF, bool COPY>
__global__ void __launch_bounds__(kThreads, kBlocks<T, VEC, HALF, COPY>) rope_kernel(const __grid_constant__ RopeArgs a) {
  using P = Vec<T, VEC>;
  constexpr bool kWithin = !HALF && VEC > 1;       // a pair lies within a piece
  constexpr int kPairs = kWithin ? VEC / 2 : VEC;  // of a piece
  extern __shared__ __align__(16) float angles[];  // [2][cos | sin][block_tokens * half]
  __shared__ uint64_t turns[kMaxPairs];
  const int half = a.rot / 2;
  const int turned_pieces = kWithin ? a.rot / VEC : 0;
  const int turned = kWithin ? (turned_pieces + 1) / 2 : half / VEC;  // units that turn
  const int copied_pieces = COPY ? (a.dim - a.rot) / VEC : 0, copied = (copied_pieces + 1) / 2;
  const int units = turned + copied;
  const int per_tok = a.block_groups * units;
  const int n_angles = a.block_tokens * half;
  const long long tiles = (a.tokens + a.block_tokens - 1) / a.block_tokens;

  // this thread's place (a tile has at most kThreads of them)
  const int tl = static_cast<int>(threadIdx.x) / per_tok, gu = static_cast<int>(threadIdx.x) - tl * per_tok;
  const int group = static_cast<int>(blockIdx.y) * a.block_groups + gu / units, u = gu % units;
  int ti = 0;
  while (ti + 1 < a.count && group >= a.t[ti + 1].group0) ++ti;
  const RopeTensorArg t = a.t[ti];
  const int h0 = (group - t.group0) * a.heads_per_thread;
  const bool turn = !COPY || u < turned;
  int nh = tl < a.block_tokens && group < a.groups ? min(a.heads_per_thread, t.heads - h0) : 0;
  if (!turn && t.x == t.out) nh = 0;
  // its first piece, and from there to its second (0: it has none)
  int at, step;
  if (turn) {
    at = kWithin || HALF ? u * VEC : 2 * u;
    step = kWithin ? (u + turned < turned_pieces ? turned * VEC : 0) : HALF ? half : 1;
  } else {
    at = a.rot + (u - turned) * VEC;
    step = u - turned + copied < copied_pieces ? copied * VEC : 0;
  }
  const T* const x0 = static_cast<const T*>(t.x) + h0 * t.x_head + at;
  T* const o0 = static_cast<T*>(t.out) + h0 * t.out_head + at;
  // the first of the angles it computes, and the way to its next
  const int step_at = kThreads / half, step_j = kThreads - step_at * half;
  const int my_at = static_cast<int>(threadIdx.x) / half, my_j = static_cast<int>(threadIdx.x) - my_at * half;

  // lanes that read different parameters take turns; here they do so once a block
  // (65536 tokens of one head of 128, where angles are half the work: 44 -> 30 us)
  for (int j = threadIdx.x; j < half; j += kThreads) turns[j] = a.turns[j];
  __syncthreads();
  grid_dep_wait();  // positions and inputs may come from the launch before
  grid_dep_trigger();

  auto compute_angles = [&](long long tile, float* buf) {
    int tok_at = my_at, j = my_j;
    for (int i = threadIdx.x; i < n_angles; i += kThreads) {
      const long long tok = tile * a.block_tokens + tok_at;
      if (tok < a.tokens) {
        const long long pos = a.pos ? __ldg(a.pos + tok) : a.pos0 + tok;
        float c, s;
        rope_angle(turns[j], pos, c, s);
        buf[i] = c * a.mscale;
        buf[n_angles + i] = s * (a.mscale * a.sign);
      }
      tok_at += step_at;
      j += step_j;
      if (j >= half) {
        j -= half;
        ++tok_at;
      }
    }
  };

  long long tile = blockIdx.x;
  if (tile < tiles) compute_angles(tile, angles);
  int parity = 0;
  for (; tile < tiles; tile += gridDim.x, parity ^= 1) {
    const long long tok = tile * a.block_tokens + tl;
    const int n = tok < a.tokens ? nh : 0, n2 = (HALF && !COPY) || step ? n : 0;
    const T* x = x0 + tok * t.x_token;
    T* o = o0 + tok * t.out_token;
    P p[kMaxHeads], q[kMaxHeads];
#pragma unroll
    for (int k = 0; k < kMaxHeads; ++k) {
      if (k < n) p[k] = *reinterpret_cast<const P*>(x + k * t.x_head);
      if (k < n2) q[k] = *reinterpret_cast<const P*>(x + k * t.x_head + step);
    }
    __syncthreads();  // this tile's angles are there; the other buffer was read
    if (tile + gridDim.x < tiles) compute_angles(tile + gridDim.x, angles + (parity ^ 1) * 2 * n_angles);
    if (n <= 0) continue;
    if (turn) {
      float c[kPairs], s[kPairs];
      const float* cs = angles + parity * 2 * n_angles + tl * half + u * kPairs;
      auto load_angles = [&] {
#pragma unroll
        for (int j = 0; j < kPairs; ++j) {
          c[j] = cs[j];
          s[j] = cs[n_angles + j];
        }
      };
      load_angles();
      if constexpr (kWithin) {
#pragma unroll
        for (int k = 0; k < kMaxHeads; ++k) turn_within<T, VEC>(p[k], c, s);
        if (n2 > 0) {
          cs += turned * kPairs;
          load_angles();
        }
#pragma unroll
        for (int k = 0; k < kMaxHeads; ++k) turn_within<T, VEC>(q[k], c, s);
      } else {
#pragma unroll
        for (int k = 0; k < kMaxHeads; ++k) turn_across<T, VEC>(p[k], q[k], c, s);
      }
    }
#pragma unroll
    for (int k = 0; k < kMaxHeads; ++k) {
      if (k < n) *reinterpret_cast<P*>(o + k * t.out_head) = p[k];
      if (k < n2) *reinterpret_cast<P*>(o + k * t.out_head + step) = q[k];
    }
  }
}

struct TableArgs {
  uint64_t turns[32];
  int n, positions;
  float mscale;
  float* cosb;
  float* sinb;
};

__global__ void __launch_bounds__(256) rope_table_kernel(const __grid_constant__ TableArgs a) {
  grid_dep_wait();
  grid_dep_trigger();
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i >= a.positions * a.n) return;
  float c, s;
  rope_angle(a.turns[i % a.n], i / a.n, c, s);
  a.cosb[i] = a.mscale * c;
  a.sinb[i] = a.mscale * s;
}

template <class T, int VEC, bool HALF, bool COPY>
cudaError_t launch_kernel(const RopeArgs& a, int num_sms, cudaStream_t st) {
  constexpr int kResident = kBlocks<T, VEC, HALF, COPY>;
  const unsigned gy = (a.groups + a.block_groups - 1) / a.block_groups;
  // the resident blocks, each walking over its share of the tiles
  const long long tiles = (a.tokens + a.block_tokens - 1) / a.block_tokens;
  long long blocks = std::max<long long>(1, static_cast<long long>(kResident) * num_sms / gy);
  // A walk of many tiles in up to 4 rounds of blocks of at least 8 tiles, so that
  // no block falls far behind (65536 tokens x 40 heads x 128, bf16: 217 -> 207 us;
  // with 4 tiles a block it costs, 9872 x 32 x 64, f16: 15.7 -> 16.7 us).
  if (kResident == 2) blocks *= std::clamp<long long>(tiles / (8 * blocks), 1, 4);
  const dim3 grid(static_cast<unsigned>(std::min(tiles, blocks)), gy);
  const size_t smem = 4 * sizeof(float) * a.block_tokens * (a.rot / 2);
  // Shared memory for the resident blocks' largest angles, the rest of the SM's
  // 228 KB as L1 for the loads in flight: all of it as shared memory, 9872 x 32 x
  // 64 takes 18.0 us, so 15.0.  Without a preference the split stays as the kernel
  // before left it (in turn with the adapter projection: 3.5 us more).
  static std::atomic<bool> configured[64] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  if (!configured[dev]) {
    constexpr int kBytes = kResident * (4 * static_cast<int>(sizeof(float)) * kThreads * VEC + 3072), kSm = 228 * 1024;
    e = cudaFuncSetAttribute(rope_kernel<T, VEC, HALF, COPY>, cudaFuncAttributePreferredSharedMemoryCarveout,
                             (100 * kBytes + kSm - 1) / kSm);
    if (e != cudaSuccess) return e;
    configured[dev] = true;
  }
  return launch_pdl(rope_kernel<T, VEC, HALF, COPY>, grid, dim3(kThreads), smem, st, nullptr, 0, a);
}

template <class T, int VEC>
cudaError_t launch_vec(const RopeArgs& a, bool half, int num_sms, cudaStream_t st) {
  if (a.dim == a.rot)
    return half ? launch_kernel<T, VEC, true, false>(a, num_sms, st)
                : launch_kernel<T, VEC, false, false>(a, num_sms, st);
  return half ? launch_kernel<T, VEC, true, true>(a, num_sms, st)
              : launch_kernel<T, VEC, false, true>(a, num_sms, st);
}

// Whether pieces of `v` elements of `es` bytes fit the head, every stride and
// every address.
bool pieces_fit(const RopeArgs& a, bool half, int es, int v) {
  if ((half ? a.rot / 2 : a.rot) % v || (a.dim - a.rot) % v) return false;
  for (int i = 0; i < a.count; ++i) {
    const RopeTensorArg& t = a.t[i];
    if ((reinterpret_cast<uintptr_t>(t.x) | reinterpret_cast<uintptr_t>(t.out)) % (es * v)) return false;
    if ((t.x_token | t.x_head | t.out_token | t.out_head) % v) return false;
  }
  return true;
}

template <class T>
cudaError_t launch_rope(RopeArgs& a, bool half, int num_sms, cudaStream_t st) {
  constexpr int es = sizeof(T), kMaxVec = 16 / es;
  int v = kMaxVec;
  while (v > 1 && !pieces_fit(a, half, es, v)) v /= 2;
  const int units = (half || v == 1 ? a.rot / 2 / v : (a.rot / v + 1) / 2) + ((a.dim - a.rot) / v + 1) / 2;
  // heads a thread: 4, fewer while there would be under 192 threads an SM (500
  // tokens x 15 heads x 80, f32: 4 heads 2.9 us, 1 head 4.5 us; 700 x 32 x 64, f16:
  // 2 heads 3.3, 4 heads 3.5; 1 x 32 x 64, f16: 1 head 2.1 us, 4 heads 2.5 us)
  int heads = 0;
  for (int i = 0; i < a.count; ++i) heads += a.t[i].heads;
  a.heads_per_thread = kMaxHeads;
  while (a.heads_per_thread > 1 && a.tokens * units * heads < 192ll * num_sms * a.heads_per_thread)
    a.heads_per_thread /= 2;
  a.groups = 0;
  for (int i = 0; i < a.count; ++i) {
    a.t[i].group0 = a.groups;
    a.groups += (a.t[i].heads + a.heads_per_thread - 1) / a.heads_per_thread;
  }
  a.block_groups = std::min(a.groups, std::max(1, kThreads / units));
  a.block_tokens = std::max(1, kThreads / (a.block_groups * units));
  switch (v) {
    case 8: return launch_vec<T, kMaxVec>(a, half, num_sms, st);
    case 4: return launch_vec<T, 4>(a, half, num_sms, st);
    case 2: return launch_vec<T, 2>(a, half, num_sms, st);
    default: return launch_vec<T, 1>(a, half, num_sms, st);
  }
}

bool finite_positive(double v) { return std::isfinite(v) && v > 0; }

}  // namespace

float rope_stretch(double* f, int rot, const laya_rope_scaling* s) {
  if (!s) return 1.0f;
  op_require(s->attn >= 0 && std::isfinite(static_cast<float>(s->attn)),
             "rope scaling: attn must not be negative, and finite in 32 bits");
  if (s->kind == LAYA_ROPE_NONE) return s->attn != 0 ? static_cast<float>(s->attn) : 1.0f;
  op_require(s->kind == LAYA_ROPE_LINEAR || s->kind == LAYA_ROPE_BASE || s->kind == LAYA_ROPE_PARTS,
             "rope scaling: unknown kind");
  op_require(std::isfinite(s->factor) && s->factor >= 1, "rope scaling: factor must be at least 1");
  const int n = rot / 2;
  double m = 1.0;
  if (s->kind == LAYA_ROPE_LINEAR) {
    for (int j = 0; j < n; ++j) f[j] /= s->factor;
  } else if (s->kind == LAYA_ROPE_BASE) {
    op_require(rot > 2, "rope scaling: LAYA_ROPE_BASE needs rot > 2");
    for (int j = 0; j < n; ++j) f[j] *= std::pow(s->factor, -2.0 * j / (rot - 2));
  } else {
    op_require(finite_positive(s->trained_len) && std::isfinite(s->low) && std::isfinite(s->high) && s->low < s->high,
               "rope scaling: LAYA_ROPE_PARTS needs trained_len > 0 and low < high");
    for (int j = 0; j < n; ++j) {
      const double turns = s->trained_len * f[j] / (2.0 * M_PI);
      const double g = std::min(1.0, std::max(0.0, (turns - s->low) / (s->high - s->low)));
      f[j] *= g + (1.0 - g) / s->factor;
    }
    m = 0.1 * std::log(s->factor) + 1.0;
  }
  return static_cast<float>(s->attn != 0 ? s->attn : m);
}

bool rope_freq_fits(double f) { return std::fabs(f) <= kMaxFreq; }

uint64_t rope_turns(double f) {
  // below, f >= 0: a negative frequency turns the other way, and the fraction of a
  // negative product would not be exact
  if (f < 0) return 0 - rope_turns(-f);
  // f / (2 pi) as the product with 1 / (2 pi) in two doubles: the leading
  // product, its exact error, and the constant's tail
  constexpr double kInvHi = 0.15915494309189535, kInvLo = -9.839338337591243e-18;
  const double hi = f * kInvHi, lo = std::fma(f, kInvHi, -hi) + f * kInvLo;
  constexpr double kUnits = 18446744073709551616.0;
  const double frac = (hi - std::floor(hi)) * kUnits;  // exact
  const double whole = std::floor(frac);
  // one rounding, of what is not whole and the low parts together
  return static_cast<uint64_t>(whole) + static_cast<uint64_t>(std::llrint((frac - whole) + lo * kUnits));
}

cudaError_t launch_rope_table(const double* freqs, int n, float mscale, int positions, float* cosb, float* sinb,
                              cudaStream_t s) {
  if (n < 1 || n > 32 || positions < 0 || !std::all_of(freqs, freqs + n, rope_freq_fits)) return cudaErrorInvalidValue;
  if (positions == 0) return cudaSuccess;
  TableArgs a{};
  for (int j = 0; j < n; ++j) a.turns[j] = rope_turns(freqs[j]);
  a.n = n;
  a.positions = positions;
  a.mscale = mscale;
  a.cosb = cosb;
  a.sinb = sinb;
  return launch_pdl(rope_table_kernel, dim3((positions * n + 255) / 256), dim3(256), 0, s, nullptr, 0, a);
}

}  // namespace laya

using namespace laya;

extern "C" int laya_rope_freqs(double base, int rot, const laya_rope_scaling* s, double* freqs, float* mscale) {
  return op_guard([&] {
    op_require(freqs && mscale, "rope_freqs: null argument");
    op_require(std::isfinite(base) && base > 0, "rope_freqs: base must be positive");
    op_require(rot >= 2 && rot <= LAYA_ROPE_MAX_DIM && rot % 2 == 0, "rope_freqs: rot must be even, 2..LAYA_ROPE_MAX_DIM");
    std::vector<double> f(rot / 2);
    for (int j = 0; j < rot / 2; ++j) f[j] = std::pow(base, -2.0 * j / rot);
    *mscale = rope_stretch(f.data(), rot, s);
    std::copy(f.begin(), f.end(), freqs);
  });
}

extern "C" int laya_rope_turns(double freq, uint64_t* turns) {
  return op_guard([&] {
    op_require(turns, "rope_turns: null argument");
    op_require(rope_freq_fits(freq), "rope_turns: a frequency is not finite, or above 2^20");
    *turns = rope_turns(freq);
  });
}

extern "C" int laya_rope(int device, const laya_rope_spec* spec, const laya_rope_tensor* tensors, int count,
                         int64_t tokens, const int32_t* pos, int64_t pos0, void* stream) {
  return op_guard([&] {
    op_require(spec && tensors && spec->freqs, "rope: null argument");
    op_require(spec->type == LAYA_F16 || spec->type == LAYA_BF16 || spec->type == LAYA_F32, "rope: unknown type");
    op_require(spec->layout == LAYA_ROPE_HALF || spec->layout == LAYA_ROPE_INTERLEAVED, "rope: unknown layout");
    op_require(spec->dim >= 2 && spec->dim <= LAYA_ROPE_MAX_DIM, "rope: dim must be 2..LAYA_ROPE_MAX_DIM");
    op_require(spec->rot >= 2 && spec->rot <= spec->dim && spec->rot % 2 == 0, "rope: rot must be even, 2..dim");
    op_require(std::isfinite(spec->mscale), "rope: mscale is not finite");
    op_require(count >= 1 && count <= kMaxTensors, "rope: 1 to 4 tensors");
    constexpr int64_t kMaxPos = 2147483647;
    op_require(tokens >= 0 && tokens <= kMaxPos, "rope: tokens out of range");
    op_require(pos || (pos0 >= -kMaxPos - 1 && pos0 <= kMaxPos && pos0 + tokens <= kMaxPos + 1),
               "rope: positions must fit 32 bits");
    op_require(reinterpret_cast<uintptr_t>(pos) % 4 == 0, "rope: pos is not aligned");
    RopeArgs a{};
    int64_t heads = 0;
    const size_t es = spec->type == LAYA_F32 ? 4 : 2;
    for (int i = 0; i < count; ++i) {
      const laya_rope_tensor& t = tensors[i];
      op_require(t.heads >= 0 && t.heads <= 65535, "rope: heads must be 0..65535");
      heads += t.heads;
      op_require(heads <= 65535, "rope: more than 65535 heads in all");
      if (t.heads == 0 || tokens == 0) continue;
      op_require(t.x && t.out, "rope: null tensor");
      op_require(reinterpret_cast<uintptr_t>(t.x) % es == 0 && reinterpret_cast<uintptr_t>(t.out) % es == 0,
                 "rope: address not aligned to its elements");
      op_require(t.x_token >= 0 && t.x_head >= 0 && t.out_token >= 0 && t.out_head >= 0, "rope: negative stride");
      constexpr int64_t kMaxStride = int64_t{1} << 40;
      op_require(t.x_token <= kMaxStride && t.x_head <= kMaxStride && t.out_token <= kMaxStride && t.out_head <= kMaxStride,
                 "rope: stride too large");
      // distinct output elements: the smaller stride steps over a head's dims,
      // the larger over everything the smaller one reaches
      const int64_t sh = t.heads > 1 ? t.out_head : 0, sk = tokens > 1 ? t.out_token : 0;
      const int64_t lo = std::min(sh, sk), hi = std::max(sh, sk), nlo = sh <= sk ? t.heads : tokens;
      op_require(t.heads == 1 || tokens == 1
                     ? hi >= spec->dim || (t.heads == 1 && tokens == 1)
                     : lo >= spec->dim && hi >= static_cast<__int128>(lo) * (nlo - 1) + spec->dim,
                 "rope: output elements overlap");
      if (t.x == t.out)
        op_require((t.x_token == t.out_token || tokens == 1) && (t.x_head == t.out_head || t.heads == 1),
                   "rope: in place needs equal strides");
      RopeTensorArg& r = a.t[a.count++];
      r.x = t.x;
      r.out = t.out;
      r.x_token = t.x_token;
      r.x_head = t.x_head;
      r.out_token = t.out_token;
      r.out_head = t.out_head;
      r.heads = static_cast<int>(t.heads);
    }
    for (int j = 0; j < spec->rot / 2; ++j) {
      op_require(rope_freq_fits(spec->freqs[j]), "rope: a frequency is not finite, or above 2^20");
      a.turns[j] = rope_turns(spec->freqs[j]);
    }
    if (a.count == 0) return;
    DeviceScope scope(device);
    for (int i = 0; i < a.count; ++i) {
      require_device_ptr(a.t[i].x, device, "rope: x");
      require_device_ptr(a.t[i].out, device, "rope: out");
    }
    if (pos) require_device_ptr(pos, device, "rope: pos");
    a.dim = spec->dim;
    a.rot = spec->rot;
    a.tokens = tokens;
    a.pos = pos;
    a.pos0 = pos0;
    a.mscale = spec->mscale;
    a.sign = spec->inverse ? -1.0f : 1.0f;
    const bool half = spec->layout == LAYA_ROPE_HALF;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int sms = device_sms(device);
    cudaError_t e = spec->type == LAYA_F16    ? launch_rope<__half>(a, half, sms, st)
                    : spec->type == LAYA_BF16 ? launch_rope<__nv_bfloat16>(a, half, sms, st)
                                              : launch_rope<float>(a, half, sms, st);
    op_check(e, "rope launch");
  });
}
