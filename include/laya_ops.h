/*
 * laya_ops.h -- C ABI of the operators a host runs on its own device buffers,
 * beside the engine (laya_b200.h):
 *
 *   laya_lora_*   a projection shared by many requests, each segment of rows
 *                 with its own low-rank adapter or none
 *   laya_rope     rotary positions of queries and keys
 *
 * Neither has a counterpart in the reference (zerodegress/laya-rust), whose
 * rotation exists only inside its attention (src/graph.rs:62-84,
 * src/backend/cuda/kernels.rs:135-163) and which has no adapters.  The engine
 * runs them too: laya_forward_adapted, laya_set_rope_scaling.
 *
 * Conventions are those of laya_b200.h: LAYA_OK (0) or a nonzero status with
 * the message in laya_last_error(), nothing aborts.  Device buffers are the
 * caller's; an address that is not memory of the call's device is refused.
 * Every call runs on the device it names (or its handle was made on) and
 * restores the caller's current device.  `stream` is a cudaStream_t of that
 * device (NULL: the default stream); calls enqueue work and return without
 * waiting for it, and may be captured into a graph (make the first call of a kind
 * on a device before any capture: it loads and configures the kernels).
 *
 * Threads: laya_rope and the calls on one laya_lora and its plans may come from
 * several threads at once.  A run has the whole of an adapter that another thread
 * sets, or none of it.  What is left to the caller: a plan's runs are ordered on
 * the device (see laya_lora_run), no captured graph of runs is replayed while
 * laya_lora_set is in progress, and no call is in progress on a handle that is
 * destroyed.  The calls on an engine follow the rule of laya_b200.h.
 */
#ifndef LAYA_OPS_H
#define LAYA_OPS_H

#include <stddef.h>
#include <stdint.h>

#include "laya_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Element types. */
enum { LAYA_F16 = 0, LAYA_BF16 = 1, LAYA_F32 = 2 };

/* ---- rotary positions ----------------------------------------------------------
 * With c = mscale cos(p f_j), s = mscale sin(p f_j) for a token's position p:
 *   LAYA_ROPE_HALF         (x[j], x[j + rot/2]) -> (x[j] c - x[j+rot/2] s, x[j+rot/2] c + x[j] s)
 *   LAYA_ROPE_INTERLEAVED  (x[2j], x[2j+1])     -> the same rotation
 * for j < rot/2; dims from rot on are copied.  inverse != 0 turns the other way
 * (s -> -s): the gradient of the rotation.  The rotation is computed in 32 bits
 * and rounded once; angles are exact to 2^-32 of a turn at any 32-bit position. */
enum { LAYA_ROPE_HALF = 0, LAYA_ROPE_INTERLEAVED = 1 };

/* How frequencies are stretched for contexts `factor` (>= 1) times the trained
 * length:
 *   LINEAR  f_j / factor
 *   BASE    f_j factor^(-2j / (rot - 2)): the base grows so that the slowest
 *           pair turns `factor` times slower and the fastest as before
 *   PARTS   with n_j = trained_len f_j / (2 pi) turns over the trained length
 *           and g = clamp((n_j - low) / (high - low), 0, 1):
 *           f_j (g + (1 - g) / factor); low < high
 * attn: the factor on cos and sin; 0 takes the scheme's own, 0.1 ln(factor) + 1
 * for PARTS and 1 for the others. */
enum { LAYA_ROPE_NONE = 0, LAYA_ROPE_LINEAR = 1, LAYA_ROPE_BASE = 2, LAYA_ROPE_PARTS = 3 };
typedef struct laya_rope_scaling {
  int32_t kind;
  double factor;
  double trained_len, low, high; /* LAYA_ROPE_PARTS only */
  double attn;
} laya_rope_scaling;

#define LAYA_ROPE_MAX_DIM 512
/* freqs[j] = base^(-2j / rot), j < rot / 2, stretched by `s` (NULL: none);
 * *mscale the factor on cos and sin.  Host only, no device needed. */
int laya_rope_freqs(double base, int rot, const laya_rope_scaling *s, double *freqs, float *mscale);
/* What laya_rope computes angles with (tests and diagnostics, host only): `freq`
 * radians per position as a 64-bit fraction of a turn, so that position * *turns
 * (mod 2^64) is the angle with whole turns dropped. */
int laya_rope_turns(double freq, uint64_t *turns);

typedef struct {
  int32_t type;        /* LAYA_F16, LAYA_BF16 or LAYA_F32 */
  int32_t layout;      /* LAYA_ROPE_HALF or LAYA_ROPE_INTERLEAVED */
  int32_t inverse;
  int32_t dim, rot;    /* head size (<= LAYA_ROPE_MAX_DIM) and its rotated part (even, 2..dim) */
  float mscale;
  const double *freqs; /* host, [rot / 2], radians per position, of magnitude at most 2^20, negative ones
                        * turn the other way; read during the call */
} laya_rope_spec;

/* A [tokens, heads, dim] view and where its rotation goes; strides in elements,
 * not negative, dim contiguous.  out == x (with equal strides) rotates in
 * place; any other overlap of the two gives undefined values.  Elements of the
 * output must be distinct.  A stride of 0 repeats an input. */
typedef struct {
  const void *x;
  void *out;
  int64_t x_token, x_head, out_token, out_head;
  int64_t heads;
} laya_rope_tensor;

/* Rotates `count` (1..4) tensors over the same tokens, e.g. q and k, in one
 * launch, 65535 heads in all.  pos: device int32 [tokens], any values, or NULL for
 * pos0, pos0 + 1, ...  (all of them 32-bit numbers).  tokens == 0 does nothing. */
int laya_rope(int device, const laya_rope_spec *spec, const laya_rope_tensor *tensors, int count, int64_t tokens,
              const int32_t *pos, int64_t pos0, void *stream);

/* ---- a shared projection with low-rank adapters ------------------------------------
 *   y[m] = x[m] W^T + bias + scale_a (x[m] A_a^T) B_a^T
 * for row m of a segment with adapter a, without the last term for a segment
 * that has none.  W [out, in], A_a [rank_a, in], B_a [out, rank_a]; x, W, A, B
 * and y of one 16-bit type (LAYA_F16 or LAYA_BF16), bias f32.  Sums are f32.
 * The rank-space vector scale x A^T passes between the two products as a pair of
 * the 16-bit type (value and remainder), off by 2^-22 of it in f16 and 2^-16 in
 * bf16; y is rounded once.  With LAYA_F16 the magnitude of scale x A^T must stay
 * below 65504, as every f16 activation must, and values of it below 2^-3 are
 * off by up to 2^-25.  A row's sums never meet another row's values; equal calls
 * give equal bits.
 *
 * A laya_lora holds the adapters of one projection; W and bias stay the
 * caller's (read at every run).  A laya_lora_plan holds the segments of one
 * batch and the workspace of its runs. */
typedef struct laya_lora laya_lora;
typedef struct laya_lora_plan laya_lora_plan;

#define LAYA_LORA_NONE (-1)      /* a segment without an adapter */
#define LAYA_LORA_MAX_RANK 256
#define LAYA_LORA_MAX_SLOTS 4096
#define LAYA_LORA_MAX_ROWS (1 << 24)

/* `slots` adapters of rank <= max_rank beside W [out, in] (device, row pitch
 * ldw elements; W and ldw * 2 multiples of 16 bytes).  bias: device f32 [out]
 * or NULL.  Device memory for all slots is taken here: slots * up16(max_rank)
 * * (in + out, rounded up to 64 and 256) * 2 bytes. */
int laya_lora_create(int device, int type, int64_t in, int64_t out, const void *w, int64_t ldw, const float *bias,
                     int slots, int max_rank, laya_lora **lora);
/* Puts an adapter into a slot: a [rank, in], b [out, rank], host arrays of
 * `host_type` (LAYA_F16, LAYA_BF16, LAYA_F32; rounded to the projection's
 * type).  Values must be finite in that type: a broken adapter would otherwise
 * reach the rows of the others.  Waits for the device's queued work, complete
 * on return; not during a stream capture.  A plan made before stays valid if
 * up16(rank) is what it was then. */
int laya_lora_set(laya_lora *lora, int slot, int rank, const void *a, const void *b, int host_type, float scale);
int laya_lora_clear(laya_lora *lora, int slot);
void laya_lora_destroy(laya_lora *lora);

/* The segments of a batch, in row order: rows[i] >= 0 rows with the adapter
 * slot[i], or LAYA_LORA_NONE.  Host arrays, read during the call.  The plan
 * keeps what it needs of `lora` alive.  Takes device memory: not during a
 * stream capture.  A graph captured from runs reads the plan at every replay:
 * destroy it first. */
int laya_lora_plan_create(laya_lora *lora, const int32_t *rows, const int32_t *slot, int n, laya_lora_plan **plan);
/* Enqueues y = the projection of x on `stream`.  x [rows, in] with row pitch
 * ldx, y [rows, out] with row pitch ldy, in elements; addresses and pitches
 * multiples of 16 bytes, x and y apart.  Only elements of y's rows and
 * columns are written.  A plan's runs share its workspace: give them one
 * stream, or order them (a graph's replays count).  LAYA_E_STATE: an adapter
 * of the plan was cleared, or changed its up16(rank).  A graph captured from a
 * run cannot be told: it goes on with what the slots' memory holds, so capture
 * again where a new run would ask for a new plan. */
int laya_lora_run(laya_lora *lora, laya_lora_plan *plan, const void *x, int64_t ldx, void *y, int64_t ldy,
                  void *stream);
/* Waits for the device and reports a bounded wait that expired in a run of
 * this plan (LAYA_E_DEVICE_TIMEOUT; its y is then undefined). */
int laya_lora_status(laya_lora_plan *plan);
/* Test of the bounded waits, as laya_test_timeout_next: in the plan's next run the
 * loads of the launch that computes scale x A^T (kind 0; LAYA_E_INVALID where the
 * plan has none that loads through a barrier), those of the projection (kind
 * 1), or the exchange between the thread blocks of a cluster (kind 2; nothing where
 * none work together) wait for something that never comes, for limit_ns (at most 2
 * s).  That run's y is undefined, laya_lora_status reports it, and the plan stays
 * usable. */
int laya_lora_test_timeout_next(laya_lora_plan *plan, int kind, uint64_t limit_ns);
void laya_lora_plan_destroy(laya_lora_plan *plan);
/* The host side of a plan with no device (tests and diagnostics): for each
 * block of 256 rows the adapters it needs, in order of first use.  ranks[s]: the
 * rank of slot s, 0 if empty.  off [blocks + 1], then per entry e the 16-column
 * chunk (slot, chunk) as chunks[2 e], chunks[2 e + 1].  *blocks and *entries
 * are always written; chunks may be NULL, else must hold cap entries. */
int laya_lora_layout(const int32_t *rows, const int32_t *slot, int n, const int32_t *ranks, int slots,
                     int64_t *blocks, int64_t *entries, int32_t *off, int64_t cap_blocks, int32_t *chunks,
                     int64_t cap_entries);

/* ---- the engine --------------------------------------------------------------------
 * Adapters of many tenants in one forward: each sequence of a request names its
 * adapter, or none, and the encoder's four projections (Wqkv, Wo, Wi, mlp.Wo) add
 * that adapter's part in their accumulator, before RoPE, GeGLU and the residual.
 * All sequences still share every launch.
 *
 * laya_adapters_create: room for `slots` adapters of rank <= max_rank on every
 * encoder projection (14.5 MB per slot and 16 ranks); replaces the slots there
 * were.  laya_adapter_create empties a slot and gives it its rank and scale,
 * with no matrices: it then changes nothing.  laya_adapter_upload sets the
 * matrices of one projection, named like its weight
 * ("encoder.layers.{i}.attn.Wqkv.weight", "...attn.Wo.weight",
 * "...mlp.Wi.weight", "...mlp.Wo.weight"): a [rank, in] and b [out, rank] with
 * in and out as the weight is stored, host arrays of `host_type`, rounded to f16
 * (values must be finite in f16).  laya_adapter_drop empties the slot.  These
 * wait for the engine's queued work and retire captured graphs, as a weight
 * upload does.  A forward's scale x A^T has the range and the rounding that
 * LAYA_F16 gives it in a laya_lora: an adapter that takes it to 65504 or beyond
 * makes infinities of that sequence's activations. */
int laya_adapters_create(laya_engine *e, int slots, int max_rank);
int laya_adapter_create(laya_engine *e, int slot, int rank, float scale);
int laya_adapter_upload(laya_engine *e, int slot, const char *name, const void *a, const void *b, int host_type);
int laya_adapter_drop(laya_engine *e, int slot);
/* laya_forward, sequence i with the adapter adapter[i] (a created slot) or
 * LAYA_LORA_NONE; adapter [n], host.  A sequence's answer does not depend, not
 * by a bit, on which adapters the other sequences of the request have; one
 * without an adapter gets its answer of laya_forward on the same request. */
int laya_forward_adapted(laya_engine *e, const laya_req *req, const int32_t *adapter, float *logits, float *act);
/* laya_plan_create with adapters; run, capture, outputs and layers as for any
 * plan.  LAYA_E_STATE from a run: one of its slots was dropped, or changed its
 * up16(rank), since. */
int laya_plan_create_adapted(laya_engine *e, const laya_req *req, const int32_t *adapter, laya_plan **out);
/* The engine's rotation with stretched frequencies, for requests longer than
 * the model was trained on: `full` for the global layers' frequencies
 * (rope.freq_full), `sliding` for the windowed layers' (rope.freq_sliding);
 * NULL leaves one as the model has it, both NULL takes the scaling back (the
 * tables are then those of an engine that was never scaled, bit for bit).  The
 * angles of stretched frequencies are computed as in laya_rope.  Waits for the
 * engine's queued work; captured graphs are retired. */
int laya_set_rope_scaling(laya_engine *e, const laya_rope_scaling *full, const laya_rope_scaling *sliding);

#ifdef __cplusplus
}
#endif

#endif /* LAYA_OPS_H */
