/*
 * hydra_optim.h -- C-ABI of the optimizer step on a reduced gradient bucket (MI355X, gfx950).
 *
 * What follows an allreduce of a gradient bucket, on the device and without a host round trip:
 * the norm of all gradients with its clip factor and the finite check, the AdamW step over many
 * tensors in one launch with moments in 32 or in 8 bits, and the conversion of 8-bit moments from
 * and to values.  Part of libhydra_hip.so; error codes and hydra_last_error() as in hydra_hip.h.
 * No counterpart in the reference.
 */
#ifndef HYDRA_OPTIM_H_
#define HYDRA_OPTIM_H_

#include "hydra_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- the tensors of a step ------------------------------------------------------------------
 * A plan is the list of tensors a training program steps together, laid out once on the device.
 * Per element i of a tensor, with t the number of the step (1, 2, ...), lr' = lr * lr_scale,
 * c1 = 1 / (1 - beta1^t) and c2 = 1 / sqrt(1 - beta2^t) (those and 1 - beta in fp64, rounded once) and
 * every operation rounded to fp32 in the order written:
 *     g = float(grad[i]) * mult
 *     m = m * beta1 + g * (1 - beta1)
 *     v = v * beta2 + (g * (1 - beta2)) * g
 *     p = p * (1 - lr' * weight_decay) - (m / (sqrt(v) * c2 + eps)) * (lr' * c1)
 * p is the fp32 master where there is one (`param` is then written only: the master rounded to
 * nearest even), else `param` widened, and rounded to nearest even on its way back.  A 16-bit
 * `param` without a master loses updates below half a step of its type.
 *
 * 8-bit moments (state_dtype HYDRA_UINT8): each 256 consecutive elements of a tensor share one
 * fp32 scale per moment, s = (their largest finite magnitude) * fp32(1 / 1.875); a block whose
 * magnitudes all lie below 2^-100 has scale 0 and reads as zeros.
 *     m        byte = sign << 7 | c;  value = +-F3(c) * s;  byte 0x80: not finite, reads as NaN
 *     sqrt(v)  byte = c;              value = F4(c) * s, v = value^2;  255: not finite, reads as inf
 * with Fk the float of 4 exponent bits and k mantissa bits whose largest power of two is 1:
 * Fk(c) = c * 2^-(14 + k) for c < 2^k, else 2^((c >> k) - 15) * (1 + (c mod 2^k) / 2^k).  The byte
 * of a v above zero is at least 1, so no step divides by eps alone where fp32 holds v at all.  m, v
 * and the bytes come from the operations above, each rounded to fp32; the magnitude over s is the
 * product with fp32's 1 / s, rounded to fp32 or, below 2^-14, to a multiple of 2^-37.  The quotient in
 * p's update is within 2 units in the last place, and its product with lr' * c1 may not be rounded
 * before the difference.
 * A step rounds its new moments stochastically: with x the magnitude over s, the two bytes around
 * x are taken with probabilities that make the mean x, by 16 random bits for each moment from a
 * 32-bit hash of (seed, t, the tensor's place in the plan, i) -- the same bits on every run and
 * every rank.  beta2 = 0.999 moves v by 0.1 % a step where a byte's step is 3 to 6 %: rounded to
 * nearest, v would stand still.  seed 0 rounds to nearest (a half up).                          */
typedef struct {
  void* param;        /* param_dtype; read and written (with HYDRA_ADAMW_MASTER only written) */
  float* master;      /* fp32 master weights (HYDRA_ADAMW_MASTER), else NULL */
  const void* grad;   /* grad_dtype; with HYDRA_ADAMW_BUCKET the BYTE OFFSET in the step's bucket */
  void* m;            /* first moment: float, or uint8_t with m_scale */
  void* v;            /* second moment: float, or uint8_t with v_scale */
  float* m_scale;     /* ceil(n / 256) scales (HYDRA_UINT8), else NULL */
  float* v_scale;
  size_t n;           /* elements; 0 is allowed */
  float lr_scale;     /* this tensor's learning rate is lr * lr_scale */
  float weight_decay;
} hydra_adamw_tensor_t;

#define HYDRA_ADAMW_MASTER 1    /* fp32 master beside a 16-bit param */
#define HYDRA_ADAMW_BUCKET 2    /* gradients lie in a bucket whose address each call gives */
#define HYDRA_ADAMW_NORM_ONLY 4 /* gradients alone, for hydra_adamw_grad_norm */

typedef struct {
  int32_t param_dtype; /* HYDRA_FLOAT32, HYDRA_BFLOAT16 or HYDRA_FLOAT16 (IEEE half) */
  int32_t grad_dtype;  /* the same choices */
  int32_t state_dtype; /* HYDRA_FLOAT32 or HYDRA_UINT8 */
  int32_t flags;
  double beta1, beta2; /* in [0, 1) */
  double eps;          /* >= 0 */
} hydra_adamw_config_t;

/* Device memory of the caller's (64 bytes, 8-byte aligned, zeroed, then `lr` and `step` set):
 * what a step takes from the device instead of from its arguments, so a captured graph of
 * grad_norm + step does the next step at every replay.  Write lr between steps to schedule it. */
typedef struct {
  int64_t step;       /* steps done; grad_norm adds 1, unless it skips */
  int64_t skipped;    /* steps that grad_norm skipped */
  float lr;           /* the learning rate: only read */
  float mult;         /* out: what the step multiplies every gradient by */
  float norm;         /* out: the norm of all gradients, before clipping */
  int32_t skip;       /* out: 1 if a gradient was not finite: the step leaves everything as it is */
  float inv_bc1;      /* out: 1 / (1 - beta1^step) */
  float inv_sqrt_bc2; /* out: 1 / sqrt(1 - beta2^step) */
  int32_t reserved[6];
} hydra_adamw_ctrl_t;

typedef struct hydra_adamw* hydra_adamw_t;

/* Lays out `count` tensors on `device` (allocates and copies: not while a stream is being
 * captured).  The list is copied; the memory it names stays the caller's and has to outlive the
 * plan's calls and every graph that holds one.  Refused with HYDRA_ERR_INVALID: null or
 * misaligned pointers (each to its element size), a range whose first or last byte is not memory
 * of this device, and any overlap of what a step writes with anything else in the plan (gradients
 * may overlap one another; those of a bucket are checked by the calls).  Plans are only read by the calls below: threads
 * may share one. */
int hydra_adamw_create(int device, const hydra_adamw_config_t* config,
                       const hydra_adamw_tensor_t* tensors, size_t count, hydra_adamw_t* out);
/* Waits for the device's work, then releases the plan (not the tensors). */
int hydra_adamw_destroy(hydra_adamw_t plan);

#define HYDRA_ADAMW_WORKSPACE_MAX 16384 /* bytes: no plan needs a larger workspace */

/* All calls below enqueue on `stream` of the plan's device whatever the caller's current device
 * is: asynchronous, no allocation, no synchronisation, graph-capturable.  They are ordered like
 * any in-place update: two calls on the same tensors (or the same ctrl or workspace) go to one
 * stream or are ordered by events.  `bucket`: the address that the plan's gradient offsets count
 * from (HYDRA_ADAMW_BUCKET; aligned to the gradients' element size), NULL without that flag.
 *
 * norm = |grad_scale| * sqrt(sum of all grad^2), summed in fp64 in an order fixed by the tensors'
 * lengths and the gradients' type, whatever the addresses: the same bits on every call and on every
 * rank that holds the same bits.  max_norm > 0 clips:
 * mult = grad_scale * min(1, max_norm / (norm + 1e-6)); 0: mult = grad_scale.  (Both are arguments: a
 * captured graph keeps those of its capture.)  If the sum is not
 * finite, skip = 1 and skipped += 1; else step += 1 and the fields for that step are set.
 * workspace: hydra_adamw_workspace() bytes of device memory or more (none for a small plan: may be
 * NULL then), 8-byte aligned, needed until the call has run, and by graphs that hold it; its contents
 * do not matter.  It is written on `stream`: memory that another stream's work may still use has to be
 * ordered first. */
int hydra_adamw_workspace(hydra_adamw_t plan, size_t* bytes);
int hydra_adamw_grad_norm(hydra_adamw_t plan, const void* bucket, double grad_scale,
                          double max_norm, hydra_adamw_ctrl_t* ctrl, void* workspace,
                          size_t workspace_bytes, hydra_stream_t stream);
/* Step number `step` (1, 2, ...) with mult = grad_scale.  seed: see above; unused by fp32 moments. */
int hydra_adamw_step(hydra_adamw_t plan, const void* bucket, double lr, int64_t step,
                     double grad_scale, uint64_t seed, hydra_stream_t stream);
/* The step that the last hydra_adamw_grad_norm on `ctrl` set up (it precedes this call on the
 * stream): number, mult, skip and lr come from ctrl.  A skipped step writes nothing. */
int hydra_adamw_step_ctrl(hydra_adamw_t plan, const void* bucket, const hydra_adamw_ctrl_t* ctrl,
                          uint64_t seed, hydra_stream_t stream);

/* ---- 8-bit moments from and to values ---------------------------------------------------------
 * encode: m and v (fp32 or bf16, `dtype`) of one tensor of n elements into bytes and
 * ceil(n / 256) scales each, rounded to nearest (a half up); v is taken as |v|.  decode: the values
 * that the bytes stand for, fp32, or bf16 rounded to nearest even.  Either moment may be left out
 * (all three of its pointers NULL).  On `stream` of the current device, graph-capturable; pointers
 * aligned to their element size; outputs overlap nothing. */
int hydra_moments8_encode(uint8_t* m8, float* m_scale, uint8_t* v8, float* v_scale, const void* m,
                          const void* v, int dtype, size_t n, hydra_stream_t stream);
int hydra_moments8_decode(void* m, void* v, int dtype, const uint8_t* m8, const float* m_scale,
                          const uint8_t* v8, const float* v_scale, size_t n,
                          hydra_stream_t stream);

#ifdef __cplusplus
}
#endif
#endif /* HYDRA_OPTIM_H_ */
