/*
 * prl_optim.h — C-ABI of libprl_hip.so's optimizer operators over LISTS of tensors: the global
 * gradient norm and one clipped AdamW step with moments in 32 or in 8 bits (csrc/prl_optim.hip).
 * prl_flat_adamw (prl_abi.h) is the same step on one flat float32 vector; these take the tensors
 * where they lie, in float32, bfloat16 or float16.  The conventions are prl_abi.h's: device
 * pointers unless a comment says host, asynchronous on `stream`, nothing allocates, graph-capturable,
 * 0 or a negative prl_status with prl_last_error().  No reference counterpart (the reference calls
 * torch's clip_grad_norm_ and AdamW, PPO/PPO.py:248-250).
 */
#ifndef PRL_OPTIM_H
#define PRL_OPTIM_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

enum prl_list_dtype { PRL_LIST_F32 = 0, PRL_LIST_BF16 = 1, PRL_LIST_F16 = 2 };

/* Values of an 8-bit moment that share one float32 scale: consecutive in the flattened tensor,
 * counted from its first value; a tensor has ceil(numel / 256) scales per moment. */
#define PRL_LIST_BLOCK 256

/* One tensor of a list (host struct, pointers on the device).  Tensors are contiguous and need
 * only their element type's alignment.  What a call writes shares no memory with anything else of
 * the call (entries may have one grad in common).  numel == 0 is allowed (the tensor is skipped, its step
 * count still advances). */
typedef struct prl_list_entry {
  void* param;        /* [numel] of dtype */
  const void* grad;   /* [numel] of dtype, left as it is */
  float* master;      /* NULL, or the float32 weights behind a 16-bit param: they are updated,
                         param receives their rounding */
  void* exp_avg;      /* bits 32: float32 [numel]; bits 8: e4m3 codes [numel] */
  void* second;       /* bits 32: exp_avg_sq, float32 [numel]; bits 8: codes of its square root */
  float* exp_avg_scale;   /* bits 8: [ceil(numel / 256)] */
  float* second_scale;
  float* step;        /* one float32, the steps taken; a tensor has its own */
  int64_t numel;
  int32_t dtype;      /* prl_list_dtype of param and grad */
  int32_t bits;       /* 32 or 8 */
  int64_t group;      /* index into the groups */
} prl_list_entry;

typedef struct prl_list_group {   /* host */
  double lr, beta1, beta2, eps, weight_decay;
  const float* lr_dev;  /* NULL, or one float32 on the device that stands in for lr (a captured
                           graph then follows a schedule) */
} prl_list_group;

/* Workspace of the two calls below for a list of these sizes (prl_list_norm: n_groups 0); 0 for a
 * short list, which needs none (NULL will do); -1 if the number of tensors or one of the sizes is out
 * of range (nothing else of the list is looked at).  It holds nothing
 * between calls and needs no initial value; two calls that may run at once need one each. */
int64_t prl_list_workspace_bytes(const prl_list_entry* entries, int64_t count, int64_t n_groups);

/* *norm = sqrt(sum over the tensors' grads of their squares), summed in float64 in a fixed order. */
int prl_list_norm(const prl_list_entry* entries, int64_t count, float* norm, void* workspace,
                  int64_t workspace_bytes, void* stream);

/* One AdamW step of every tensor: step += 1, then with t = step and c = 1 or, if norm is given,
 * *norm as above and c = min(1, max_norm / (*norm + 1e-6)) (a NaN norm gives c = NaN):
 *   g = c * grad;  m = m + (1 - beta1) (g - m);  v = beta2 v + (1 - beta2) g^2
 *   w = w (1 - lr weight_decay) - lr / (1 - beta1^t) * m / (sqrt(v) / sqrt(1 - beta2^t) + eps)
 * in float32 (bias corrections in float64), w rounded once to a 16-bit param.
 *
 * bits 8: with A = the largest |x| of a block of 256 (its scale), m and r = sqrt(v) are held as
 * e4m3 values q of x / A * 256, so x = q * A / 256.  Rounding is stochastic (to the upper neighbour
 * with probability equal to the way past the lower one, in 2^-16ths) with bits hashed from the
 * value's index and t, so a run repeats itself bit for bit; for that, the step count of 8-bit
 * moments does not stay at 2^24, where float32's whole numbers end, but goes on by the next
 * float32 (t is then that, and its bits are hashed).  An r above 0 is held as at least the
 * smallest code.  A block with a value that is not finite gets the scale NaN: all its 256 moments
 * are NaN from then on.  One whose A is below 2^-118 is held as zeros. */
int prl_list_adamw(const prl_list_entry* entries, int64_t count, const prl_list_group* groups,
                   int64_t n_groups, float max_norm, float* norm, void* workspace,
                   int64_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* PRL_OPTIM_H */
