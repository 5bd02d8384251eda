#ifndef K3_HIP_SAMPLE_ABI_H
#define K3_HIP_SAMPLE_ABI_H
/*
 * Token sampling from rows of logits with temperature, top-k, top-p and min-p and given
 * random numbers, for gfx950 (MI355X): what follows the last projection of a decode or
 * verify step.
 *
 * Conventions as k3_hip_dense_abi.h's: K3_SPINE_* statuses with the reason in
 * k3_hip_spine_last_error(); nothing allocates or synchronises; the caller's workspace is
 * 256-byte aligned, holds nothing between calls, and each call that may run at the same
 * time needs its own; calls may be captured into a graph.
 *
 * A row's tokens are ordered by logit, the larger first, and by index, the lower first,
 * where logits are equal.  With T = temperature and max the row's largest logit, token i
 * weighs w_i = exp((logit_i - max) / T).  Three prefixes of that order are formed:
 *   top-k   the first top_k tokens (top_k < 1: all of them);
 *   top-p   the shortest prefix whose weights sum to at least top_p times the sum over the
 *           top-k prefix (at least one token; top_p not below 1: all of them);
 *   min-p   the tokens with w_i >= min_p (min_p not above 0: all; above 1 counts as 1);
 * and the shortest of the three is kept.  The token drawn is the first one at which the
 * running sum of weights exceeds u times the sum over the kept ones.  T not above 0 takes
 * the first token of the order.  u outside [0, 1) (NaN included) counts as the nearest
 * value inside (as the largest).
 *
 * -inf and NaN logits weigh nothing and are never drawn; a row with nothing else gives -1.
 * +inf logits, if there are any, share all the weight.
 *
 * Weights are taken in fp64 and summed as 64-bit integers (w_i times a power of two that
 * depends on the vocabulary alone: 2^45 at 131072 tokens), so a result has the same bits
 * whatever the order of the sums and whatever other rows a call holds.
 */
#include <stdint.h>

#include "k3_hip_moe_abi.h"
#include "k3_hip_spine_abi.h"

#ifdef __cplusplus
extern "C" {
#endif

#define K3_SAMPLE_ABI_V1 1u
#define K3_SAMPLE_MAX_ROWS 32768u
#define K3_SAMPLE_MAX_VOCABULARY 16777216u

typedef struct K3HipSampleV1 {
  uint32_t abi_version;     /* K3_SAMPLE_ABI_V1 */
  uint32_t struct_bytes;    /* sizeof(K3HipSampleV1) == 80 */
  uint32_t logits_dtype;    /* K3_DTYPE_* */
  uint32_t rows;            /* 1..K3_SAMPLE_MAX_ROWS */
  uint32_t vocabulary;      /* 1..K3_SAMPLE_MAX_VOCABULARY */
  uint32_t reserved;        /* 0 */
  const void* logits;       /* [rows, vocabulary], row-major and dense */
  const float* u;           /* [rows] */
  const float* temperature; /* [rows], or NULL for 1 */
  const int32_t* top_k;     /* [rows], or NULL for none */
  const float* top_p;       /* [rows], or NULL for none */
  const float* min_p;       /* [rows], or NULL for none */
  int32_t* tokens;          /* [rows] */
} K3HipSampleV1;

uint64_t k3_hip_sample_workspace_bytes(const K3HipSampleV1* op);
int k3_hip_sample(const K3HipSampleV1* op, void* workspace, uint64_t workspace_bytes,
                  void* stream);

#ifdef __cplusplus
}
#endif
#endif /* K3_HIP_SAMPLE_ABI_H */
