#ifndef K3_HIP_DENSE_ABI_H
#define K3_HIP_DENSE_ABI_H
/*
 * Dense layers over any number of positions, for gfx950 (MI355X): a projection with
 * bias, activation and residual, and a gated feed-forward block (both projections, the
 * activation and the product in one kernel) with its gradient.  They take the same
 * resident matrices as the spine projections (k3_hip_spine_abi.h, at most 64 positions)
 * and the shared expert of k3_hip_moe_block_device (at most 16), at the lengths of a
 * prompt or a training batch.  The reference runs these steps through ATen
 * (row_int8_linear, native/provider_gate/provider_moe.cpp:507-516; situ, :524-533).
 *
 * Conventions, as k3_hip_spine_abi.h's:
 *   - statuses K3_SPINE_OK, K3_SPINE_E_INVALID, K3_SPINE_E_RUNTIME,
 *     K3_SPINE_E_UNSUPPORTED; the reason is in k3_hip_spine_last_error();
 *   - nothing allocates, synchronises, creates a stream or keeps a pointer; work is
 *     enqueued on `stream` of the current device, where every buffer lives, and may be
 *     captured into a graph; a failed call enqueues nothing (a launch that the runtime
 *     refuses midway excepted);
 *   - matrices, activations and outputs are row-major and dense, aligned to their
 *     elements (16-byte aligned buffers with rows of whole 16-byte pieces are used in
 *     place, others are laid out again in the workspace within the call);
 *   - outputs must not overlap inputs or one another, except that a residual may be the
 *     output itself;
 *   - scratch memory is the caller's: the matching *_workspace_bytes gives its size for
 *     a descriptor (0 with a reason for an invalid one; pointers count by their
 *     alignment only, NULL as an aligned one where the operand is not optional).  A size
 *     of K3_DENSE_NO_WORKSPACE means that the call uses none and takes NULL as well.  The
 *     workspace is 256-byte aligned and holds nothing between calls.  Calls that may
 *     run at the same time, replays of captured graphs among them, need one each.
 * rows, columns and positions are 1..1048576.
 *
 * Numbers.  BF16 weights are exact, int8 ones are exact integers scaled per row after
 * the sum; products are exact and sums are fp32.  BF16 activations enter as they are;
 * fp32 ones as three BF16 terms, whose sum has all 24 bits.  Outputs are rounded once.
 * A result does not depend on what other calls ran, but may differ in its last bits
 * with the number of positions (the order of its sum goes by the shape).  Infinities and
 * NaN in BF16 activations act as in fp32 sums, in fp32 activations too as long as the
 * matrix row is finite; a matrix value that is not finite makes its row's outputs for
 * fp32 activations not finite (NaN where an fp32 sum may give an infinity), and in the
 * fp32 gradient any value that is not finite does so to the outputs that it enters.
 */
#include <stdint.h>

#include "k3_hip_moe_abi.h"
#include "k3_hip_spine_abi.h"

#ifdef __cplusplus
extern "C" {
#endif

#define K3_DENSE_ABI_V1 1u
#define K3_DENSE_MAX_EXTENT 1048576u /* of rows, columns and positions */
#define K3_DENSE_NO_WORKSPACE 256u   /* size of a call that uses no scratch memory */

/* Activation of a projection: z, z / (1 + exp(-z)), z / 2 (1 + erf(z / sqrt 2)). */
enum { K3_DENSE_ACT_NONE = 0, K3_DENSE_ACT_SILU = 1, K3_DENSE_ACT_GELU = 2 };

/* out[p, r] = activation(row_scales[r] * sum_c weights[r, c] * x[p, c] + bias[r])
 *             + residual[p, r] */
typedef struct K3HipLinearV1 {
  uint32_t abi_version;    /* K3_DENSE_ABI_V1 */
  uint32_t struct_bytes;   /* sizeof(K3HipLinearV1) == 88 */
  uint32_t matrix_kind;    /* K3_SPINE_MATRIX_* */
  uint32_t activation;     /* K3_DENSE_ACT_* */
  uint32_t x_dtype;        /* K3_DTYPE_* of x */
  uint32_t out_dtype;      /* K3_DTYPE_* of out and residual */
  uint32_t rows, columns, positions;
  uint32_t reserved;       /* 0 */
  const void* weights;     /* BF16 bits or int8 [rows, columns] */
  const float* row_scales; /* int8: [rows]; BF16: NULL */
  const float* bias;       /* [rows] or NULL */
  const void* x;           /* [positions, columns] */
  const void* residual;    /* [positions, rows] or NULL; may be out */
  void* out;               /* [positions, rows] */
} K3HipLinearV1;

/* out = f(g, u), g[p, r] = gate_scales[r] * sum_c gate[r, c] x[p, c] and u alike from up;
 * f is SiLU(g) u (K3_ACT_SILU) or the K3 SiTU 4 tanh(g/4) sigmoid(g) 25 tanh(u/25). */
typedef struct K3HipGatedV1 {
  uint32_t abi_version;      /* K3_DENSE_ABI_V1 */
  uint32_t struct_bytes;     /* sizeof(K3HipGatedV1) == 104 */
  uint32_t matrix_kind;      /* K3_SPINE_MATRIX_* */
  uint32_t activation;       /* K3_ACT_* */
  uint32_t x_dtype;          /* K3_DTYPE_* of x */
  uint32_t out_dtype;        /* K3_DTYPE_* of out, out_gate and out_up */
  uint32_t rows, columns, positions;
  uint32_t reserved;         /* 0 */
  const void* gate;          /* [rows, columns] */
  const void* up;            /* [rows, columns] */
  const float* gate_scales;  /* int8: [rows]; BF16: NULL */
  const float* up_scales;
  const void* x;             /* [positions, columns] */
  void* out;                 /* [positions, rows] */
  void* out_gate;            /* g, u [positions, rows] for the gradient, both or neither */
  void* out_up;
} K3HipGatedV1;

/* The gradient of K3HipGatedV1 with BF16 matrices.  From grad = d(loss)/d(out) and the
 * kept g and u:  dg = grad f_g(g, u), du = grad f_u(g, u),
 *   d_x = dg gate + du up,  d_gate[r, c] = sum_p dg[p, r] x[p, c],  d_up alike from du.
 * Every activation, gradient and output has the one dtype.  BF16: dg and du are rounded
 * to BF16 before the products.  fp32: both operands of d_gate and d_up are three BF16
 * terms and the six leading products are kept; values under 2^-110 lose low bits (an
 * absolute error under 2^-133 of a term's other factor). */
typedef struct K3HipGatedGradV1 {
  uint32_t abi_version;      /* K3_DENSE_ABI_V1 */
  uint32_t struct_bytes;     /* sizeof(K3HipGatedGradV1) == 104 */
  uint32_t activation;       /* K3_ACT_* */
  uint32_t dtype;            /* K3_DTYPE_* */
  uint32_t rows, columns, positions;
  uint32_t reserved;         /* 0 */
  const void* gate;          /* BF16 bits [rows, columns] */
  const void* up;
  const void* x;             /* [positions, columns] */
  const void* g;             /* [positions, rows] */
  const void* u;
  const void* grad;          /* [positions, rows] */
  void* d_x;                 /* [positions, columns] */
  void* d_gate;              /* [rows, columns] */
  void* d_up;
} K3HipGatedGradV1;

uint64_t k3_hip_linear_workspace_bytes(const K3HipLinearV1* op);
int k3_hip_linear(const K3HipLinearV1* op, void* workspace, uint64_t workspace_bytes,
                  void* stream);

uint64_t k3_hip_gated_ffn_workspace_bytes(const K3HipGatedV1* op);
int k3_hip_gated_ffn(const K3HipGatedV1* op, void* workspace, uint64_t workspace_bytes,
                     void* stream);

uint64_t k3_hip_gated_ffn_grad_workspace_bytes(const K3HipGatedGradV1* op);
int k3_hip_gated_ffn_grad(const K3HipGatedGradV1* op, void* workspace,
                          uint64_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* K3_HIP_DENSE_ABI_H */
