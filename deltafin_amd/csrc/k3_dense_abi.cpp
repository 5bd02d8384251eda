// C ABI of the dense layers (include/k3_hip_dense_abi.h): argument checks.  The kernels
// are in k3_dense.hip.
#include <hip/hip_runtime_api.h>

#include "k3_dense.h"
#include "k3_internal.h"

namespace k3 {
namespace {

// A buffer of a call: who it is, where it lies, what its elements are.
struct Span {
  const char* name;
  const void* p;
  uint64_t bytes;
  unsigned align;
};

uint64_t elem(uint32_t dtype) { return dtype == K3_DTYPE_F32 ? 4 : 2; }

bool overlap(const Span& a, const Span& b) {
  const uintptr_t x = (uintptr_t)a.p, y = (uintptr_t)b.p;
  return a.p && b.p && x < y + b.bytes && y < x + a.bytes;
}

int check_extents(const char* what, uint32_t rows, uint32_t columns, uint32_t positions) {
  if (rows == 0 || columns == 0 || positions == 0 || rows > K3_DENSE_MAX_EXTENT ||
      columns > K3_DENSE_MAX_EXTENT || positions > K3_DENSE_MAX_EXTENT)
    return spine_fail(K3_SPINE_E_INVALID,
                      "%s: rows (%u), columns (%u) and positions (%u) must be 1..%u", what, rows,
                      columns, positions, K3_DENSE_MAX_EXTENT);
  return K3_SPINE_OK;
}

int check_header(const char* what, uint32_t abi, uint32_t bytes, uint64_t want, uint32_t reserved) {
  if (abi != K3_DENSE_ABI_V1 || bytes != want || reserved != 0)
    return spine_fail(K3_SPINE_E_INVALID,
                      "%s: descriptor version %u, size %u or reserved field is not this ABI's "
                      "(%u, %llu, 0)",
                      what, abi, bytes, K3_DENSE_ABI_V1, (unsigned long long)want);
  return K3_SPINE_OK;
}

int check_dtype(const char* what, const char* name, uint32_t dtype) {
  if (dtype != K3_DTYPE_F32 && dtype != K3_DTYPE_BF16)
    return spine_fail(K3_SPINE_E_INVALID, "%s: %s is neither fp32 nor BF16", what, name);
  return K3_SPINE_OK;
}

// sizes: whether the pointers are checked, too (a size query has no buffers yet).
template <int NI, int NO>
int check_spans(const char* what, const Span (&in)[NI], const Span (&out)[NO], bool sizes) {
  for (const Span& s : in)
    if (((uintptr_t)s.p & (s.align - 1)) != 0)
      return spine_fail(K3_SPINE_E_INVALID, "%s: %s is not aligned to %u bytes", what, s.name,
                        s.align);
  for (const Span& s : out)
    if (((uintptr_t)s.p & (s.align - 1)) != 0)
      return spine_fail(K3_SPINE_E_INVALID, "%s: %s is not aligned to %u bytes", what, s.name,
                        s.align);
  if (sizes) return K3_SPINE_OK;
  for (int i = 0; i < NO; ++i) {
    for (const Span& s : in)
      if (overlap(out[i], s))
        return spine_fail(K3_SPINE_E_INVALID, "%s: %s overlaps %s", what, out[i].name, s.name);
    for (int j = 0; j < i; ++j)
      if (overlap(out[i], out[j]))
        return spine_fail(K3_SPINE_E_INVALID, "%s: %s overlaps %s", what, out[i].name,
                          out[j].name);
  }
  return K3_SPINE_OK;
}

#define K3_TRY(call)                       \
  do {                                     \
    const int rc_ = (call);                \
    if (rc_ != K3_SPINE_OK) return rc_;    \
  } while (0)

int check_linear(const K3HipLinearV1* op, bool sizes) {
  const char* what = "linear";
  if (!op) return spine_fail(K3_SPINE_E_INVALID, "%s: null descriptor", what);
  K3_TRY(check_header(what, op->abi_version, op->struct_bytes, sizeof(*op), op->reserved));
  K3_TRY(check_extents(what, op->rows, op->columns, op->positions));
  K3_TRY(check_dtype(what, "x_dtype", op->x_dtype));
  K3_TRY(check_dtype(what, "out_dtype", op->out_dtype));
  if (op->matrix_kind != K3_SPINE_MATRIX_BF16 && op->matrix_kind != K3_SPINE_MATRIX_INT8)
    return spine_fail(K3_SPINE_E_INVALID, "%s: unknown matrix kind %u", what, op->matrix_kind);
  if (op->activation > K3_DENSE_ACT_GELU)
    return spine_fail(K3_SPINE_E_INVALID, "%s: unknown activation %u", what, op->activation);
  const bool int8 = op->matrix_kind == K3_SPINE_MATRIX_INT8;
  if (!sizes && (!op->weights || !op->x || !op->out || (int8 && !op->row_scales)))
    return spine_fail(K3_SPINE_E_INVALID, "%s: null weights, row scales, x or out", what);
  if (!int8 && op->row_scales)
    return spine_fail(K3_SPINE_E_INVALID, "%s: BF16 weights take no row scales", what);
  const uint64_t R = op->rows, C = op->columns, P = op->positions;
  const unsigned ex = (unsigned)elem(op->x_dtype), eo = (unsigned)elem(op->out_dtype);
  const bool in_place = op->residual == op->out;
  const Span in[] = {{"weights", op->weights, R * C * (int8 ? 1 : 2), int8 ? 1u : 2u},
                     {"row_scales", op->row_scales, R * 4, 4},
                     {"bias", op->bias, R * 4, 4},
                     {"x", op->x, P * C * ex, ex},
                     {"residual", in_place ? nullptr : op->residual, P * R * eo, eo}};
  const Span out[] = {{"out", op->out, P * R * eo, eo}};
  return check_spans(what, in, out, sizes);
}

int check_gated(const K3HipGatedV1* op, bool sizes) {
  const char* what = "gated feed-forward";
  if (!op) return spine_fail(K3_SPINE_E_INVALID, "%s: null descriptor", what);
  K3_TRY(check_header(what, op->abi_version, op->struct_bytes, sizeof(*op), op->reserved));
  K3_TRY(check_extents(what, op->rows, op->columns, op->positions));
  K3_TRY(check_dtype(what, "x_dtype", op->x_dtype));
  K3_TRY(check_dtype(what, "out_dtype", op->out_dtype));
  if (op->matrix_kind != K3_SPINE_MATRIX_BF16 && op->matrix_kind != K3_SPINE_MATRIX_INT8)
    return spine_fail(K3_SPINE_E_INVALID, "%s: unknown matrix kind %u", what, op->matrix_kind);
  if (op->activation != K3_ACT_SITU && op->activation != K3_ACT_SILU)
    return spine_fail(K3_SPINE_E_INVALID, "%s: unknown activation %u", what, op->activation);
  const bool int8 = op->matrix_kind == K3_SPINE_MATRIX_INT8;
  if (!sizes && (!op->gate || !op->up || !op->x || !op->out ||
                 (int8 && (!op->gate_scales || !op->up_scales))))
    return spine_fail(K3_SPINE_E_INVALID, "%s: null matrix, scales, x or out", what);
  if (!sizes && !op->out_gate != !op->out_up)
    return spine_fail(K3_SPINE_E_INVALID, "%s: out_gate and out_up are kept together", what);
  if (!int8 && (op->gate_scales || op->up_scales))
    return spine_fail(K3_SPINE_E_INVALID, "%s: BF16 weights take no row scales", what);
  const uint64_t R = op->rows, C = op->columns, P = op->positions;
  const unsigned ex = (unsigned)elem(op->x_dtype), eo = (unsigned)elem(op->out_dtype);
  const Span in[] = {{"gate", op->gate, R * C * (int8 ? 1 : 2), int8 ? 1u : 2u},
                     {"up", op->up, R * C * (int8 ? 1 : 2), int8 ? 1u : 2u},
                     {"gate_scales", op->gate_scales, R * 4, 4},
                     {"up_scales", op->up_scales, R * 4, 4},
                     {"x", op->x, P * C * ex, ex}};
  const Span out[] = {{"out", op->out, P * R * eo, eo},
                      {"out_gate", op->out_gate, P * R * eo, eo},
                      {"out_up", op->out_up, P * R * eo, eo}};
  return check_spans(what, in, out, sizes);
}

int check_grad(const K3HipGatedGradV1* op, bool sizes) {
  const char* what = "gated feed-forward gradient";
  if (!op) return spine_fail(K3_SPINE_E_INVALID, "%s: null descriptor", what);
  K3_TRY(check_header(what, op->abi_version, op->struct_bytes, sizeof(*op), op->reserved));
  K3_TRY(check_extents(what, op->rows, op->columns, op->positions));
  K3_TRY(check_dtype(what, "dtype", op->dtype));
  if (op->activation != K3_ACT_SITU && op->activation != K3_ACT_SILU)
    return spine_fail(K3_SPINE_E_INVALID, "%s: unknown activation %u", what, op->activation);
  if (!sizes && (!op->gate || !op->up || !op->x || !op->g || !op->u || !op->grad || !op->d_x ||
                 !op->d_gate || !op->d_up))
    return spine_fail(K3_SPINE_E_INVALID, "%s: null input or output pointer", what);
  const uint64_t R = op->rows, C = op->columns, P = op->positions;
  const unsigned e = (unsigned)elem(op->dtype);
  const Span in[] = {{"gate", op->gate, R * C * 2, 2}, {"up", op->up, R * C * 2, 2},
                     {"x", op->x, P * C * e, e},       {"g", op->g, P * R * e, e},
                     {"u", op->u, P * R * e, e},       {"grad", op->grad, P * R * e, e}};
  const Span out[] = {{"d_x", op->d_x, P * C * e, e},
                      {"d_gate", op->d_gate, R * C * e, e},
                      {"d_up", op->d_up, R * C * e, e}};
  return check_spans(what, in, out, sizes);
}

int check_workspace(const char* what, const void* ws, uint64_t bytes, uint64_t need) {
  const bool none = need == K3_DENSE_NO_WORKSPACE && !ws;
  if (!none && (!ws || ((uintptr_t)ws & 255u) != 0 || bytes < need))
    return spine_fail(K3_SPINE_E_INVALID,
                      "%s: the workspace must be %llu bytes at a 256-byte boundary, got %llu at %p",
                      what, (unsigned long long)need, (unsigned long long)bytes, ws);
  const hipError_t e = hipGetLastError();  // an earlier call's, not this one's
  if (e != hipSuccess)
    return spine_fail(K3_SPINE_E_RUNTIME, "%s preflight: %s", what, hipGetErrorString(e));
  return K3_SPINE_OK;
}

// Nothing that the host code throws leaves the C surface.
template <typename F>
int guarded(const char* what, F f) {
  try {
    return f();
  } catch (...) {
    return spine_fail(K3_SPINE_E_RUNTIME, "%s: out of host memory", what);
  }
}
template <typename F>
uint64_t guarded_size(const char* what, F f) {
  uint64_t n = 0;
  (void)guarded(what, [&] {
    n = f();
    return K3_SPINE_OK;
  });
  return n;
}

}  // namespace
}  // namespace k3

using namespace k3;

static_assert(sizeof(K3HipLinearV1) == 88, "descriptor ABI drift");
static_assert(sizeof(K3HipGatedV1) == 104, "descriptor ABI drift");
static_assert(sizeof(K3HipGatedGradV1) == 104, "descriptor ABI drift");

extern "C" {

uint64_t k3_hip_linear_workspace_bytes(const K3HipLinearV1* op) {
  if (check_linear(op, true) != K3_SPINE_OK) return 0;
  return guarded_size("linear", [&] { return dense_linear_workspace(*op); });
}

int k3_hip_linear(const K3HipLinearV1* op, void* workspace, uint64_t workspace_bytes,
                  void* stream) {
  K3_TRY(check_linear(op, false));
  return guarded("linear", [&] {
    K3_TRY(check_workspace("linear", workspace, workspace_bytes, dense_linear_workspace(*op)));
    return dense_linear(*op, workspace, static_cast<hipStream_t>(stream));
  });
}

uint64_t k3_hip_gated_ffn_workspace_bytes(const K3HipGatedV1* op) {
  if (check_gated(op, true) != K3_SPINE_OK) return 0;
  return guarded_size("gated feed-forward", [&] { return dense_gated_workspace(*op); });
}

int k3_hip_gated_ffn(const K3HipGatedV1* op, void* workspace, uint64_t workspace_bytes,
                     void* stream) {
  K3_TRY(check_gated(op, false));
  return guarded("gated feed-forward", [&] {
    K3_TRY(check_workspace("gated feed-forward", workspace, workspace_bytes,
                           dense_gated_workspace(*op)));
    return dense_gated(*op, workspace, static_cast<hipStream_t>(stream));
  });
}

uint64_t k3_hip_gated_ffn_grad_workspace_bytes(const K3HipGatedGradV1* op) {
  if (check_grad(op, true) != K3_SPINE_OK) return 0;
  return guarded_size("gated feed-forward gradient",
                      [&] { return dense_gated_grad_workspace(*op); });
}

int k3_hip_gated_ffn_grad(const K3HipGatedGradV1* op, void* workspace, uint64_t workspace_bytes,
                          void* stream) {
  K3_TRY(check_grad(op, false));
  return guarded("gated feed-forward gradient", [&] {
    K3_TRY(check_workspace("gated feed-forward gradient", workspace, workspace_bytes,
                           dense_gated_grad_workspace(*op)));
    return dense_gated_grad(*op, workspace, static_cast<hipStream_t>(stream));
  });
}

}  // extern "C"
