/* Compiled as plain C11 against include/k3_hip_dense_abi.h and k3_hip_sample_abi.h and
 * linked to the library: sizes and refusals, nothing that needs a device. */
#include <stdio.h>
#include <string.h>

#include "k3_hip_dense_abi.h"
#include "k3_hip_sample_abi.h"

#define CHECK(c)                                                     \
  do {                                                               \
    if (!(c)) {                                                      \
      fprintf(stderr, "check failed: %s (line %d)\n", #c, __LINE__); \
      return 1;                                                      \
    }                                                                \
  } while (0)

_Static_assert(sizeof(K3HipLinearV1) == 88, "descriptor size");
_Static_assert(sizeof(K3HipGatedV1) == 104, "descriptor size");
_Static_assert(sizeof(K3HipGatedGradV1) == 104, "descriptor size");
_Static_assert(sizeof(K3HipSampleV1) == 80, "descriptor size");

int main(void) {
  K3HipLinearV1 down = {K3_DENSE_ABI_V1, sizeof down, K3_SPINE_MATRIX_BF16, K3_DENSE_ACT_NONE,
                        K3_DTYPE_BF16, K3_DTYPE_BF16, 7168, 6144, 1, 0,
                        NULL, NULL, NULL, NULL, NULL, NULL};
  CHECK(k3_hip_linear_workspace_bytes(&down) == K3_DENSE_NO_WORKSPACE);
  CHECK(k3_hip_linear(&down, NULL, 0, NULL) == K3_SPINE_E_INVALID);
  CHECK(strstr(k3_hip_spine_last_error(), "null") != NULL);
  down.x_dtype = K3_DTYPE_F32;
  down.positions = 1000;
  CHECK(k3_hip_linear_workspace_bytes(&down) >= UINT64_C(3) * 1000 * 6144 * 2);
  down.reserved = 1;
  CHECK(k3_hip_linear_workspace_bytes(&down) == 0);
  K3HipGatedV1 gated;
  memset(&gated, 0, sizeof gated);
  CHECK(k3_hip_gated_ffn(&gated, NULL, 0, NULL) == K3_SPINE_E_INVALID);
  CHECK(k3_hip_gated_ffn_workspace_bytes(&gated) == 0);
  CHECK(k3_hip_gated_ffn_grad(NULL, NULL, 0, NULL) == K3_SPINE_E_INVALID);
  CHECK(k3_hip_gated_ffn_grad_workspace_bytes(NULL) == 0);
  CHECK(k3_hip_sample(NULL, NULL, 0, NULL) == K3_SPINE_E_INVALID);
  printf("ok\n");
  return 0;
}
