// Dense layers over many positions (k3_dense.hip); include/k3_hip_dense_abi.h states
// what they compute.  Statuses are the K3_SPINE_* codes.
#pragma once

#include <hip/hip_runtime_api.h>
#include <stdint.h>

#include "../../include/k3_hip_dense_abi.h"

namespace k3 {

// Scratch bytes of a valid descriptor (K3_DENSE_NO_WORKSPACE: none).
uint64_t dense_linear_workspace(const K3HipLinearV1& op);
uint64_t dense_gated_workspace(const K3HipGatedV1& op);
uint64_t dense_gated_grad_workspace(const K3HipGatedGradV1& op);

// The descriptor is valid and the workspace is large enough and aligned.
int dense_linear(const K3HipLinearV1& op, void* ws, hipStream_t st);
int dense_gated(const K3HipGatedV1& op, void* ws, hipStream_t st);
int dense_gated_grad(const K3HipGatedGradV1& op, void* ws, hipStream_t st);

}  // namespace k3
