// Two independent matrices or products in one launch each, for a layer's operands and its gradients: a launch of few workgroups costs some 4 us however
// little it does, and two of them side by side fill more of the chip.  What has no such form is enqueued one after the other.
#pragma once
#include "geneface_train_hip.h"

namespace gf {

int quantize_two(const gf_fp8_quantize_t& a, const gf_fp8_quantize_t& b, void* stream);
int matmul_two(const gf_fp8_matmul_t& a, const gf_fp8_matmul_t& b, void* stream);

}  // namespace gf
