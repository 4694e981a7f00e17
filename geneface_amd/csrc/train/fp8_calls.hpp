// What a layer's calls enqueue together: a launch of few workgroups costs some 4 us however little it does, and two of them side by side fill more of the chip.
#pragma once
#include "geneface_train_hip.h"

namespace gf {

// Two independent matrices or products in one launch each; what has no such form is enqueued one after the other.
int quantize_two(const gf_fp8_quantize_t& a, const gf_fp8_quantize_t& b, void* stream);
int matmul_two(const gf_fp8_matmul_t& a, const gf_fp8_matmul_t& b, void* stream);

// gf_fp8_thin with the weight as values [n, k]: brought to 8 bits on the way, and left by columns with its scale for the backward call where that is wanted
// (col_codes, scale; or both NULL).  codes and scale of the descriptor are not read then.
struct ThinWeight { const void* w; uint64_t ldw; uint32_t dtype; uint8_t *col_codes, *scale; };
int thin_forward(const gf_fp8_thin_t& d, const ThinWeight* w, void* stream);

}  // namespace gf
