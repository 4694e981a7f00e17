// gf_fp8_quantize: a matrix to block-scaled 8-bit values, along its rows, along its columns (written transposed), or both at once.
//
// Memory bounds it: a value is read once and leaves as one byte for each form.  A workgroup takes a tile of 128 x 128, which is a block of either
// form, so every scale is known inside it.  A thread holds 8 x 8 values: its 8 columns of a row are one 16-byte load of 16-bit values and one
// 8-byte store of codes, its 8 rows of a column are one 8-byte store into the transposed tile in LDS.
#include "../common.hpp"
#include "fp8.hpp"
#include "geneface_train_hip.h"

namespace gf {

constexpr int kTile = 128, kPitch = 144;      // bytes of a row of the transposed tile; 144: eight bytes of 16 lanes fall on different banks

// wide: 2: the address is a multiple of 16 bytes, 1: of four values, 0: of one
template <typename T>
__device__ __forceinline__ void load8_of(const T* src, int left, int wide, float out[8]) {
    if (left >= 8 && wide == 2) {
        typedef T vec __attribute__((ext_vector_type(16 / sizeof(T))));
#pragma unroll
        for (int q = 0; q < (int)sizeof(T) / 2; ++q) {
            const vec v = reinterpret_cast<const vec*>(src)[q];
#pragma unroll
            for (int i = 0; i < 16 / (int)sizeof(T); ++i) out[q * (16 / sizeof(T)) + i] = (float)v[i];
        }
        return;
    }
    if (left >= 8 && wide == 1) { load4(src, out); load4(src + 4, out + 4); return; }
#pragma unroll
    for (int i = 0; i < 8; ++i) out[i] = i < left ? (float)src[i] : 0.0f;
}

template <typename T>
__global__ __launch_bounds__(256) void k_quantize(const gf_fp8_quantize_t d, const uint32_t blocks_r, const uint32_t blocks_c, const int wide) {
    __shared__ uint32_t colmax[kTile];
    __shared__ uint32_t rowmax_all;
    __shared__ __align__(16) uint8_t turned[kTile * kPitch];
    const int t = threadIdx.x, j = t & 15, g = t >> 4;                 // columns 8j..8j+7 of the tile, rows 8g..8g+7
    const uint32_t br = blockIdx.x / blocks_c, bc = blockIdx.x % blocks_c;
    const uint64_t r0 = (uint64_t)br * kTile + 8 * g, c0 = (uint64_t)bc * kTile + 8 * j;
    const bool by_tile = d.tiles != 0;
    if (t < kTile) colmax[t] = 0;
    if (t == 0) rowmax_all = 0;
    __syncthreads();

    float x[8][8];
    const int left = c0 < d.cols ? (int)min((uint64_t)8, d.cols - c0) : 0;
    const T* src = (const T*)d.src;
#pragma unroll
    for (int r = 0; r < 8; ++r) {
        const bool there = r0 + r < d.rows && left > 0;
        load8_of(src + (there ? (r0 + r) * d.ld + c0 : 0), there ? left : 0, wide, x[r]);
    }
    uint32_t rm[8], cm[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        rm[k] = cm[k] = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            rm[k] = max(rm[k], abs_bits(x[k][i]));
            cm[k] = max(cm[k], abs_bits(x[i][k]));
        }
    }
    if (by_tile) {
        uint32_t m = 0;
#pragma unroll
        for (int k = 0; k < 8; ++k) m = max(m, rm[k]);
        m = row_max_u32(m);
        if (j == 0) atomicMax(&rowmax_all, m);
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) rm[k] = row_max_u32(rm[k]);
        if (d.col_codes) {
#pragma unroll
            for (int k = 0; k < 8; ++k) atomicMax(&colmax[8 * j + k], cm[k]);
        }
    }
    __syncthreads();
    if (by_tile) {
        const uint32_t b = scale_byte(rowmax_all);
#pragma unroll
        for (int k = 0; k < 8; ++k) rm[k] = cm[k] = b;
        if (t == 0) d.tile_scales[(uint64_t)br * blocks_c + bc] = (uint8_t)b;
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            rm[k] = scale_byte(rm[k]);
            cm[k] = d.col_codes ? scale_byte(colmax[8 * j + k]) : 0;
        }
    }
    if (d.row_codes) {
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            if (r0 + r >= d.rows) break;
            const float inv = scale_inverse(rm[r]);
            uint2 w = {encode4(x[r], inv), encode4(x[r] + 4, inv)};
            *reinterpret_cast<uint2*>(d.row_codes + (r0 + r) * ((uint64_t)blocks_c * kTile) + c0) = w;
            if (!by_tile && j == 0) d.row_scales[(uint64_t)bc * d.row_pitch + r0 + r] = (uint8_t)rm[r];
        }
    }
    if (!d.col_codes) return;
#pragma unroll
    for (int c = 0; c < 8; ++c) {
        float y[8];
#pragma unroll
        for (int r = 0; r < 8; ++r) y[r] = x[r][c];
        const float inv = scale_inverse(cm[c]);
        uint2 w = {encode4(y, inv), encode4(y + 4, inv)};
        *reinterpret_cast<uint2*>(turned + (8 * j + c) * kPitch + 8 * g) = w;
        if (!by_tile && g == 0 && c0 + c < d.cols) d.col_scales[(uint64_t)br * d.col_pitch + c0 + c] = (uint8_t)cm[c];
    }
    __syncthreads();
    const uint64_t pitch = (uint64_t)blocks_r * kTile;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const int c = q * 32 + (t >> 3), at = (t & 7) * 16;
        const uint64_t col = (uint64_t)bc * kTile + c;
        if (col < d.cols) *reinterpret_cast<i32x4*>(d.col_codes + col * pitch + (uint64_t)br * kTile + at) = *reinterpret_cast<const i32x4*>(turned + c * kPitch + at);
    }
}

}  // namespace gf

using namespace gf;

GF_EXPORT int gf_fp8_quantize(const gf_fp8_quantize_t* d, void* stream) {
    if (!d) return gf_set_error(GF_ERR_INVALID, "gf_fp8_quantize: null descriptor");
    if (d->rows == 0 || d->cols == 0) return GF_OK;
    if (!d->src || (!d->row_codes && !d->col_codes)) return gf_set_error(GF_ERR_INVALID, "gf_fp8_quantize: null pointer");
    if (d->tiles ? !d->tile_scales : ((d->row_codes && !d->row_scales) || (d->col_codes && !d->col_scales)))
        return gf_set_error(GF_ERR_INVALID, "gf_fp8_quantize: null scales");
    if (d->dtype > F16) return gf_set_error(GF_ERR_INVALID, "gf_fp8_quantize: unknown dtype %u", d->dtype);
    if (d->ld < d->cols) return gf_set_error(GF_ERR_INVALID, "gf_fp8_quantize: ld < cols");
    if (!d->tiles && ((d->row_codes && d->row_pitch < d->rows) || (d->col_codes && d->col_pitch < d->cols)))
        return gf_set_error(GF_ERR_INVALID, "gf_fp8_quantize: scale pitch too small");
    const uint64_t rb = (d->rows + kTile - 1) / kTile, cb = (d->cols + kTile - 1) / kTile;
    if (rb > 0x7fffffffull || cb > 0x7fffffffull / rb) return gf_set_error(GF_ERR_INVALID, "gf_fp8_quantize: matrix too large");
    const uint64_t size = d->dtype == F32 ? 4 : 2, at = (uintptr_t)d->src | d->ld * size;
    const int wide = at % 16 == 0 ? 2 : at % (4 * size) == 0 ? 1 : 0;
    const uint32_t grid = (uint32_t)(rb * cb);
    const hipStream_t s = gf_stream(stream);
    if (d->dtype == F32) k_quantize<float><<<grid, 256, 0, s>>>(*d, (uint32_t)rb, (uint32_t)cb, wide);
    else if (d->dtype == BF16) k_quantize<__bf16><<<grid, 256, 0, s>>>(*d, (uint32_t)rb, (uint32_t)cb, wide);
    else k_quantize<_Float16><<<grid, 256, 0, s>>>(*d, (uint32_t)rb, (uint32_t)cb, wide);
    return gf_check_launch("gf_fp8_quantize");
}
