// gf_fp8_quantize: a matrix to block-scaled 8-bit values, along its rows, along its columns (written transposed), or both at once.
//
// Memory bounds it: a value is read once and leaves as one byte for each form.  A workgroup takes a tile of 128 x 128, which is a block of either
// form, so every scale is known inside it.  A thread holds 8 x 8 values: its 8 columns of a row are one 16-byte load of 16-bit values and one
// 8-byte store of codes, its 8 rows of a column are one 8-byte store into the transposed tile in LDS.  Along the rows alone nothing is shared beyond
// 16 lanes: tiles are 32 rows then, without LDS, so that a few hundred rows still fill the chip.  Measured: 8192 x 4096 bfloat16 values along the rows in
// 18 us (5.5 TB/s); 4096 x 4096 both ways, float32 as a weight and bfloat16 as its input in one launch, in 31-36 us (168 MB, 4.7-5.4 TB/s).
#include "../common.hpp"
#include "fp8.hpp"
#include "fp8_calls.hpp"
#include "geneface_train_hip.h"

namespace gf {

constexpr int kTile = 128;

struct Scratch {
    uint32_t most[4][kTile];                                           // a wave's largest magnitudes by column
    uint8_t turned[kTile * kTile];
};

// tile `at` of a matrix
template <typename T>
__device__ __forceinline__ void quantize_tile(const gf_fp8_quantize_t& d, const uint32_t at, Scratch& lds) {
    auto& most = lds.most;
    uint8_t* turned = lds.turned;
    const uint32_t blocks_r = (uint32_t)((d.rows + kTile - 1) / kTile), blocks_c = (uint32_t)((d.cols + kTile - 1) / kTile);
    const int t = threadIdx.x, j = t & 15, g = t >> 4, wave = t >> 6;  // columns 8j..8j+7 of the tile, rows 8g..8g+7
    const uint32_t br = at / blocks_c, bc = at % blocks_c;
    if (br >= blocks_r) return;
    const uint64_t r0 = (uint64_t)br * kTile + 8 * g, c0 = (uint64_t)bc * kTile + 8 * j;
    const bool by_tile = d.tiles != 0;

    Eight<T> x[8];
    const int left = c0 < d.cols ? (int)min((uint64_t)8, d.cols - c0) : 0;
    const T* src = (const T*)d.src;
#pragma unroll
    for (int r = 0; r < 8; ++r) {
        const bool there = r0 + r < d.rows && left > 0;
        x[r].load(src + (there ? (r0 + r) * d.ld + c0 : 0), there ? left : 0);
    }
    uint32_t rm[8], cm[8];
#pragma unroll
    for (int r = 0; r < 8; ++r) rm[r] = x[r].amax();
    if (by_tile) {
        uint32_t m = 0;
#pragma unroll
        for (int r = 0; r < 8; ++r) m = max(m, rm[r]);
        m = row_max_u32(m);
        m = max(m, (uint32_t)__shfl_xor((int)m, 16));
        m = max(m, (uint32_t)__shfl_xor((int)m, 32));
        if ((t & 63) == 0) most[wave][0] = m;
    } else {
#pragma unroll
        for (int r = 0; r < 8; ++r) rm[r] = row_max_u32(rm[r]);
        column_amax(x, cm);
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            cm[c] = max(cm[c], (uint32_t)__shfl_xor((int)cm[c], 16));
            cm[c] = max(cm[c], (uint32_t)__shfl_xor((int)cm[c], 32));
        }
        if ((g & 3) == 0) {
#pragma unroll
            for (int c = 0; c < 8; ++c) most[wave][8 * j + c] = cm[c];
        }
    }
    __syncthreads();
    if (by_tile) {
        const uint32_t b = scale_byte(max(max(most[0][0], most[1][0]), max(most[2][0], most[3][0])));
#pragma unroll
        for (int k = 0; k < 8; ++k) rm[k] = cm[k] = b;
        if (t == 0) d.tile_scales[(uint64_t)br * blocks_c + bc] = (uint8_t)b;
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            rm[k] = scale_byte(rm[k]);
            cm[k] = scale_byte(max(max(most[0][8 * j + k], most[1][8 * j + k]), max(most[2][8 * j + k], most[3][8 * j + k])));
        }
    }
    if (d.row_codes) {
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            if (r0 + r >= d.rows) break;
            *reinterpret_cast<uint2*>(d.row_codes + (r0 + r) * ((uint64_t)blocks_c * kTile) + c0) = coded(x[r].encode(scale_value(rm[r])), rm[r]);
            if (!by_tile && j == 0) d.row_scales[(uint64_t)bc * d.row_pitch + r0 + r] = (uint8_t)rm[r];
        }
    }
    if (!d.col_codes) return;
    // column c of the tile is 128 bytes, its 16-byte piece p at place p ^ ((c >> 3) & 7): the lanes of a store differ in c >> 3
#pragma unroll
    for (int c = 0; c < 8; ++c) {
        *reinterpret_cast<uint2*>(turned + (8 * j + c) * kTile + (((g >> 1) ^ (j & 7)) << 4) + (g & 1) * 8) = coded(encode_column(x, c, scale_value(cm[c])), cm[c]);
        if (!by_tile && g == 0 && c0 + c < d.cols) d.col_scales[(uint64_t)br * d.col_pitch + c0 + c] = (uint8_t)cm[c];
    }
    __syncthreads();
    const uint64_t pitch = (uint64_t)blocks_r * kTile;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const int c = q * 32 + (t >> 3), p = t & 7;
        const uint64_t col = (uint64_t)bc * kTile + c;
        if (col < d.cols)
            *reinterpret_cast<i32x4*>(d.col_codes + col * pitch + (uint64_t)br * kTile + p * 16) = *reinterpret_cast<const i32x4*>(turned + c * kTile + ((p ^ ((c >> 3) & 7)) << 4));
    }
}

template <typename T>
__global__ __launch_bounds__(256) void k_quantize(const gf_fp8_quantize_t d) {
    __shared__ __align__(16) Scratch lds;
    quantize_tile<T>(d, blockIdx.y * gridDim.x + blockIdx.x, lds);
}

template <typename A, typename B>
__global__ __launch_bounds__(256) void k_quantize_two(const gf_fp8_quantize_t a, const gf_fp8_quantize_t b, const uint32_t tiles_a) {
    __shared__ __align__(16) Scratch lds;
    if (blockIdx.x < tiles_a) quantize_tile<A>(a, blockIdx.x, lds);
    else quantize_tile<B>(b, blockIdx.x - tiles_a, lds);
}

template <typename T>
__global__ __launch_bounds__(256) void k_quantize_rows(const gf_fp8_quantize_t d, const uint32_t blocks_c) {
    const int j = threadIdx.x & 15, g = threadIdx.x >> 4;
    const uint32_t at = blockIdx.y * gridDim.x + blockIdx.x, br = at / blocks_c, bc = at % blocks_c;      // behind the last: rows that are not there
    const uint64_t r0 = (uint64_t)br * 32 + 2 * g, c0 = (uint64_t)bc * kTile + 8 * j;
    Eight<T> x[2];
    const int left = c0 < d.cols ? (int)min((uint64_t)8, d.cols - c0) : 0;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        const bool there = r0 + r < d.rows && left > 0;
        x[r].load((const T*)d.src + (there ? (r0 + r) * d.ld + c0 : 0), there ? left : 0);
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        const uint32_t b = scale_byte(row_max_u32(x[r].amax()));
        if (r0 + r >= d.rows) break;
        *reinterpret_cast<uint2*>(d.row_codes + (r0 + r) * ((uint64_t)blocks_c * kTile) + c0) = coded(x[r].encode(scale_value(b)), b);
        if (j == 0) d.row_scales[(uint64_t)bc * d.row_pitch + r0 + r] = (uint8_t)b;
    }
}

static uint64_t tiles_of(const gf_fp8_quantize_t& d) { return ((d.rows + kTile - 1) / kTile) * ((d.cols + kTile - 1) / kTile); }
static bool rows_alone(const gf_fp8_quantize_t& d) { return !d.col_codes && !d.tiles; }

// f(T()) with the type that dtype names
template <typename F>
static void with_type(uint32_t dtype, F f) {
    if (dtype == F32) f(float());
    else if (dtype == BF16) f(__bf16());
    else f(_Float16());
}

static void launch_quantize(const gf_fp8_quantize_t& d, hipStream_t s) {
    auto grid = [](uint64_t n) { const uint64_t wide = 1u << 22; return dim3((uint32_t)(n < wide ? n : wide), (uint32_t)((n + wide - 1) / wide)); };      // work-items along x lie below 2^32
    const uint64_t cb = (d.cols + kTile - 1) / kTile;
    with_type(d.dtype, [&](auto t) {
        if (rows_alone(d)) k_quantize_rows<decltype(t)><<<grid((d.rows + 31) / 32 * cb), 256, 0, s>>>(d, (uint32_t)cb);
        else k_quantize<decltype(t)><<<grid(tiles_of(d)), 256, 0, s>>>(d);
    });
}

static int quantize_error(const gf_fp8_quantize_t& d) {
    if (!d.src || (!d.row_codes && !d.col_codes)) return gf_set_error(GF_ERR_INVALID, "gf_fp8_quantize: null pointer");
    if (d.tiles ? !d.tile_scales : ((d.row_codes && !d.row_scales) || (d.col_codes && !d.col_scales)))
        return gf_set_error(GF_ERR_INVALID, "gf_fp8_quantize: null scales");
    if (d.dtype > F16) return gf_set_error(GF_ERR_INVALID, "gf_fp8_quantize: unknown dtype %u", d.dtype);
    if (d.ld < d.cols) return gf_set_error(GF_ERR_INVALID, "gf_fp8_quantize: ld < cols");
    if (!d.tiles && ((d.row_codes && d.row_pitch < d.rows) || (d.col_codes && d.col_pitch < d.cols)))
        return gf_set_error(GF_ERR_INVALID, "gf_fp8_quantize: scale pitch too small");
    const uint64_t rb = (d.rows + kTile - 1) / kTile, cb = (d.cols + kTile - 1) / kTile;
    if (rb > 0x1fffffffull || cb > 0x1fffffffull / rb) return gf_set_error(GF_ERR_INVALID, "gf_fp8_quantize: matrix too large");
    return GF_OK;
}

int quantize_two(const gf_fp8_quantize_t& a, const gf_fp8_quantize_t& b, void* stream) {
    if (const int rc = quantize_error(a)) return rc;
    if (const int rc = quantize_error(b)) return rc;
    const hipStream_t s = gf_stream(stream);
    const uint64_t ta = tiles_of(a), tb = tiles_of(b);
    if (rows_alone(a) || rows_alone(b) || ta + tb > 1u << 22) {
        launch_quantize(a, s);
        launch_quantize(b, s);
    } else {
        with_type(a.dtype, [&](auto x) {
            with_type(b.dtype, [&](auto y) { k_quantize_two<decltype(x), decltype(y)><<<(uint32_t)(ta + tb), 256, 0, s>>>(a, b, (uint32_t)ta); });
        });
    }
    return gf_check_launch("gf_fp8_quantize");
}

}  // namespace gf

using namespace gf;

GF_EXPORT int gf_fp8_quantize(const gf_fp8_quantize_t* d, void* stream) {
    if (!d) return gf_set_error(GF_ERR_INVALID, "gf_fp8_quantize: null descriptor");
    if (d->rows == 0 || d->cols == 0) return GF_OK;
    if (const int rc = quantize_error(*d)) return rc;
    launch_quantize(*d, gf_stream(stream));
    return gf_check_launch("gf_fp8_quantize");
}
