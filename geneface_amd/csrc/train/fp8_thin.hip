// gf_fp8_thin and gf_fp8_thin_backward: the linear layer where both of the weight's sides lie within one block of 128 -- the layers of the field's
// MLPs, over the samples of a training batch.
//
// Such a layer does 2 N K <= 32768 operations on N + K values of a row, far below what would keep the matrix units busy: memory bounds it.  What
// the general path moves besides x and y -- row codes of 128 bytes a row however short the row, written and read again -- is what these kernels
// avoid: a workgroup brings its 128 rows to 8 bits in LDS and multiplies them there.  The weight's codes stay in LDS for all its tiles.  Forward: x is
// read once, y and (for the weight's gradient) x by columns are written.  Backward: dy is read once for both products; the weight's gradient is
// added up in the registers of the workgroup over all its tiles, so that only a part per workgroup has to be joined.
// Measured, 262221 rows, 96 -> 128, float32: forward 52-55 us with the weight's own quantisation (260 MB, 4.7-5.0 TB/s), backward 61-65 (285 MB, 4.4-4.7 TB/s), the join of its 512 parts 8.
#include "../common.hpp"
#include "fp8.hpp"
#include "fp8_calls.hpp"
#include "fp8_join.hpp"
#include "geneface_train_hip.h"

namespace gf {

constexpr int kEdge = 128;

// Where byte 16 p of row r lies in a tile of rows of 128 bytes: the same piece of 16 consecutive rows on different banks (as the matrix
// instructions read them), and of rows 8 apart (as a thread of the transposition writes them) on at least eight.
__device__ __forceinline__ int spot(int r, int p) { return r * kEdge + ((p ^ ((r >> 1) & 7) ^ ((r >> 4) & 7)) << 4); }

// lane's 32 codes of row r, half `half` of the block
__device__ __forceinline__ i32x8 fragment(const uint8_t* tile, int r, int half, int lane) {
    const int p = half * 4 + (lane >> 5) * 2;
    const i32x4 lo = *reinterpret_cast<const i32x4*>(tile + spot(r, p)), hi = *reinterpret_cast<const i32x4*>(tile + spot(r, p + 1));
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}

// acc += a b^T over half a block
template <bool EXACT>
__device__ __forceinline__ f32x16 multiply_half(i32x8 a, i32x8 b, f32x16 acc, uint32_t sa, uint32_t sb) {
    if constexpr (EXACT) {
        const float wa = scale_value(sa), wb = scale_value(sb);
#pragma unroll
        for (int s = 0; s < 4; ++s)
            acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(widen8(a[2 * s], a[2 * s + 1], wa), widen8(b[2 * s], b[2 * s + 1], wb), acc, 0, 0, 0);
        return acc;
    } else {
        return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, acc, 0, 0, 0, (int)sa, 0, (int)sb);
    }
}

// A tile's 128 x 128 values in the threads' registers (thread: 8 columns from 8 (t % 16), 8 rows from 8 (t / 16)), and their blocks' scales.
template <typename T>
struct Tile {
    Eight<T> x[8];
    uint32_t rows[8], cols[8];      // scale bytes

    __device__ __forceinline__ void load(const T* src, uint64_t ld, uint64_t r0, uint64_t m, int width) {
        const int c0 = 8 * (threadIdx.x & 15), left = max(0, min(8, width - c0));
        const uint64_t row = r0 + 8 * (threadIdx.x >> 4);
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            const bool there = row + r < m && left > 0;
            x[r].load(src + (there ? (row + r) * ld + c0 : 0), there ? left : 0);
        }
    }
    __device__ __forceinline__ void scale_rows() {
#pragma unroll
        for (int r = 0; r < 8; ++r) rows[r] = scale_byte(row_max_u32(x[r].amax()));
    }
    // before and behind a barrier
    __device__ __forceinline__ void columns_to(uint32_t most[4][kEdge]) {
        column_amax(x, cols);
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            cols[c] = max(cols[c], (uint32_t)__shfl_xor((int)cols[c], 16));
            cols[c] = max(cols[c], (uint32_t)__shfl_xor((int)cols[c], 32));
        }
        if ((threadIdx.x & 48) == 0) {
#pragma unroll
            for (int c = 0; c < 8; ++c) most[threadIdx.x >> 6][8 * (threadIdx.x & 15) + c] = cols[c];
        }
    }
    __device__ __forceinline__ void scale_columns(const uint32_t most[4][kEdge]) {
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            const int at = 8 * (threadIdx.x & 15) + c;
            cols[c] = scale_byte(max(max(most[0][at], most[1][at]), max(most[2][at], most[3][at])));
        }
    }
    __device__ __forceinline__ void row_codes_to(uint8_t* tile, uint8_t* scales) const {      // a wave writes its own 32 rows
        const int j = threadIdx.x & 15, r0 = 8 * (threadIdx.x >> 4);
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            *reinterpret_cast<uint2*>(tile + spot(r0 + r, j >> 1) + (j & 1) * 8) = coded(x[r].encode(scale_value(rows[r])), rows[r]);
            if (j == 0) scales[r0 + r] = (uint8_t)rows[r];
        }
    }
    __device__ __forceinline__ void column_codes_to(uint8_t* tile) const {
        int t = threadIdx.x;
        asm volatile("" : "+v"(t));      // its places are worked out here, not kept in registers over all tiles: three workgroups' have to fit a CU
        const int c0 = 8 * (t & 15), g = t >> 4;
#pragma unroll
        for (int c = 0; c < 8; ++c) *reinterpret_cast<uint2*>(tile + spot(c0 + c, g >> 1) + (g & 1) * 8) = coded(encode_column(x, c, scale_value(cols[c])), cols[c]);
    }
};

// rows of 128 codes, `pitch` bytes apart, into a tile; rows from `rows` on become zeros
struct CodesTile {
    i32x4 v[4];
    __device__ __forceinline__ void load(const uint8_t* src, uint64_t pitch, int rows) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int r = q * 32 + (threadIdx.x >> 3), p = threadIdx.x & 7;
            v[q] = r < rows ? *reinterpret_cast<const i32x4*>(src + r * pitch + p * 16) : i32x4{0, 0, 0, 0};
        }
    }
    __device__ __forceinline__ void to(uint8_t* tile) const {
#pragma unroll
        for (int q = 0; q < 4; ++q) *reinterpret_cast<i32x4*>(tile + spot(q * 32 + (threadIdx.x >> 3), threadIdx.x & 7)) = v[q];
    }
};

// A wave's 32 rows times the 32 N' rows of `other`, to out [m, width]: `mine` holds the wave's codes and is overwritten as staging.
template <typename T>
__device__ __forceinline__ void rows_product(uint8_t* codes, const uint8_t* scales, const uint8_t* other, uint32_t other_scale, T* out, uint64_t r0, uint64_t m, int width) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, row = wave * 32 + (lane & 31);
    const i32x8 x0 = fragment(codes, row, 0, lane), x1 = fragment(codes, row, 1, lane);
    const uint32_t sx = scales[row];
    uint8_t* mine = codes + wave * 32 * kEdge;      // (spot() keeps a row's bytes within its 128)
    constexpr int EACH = 16 / (int)sizeof(T), PIECES = 32 / EACH, PITCH = 32 * (int)sizeof(T);
#pragma unroll 1
    for (int k = 0; 32 * k < width; ++k) {
        f32x16 acc;
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[e] = 0.0f;
        const int r = k * 32 + (lane & 31);
        acc = multiply_half<kExact<T>>(fragment(other, r, 0, lane), x0, acc, other_scale, sx);
        acc = multiply_half<kExact<T>>(fragment(other, r, 1, lane), x1, acc, other_scale, sx);
        // 32 x 32 results through LDS, so that a row's 128 (64) bytes leave together
        __builtin_amdgcn_s_waitcnt(0xc07f);
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const float v[4] = {acc[4 * g], acc[4 * g + 1], acc[4 * g + 2], acc[4 * g + 3]};
            const int at = (g * 8 + (lane >> 5) * 4) * (int)sizeof(T);
            store4((T*)(mine + (lane & 31) * PITCH + ((((at >> 4) ^ (lane >> 1)) & (PIECES - 1)) << 4) + (at & 15)), v);
        }
        __builtin_amdgcn_s_waitcnt(0xc07f);
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int q = 0; q < PIECES / 2; ++q) {
            const int rr = (q * 64 + lane) / PIECES, c = (q * 64 + lane) % PIECES;
            const i32x4 v = *reinterpret_cast<const i32x4*>(mine + rr * PITCH + (((c ^ (rr >> 1)) & (PIECES - 1)) << 4));
            const uint64_t to_row = r0 + wave * 32 + rr;
            const int col = k * 32 + c * EACH;
            if (to_row >= m || col >= width) continue;
            T* to = out + to_row * width + col;
            if (col + EACH <= width) {
                typedef int piece __attribute__((ext_vector_type(4), aligned(2)));
                *reinterpret_cast<piece*>(to) = v;
            } else {
                const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
                for (int i = 0; i < EACH; ++i) if (col + i < width) to[i] = e[i];
            }
        }
        __builtin_amdgcn_s_waitcnt(0xc07f);
        __builtin_amdgcn_wave_barrier();
    }
}

struct ThinForward {
    const void* x;
    uint64_t ldx, m;
    uint32_t n, k, tiles;
    const uint8_t *w_codes, *w_scale;      // [n, 128] and one byte
    void* y;
    uint8_t *col_codes, *col_scales;       // x by columns [k, 128 tiles] and [tiles, k], or NULL
    ThinWeight w;                          // the weight as values, or w.w NULL
};

// The weight's values to its codes in LDS, by every workgroup for itself (48 KB out of L2; a launch ahead that does it once
// takes 6 us), and by the first one for the backward call.  Returns the scale's byte.
template <typename W>
__device__ __forceinline__ uint32_t weight_to(uint8_t* weight, uint8_t* turned, uint32_t most[4][kEdge], uint8_t* scales, const ThinForward& d) {
    Tile<W> w;
    w.load((const W*)d.w.w, d.w.ldw, 0, d.n, d.k);
    uint32_t m = 0;
#pragma unroll
    for (int r = 0; r < 8; ++r) m = max(m, w.x[r].amax());
    m = row_max_u32(m);
    m = max(m, (uint32_t)__shfl_xor((int)m, 16));
    m = max(m, (uint32_t)__shfl_xor((int)m, 32));
    if ((threadIdx.x & 63) == 0) most[threadIdx.x >> 6][0] = m;
    __syncthreads();
    const uint32_t byte = scale_byte(max(max(most[0][0], most[1][0]), max(most[2][0], most[3][0])));
#pragma unroll
    for (int i = 0; i < 8; ++i) w.rows[i] = w.cols[i] = byte;
    w.row_codes_to(weight, scales);
    if (blockIdx.x == 0 && d.w.col_codes) {
        w.column_codes_to(turned);
        __syncthreads();
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int c = q * 32 + (threadIdx.x >> 3), p = threadIdx.x & 7;
            if (c < (int)d.k) *reinterpret_cast<i32x4*>(d.w.col_codes + c * kEdge + p * 16) = *reinterpret_cast<const i32x4*>(turned + spot(c, p));
        }
        if (threadIdx.x == 0) *d.w.scale = (uint8_t)byte;
    }
    return byte;
}

// Three workgroups a CU, as its LDS holds: 120 us for the layer in 32 bits, with two 129.
template <typename T>
__global__ __launch_bounds__(256, 3) void k_thin_forward(const ThinForward d) {
    __shared__ __align__(16) uint8_t weight[kEdge * kEdge], codes[kEdge * kEdge], turned[kEdge * kEdge];
    __shared__ uint32_t most[4][kEdge];
    __shared__ uint8_t scales[kEdge];
    uint32_t sw;
    if (d.w.w) {
        sw = d.w.dtype == F32 ? weight_to<float>(weight, turned, most, scales, d) : d.w.dtype == BF16 ? weight_to<__bf16>(weight, turned, most, scales, d)
                                                                                                      : weight_to<_Float16>(weight, turned, most, scales, d);
    } else {
        CodesTile w;
        w.load(d.w_codes, kEdge, d.n);
        w.to(weight);
        sw = *d.w_scale;
    }
    __syncthreads();
    for (uint32_t t = blockIdx.x; t < d.tiles; t += gridDim.x) {
        const uint64_t r0 = (uint64_t)t * kEdge;
        Tile<T> x;
        x.load((const T*)d.x, d.ldx, r0, d.m, d.k);
        x.scale_rows();
        x.row_codes_to(codes, scales);      // a wave's own rows: no barrier between writing and reading them
        if (d.col_codes) {
            x.columns_to(most);
            __syncthreads();      // also: everyone is done with the last tile
            x.scale_columns(most);
            x.column_codes_to(turned);
            if ((threadIdx.x >> 4) == 0) {
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    const uint32_t col = 8 * threadIdx.x + c;
                    if (col < d.k) d.col_scales[(uint64_t)t * d.k + col] = (uint8_t)x.cols[c];
                }
            }
        }
        __builtin_amdgcn_s_waitcnt(0xc07f);
        __builtin_amdgcn_wave_barrier();
        if (d.col_codes) {
            __syncthreads();
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int c = q * 32 + (threadIdx.x >> 3), p = threadIdx.x & 7;
                if (c < (int)d.k) *reinterpret_cast<i32x4*>(d.col_codes + ((uint64_t)c * d.tiles + t) * kEdge + p * 16) = *reinterpret_cast<const i32x4*>(turned + spot(c, p));
            }
        }
        rows_product<T>(codes, scales, weight, sw, (T*)d.y, r0, d.m, d.n);
    }
}

struct ThinBackward {
    const void* dy;
    uint64_t lddy, m;
    uint32_t n, k, tiles;
    const uint8_t *w_codes, *w_scale;          // the weight by columns [k, 128] and one byte
    const uint8_t *x_codes, *x_scales;         // x by columns, as above
    void* dx;                                  // [m, k], or NULL
    float* part;                               // [workgroups, n, k], or NULL
};

template <typename T>
__global__ __launch_bounds__(256, 2) void k_thin_backward(const ThinBackward d) {
    __shared__ __align__(16) uint8_t weight[kEdge * kEdge], codes[kEdge * kEdge], turned[kEdge * kEdge], xs[kEdge * kEdge];
    __shared__ uint32_t most[4][kEdge];
    __shared__ uint8_t scales[kEdge], col_scales[kEdge], x_scales[kEdge];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n0 = (wave >> 1) * 64, k0 = (wave & 1) * 64;
    uint32_t sw = 0;
    if (d.dx) {
        CodesTile w;
        w.load(d.w_codes, kEdge, d.k);
        w.to(weight);
        sw = *d.w_scale;
    }
    f32x16 acc[2][2];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[i >> 1][i & 1][e] = 0.0f;
    __syncthreads();
    for (uint32_t t = blockIdx.x; t < d.tiles; t += gridDim.x) {
        const uint64_t r0 = (uint64_t)t * kEdge;
        Tile<T> g;
        CodesTile x;
        uint8_t sx = 0;
        g.load((const T*)d.dy, d.lddy, r0, d.m, d.n);
        if (d.part) {
            x.load(d.x_codes + (uint64_t)t * kEdge, (uint64_t)d.tiles * kEdge, d.k);
            if (threadIdx.x < d.k) sx = d.x_scales[(uint64_t)t * d.k + threadIdx.x];
        }
        if (d.part) g.columns_to(most);
        __syncthreads();      // also: everyone is done with the last tile
        if (d.dx) {
            g.scale_rows();
            g.row_codes_to(codes, scales);
            __builtin_amdgcn_s_waitcnt(0xc07f);
            __builtin_amdgcn_wave_barrier();
        }
        if (d.part) {
            g.scale_columns(most);
            g.column_codes_to(turned);
            if ((threadIdx.x >> 4) == 0) {
#pragma unroll
                for (int c = 0; c < 8; ++c) col_scales[8 * threadIdx.x + c] = (uint8_t)g.cols[c];
            }
            x.to(xs);
            if (threadIdx.x < kEdge) x_scales[threadIdx.x] = sx;
            __syncthreads();
        }
        if (d.dx) rows_product<T>(codes, scales, weight, sw, (T*)d.dx, r0, d.m, d.k);
        if (d.part) {
#pragma unroll 1
            for (int half = 0; half < 2; ++half)      // (unrolled, their fragments would not fit beside the sums: two workgroups share a CU's registers)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int rn = n0 + 32 * i + (lane & 31);
                    if (n0 + 32 * i >= (int)d.n) break;
                    const i32x8 a = fragment(turned, rn, half, lane);
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const int rk = k0 + 32 * k + (lane & 31);
                        if (k0 + 32 * k >= (int)d.k) break;
                        acc[i][k] = multiply_half<true>(a, fragment(xs, rk, half, lane), acc[i][k], col_scales[rn], x_scales[rk]);
                    }
                }
        }
    }
    if (!d.part) return;
    float* part = d.part + (uint64_t)blockIdx.x * d.n * d.k;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const uint32_t col = k0 + 32 * k + (lane & 31);
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const uint32_t row = n0 + 32 * i + (e >> 2) * 8 + (lane >> 5) * 4 + (e & 3);
                if (row < d.n && col < d.k) part[row * d.k + col] = acc[i][k][e];
            }
        }
}

// Workgroups of a launch: three (forward) or two (backward) fit a CU's LDS.
static uint32_t groups_of(uint32_t tiles, uint32_t per_cu) { return tiles < 256 * per_cu ? tiles : 256 * per_cu; }

static int thin_error(const char* what, uint64_t m, uint64_t n, uint64_t k, uint32_t dtype) {
    if (n == 0 || k == 0 || n > kEdge || k > kEdge) return gf_set_error(GF_ERR_INVALID, "%s: 1 to 128 values on either side", what);
    if (m == 0 || m >> 31) return gf_set_error(GF_ERR_INVALID, "%s: rows out of range", what);
    if (dtype > F16) return gf_set_error(GF_ERR_INVALID, "%s: unknown dtype %u", what, dtype);
    return GF_OK;
}

int thin_forward(const gf_fp8_thin_t& d, const ThinWeight* w, void* stream) {
    if (const int rc = thin_error("gf_fp8_thin", d.m, d.n, d.k, d.dtype)) return rc;
    if (!d.x || (w ? !w->w || (!w->col_codes) != (!w->scale) : !d.codes || !d.scale) || !d.y || (!d.col_codes) != (!d.col_scales))
        return gf_set_error(GF_ERR_INVALID, "gf_fp8_thin: null pointer");
    if ((uintptr_t)(w ? w->col_codes : d.codes) % 16 || (uintptr_t)d.col_codes % 16) return gf_set_error(GF_ERR_INVALID, "gf_fp8_thin: codes must start at a multiple of 16 bytes");
    if (d.ldx < d.k || (w && w->ldw < d.k)) return gf_set_error(GF_ERR_INVALID, "gf_fp8_thin: ldx < k");
    if (w && w->dtype > F16) return gf_set_error(GF_ERR_INVALID, "gf_fp8_thin: unknown dtype %u", w->dtype);
    const uint32_t tiles = (uint32_t)((d.m + kEdge - 1) / kEdge), grid = groups_of(tiles, 3);
    const ThinForward a = {d.x, d.ldx, d.m, (uint32_t)d.n, (uint32_t)d.k, tiles, d.codes, d.scale, d.y, d.col_codes, d.col_scales, w ? *w : ThinWeight{}};
    const hipStream_t s = gf_stream(stream);
    if (d.dtype == F32) k_thin_forward<float><<<grid, 256, 0, s>>>(a);
    else if (d.dtype == BF16) k_thin_forward<__bf16><<<grid, 256, 0, s>>>(a);
    else k_thin_forward<_Float16><<<grid, 256, 0, s>>>(a);
    return gf_check_launch("gf_fp8_thin");
}

}  // namespace gf

using namespace gf;

GF_EXPORT int gf_fp8_thin(const gf_fp8_thin_t* d, void* stream) {
    if (!d) return gf_set_error(GF_ERR_INVALID, "gf_fp8_thin: null descriptor");
    return thin_forward(*d, nullptr, stream);
}

GF_EXPORT uint64_t gf_fp8_thin_workspace_bytes(uint64_t m, uint64_t n, uint64_t k) {
    return m >> 31 || n > kEdge || k > kEdge ? 0 : 4ull * groups_of((uint32_t)((m + kEdge - 1) / kEdge), 2) * n * k;
}

GF_EXPORT int gf_fp8_thin_backward(const gf_fp8_thin_backward_t* d, void* stream) {
    if (!d) return gf_set_error(GF_ERR_INVALID, "gf_fp8_thin_backward: null descriptor");
    if (const int rc = thin_error("gf_fp8_thin_backward", d->m, d->n, d->k, d->dtype)) return rc;
    if (!d->dx && !d->dw) return GF_OK;
    if (!d->dy || (d->dx && (!d->codes || !d->scale)) || (d->dw && (!d->col_codes || !d->col_scales || !d->workspace)))
        return gf_set_error(GF_ERR_INVALID, "gf_fp8_thin_backward: null pointer");
    if (d->w_dtype > F16) return gf_set_error(GF_ERR_INVALID, "gf_fp8_thin_backward: unknown dtype %u", d->w_dtype);
    if ((uintptr_t)d->codes % 16 || (uintptr_t)d->col_codes % 16) return gf_set_error(GF_ERR_INVALID, "gf_fp8_thin_backward: codes must start at a multiple of 16 bytes");
    if (d->lddy < d->n) return gf_set_error(GF_ERR_INVALID, "gf_fp8_thin_backward: lddy < n");
    const uint32_t tiles = (uint32_t)((d->m + kEdge - 1) / kEdge), grid = groups_of(tiles, 2);
    const ThinBackward a = {d->dy, d->lddy, d->m, (uint32_t)d->n, (uint32_t)d->k, tiles, d->codes, d->scale, d->col_codes, d->col_scales, d->dx, d->dw ? (float*)d->workspace : nullptr};
    const hipStream_t s = gf_stream(stream);
    if (d->dtype == F32) k_thin_backward<float><<<grid, 256, 0, s>>>(a);
    else if (d->dtype == BF16) k_thin_backward<__bf16><<<grid, 256, 0, s>>>(a);
    else k_thin_backward<_Float16><<<grid, 256, 0, s>>>(a);
    if (d->dw) {
        const float* part = (const float*)d->workspace;
        if (d->w_dtype == F32) launch_join<float>(part, grid, d->n * d->k, (float*)d->dw, s);
        else if (d->w_dtype == BF16) launch_join<__bf16>(part, grid, d->n * d->k, (__bf16*)d->dw, s);
        else launch_join<_Float16>(part, grid, d->n * d->k, (_Float16*)d->dw, s);
    }
    return gf_check_launch("gf_fp8_thin_backward");
}
