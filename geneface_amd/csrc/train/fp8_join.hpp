// The parts of a product whose sum was split, added up.
#pragma once
#include "fp8.hpp"

namespace gf {

// out = the sum of the splits' parts in a fixed order: a wave adds up every WAVES-th of them for 256 values, then the waves' sums are added.  Eight
// loads are under way at a time: the parts of a tall product's weight gradient are hundreds, of few values each, and latency is all they cost
// (512 parts of 128 x 96: 8 us).
template <typename T, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void k_join(const float* part, uint32_t splits, uint64_t count, T* out) {
    __shared__ f32x4 sums[WAVES][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint64_t i = ((uint64_t)blockIdx.x * 64 + lane) * 4;
    const int left = i < count ? (int)min((uint64_t)4, count - i) : 0;
    const float* at = part + (left ? i : 0);
    f32x4 s = {0, 0, 0, 0};
    for (uint32_t k = wave; k < splits; k += 8 * WAVES) {
        float v[8][4];
#pragma unroll
        for (int u = 0; u < 8; ++u) load4_of(at + min(k + u * WAVES, splits - 1) * count, k + u * WAVES < splits ? left : 0, v[u]);
#pragma unroll
        for (int u = 0; u < 8; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[e] += v[u][e];
    }
    sums[wave][lane] = s;
    __syncthreads();
    if (wave) return;
    float r[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
    for (int w = 1; w < WAVES; ++w)
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] += sums[w][lane][e];
    store4_of(out + (left ? i : 0), left, r);
}

template <typename T>
static void launch_join(const float* part, uint32_t splits, uint64_t count, T* out, hipStream_t s) {
    const uint32_t grid = (uint32_t)((count + 255) / 256);
    if (splits > 16) k_join<T, 16><<<grid, 1024, 0, s>>>(part, splits, count, out);
    else k_join<T, 4><<<grid, 256, 0, s>>>(part, splits, count, out);
}

}  // namespace gf
