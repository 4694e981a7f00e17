// gf_fp8_matmul and gf_fp8_rows: products of block-scaled 8-bit values on the scaled matrix instructions.
//
// A block of 128 has one power-of-two scale, which is what v_mfma_scale_* take (as a byte per lane, for each 32 values): the products of all blocks
// are added up in the accumulator itself, with no rescaling between them.  Since a block's 128 values share their scale, the order in which
// they reach a lane does not matter as long as both operands have the same.
#include "../common.hpp"
#include "fp8.hpp"
#include "fp8_calls.hpp"
#include "fp8_join.hpp"
#include "geneface_train_hip.h"
#include <utility>

namespace gf {

struct Operand {
    const uint8_t* codes;
    const uint8_t* scales;
    uint64_t pitch, stride_row, stride_block;      // pitch > 0: scales by row; 0: by tile
    __device__ __forceinline__ uint64_t step() const { return pitch ? pitch : stride_block; }
    __device__ __forceinline__ uint64_t at(uint64_t row) const { return pitch ? row : (row >> 7) * stride_row; }
};

struct MatmulArgs {
    Operand a, b;
    uint32_t m, n, blocks, per_split;      // blocks of 128, and how many of them each split adds up
    uint32_t tiles_m, tiles_n;
    void* out;                             // [m, n], or with several splits float [splits, m, n]
};

typedef __attribute__((address_space(3))) void lds_t;

#define GF_FENCE __builtin_amdgcn_sched_barrier(0)      // the scheduler moves nothing across

// An array in LDS of its own for each TAG: the compiler then knows that a load into one is not what a read of another waits for.
template <int BYTES, int TAG>
__device__ __forceinline__ uint8_t* lds_array() {
    __shared__ __align__(16) uint8_t bytes[BYTES];
    return bytes;
}

template <int N> using Const = std::integral_constant<int, N>;
template <int N, typename F, int... I>
__device__ __forceinline__ void each(F f, std::integer_sequence<int, I...>) { (f(Const<I>{}), ...); }
template <int N, typename F>
__device__ __forceinline__ void each(F f) { each<N>(f, std::make_integer_sequence<int, N>{}); }      // f(Const<0>), f(Const<1>), ..

// s_waitcnt: at most vm loads and lgkm LDS reads still under way
constexpr int waitcnt(int vm, int lgkm) { return (vm & 15) | 7 << 4 | lgkm << 8 | (vm >> 4) << 14; }

// A workgroup of 2 x 2 waves makes a tile of 64 TM x 64 TN of the product, a wave TM x TN tiles of 32 x 32.
//
// Blocks of codes come straight from memory to LDS, STAGES of them under way (the buffer descriptor ends with the tile's last row: rows behind it
// read as zero).  Row r is 128 bytes, its 16-byte piece c at place c ^ ((r >> 1) & 7), so that the same piece of any 16 consecutive rows lies on
// different banks.  A step multiplies one block in two halves of 64, and the fragments of a half are read from LDS while the half before it is
// multiplied, so the matrix unit waits for nothing but the one barrier of a step: behind it everyone has read the block, whose place the block
// STAGES further on is then loaded into.  With one wave on each SIMD there is nobody else to fill a gap, hence the interleaving by hand (weave): an
// LDS read or two and a load beside each matrix instruction.  (Two waves on each, with 128 x 64 each of a tile of 256, take as long: 104 us for 4096 x 4096 x
// 8192, 233 against 223 for 8192 x 8192 x 4096.)
//
// Measured: m 8192, n 8192, k 4096 to bfloat16 in 222-250 us (2 200-2 480 TFLOP/s; the library's tensor-scaled product 226), 4096 each 58-65; to float32 (EXACT)
// 4096 each 106-116 us (1 180-1 300 TFLOP/s).  The matrix units are busy for two thirds of a wave's life; the rest is the barrier of a step, first loads and last stores.
//
// EXACT (kExact<T>): codes are widened to bfloat16 on the way out of LDS and added up on its instruction, in 32 bits.  8192 x 8192 x 4096 to binary16 takes
// 403 us that way, 222 on the 8-bit instruction; 333 rows, 8192 -> 2048 29.5 for 22.4; a few rows 5.8 for 5.4.
template <typename T, bool EXACT, int TM, int TN, int STAGES>
__device__ __forceinline__ void matmul_tile(const MatmulArgs& d, const uint32_t block, const uint32_t split) {
    constexpr int BM = 64 * TM, BN = 64 * TN, LA = BM / 32, LB = BN / 32;      // 32 rows of 128 bytes a load of the workgroup
    auto stage_a = [](auto j) __attribute__((always_inline)) { return lds_array<BM * 128, decltype(j)::value>(); };
    auto stage_b = [](auto j) __attribute__((always_inline)) { return lds_array<BN * 128, 16 + decltype(j)::value>(); };
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wr = wave >> 1, wc = wave & 1;

    // Workgroups go to the 8 XCDs in turn.  Each XCD gets a contiguous range of tiles, walked in bands of 8 rows of tiles, so that what its
    // workgroups read at one time is a few rows and columns of tiles, in its own L2.
    uint32_t tile_m, tile_n;
    {
        const uint32_t total = d.tiles_m * d.tiles_n, xcd = block & 7, full = total / 8, rest = total % 8;
        const uint32_t t = xcd * full + min(xcd, rest) + (block >> 3), band = t / (8 * d.tiles_n), in = t % (8 * d.tiles_n);
        const uint32_t high = min(8u, d.tiles_m - band * 8);
        tile_m = __builtin_amdgcn_readfirstlane(band * 8 + in % high);
        tile_n = __builtin_amdgcn_readfirstlane(in / high);
    }
    const uint64_t m0 = (uint64_t)tile_m * BM, n0 = (uint64_t)tile_n * BN;
    const uint32_t kb0 = split * d.per_split, nb = min(d.blocks, kb0 + d.per_split) - kb0, width = d.blocks * 128;

    auto buffer = [&](const uint8_t* codes, uint64_t row0, uint32_t rows, uint32_t tile) {
        const uint64_t have = (uint64_t)min(tile, rows - (uint32_t)row0) * width - (uint64_t)kb0 * 128;
        return __builtin_amdgcn_make_buffer_rsrc((void*)(codes + row0 * width + (uint64_t)kb0 * 128), 0, (int)(uint32_t)have, 0x00027000);
    };
    const auto ra = buffer(d.a.codes, m0, d.m, BM), rb = buffer(d.b.codes, n0, d.n, BN);
    const uint32_t r8 = wave * 8 + (lane >> 3);      // the row of the first load; the others' differ by multiples of 32 and swizzle alike
    const uint32_t off = r8 * width + (((lane & 7) ^ ((r8 >> 1) & 7)) << 4);
    auto load = [&](uint8_t* A, uint8_t* B, uint32_t kb) __attribute__((always_inline)) {
        // The row goes into the offset that the descriptor's bound is held against, the block into the one that is not: a row behind the last is out
        // of bounds by itself.  Behind the last block: that one again, for nobody.
        const uint32_t at = min(kb, nb - 1) * 128;
#pragma unroll
        for (int i = 0; i < LA; ++i) __builtin_amdgcn_raw_ptr_buffer_load_lds(ra, (lds_t*)(A + (i * 4 + wave) * 1024), 16, off + i * 32 * width, at, 0, 0);
#pragma unroll
        for (int i = 0; i < LB; ++i) __builtin_amdgcn_raw_ptr_buffer_load_lds(rb, (lds_t*)(B + (i * 4 + wave) * 1024), 16, off + i * 32 * width, at, 0, 0);
    };

    // Scales: a byte for each row of a fragment, read at least STAGES - 1 steps before it is used.
    const uint64_t step_a = d.a.step(), step_b = d.b.step();
    const uint8_t *sa = d.a.scales + d.a.at(m0) + kb0 * step_a, *sb = d.b.scales + d.b.at(n0) + kb0 * step_b;
    uint32_t ca[TM], cb[TN];
#pragma unroll
    for (int i = 0; i < TM; ++i) ca[i] = (uint32_t)d.a.at(min((uint32_t)((wr * TM + i) * 32 + (lane & 31)), (uint32_t)(d.m - 1 - m0)));
#pragma unroll
    for (int i = 0; i < TN; ++i) cb[i] = (uint32_t)d.b.at(min((uint32_t)((wc * TN + i) * 32 + (lane & 31)), (uint32_t)(d.n - 1 - n0)));
    int xa[STAGES][TM], xb[STAGES][TN], nxa[STAGES][TM], nxb[STAGES][TN];      // of the STAGES blocks at hand, and of the next
    auto read_scales = [&](uint32_t kb) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < STAGES; ++j) {
            const uint32_t at = min(kb + j, nb - 1);
            const uint8_t *u = sa + at * step_a, *v = sb + at * step_b;
#pragma unroll
            for (int i = 0; i < TM; ++i) nxa[j][i] = u[ca[i]];
#pragma unroll
            for (int i = 0; i < TN; ++i) nxb[j][i] = v[cb[i]];
        }
    };
    auto take_scales = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < STAGES; ++j) {
#pragma unroll
            for (int i = 0; i < TM; ++i) xa[j][i] = nxa[j][i];
#pragma unroll
            for (int i = 0; i < TN; ++i) xb[j][i] = nxb[j][i];
        }
        GF_FENCE;
    };

    // Fragments: lane l holds row l % 32 and 32 of the half's 64 codes, the pieces 4 half + 2 (l / 32) and the next.
    uint32_t pa[4], pb[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const int piece = (((q >> 1) * 4 + (lane >> 5) * 2 + (q & 1)) ^ ((lane >> 1) & 7)) << 4;
        pa[q] = (wr * TM * 32 + (lane & 31)) * 128 + piece;
        pb[q] = (wc * TN * 32 + (lane & 31)) * 128 + piece;
    }
    auto fragment = [&](const uint8_t* base, uint32_t lo, uint32_t hi) __attribute__((always_inline)) {
        const i32x4 x = *reinterpret_cast<const i32x4*>(base + lo), y = *reinterpret_cast<const i32x4*>(base + hi);
        return __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
    };
    auto read = [&](const uint8_t* A, const uint8_t* B, int half, i32x8* fa, i32x8* fb) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < TN; ++i) fb[i] = fragment(B + i * 4096, pb[half * 2], pb[half * 2 + 1]);
#pragma unroll
        for (int i = 0; i < TM; ++i) fa[i] = fragment(A + i * 4096, pa[half * 2], pa[half * 2 + 1]);
    };

    f32x16 acc[TM][TN];      // transposed: b's rows in the registers, a's in the lanes, so that a lane holds neighbours of a row of the result
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int k = 0; k < TN; ++k)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][k][e] = 0.0f;
    auto multiply = [&](const i32x8* fa, const i32x8* fb, const int* p, const int* q) __attribute__((always_inline)) {
        if constexpr (EXACT) {
            bf16x8 wb[TN][4];
#pragma unroll
            for (int k = 0; k < TN; ++k)
#pragma unroll
                for (int s = 0; s < 4; ++s) wb[k][s] = widen8(fb[k][2 * s], fb[k][2 * s + 1], scale_value(q[k]));
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int s = 0; s < 4; ++s) {
                    const bf16x8 wa = widen8(fa[i][2 * s], fa[i][2 * s + 1], scale_value(p[i]));
#pragma unroll
                    for (int k = 0; k < TN; ++k) acc[i][k] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(wb[k][s], wa, acc[i][k], 0, 0, 0);
                }
        } else {
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int k = 0; k < TN; ++k)
                    acc[i][k] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fb[k], fa[i], acc[i][k], 0, 0, 0, q[k], 0, p[i]);
        }
    };
    auto weave = [&](auto loads) __attribute__((always_inline)) {
        constexpr int MF = TM * TN * (EXACT ? 4 : 1), DS = 2 * (TM + TN), LD = LA + LB;
        // the reads beside the first half of the matrix instructions, so that the last of them is back when those are through (512 x 4096 x 4096: 13.8 -> 13.4 us)
        constexpr int per_ds = 2 * DS > MF ? 2 * DS / MF : 1, per_ld = LD > MF ? LD / MF : 1;
#pragma unroll
        for (int i = 0; i < MF; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);                                          // a matrix instruction,
            if constexpr (decltype(loads)::value) __builtin_amdgcn_sched_group_barrier(0x010, per_ld, 0);    // a load,
            __builtin_amdgcn_sched_group_barrier(0x100, per_ds, 0);                                     // a read from LDS
        }
    };

    i32x8 fa0[TM], fb0[TN], fa1[TM], fb1[TN];
    auto step = [&](auto j, uint32_t kb) __attribute__((always_inline)) {
        constexpr int J = decltype(j)::value;
        uint8_t *A = stage_a(j), *B = stage_b(j);
        const uint8_t *A2 = stage_a(Const<(J + 1) % STAGES>{}), *B2 = stage_b(Const<(J + 1) % STAGES>{});
        __builtin_amdgcn_s_waitcnt(waitcnt(63, 0));      // the first half's fragments
        GF_FENCE;
        read(A, B, 1, fa1, fb1);
        multiply(fa0, fb0, xa[J], xb[J]);
        weave(Const<0>{});
        GF_FENCE;
        // The next block is there and this one is read.  STAGES - 2 blocks were asked for behind the next one; scales that were asked for in between
        // only make the wait a longer one.
        __builtin_amdgcn_s_waitcnt(waitcnt((STAGES - 2) * (LA + LB), 0));
        __builtin_amdgcn_s_barrier();
        GF_FENCE;
        if constexpr (J == 0) {
            read_scales(kb + STAGES);
            GF_FENCE;
        }
        load(A, B, kb + STAGES);
        read(A2, B2, 0, fa0, fb0);
        multiply(fa1, fb1, xa[J], xb[J]);
        weave(Const<1>{});
        GF_FENCE;
    };

    read_scales(0);
    GF_FENCE;
    each<STAGES>([&](auto j) __attribute__((always_inline)) { load(stage_a(j), stage_b(j), decltype(j)::value); });
    __builtin_amdgcn_s_waitcnt(waitcnt((STAGES - 1) * (LA + LB), 0));
    __builtin_amdgcn_s_barrier();
    GF_FENCE;
    read(stage_a(Const<0>{}), stage_b(Const<0>{}), 0, fa0, fb0);
    uint32_t kb = 0;
    for (; kb + STAGES <= nb; kb += STAGES) {
        take_scales();
        each<STAGES>([&](auto j) __attribute__((always_inline)) { step(j, kb + decltype(j)::value); });
    }
    if (kb < nb) {
        take_scales();
        each<STAGES - 1>([&](auto j) __attribute__((always_inline)) {
            if (kb + decltype(j)::value < nb) step(j, kb + decltype(j)::value);
        });
    }
    __builtin_amdgcn_s_waitcnt(waitcnt(0, 0));      // no load is under way and nobody reads any more: LDS is free
    __builtin_amdgcn_s_barrier();

    // 32 rows of the wave's part at a time through LDS, so that a row leaves in pieces of 16 bytes.
    constexpr int COLS = 32 * TN, PITCH = COLS * (int)sizeof(T) + 16, EACH = 16 / (int)sizeof(T), PIECES = COLS / EACH;
    static_assert(32 * PITCH <= BN * 128 && 32 * PITCH <= BM * 128, "staging");
    uint8_t* mine = wave == 0 ? stage_a(Const<0>{}) : wave == 1 ? stage_a(Const<1>{}) : wave == 2 ? stage_b(Const<0>{}) : stage_b(Const<1>{});
    T* out = (T*)d.out + (uint64_t)split * d.m * d.n;
#pragma unroll
    for (int i = 0; i < TM; ++i) {
#pragma unroll
        for (int k = 0; k < TN; ++k)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const float v[4] = {acc[i][k][4 * g], acc[i][k][4 * g + 1], acc[i][k][4 * g + 2], acc[i][k][4 * g + 3]};
                store4((T*)(mine + (lane & 31) * PITCH) + k * 32 + g * 8 + (lane >> 5) * 4, v);
            }
        __builtin_amdgcn_s_waitcnt(waitcnt(63, 0));      // the wave's own stores (it alone reads them)
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int q = 0; q < 32 * PIECES / 64; ++q) {
            const int r = (q * 64 + lane) / PIECES, c = (q * 64 + lane) % PIECES;
            const uint64_t row = m0 + (wr * TM + i) * 32 + r, col = n0 + wc * COLS + c * EACH;
            const i32x4 v = *reinterpret_cast<const i32x4*>(mine + r * PITCH + c * 16);
            if (row >= d.m || col >= d.n) continue;
            T* to = out + row * d.n + col;
            if (col + EACH <= d.n) {
                typedef int piece __attribute__((ext_vector_type(4), aligned(2)));
                *reinterpret_cast<piece*>(to) = v;
            } else {
                const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
                for (int k = 0; k < EACH; ++k) if (col + k < d.n) to[k] = e[k];
            }
        }
        __builtin_amdgcn_wave_barrier();
    }
}

template <typename T, bool EXACT, int TM, int TN, int STAGES>
__global__ __launch_bounds__(256) void k_matmul(const MatmulArgs d) { matmul_tile<T, EXACT, TM, TN, STAGES>(d, blockIdx.x, blockIdx.y); }

// Two products of small tiles and sums that are not split; the second one's begin at a multiple of 8, for the XCDs.
template <typename A, typename B>
__global__ __launch_bounds__(256) void k_matmul_two(const MatmulArgs a, const MatmulArgs b) {
#ifdef __HIP_DEVICE_COMPILE__      // (the host's pass finds no candidate for these calls, and has no use for them)
    const uint32_t tiles = a.tiles_m * a.tiles_n, first = (tiles + 7) & ~7u;
    if (blockIdx.x >= first) matmul_tile<B, kExact<B>, 1, 1, 4>(b, blockIdx.x - first, 0);
    else if (blockIdx.x < tiles) matmul_tile<A, kExact<A>, 1, 1, 4>(a, blockIdx.x, 0);
#endif
}

// ---- a few rows ----------------------------------------------------------------------------------------------------------------------------
// The weight's bytes bound it, and at the sizes it is called with, how many of them are under way at once and how long the way to the first product is.
// A wave takes 16 rows of the weight (one row of codes is 128 bytes a block: whole cache lines, straight into registers) and every 16th block, two
// blocks ahead; 16 waves of a workgroup share the rows and add up through LDS.  While the first blocks of the weight are under way the workgroup
// brings x to 8 bits in LDS, 16 lanes to a block of a row: 8 values a lane, as few as they can be shared out.  Measured: one row, n = k = 4096, 4.7-5.3 us
// with its launch (3.2-3.6 TB/s); 7 rows, n 1111, k 2050 5.3, which is what the steps one behind another take whatever the sizes.
constexpr int kRowWaves = 16, kRowBlocks = 2, kRowBytes = 128 * 1024;      // codes of x at a time

template <typename T>
__global__ __launch_bounds__(64 * kRowWaves) void k_rows(const gf_fp8_rows_t d) {
    __shared__ f32x4 part[kRowWaves][64];
    __shared__ __align__(16) uint8_t codes[kRowBytes + 16 * 16];
    __shared__ uint8_t bytes[kRowBytes / 128];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, q = lane >> 4;
    const uint64_t n0 = ((uint64_t)blockIdx.y * gridDim.x + blockIdx.x) * 16;
    if (n0 >= d.n) return;
    const uint32_t blocks = (uint32_t)((d.k + 127) / 128), rows = (uint32_t)d.m;
    const uint64_t row = min(n0 + r, d.n - 1);
    const uint8_t* w = d.codes + row * blocks * 128 + q * 32;
    const uint8_t* ws = d.scales + (row >> 7) * blocks;
    const uint32_t room = kRowBytes / 128 / rows;                          // blocks of x that fit
    f32x4 acc = {0, 0, 0, 0};
    for (uint32_t c0 = 0; c0 < blocks; c0 += room) {
        const uint32_t here = min(room, blocks - c0), pitch = here * 128 + 16;      // 16: the rows' same piece on different banks
        i32x4 lo[kRowBlocks], hi[kRowBlocks];
        int sw[kRowBlocks];
        auto ahead = [&](uint32_t b0) __attribute__((always_inline)) {
#pragma unroll
            for (int u = 0; u < kRowBlocks; ++u) {
                const uint64_t b = c0 + min(b0 + u * kRowWaves, here - 1);          // behind the last block: that one again, for nobody
                lo[u] = *reinterpret_cast<const i32x4*>(w + b * 128);
                hi[u] = *reinterpret_cast<const i32x4*>(w + b * 128 + 16);
                sw[u] = ws[b];
            }
        };
        ahead(wave);
        if (c0) __syncthreads();                                            // everyone is done with the last codes
        for (uint32_t t = threadIdx.x >> 4; t < rows * here; t += 4 * kRowWaves) {
            const uint32_t xr = t / here, b = t % here;
            const uint64_t k = (uint64_t)(c0 + b) * 128 + 8 * r;
            const int left = k < d.k ? (int)min((uint64_t)8, d.k - k) : 0;
            Eight<T> v;
            v.load((const T*)d.x + xr * d.ldx + (left ? k : 0), left);
            const uint32_t byte = scale_byte(row_max_u32(v.amax()));
            *reinterpret_cast<uint2*>(codes + xr * pitch + b * 128 + 8 * r) = coded(v.encode(scale_value(byte)), byte);
            if (r == 0) bytes[xr * here + b] = (uint8_t)byte;
        }
        __syncthreads();
        const uint32_t xr = min((uint32_t)r, rows - 1);                     // rows behind the last: its results again, for nobody
        for (uint32_t b0 = wave; b0 < here; b0 += kRowWaves * kRowBlocks) {
            if (b0 != (uint32_t)wave) ahead(b0);
#pragma unroll
            for (int u = 0; u < kRowBlocks; ++u) {
                const uint32_t b = b0 + u * kRowWaves;
                if (b >= here) break;
                const i32x4 xl = *reinterpret_cast<const i32x4*>(codes + xr * pitch + b * 128 + q * 32), xh = *reinterpret_cast<const i32x4*>(codes + xr * pitch + b * 128 + q * 32 + 16);
                const uint32_t sx = bytes[xr * here + b];
                if constexpr (kExact<T>) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const i32x4 pw = i < 2 ? lo[u] : hi[u], px = i < 2 ? xl : xh;
                        acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen8(pw[2 * (i & 1)], pw[2 * (i & 1) + 1], scale_value(sw[u])),
                                                                      widen8(px[2 * (i & 1)], px[2 * (i & 1) + 1], scale_value(sx)), acc, 0, 0, 0);
                    }
                } else {
                    acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(__builtin_shufflevector(lo[u], hi[u], 0, 1, 2, 3, 4, 5, 6, 7),
                                                                           __builtin_shufflevector(xl, xh, 0, 1, 2, 3, 4, 5, 6, 7), acc, 0, 0, 0, sw[u], 0, (int)sx);
                }
            }
        }
    }
    part[wave][lane] = acc;
    __syncthreads();
    if (threadIdx.x >= 256) return;
    const int e = threadIdx.x & 3, l = threadIdx.x >> 2;      // part[.][l][e]: row l % 16 of x, row 4 (l / 16) + e of the weight
    float s = 0;
#pragma unroll
    for (int k = 0; k < kRowWaves; ++k) s += part[k][l][e];
    const uint64_t m = l & 15, n = n0 + 4 * (l >> 4) + e;
    if (m < d.m && n < d.n) ((T*)d.out)[m * d.n + n] = (T)s;
}

// The tile and how many ways the sum over K is split: the choice with the least time of its longest CU, in units of 0.11 us.  A workgroup's step over
// one block takes 2 of them for a tile of 64 x 64, 3 for 128 x 64, 5 for 128 x 128 and 17 for 256 x 256 (about 1.7 times that each for EXACT
// ones): large tiles read less per product, small ones give every CU one (the three small tiles all read some 32 bytes a clock and CU, which is what
// bounds them; fragments straight from memory to registers, without LDS, read half of that).  A split's parts cost 45, their launch among it, and the way to memory and
// back.  Measured, us, 64 x 64 / 128 x 64 / 128 x 128 / 256 x 256: m 333, n 2048, k 8192 16.9 / 21 / 22 / -, split in two 128 x 64 18.3, in four
// 128 x 128 18.1; 512, 4096, 4096 16.6 / 13.7 / 17.1 / -; 2048 each 17.7 / 15.9 / 13.8 / 25.5; 4096 each 111 / 103 / 70 / 62.
struct Plan { uint32_t edge_m, edge_n, tiles_m, tiles_n, splits, per_split; };

static Plan plan_of(uint64_t m, uint64_t n, uint64_t blocks) {
    struct Kind { uint32_t edge_m, edge_n, units; };
    constexpr Kind kinds[] = {{64, 64, 2}, {128, 64, 3}, {128, 128, 5}, {256, 256, 17}};
    constexpr uint64_t kCus = 256;
    Plan best = {};
    double least = 0;
    for (const Kind& k : kinds) {
        Plan p = {k.edge_m, k.edge_n, (uint32_t)((m + k.edge_m - 1) / k.edge_m), (uint32_t)((n + k.edge_n - 1) / k.edge_n), 1, (uint32_t)blocks};
        const uint64_t t = (uint64_t)p.tiles_m * p.tiles_n;
        for (uint64_t want = 1;; want = kCus / t < blocks / 4 ? kCus / t : blocks / 4) {      // at least four blocks in each
            p.per_split = (uint32_t)((blocks + want - 1) / want);
            p.splits = (uint32_t)((blocks + p.per_split - 1) / p.per_split);                  // none of them empty
            const double cost = (double)((t * p.splits + kCus - 1) / kCus) * p.per_split * k.units + (p.splits > 1 ? 45 + 1.8e-5 * (double)(m * n) * p.splits : 0);
            if (!best.edge_m || cost < least) { best = p; least = cost; }
            if (want > 1 || kCus / t < 2 || blocks < 8) break;
        }
    }
    return best;
}

template <typename T, bool EXACT>
static void launch_tiles(const MatmulArgs& a, const Plan& p, hipStream_t s) {
    const dim3 grid(p.tiles_m * p.tiles_n, p.splits);
    if (p.edge_m == 256) k_matmul<T, EXACT, 4, 4, 2><<<grid, 256, 0, s>>>(a);
    else if (p.edge_n == 64 && p.edge_m == 64) k_matmul<T, EXACT, 1, 1, 4><<<grid, 256, 0, s>>>(a);
    else if (p.edge_n == 64) k_matmul<T, EXACT, 2, 1, 4><<<grid, 256, 0, s>>>(a);
    // four blocks under way where a CU has one workgroup (2048 each: 13.8 us, with two blocks 15.0), two where it has more (2500 each: 22.0, with four 26.5)
    else if (grid.x * grid.y <= 256) k_matmul<T, EXACT, 2, 2, 4><<<grid, 256, 0, s>>>(a);
    else k_matmul<T, EXACT, 2, 2, 2><<<grid, 256, 0, s>>>(a);
}

template <typename T>
static void launch_matmul(MatmulArgs a, const Plan& p, void* workspace, hipStream_t s) {
    constexpr bool exact = kExact<T>;
    if (p.splits == 1) { launch_tiles<T, exact>(a, p, s); return; }
    T* out = (T*)a.out;
    a.out = workspace;
    launch_tiles<float, exact>(a, p, s);
    const uint64_t count = (uint64_t)a.m * a.n;
    launch_join<T>((const float*)workspace, p.splits, count, out, s);
}

static const char* operand_error(const gf_fp8_operand_t& o, uint64_t rows) {
    if (!o.codes || !o.scales) return "null operand";
    if ((uintptr_t)o.codes % 16) return "codes must start at a multiple of 16 bytes";
    if (o.pitch && o.pitch < rows) return "scale pitch smaller than the rows";
    if (!o.pitch && o.stride_row >> 24) return "scale stride too large";
    return nullptr;
}

static bool too_large(uint64_t m, uint64_t n, uint64_t blocks) {      // blocks: a tile's rows have to lie within 4 GB; tiles: a launch's work-items below 2^32
    return m >> 31 || n >> 31 || blocks > 65535 || ((m + 127) / 128) * ((n + 127) / 128) >> 22;
}

static int matmul_error(const gf_fp8_matmul_t& d) {
    if (!d.out) return gf_set_error(GF_ERR_INVALID, "gf_fp8_matmul: null output");
    if (d.dtype > F16) return gf_set_error(GF_ERR_INVALID, "gf_fp8_matmul: unknown dtype %u", d.dtype);
    if (d.blocks == 0) return gf_set_error(GF_ERR_INVALID, "gf_fp8_matmul: no blocks to add up");
    if (const char* e = operand_error(d.a, d.m)) return gf_set_error(GF_ERR_INVALID, "gf_fp8_matmul: a: %s", e);
    if (const char* e = operand_error(d.b, d.n)) return gf_set_error(GF_ERR_INVALID, "gf_fp8_matmul: b: %s", e);
    if (too_large(d.m, d.n, d.blocks)) return gf_set_error(GF_ERR_INVALID, "gf_fp8_matmul: matrix too large (at most 65535 blocks along the sum)");
    if (plan_of(d.m, d.n, d.blocks).splits > 1 && (!d.workspace || (uintptr_t)d.workspace % 16))
        return gf_set_error(GF_ERR_INVALID, "gf_fp8_matmul: null or unaligned workspace");
    return GF_OK;
}

static MatmulArgs args_of(const gf_fp8_matmul_t& d, const Plan& p) {
    MatmulArgs a;
    a.a = {d.a.codes, d.a.scales, d.a.pitch, d.a.stride_row, d.a.stride_block};
    a.b = {d.b.codes, d.b.scales, d.b.pitch, d.b.stride_row, d.b.stride_block};
    a.m = (uint32_t)d.m; a.n = (uint32_t)d.n; a.blocks = (uint32_t)d.blocks;
    a.per_split = p.per_split; a.tiles_m = p.tiles_m; a.tiles_n = p.tiles_n;
    a.out = d.out;
    return a;
}

// f(T()) with the type that dtype names
template <typename F>
static void with_type(uint32_t dtype, F f) {
    if (dtype == F32) f(float());
    else if (dtype == BF16) f(__bf16());
    else f(_Float16());
}

static void launch(const gf_fp8_matmul_t& d, hipStream_t s) {
    const Plan p = plan_of(d.m, d.n, d.blocks);
    with_type(d.dtype, [&](auto t) { launch_matmul<decltype(t)>(args_of(d, p), p, d.workspace, s); });
}

template <typename A, typename B>
static void launch_matmul_two(const MatmulArgs& a, const MatmulArgs& b, uint32_t grid, hipStream_t s) { k_matmul_two<A, B><<<grid, 256, 0, s>>>(a, b); }

int matmul_two(const gf_fp8_matmul_t& a, const gf_fp8_matmul_t& b, void* stream) {
    if (const int rc = matmul_error(a)) return rc;
    if (const int rc = matmul_error(b)) return rc;
    const hipStream_t s = gf_stream(stream);
    const Plan p = plan_of(a.m, a.n, a.blocks), q = plan_of(b.m, b.n, b.blocks);
    const uint64_t ta = (uint64_t)p.tiles_m * p.tiles_n, tb = (uint64_t)q.tiles_m * q.tiles_n;
    if (p.edge_m == 64 && q.edge_m == 64 && p.splits == 1 && q.splits == 1 && ta + tb < 1u << 22) {
        with_type(a.dtype, [&](auto x) {
            with_type(b.dtype, [&](auto y) { launch_matmul_two<decltype(x), decltype(y)>(args_of(a, p), args_of(b, q), (uint32_t)((ta + 7) / 8 * 8 + tb), s); });
        });
    } else {
        launch(a, s);
        launch(b, s);      // (their parts may lie in one workspace: the first product's are read before the second's are written)
    }
    return gf_check_launch("gf_fp8_matmul");
}

}  // namespace gf

using namespace gf;

GF_EXPORT uint64_t gf_fp8_matmul_workspace_bytes(uint64_t m, uint64_t n, uint64_t blocks) {
    if (!m || !n || !blocks || too_large(m, n, blocks)) return 0;
    const Plan p = plan_of(m, n, blocks);
    return p.splits > 1 ? 4ull * p.splits * m * n : 0;
}

GF_EXPORT int gf_fp8_matmul(const gf_fp8_matmul_t* d, void* stream) {
    if (!d) return gf_set_error(GF_ERR_INVALID, "gf_fp8_matmul: null descriptor");
    if (d->m == 0 || d->n == 0) return GF_OK;
    if (const int rc = matmul_error(*d)) return rc;
    launch(*d, gf_stream(stream));
    return gf_check_launch("gf_fp8_matmul");
}

GF_EXPORT int gf_fp8_rows(const gf_fp8_rows_t* d, void* stream) {
    if (!d) return gf_set_error(GF_ERR_INVALID, "gf_fp8_rows: null descriptor");
    if (d->m == 0 || d->n == 0) return GF_OK;
    if (!d->x || !d->codes || !d->scales || !d->out) return gf_set_error(GF_ERR_INVALID, "gf_fp8_rows: null pointer");
    if (d->m > 16) return gf_set_error(GF_ERR_INVALID, "gf_fp8_rows: at most 16 rows, got %llu", (unsigned long long)d->m);
    if (d->dtype > F16) return gf_set_error(GF_ERR_INVALID, "gf_fp8_rows: unknown dtype %u", d->dtype);
    if (d->k == 0 || d->ldx < d->k) return gf_set_error(GF_ERR_INVALID, "gf_fp8_rows: ldx < k, or k = 0");
    if (d->k >> 31) return gf_set_error(GF_ERR_INVALID, "gf_fp8_rows: matrix too large");
    if ((uintptr_t)d->codes % 16) return gf_set_error(GF_ERR_INVALID, "gf_fp8_rows: codes must start at a multiple of 16 bytes");
    if ((d->n + 15) / 16 >> 31) return gf_set_error(GF_ERR_INVALID, "gf_fp8_rows: matrix too large");
    const uint32_t groups = (uint32_t)((d->n + 15) / 16), wide = 1u << 20;      // a launch's work-items along x lie below 2^32
    const dim3 grid(groups < wide ? groups : wide, (groups + wide - 1) / wide);
    const hipStream_t s = gf_stream(stream);
    with_type(d->dtype, [&](auto t) { k_rows<decltype(t)><<<grid, 64 * kRowWaves, 0, s>>>(*d); });
    return gf_check_launch("gf_fp8_rows");
}
