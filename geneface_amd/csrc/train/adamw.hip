// AdamW over many tensors in one launch (gf_adamw_step) and the global norm of their gradients (gf_grad_norm); declared in
// include/geneface_train_hip.h.
//
// Both read and write each value once and do some twenty operations on it, so memory bounds them.  The tensors' addresses travel in the kernel
// arguments (no table in memory that a replayed graph could find changed): a launch takes as many tensors as 4 KB of arguments hold, and every
// workgroup finds its tensor by one comparison per lane with the first workgroups of all of them.
#include "../common.hpp"
#include "elem.hpp"
#include "geneface_train_hip.h"

namespace gf {

constexpr int kThreads = 256;
constexpr int kTensors = 56;              // per launch: 56 x 64 bytes + first workgroups + scalars < 4096

struct AdamwArgs {
    gf_adamw_tensor_t t[kTensors];
    uint32_t first[kTensors];             // first workgroup of each tensor, 0xffffffff behind the last
    double beta1, beta2, lr, weight_decay, max_norm;
    float eps;
    uint32_t chunk;                       // values per workgroup, a multiple of 1024
    const float* lr_device;
    const float* grad_scale;
    const float* found_inf;
    const float* grad_norm;
    const double* grad_norm_wide;
    uint32_t count_steps;                 // 1: every tensor of the call has one workgroup, which counts its step itself
};
static_assert(sizeof(AdamwArgs) <= 4096, "kernel arguments");

struct StepArgs {
    float* step[496];
    const float* found_inf;
    uint32_t count;
};
static_assert(sizeof(StepArgs) <= 4096, "kernel arguments");

struct Hyper { float shrink, om_beta1, beta2, om_beta2, rate, inv_root, eps, grad; };

__device__ __forceinline__ double pow_int(double b, uint32_t t) {
    double r = 1.0;
    for (; t; t >>= 1, b *= b) if (t & 1) r *= b;
    return r;
}

// Scalars of one tensor in 64 bits, rounded once.  1 - beta^t keeps its digits at small t that way.
__device__ __forceinline__ Hyper hyper_of(const AdamwArgs& a, float t) {
    const double lr = a.lr_device ? (double)*a.lr_device : a.lr;
    const uint32_t ti = (uint32_t)t;
    Hyper h;
    h.shrink = (float)(1.0 - lr * a.weight_decay);
    h.om_beta1 = (float)(1.0 - a.beta1);
    h.beta2 = (float)a.beta2;
    h.om_beta2 = (float)(1.0 - a.beta2);
    h.rate = (float)(lr / (1.0 - pow_int(a.beta1, ti)));
    h.inv_root = (float)(1.0 / sqrt(1.0 - pow_int(a.beta2, ti)));
    h.eps = a.eps;
    double c = a.grad_scale ? 1.0 / (double)*a.grad_scale : 1.0;
    if (a.grad_norm) {
        double norm = *a.grad_norm;
        if (a.grad_norm_wide && (float)*a.grad_norm_wide == *a.grad_norm) norm = *a.grad_norm_wide;      // (the 32-bit one as it was written)
        const double q = a.max_norm / (norm + 1e-6);
        c *= q >= 1.0 ? 1.0 : q;          // a norm that is no number leaves none
    }
    h.grad = (float)c;
    return h;
}

// Every operation on the moments rounds by itself, as a formula written out in 32-bit operations does.  An 8-bit code is a step function of its
// value: with the same roundings the state is the same bit for bit, however long two runs of the formula go side by side.
__device__ __forceinline__ float moment1(const Hyper& h, float m, float g) {
#pragma clang fp contract(off)
    return m + h.om_beta1 * (g - m);
}
__device__ __forceinline__ float moment2(const Hyper& h, float v, float g) {
#pragma clang fp contract(off)
    return h.beta2 * v + h.om_beta2 * g * g;
}
__device__ __forceinline__ float updated(const Hyper& h, float p, float m, float r) { return p * h.shrink - h.rate * m / (r * h.inv_root + h.eps); }

__device__ __forceinline__ uint32_t tensor_of(const AdamwArgs& a, uint32_t block) {
    const uint32_t lane = threadIdx.x & 63;
    const uint64_t has = __ballot(lane < kTensors && a.first[lane < kTensors ? lane : 0] <= block);
    return __builtin_amdgcn_readfirstlane((uint32_t)__popcll(has) - 1u);
}

// 32-bit moments: four consecutive values a thread.  28 bytes a value: 250 M float32 values in 1 330 us, 5.3 TB/s (a large copy reaches 4.65).
template <typename T>
__device__ __forceinline__ void step32(const gf_adamw_tensor_t& t, const Hyper& h, uint64_t begin, uint64_t end) {
    T* p = (T*)t.p;
    const T* g = (const T*)t.g;
    float *m = (float*)t.m, *v = (float*)t.v;
    for (uint64_t i = begin + threadIdx.x * 4; i < end; i += kThreads * 4) {
        const int left = (int)min((uint64_t)4, end - i);
        float fp[4], fg[4], fm[4], fv[4];
        load4_of(g + i, left, fg);
        load4_of(m + i, left, fm);
        load4_of(v + i, left, fv);
        load4_of(p + i, left, fp);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float x = fg[k] * h.grad;
            fm[k] = moment1(h, fm[k], x);
            fv[k] = moment2(h, fv[k], x);
            fp[k] = updated(h, fp[k], fm[k], sqrtf(fv[k]));
        }
        store4_of(m + i, left, fm);
        store4_of(v + i, left, fv);
        store4_of(p + i, left, fp);
    }
}

// ---- 8-bit moments -------------------------------------------------------------------------------------------------------------------------
// A block of 128 values has one 32-bit scale a * (1 / 448), a its largest magnitude (2^-100 at least, so that its reciprocal is finite).  Sixteen lanes share a
// block: lane j holds values 4j .. 4j+3 and 64+4j .. 64+4j+3, so that every load of a row of lanes is 256 consecutive bytes of 32-bit values.
// Rounding to nearest would lose every change below half a spacing (up to 6 % of the value; the second moment moves by 1 - beta2 a step).  The
// value is therefore rounded to floor(value / spacing + u) with u the fractional part of index phi_1 + step phi_2 (a two-dimensional Weyl
// sequence): over successive steps u is evenly spread, so the stored values are right on average, with no random numbers and no state.
// 10 bytes a bfloat16 value: 200 M of them in 444 us, 4.5 TB/s; the conversions and the roundings that are asked for leave little beside it.
constexpr uint32_t kDitherIndex = 3242174889u, kDitherStep = 2447445414u;     // 2^32 / rho, 2^32 / rho^2; rho the real root of x^3 = x + 1
constexpr float kTiny = 7.888609052210118e-31f;                                // 2^-100

// Four values with |y| <= 448 to their e4m3 codes.  v_cvt_sr_fp8_f32 adds the top 20 bits of its seed below the three fraction bits that stay and
// truncates, at values below 2^-6 the same at their spacing of 2^-9: floor(|y| / spacing + u), for every u and y (compared over 4 M pairs).
__device__ __forceinline__ uint32_t encode_dithered4(const float y[4], uint32_t seed) {
    int w = __builtin_amdgcn_cvt_sr_fp8_f32(y[0], (int)seed, 0, 0);
    w = __builtin_amdgcn_cvt_sr_fp8_f32(y[1], (int)(seed + kDitherIndex), w, 1);
    w = __builtin_amdgcn_cvt_sr_fp8_f32(y[2], (int)(seed + 2 * kDitherIndex), w, 2);
    return (uint32_t)__builtin_amdgcn_cvt_sr_fp8_f32(y[3], (int)(seed + 3 * kDitherIndex), w, 3);
}

__device__ __forceinline__ void decode4(uint32_t w, float scale, float out[4]) {
    typedef float f2 __attribute__((ext_vector_type(2)));
    const f2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    out[0] = lo[0] * scale; out[1] = lo[1] * scale; out[2] = hi[0] * scale; out[3] = hi[1] * scale;
}

typedef uint32_t codes4 __attribute__((aligned(1)));
__device__ __forceinline__ uint32_t load_codes(const uint8_t* src, int left) {
    if (left >= 4) return *reinterpret_cast<const codes4*>(src);
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) if (i < left) w |= (uint32_t)src[i] << (8 * i);
    return w;
}
__device__ __forceinline__ void store_codes(uint8_t* dst, uint32_t w, int left) {
    if (left >= 4) { *reinterpret_cast<codes4*>(dst) = w; return; }
#pragma unroll
    for (int i = 0; i < 4; ++i) if (i < left) dst[i] = (uint8_t)(w >> (8 * i));
}

// The square root to nearest from one to a unit in the last place: a neighbour is the nearer one where the residual of the middle says so.  (The
// compiler's own also scales values below 2^-96, whose residual leaves the type's range; here those may be a unit off.  That scaling is half as
// many operations again, and they are what this kernel has least room for: 506 us with it, 482 so, for 200 M values.)
__device__ __forceinline__ float sqrt_nearest(float x) {
    const float s = __builtin_amdgcn_sqrtf(x);
    const float below = __uint_as_float(__float_as_uint(s) - 1), above = __uint_as_float(__float_as_uint(s) + 1);
    const float down = __builtin_fmaf(-below, s, x), up = __builtin_fmaf(-above, s, x);
    const float r = down <= 0.0f ? below : s;
    return up > 0.0f ? above : r;
}

template <typename T>
__device__ __forceinline__ void step8(const gf_adamw_tensor_t& t, const Hyper& h, uint64_t begin, uint64_t end, uint32_t word) {
    T* p = (T*)t.p;
    const T* g = (const T*)t.g;
    uint8_t *m = (uint8_t*)t.m, *v = (uint8_t*)t.v;
    const int lane16 = threadIdx.x & 15;
    // all lanes of a row run the same blocks; a ragged last block is whole lanes with nothing left
    for (uint64_t b = begin / 128 + (threadIdx.x >> 4); b * 128 < end; b += kThreads / 16) {
        const uint64_t i0 = b * 128 + 4 * lane16;
        float fp[8], fg[8], fm[8], fr[8];
        int left[2];
        const float ms = t.m_scale[b], vs = t.v_scale[b];
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const uint64_t i = i0 + 64 * q;
            left[q] = i < end ? (int)min((uint64_t)4, end - i) : 0;
            const uint64_t at = left[q] ? i : begin;
            load4_of(g + at, left[q], fg + 4 * q);
            load4_of(p + at, left[q], fp + 4 * q);
            decode4(load_codes(m + at, left[q]), ms, fm + 4 * q);
            decode4(load_codes(v + at, left[q]), vs, fr + 4 * q);
        }
        float am = 0, ar = 0;
#pragma unroll
        for (int k = 0; k < 8; ++k) {      // (values that are not there are zeros and stay so)
            const float x = fg[k] * h.grad;
            fm[k] = moment1(h, fm[k], x);
            fr[k] = sqrt_nearest(moment2(h, fr[k] * fr[k], x));
            // the reciprocal to one unit in the last place: nothing but this step's p depends on it
            fp[k] = fp[k] * h.shrink - h.rate * fm[k] * __builtin_amdgcn_rcpf(fr[k] * h.inv_root + h.eps);
            am = max_abs(am, fm[k]);
            ar = max_abs(ar, fr[k]);
        }
        // A root whose square leaves the type's range: a gradient above 1.8e19 / sqrt(1 - beta2), or a root above 1.8e19 that is still held.  The root itself does
        // not, and an infinite one would freeze all 128 values for good: it is formed again from what is still in memory, scaled.
        if (ar == __builtin_inff()) {
            ar = 0;
#pragma unroll 1
            for (int k = 0; k < 8; ++k) {
                if (fr[k] == __builtin_inff() && __builtin_fabsf(fm[k]) < __builtin_inff() && (k & 3) < left[k >> 2]) {
                    const uint64_t i = i0 + 64 * (k >> 2) + (k & 3);
                    const float r = __builtin_amdgcn_cvt_f32_fp8((int)v[i], 0) * vs * 0x1p-66f, x = (float)g[i] * h.grad * 0x1p-66f;
                    fr[k] = fminf(sqrtf(moment2(h, r * r, x)) * 0x1p66f, 3.4028234663852886e38f);
                    fp[k] = updated(h, (float)p[i], fm[k], fr[k]);
                }
                ar = max_abs(ar, fr[k]);
            }
        }
        // as integers: what is no number stays the largest and makes the whole block none
        const uint32_t bm = row_max_u32(__float_as_uint(am)), br = row_max_u32(__float_as_uint(ar));
        const float a_m = max_abs(kTiny, __uint_as_float(bm)), a_r = max_abs(kTiny, __uint_as_float(br));
        const float inv_m = 1.0f / a_m * 448.0f, inv_r = 1.0f / a_r * 448.0f;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const uint32_t seed = (uint32_t)(i0 + 64 * q) * kDitherIndex + word;
            float ym[4], yr[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                ym[k] = __builtin_amdgcn_fmed3f(fm[4 * q + k] * inv_m, -448.0f, 448.0f);
                // a second moment above zero stays so (the smallest code is 2^-9): m / sqrt(v) must not meet a lost one
                yr[k] = __builtin_amdgcn_fmed3f(fr[4 * q + k] * inv_r, fr[4 * q + k] > 0.0f ? 0x1p-9f : 0.0f, 448.0f);
            }
            const uint32_t wm = encode_dithered4(ym, seed), wr = encode_dithered4(yr, seed ^ 0x80000000u);
            if (left[q]) {
                const uint64_t i = i0 + 64 * q;
                store_codes(m + i, wm, left[q]);
                store_codes(v + i, wr, left[q]);
                store4_of(p + i, left[q], fp + 4 * q);
            }
        }
        if (lane16 == 0) { t.m_scale[b] = a_m * (1.0f / 448.0f); t.v_scale[b] = a_r * (1.0f / 448.0f); }
    }
}

template <typename T, int BITS>
__global__ __launch_bounds__(kThreads) void k_adamw(const AdamwArgs a) {
    if (a.found_inf && *a.found_inf != 0.0f) return;
    const uint32_t at = tensor_of(a, blockIdx.x);
    const gf_adamw_tensor_t t = a.t[at];
    const uint64_t begin = (uint64_t)(blockIdx.x - a.first[at]) * a.chunk, end = min(t.n, begin + a.chunk);
    const float now = *t.step + 1.0f;
    const Hyper h = hyper_of(a, now);
    if constexpr (BITS == 32) step32<T>(t, h, begin, end);
    else step8<T>(t, h, begin, end, (uint32_t)now * kDitherStep);
    if (a.count_steps) {
        __syncthreads();                  // the tensor's only workgroup: every thread has read the count
        if (threadIdx.x == 0) *t.step = now;
    }
}

// The counts of a call in which a tensor has several workgroups: raised when all of those have read them, i.e. by a launch behind.
__global__ __launch_bounds__(512) void k_count_steps(const StepArgs a) {
    if (a.found_inf && *a.found_inf != 0.0f) return;
    if (threadIdx.x < a.count) *a.step[threadIdx.x] += 1.0f;
}

template <typename T>
static void launch_adamw(const AdamwArgs& a, uint32_t blocks, uint32_t bits, hipStream_t s) {
    if (bits == 32) k_adamw<T, 32><<<blocks, kThreads, 0, s>>>(a);
    else k_adamw<T, 8><<<blocks, kThreads, 0, s>>>(a);
}

// ---- the gradients' norm -------------------------------------------------------------------------------------------------------------------
constexpr int kNormTensors = 140;         // per launch, as many as 4 KB of arguments hold
constexpr uint32_t kNormBlocks = 2048;    // sums of one call, apart from one per tensor

struct NormArgs {
    gf_norm_tensor_t t[kNormTensors];
    uint32_t first[kNormTensors];
    uint64_t chunk;                       // values per workgroup, a multiple of 4096
    double* sums;
};
static_assert(sizeof(NormArgs) <= 4096, "kernel arguments");

__device__ __forceinline__ double block_sum(double x, double* lds) {
#pragma unroll
    for (int o = 32; o; o >>= 1) x += __shfl_xor(x, o);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = x;
    __syncthreads();
    double r = 0;
    for (uint32_t w = 0; w < blockDim.x / 64; ++w) r += lds[w];
    return r;
}

// Squares are added up in 64 bits: a 32-bit square leaves the type's range at 1e19 and at 1e-23, and the sum is one over all values of a model.
// 250 M float32 gradients in 220 us, 4.5 TB/s.
template <typename T>
__device__ __forceinline__ double squares(const T* g, uint64_t begin, uint64_t end) {
    double s[4] = {0, 0, 0, 0};
    uint64_t i = begin + threadIdx.x * 4;
    constexpr int U = 8;                  // loads under way
    for (; i + (U - 1) * kThreads * 4 + 4 <= end; i += U * kThreads * 4) {
        float f[U][4];
#pragma unroll
        for (int q = 0; q < U; ++q) load4(g + i + q * kThreads * 4, f[q]);
#pragma unroll
        for (int q = 0; q < U; ++q)
#pragma unroll
            for (int k = 0; k < 4; ++k) s[k] = fma((double)f[q][k], (double)f[q][k], s[k]);
    }
    for (; i < end; i += kThreads * 4) {
        float f[4];
        load4_of(g + i, (int)min((uint64_t)4, end - i), f);
#pragma unroll
        for (int k = 0; k < 4; ++k) s[k] = fma((double)f[k], (double)f[k], s[k]);
    }
    return (s[0] + s[1]) + (s[2] + s[3]);
}

__global__ __launch_bounds__(kThreads) void k_norm(const NormArgs a) {
    __shared__ double lds[kThreads / 64];
    const uint32_t lane = threadIdx.x & 63;
    uint32_t at = 0;
    for (uint32_t r = 0; r < kNormTensors; r += 64)
        at += (uint32_t)__popcll(__ballot(r + lane < kNormTensors && a.first[r + lane < kNormTensors ? r + lane : 0] <= blockIdx.x));
    at = __builtin_amdgcn_readfirstlane(at) - 1;
    const gf_norm_tensor_t t = a.t[at];
    const uint64_t begin = (blockIdx.x - a.first[at]) * a.chunk, end = min(t.n, begin + a.chunk);
    double s;
    if (t.dtype == F32) s = squares((const float*)t.g, begin, end);
    else if (t.dtype == BF16) s = squares((const __bf16*)t.g, begin, end);
    else s = squares((const _Float16*)t.g, begin, end);
    s = block_sum(s, lds);
    if (threadIdx.x == 0) a.sums[blockIdx.x] = s;
}

__global__ __launch_bounds__(1024) void k_norm_finish(const double* sums, uint32_t count, const float* grad_scale, float* out, double* wide) {
    __shared__ double lds[16];
    double s = 0;
    for (uint32_t i = threadIdx.x; i < count; i += 1024) s += sums[i];
    s = block_sum(s, lds);
    if (threadIdx.x) return;
    const double norm = sqrt(s) * (grad_scale ? 1.0 / (double)*grad_scale : 1.0);
    *out = (float)norm;
    if (wide) *wide = norm;
}

}  // namespace gf

using namespace gf;

GF_EXPORT int gf_adamw_step(const gf_adamw_t* d, void* stream) {
    if (!d) return gf_set_error(GF_ERR_INVALID, "gf_adamw_step: null descriptor");
    if (d->count == 0) return GF_OK;
    if (!d->tensors_host) return gf_set_error(GF_ERR_INVALID, "gf_adamw_step: null tensor list");
    if (d->dtype > F16) return gf_set_error(GF_ERR_INVALID, "gf_adamw_step: unknown dtype %u", d->dtype);
    if (d->state_bits != 32 && d->state_bits != 8) return gf_set_error(GF_ERR_INVALID, "gf_adamw_step: state_bits must be 32 or 8, got %u", d->state_bits);
    if (!(d->beta1 >= 0 && d->beta1 < 1 && d->beta2 >= 0 && d->beta2 < 1)) return gf_set_error(GF_ERR_INVALID, "gf_adamw_step: betas must be in [0, 1)");
    uint64_t total = 0, most = 0;
    for (uint32_t i = 0; i < d->count; ++i) {
        const gf_adamw_tensor_t& t = d->tensors_host[i];
        if (!t.step || (t.n && (!t.p || !t.g || !t.m || !t.v || (d->state_bits == 8 && (!t.m_scale || !t.v_scale)))))
            return gf_set_error(GF_ERR_INVALID, "gf_adamw_step: null pointer in tensor %u", i);
        if (t.n >> 40) return gf_set_error(GF_ERR_INVALID, "gf_adamw_step: tensor %u has too many values", i);
        total += t.n;
        most = t.n > most ? t.n : most;
    }
    // Values per workgroup: as many workgroups as keep the chip's 256 CUs busy where there is work for them, few enough that each amortises its
    // scalars (two powers in 64 bits, about half a microsecond) where there is more.
    uint32_t chunk = 1024;
    while (chunk < 8192 && total / chunk > 4096) chunk *= 2;
    while (total / chunk > (1ull << 23)) chunk *= 2;      // a launch's work-items lie below 2^32

    AdamwArgs a;
    a.beta1 = d->beta1; a.beta2 = d->beta2; a.lr = d->lr;
    a.weight_decay = d->weight_decay; a.max_norm = d->max_norm; a.eps = (float)d->eps;
    a.chunk = chunk;
    a.count_steps = most <= chunk;
    a.lr_device = d->lr_device; a.grad_scale = d->grad_scale; a.found_inf = d->found_inf; a.grad_norm = d->grad_norm; a.grad_norm_wide = d->grad_norm_wide;
    const hipStream_t s = gf_stream(stream);
    for (uint32_t i = 0; i < d->count;) {
        uint32_t k = 0, blocks = 0;
        for (; i < d->count && k < kTensors; ++i, ++k) {
            const gf_adamw_tensor_t& t = d->tensors_host[i];
            const uint32_t need = t.n ? (uint32_t)((t.n + chunk - 1) / chunk) : 1;       // an empty tensor's step is counted too
            a.t[k] = t;
            a.first[k] = blocks;
            blocks += need;
        }
        for (; k < kTensors; ++k) { a.t[k] = a.t[0]; a.first[k] = 0xffffffffu; }
        if (d->dtype == F32) launch_adamw<float>(a, blocks, d->state_bits, s);
        else if (d->dtype == BF16) launch_adamw<__bf16>(a, blocks, d->state_bits, s);
        else launch_adamw<_Float16>(a, blocks, d->state_bits, s);
    }
    if (!a.count_steps) {
        StepArgs c;
        c.found_inf = d->found_inf;
        for (uint32_t i = 0; i < d->count;) {
            for (c.count = 0; i < d->count && c.count < 496; ++i) c.step[c.count++] = d->tensors_host[i].step;
            k_count_steps<<<1, 512, 0, s>>>(c);
        }
    }
    return gf_check_launch("gf_adamw_step");
}

GF_EXPORT uint64_t gf_grad_norm_workspace_bytes(uint32_t count) { return 8ull * ((uint64_t)kNormBlocks + count); }

GF_EXPORT int gf_grad_norm(const gf_grad_norm_t* d, void* stream) {
    if (!d) return gf_set_error(GF_ERR_INVALID, "gf_grad_norm: null descriptor");
    if (!d->norm_out || !d->workspace || (d->count && !d->tensors_host)) return gf_set_error(GF_ERR_INVALID, "gf_grad_norm: null pointer");
    uint64_t total = 0;
    for (uint32_t i = 0; i < d->count; ++i) {
        const gf_norm_tensor_t& t = d->tensors_host[i];
        if (t.n && !t.g) return gf_set_error(GF_ERR_INVALID, "gf_grad_norm: null pointer in tensor %u", i);
        if (t.dtype > F16) return gf_set_error(GF_ERR_INVALID, "gf_grad_norm: unknown dtype %u in tensor %u", t.dtype, i);
        if (t.n >> 40) return gf_set_error(GF_ERR_INVALID, "gf_grad_norm: tensor %u has too many values", i);
        total += t.n;
    }
    const hipStream_t s = gf_stream(stream);
    NormArgs a;
    a.chunk = (total / kNormBlocks + 4096) / 4096 * 4096;
    uint32_t done = 0;
    for (uint32_t i = 0; i < d->count;) {
        int k = 0;
        uint32_t blocks = 0;
        for (; i < d->count && k < kNormTensors; ++i) {
            const gf_norm_tensor_t& t = d->tensors_host[i];
            if (!t.n) continue;
            const uint32_t need = (uint32_t)((t.n + a.chunk - 1) / a.chunk);
            a.t[k] = t;
            a.first[k++] = blocks;
            blocks += need;
        }
        if (!blocks) break;
        for (; k < kNormTensors; ++k) { a.t[k] = a.t[0]; a.first[k] = 0xffffffffu; }
        a.sums = (double*)d->workspace + done;
        k_norm<<<blocks, kThreads, 0, s>>>(a);
        done += blocks;
    }
    k_norm_finish<<<1, 1024, 0, s>>>((const double*)d->workspace, done, d->grad_scale, d->norm_out, d->norm_out_wide);
    return gf_check_launch("gf_grad_norm");
}
