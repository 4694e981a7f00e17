/*
 * geneface_train_hip.h -- the part of libgeneface_hip.so's C ABI that a training step needs beside the field's own nodes: AdamW over many
 * tensors at once, the global norm of their gradients, and block-scaled 8-bit linear products.
 *
 * Conventions are those of geneface_hip.h: device pointers unless a name ends in _host, outputs allocated by the caller, `stream` a hipStream_t,
 * calls only enqueue work, 0 on success and gf_last_error() otherwise.  `dtype` is one of GF_F32 / GF_BF16 / GF_F16.
 */
#ifndef GENEFACE_TRAIN_HIP_H
#define GENEFACE_TRAIN_HIP_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define GF_F32 0
#define GF_BF16 1
#define GF_F16 2

/* One tensor of gf_adamw_step: n values of p (updated), g (read), the moments m and v (updated) and the step count (one float, incremented).
 * With 32-bit moments m and v are float[n] and the scales NULL.  With 8-bit moments m and v are e4m3 codes [n] and m_scale / v_scale
 * float[ceil(n / 128)]: m[i] = m_code[i] m_scale[i / 128] and sqrt(v[i]) = v_code[i] v_scale[i / 128]. */
typedef struct {
    void* p;
    const void* g;
    void* m;
    void* v;
    float* m_scale;
    float* v_scale;
    float* step;
    uint64_t n;
} gf_adamw_tensor_t;

/* Host descriptor; tensors_host is read during the call.  grad_scale, found_inf, grad_norm and lr_device are one float on the device each, or
 * NULL.  The gradients that enter are g / grad_scale min(1, max_norm / (grad_norm + 1e-6)); grad_norm_wide:
 * the norm in 64 bits, taken where it rounds to *grad_norm, or NULL.  Where *found_inf is not 0 nothing is changed, the
 * step counts included.  What is written is read through no other pointer; g may be its own p.  lr_device replaces lr.  dtype: of p and g.  state_bits: 32 or 8. */
typedef struct {
    const gf_adamw_tensor_t* tensors_host;
    uint32_t count;
    uint32_t dtype;
    uint32_t state_bits;
    uint32_t _pad;
    double lr, beta1, beta2, eps, weight_decay, max_norm;
    const float* lr_device;
    const float* grad_scale;
    const float* found_inf;
    const float* grad_norm;
    const double* grad_norm_wide;
} gf_adamw_t;

/* p <- p (1 - lr wd);  m <- m + (1 - beta1)(g - m);  v <- beta2 v + (1 - beta2) g^2;
 * p <- p - lr / (1 - beta1^t) m / (sqrt(v) / sqrt(1 - beta2^t) + eps), t the incremented step. */
int gf_adamw_step(const gf_adamw_t* desc, void* stream);

/* One tensor of gf_grad_norm: n values of `dtype`. */
typedef struct {
    const void* g;
    uint64_t n;
    uint32_t dtype;
    uint32_t _pad;
} gf_norm_tensor_t;

/* Host descriptor; tensors_host is read during the call.  norm_out[0] = sqrt(sum over all tensors of g^2) / grad_scale, added up in 64 bits in
 * a fixed order; grad_scale: one float on the device, or NULL.  workspace: gf_grad_norm_workspace_bytes(count) device bytes of this call's own. */
typedef struct {
    const gf_norm_tensor_t* tensors_host;
    uint32_t count;
    uint32_t _pad;
    const float* grad_scale;
    float* norm_out;
    void* workspace;
    double* norm_out_wide;      /* the same in 64 bits, or NULL */
} gf_grad_norm_t;

uint64_t gf_grad_norm_workspace_bytes(uint32_t count);
int gf_grad_norm(const gf_grad_norm_t* desc, void* stream);

/* ------------------------------------------------------------------------------------------------
 * Products of block-scaled 8-bit values.
 *
 * Codes are e4m3 (largest 448).  A block of 128 values has the scale 2^(byte - 127): the smallest power of two >= 2^-127 with
 * (largest magnitude) <= 448 * scale; the byte is 255 and every code NaN where the block holds an infinity or a NaN.  Codes are
 * rounded to nearest even.  Products are added up in 32 bits where the result is float32 or binary16; where it is bfloat16, products of eight neighbours
 * along the sum are first added with what each has above 2^-13 of the largest of them (at most 7 * 2^-13 of that is lost), the eights in 32 bits.  An operand [R, K] that is summed over K is held as codes [R, Kp], Kp = K rounded up to a multiple of 128 and the
 * codes behind K zero, and scales either by row, byte (r, b) at [b * pitch + r], or by tile of 128 x 128, byte at [(r / 128) * stride_row + b *
 * stride_block].
 * ---------------------------------------------------------------------------------------------- */

/* src [rows, cols] of `dtype`, ld values from row to row.  row_codes [rows, up(cols)] with row_scales [up(cols)/128, row_pitch]: blocks along the
 * rows; col_codes [cols, up(rows)] with col_scales [up(rows)/128, col_pitch]: blocks along the columns, transposed.  Either may be NULL.
 * tiles != 0: one scale for each 128 x 128 in tile_scales [up(rows)/128, up(cols)/128] for both, row_scales and col_scales unused. */
typedef struct {
    const void* src;
    uint64_t rows, cols, ld;
    uint32_t dtype;
    uint32_t tiles;
    uint8_t* row_codes;
    uint8_t* row_scales;
    uint8_t* col_codes;
    uint8_t* col_scales;
    uint8_t* tile_scales;
    uint64_t row_pitch, col_pitch;
} gf_fp8_quantize_t;
int gf_fp8_quantize(const gf_fp8_quantize_t* desc, void* stream);

/* One operand of gf_fp8_matmul: codes [rows, 128 * blocks].  pitch > 0: scales by row; 0: by tile. */
typedef struct {
    const uint8_t* codes;
    const uint8_t* scales;
    uint64_t pitch;
    uint64_t stride_row, stride_block;
} gf_fp8_operand_t;

/* out [m, n] of `dtype` (contiguous) = a [m, 128 blocks] b [n, 128 blocks]^T; blocks <= 65535.
 * workspace: gf_fp8_matmul_workspace_bytes(m, n, blocks) device bytes of this call's own (NULL where that is 0). */
typedef struct {
    gf_fp8_operand_t a, b;
    uint64_t m, n, blocks;
    void* out;
    uint32_t dtype;
    uint32_t _pad;
    void* workspace;
} gf_fp8_matmul_t;
uint64_t gf_fp8_matmul_workspace_bytes(uint64_t m, uint64_t n, uint64_t blocks);
int gf_fp8_matmul(const gf_fp8_matmul_t* desc, void* stream);

/* out [m, n] = Q(x) w^T for m <= 16 rows x [m, k] of `dtype` (ldx values from row to row): x is brought to 8 bits on the way, w is held as codes
 * [n, up(k)] with one scale for each 128 x 128 at [(n / 128) * ceil(k / 128) + k / 128].  out: `dtype`, contiguous. */
typedef struct {
    const void* x;
    uint64_t m, n, k, ldx;
    const uint8_t* codes;
    const uint8_t* scales;
    void* out;
    uint32_t dtype;
    uint32_t _pad;
} gf_fp8_rows_t;
int gf_fp8_rows(const gf_fp8_rows_t* desc, void* stream);

/* The same products where n and k are at most 128, a block each, in one launch over the rows: y [m, n] = Q_row(x) w^T with w as codes [n, 128] and the
 * byte of its one scale; x by columns is left in col_codes [k, up(m)] and col_scales [up(m)/128, k], or both are NULL. */
typedef struct {
    const void* x;
    uint64_t ldx, m, n, k;
    const uint8_t* codes;
    const uint8_t* scale;
    void* y;
    uint8_t* col_codes;
    uint8_t* col_scales;
    uint32_t dtype;
    uint32_t _pad;
} gf_fp8_thin_t;
int gf_fp8_thin(const gf_fp8_thin_t* desc, void* stream);

/* dx [m, k] of dtype (or NULL) from the weight by columns, codes [k, 128] and the byte of its scale; dw [n, k] of w_dtype (or NULL) from x by columns
 * as gf_fp8_thin left it.  workspace: gf_fp8_thin_workspace_bytes(m, n, k) device bytes of this call's own, where dw is given. */
typedef struct {
    const void* dy;
    uint64_t lddy, m, n, k;
    const uint8_t* codes;
    const uint8_t* scale;
    const uint8_t* col_codes;
    const uint8_t* col_scales;
    void* dx;
    void* dw;
    void* workspace;
    uint32_t dtype, w_dtype;
} gf_fp8_thin_backward_t;
uint64_t gf_fp8_thin_workspace_bytes(uint64_t m, uint64_t n, uint64_t k);
int gf_fp8_thin_backward(const gf_fp8_thin_backward_t* desc, void* stream);

/* A linear layer, y [m, n] = Q_row(x) Q_tile(w)^T, and its gradients dx [m, k] = Q_row(dy) Q_tile(w), dw [n, k] = Q_col(dy)^T Q_col(x), each as one
 * call that enqueues all its launches.  x, dy: ldx / lddy values from row to row.  The weight is given as values w [n, k] of w_dtype (ldw values from
 * row to row), or as codes and scales as gf_fp8_rows takes them (w NULL).  y and dx have dtype, dw has w_dtype; all contiguous.
 * keep_w, keep_x: what the backward call will need is left in `saved` (keep_w for dx: w by columns; keep_x for dw: x by columns, one byte a value).
 * gf_fp8_linear_plan fills saved_bytes, workspace_bytes and backward_bytes (the workspace of the backward call); the buffers start at multiples of
 * 256 bytes, and a workspace is one call's own until the stream has passed it.  No size may be 0. */
typedef struct {
    const void* x;
    uint64_t ldx;
    const void* w;
    uint64_t ldw;
    const uint8_t* codes;
    const uint8_t* scales;
    uint64_t m, n, k;
    void* y;
    void* saved;
    void* workspace;
    uint32_t dtype, w_dtype, keep_w, keep_x;
    uint64_t saved_bytes, workspace_bytes, backward_bytes;
} gf_fp8_linear_t;
int gf_fp8_linear_plan(gf_fp8_linear_t* desc_host);
int gf_fp8_linear(const gf_fp8_linear_t* desc, void* stream);

typedef struct {
    const void* dy;
    uint64_t lddy;
    const void* saved;
    uint64_t m, n, k;
    void* dx;            /* NULL: not wanted (keep_w was 0 or the caller has no use for it) */
    void* dw;            /* NULL: not wanted */
    void* workspace;
    uint32_t dtype, w_dtype, keep_w, keep_x;
} gf_fp8_linear_backward_t;
int gf_fp8_linear_backward(const gf_fp8_linear_backward_t* desc, void* stream);

#ifdef __cplusplus
}
#endif
#endif
