// gf_fp8_linear and gf_fp8_linear_backward: a layer's products with what they need around them, as one call each.  Host code over the entry points of
// fp8_quantize.hip and fp8_matmul.hip; what it decides is where everything lies in the caller's two buffers.
#include "../common.hpp"
#include "fp8_calls.hpp"
#include "geneface_train_hip.h"

namespace gf {

// One block of 128 on either side: gf_fp8_thin (262221 rows, 96 -> 128, 32 bits, both directions: 120 us, by the general path 179).
static bool thin(uint64_t n, uint64_t k) { return n <= 128 && k <= 128; }

static uint64_t blocks_of(uint64_t n) { return (n + 127) / 128; }

// Hands out pieces of a buffer at multiples of 256 bytes; with base NULL it only measures.
struct Pieces {
    uint8_t* base;
    uint64_t used = 0;
    uint8_t* take(uint64_t bytes) {
        uint8_t* p = base ? base + used : nullptr;
        used += (bytes + 255) / 256 * 256;
        return p;
    }
};

struct Saved { uint8_t *w_codes, *w_scales, *x_codes, *x_scales; };      // w by columns [k, up(n)] and its tiles' scales, x by columns [k, up(m)]

static Saved saved_pieces(Pieces& p, uint64_t m, uint64_t n, uint64_t k, bool keep_w, bool keep_x) {
    Saved s = {};
    if (keep_w) { s.w_codes = p.take(k * blocks_of(n) * 128); s.w_scales = p.take(blocks_of(n) * blocks_of(k)); }
    if (keep_x) { s.x_codes = p.take(k * blocks_of(m) * 128); s.x_scales = p.take(blocks_of(m) * k); }
    return s;
}

struct Forward { uint8_t *x_codes, *x_scales, *w_codes, *w_scales, *parts; };

static Forward forward_pieces(Pieces& p, const gf_fp8_linear_t& d) {
    Forward f = {};
    if (!d.w && d.m <= 16) return f;      // gf_fp8_rows needs nothing
    if (thin(d.n, d.k)) return f;         // and neither does gf_fp8_thin
    f.x_codes = p.take(d.m * blocks_of(d.k) * 128);
    f.x_scales = p.take(blocks_of(d.k) * d.m);
    f.parts = p.take(gf_fp8_matmul_workspace_bytes(d.m, d.n, blocks_of(d.k)));
    if (d.w) f.w_codes = p.take(d.n * blocks_of(d.k) * 128);
    if (d.w && !d.keep_w) f.w_scales = p.take(blocks_of(d.n) * blocks_of(d.k));
    return f;
}

struct Backward { uint8_t *row_codes, *row_scales, *col_codes, *col_scales, *parts; };

static Backward backward_pieces(Pieces& p, uint64_t m, uint64_t n, uint64_t k, bool dx, bool dw) {
    Backward b = {};
    uint64_t parts = 0;
    if (thin(n, k)) {
        if (dw) b.parts = p.take(gf_fp8_thin_workspace_bytes(m, n, k));
        return b;
    }
    if (dx) {
        b.row_codes = p.take(m * blocks_of(n) * 128);
        b.row_scales = p.take(blocks_of(n) * m);
        parts = gf_fp8_matmul_workspace_bytes(m, k, blocks_of(n));
    }
    if (dw) {
        b.col_codes = p.take(n * blocks_of(m) * 128);
        b.col_scales = p.take(blocks_of(m) * n);
        const uint64_t need = gf_fp8_matmul_workspace_bytes(n, k, blocks_of(m));
        parts = parts > need ? parts : need;
    }
    b.parts = p.take(parts);
    return b;
}

static int size_error(const char* what, uint64_t m, uint64_t n, uint64_t k) {
    if (m == 0 || n == 0 || k == 0) return gf_set_error(GF_ERR_INVALID, "%s: an empty matrix", what);
    if (m >> 31 || n >> 31 || k >> 31) return gf_set_error(GF_ERR_INVALID, "%s: matrix too large", what);
    return GF_OK;
}

// gf_fp8_matmul adds up at most 65535 blocks: what the backward call would refuse is refused before there is anything to go back to.
static int sum_error(const gf_fp8_linear_t& d) {
    if (thin(d.n, d.k)) return GF_OK;
    const uint64_t most = 65535ull * 128;
    if (d.k > most || (d.keep_w && d.n > most) || (d.keep_x && d.m > most))
        return gf_set_error(GF_ERR_INVALID, "gf_fp8_linear: more than %llu values along a sum", (unsigned long long)most);
    return GF_OK;
}

}  // namespace gf

using namespace gf;

GF_EXPORT int gf_fp8_linear_plan(gf_fp8_linear_t* d) {
    if (!d) return gf_set_error(GF_ERR_INVALID, "gf_fp8_linear_plan: null descriptor");
    if (const int rc = size_error("gf_fp8_linear_plan", d->m, d->n, d->k)) return rc;
    if (const int rc = sum_error(*d)) return rc;
    Pieces s{nullptr}, f{nullptr}, b{nullptr};
    saved_pieces(s, d->m, d->n, d->k, d->keep_w, d->keep_x);
    forward_pieces(f, *d);
    backward_pieces(b, d->m, d->n, d->k, d->keep_w, d->keep_x);
    d->saved_bytes = s.used;
    d->workspace_bytes = f.used;
    d->backward_bytes = b.used;
    return GF_OK;
}

GF_EXPORT int gf_fp8_linear(const gf_fp8_linear_t* d, void* stream) {
    if (!d) return gf_set_error(GF_ERR_INVALID, "gf_fp8_linear: null descriptor");
    if (const int rc = size_error("gf_fp8_linear", d->m, d->n, d->k)) return rc;
    if (const int rc = sum_error(*d)) return rc;
    if (!d->x || !d->y || (!d->w && (!d->codes || !d->scales))) return gf_set_error(GF_ERR_INVALID, "gf_fp8_linear: null pointer");
    if (!d->w && (d->keep_w || d->keep_x)) return gf_set_error(GF_ERR_INVALID, "gf_fp8_linear: a weight given as codes has no backward call");
    if (!d->w && d->m <= 16) {
        const gf_fp8_rows_t r = {d->x, d->m, d->n, d->k, d->ldx, d->codes, d->scales, d->y, d->dtype, 0};
        return gf_fp8_rows(&r, stream);
    }
    if ((!d->workspace && !thin(d->n, d->k)) || ((d->keep_w || d->keep_x) && !d->saved)) return gf_set_error(GF_ERR_INVALID, "gf_fp8_linear: null buffer");
    if ((uintptr_t)d->workspace % 256 || (uintptr_t)d->saved % 256) return gf_set_error(GF_ERR_INVALID, "gf_fp8_linear: buffers must start at multiples of 256 bytes");
    Pieces ps{(uint8_t*)d->saved}, pf{(uint8_t*)d->workspace};
    const Saved s = saved_pieces(ps, d->m, d->n, d->k, d->keep_w, d->keep_x);
    const Forward f = forward_pieces(pf, *d);
    const uint64_t kb = blocks_of(d->k);
    const uint8_t *w_codes = d->w ? f.w_codes : d->codes, *w_scales = d->w ? (d->keep_w ? s.w_scales : f.w_scales) : d->scales;
    const gf_fp8_quantize_t qw = {d->w, d->n, d->k, d->ldw, d->w_dtype, 1, f.w_codes, nullptr, s.w_codes, nullptr, d->keep_w ? s.w_scales : f.w_scales, 0, 0};
    const gf_fp8_quantize_t qx = {d->x, d->m, d->k, d->ldx, d->dtype, 0, f.x_codes, f.x_scales, s.x_codes, s.x_scales, nullptr, d->m, d->k};
    if (thin(d->n, d->k)) {
        const gf_fp8_thin_t t = {d->x, d->ldx, d->m, d->n, d->k, w_codes, w_scales, d->y, s.x_codes, s.x_scales, d->dtype, 0};
        const ThinWeight w = {d->w, d->ldw, d->w_dtype, s.w_codes, s.w_scales};
        return thin_forward(t, d->w ? &w : nullptr, stream);
    }
    if (const int rc = d->w ? quantize_two(qw, qx, stream) : gf_fp8_quantize(&qx, stream)) return rc;
    const gf_fp8_matmul_t p = {{f.x_codes, f.x_scales, d->m, 0, 0}, {w_codes, w_scales, 0, kb, 1}, d->m, d->n, kb, d->y, d->dtype, 0, f.parts};
    return gf_fp8_matmul(&p, stream);
}

GF_EXPORT int gf_fp8_linear_backward(const gf_fp8_linear_backward_t* d, void* stream) {
    if (!d) return gf_set_error(GF_ERR_INVALID, "gf_fp8_linear_backward: null descriptor");
    if (const int rc = size_error("gf_fp8_linear_backward", d->m, d->n, d->k)) return rc;
    if (!d->dx && !d->dw) return GF_OK;
    if (!d->dy || !d->saved || (!d->workspace && (d->dw || !thin(d->n, d->k)))) return gf_set_error(GF_ERR_INVALID, "gf_fp8_linear_backward: null pointer");
    if ((d->dx && !d->keep_w) || (d->dw && !d->keep_x)) return gf_set_error(GF_ERR_INVALID, "gf_fp8_linear_backward: a gradient whose operand was not kept");
    if ((uintptr_t)d->workspace % 256 || (uintptr_t)d->saved % 256)
        return gf_set_error(GF_ERR_INVALID, "gf_fp8_linear_backward: buffers must start at multiples of 256 bytes");
    Pieces ps{(uint8_t*)d->saved}, pb{(uint8_t*)d->workspace};
    const Saved s = saved_pieces(ps, d->m, d->n, d->k, d->keep_w, d->keep_x);
    const Backward b = backward_pieces(pb, d->m, d->n, d->k, d->dx != nullptr, d->dw != nullptr);
    if (thin(d->n, d->k)) {
        const gf_fp8_thin_backward_t t = {d->dy, d->lddy, d->m, d->n, d->k, s.w_codes, s.w_scales, s.x_codes, s.x_scales, d->dx, d->dw, b.parts, d->dtype, d->w_dtype};
        return gf_fp8_thin_backward(&t, stream);
    }
    const gf_fp8_quantize_t q = {d->dy, d->m, d->n, d->lddy, d->dtype, 0, b.row_codes, b.row_scales, b.col_codes, b.col_scales, nullptr, d->m, d->n};
    if (const int rc = gf_fp8_quantize(&q, stream)) return rc;
    // dx: b is w by columns, its scales those of the tiles, transposed
    const gf_fp8_matmul_t x = {{b.row_codes, b.row_scales, d->m, 0, 0}, {s.w_codes, s.w_scales, 0, 1, blocks_of(d->k)}, d->m, d->k, blocks_of(d->n), d->dx, d->dtype, 0, b.parts};
    const gf_fp8_matmul_t w = {{b.col_codes, b.col_scales, d->n, 0, 0}, {s.x_codes, s.x_scales, d->k, 0, 0}, d->n, d->k, blocks_of(d->m), d->dw, d->w_dtype, 0, b.parts};
    if (d->dx && d->dw) return matmul_two(x, w, stream);
    return gf_fp8_matmul(d->dx ? &x : &w, stream);
}
