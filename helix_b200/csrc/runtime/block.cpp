// block.cpp -- entry points of the recurrent block's operators
// (helix_block.h): checks of arguments, plans, launches on the caller's
// stream.  Nothing here synchronises or allocates device memory, and no C++
// exception leaves an entry point.
#include "block_internal.h"

#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <string>
#include <utility>

namespace {

// Makes ctx's device current for a call, and the caller's again after it.
struct DeviceScope {
    int restore = -1;
    explicit DeviceScope(int dev) {
        int cur = dev;
        if (cudaGetDevice(&cur) == cudaSuccess && cur == dev) return;
        if (cudaSetDevice(dev) == cudaSuccess) restore = cur;
    }
    ~DeviceScope() {
        if (restore >= 0) cudaSetDevice(restore);
    }
};

// A refusal: the status and its message.
struct Refused {
    helix_status status;
    std::string  why;
};
[[noreturn]] void refuse(helix_status st, const std::string& why) { throw Refused{st, why}; }
[[noreturn]] void invalid(const std::string& why) { refuse(HELIX_ERR_INVALID_ARG, why); }
[[noreturn]] void unsupported(const std::string& why) { refuse(HELIX_ERR_UNSUPPORTED_SHAPE, why); }

// Runs the body of an entry point; its exceptions become a status.
template <class F>
helix_status entry(helix_ctx* ctx, const void* d, F body) noexcept {
    if (!ctx || !d) return HELIX_ERR_INVALID_ARG;
    try {
        try {
            DeviceScope scope(ctx->device);
            const int rc = body();
            if (rc == cudaSuccess) return HELIX_OK;
            hx::set_error(ctx, std::string("kernel launch failed: ") +
                                   cudaGetErrorString(static_cast<cudaError_t>(rc)));
            return HELIX_ERR_PIPELINE;
        } catch (const Refused& r) {
            hx::set_error(ctx, r.why);
            return r.status;
        }
    } catch (...) {  // out of host memory
        return HELIX_ERR_PIPELINE;
    }
}

uintptr_t addr(helix_tensor t) { return reinterpret_cast<uintptr_t>(t.buf) + t.offset; }
template <class T = void>
T* ptr(helix_tensor t) {
    return t.buf ? reinterpret_cast<T*>(addr(t)) : nullptr;
}

int64_t elem(helix_dtype t) { return t == HELIX_F32 ? 4 : t == HELIX_E4M3 ? 1 : 2; }
bool io(helix_dtype t) { return t == HELIX_F32 || t == HELIX_BF16; }

// A matrix argument of a call: `rows` rows of `cols` elements, `ld` apart; or
// `stack` such matrices, `step` elements apart.
struct Mat {
    const char*  name;
    helix_tensor t;
    int64_t      rows, cols, ld, size;
    bool         written;
    int64_t      stack = 1, step = 0;

    uintptr_t end() const {
        return addr(t) + (uintptr_t)(((stack - 1) * step + (rows - 1) * ld + cols) * size);
    }
};

void check_mat(const Mat& m) {
    if (!m.t.buf) return;
    const std::string n = m.name;
    if (addr(m.t) % (uintptr_t)m.size) invalid(n + " is not aligned to its elements");
    if (m.ld < 0 || (m.written && m.rows > 1 && m.ld < m.cols)) invalid(n + ": row stride too small");
    const int64_t most = INT64_MAX / 16;
    if (m.rows > 1 && m.ld > 0 && (m.rows - 1) > most / m.ld) invalid(n + ": rows reach past 64-bit offsets");
}

// Whether a row of one of two stacks with the same strides shares bytes with a
// row of the other: whether, for some difference i of their places in the
// stacks and j of their rows, the distance of the rows is less than their width.
// Exact, unless both differences have more than 2^16 values (then: they may).
bool stacks_overlap(const Mat& a, const Mat& b) {
    int64_t n = a.stack, m = a.rows, p = a.step * a.size, q = a.ld * a.size;
    if (n > m) std::swap(n, m), std::swap(p, q);
    const int64_t wa = a.cols * a.size, wb = b.cols * b.size;
    if (n > 1 << 16 || q <= 0) return true;
    const int64_t apart = (int64_t)(addr(b.t) - addr(a.t));
    for (int64_t i = 1 - n; i < n; ++i) {
        const int64_t d = apart + i * p;  // -wb < d + j q < wa
        int64_t j = (wa - 1 - d) / q;     // the largest such j, and what is below
        if ((wa - 1 - d) % q < 0) --j;
        j = std::min(j, m - 1);
        if (j > -m && d + j * q > -wb) return true;
    }
    return false;
}

// Whether two matrices share bytes.  Matrices with one row pitch may lie
// side by side in it (slices of one wider matrix).
bool overlap(const Mat& a, const Mat& b) {
    if (!a.t.buf || !b.t.buf || !a.rows || !b.rows || !a.cols || !b.cols) return false;
    const uintptr_t a0 = addr(a.t), b0 = addr(b.t);
    if (a.end() <= b0 || b.end() <= a0) return false;
    if (a.stack > 1 || b.stack > 1) {
        const bool alike = a.stack == b.stack && a.rows == b.rows && a.step * a.size == b.step * b.size &&
                           a.ld * a.size == b.ld * b.size;
        return !alike || stacks_overlap(a, b);
    }
    const uintptr_t pitch = (uintptr_t)(a.ld * a.size);
    if (a.rows > 1 && b.rows > 1 && pitch && pitch == (uintptr_t)(b.ld * b.size)) {
        const uintptr_t wa = (uintptr_t)(a.cols * a.size), wb = (uintptr_t)(b.cols * b.size);
        const uintptr_t off = b0 >= a0 ? (b0 - a0) % pitch : (pitch - (a0 - b0) % pitch) % pitch;
        if (off >= wa && off + wb <= pitch) return false;
    }
    return true;
}
bool same(const Mat& a, const Mat& b) {
    return addr(a.t) == addr(b.t) && a.size == b.size && (a.rows <= 1 || a.ld == b.ld);
}

// Checks every matrix, and each written one against all others; pairs in
// `in_place` (by index: the written one, the read one) may be one and the same.
template <size_t N, size_t M>
void check_mats(const Mat (&m)[N], const int (&in_place)[M][2]) {
    for (const Mat& x : m) check_mat(x);
    for (size_t i = 0; i < N; ++i) {
        if (!m[i].written) continue;
        for (size_t j = 0; j < N; ++j) {
            if (j == i || (m[j].written && j < i) || !overlap(m[i], m[j])) continue;
            bool ok = false;
            for (const auto& q : in_place)
                ok = ok || ((size_t)q[0] == i && (size_t)q[1] == j && same(m[i], m[j]));
            if (!ok) invalid(std::string(m[i].name) + " overlaps " + m[j].name);
        }
    }
}
constexpr int kNoneInPlace[1][2] = {{-1, -1}};

void need(helix_tensor t, const char* name) {
    if (!t.buf) invalid(std::string("null tensor: ") + name);
}

void check_scratch(helix_tensor s, size_t bytes, const char* size_fn) {
    if (!bytes) return;
    if (!s.buf) refuse(HELIX_ERR_SCRATCH_TOO_SMALL, std::string("a scratch buffer of ") + size_fn + "() is required");
    if (addr(s) & 255) invalid("scratch must be 256-byte aligned");
    if (!hx::scratch_fits(ptr(s), bytes))
        refuse(HELIX_ERR_SCRATCH_TOO_SMALL, std::string("scratch allocation smaller than ") + size_fn + "()");
}

// Whether rows of the matrix can be accessed in whole `bytes`-byte pieces at
// multiples of that many bytes.
bool whole(const Mat& m, int64_t bytes) {
    return !m.t.buf || (addr(m.t) % (uintptr_t)bytes == 0 && (m.rows <= 1 || m.ld * m.size % bytes == 0));
}

}  // namespace

// ---------------------------------------------------------------------------
// Norm
// ---------------------------------------------------------------------------
namespace {

void check_norm_desc(const helix_rms_norm_desc& d) {
    if (d.n_row < 0 || d.n_col < 1) unsupported("n_row must be >= 0 and n_col >= 1");
    if (d.n_col > 16384) unsupported("n_col must be at most 16384");
    if (d.n_row > INT_MAX) unsupported("n_row must be at most 2^31 - 1");
    if (!io(d.x_dtype)) unsupported("x_dtype must be F32 or BF16");
    if (d.sum_dtype != HELIX_F32 && d.sum_dtype != d.x_dtype) unsupported("sum_dtype must be F32 or x_dtype");
    if (!io(d.out_dtype) && d.out_dtype != HELIX_E4M3) unsupported("out_dtype must be F32, BF16 or E4M3");
    if (!io(d.w_dtype)) unsupported("w_dtype must be F32 or BF16");
    if (!(d.eps >= 0.0f)) invalid("eps must be >= 0");
}

}  // namespace

extern "C" void helix_rms_norm_desc_init(helix_rms_norm_desc* d, int64_t n_row, int32_t n_col) {
    if (!d) return;
    *d = helix_rms_norm_desc{};
    d->n_row = n_row;
    d->n_col = n_col;
    d->eps = 1e-6f;
    d->x_dtype = d->sum_dtype = d->out_dtype = d->w_dtype = HELIX_F32;
    d->ld_x = d->ld_res = d->ld_sum = d->ld_out = n_col;
    d->ld_dout = d->ld_dsum = d->ld_dx = d->ld_dres = n_col;
    d->ld_scale = ((int64_t)n_col + HELIX_GROUP - 1) / HELIX_GROUP;
}

extern "C" helix_status helix_rms_norm_encode(helix_ctx* ctx, void* stream, const helix_rms_norm_desc* d,
                                              helix_tensor x, helix_tensor residual, helix_tensor weight,
                                              helix_tensor out, helix_tensor scale, helix_tensor sum,
                                              helix_tensor rstd) {
    return entry(ctx, d, [&]() -> int {
        check_norm_desc(*d);
        if (d->n_row == 0) return cudaSuccess;
        need(x, "x");
        need(weight, "weight");
        need(out, "out");
        const bool q = d->out_dtype == HELIX_E4M3;
        if (q) need(scale, "scale");
        const int64_t n = d->n_row, c = d->n_col, groups = (c + HELIX_GROUP - 1) / HELIX_GROUP;
        const Mat m[] = {{"x", x, n, c, d->ld_x, elem(d->x_dtype), false},
                         {"residual", residual, n, c, d->ld_res, elem(d->sum_dtype), false},
                         {"weight", weight, 1, c, c, elem(d->w_dtype), false},
                         {"out", out, n, c, d->ld_out, elem(d->out_dtype), true},
                         {"sum", sum, n, c, d->ld_sum, elem(d->sum_dtype), true},
                         {"scale", q ? scale : HELIX_TENSOR_NULL, n, groups, d->ld_scale, 4, true},
                         {"rstd", rstd, 1, n, n, 4, true}};
        const int in_place[][2] = {{4, 1}, {4, 0}};
        check_mats(m, in_place);
        hx::NormParams p{};
        p.n_row = n;
        p.n_col = d->n_col;
        p.inv_col = 1.0f / (float)d->n_col;
        const hx::NormShape s = hx::norm_shape(*d);
        p.wpr = s.wpr;
        p.rpb = s.rpb;
        p.eps = d->eps;
        p.out_dtype = d->out_dtype;
        p.w_bf16 = d->w_dtype == HELIX_BF16;
        p.ld_x = d->ld_x, p.ld_res = d->ld_res, p.ld_sum = d->ld_sum, p.ld_out = d->ld_out, p.ld_scale = d->ld_scale;
        p.x = ptr(x), p.res = ptr(residual), p.w = ptr(weight);
        p.out = ptr(out), p.sum = ptr(sum);
        p.scale = ptr<float>(scale), p.rstd = ptr<float>(rstd);
        const bool vec = whole(m[0], 16) && whole(m[1], 16) && whole(m[2], 16) && whole(m[3], q ? 8 : 16) &&
                         whole(m[4], 16);
        return hx::launch_norm(ctx, *d, p, vec, stream);
    });
}

extern "C" size_t helix_rms_norm_grad_scratch_size(helix_ctx* ctx, const helix_rms_norm_desc* d) {
    if (!d || d->n_row < 0 || d->n_col < 1 || d->n_col > 16384) return 0;
    return hx::norm_grad_plan(ctx, *d).total;
}

extern "C" helix_status helix_rms_norm_grad_encode(helix_ctx* ctx, void* stream, const helix_rms_norm_desc* d,
                                                   helix_tensor dout, helix_tensor sum, helix_tensor rstd,
                                                   helix_tensor weight, helix_tensor dsum, helix_tensor dx,
                                                   helix_tensor dres, helix_tensor dweight,
                                                   helix_tensor scratch) {
    return entry(ctx, d, [&]() -> int {
        check_norm_desc(*d);
        need(dweight, "dweight");
        need(weight, "weight");
        if (d->n_row > 0) {
            need(dout, "dout");
            need(sum, "sum");
            need(rstd, "rstd");
            need(dx, "dx");
        }
        const hx::NormGradPlan pl = hx::norm_grad_plan(ctx, *d);
        check_scratch(scratch, pl.total, "helix_rms_norm_grad_scratch_size");
        const int64_t n = d->n_row, c = d->n_col, ts = elem(d->sum_dtype), tx = elem(d->x_dtype);
        const Mat m[] = {{"dout", dout, n, c, d->ld_dout, tx, false},
                         {"sum", sum, n, c, d->ld_sum, ts, false},
                         {"rstd", rstd, 1, n, n, 4, false},
                         {"weight", weight, 1, c, c, elem(d->w_dtype), false},
                         {"dsum", dsum, n, c, d->ld_dsum, ts, false},
                         {"dx", dx, n, c, d->ld_dx, tx, true},
                         {"dres", dres, n, c, d->ld_dres, ts, true},
                         {"dweight", dweight, 1, c, c, 4, true},
                         {"scratch", scratch, 1, (int64_t)pl.total, (int64_t)pl.total, 1, true}};
        const int in_place[][2] = {{5, 0}, {6, 4}};
        check_mats(m, in_place);
        hx::NormParams p{};
        p.n_row = n;
        p.n_col = d->n_col;
        p.inv_col = 1.0f / (float)d->n_col;
        p.w_bf16 = d->w_dtype == HELIX_BF16;
        p.ld_dout = d->ld_dout, p.ld_sum = d->ld_sum, p.ld_dsum = d->ld_dsum;
        p.ld_dx = d->ld_dx, p.ld_dres = d->ld_dres;
        p.dout = ptr(dout), p.sum = ptr(sum), p.dsum = ptr(dsum), p.w = ptr(weight);
        p.dx = ptr(dx), p.dres = ptr(dres), p.rstd = ptr<float>(rstd);
        p.partial = ptr<float>(scratch);
        const bool vec = whole(m[0], 16) && whole(m[1], 16) && whole(m[3], 16) && whole(m[4], 16) &&
                         whole(m[5], 16) && whole(m[6], 16);
        p.wpr = pl.shape.wpr;
        p.rpb = pl.shape.rpb;
        return hx::launch_norm_grad(*d, pl, p, vec, ptr<float>(dweight), stream);
    });
}

// ---------------------------------------------------------------------------
// Quantiser
// ---------------------------------------------------------------------------
extern "C" void helix_quant8_desc_init(helix_quant8_desc* d, int64_t n_row, int64_t n_col, helix_scale_form form,
                                       bool transpose) {
    if (!d) return;
    *d = helix_quant8_desc{};
    d->n_row = n_row;
    d->n_col = n_col;
    d->x_dtype = HELIX_F32;
    d->form = form;
    d->transpose = transpose;
    const int64_t q_cols = transpose ? n_row : n_col;
    d->ld_x = n_col;
    d->ld_q = (q_cols + 15) / 16 * 16;
    d->ld_scale = (q_cols + HELIX_GROUP - 1) / HELIX_GROUP;
}

extern "C" helix_status helix_quant8_encode(helix_ctx* ctx, void* stream, const helix_quant8_desc* d,
                                            helix_tensor x, helix_tensor q, helix_tensor scale) {
    return entry(ctx, d, [&]() -> int {
        if (d->n_row < 0 || d->n_col < 0) unsupported("n_row and n_col must be >= 0");
        if (d->n_row > INT_MAX || d->n_col > INT_MAX) unsupported("n_row and n_col must be at most 2^31 - 1");
        if (!io(d->x_dtype)) unsupported("x_dtype must be F32 or BF16");
        if (d->form != HELIX_SCALE_ROWS && d->form != HELIX_SCALE_BLOCKS) unsupported("unknown scale form");
        if (d->n_row == 0 || d->n_col == 0) return cudaSuccess;
        const int64_t tr = (d->n_row + HELIX_GROUP - 1) / HELIX_GROUP, tc = (d->n_col + HELIX_GROUP - 1) / HELIX_GROUP;
        if (tr * tc > INT_MAX) unsupported("problem too large for one launch");
        need(x, "x");
        need(q, "q");
        need(scale, "scale");
        const bool t = d->transpose, blocks = d->form == HELIX_SCALE_BLOCKS;
        const int64_t qr = t ? d->n_col : d->n_row, qc = t ? d->n_row : d->n_col;
        const Mat m[] = {{"x", x, d->n_row, d->n_col, d->ld_x, elem(d->x_dtype), false},
                         {"q", q, qr, qc, d->ld_q, 1, true},
                         {"scale", scale, blocks ? (t ? tc : tr) : qr, t ? tr : tc, d->ld_scale, 4, true}};
        check_mats(m, kNoneInPlace);
        hx::QuantParams p{};
        p.n_row = d->n_row, p.n_col = d->n_col;
        p.ld_x = d->ld_x, p.ld_q = d->ld_q, p.ld_scale = d->ld_scale;
        p.n_tile_col = (int32_t)tc;
        p.x = ptr(x), p.q = ptr<uint8_t>(q), p.scale = ptr<float>(scale);
        p.q_vec = whole(m[1], 8);
        return hx::launch_quant(*d, p, whole(m[0], 16), stream);
    });
}

// ---------------------------------------------------------------------------
// Product
// ---------------------------------------------------------------------------
extern "C" void helix_matmul8_desc_init(helix_matmul8_desc* d, int32_t m, int32_t n, int32_t k,
                                        helix_scale_form b_form) {
    if (!d) return;
    *d = helix_matmul8_desc{};
    d->m = m, d->n = n, d->k = k;
    d->b_form = b_form;
    d->out_dtype = HELIX_BF16;
    d->ld_a = d->ld_b = ((int64_t)k + 15) / 16 * 16;
    d->ld_out = n;
    d->ld_a_scale = d->ld_b_scale = ((int64_t)k + HELIX_GROUP - 1) / HELIX_GROUP;
}

extern "C" helix_status helix_matmul8_encode(helix_ctx* ctx, void* stream, const helix_matmul8_desc* d,
                                             helix_tensor a, helix_tensor a_scale, helix_tensor b,
                                             helix_tensor b_scale, helix_tensor out) {
    return entry(ctx, d, [&]() -> int {
        if (d->m < 0 || d->n < 0 || d->k < 1) unsupported("m and n must be >= 0 and k >= 1");
        if (d->b_form != HELIX_SCALE_ROWS && d->b_form != HELIX_SCALE_BLOCKS) unsupported("unknown scale form");
        if (!io(d->out_dtype)) unsupported("out_dtype must be F32 or BF16");
        // the kernel's coordinates are 32-bit, and reach a tile past the end
        if (d->m > INT_MAX - 512 || d->n > INT_MAX - 512 || d->k > INT_MAX - 512)
            unsupported("m, n and k must be at most 2^31 - 513");
        if (d->m == 0 || d->n == 0) return cudaSuccess;
        if (!ctx->encode_tiled) unsupported("tensor maps are unavailable on this device");
        need(a, "a");
        need(a_scale, "a_scale");
        need(b, "b");
        need(b_scale, "b_scale");
        need(out, "out");
        const int64_t kb = ((int64_t)d->k + HELIX_GROUP - 1) / HELIX_GROUP;
        const bool blocks = d->b_form == HELIX_SCALE_BLOCKS;
        const int64_t nb = blocks ? ((int64_t)d->n + HELIX_GROUP - 1) / HELIX_GROUP : d->n;
        const Mat m[] = {{"a", a, d->m, d->k, d->ld_a, 1, false},
                         {"a_scale", a_scale, d->m, kb, d->ld_a_scale, 4, false},
                         {"b", b, d->n, d->k, d->ld_b, 1, false},
                         {"b_scale", b_scale, nb, kb, d->ld_b_scale, 4, false},
                         {"out", out, d->m, d->n, d->ld_out, elem(d->out_dtype), true}};
        check_mats(m, kNoneInPlace);
        if (!whole(m[0], 16) || !whole(m[2], 16)) unsupported("a and b need 16-byte aligned rows");
        if (d->m > 1 && d->ld_a < d->k) invalid("a: row stride too small");
        if (d->n > 1 && d->ld_b < d->k) invalid("b: row stride too small");
        const hx::Mm8Plan pl = hx::mm8_plan(ctx, *d);
        hx::Mm8Params p{};
        const hx::Mm8Operand oa{ptr<float>(a_scale), d->ld_a_scale, d->m, 1, whole(m[1], 16)};
        const hx::Mm8Operand ob{ptr<float>(b_scale), d->ld_b_scale, d->n, blocks ? HELIX_GROUP : 1, whole(m[3], 16)};
        p.p = pl.swap ? ob : oa;
        p.q = pl.swap ? oa : ob;
        p.k_blocks = (int32_t)kb;
        p.splits = pl.splits;
        p.swap = pl.swap;
        p.ld_out = d->ld_out;
        p.out = ptr(out);
        p.vec_out = whole(m[4], 16);
        p.fault = ctx->fault_word;
        return hx::launch_mm8(ctx, *d, pl, p, ptr(a), ptr(b), stream);
    });
}

// ---------------------------------------------------------------------------
// Gated linear recurrence
// ---------------------------------------------------------------------------
namespace {

// A token tensor [n_seq][n_tok][n_chan].
struct Tok {
    const char*  name;
    helix_tensor t;
    int64_t      s_tok, s_seq;
    bool         written;
};

void check_tok(const helix_gated_scan_desc& d, const Tok& x) {
    const std::string n = x.name;
    if (addr(x.t) % (uintptr_t)elem(d.io_dtype)) invalid(n + " is not aligned to its elements");
    if (x.s_tok < 0 || x.s_seq < 0) invalid(n + ": negative stride");
    if (x.written) {
        // distinct elements have distinct addresses: the token rows do not
        // overlap within a sequence, nor the sequences (or they interleave)
        const bool rows = d.n_tok <= 1 || x.s_tok >= d.n_chan;
        const int64_t span = (int64_t)(d.n_tok - 1) * x.s_tok + d.n_chan;
        const bool seqs = d.n_seq <= 1 || x.s_seq >= span ||
                          (x.s_seq >= d.n_chan && (int64_t)(d.n_seq - 1) * x.s_seq + d.n_chan <= x.s_tok);
        if (!rows || !seqs) invalid(n + ": strides make its elements overlap");
    }
    const int64_t most = INT64_MAX / 64;
    if ((d.n_tok > 1 && x.s_tok > most / d.n_tok) || (d.n_seq > 1 && x.s_seq > most / d.n_seq))
        invalid(n + ": reaches past 64-bit offsets");
}

// A matrix where tokens follow one another at one pitch through all sequences,
// else a stack of the sequences' (slices of one wider tensor may lie side by
// side in both).
Mat mat_of(const helix_gated_scan_desc& d, const Tok& x) {
    const int64_t size = elem(d.io_dtype);
    if (d.n_seq <= 1 || x.s_seq == (int64_t)d.n_tok * x.s_tok)
        return {x.name, x.t, (int64_t)d.n_tok * d.n_seq, d.n_chan, x.s_tok, size, x.written};
    if (d.n_tok <= 1) return {x.name, x.t, d.n_seq, d.n_chan, x.s_seq, size, x.written};
    return {x.name, x.t, d.n_tok, d.n_chan, x.s_tok, size, x.written, d.n_seq, x.s_seq};
}
bool same_tok(const helix_gated_scan_desc& d, const Tok& a, const Tok& b) {
    return addr(a.t) == addr(b.t) && (d.n_tok <= 1 || a.s_tok == b.s_tok) && (d.n_seq <= 1 || a.s_seq == b.s_seq);
}

void check_gated_desc(const helix_gated_scan_desc& d) {
    if (d.n_tok < 0 || d.n_seq < 0 || d.n_chan < 0) unsupported("n_tok, n_seq and n_chan must be >= 0");
    if (!io(d.io_dtype)) unsupported("io_dtype must be F32 or BF16");
    // chunk indexes, the grid and the channels of a slab (64) are 32-bit
    if (d.n_tok > INT_MAX - 4096) unsupported("n_tok must be at most 2^31 - 4097");
    if (d.n_chan > INT_MAX - 64) unsupported("n_chan must be at most 2^31 - 65");
    const int64_t slabs = ((int64_t)d.n_chan + 31) / 32;
    if ((int64_t)d.n_seq * slabs > INT_MAX / 16) unsupported("problem too large for one launch");
}

// Two channels at once: 4-byte aligned rows.
bool pairs(const helix_gated_scan_desc& d, const Tok& x) {
    return !x.t.buf || (addr(x.t) % 4 == 0 && (d.n_tok <= 1 || x.s_tok % 2 == 0) && (d.n_seq <= 1 || x.s_seq % 2 == 0));
}

int64_t gated_chunks(const helix_gated_scan_desc& d) {
    return ((int64_t)d.n_tok + HELIX_GATED_CHUNK - 1) / HELIX_GATED_CHUNK;
}

}  // namespace

extern "C" void helix_gated_scan_desc_init(helix_gated_scan_desc* d, int32_t n_tok, int32_t n_seq, int32_t n_chan) {
    if (!d) return;
    *d = helix_gated_scan_desc{};
    d->n_tok = n_tok, d->n_seq = n_seq, d->n_chan = n_chan;
    d->io_dtype = HELIX_F32;
    d->s_v = d->s_g = d->s_y = d->s_dy = d->s_dv = d->s_dg = n_chan;
    d->seq_v = d->seq_g = d->seq_y = d->seq_dy = d->seq_dv = d->seq_dg = (int64_t)n_tok * n_chan;
    d->seq_h0 = d->seq_h1 = d->seq_dh1 = d->seq_dh0 = n_chan;
}

extern "C" size_t helix_gated_scan_states_size(const helix_gated_scan_desc* d) {
    if (!d || d->n_tok < 0 || d->n_seq < 0 || d->n_chan < 0) return 0;
    return (size_t)d->n_seq * (size_t)gated_chunks(*d) * (size_t)d->n_chan * sizeof(float);
}

extern "C" helix_status helix_gated_scan_encode(helix_ctx* ctx, void* stream, const helix_gated_scan_desc* d,
                                                helix_tensor v, helix_tensor g, helix_tensor h0,
                                                helix_tensor lengths, helix_tensor y, helix_tensor h1,
                                                helix_tensor states) {
    return entry(ctx, d, [&]() -> int {
        check_gated_desc(*d);
        if (d->n_seq == 0 || d->n_chan == 0) return cudaSuccess;
        need(h1, "h1");
        const Tok tv{"v", v, d->s_v, d->seq_v, false}, tg{"g", g, d->s_g, d->seq_g, false},
            ty{"y", y, d->s_y, d->seq_y, true};
        if (d->n_tok > 0) {
            need(v, "v");
            need(g, "g");
            need(y, "y");
            for (const Tok* t : {&tv, &tg, &ty}) check_tok(*d, *t);
        }
        const bool any = d->n_tok > 0;
        const int64_t ns = d->n_seq, nc = d->n_chan;
        Mat none{"", HELIX_TENSOR_NULL, 0, 0, 0, 1, false};
        const Mat m[] = {any ? mat_of(*d, tv) : none,
                         any ? mat_of(*d, tg) : none,
                         {"h0", h0, ns, nc, d->seq_h0, 4, false},
                         {"lengths", lengths, 1, ns, ns, 4, false},
                         any ? mat_of(*d, ty) : none,
                         {"h1", h1, ns, nc, d->seq_h1, 4, true},
                         {"states", states, 1, ns * gated_chunks(*d) * nc, ns * gated_chunks(*d) * nc, 4, true}};
        const int in_place[][2] = {{5, 2}};
        check_mats(m, in_place);
        hx::GatedParams p{};
        p.n_tok = d->n_tok, p.n_seq = d->n_seq, p.n_chan = d->n_chan;
        p.n_chunk = (int32_t)gated_chunks(*d);
        p.s_v = d->s_v, p.s_g = d->s_g, p.s_y = d->s_y;
        p.seq_v = d->seq_v, p.seq_g = d->seq_g, p.seq_y = d->seq_y;
        p.seq_h0 = d->seq_h0, p.seq_h1 = d->seq_h1;
        p.v = ptr(v), p.g = ptr(g), p.y = ptr(y);
        p.h0 = ptr<float>(h0), p.h1 = ptr<float>(h1), p.states = ptr<float>(states);
        p.lengths = ptr<int32_t>(lengths);
        p.fault = ctx->fault_word;
        return hx::launch_gated(ctx, *d, p, pairs(*d, tv) && pairs(*d, tg) && pairs(*d, ty), stream);
    });
}

extern "C" helix_status helix_gated_scan_grad_encode(helix_ctx* ctx, void* stream, const helix_gated_scan_desc* d,
                                                     helix_tensor dy, helix_tensor v, helix_tensor g,
                                                     helix_tensor states, helix_tensor dh1, helix_tensor lengths,
                                                     helix_tensor dv, helix_tensor dg, helix_tensor dh0) {
    return entry(ctx, d, [&]() -> int {
        check_gated_desc(*d);
        if (d->n_seq == 0 || d->n_chan == 0) return cudaSuccess;
        const Tok tdy{"dy", dy, d->s_dy, d->seq_dy, false}, tv{"v", v, d->s_v, d->seq_v, false},
            tg{"g", g, d->s_g, d->seq_g, false}, tdv{"dv", dv, d->s_dv, d->seq_dv, true},
            tdg{"dg", dg, d->s_dg, d->seq_dg, true};
        const bool any = d->n_tok > 0;
        if (any) {
            need(dy, "dy");
            need(v, "v");
            need(g, "g");
            need(states, "states");
            need(dv, "dv");
            need(dg, "dg");
            for (const Tok* t : {&tdy, &tv, &tg, &tdv, &tdg}) check_tok(*d, *t);
        }
        const int64_t ns = d->n_seq, nc = d->n_chan;
        Mat none{"", HELIX_TENSOR_NULL, 0, 0, 0, 1, false};
        const Mat m[] = {any ? mat_of(*d, tdy) : none,
                         any ? mat_of(*d, tv) : none,
                         any ? mat_of(*d, tg) : none,
                         {"states", states, 1, ns * gated_chunks(*d) * nc, ns * gated_chunks(*d) * nc, 4, false},
                         {"dh1", dh1, ns, nc, d->seq_dh1, 4, false},
                         {"lengths", lengths, 1, ns, ns, 4, false},
                         any ? mat_of(*d, tdv) : none,
                         any ? mat_of(*d, tdg) : none,
                         {"dh0", dh0, ns, nc, d->seq_dh0, 4, true}};
        const int dv_on_dy = any && same_tok(*d, tdv, tdy) ? 6 : -1;
        const int in_place[][2] = {{dv_on_dy, 0}, {8, 4}};
        check_mats(m, in_place);
        hx::GatedParams p{};
        p.n_tok = d->n_tok, p.n_seq = d->n_seq, p.n_chan = d->n_chan;
        p.n_chunk = (int32_t)gated_chunks(*d);
        p.s_v = d->s_v, p.s_g = d->s_g, p.s_dy = d->s_dy, p.s_dv = d->s_dv, p.s_dg = d->s_dg;
        p.seq_v = d->seq_v, p.seq_g = d->seq_g, p.seq_dy = d->seq_dy, p.seq_dv = d->seq_dv, p.seq_dg = d->seq_dg;
        p.seq_dh1 = d->seq_dh1, p.seq_dh0 = d->seq_dh0;
        p.v = ptr(v), p.g = ptr(g), p.dy = ptr(dy), p.dv = ptr(dv), p.dg = ptr(dg);
        p.dh1 = ptr<float>(dh1), p.dh0 = ptr<float>(dh0), p.states = ptr<float>(states);
        p.lengths = ptr<int32_t>(lengths);
        p.fault = ctx->fault_word;
        if (!any && !dh0.buf) return cudaSuccess;
        const bool vec = pairs(*d, tdy) && pairs(*d, tv) && pairs(*d, tg) && pairs(*d, tdv) && pairs(*d, tdg);
        return hx::launch_gated_grad(ctx, *d, p, vec, stream);
    });
}
