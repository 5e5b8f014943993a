// block.cpp -- entry points of the recurrent block's operators
// (helix_block.h): checks of arguments, plans, launches on the caller's
// stream.  Nothing here synchronises or allocates device memory, and no C++
// exception leaves an entry point.
#include "block_internal.h"

#include <cuda_runtime.h>

#include <climits>
#include <cstdlib>
#include <string>

namespace {

struct DeviceScope {
    int prev = -1;
    explicit DeviceScope(int dev) {
        if (cudaGetDevice(&prev) != cudaSuccess) prev = -1;
        if (prev != dev) cudaSetDevice(dev);
    }
    ~DeviceScope() {
        int cur = -1;
        if (prev >= 0 && cudaGetDevice(&cur) == cudaSuccess && cur != prev) cudaSetDevice(prev);
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

// A matrix argument of a call: `rows` rows of `cols` elements, `ld` apart.
struct Mat {
    const char*  name;
    helix_tensor t;
    int64_t      rows, cols, ld, size;
    bool         written;
};

void check_mat(const Mat& m) {
    if (!m.t.buf) return;
    const std::string n = m.name;
    if (addr(m.t) % (uintptr_t)m.size) invalid(n + " is not aligned to its elements");
    if (m.ld < 0 || (m.written && m.rows > 1 && m.ld < m.cols)) invalid(n + ": row stride too small");
    const int64_t most = INT64_MAX / 16;
    if (m.rows > 1 && m.ld > 0 && (m.rows - 1) > most / m.ld) invalid(n + ": rows reach past 64-bit offsets");
}

// Whether two matrices share bytes.  Matrices with one row pitch may lie
// side by side in it (slices of one wider matrix).
bool overlap(const Mat& a, const Mat& b) {
    if (!a.t.buf || !b.t.buf || !a.rows || !b.rows || !a.cols || !b.cols) return false;
    const uintptr_t a0 = addr(a.t), b0 = addr(b.t);
    const uintptr_t a1 = a0 + (uintptr_t)(((a.rows - 1) * a.ld + a.cols) * a.size);
    const uintptr_t b1 = b0 + (uintptr_t)(((b.rows - 1) * b.ld + b.cols) * b.size);
    if (a1 <= b0 || b1 <= a0) return false;
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
        return hx::launch_norm(*d, p, vec, stream);
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
        p.wpr = pl.shape.wpr;
        p.rpb = pl.shape.rpb;
        p.w_bf16 = d->w_dtype == HELIX_BF16;
        p.ld_dout = d->ld_dout, p.ld_sum = d->ld_sum, p.ld_dsum = d->ld_dsum, p.ld_dx = d->ld_dx, p.ld_dres = d->ld_dres;
        p.dout = ptr(dout), p.sum = ptr(sum), p.dsum = ptr(dsum), p.w = ptr(weight);
        p.dx = ptr(dx), p.dres = ptr(dres), p.rstd = ptr<float>(rstd);
        p.partial = ptr<float>(scratch);
        const bool vec = whole(m[0], 16) && whole(m[1], 16) && whole(m[3], 16) && whole(m[4], 16) &&
                         whole(m[5], 16) && whole(m[6], 16);
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
        return hx::launch_quant(*d, p, whole(m[0], 16) && whole(m[1], 8), stream);
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
        const hx::Mm8Operand oa{ptr<float>(a_scale), d->ld_a_scale, d->m, 1};
        const hx::Mm8Operand ob{ptr<float>(b_scale), d->ld_b_scale, d->n, blocks ? HELIX_GROUP : 1};
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
