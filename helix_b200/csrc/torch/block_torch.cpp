// block_torch.cpp -- the block operators (helix_block.h) for torch tensors:
// the extension module helix_b200._block_torch behind helix_b200/block.py.
//
// Each function checks its tensors, allocates the outputs and the scratch with
// torch's allocator and makes one call of the C ABI on torch's current stream.
// There is no compute here.  It is compiled because a step of a decoder costs
// a few microseconds on the GPU, and the same checks and allocations cost 12
// to 18 from Python through ctypes.
//
// Arguments are positional (block.py has the names and defaults); the first
// is the helix_ctx as an integer.
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <optional>
#include <stdexcept>
#include <string>

#include "helix/helix_block.h"

namespace {

using at::ScalarType;
using at::Tensor;

// Errors by the Python exception they become.
struct Value : std::runtime_error {
    using std::runtime_error::runtime_error;
};
struct Type : std::runtime_error {
    using std::runtime_error::runtime_error;
};
struct Set {};  // the Python error is set already

std::string str(at::IntArrayRef s) {
    std::string out = "(";
    for (size_t i = 0; i < s.size(); ++i) out += (i ? ", " : "") + std::to_string(s[i]);
    return out + ")";
}

// --- arguments -------------------------------------------------------------
struct Args {
    PyObject* const* at;
    helix_ctx*       ctx;
    int              device = -1;

    Args(PyObject* const* a, Py_ssize_t n, Py_ssize_t want) : at(a) {
        if (n != want) throw Type("wrong number of arguments");
        ctx = static_cast<helix_ctx*>(PyLong_AsVoidPtr(a[0]));
        if (PyErr_Occurred()) throw Set{};
    }
    // Tensor i; all of a call's are on one CUDA device.
    const Tensor& tensor(int i, const char* name) {
        if (!THPVariable_Check(at[i])) throw Type(std::string(name) + " must be a tensor");
        const Tensor& t = THPVariable_Unpack(at[i]);
        if (!t.is_cuda()) throw Value("tensors must be on a CUDA device");
        if (device < 0)
            device = t.get_device();
        else if (t.get_device() != device)
            throw Value("tensors are on different devices");
        return t;
    }
    const Tensor* maybe(int i, const char* name) { return at[i] == Py_None ? nullptr : &tensor(i, name); }
    bool flag(int i) const {
        const int v = PyObject_IsTrue(at[i]);
        if (v < 0) throw Set{};
        return v != 0;
    }
    double number(int i) const {
        const double v = PyFloat_AsDouble(at[i]);
        if (v == -1.0 && PyErr_Occurred()) throw Set{};
        return v;
    }
    std::optional<ScalarType> dtype(int i, const char* name) const {
        if (at[i] == Py_None) return std::nullopt;
        if (!THPDtype_Check(at[i])) throw Type(std::string(name) + " must be a torch.dtype");
        return reinterpret_cast<THPDtype*>(at[i])->scalar_type;
    }
    void* stream() const { return c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream(); }

    void check(helix_status st) const {
        if (st == HELIX_OK) return;
        PyObject* mod = PyImport_ImportModule("helix_b200");
        PyObject* cls = mod ? PyObject_GetAttrString(mod, "HelixError") : nullptr;
        PyObject* err = cls ? PyObject_CallFunction(cls, "is", (int)st, helix_ctx_last_error(ctx)) : nullptr;
        if (err) PyErr_SetObject(cls, err);
        Py_XDECREF(err);
        Py_XDECREF(cls);
        Py_XDECREF(mod);
        throw Set{};
    }
};

helix_dtype io_type(const char* name, ScalarType t, bool also8 = false) {
    if (t == at::kFloat) return HELIX_F32;
    if (t == at::kBFloat16) return HELIX_BF16;
    if (also8 && t == at::kFloat8_e4m3fn) return HELIX_E4M3;
    throw Type(std::string(name) + ": " + c10::toString(t) + " is not supported");
}

helix_tensor arg(const Tensor& t) { return helix_tensor{t.data_ptr(), 0}; }
helix_tensor arg(const Tensor* t) { return t ? arg(*t) : helix_tensor{nullptr, 0}; }

void same_shape(const char* name, const Tensor& t, at::IntArrayRef want) {
    if (t.sizes() != want)
        throw Value(std::string(name) + " has shape " + str(t.sizes()) + ", expected " + str(want));
}

// Row stride of t seen as rows of its last dimension.
int64_t pitch(const char* name, const Tensor& t) {
    const auto size = t.sizes(), stride = t.strides();
    const int64_t n = t.dim();
    if (n < 1) throw Value(std::string(name) + " needs a dimension");
    if (t.is_contiguous()) return size[n - 1];
    if (size[n - 1] > 1 && stride[n - 1] != 1)
        throw Value(std::string(name) + " needs unit stride along its last dimension");
    int64_t rows = -1, next = 0;  // the innermost leading dimension that counts, and what the next one's stride must be
    for (int64_t i = n - 2; i >= 0; --i) {
        if (size[i] == 1) continue;
        if (rows < 0)
            rows = stride[i];
        else if (stride[i] != next)
            throw Value(std::string(name) + ": rows must be equally far apart");
        next = stride[i] * size[i];
    }
    return rows < 0 ? size[n - 1] : rows;
}
int64_t pitch(const char* name, const Tensor& t, at::IntArrayRef want) {
    same_shape(name, t, want);
    return pitch(name, t);
}
int64_t rows_of(const Tensor& t) {
    const int64_t c = t.size(-1);
    return c ? t.numel() / c : 0;
}
void vector(const char* name, const Tensor& t, int64_t n) {
    if (t.dim() != 1 || t.size(0) != n || !t.is_contiguous())
        throw Value(std::string(name) + " must be a dense vector of " + std::to_string(n));
}
void of_type(const char* name, const Tensor& t, ScalarType want) {
    if (t.scalar_type() != want) throw Type(std::string(name) + " must be " + c10::toString(want));
}
int32_t narrow(const char* name, int64_t v) {
    if (v > INT32_MAX) throw Value(std::string(name) + " is too large");
    return (int32_t)v;
}

Tensor make(const Tensor& like, at::IntArrayRef size, ScalarType t) {
    return at::detail::empty_cuda(size, t, like.device(), std::nullopt);
}
int64_t groups(int64_t n) { return (n + HELIX_GROUP - 1) / HELIX_GROUP; }
int64_t whole16(int64_t n) { return (n + 15) / 16 * 16; }

using Shape = c10::SmallVector<int64_t, 4>;
Shape with_last(at::IntArrayRef size, int64_t last) {
    Shape s(size.begin(), size.end());
    s.back() = last;
    return s;
}
// 8-bit tensor whose rows start at multiples of 16 bytes.
Tensor make8(const Tensor& like, at::IntArrayRef size) {
    const int64_t cols = size.back();
    Tensor held = make(like, with_last(size, whole16(cols)), at::kFloat8_e4m3fn);
    return cols % 16 == 0 ? held : held.narrow(-1, 0, cols);
}

PyObject* wrap(const Tensor* t) {
    if (!t || !t->defined()) Py_RETURN_NONE;
    return THPVariable_Wrap(*t);
}
template <typename... T>
PyObject* tuple_of(const T&... t) {
    PyObject* out = PyTuple_New(sizeof...(t));
    if (!out) throw Set{};
    Py_ssize_t i = 0;
    bool ok = true;
    for (PyObject* o : {wrap(&t)...}) {
        ok = ok && o;
        PyTuple_SET_ITEM(out, i++, o);
    }
    if (!ok) {
        Py_DECREF(out);
        throw Set{};
    }
    return out;
}

template <typename F>
PyObject* guarded(F body) {
    try {
        return body();
    } catch (const Set&) {
    } catch (const Value& e) {
        PyErr_SetString(PyExc_ValueError, e.what());
    } catch (const Type& e) {
        PyErr_SetString(PyExc_TypeError, e.what());
    } catch (const c10::OutOfMemoryError& e) {
        PyObject* mod = PyImport_ImportModule("torch");
        PyObject* cls = mod ? PyObject_GetAttrString(mod, "OutOfMemoryError") : nullptr;
        if (cls) PyErr_SetString(cls, e.what_without_backtrace());
        Py_XDECREF(cls);
        Py_XDECREF(mod);
    } catch (const c10::Error& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    }
    return nullptr;
}

// --- norm ------------------------------------------------------------------
// (ctx, x, weight, residual, eps, out_dtype, keep_rstd) -> (out, scale, sum, rstd)
PyObject* rms_norm(PyObject*, PyObject* const* argv, Py_ssize_t n) {
    return guarded([&] {
        Args a(argv, n, 7);
        const Tensor& x = a.tensor(1, "x");
        const Tensor& w = a.tensor(2, "weight");
        const Tensor* res = a.maybe(3, "residual");
        const auto size = x.sizes();
        helix_rms_norm_desc d{};
        d.ld_x = pitch("x", x);
        const int64_t cols = size.back();
        d.n_row = rows_of(x);
        d.n_col = narrow("x", cols);
        d.eps = (float)a.number(4);
        d.x_dtype = d.sum_dtype = io_type("x", x.scalar_type());
        if (res) {
            d.sum_dtype = io_type("residual", res->scalar_type());
            d.ld_res = pitch("residual", *res, size);
        }
        vector("weight", w, cols);
        d.w_dtype = io_type("weight", w.scalar_type());
        const ScalarType to = a.dtype(5, "out_dtype").value_or(x.scalar_type());
        d.out_dtype = io_type("out_dtype", to, true);
        Tensor out, scale, sum, rstd;
        d.ld_sum = cols;
        d.ld_scale = groups(cols);
        if (d.out_dtype == HELIX_E4M3) {
            out = make8(x, size);
            scale = make(x, with_last(size, d.ld_scale), at::kFloat);
            d.ld_out = whole16(cols);
        } else {
            out = make(x, size, to);
            d.ld_out = cols;
        }
        if (res) sum = make(x, size, res->scalar_type());
        if (a.flag(6)) rstd = make(x, size.slice(0, size.size() - 1), at::kFloat);
        a.check(helix_rms_norm_encode(a.ctx, a.stream(), &d, arg(x), arg(res), arg(w), arg(out),
                                      scale.defined() ? arg(scale) : arg(nullptr), res ? arg(sum) : arg(nullptr),
                                      rstd.defined() ? arg(rstd) : arg(nullptr)));
        return tuple_of(out, scale, res ? sum : x, rstd);
    });
}

// (ctx, dout, sum, rstd, weight, dsum, keep_dres) -> (dx, dweight, dres)
PyObject* rms_norm_grad(PyObject*, PyObject* const* argv, Py_ssize_t n) {
    return guarded([&] {
        Args a(argv, n, 7);
        const Tensor& dout = a.tensor(1, "dout");
        const Tensor& sum = a.tensor(2, "sum");
        const Tensor& rstd = a.tensor(3, "rstd");
        const Tensor& w = a.tensor(4, "weight");
        const Tensor* dsum = a.maybe(5, "dsum");
        const auto size = dout.sizes();
        helix_rms_norm_desc d{};
        d.ld_dout = pitch("dout", dout);
        const int64_t cols = size.back();
        d.n_row = rows_of(dout);
        d.n_col = narrow("dout", cols);
        d.x_dtype = d.out_dtype = io_type("dout", dout.scalar_type());
        d.sum_dtype = io_type("sum", sum.scalar_type());
        d.ld_sum = pitch("sum", sum, size);
        if (dsum) {
            of_type("dsum", *dsum, sum.scalar_type());
            d.ld_dsum = pitch("dsum", *dsum, size);
        }
        if (rstd.scalar_type() != at::kFloat || rstd.sizes() != size.slice(0, size.size() - 1) || !rstd.is_contiguous())
            throw Value("rstd must be a dense float32 tensor with one value per row");
        vector("weight", w, cols);
        d.w_dtype = io_type("weight", w.scalar_type());
        d.ld_dx = d.ld_dres = cols;
        const size_t bytes = helix_rms_norm_grad_scratch_size(a.ctx, &d);
        Tensor dx = make(dout, size, dout.scalar_type()), dweight = make(dout, {cols}, at::kFloat), dres, scratch;
        const bool keep = a.flag(6);
        if (keep && d.sum_dtype != d.x_dtype) dres = make(dout, size, sum.scalar_type());
        if (bytes) scratch = make(dout, {(int64_t)bytes}, at::kByte);
        a.check(helix_rms_norm_grad_encode(a.ctx, a.stream(), &d, arg(dout), arg(sum), arg(rstd), arg(w), arg(dsum),
                                           arg(dx), dres.defined() ? arg(dres) : arg(nullptr), arg(dweight),
                                           bytes ? arg(scratch) : arg(nullptr)));
        if (!keep) return tuple_of(dx, dweight);
        return tuple_of(dx, dweight, dres.defined() ? dres : dx);
    });
}

// --- quantiser -------------------------------------------------------------
// (ctx, x, blocks, transpose) -> (q, scale)
PyObject* quantize8(PyObject*, PyObject* const* argv, Py_ssize_t n) {
    return guarded([&] {
        Args a(argv, n, 4);
        const Tensor& x = a.tensor(1, "x");
        if (x.dim() != 2) throw Value("x must be a matrix");
        helix_quant8_desc d{};
        d.n_row = x.size(0), d.n_col = x.size(1);
        d.x_dtype = io_type("x", x.scalar_type());
        d.ld_x = pitch("x", x);
        const bool blocks = a.flag(2);
        d.form = blocks ? HELIX_SCALE_BLOCKS : HELIX_SCALE_ROWS;
        d.transpose = a.flag(3);
        const int64_t rows = d.transpose ? d.n_col : d.n_row, cols = d.transpose ? d.n_row : d.n_col;
        Tensor q = make8(x, {rows, cols});
        Tensor scale = make(x, {blocks ? groups(rows) : rows, groups(cols)}, at::kFloat);
        d.ld_q = whole16(cols);
        d.ld_scale = groups(cols);
        a.check(helix_quant8_encode(a.ctx, a.stream(), &d, arg(x), arg(q), arg(scale)));
        return tuple_of(q, scale);
    });
}

// --- product ---------------------------------------------------------------
// (ctx, a, a_scale, b, b_scale, out_dtype) -> out
PyObject* matmul8(PyObject*, PyObject* const* argv, Py_ssize_t n) {
    return guarded([&] {
        Args a(argv, n, 6);
        const Tensor& x = a.tensor(1, "a");
        const Tensor& sx = a.tensor(2, "a_scale");
        const Tensor& y = a.tensor(3, "b");
        const Tensor& sy = a.tensor(4, "b_scale");
        if (x.scalar_type() != at::kFloat8_e4m3fn || y.scalar_type() != at::kFloat8_e4m3fn)
            throw Type("a and b must be torch.float8_e4m3fn");
        if (sx.scalar_type() != at::kFloat || sy.scalar_type() != at::kFloat)
            throw Type("scales must be torch.float32");
        if (y.dim() != 2 || x.dim() < 1 || x.size(-1) != y.size(1))
            throw Value("b must be a matrix with as many columns as a");
        const auto size = x.sizes();
        const int64_t cols = y.size(0), k = y.size(1), g = groups(k);
        helix_matmul8_desc d{};
        d.m = narrow("a", rows_of(x)), d.n = narrow("b", cols), d.k = narrow("a", k);
        const bool rows = sy.dim() == 2 && sy.size(0) == cols && sy.size(1) == g;
        d.b_form = rows ? HELIX_SCALE_ROWS : HELIX_SCALE_BLOCKS;
        const ScalarType to = a.dtype(5, "out_dtype").value_or(at::kBFloat16);
        d.out_dtype = io_type("out_dtype", to);
        d.ld_a = pitch("a", x), d.ld_b = pitch("b", y);
        d.ld_a_scale = pitch("a_scale", sx, with_last(size, g));
        d.ld_b_scale = pitch("b_scale", sy, {rows ? cols : groups(cols), g});
        d.ld_out = cols;
        Tensor out = make(x, with_last(size, cols), to);
        a.check(helix_matmul8_encode(a.ctx, a.stream(), &d, arg(x), arg(sx), arg(y), arg(sy), arg(out)));
        return wrap(&out);
    });
}

// --- gated recurrence ------------------------------------------------------
// Token and sequence stride of a (sequences, tokens, channels) tensor.
void token_strides(const char* name, const Tensor& t, const Tensor& v, int64_t* tok, int64_t* seq) {
    same_shape(name, t, v.sizes());
    of_type(name, t, v.scalar_type());
    if (t.size(2) > 1 && t.stride(2) != 1) throw Value(std::string(name) + " needs unit stride along the channels");
    *tok = t.stride(1);
    *seq = t.stride(0);
}
int64_t state_pitch(const char* name, const Tensor& t, at::IntArrayRef want) {
    of_type(name, t, at::kFloat);
    return pitch(name, t, want);
}
void lengths_of(const Tensor* t, int64_t seqs) {
    if (!t) return;
    vector("lengths", *t, seqs);
    of_type("lengths", *t, at::kInt);
}
helix_gated_scan_desc gated_desc(const Tensor& v) {
    if (v.dim() != 3) throw Value("v must be (sequences, tokens, channels)");
    helix_gated_scan_desc d{};
    d.n_seq = narrow("v", v.size(0)), d.n_tok = narrow("v", v.size(1)), d.n_chan = narrow("v", v.size(2));
    d.io_dtype = io_type("v", v.scalar_type());
    return d;
}
int64_t chunks(int64_t n) { return (n + HELIX_GATED_CHUNK - 1) / HELIX_GATED_CHUNK; }

// (ctx, v, g, h0, lengths, h1, keep_states) -> (y, h1[, states])
PyObject* gated_scan(PyObject*, PyObject* const* argv, Py_ssize_t n) {
    return guarded([&] {
        Args a(argv, n, 7);
        const Tensor& v = a.tensor(1, "v");
        const Tensor& g = a.tensor(2, "g");
        const Tensor* h0 = a.maybe(3, "h0");
        const Tensor* len = a.maybe(4, "lengths");
        const Tensor* into = a.maybe(5, "h1");
        helix_gated_scan_desc d = gated_desc(v);
        const int64_t S = d.n_seq, L = d.n_tok, C = d.n_chan;
        token_strides("v", v, v, &d.s_v, &d.seq_v);
        token_strides("g", g, v, &d.s_g, &d.seq_g);
        lengths_of(len, S);
        if (h0) d.seq_h0 = state_pitch("h0", *h0, {S, C});
        d.seq_h1 = into ? state_pitch("h1", *into, {S, C}) : C;
        Tensor y = make(v, v.sizes(), v.scalar_type()), states;
        Tensor h1 = into ? *into : make(v, {S, C}, at::kFloat);
        const bool keep = a.flag(6);
        if (keep) states = make(v, {S, chunks(L), C}, at::kFloat);
        d.s_y = C, d.seq_y = L * C;
        a.check(helix_gated_scan_encode(a.ctx, a.stream(), &d, arg(v), arg(g), arg(h0), arg(len), arg(y), arg(h1),
                                        keep ? arg(states) : arg(nullptr)));
        return keep ? tuple_of(y, h1, states) : tuple_of(y, h1);
    });
}

// (ctx, dy, v, g, states, dh1, lengths, dv, dg) -> (dv, dg, dh0)
PyObject* gated_scan_grad(PyObject*, PyObject* const* argv, Py_ssize_t n) {
    return guarded([&] {
        Args a(argv, n, 9);
        const Tensor& dy = a.tensor(1, "dy");
        const Tensor& v = a.tensor(2, "v");
        const Tensor& g = a.tensor(3, "g");
        const Tensor& states = a.tensor(4, "states");
        const Tensor* dh1 = a.maybe(5, "dh1");
        const Tensor* len = a.maybe(6, "lengths");
        const Tensor* into_v = a.maybe(7, "dv");
        const Tensor* into_g = a.maybe(8, "dg");
        helix_gated_scan_desc d = gated_desc(v);
        const int64_t S = d.n_seq, L = d.n_tok, C = d.n_chan;
        token_strides("v", v, v, &d.s_v, &d.seq_v);
        token_strides("g", g, v, &d.s_g, &d.seq_g);
        token_strides("dy", dy, v, &d.s_dy, &d.seq_dy);
        if (states.scalar_type() != at::kFloat || !states.is_contiguous() || states.dim() != 3 || states.size(0) != S ||
            states.size(1) != chunks(L) || states.size(2) != C)
            throw Value("states must be what gated_scan(keep_states=True) gave");
        lengths_of(len, S);
        if (dh1) d.seq_dh1 = state_pitch("dh1", *dh1, {S, C});
        if (into_v) token_strides("dv", *into_v, v, &d.s_dv, &d.seq_dv);
        if (into_g) token_strides("dg", *into_g, v, &d.s_dg, &d.seq_dg);
        Tensor dv = into_v ? *into_v : make(v, v.sizes(), v.scalar_type());
        Tensor dg = into_g ? *into_g : make(v, v.sizes(), v.scalar_type());
        Tensor dh0 = make(v, {S, C}, at::kFloat);
        if (!into_v) d.s_dv = C, d.seq_dv = L * C;
        if (!into_g) d.s_dg = C, d.seq_dg = L * C;
        d.seq_dh0 = C;
        a.check(helix_gated_scan_grad_encode(a.ctx, a.stream(), &d, arg(dy), arg(v), arg(g), arg(states), arg(dh1),
                                             arg(len), arg(dv), arg(dg), arg(dh0)));
        return tuple_of(dv, dg, dh0);
    });
}

#define FAST(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef kMethods[] = {FAST(rms_norm), FAST(rms_norm_grad),   FAST(quantize8),        FAST(matmul8),
                          FAST(gated_scan), FAST(gated_scan_grad), {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_block_torch", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__block_torch() { return PyModule_Create(&kModule); }
