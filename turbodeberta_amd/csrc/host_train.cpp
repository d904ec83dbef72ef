// Native front of the training operators (include/tdb_train.h): CPython functions that take the operators' arguments as they are, check the well-formed case, and record a node
// of autograd whose backward pass is native too.  A small call is bound by the host: ctypes, the Python checks and torch.autograd.Function took 92 us for a forward and a backward
// pass of dropout over 29 x 768 values, where the two kernels take 5.  Anything out of the ordinary returns None, as in host.cpp, and the caller takes the Python path.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/core/GradMode.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <cstring>

#include "host.h"
#include "tdb_train.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct {
    decltype(&tdb_dropout) dropout;
    decltype(&tdb_norm_fwd) norm_fwd;
    decltype(&tdb_norm_bwd) norm_bwd;
    decltype(&tdb_norm_workspace) norm_workspace;
    decltype(&tdb_attn_train_fwd) attn_fwd;
    decltype(&tdb_attn_train_bwd) attn_bwd;
    decltype(&tdb_attn_train_workspace) attn_workspace;
    decltype(&tdb_last_error) last_error;
} g;

// A forward call that the C ABI refuses: the Python path repeats it and raises the message.
struct Refused {};
void forward_ok(int rc) {
    if (rc != TDB_OK) throw Refused();
}
void backward_ok(int rc) { TORCH_CHECK(rc == TDB_OK, g.last_error()); }

void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
int dtype_code(const Tensor& t) {
    const auto s = t.scalar_type();
    return s == at::kFloat ? TDB_F32 : s == at::kBFloat16 ? TDB_BF16 : s == at::kHalf ? TDB_F16 : -1;
}
Tensor empty(at::IntArrayRef sizes, at::ScalarType type, const Tensor& like) { return at::detail::empty_cuda(sizes, type, like.device(), std::nullopt); }
Tensor empty(at::IntArrayRef sizes, const Tensor& like) { return empty(sizes, like.scalar_type(), like); }
// Arguments of a node that may be absent.
using Optional = std::optional<Tensor>;
Optional optional(const Tensor& t) { return t.defined() ? Optional(t) : std::nullopt; }
Tensor plain(const Optional& t) { return t.value_or(Tensor()); }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// Whether the node whose backward pass runs hands a gradient to a leaf whose accumulation belongs to another stream: that of the first graph of the leaf that still lives.
bool tied_to_another_stream() {
    const auto node = torch::autograd::get_current_node();
    if (!node) return false;
    for (const auto& edge : node->next_edges()) {
        if (!dynamic_cast<torch::autograd::AccumulateGrad*>(edge.function.get())) continue;
        const auto stream = edge.function->stream();
        if (stream && stream->id() != c10::hip::getCurrentHIPStream(stream->device_index()).id()) return true;
    }
    return false;
}
// Under capture autograd's engine would wait across the two streams, and the process ends.
void capturable() {
    if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
    TORCH_CHECK(!tied_to_another_stream(), "a backward pass cannot be captured while a graph of autograd's that was recorded on another stream holds the same leaves: drop its results first");
}

// The gradient that arrives has to be a tensor of the device's memory, with no transform around it.
void arrived(const Tensor& dy, const Tensor& x) {
    TORCH_CHECK(tdb_host_plain(dy, x, false), "the gradient must be an ordinary tensor on ", x.device());
    capturable();
}

// Results of a backward pass, which is not differentiable itself: asked for a second gradient they raise.
variable_list once(variable_list grads) {
    if (!c10::GradMode::is_enabled()) return grads;
    variable_list some;
    for (const Tensor& t : grads)
        if (t.defined()) some.push_back(t.detach().requires_grad_(true));
    const auto raises = std::make_shared<torch::autograd::DelayedError>("trying to differentiate twice an operator that is differentiable once", int64_t(some.size()));
    variable_list out = (*raises)(std::move(some));
    size_t n = 0;
    for (Tensor& t : grads)
        if (t.defined()) t = out[n++];
    return grads;
}

// ---------------------------------------------------------------------------------------------------------------- dropout

Tensor drop(const Tensor& x, int64_t threshold, const Tensor& seed, int& rc) {
    const Tensor from = x.contiguous();
    Tensor y = empty(x.sizes(), x);
    rc = g.dropout(from.data_ptr(), y.data_ptr(), x.numel(), dtype_code(x), int32_t(threshold), static_cast<const int64_t*>(seed.data_ptr()), stream_of(x));
    return y;
}

struct Dropout : torch::autograd::Function<Dropout> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& seed, int64_t threshold) {
        int rc;
        Tensor y = drop(x, threshold, seed, rc);
        forward_ok(rc);
        ctx->save_for_backward({seed});
        ctx->saved_data["threshold"] = threshold;
        return y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list dy) {
        const Tensor seed = ctx->get_saved_variables()[0];
        arrived(dy[0], seed);
        variable_list out(3);
        {
            const at::NoGradGuard off;
            int rc;
            out[0] = drop(dy[0], ctx->saved_data["threshold"].toInt(), seed, rc);
            backward_ok(rc);
        }
        return once(std::move(out));
    }
};

// -------------------------------------------------------------------------------------------------------------------- norm

// t as rows of `hidden` values side by side, `stride` apart: t itself where it lies so
Tensor as_rows(const Tensor& t, int64_t hidden, int64_t& stride) {
    if (t.is_contiguous()) {
        stride = hidden;
        return t;
    }
    Tensor rows = t.reshape({-1, hidden});
    if (hidden > 1 && rows.stride(1) != 1) rows = rows.contiguous();
    stride = rows.stride(0);
    return rows;
}

struct NormCall {
    tdb_norm_args a;
    Tensor x, residual, weight, bias;
    NormCall(const Tensor& of_x, const Tensor& of_residual, const Tensor& of_weight, const Tensor& of_bias, const Tensor& seed, int64_t threshold, double eps) {
        memset(&a, 0, sizeof(a));
        const int64_t hidden = of_x.size(-1);
        a.dtype = dtype_code(of_x), a.hidden = int32_t(hidden), a.threshold = int32_t(threshold), a.rows = of_x.numel() / hidden, a.eps = float(eps);
        x = as_rows(of_x, hidden, a.x_stride);
        if (of_residual.defined()) residual = as_rows(of_residual, hidden, a.residual_stride);
        if (of_weight.defined()) weight = of_weight.contiguous(), bias = of_bias.contiguous();
        a.weight_dtype = weight.defined() ? dtype_code(weight) : a.dtype;
        a.x = ptr(x), a.residual = ptr(residual), a.weight = ptr(weight), a.bias = ptr(bias), a.seed = static_cast<const int64_t*>(ptr(seed));
        a.y_stride = a.dx_stride = a.dresidual_stride = hidden;
    }
};

struct Norm : torch::autograd::Function<Norm> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Optional& of_residual, const Optional& of_weight, const Optional& of_bias, const Optional& of_seed, int64_t threshold,
                          double eps) {
        const Tensor residual = plain(of_residual), weight = plain(of_weight), bias = plain(of_bias), seed = plain(of_seed);
        NormCall c(x, residual, weight, bias, seed, threshold, eps);
        Tensor y = empty(x.sizes(), x);
        c.a.y = y.data_ptr();
        forward_ok(g.norm_fwd(&c.a, stream_of(x)));
        ctx->save_for_backward({x, residual, weight, bias, seed});
        ctx->saved_data["threshold"] = threshold, ctx->saved_data["eps"] = eps;
        return y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &residual = saved[1], &weight = saved[2], &bias = saved[3];
        arrived(grads[0], x);
        variable_list out(7);
        {
            const at::NoGradGuard off;
            NormCall c(x, residual, weight, bias, saved[4], ctx->saved_data["threshold"].toInt(), ctx->saved_data["eps"].toDouble());
            const Tensor dy = as_rows(grads[0], x.size(-1), c.a.dy_stride);
            c.a.dy = dy.data_ptr();
            const int at = residual.defined() ? 2 : 1;          // number of the weight among the tensors that are there
            const bool wants_weight = weight.defined() && ctx->needs_input_grad(at), wants_bias = weight.defined() && ctx->needs_input_grad(at + 1);
            if (ctx->needs_input_grad(0)) out[0] = empty(x.sizes(), x), c.a.dx = out[0].data_ptr();
            if (residual.defined() && ctx->needs_input_grad(1)) out[1] = empty(residual.sizes(), residual), c.a.dresidual = out[1].data_ptr();
            Tensor work;
            if (wants_weight || wants_bias) {
                out[2] = empty(weight.sizes(), weight), out[3] = empty(bias.sizes(), bias);
                work = empty({g.norm_workspace(c.a.rows, c.a.hidden)}, at::kFloat, x);
                c.a.dweight = out[2].data_ptr(), c.a.dbias = out[3].data_ptr(), c.a.workspace = static_cast<float*>(work.data_ptr());
            }
            backward_ok(g.norm_bwd(&c.a, stream_of(x)));
            if (!wants_weight) out[2] = Tensor();
            if (!wants_bias) out[3] = Tensor();
        }
        return once(std::move(out));
    }
};

// --------------------------------------------------------------------------------------------------------------- attention

// Rows that do not share memory and are not too far apart for 32-bit offsets.
bool apart(const Tensor& t) {
    const int64_t row = t.stride(t.dim() == 4 ? 2 : 0);
    return tdb_host_rows_ok(t) && t.size(-1) <= row && row * t.element_size() <= int64_t(1) << 24;
}
Tensor result_like(const Tensor& t) {
    Tensor o;
    return tdb_host_output_like(t, o) && apart(o) ? o : empty(t.sizes(), t);
}

// A table [H, rows, D]: as it is handed in, or without a leading 1.  (Taken off within a node, so that a leaf's accumulation is that node's own edge, which tied_to_another_stream
// looks at.)
Tensor table_of(const Tensor& t) { return t.defined() && t.dim() == 4 ? t.select(0, 0) : t; }

// (batch, head, row) strides of [B, H, L, D], or of packed [T, H, D]
void strides(const Tensor& t, int64_t* to) { to[0] = t.dim() == 4 ? t.stride(0) : 0, to[1] = t.stride(1), to[2] = t.stride(t.dim() == 4 ? 2 : 0); }

struct Attention : torch::autograd::Function<Attention> {
    static tdb_train_attn_args args(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& pk, const Tensor& pq, const Tensor& lens, const Tensor& cu, const Tensor& seed,
                                    const Tensor& lut, int64_t longest, double scale, int64_t span, int64_t threshold) {
        tdb_train_attn_args a;
        memset(&a, 0, sizeof(a));
        a.dtype = dtype_code(q), a.heads = int32_t(q.size(1)), a.head_dim = int32_t(q.size(-1)), a.max_seqlen = int32_t(longest), a.threshold = int32_t(threshold), a.sm_scale = float(scale);
        a.batch = int32_t(cu.defined() ? cu.numel() - 1 : q.size(0)), a.total_tokens = int32_t(cu.defined() ? q.size(0) : 0);
        a.q = q.data_ptr(), a.k = k.data_ptr(), a.v = v.data_ptr();
        strides(q, &a.q_stride_b), strides(k, &a.k_stride_b), strides(v, &a.v_stride_b);
        a.seqlens_k = static_cast<const int32_t*>(ptr(lens)), a.cu_seqlens = static_cast<const int32_t*>(ptr(cu)), a.seed = static_cast<const int64_t*>(ptr(seed));
        if (lut.defined()) a.delta_lut = static_cast<const int32_t*>(lut.data_ptr()), a.lut_half = int32_t(lut.numel() / 2), a.span = int32_t(span);
        if (pk.defined()) a.pos_key = pk.data_ptr(), a.pos_key_stride_h = pk.stride(0), a.pos_key_stride_r = pk.stride(1);
        if (pq.defined()) a.pos_query = pq.data_ptr(), a.pos_query_stride_h = pq.stride(0), a.pos_query_stride_r = pq.stride(1);
        return a;
    }
    static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const Optional& of_pk, const Optional& of_pq, const Optional& of_lens, const Optional& of_cu,
                          const Optional& of_seed, const Optional& of_lut, int64_t longest, double scale, int64_t span, int64_t threshold) {
        const Tensor pk = table_of(plain(of_pk)), pq = table_of(plain(of_pq)), lens = plain(of_lens), cu = plain(of_cu), seed = plain(of_seed), lut = plain(of_lut);
        tdb_train_attn_args a = args(q, k, v, pk, pq, lens, cu, seed, lut, longest, scale, span, threshold);
        Tensor o = result_like(q), rest;
        const int64_t rows = q.numel() / (q.size(1) * q.size(-1));
        const Tensor lse = empty({q.size(1), rows}, at::kFloat, q);
        if (q.scalar_type() != at::kFloat) rest = empty({q.size(1), rows, q.size(-1)}, q);
        a.o = o.data_ptr(), a.lse = static_cast<float*>(lse.data_ptr()), a.o_rest = ptr(rest);
        strides(o, &a.o_stride_b);
        forward_ok(g.attn_fwd(&a, stream_of(q)));
        ctx->save_for_backward({q, k, v, o, rest, lse, plain(of_pk), plain(of_pq), lens, cu, seed, lut});
        ctx->saved_data["longest"] = longest, ctx->saved_data["scale"] = scale, ctx->saved_data["span"] = span, ctx->saved_data["threshold"] = threshold;
        return o;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &q = saved[0], &k = saved[1], &v = saved[2], &o = saved[3], &rest = saved[4], &lse = saved[5];
        arrived(grads[0], q);
        variable_list out(13);
        {
            const at::NoGradGuard off;
            const Tensor pk = table_of(saved[6]), pq = table_of(saved[7]);
            const Tensor dout = apart(grads[0]) ? grads[0] : grads[0].clone(at::MemoryFormat::Contiguous);
            const int64_t span = ctx->saved_data["span"].toInt();
            tdb_train_attn_args a = args(q, k, v, pk, pq, saved[8], saved[9], saved[10], saved[11], ctx->saved_data["longest"].toInt(), ctx->saved_data["scale"].toDouble(), span,
                                         ctx->saved_data["threshold"].toInt());
            out[0] = result_like(q), out[1] = result_like(k), out[2] = result_like(v);
            a.o = o.data_ptr(), a.o_rest = ptr(rest), a.lse = static_cast<float*>(lse.data_ptr()), a.dout = dout.data_ptr();
            a.dq = out[0].data_ptr(), a.dk = out[1].data_ptr(), a.dv = out[2].data_ptr();
            strides(o, &a.o_stride_b), strides(dout, &a.dout_stride_b), strides(out[0], &a.dq_stride_b), strides(out[1], &a.dk_stride_b), strides(out[2], &a.dv_stride_b);
            for (int n = 0; n < 2; ++n) {
                const Tensor& t = n ? pq : pk;
                if (!t.defined()) continue;
                Tensor& d = out[3 + n];
                d = empty(saved[6 + n].sizes(), t);
                if (t.size(1) != 2 * span) d.zero_();       // (rows that no offset has)
                (n ? a.dpos_query : a.dpos_key) = d.data_ptr();
                (n ? a.dpos_query_stride_h : a.dpos_key_stride_h) = t.size(1) * t.size(2);
            }
            a.workspace_bytes = g.attn_workspace(&a);
            const Tensor work = empty({a.workspace_bytes}, at::kByte, q);
            a.workspace = work.data_ptr();
            backward_ok(g.attn_bwd(&a, stream_of(q)));
        }
        return once(std::move(out));
    }
};

// ----------------------------------------------------------------------------------------------------------------- CPython

// One tensor argument, undefined for None; `ok` is cleared for anything but a plain tensor on x's device.
Tensor take(PyObject* o, const Tensor* x, bool& ok) {
    if (o == Py_None) return Tensor();
    if (!THPVariable_CheckExact(o)) {
        ok = false;
        return Tensor();
    }
    const Tensor& t = THPVariable_Unpack(o);
    ok = ok && tdb_host_plain(t, x ? *x : t, false);
    return t;
}
// The tensor whose device decides: on the current one, of a type that the kernels have.
Tensor first(PyObject* o, bool& ok) {
    Tensor t = take(o, nullptr, ok);
    ok = ok && t.defined() && t.is_cuda() && dtype_code(t) >= 0 && t.numel() > 0 && t.device().index() == c10::hip::current_device();
    return t;
}
bool as_double(PyObject* o, double& x) {
    if (PyFloat_CheckExact(o)) x = PyFloat_AS_DOUBLE(o);
    else if (PyLong_CheckExact(o)) x = PyLong_AsDouble(o);
    else return false;
    if (PyErr_Occurred()) {
        PyErr_Clear();
        return false;
    }
    return true;
}
bool as_threshold(PyObject* o, int64_t& threshold) {
    double p;
    if (!as_double(o, p) || !(p >= 0.0 && p <= 1.0)) return false;
    threshold = int64_t(std::nearbyint(65536.0 * p));
    return true;
}
bool as_int(PyObject* o, int64_t& x) {
    if (!PyLong_CheckExact(o)) return false;
    x = PyLong_AsLongLong(o);
    if (x == -1 && PyErr_Occurred()) {
        PyErr_Clear();
        return false;
    }
    return x >= INT32_MIN && x <= INT32_MAX;
}
// The seed of a call that drops anything.
Tensor as_seed(PyObject* o, int64_t threshold, const Tensor& x, bool& ok) {
    if (!ok || threshold == 0) return Tensor();
    Tensor seed = take(o, &x, ok);
    ok = ok && seed.defined() && seed.scalar_type() == at::kLong && seed.numel() == 1;
    return seed;
}

template <class F>
PyObject* native(F call) {
    if (!g.dropout || tdb_host_observed()) Py_RETURN_NONE;
    HANDLE_TH_ERRORS                    // (what hooks of saved tensors raise passes through as it is)
    try {
        Tensor out = call();
        if (!out.defined()) Py_RETURN_NONE;
        return THPVariable_Wrap(std::move(out));
    } catch (const Refused&) {
        Py_RETURN_NONE;
    }
    END_HANDLE_TH_ERRORS
}

// train_dropout(x, p, seed)
PyObject* py_dropout(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    if (nargs != 3) Py_RETURN_NONE;
    return native([&]() -> Tensor {
        bool ok = true;
        int64_t threshold;
        const Tensor x = first(args[0], ok);
        if (!ok || !as_threshold(args[1], threshold) || threshold == 0) return Tensor();
        const Tensor seed = as_seed(args[2], threshold, x, ok);
        return ok ? Dropout::apply(x, seed, threshold) : Tensor();
    });
}

// train_norm(x, residual, weight, bias, p, seed, eps)
PyObject* py_norm(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    if (nargs != 7) Py_RETURN_NONE;
    return native([&]() -> Tensor {
        bool ok = true;
        int64_t threshold;
        double eps;
        const Tensor x = first(args[0], ok);
        if (!ok || !as_threshold(args[4], threshold) || !as_double(args[6], eps) || !(eps >= 0.0) || x.dim() < 1 || x.size(-1) > 32768) return Tensor();
        const Tensor residual = take(args[1], &x, ok), weight = take(args[2], &x, ok), bias = take(args[3], &x, ok), seed = as_seed(args[5], threshold, x, ok);
        if (!ok || (residual.defined() && (residual.sizes() != x.sizes() || residual.scalar_type() != x.scalar_type())) || weight.defined() != bias.defined()) return Tensor();
        if (weight.defined() && (weight.dim() != 1 || weight.size(0) != x.size(-1) || bias.sizes() != weight.sizes() || weight.scalar_type() != bias.scalar_type() ||
                                 (weight.scalar_type() != x.scalar_type() && weight.scalar_type() != at::kFloat)))
            return Tensor();
        return Norm::apply(x, optional(residual), optional(weight), optional(bias), optional(seed), threshold, eps);
    });
}

// train_attention(q, k, v, pos_key_layer, pos_query_layer, sm_scale, position_buckets, max_relative_distance, seqlens_k, cu_seqlens, max_seqlen, p, seed)
PyObject* py_attention(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    if (nargs != 13) Py_RETURN_NONE;
    return native([&]() -> Tensor {
        bool ok = true;
        int64_t buckets, max_rel, threshold, longest = 0;
        double scale;
        const Tensor q = first(args[0], ok);
        if (!ok || !as_int(args[6], buckets) || !as_int(args[7], max_rel) || !as_threshold(args[11], threshold)) return Tensor();
        const Tensor k = take(args[1], &q, ok), v = take(args[2], &q, ok), lens = take(args[8], &q, ok), cu = take(args[9], &q, ok), seed = as_seed(args[12], threshold, q, ok);
        const Tensor pk = take(args[3], &q, ok), pq = take(args[4], &q, ok);
        const int64_t dims = cu.defined() ? 3 : 4;
        if (!ok || !k.defined() || !v.defined() || q.dim() != dims || k.sizes() != q.sizes() || v.sizes() != q.sizes() || k.scalar_type() != q.scalar_type() ||
            v.scalar_type() != q.scalar_type() || !apart(q) || !apart(k) || !apart(v))
            return Tensor();
        const int64_t heads = q.size(1), D = q.size(-1);
        if (D % 8 || D < 8 || D > 64 || q.size(0) > INT32_MAX) return Tensor();
        if (args[5] == Py_None) scale = 1.0 / std::sqrt(double(D));
        else if (!as_double(args[5], scale)) return Tensor();
        if (!(scale > 0.0 && scale < 1e30)) return Tensor();
        for (const Tensor* t : {&lens, &cu})
            if (t->defined() && (t->dim() != 1 || t->scalar_type() != at::kInt || !t->is_contiguous())) return Tensor();
        if (cu.defined()) {
            if (cu.numel() < 2 || !as_int(args[10], longest)) return Tensor();
            longest = std::max<int64_t>(longest, 1);
        } else {
            longest = q.size(2);
            if (longest > INT32_MAX || (lens.defined() && lens.numel() != q.size(0))) return Tensor();
        }
        Tensor lut;
        const int64_t span = buckets > 0 ? buckets : max_rel;
        if (pk.defined() || pq.defined()) {
            const Tensor* table = span < 1 ? nullptr : tdb_host_lut(buckets, max_rel, longest, cu.defined() ? std::min(longest, q.size(0)) : longest, q.device().index());
            if (!table) return Tensor();
            lut = *table;
        }
        for (const Tensor* t : {&pk, &pq}) {
            if (!t->defined()) continue;
            const int64_t at = t->dim() - 3;
            if (!(at == 0 || (at == 1 && t->size(0) == 1)) || t->size(at) != heads || t->size(at + 1) < 2 * span || t->size(at + 2) != D || t->scalar_type() != q.scalar_type() ||
                !tdb_host_rows_ok(*t))
                return Tensor();
        }
        return Attention::apply(q, k, v, optional(pk), optional(pq), optional(lens), optional(cu), optional(seed), optional(lut), longest, scale, span, threshold);
    });
}

// bind_train(addresses of the entry points of tdb_train.h in its order, address of tdb_last_error)
PyObject* py_bind_train(PyObject*, PyObject* args) {
    unsigned long long at[8];
    if (!PyArg_ParseTuple(args, "KKKKKKKK", at, at + 1, at + 2, at + 3, at + 4, at + 5, at + 6, at + 7)) return nullptr;
    static_assert(sizeof(g) == sizeof(at), "");
    memcpy(&g, at, sizeof(g));
    Py_RETURN_NONE;
}

// backward_begins(): what the Python path's backward passes ask first, see capturable; returns what it looks at
PyObject* py_backward_begins(PyObject*, PyObject*) {
    HANDLE_TH_ERRORS
    capturable();
    return PyBool_FromLong(tied_to_another_stream());
    END_HANDLE_TH_ERRORS
}

PyMethodDef kTrain[] = {
    {"backward_begins", py_backward_begins, METH_NOARGS, nullptr},
    {"bind_train", py_bind_train, METH_VARARGS, nullptr},
    {"train_dropout", reinterpret_cast<PyCFunction>(py_dropout), METH_FASTCALL, nullptr},
    {"train_norm", reinterpret_cast<PyCFunction>(py_norm), METH_FASTCALL, nullptr},
    {"train_attention", reinterpret_cast<PyCFunction>(py_attention), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};

}  // namespace

bool tdb_host_add_train(PyObject* module) { return PyModule_AddFunctions(module, kTrain) == 0; }
