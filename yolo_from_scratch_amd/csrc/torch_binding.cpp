// Tensor side of the head operators: layer norm, dropout, the 8-bit product served and trained.  Argument checks,
// output allocation and the autograd nodes run here instead of in Python, whose interpreter time was several times the
// kernels' (forward and backward of a layer norm of 64 x 4096: 121 us, 12 of them on the GPU).  The kernels are reached through
// the addresses of the C ABI's entry points (include/yfs.h) that the Python side hands over from the library it has loaded.
#include <torch/extension.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <optional>
#include <stdexcept>
#include <string>

#include "../../include/yfs.h"

namespace {
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

struct YfsException : std::runtime_error {
    using std::runtime_error::runtime_error;
};
PyObject* g_error = nullptr;

struct Entries {
    decltype(&yfs_last_error) last_error;
    decltype(&yfs_layer_norm_fwd) ln_fwd;
    decltype(&yfs_layer_norm_bwd) ln_bwd;
    decltype(&yfs_layer_norm_bwd_workspace_bytes) ln_ws;
    decltype(&yfs_dropout_fwd) drop_fwd;
    decltype(&yfs_dropout_bwd) drop_bwd;
    decltype(&yfs_fp8_matmul) matmul;
    decltype(&yfs_fp8_matmul_workspace_bytes) matmul_ws;
    decltype(&yfs_fp8_linear_saved_bytes) lin_saved;
    decltype(&yfs_fp8_linear_fwd_workspace_bytes) lin_fwd_ws;
    decltype(&yfs_fp8_linear_bwd_workspace_bytes) lin_bwd_ws;
    decltype(&yfs_fp8_linear_fwd) lin_fwd;
    decltype(&yfs_fp8_linear_bwd) lin_bwd;
} yfs;

[[noreturn]] void fail(const std::string& what) { throw YfsException(what); }
std::string str(const Tensor& t) { return c10::str(t.scalar_type(), " ", t.sizes()); }
void check(int status, const char* what) {
    if (status == YFS_OK) return;
    char buf[512];
    yfs.last_error(buf, sizeof(buf));
    fail(c10::str(what, " failed with status ", status, ": ", buf));
}
int code(at::ScalarType t) {
    return t == at::kFloat ? YFS_F32 : (t == at::kBFloat16 ? YFS_BF16 : (t == at::kHalf ? YFS_F16 : -1));
}
// a tangent of forward-mode differentiation would be dropped without a word where no gradient is required
void no_tangent(const char* what, std::initializer_list<const Tensor*> ts) {
    for (const Tensor* t : ts)
        if (t && t->defined() && t->_fw_grad(/*level=*/0).defined())
            fail(c10::str(what, ": forward-mode derivatives are not implemented, and an argument carries a tangent"));
}
// all on one GPU, without tangents
void on_one_gpu(const char* what, std::initializer_list<const Tensor*> ts) {
    no_tangent(what, ts);
    const Tensor* first = nullptr;
    for (const Tensor* t : ts) {
        if (!t || !t->defined()) continue;
        if (!t->is_cuda())
            fail("yolo_from_scratch_amd ops run on the MI355X only: got a CPU tensor (there is no CPU fallback; the CPU oracle "
                 "lives in oracle/ and is test-only)");
        if (first && t->device() != first->device()) fail(c10::str(what, ": tensors on devices ", first->device(), " and ", t->device()));
        if (!first) first = t;
    }
}
void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }
const void* ptr(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
float* f32(const Tensor& t) { return t.defined() ? t.mutable_data_ptr<float>() : nullptr; }
Tensor get(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }

// a tensor as rows of its last axis, unit stride inside a row
struct Rows {
    Tensor t;
    int64_t rows, cols, stride;
    explicit Rows(const Tensor& x) : t(x), cols(x.size(-1)) {
        if (x.dim() == 2 && (cols == 1 || x.stride(1) == 1)) {
            rows = x.size(0);
            stride = x.stride(0);
        } else {
            t = x.contiguous();
            rows = t.numel() / cols;
            stride = cols;
        }
    }
};
Tensor f32_vector(const Tensor& t) {
    return t.defined() ? (t.scalar_type() == at::kFloat ? t : t.to(at::kFloat)).contiguous() : t;
}
void once(const char* what) {
    if (at::GradMode::is_enabled()) fail(c10::str(what, ": the gradient is not differentiable (create_graph=True)"));
}

// ---- layer norm ------------------------------------------------------------------------------------------------------
Tensor ln_forward(const Tensor& x, const Tensor& weight, const Tensor& bias, double eps, Tensor* stats) {
    const c10::DeviceGuard guard(x.device());
    const Rows r(x);
    const Tensor w = f32_vector(weight), b = f32_vector(bias);
    Tensor y = at::empty(x.sizes(), x.options());
    if (stats) *stats = at::empty({2, r.rows}, x.options().dtype(at::kFloat));
    if (r.rows) {
        float* mean = stats ? f32(*stats) : nullptr;
        check(yfs.ln_fwd(ptr(r.t), r.stride, f32(w), f32(b), y.mutable_data_ptr(), mean, mean ? mean + r.rows : nullptr, r.rows, r.cols,
                         (float)eps, code(x.scalar_type()), stream_of(x)),
              "yfs_layer_norm_fwd");
    }
    return y;
}

struct LayerNormFn : torch::autograd::Function<LayerNormFn> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptTensor& weight_, const OptTensor& bias_, double eps) {
        const Tensor weight = get(weight_), bias = get(bias_);
        Tensor stats;
        Tensor y = ln_forward(x, weight, bias, eps, &stats);
        ctx->save_for_backward({x, weight, stats});
        ctx->saved_data["bias"] = bias.defined() ? (int64_t)bias.scalar_type() : -1;
        return y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        once("layer_norm");
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &weight = saved[1], &stats = saved[2];
        if (!grads[0].defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
        const bool need_x = ctx->needs_input_grad(0);
        // (the inputs that are there are counted through)
        const int64_t bias_type = ctx->saved_data["bias"].toInt();
        const bool need_w = weight.defined() && ctx->needs_input_grad(1);
        const bool need_b = bias_type >= 0 && ctx->needs_input_grad(weight.defined() ? 2 : 1);
        const c10::DeviceGuard guard(x.device());
        const Rows r(x), d(grads[0].scalar_type() == x.scalar_type() ? grads[0] : grads[0].to(x.scalar_type()));
        const Tensor w = f32_vector(weight);
        const auto f = x.options().dtype(at::kFloat);
        Tensor dx = need_x ? at::empty(x.sizes(), x.options()) : Tensor();
        Tensor dw = need_w ? (r.rows ? at::empty({r.cols}, f) : at::zeros({r.cols}, f)) : Tensor();
        Tensor db = need_b ? (r.rows ? at::empty({r.cols}, f) : at::zeros({r.cols}, f)) : Tensor();
        if (r.rows) {
            const int type = code(x.scalar_type());
            const size_t bytes = need_w || need_b ? yfs.ln_ws(r.rows, r.cols, type) : 0;
            Tensor ws = bytes ? at::empty({(int64_t)bytes}, x.options().dtype(at::kByte)) : Tensor();
            check(yfs.ln_bwd(ptr(d.t), d.stride, ptr(r.t), r.stride, f32(w), f32(stats), f32(stats) + r.rows,
                             dx.defined() ? dx.mutable_data_ptr() : nullptr, f32(dw), f32(db), r.rows, r.cols, type,
                             bytes ? ws.mutable_data_ptr() : nullptr, bytes, stream_of(x)),
                  "yfs_layer_norm_bwd");
        }
        if (need_w && weight.scalar_type() != at::kFloat) dw = dw.to(weight.scalar_type());
        if (need_b && bias_type != (int64_t)at::kFloat) db = db.to((at::ScalarType)bias_type);
        return {dx, dw, db, Tensor()};
    }
};

Tensor layer_norm(const Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps) {
    if (code(x.scalar_type()) < 0) fail(c10::str("layer_norm: x must be fp32, bf16 or fp16, got ", x.scalar_type()));
    if (x.dim() == 0 || x.size(-1) == 0) fail(c10::str("layer_norm: x needs a last axis of at least one element, got ", x.sizes()));
    if (!(eps >= 0)) fail(c10::str("layer_norm: eps must not be negative, got ", eps));
    const Tensor w = get(weight), b = get(bias);
    for (const auto& [name, t] : {std::pair<const char*, const Tensor&>("weight", w), std::pair<const char*, const Tensor&>("bias", b)})
        if (t.defined() && (t.dim() != 1 || t.size(0) != x.size(-1) || !t.is_floating_point()))
            fail(c10::str("layer_norm: ", name, " must be floating point [", x.size(-1), "], got ", str(t)));
    on_one_gpu("layer_norm", {&x, &w, &b});
    if (at::GradMode::is_enabled() && (x.requires_grad() || (w.defined() && w.requires_grad()) || (b.defined() && b.requires_grad())))
        return LayerNormFn::apply(x, weight, bias, eps);
    at::AutoDispatchBelowADInplaceOrView below;
    return ln_forward(x, w, b, eps, nullptr);
}

// ---- dropout ---------------------------------------------------------------------------------------------------------
Tensor drop(bool backward, const Tensor& in, const Tensor& y, double p, double slope, int64_t seed, const Tensor& seed_dev) {
    const c10::DeviceGuard guard(in.device());
    Tensor out = at::empty(in.sizes(), in.options());
    if (in.numel() == 0) return out;
    const int64_t* where = seed_dev.defined() ? seed_dev.const_data_ptr<int64_t>() : nullptr;
    const int type = code(in.scalar_type());
    if (backward)
        check(yfs.drop_bwd(ptr(in), ptr(y), out.mutable_data_ptr(), in.numel(), p, (float)slope, (uint64_t)seed, where, type, stream_of(in)),
              "yfs_dropout_bwd");
    else
        check(yfs.drop_fwd(ptr(in), out.mutable_data_ptr(), in.numel(), p, (float)slope, (uint64_t)seed, where, type, stream_of(in)),
              "yfs_dropout_fwd");
    return out;
}

struct DropoutFn : torch::autograd::Function<DropoutFn> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, double p, double slope, int64_t seed, const OptTensor& seed_) {
        const Tensor seed_dev = get(seed_);
        Tensor y = drop(false, x.contiguous(), Tensor(), p, slope, seed, seed_dev);
        // y is kept for the sign of its elements, a seed in device memory so that a change before backward is noticed
        ctx->save_for_backward({slope != 1.0 ? y : Tensor(), seed_dev});
        ctx->saved_data["p"] = p;
        ctx->saved_data["slope"] = slope;
        ctx->saved_data["seed"] = seed;
        return y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        once("dropout");
        const variable_list saved = ctx->get_saved_variables();
        if (!grads[0].defined()) return {Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
        Tensor dx = drop(true, grads[0].contiguous(), saved[0], ctx->saved_data["p"].toDouble(), ctx->saved_data["slope"].toDouble(),
                         ctx->saved_data["seed"].toInt(), saved[1]);
        return {dx, Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

Tensor dropout(const Tensor& x, double p, const py::object& seed, double slope) {
    if (code(x.scalar_type()) < 0) fail(c10::str("dropout: x must be fp32, bf16 or fp16, got ", x.scalar_type()));
    if (!(p >= 0.0 && p <= 1.0)) fail(c10::str("dropout: p must lie in [0, 1], got ", p));
    if (!(slope >= 0.0 && slope <= 1.0)) fail(c10::str("dropout: slope must lie in [0, 1], got ", slope));
    Tensor dev;
    int64_t value = 0;
    if (THPVariable_Check(seed.ptr())) {
        dev = THPVariable_Unpack(seed.ptr());
        if (dev.scalar_type() != at::kLong || dev.numel() != 1) fail(c10::str("dropout: a seed tensor must hold one int64, got ", str(dev)));
    } else if (PyIndex_Check(seed.ptr())) {
        const py::object whole = py::reinterpret_steal<py::object>(PyNumber_Index(seed.ptr()));
        if (!whole) throw py::error_already_set();
        value = (int64_t)PyLong_AsUnsignedLongLongMask(whole.ptr());
    } else fail(c10::str("dropout: seed must be an int or an int64 tensor, got ", Py_TYPE(seed.ptr())->tp_name));
    on_one_gpu("dropout", {&x, &dev});
    if (at::GradMode::is_enabled() && x.requires_grad()) return DropoutFn::apply(x, p, slope, value, dev.defined() ? OptTensor(dev) : std::nullopt);
    at::AutoDispatchBelowADInplaceOrView below;
    return drop(false, x.contiguous(), Tensor(), p, slope, value, dev);
}

// ---- served 8-bit product --------------------------------------------------------------------------------------------
Tensor matmul_forward(const Tensor& x, const Tensor& data, const Tensor& scale, int64_t k, const Tensor& b, std::optional<double> slope_,
                      const std::optional<at::ScalarType>& out_dtype) {
    if (x.dim() == 0 || x.size(-1) != k) fail(c10::str("fp8_matmul: x [..., ", k, "] expected, got ", x.sizes()));
    if (code(x.scalar_type()) < 0) fail(c10::str("fp8_matmul: x must be fp32, bf16 or fp16, got ", x.scalar_type()));
    const at::ScalarType out = out_dtype.value_or(x.scalar_type());
    if (code(out) < 0) fail(c10::str("fp8_matmul: out_dtype must be fp32, bf16 or fp16, got ", out));
    const double slope = slope_.value_or(1.0);
    if (!(slope >= 0.0 && slope <= 1.0)) fail(c10::str("fp8_matmul: slope must lie in [0, 1], got ", slope));
    const int64_t n = data.size(0);
    if (b.defined() && (b.dim() != 1 || b.size(0) != n || !b.is_floating_point()))
        fail(c10::str("fp8_matmul: bias must be floating point [", n, "], got ", str(b)));
    on_one_gpu("fp8_matmul", {&x, &data, &scale, &b});
    at::AutoDispatchBelowADInplaceOrView below;
    const Rows r(x);
    const Tensor bf = f32_vector(b);
    const c10::DeviceGuard guard(x.device());
    at::DimVector sizes(x.sizes());
    sizes.back() = n;
    Tensor y = at::empty(sizes, x.options().dtype(out));
    if (r.rows == 0) return y;
    const size_t bytes = yfs.matmul_ws(r.rows, n, k);
    Tensor ws = bytes ? at::empty({(int64_t)bytes}, x.options().dtype(at::kByte)) : Tensor();
    check(yfs.matmul(ptr(r.t), code(x.scalar_type()), r.stride, ptr(data), ptr(scale), f32(bf), y.mutable_data_ptr(), code(out), r.rows, n, k,
                     (float)slope, bytes ? ws.mutable_data_ptr() : nullptr, bytes, stream_of(x)),
          "yfs_fp8_matmul");
    return y;
}
Tensor fp8_matmul(const Tensor& x, const Tensor& data, const Tensor& scale, int64_t k, const OptTensor& bias, std::optional<double> slope,
                  const std::optional<at::ScalarType>& out_dtype) {
    const Tensor b = get(bias);
    Tensor y = matmul_forward(x, data, scale, k, b, slope, out_dtype);
    // A backward pass that comes here is refused.  The node has no edges: with them a result that is kept would keep the leaves'
    // graph alive, beside which no backward pass of theirs can be captured.
    if (at::GradMode::is_enabled() && (x.requires_grad() || (b.defined() && b.requires_grad())))
        torch::autograd::set_history(y, std::make_shared<torch::autograd::Error>(
            "fp8_matmul: not differentiable (fp8_linear is; without gradients: torch.no_grad() or x.detach())"));
    return y;
}

// ---- 8-bit linear layer, trained -------------------------------------------------------------------------------------
Tensor bytes_like(const Tensor& t, size_t n) { return n ? at::empty({(int64_t)n}, t.options().dtype(at::kByte)) : Tensor(); }
void* mptr(const Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }

// needs: YFS_NEED_* of the backward pass; saved: what it will multiply
Tensor linear_forward(const Tensor& x, const Tensor& weight, const Tensor& bias, int needs, Tensor& saved) {
    const c10::DeviceGuard guard(x.device());
    const int64_t n = weight.size(0), k = weight.size(1);
    const Rows r(x), w(weight);
    const Tensor b = f32_vector(bias);
    at::DimVector sizes(x.sizes());
    sizes.back() = n;
    Tensor y = at::empty(sizes, x.options());
    if (r.rows) {
        const size_t kept = yfs.lin_saved(r.rows, n, k, needs), space = yfs.lin_fwd_ws(r.rows, n, k);
        saved = bytes_like(x, kept);
        const Tensor ws = bytes_like(x, space);
        check(yfs.lin_fwd(ptr(r.t), code(x.scalar_type()), r.stride, ptr(w.t), code(weight.scalar_type()), w.stride, f32(b), mptr(y),
                          code(x.scalar_type()), r.rows, n, k, needs, mptr(saved), kept, mptr(ws), space, stream_of(x)),
              "yfs_fp8_linear_fwd");
    }
    return y;
}

struct Fp8LinearFn : torch::autograd::Function<Fp8LinearFn> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const OptTensor& bias_, int64_t needs) {
        const Tensor bias = get(bias_);
        Tensor saved, y = linear_forward(x, weight, bias, (int)needs, saved);
        ctx->save_for_backward({saved});
        ctx->saved_data["x"] = x.sizes().vec();
        ctx->saved_data["nk"] = std::vector<int64_t>{x.numel() / weight.size(1), weight.size(0), weight.size(1), needs, (int64_t)weight.scalar_type(),
                                                     bias.defined() ? (int64_t)bias.scalar_type() : -1};
        return y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        once("fp8_linear");
        const Tensor saved = ctx->get_saved_variables()[0], &dy = grads[0];
        if (!dy.defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
        const auto nk = ctx->saved_data["nk"].toIntVector();
        const int64_t m = nk[0], n = nk[1], k = nk[2];
        const int needs = (int)nk[3];
        const bool need_b = nk[5] >= 0 && ctx->needs_input_grad(2);
        const c10::DeviceGuard guard(dy.device());
        const auto f = dy.options().dtype(at::kFloat);
        Tensor dx, dw, db;
        if (needs & YFS_NEED_DX) dx = at::empty(ctx->saved_data["x"].toIntVector(), dy.options());
        if (needs & YFS_NEED_DW) dw = m ? at::empty({n, k}, f) : at::zeros({n, k}, f);
        if (m == 0) {
            if (need_b) db = at::zeros({n}, f);
        } else if (!needs) {
            if (need_b) db = dy.reshape({m, n}).to(at::kFloat).sum(0);
        } else {
            const Rows d(dy);
            if (needs & YFS_NEED_DB) db = at::empty({n}, f);
            const size_t space = yfs.lin_bwd_ws(m, n, k, needs);
            const Tensor ws = bytes_like(dy, space);
            check(yfs.lin_bwd(ptr(d.t), code(dy.scalar_type()), d.stride, mptr(dx), code(dy.scalar_type()), f32(dw), 0, f32(db), 0, m, n, k,
                              needs, ptr(saved), (size_t)saved.numel(), mptr(ws), space, stream_of(dy)),
                  "yfs_fp8_linear_bwd");
        }
        if (dw.defined() && nk[4] != (int64_t)at::kFloat) dw = dw.to((at::ScalarType)nk[4]);
        if (db.defined() && nk[5] != (int64_t)at::kFloat) db = db.to((at::ScalarType)nk[5]);
        return {dx, dw, db, Tensor()};
    }
};

void fp8_linear_check(const Tensor& x, const Tensor& weight, const OptTensor& bias_) {
    if (weight.dim() != 2 || weight.size(0) == 0 || weight.size(1) == 0 || code(weight.scalar_type()) < 0)
        fail(c10::str("fp8_linear: expected a non-empty fp32, bf16 or fp16 weight matrix, got ", str(weight)));
    if (x.dim() == 0 || x.size(-1) != weight.size(1) || code(x.scalar_type()) < 0)
        fail(c10::str("fp8_linear: x fp32, bf16 or fp16 [..., ", weight.size(1), "] expected, got ", str(x)));
    const Tensor b = get(bias_);
    if (b.defined() && (b.dim() != 1 || b.size(0) != weight.size(0) || !b.is_floating_point()))
        fail(c10::str("fp8_linear: bias must be floating point [", weight.size(0), "], got ", str(b)));
    on_one_gpu("fp8_linear", {&x, &weight, &b});
}
Tensor fp8_linear(const Tensor& x, const Tensor& weight, const OptTensor& bias) {
    fp8_linear_check(x, weight, bias);
    const Tensor b = get(bias);
    const bool grad = at::GradMode::is_enabled(), gx = grad && x.requires_grad(), gw = grad && weight.requires_grad(),
               gb = grad && b.defined() && b.requires_grad();
    // db alone is a sum of dy: nothing is kept for it
    const int needs = (gx ? YFS_NEED_DX : 0) | (gw ? YFS_NEED_DW : 0) | (gb && (gx || gw) ? YFS_NEED_DB : 0);
    if (gx || gw || gb) return Fp8LinearFn::apply(x, weight, bias, (int64_t)needs);
    at::AutoDispatchBelowADInplaceOrView below;
    Tensor saved;
    return linear_forward(x, weight, b, 0, saved);
}

template <typename F>
void take(F& f, const py::dict& at, const char* name) { f = reinterpret_cast<F>(at[name].cast<uintptr_t>()); }

// addresses: name of each entry point -> its address; error: the exception that refusals raise
void init(const py::dict& addresses, const py::object& error) {
    take(yfs.last_error, addresses, "yfs_last_error");
    take(yfs.ln_fwd, addresses, "yfs_layer_norm_fwd");
    take(yfs.ln_bwd, addresses, "yfs_layer_norm_bwd");
    take(yfs.ln_ws, addresses, "yfs_layer_norm_bwd_workspace_bytes");
    take(yfs.drop_fwd, addresses, "yfs_dropout_fwd");
    take(yfs.drop_bwd, addresses, "yfs_dropout_bwd");
    take(yfs.matmul, addresses, "yfs_fp8_matmul");
    take(yfs.matmul_ws, addresses, "yfs_fp8_matmul_workspace_bytes");
    take(yfs.lin_saved, addresses, "yfs_fp8_linear_saved_bytes");
    take(yfs.lin_fwd_ws, addresses, "yfs_fp8_linear_fwd_workspace_bytes");
    take(yfs.lin_bwd_ws, addresses, "yfs_fp8_linear_bwd_workspace_bytes");
    take(yfs.lin_fwd, addresses, "yfs_fp8_linear_fwd");
    take(yfs.lin_bwd, addresses, "yfs_fp8_linear_bwd");
    g_error = error.inc_ref().ptr();   // for the life of the process
}
}  // namespace

PYBIND11_MODULE(_binding, m) {
    py::register_exception_translator([](std::exception_ptr p) {
        try {
            if (p) std::rethrow_exception(p);
        } catch (const YfsException& e) {
            PyErr_SetString(g_error ? g_error : PyExc_RuntimeError, e.what());
        }
    });
    m.def("init", &init);
    m.def("layer_norm", &layer_norm);
    m.def("dropout", &dropout);
    m.def("fp8_matmul", &fp8_matmul);
    m.def("fp8_linear", &fp8_linear);
    m.def("fp8_linear_check", &fp8_linear_check);
}
