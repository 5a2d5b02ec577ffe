// Module vc3d._tensors, second part (host only): the gated scan and the linear cross-entropy with their gradients, as autograd
// nodes around libvc3d.so's entry points.  In C++ because a short call's time is this: 64 x 512 of 400 classes in Python took 144
// us for some 50 us of kernels, a scan of 3 x 1531 x 1000 135; here 61 to 92 (as the autograd engine's thread is placed) and 69 to 74.
#include <Python.h>
#include <dlfcn.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ops/empty.h>
#include <ATen/ops/zeros.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include <optional>
#include <sstream>
#include <string>

#include "../../include/vc3d.h"
#include "autograd.h"

namespace {

using at::Tensor;
typedef std::optional<Tensor> Maybe;

struct Library {
    decltype(&vc_last_error) last_error;
    decltype(&vc_gated_scan_workspace_bytes) scan_workspace;
    decltype(&vc_gated_scan_fwd) scan_fwd;
    decltype(&vc_gated_scan_bwd) scan_bwd;
    decltype(&vc_gated_scan_step) scan_step;
    decltype(&vc_linear_ce_workspace_bytes) lce_workspace;
    decltype(&vc_linear_ce_saved_bytes) lce_saved;
    decltype(&vc_linear_ce_fwd) lce_fwd;
    decltype(&vc_linear_ce_bwd) lce_bwd;
} lib;
PyObject* error_class = nullptr;

struct Error : std::runtime_error {
    using std::runtime_error::runtime_error;
};
template <typename... A>
[[noreturn]] void refuse(const A&... a) {
    std::ostringstream s;
    (s << ... << a);
    throw Error(s.str());
}
void check(int rc, const char* what) {
    if (rc != 0) refuse(what, " failed (", rc, "): ", lib.last_error());
}

void* stream(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
void* ptr(const Maybe& t) { return t ? t->data_ptr() : nullptr; }
Tensor bytes(size_t n, const Tensor& like) { return at::empty({(int64_t)n}, like.options().dtype(at::kByte)); }
Tensor defined(const Maybe& t) { return t ? *t : Tensor(); }

bool is_bf16(const Tensor& t, const char* name) {
    if (!t.is_cuda() || t.layout() != at::kStrided) refuse(name, " must be a CUDA/HIP tensor: the vc3d path has no CPU fallback");
    if (t.scalar_type() != at::kFloat && t.scalar_type() != at::kBFloat16) refuse(name, ": expected fp32 or bf16, got ", t.scalar_type());
    return t.scalar_type() == at::kBFloat16;
}
void same_device(const Tensor& ref, const Maybe& t, const char* name) {
    if (t && t->device() != ref.device()) refuse(name, " is on ", t->device(), ", not on ", ref.device());
}
// What autograd hands back may have passed through a caller's hooks (kept elsewhere and loaded again, at another address, with other
// strides): the backward asks of it again what its launches rely on.
std::vector<int64_t> shape_of(const Tensor& t) {
    std::vector<int64_t> v = t.sizes().vec();
    v.insert(v.end(), {(int64_t)t.scalar_type(), (int64_t)t.device().index()});
    return v;
}
void as_saved(const Tensor& t, const char* name, at::IntArrayRef sizes, at::ScalarType type, const Tensor& where) {
    if (!t.is_cuda() || t.layout() != at::kStrided || t.device() != where.device() || t.scalar_type() != type || t.sizes() != sizes)
        refuse(name, " came back from the saved tensors' hooks as another tensor: ", t.scalar_type(), " ", t.sizes(), " on ", t.device());
}
// gradients of gradients are not there: whoever asks for them is told so, not given none
torch::autograd::variable_list once(torch::autograd::variable_list grads) {
    if (!at::GradMode::is_enabled()) return grads;
    for (Tensor& g : grads)
        if (g.defined()) g = g.detach().set_requires_grad(true);
    torch::autograd::DelayedError error("this operator of vc3d is differentiable once only", (int64_t)grads.size());
    return error.apply(std::move(grads));
}

// ---------------------------------------------------------------- gated scan
vc_scan_desc scan_desc(const Tensor& gates, bool reverse) {
    vc_scan_desc d = {};
    d.B = (int32_t)gates.size(0), d.T = (int32_t)gates.size(1), d.H = (int32_t)(gates.size(2) / 2);
    d.is_bf16 = gates.scalar_type() == at::kBFloat16, d.reverse = reverse;
    d.stride_b = gates.stride(0), d.stride_t = gates.stride(1);
    return d;
}

struct GatedScan : torch::autograd::Function<GatedScan> {
    static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& gates, const Maybe& h0, const Maybe& lengths,
                                                  bool reverse, bool grad) {
        const c10::DeviceGuard guard(gates.device());
        const vc_scan_desc d = scan_desc(gates, reverse);
        const auto f32 = gates.options().dtype(at::kFloat);
        Tensor h = at::empty({d.B, d.T, d.H}, gates.options()), last, states;
        if (grad) states = at::empty({d.B, (d.T + VC_SCAN_STATE_STEPS - 1) / VC_SCAN_STATE_STEPS, d.H}, f32);
        if (d.T == 0 || d.B == 0) last = h0 ? h0->clone() : at::zeros({d.B, d.H}, f32);
        else {
            last = at::empty({d.B, d.H}, f32);
            const size_t need = lib.scan_workspace(&d, 0);
            const Tensor ws = need > 0 ? bytes(need, gates) : Tensor();
            check(lib.scan_fwd(&d, gates.data_ptr(), (const float*)ptr(h0), (const int32_t*)ptr(lengths), h.data_ptr(), (float*)last.data_ptr(),
                               (float*)ptr(states), ptr(ws), need, stream(gates)),
                  "vc_gated_scan_fwd");
        }
        if (grad) {
            ctx->set_materialize_grads(false);
            ctx->save_for_backward({gates, defined(lengths), states});
            ctx->saved_data["reverse"] = reverse;
            ctx->saved_data["h0"] = h0.has_value();
            ctx->saved_data["shape"] = shape_of(gates);
        }
        return {h, last};
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list up) {
        const auto saved = ctx->get_saved_variables();
        Tensor gates = saved[0], lengths = saved[1], states = saved[2];
        Tensor dy = up[0], dlast = up[1], dgates, dh0;
        if (!dy.defined() && !dlast.defined()) return {Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
        {
            const auto v = ctx->saved_data["shape"].toIntVector();  // B, T, 2H, type, device
            const Tensor& up = dy.defined() ? dy : dlast;
            as_saved(gates, "gates", at::IntArrayRef(v).slice(0, 3), (at::ScalarType)v[3], up);
            if (lengths.defined()) as_saved(lengths, "lengths", {v[0]}, at::kInt, up), lengths = lengths.contiguous();
            as_saved(states, "states", {v[0], (v[1] + VC_SCAN_STATE_STEPS - 1) / VC_SCAN_STATE_STEPS, v[2] / 2}, at::kFloat, up);
            if (gates.stride(2) != 1) gates = gates.contiguous();
            states = states.contiguous();
        }
        const c10::DeviceGuard guard(gates.device());
        const vc_scan_desc d = scan_desc(gates, ctx->saved_data["reverse"].toBool());
        if (dy.defined()) {  // contiguous, at a multiple of two elements (a slice's storage may begin anywhere)
            dy = dy.contiguous();
            if ((uintptr_t)dy.data_ptr() % (2 * dy.element_size()) != 0) dy = dy.clone();
        }
        if (dlast.defined()) dlast = dlast.contiguous();
        dgates = at::empty({d.B, d.T, 2 * (int64_t)d.H}, gates.options());
        const bool want_dh0 = ctx->saved_data["h0"].toBool() && ctx->needs_input_grad(1);
        if (want_dh0) dh0 = at::empty({d.B, d.H}, states.options());
        if (d.T == 0 || d.B == 0) {
            if (want_dh0) dh0 = dlast.defined() ? dlast.clone() : dh0.zero_();
        } else {
            const size_t need = lib.scan_workspace(&d, 1);
            const Tensor ws = need > 0 ? bytes(need, gates) : Tensor();
            check(lib.scan_bwd(&d, gates.data_ptr(), (const int32_t*)ptr(lengths), (const float*)states.data_ptr(), ptr(dy), (const float*)ptr(dlast),
                               dgates.data_ptr(), (float*)ptr(dh0), ptr(ws), need, stream(gates)),
                  "vc_gated_scan_bwd");
        }
        return once({ctx->needs_input_grad(0) ? dgates : Tensor(), dh0, Tensor(), Tensor(), Tensor()});
    }
};

torch::autograd::variable_list gated_scan(Tensor gates, Maybe h0, Maybe lengths, bool reverse) {
    if (!gates.is_cuda()) refuse("gated_scan runs on the GPU only (no CPU fallback)");
    is_bf16(gates, "gates");
    if (gates.dim() != 3 || gates.size(2) == 0 || gates.size(2) % 2 != 0) refuse("gated_scan: gates [B][T][2H] expected, got ", gates.sizes());
    const int64_t B = gates.size(0), T = gates.size(1), H = gates.size(2) / 2;
    if (B > INT32_MAX || T > INT32_MAX || H > INT32_MAX) refuse("gated_scan: gates ", gates.sizes(), " are too large");
    if (h0) {
        if (h0->scalar_type() != at::kFloat || h0->sizes() != at::IntArrayRef({B, H}))
            refuse("gated_scan: h0 fp32 [", B, "][", H, "] expected, got ", h0->scalar_type(), " ", h0->sizes());
        same_device(gates, h0, "h0");
        h0 = h0->contiguous();
    }
    if (lengths) {
        if ((lengths->scalar_type() != at::kInt && lengths->scalar_type() != at::kLong) || lengths->sizes() != at::IntArrayRef({B}))
            refuse("gated_scan: lengths int32 or int64 [", B, "] on the GPU expected");
        same_device(gates, lengths, "lengths");
        lengths = lengths->scalar_type() == at::kInt ? lengths->contiguous() : lengths->clamp(0, T).to(at::kInt);
    }
    if (gates.stride(2) != 1) gates = gates.contiguous();
    const bool grad = at::GradMode::is_enabled() && (gates.requires_grad() || (h0 && h0->requires_grad()));  // whether a backward may come
    return GatedScan::apply(gates, h0, lengths, reverse, grad);
}

Tensor gated_scan_step(const Tensor& gates, const Tensor& state) {
    const bool bf16 = is_bf16(gates, "gates");
    if (gates.dim() != 2 || gates.size(1) == 0 || gates.size(1) % 2 != 0 || gates.stride(1) != 1)
        refuse("gated_scan_step: gates [B][2H] with contiguous rows expected, got ", gates.sizes());
    const int64_t B = gates.size(0), H = gates.size(1) / 2;
    if (B > INT32_MAX || H > INT32_MAX) refuse("gated_scan_step: gates ", gates.sizes(), " are too large");
    if (state.scalar_type() != at::kFloat || state.sizes() != at::IntArrayRef({B, H}) || !state.is_contiguous())
        refuse("gated_scan_step: state fp32 [", B, "][", H, "], contiguous, expected, got ", state.scalar_type(), " ", state.sizes());
    same_device(gates, state, "state");
    if (at::GradMode::is_enabled() && (gates.requires_grad() || state.requires_grad()))
        refuse("gated_scan_step has no gradient, and gates or state want one: torch.no_grad() around it, or gated_scan over one step");
    const c10::DeviceGuard guard(gates.device());
    const Tensor h = at::empty({B, H}, gates.options());
    if (B > 0) {
        check(lib.scan_step(gates.data_ptr(), gates.stride(0), bf16, (float*)state.data_ptr(), h.data_ptr(), (int32_t)B, (int32_t)H, stream(gates)),
              "vc_gated_scan_step");
        if (!state.is_inference()) state.unsafeGetTensorImpl()->bump_version();
    }
    return h;
}

// ---------------------------------------------------------------- linear classifier + cross-entropy
int64_t row_stride(const Tensor& t) { return t.size(0) > 1 ? std::max(t.stride(0), t.size(1)) : t.size(1); }
// a matrix with contiguous rows that do not overlap: as it is, or a copy
Tensor rows(const Tensor& t) {
    return t.is_contiguous() || ((t.size(1) <= 1 || t.stride(1) == 1) && (t.size(0) <= 1 || t.stride(0) >= t.size(1))) ? t : t.contiguous();
}
vc_linear_ce_desc lce_desc(const Tensor& x, const Tensor& w, int64_t ignore, int64_t reduction, int64_t keep) {
    vc_linear_ce_desc d = {};
    d.N = (int32_t)x.size(0), d.D = (int32_t)x.size(1), d.V = (int32_t)w.size(0), d.is_bf16 = x.scalar_type() == at::kBFloat16;
    d.reduction = (int32_t)reduction, d.w_align = (int32_t)((uintptr_t)w.data_ptr() & 15);
    d.ldx = row_stride(x), d.ldw = row_stride(w), d.ignore_index = ignore, d.keep_bytes = keep;
    return d;
}

struct LinearCrossEntropy : torch::autograd::Function<LinearCrossEntropy> {
    static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const Tensor& w, const Tensor& labels, const Maybe& bias, int64_t ignore,
                          int64_t reduction, int64_t keep, bool grad) {
        const c10::DeviceGuard guard(x.device());
        vc_linear_ce_desc d = lce_desc(x, w, ignore, reduction, keep);
        const auto f32 = x.options().dtype(at::kFloat);
        Tensor loss = reduction == 0 ? at::empty({d.N}, f32) : at::empty({}, f32), saved;
        if (d.N == 0) {
            loss.zero_();
            saved = bytes(0, x);
        } else {
            size_t need = 0;
            Tensor ws;
            auto allocate = [&] { saved = bytes(lib.lce_saved(&d), x), need = lib.lce_workspace(&d, 0), ws = bytes(need, x); };
            try {
                allocate();
            } catch (const c10::OutOfMemoryError&) {  // what is kept by itself is kept where there is room for it
                if (keep != -1) throw;
                saved = ws = Tensor();
                d.keep_bytes = keep = 0;
                allocate();
            }
            check(lib.lce_fwd(&d, x.data_ptr(), w.data_ptr(), ptr(bias), (const int64_t*)labels.data_ptr(), (float*)loss.data_ptr(), saved.data_ptr(),
                              ws.data_ptr(), need, stream(x)),
                  "vc_linear_ce_fwd");
        }
        if (grad) {
            ctx->save_for_backward({x, w, labels, defined(bias), saved});
            ctx->saved_data["ignore"] = ignore;
            ctx->saved_data["reduction"] = reduction;
            ctx->saved_data["keep"] = keep;
            ctx->saved_data["shape"] = std::vector<int64_t>{d.N, d.D, d.V, (int64_t)x.scalar_type(), saved.numel()};
        }
        return loss;
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list up) {
        const auto saved = ctx->get_saved_variables();
        Tensor x = saved[0], w = saved[1], labels = saved[2], bias = saved[3], kept = saved[4];
        {
            const auto v = ctx->saved_data["shape"].toIntVector();  // N, D, V, type, bytes saved
            const auto type = (at::ScalarType)v[3];
            as_saved(x, "x", {v[0], v[1]}, type, up[0]), as_saved(w, "weight", {v[2], v[1]}, type, up[0]);
            as_saved(labels, "labels", {v[0]}, at::kLong, up[0]), as_saved(kept, "what the forward saved", {v[4]}, at::kByte, up[0]);
            if (bias.defined()) as_saved(bias, "bias", {v[2]}, type, up[0]), bias = bias.contiguous();
            x = rows(x), w = rows(w), labels = labels.contiguous(), kept = kept.contiguous();
            if ((uintptr_t)kept.data_ptr() % 256 != 0) kept = kept.clone();
        }
        const c10::DeviceGuard guard(x.device());
        auto desc = [&] {
            return lce_desc(x, w, ctx->saved_data["ignore"].toInt(), ctx->saved_data["reduction"].toInt(), ctx->saved_data["keep"].toInt());
        };
        vc_linear_ce_desc d = desc();
        // whether the forward left a copy of w goes by where w lay then: one that would need the copy now is laid as it was
        if (d.N > 0 && lib.lce_saved(&d) > (size_t)kept.numel()) w = w.clone(at::MemoryFormat::Contiguous), d = desc();
        if (d.N > 0 && lib.lce_saved(&d) > (size_t)kept.numel()) refuse("linear_cross_entropy: the weight came back in another layout");
        const Tensor dloss = up[0].contiguous();
        Tensor dx, dw, db;
        if (ctx->needs_input_grad(0)) dx = at::empty({d.N, d.D}, x.options());
        if (ctx->needs_input_grad(1)) dw = at::empty({d.V, d.D}, x.options());
        if (bias.defined() && ctx->needs_input_grad(3)) db = at::empty({d.V}, x.options());
        if (d.N == 0) {
            if (dw.defined()) dw.zero_();
            if (db.defined()) db.zero_();
        } else {
            const size_t need = lib.lce_workspace(&d, 1);
            const Tensor ws = bytes(need, x);
            check(lib.lce_bwd(&d, x.data_ptr(), w.data_ptr(), ptr(bias), (const int64_t*)labels.data_ptr(), kept.data_ptr(),
                              (const float*)dloss.data_ptr(), ptr(dx), ptr(dw), ptr(db), ws.data_ptr(), need, stream(x)),
                  "vc_linear_ce_bwd");
        }
        return once({dx, dw, Tensor(), db, Tensor(), Tensor(), Tensor(), Tensor()});
    }
};

Tensor linear_cross_entropy(Tensor x, Tensor w, Tensor labels, Maybe bias, int64_t ignore, int64_t reduction, int64_t keep) {
    if (!x.is_cuda()) refuse("linear_cross_entropy runs on the GPU only (no CPU fallback)");
    is_bf16(x, "x");
    if (x.dim() < 1 || w.dim() != 2 || x.size(-1) != w.size(1) || labels.sizes() != x.sizes().slice(0, x.dim() - 1))
        refuse("linear_cross_entropy: x [..., D], weight [V][D] and labels [...] expected, got ", x.sizes(), ", ", w.sizes(), ", ", labels.sizes());
    const int64_t D = w.size(1), V = w.size(0);
    if (V == 0 || D == 0) refuse("linear_cross_entropy: no classes or no features (weight ", w.sizes(), ")");
    same_device(x, w, "weight");
    same_device(x, labels, "labels");
    same_device(x, bias, "bias");
    if (w.scalar_type() != x.scalar_type() || (bias && bias->scalar_type() != x.scalar_type()))
        refuse("linear_cross_entropy: x, weight and bias are of one type, got ", x.scalar_type(), ", ", w.scalar_type(),
               bias ? std::string(", ") + c10::toString(bias->scalar_type()) : "");
    if (labels.scalar_type() != at::kLong) refuse("linear_cross_entropy: labels int64 expected, got ", labels.scalar_type());
    if (bias && bias->sizes() != at::IntArrayRef({V})) refuse("linear_cross_entropy: bias [", V, "] expected, got ", bias->sizes());
    const auto shape = labels.sizes().vec();
    if (x.dim() != 2) x = x.reshape({-1, D}), labels = labels.reshape({-1});
    if (x.size(0) > INT32_MAX || V > INT32_MAX || D > INT32_MAX) refuse("linear_cross_entropy: at most 2^23 rows and classes, 2^20 features");
    x = rows(x), w = rows(w), labels = labels.contiguous();
    if (bias) bias = bias->contiguous();
    const bool grad = at::GradMode::is_enabled() && (x.requires_grad() || w.requires_grad() || (bias && bias->requires_grad()));
    const Tensor loss = LinearCrossEntropy::apply(x, w, labels, bias, ignore, reduction, grad ? keep : 0, grad);
    return reduction == 0 && shape.size() != 1 ? loss.view(shape) : loss;
}

// ---------------------------------------------------------------- Python
// what this module refuses comes as its own exception, everything else as torch's operators would let it through (memory that runs
// out, what a caller's hooks raise)
template <typename F>
PyObject* guarded(F f) {
    HANDLE_TH_ERRORS
    try {
        return f();
    } catch (const Error& e) {
        PyErr_SetString(error_class, e.what());
        return nullptr;
    }
    END_HANDLE_TH_ERRORS
}
Tensor tensor(PyObject* o, const char* name) {
    if (!THPVariable_Check(o)) refuse(name, " is no tensor");
    return THPVariable_Unpack(o);
}
Maybe maybe(PyObject* o, const char* name) { return o == Py_None ? Maybe() : Maybe(tensor(o, name)); }
struct NoGil {
    PyThreadState* s = PyEval_SaveThread();
    ~NoGil() { PyEval_RestoreThread(s); }
};

}  // namespace

// bind(path of the loaded libvc3d.so, exception class)
PyObject* vc_bind(PyObject*, PyObject* args) {
    const char* path;
    PyObject* cls;
    if (!PyArg_ParseTuple(args, "sO", &path, &cls)) return nullptr;
    void* const so = dlopen(path, RTLD_NOW | RTLD_NOLOAD);
    if (so == nullptr) return PyErr_Format(cls, "%s is not loaded", path), nullptr;
    bool all = true;
    auto get = [&](auto& f, const char* name) { all = (f = (std::decay_t<decltype(f)>)dlsym(so, name)) != nullptr && all; };
    get(lib.last_error, "vc_last_error");
    get(lib.scan_workspace, "vc_gated_scan_workspace_bytes");
    get(lib.scan_fwd, "vc_gated_scan_fwd");
    get(lib.scan_bwd, "vc_gated_scan_bwd");
    get(lib.scan_step, "vc_gated_scan_step");
    get(lib.lce_workspace, "vc_linear_ce_workspace_bytes");
    get(lib.lce_saved, "vc_linear_ce_saved_bytes");
    get(lib.lce_fwd, "vc_linear_ce_fwd");
    get(lib.lce_bwd, "vc_linear_ce_bwd");
    if (!all) return PyErr_Format(cls, "%s lacks an entry point", path), nullptr;
    Py_INCREF(cls);
    error_class = cls;
    Py_RETURN_NONE;
}

// gated_scan(gates, h0 or None, lengths or None, reverse) -> (h, last)
PyObject* vc_gated_scan_py(PyObject*, PyObject* args) {
    PyObject *g, *h, *l;
    int reverse;
    if (!PyArg_ParseTuple(args, "OOOp", &g, &h, &l, &reverse)) return nullptr;
    return guarded([&]() -> PyObject* {
        const Tensor gates = tensor(g, "gates");
        const Maybe h0 = maybe(h, "h0"), lengths = maybe(l, "lengths");
        torch::autograd::variable_list out;
        {
            const NoGil no;
            out = gated_scan(gates, h0, lengths, reverse != 0);
        }
        return Py_BuildValue("NN", THPVariable_Wrap(out[0]), THPVariable_Wrap(out[1]));
    });
}

// gated_scan_step(gates, state) -> h
PyObject* vc_gated_scan_step_py(PyObject*, PyObject* args) {
    PyObject *g, *s;
    if (!PyArg_ParseTuple(args, "OO", &g, &s)) return nullptr;
    return guarded([&]() -> PyObject* { return THPVariable_Wrap(gated_scan_step(tensor(g, "gates"), tensor(s, "state"))); });
}

// linear_cross_entropy(x, weight, labels, bias or None, ignore_index, reduction, keep_bytes) -> loss
PyObject* vc_linear_cross_entropy_py(PyObject*, PyObject* args) {
    PyObject *xo, *wo, *yo, *bo;
    long long ignore, keep;
    int reduction;
    if (!PyArg_ParseTuple(args, "OOOOLiL", &xo, &wo, &yo, &bo, &ignore, &reduction, &keep)) return nullptr;
    return guarded([&]() -> PyObject* {
        const Tensor x = tensor(xo, "x"), w = tensor(wo, "weight"), y = tensor(yo, "labels");
        const Maybe b = maybe(bo, "bias");
        Tensor loss;
        {
            const NoGil no;
            loss = linear_cross_entropy(x, w, y, b, ignore, reduction, keep);
        }
        return THPVariable_Wrap(loss);
    });
}
