// regularise_torch.cpp -- the autograd nodes of regularise.py: tensors in, tensors out, around the C ABI of include/plenreg.h.
//
// Native because of the small calls: a training pass of a 100 x 512 layer takes 13 us on the GPU; with the nodes written in Python its two passes cost
// 120-160 us of host time (the engine's thread has to get hold of the interpreter for each node), with these about a third of that.  Nodes with plain
// members rather than torch::autograd::Function, whose context (a map of values by name, wrapped inputs and outputs) costs several us a pass.
// regularise.py's functions first hand their arguments over as they come (quick_*): what passes all of its checks here is launched at once, anything else comes back as None and
// goes through the checks in Python, which say what is wrong with it.  (A call at 100 x 512, us of host time: dropout 3.5, norm 4.0; 4.7 and 5.8 with the checks in Python; a
// library multiplication is at 4.5.)  What concerns memory is checked once more behind the C ABI.
#include <torch/extension.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include "../../include/plenreg.h"

using at::Tensor;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

namespace {

// entry points of libplenreg.so, handed over by regularise.load()
int (*dropout_entry)(const PlenRegDropout *, void *) = nullptr;
int (*forward_entry)(const PlenRegNorm *, void *) = nullptr;
int (*backward_entry)(const PlenRegNorm *, void *) = nullptr;
int64_t (*workspace_entry)(const PlenRegNorm *, int) = nullptr;

void bind(uintptr_t dropout, uintptr_t forward, uintptr_t backward, uintptr_t workspace) {
    dropout_entry = (decltype(dropout_entry))dropout;
    forward_entry = (decltype(forward_entry))forward;
    backward_entry = (decltype(backward_entry))backward;
    workspace_entry = (decltype(workspace_entry))workspace;
}

int type_of(const Tensor &t) { return t.scalar_type() == at::kFloat ? PLENREG_F32 : t.scalar_type() == at::kBFloat16 ? PLENREG_BF16 : PLENREG_F16; }
// on the tensors' device and its current stream
template <class Args> void launch(int (*entry)(const Args *, void *), const Args &a, const Tensor &x) {
    const c10::DeviceGuard guard(x.device());
    const int rc = entry(&a, c10::hip::getCurrentHIPStream(x.device().index()).stream());
    TORCH_CHECK(rc == 0, "libplenreg kernel launch failed: HIP error ", -rc);
}
// gradients of these operators are not differentiable themselves: an error when that is asked for, as torch.autograd.function.once_differentiable makes it
variable_list once(variable_list out) {
    if (!at::GradMode::is_enabled()) return out;
    const auto node = std::make_shared<torch::autograd::DelayedError>("trying to differentiate twice an operator that is differentiable once (plen_ml_walk_amd.regularise)", (int64_t)out.size());
    return (*node)(std::move(out));
}

// as saved tensors that are used after their release report it
void check_alive(bool released) {
    TORCH_CHECK(!released, "Trying to backward through the graph a second time: the saved state of this operator has been released; pass retain_graph=True to the first backward");
}
// The nodes fill their results through raw pointers, which whoever records operations does not see: a traced call would return uninitialised memory.  Refused, as are tensors without memory of their own
// (fake and functional ones, those of a functorch transform, subclasses that stand for others).
void not_recorded() {
    using Modes = c10::impl::TorchDispatchModeTLS;
    using Key = c10::impl::TorchDispatchModeKey;
    TORCH_CHECK(!torch::jit::tracer::isTracing() && !(Modes::any_modes_set() && (Modes::get_mode(Key::FAKE) || Modes::get_mode(Key::PROXY) || Modes::get_mode(Key::FUNCTIONAL))),
                "plen_ml_walk_amd.regularise cannot be traced: its kernels are no library operations that a trace could record");
}
void own_memory(const Tensor &t) {
    if (!t.defined()) return;
    static const c10::DispatchKeySet wrappers({c10::DispatchKey::Python, c10::DispatchKey::FuncTorchGradWrapper, c10::DispatchKey::FuncTorchBatched, c10::DispatchKey::Batched, c10::DispatchKey::Functionalize});
    TORCH_CHECK(!t.key_set().has_any(wrappers), "plen_ml_walk_amd.regularise needs tensors with memory of their own; functorch transforms (vmap, torch.func.grad), fake tensors and tensor subclasses are not supported");
}
void no_tangent(const Tensor &t) { TORCH_CHECK(!t.defined() || !t._fw_grad(0).defined(), "plen_ml_walk_amd.regularise has no forward-mode derivatives"); }

// ---- dropout
// x as rows of contiguous elements, a constant stride apart; what is laid out otherwise is copied first
Tensor as_rows(const Tensor &x, PlenRegDropout &a) {
    a.rows = 1; a.cols = x.numel(); a.x_stride = 0;
    if (x.is_contiguous()) return x;
    int64_t k = x.dim(), width = 1, next = 0, step = 0;
    while (k > 0 && (x.size(k - 1) == 1 || x.stride(k - 1) == width)) width *= x.size(--k);
    for (int64_t i = k - 1; i >= 0; i--) {
        if (x.size(i) == 1) continue;
        if (step == 0 && next == 0) { step = x.stride(i); next = x.size(i) * step; if (step == 0) return as_rows(x.contiguous(), a); }
        else if (x.stride(i) == next) next = x.size(i) * x.stride(i);
        else return as_rows(x.contiguous(), a);
    }
    if (width == 1) return as_rows(x.contiguous(), a);
    a.rows = x.numel() / width; a.cols = width; a.x_stride = step;
    return x;
}
Tensor run_dropout(const Tensor &x, int64_t cut, const Tensor &rng, int64_t site, const Tensor &used) {
    const Tensor y = at::empty(x.sizes(), x.options().memory_format(at::MemoryFormat::Contiguous));
    if (x.numel() == 0) return y;
    PlenRegDropout a = {};
    const Tensor rows = as_rows(x, a);
    a.x = rows.data_ptr(); a.y = y.data_ptr(); a.rng = (const uint64_t *)rng.data_ptr(); a.used = used.defined() ? (uint64_t *)used.data_ptr() : nullptr;
    a.dtype = type_of(x); a.cut = (uint32_t)cut; a.site = (int32_t)site;
    launch(dropout_entry, a, x);
    return y;
}
struct DropoutNode : torch::autograd::Node {
    Tensor used;
    int64_t cut, site;
    bool released = false;
    variable_list apply(variable_list &&dy) override {
        Tensor dx;
        {
            std::lock_guard<std::mutex> lock(mutex_);
            check_alive(released);
            not_recorded(); own_memory(dy[0]);
            const at::NoGradGuard off;
            if (dy[0].defined() && task_should_compute_output(0)) dx = run_dropout(dy[0].resolve_neg(), cut, used, site, Tensor());
        }
        return once({dx});
    }
    void release_variables() override { std::lock_guard<std::mutex> lock(mutex_); used.reset(); released = true; }
    std::string name() const override { return "RegulariseDropout"; }
};
Tensor dropout(const Tensor &x_, int64_t cut, const Tensor &rng_, int64_t site) {
    not_recorded(); own_memory(x_); own_memory(rng_);
    const Tensor x = x_.resolve_neg(), rng = rng_.resolve_neg();          // (a view whose memory holds the negatives, as the imaginary part of a conjugate)
    no_tangent(x);
    if (!x.requires_grad() || !at::GradMode::is_enabled()) return run_dropout(x, cut, rng, site, Tensor());
    const std::shared_ptr<DropoutNode> node(new DropoutNode, torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(x));
    node->cut = cut; node->site = site;
    Tensor y;
    {
        const at::AutoDispatchBelowADInplaceOrView below;
        node->used = at::empty({2}, rng.options());
        y = run_dropout(x, cut, rng, site, node->used);
    }
    torch::autograd::set_history(y, node);
    return y;
}

// ---- group norm with an activation, with dropout (cut > 0) or without
struct Form { int64_t groups, act, cut, site; double eps; };

// x with the elements of each x[n] contiguous
Tensor as_slabs(const Tensor &x, int64_t &stride) {
    stride = x.stride(0);
    if (x.is_contiguous()) return x;
    int64_t want = 1;
    for (int64_t i = x.dim() - 1; i > 0; i--) {
        if (x.size(i) != 1 && x.stride(i) != want) { const Tensor c = x.contiguous(); stride = c.stride(0); return c; }
        want *= x.size(i);
    }
    return x;
}
// a parameter in a type that the kernels read beside x's: float32 or x's own
Tensor as_param(const Tensor &t, const Tensor &x) {
    if (!t.defined()) return t;
    return (t.scalar_type() == at::kFloat || t.scalar_type() == x.scalar_type() ? t : t.to(at::kFloat)).contiguous();
}
PlenRegNorm norm_args(const Tensor &x, const Tensor &w, const Tensor &b, const Form &f) {
    PlenRegNorm a = {};
    a.N = x.size(0); a.C = (int32_t)x.size(-1); a.L = x.numel() / a.N / a.C; a.G = (int32_t)f.groups;
    a.dtype = type_of(x); a.act = (int32_t)f.act; a.cut = (uint32_t)f.cut; a.site = (int32_t)f.site; a.eps = (float)f.eps;
    if (w.defined()) { a.w = w.data_ptr(); a.w_dtype = type_of(w); }
    if (b.defined()) { a.b = b.data_ptr(); a.w_dtype = type_of(b); }
    return a;
}
Tensor workspace(PlenRegNorm &a, int backward, const Tensor &x) {
    const int64_t n = workspace_entry(&a, backward);
    TORCH_CHECK(n >= 0, "libplenreg refuses these sizes: N ", a.N, ", L ", a.L, ", C ", a.C, ", groups ", a.G);
    if (n == 0) return Tensor();
    const Tensor ws = at::empty({n}, x.options().dtype(at::kByte).memory_format(at::MemoryFormat::Contiguous));
    a.ws = ws.data_ptr();
    return ws;
}
Tensor run_forward(const Tensor &x_, const Tensor &w_, const Tensor &b_, const Form &f, const Tensor &rng, const Tensor &stats, const Tensor &used) {
    const Tensor y = at::empty(x_.sizes(), x_.options().memory_format(at::MemoryFormat::Contiguous));
    if (x_.numel() == 0) return y;
    int64_t stride;
    const Tensor x = as_slabs(x_, stride), w = as_param(w_, x_), b = as_param(b_, x_);
    PlenRegNorm a = norm_args(x, w, b, f);
    a.x = x.data_ptr(); a.x_stride = stride; a.out = y.data_ptr();
    a.stats = stats.defined() ? (double *)stats.data_ptr() : nullptr;
    if (f.cut) { a.rng = (const uint64_t *)rng.data_ptr(); a.used = used.defined() ? (uint64_t *)used.data_ptr() : nullptr; }
    const Tensor ws = workspace(a, 0, x);
    launch(forward_entry, a, x);
    return y;
}
struct NormNode : torch::autograd::Node {
    SavedVariable x_, w_, b_;
    Tensor stats, used;
    Form f;
    bool released = false;
    variable_list apply(variable_list &&grads) override {
        variable_list out(3);
        std::unique_lock<std::mutex> lock(mutex_);
        check_alive(released);
        not_recorded(); own_memory(grads[0]);
        if (grads[0].defined()) {
            const at::NoGradGuard off;
            const Tensor x0 = x_.unpack(), w0 = w_.unpack(), b0 = b_.unpack();
            const Tensor w = as_param(w0, x0), b = as_param(b0, x0);
            const bool want_w = w.defined() && task_should_compute_output(1), want_b = b.defined() && task_should_compute_output(2);
            Tensor dx = at::empty(x0.sizes(), x0.options().memory_format(at::MemoryFormat::Contiguous)), dw = want_w ? at::empty_like(w) : Tensor(), db = want_b ? at::empty_like(b) : Tensor();
            if (x0.numel()) {
                int64_t xs, dys;
                const Tensor x = as_slabs(x0, xs), dy = as_slabs(grads[0].resolve_neg(), dys);
                PlenRegNorm a = norm_args(x, w, b, f);
                a.x = x.data_ptr(); a.x_stride = xs; a.dy = dy.data_ptr(); a.dy_stride = dys; a.out = dx.data_ptr(); a.stats = (double *)stats.data_ptr();
                a.dw = want_w ? dw.data_ptr() : nullptr; a.db = want_b ? db.data_ptr() : nullptr;
                a.rng = f.cut ? (const uint64_t *)used.data_ptr() : nullptr;
                const Tensor ws = workspace(a, 1, x);
                launch(backward_entry, a, x);
            } else {
                if (want_w) dw.zero_();
                if (want_b) db.zero_();
            }
            if (task_should_compute_output(0)) out[0] = std::move(dx);
            if (want_w) out[1] = dw.scalar_type() == w0.scalar_type() ? std::move(dw) : dw.to(w0.scalar_type());
            if (want_b) out[2] = db.scalar_type() == b0.scalar_type() ? std::move(db) : db.to(b0.scalar_type());
        }
        lock.unlock();
        return once(std::move(out));
    }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        x_.reset_data(); w_.reset_data(); b_.reset_data(); stats.reset(); used.reset();
        released = true;
    }
    std::string name() const override { return "RegulariseNormAct"; }
};
Tensor norm(const Tensor &x_, const std::optional<Tensor> &weight, const std::optional<Tensor> &bias, int64_t groups, double eps, int64_t act, int64_t cut, const std::optional<Tensor> &rng_, int64_t site) {
    const auto values = [](const std::optional<Tensor> &t) { return t && t->defined() ? t->resolve_neg() : Tensor(); };
    const Form f = {groups, act, cut, site, eps};
    not_recorded(); own_memory(x_);
    for (const auto *t : {&weight, &bias, &rng_}) if (*t) own_memory(**t);
    const Tensor x = x_.resolve_neg(), w = values(weight), b = values(bias), rng = values(rng_);
    no_tangent(x); no_tangent(w); no_tangent(b);
    if (!at::GradMode::is_enabled() || !(x.requires_grad() || (w.defined() && w.requires_grad()) || (b.defined() && b.requires_grad())))
        return run_forward(x, w, b, f, rng, Tensor(), Tensor());
    const std::shared_ptr<NormNode> node(new NormNode, torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(x, w, b));
    node->f = f;
    node->x_ = SavedVariable(x, false);
    if (w.defined()) node->w_ = SavedVariable(w, false);
    if (b.defined()) node->b_ = SavedVariable(b, false);
    Tensor y;
    {
        const at::AutoDispatchBelowADInplaceOrView below;
        node->stats = at::empty({x.size(0), groups, 2}, x.options().dtype(at::kDouble).memory_format(at::MemoryFormat::Contiguous));
        if (cut) node->used = at::empty({2}, rng.options());
        y = run_forward(x, w, b, f, rng, node->stats, node->used);
    }
    torch::autograd::set_history(y, node);
    return y;
}

// ---- the checks of regularise.py, as yes or no
bool float_type(const Tensor &t) { const auto k = t.scalar_type(); return k == at::kFloat || k == at::kBFloat16 || k == at::kHalf; }
bool good_x(PyObject *o) {
    if (!THPVariable_Check(o)) return false;
    const Tensor &x = THPVariable_Unpack(o);
    own_memory(x);                                        // (before sizes are asked for, which may be symbols)
    return x.is_cuda() && x.layout() == at::kStrided && float_type(x);
}
bool to_int(PyObject *o, int64_t &v) {
    if (!PyLong_Check(o)) return false;
    int overflow = 0;
    v = PyLong_AsLongLongAndOverflow(o, &overflow);
    return !overflow;
}
bool to_double(PyObject *o, double &v) {
    if (!PyFloat_Check(o)) return false;
    v = PyFloat_AS_DOUBLE(o);
    return true;
}
struct DrawArgs { int64_t cut, site; };
bool good_draw(const Tensor &x, PyObject *p, PyObject *rng_, PyObject *site, DrawArgs &d) {
    double prob;
    if (!to_double(p, prob) || !(prob >= 0.0 && prob <= 1.0) || !to_int(site, d.site) || d.site < 0 || d.site >= (INT64_C(1) << 31) - 16 || !THPVariable_Check(rng_)) return false;
    const Tensor &rng = THPVariable_Unpack(rng_);
    if (rng.scalar_type() != at::kLong || rng.dim() != 1 || rng.size(0) != 2 || rng.device() != x.device() || !rng.is_contiguous() || x.numel() > INT64_C(1) << 35) return false;
    d.cut = llrint(prob * 65536);                                   // (to even, as Python rounds)
    return true;
}
bool good_param(const Tensor &x, PyObject *o, std::optional<Tensor> &t) {
    if (o == Py_None) return true;
    if (!THPVariable_Check(o)) return false;
    t = THPVariable_Unpack(o);
    return t->dim() == 1 && t->size(0) == x.size(-1) && float_type(*t) && t->device() == x.device() && t->layout() == at::kStrided;
}
struct NormCall { std::optional<Tensor> w, b; int64_t groups, act; double eps; };
bool good_norm(const Tensor &x, PyObject *groups, PyObject *w, PyObject *b, PyObject *eps, PyObject *act, NormCall &n) {
    if (x.dim() < 2 || x.numel() == 0 || !to_int(groups, n.groups) || !to_double(eps, n.eps) || !PyUnicode_Check(act)) return false;
    const int64_t ch = x.size(-1), positions = x.numel() / x.size(0) / ch;
    if (n.groups < 1 || n.groups > ch || ch % n.groups || ch > (positions > 1 ? PLENREG_MAX_C_LONG : PLENREG_MAX_C)) return false;
    if (!good_param(x, w, n.w) || !good_param(x, b, n.b) || (n.w && n.b && n.w->scalar_type() != n.b->scalar_type())) return false;
    if (!(n.eps > 0.0) || std::isinf(n.eps) || (float)n.eps == 0.f) return false;
    n.act = -1;
    static const char *const names[3] = {"none", "relu", "silu"};
    for (int k = 0; k < 3; k++)
        if (PyUnicode_CompareWithASCIIString(act, names[k]) == 0) n.act = k;
    return n.act >= 0;
}
// (x, p, rng, site)
PyObject *quick_dropout(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    DrawArgs d;
    if (n != 4 || !good_x(a[0]) || !good_draw(THPVariable_Unpack(a[0]), a[1], a[2], a[3], d)) Py_RETURN_NONE;
    return THPVariable_Wrap(dropout(THPVariable_Unpack(a[0]), d.cut, THPVariable_Unpack(a[2]), d.site));
    END_HANDLE_TH_ERRORS
}
// (x, groups, weight, bias, eps, act)
PyObject *quick_norm(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    NormCall c;
    if (n != 6 || !good_x(a[0]) || !good_norm(THPVariable_Unpack(a[0]), a[1], a[2], a[3], a[4], a[5], c)) Py_RETURN_NONE;
    return THPVariable_Wrap(norm(THPVariable_Unpack(a[0]), c.w, c.b, c.groups, c.eps, c.act, 0, std::nullopt, 0));
    END_HANDLE_TH_ERRORS
}
// (x, p, rng, groups, weight, bias, site, eps, act)
PyObject *quick_layer(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    DrawArgs d;
    NormCall c;
    if (n != 9 || !good_x(a[0]) || !good_draw(THPVariable_Unpack(a[0]), a[1], a[2], a[6], d) || !good_norm(THPVariable_Unpack(a[0]), a[3], a[4], a[5], a[7], a[8], c)) Py_RETURN_NONE;
    return THPVariable_Wrap(norm(THPVariable_Unpack(a[0]), c.w, c.b, c.groups, c.eps, c.act, d.cut, THPVariable_Unpack(a[2]), d.site));
    END_HANDLE_TH_ERRORS
}
PyMethodDef quick[] = {{"quick_dropout", (PyCFunction)(void *)quick_dropout, METH_FASTCALL, nullptr},
                       {"quick_norm", (PyCFunction)(void *)quick_norm, METH_FASTCALL, nullptr},
                       {"quick_layer", (PyCFunction)(void *)quick_layer, METH_FASTCALL, nullptr},
                       {nullptr, nullptr, 0, nullptr}};

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    m.def("bind", &bind);
    m.def("dropout", &dropout);
    m.def("norm", &norm);
    if (PyModule_AddFunctions(m.ptr(), quick) != 0) throw py::error_already_set();
}
