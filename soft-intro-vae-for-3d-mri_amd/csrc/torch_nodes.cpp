// Autograd nodes of layer_norm, add_layer_norm and dropout over the C entry points, as a Python extension module.
//
// A training call on a small tensor is host time: the same operators as Python autograd functions spend most of it in
// interpreted code on autograd's own thread (a layer norm of 8 x 1200 and its gradients: 107 us, and 59 us for a native
// operator of torch).  The functions here take the common case -- plain dense device tensors (or slices of wider
// rows) on the current device, arguments in range, no trace being recorded -- and return None for everything else; the
// caller then takes the Python path, which knows every layout and words every refusal.  Both call the same entry points of libsiv, whose
// addresses are handed in by `bind`, so that whichever build of the library is loaded is the one that runs.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/TracerMode.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/utils/pybind.h>

#include "siv.h"

namespace {

using at::Tensor;
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

struct {
    decltype(&siv_layer_norm_workspace) norm_workspace;
    decltype(&siv_layer_norm_fwd) norm_fwd;
    decltype(&siv_layer_norm_bwd) norm_bwd;
    decltype(&siv_add_layer_norm_fwd) add_fwd;
    decltype(&siv_add_layer_norm_bwd) add_bwd;
    decltype(&siv_dropout_fwd) drop_fwd;
    decltype(&siv_dropout_bwd) drop_bwd;
    decltype(&siv_last_error) last_error;
} lib;

int type_code(at::ScalarType t) {
    return t == at::kFloat ? SIV_F32 : t == at::kBFloat16 ? SIV_BF16 : t == at::kHalf ? SIV_F16 : -1;
}
bool on_current_device(const Tensor& t) {
    return t.is_cuda() && t.layout() == at::kStrided && t.get_device() == c10::hip::current_device();
}
// torch.func's wrappers (vmap, grad, functionalize) and batched gradients: tensors without memory of their own
bool wrapped(const Tensor& t) {
    constexpr c10::DispatchKeySet keys({c10::DispatchKey::FuncTorchGradWrapper, c10::DispatchKey::FuncTorchBatched,
                                        c10::DispatchKey::Functionalize, c10::DispatchKey::Batched});
    return t.defined() && t.key_set().has_any(keys);
}
void require_plain(const variable_list& grads, const char* what) {
    for (const Tensor& g : grads)
        TORCH_CHECK(!wrapped(g), "the backward pass of ", what, " takes no batched or transformed gradients (torch.func, vmap)");
}
at::MemoryFormat format_of(const Tensor& t) {
    return t.dim() == 5 ? at::MemoryFormat::ChannelsLast3d : at::MemoryFormat::Contiguous;
}
bool dense(const Tensor& t) { return t.is_contiguous(format_of(t)); }
Tensor made_dense(const Tensor& t) { return t.contiguous(format_of(t)); }
Tensor empty_like_dense(const Tensor& t) { return at::empty(t.sizes(), t.options(), format_of(t)); }
bool same_kind(const Tensor& a, const Tensor& x) {
    return a.scalar_type() == x.scalar_type() && a.device() == x.device() && a.sizes() == x.sizes() && dense(a);
}
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
void* stream_of(const Tensor& t) { return (void*)c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

// A saved tensor as it comes back.  Hooks (torch.autograd.graph.save_on_cpu and the like) keep values, not strides, and may
// hand back anything: the kernels take no other type, sizes or device than those that were saved.
Tensor unpacked(const SavedVariable& v, at::ScalarType type, at::IntArrayRef sizes, at::Device device,
                std::shared_ptr<Node> saved_for = nullptr, bool any_rows = false) {
    Tensor t = v.unpack(std::move(saved_for));
    if (!t.defined()) return t;
    TORCH_CHECK(t.scalar_type() == type && t.sizes() == sizes && t.device() == device && t.layout() == at::kStrided,
                "a saved tensor came back as ", t.scalar_type(), " ", t.sizes(), " on ", t.device(), " where ", type, " ", sizes,
                " on ", device, " was saved");
    return any_rows || dense(t) ? t : made_dense(t);
}

struct Rows {
    int64_t rows, C;
};
Rows rows_of(const Tensor& x) {
    const int64_t C = x.dim() == 5 ? x.size(1) : x.size(-1);
    return {x.numel() / C, C};
}
// elements between rows: dense tensors, and rows that are slices of wider ones; -1: neither
int64_t row_stride(const Tensor& x, const Rows& r) {
    if (dense(x)) return r.C;
    if (x.dim() == 2 && x.stride(1) == 1) return r.rows == 1 ? r.C : x.stride(0) >= r.C ? x.stride(0) : -1;
    return -1;
}
bool plain_activation(const Tensor& x) {
    return x.defined() && x.dim() > 0 && x.numel() > 0 && type_code(x.scalar_type()) >= 0 && on_current_device(x);
}
// type code of weight / bias, or -1 where the Python path has to look at them
int affine_type(const Tensor& x, const Rows& r, const Tensor& w, const Tensor& b) {
    int code = SIV_F32;
    for (const Tensor* t : {&w, &b}) {
        if (!t->defined()) continue;
        if ((t->scalar_type() != at::kFloat && t->scalar_type() != x.scalar_type()) || t->device() != x.device() ||
            t->dim() != 1 || t->numel() != r.C || !t->is_contiguous())
            return -1;
        code = type_code(t->scalar_type());
    }
    return w.defined() && b.defined() && w.scalar_type() != b.scalar_type() ? -1 : code;
}
struct Scratch {
    Tensor t;
    size_t bytes = 0;
    Scratch(const Rows& r, int type, int backward, const Tensor& like) {
        if (lib.norm_workspace(r.rows, r.C, type, backward, &bytes) == 0 && bytes)
            t = at::empty({(int64_t)bytes}, like.options().dtype(at::kByte));
    }
};

// where a dropout mask comes from
struct Mask {
    bool on = false;
    Tensor keep, epoch;                    // a stored mask; the device epoch of a key
    uint64_t seed = 0, sid = 0;
    float p = 0.f;
    const uint8_t* stored() const { return keep.defined() ? (const uint8_t*)keep.data_ptr() : nullptr; }
    const uint64_t* epoch_ptr() const { return epoch.defined() ? (const uint64_t*)epoch.data_ptr() : nullptr; }
};
bool plain_mask(const Mask& m, const Tensor& x) {
    if (!(m.p >= 0.f && m.p < 1.f)) return false;
    if (m.keep.defined() && (m.keep.scalar_type() != at::kByte || m.keep.device() != x.device() ||
                             m.keep.sizes() != x.sizes() || !dense(m.keep)))
        return false;
    return !m.epoch.defined() ||
           (m.epoch.scalar_type() == at::kLong && m.epoch.numel() == 1 && m.epoch.device() == x.device());
}

void require(int rc, const char* what) {
    TORCH_CHECK(rc == 0, what, " failed (code ", rc, "): ", lib.last_error());
}
// Gradients under create_graph.  They have no derivative of their own: each gets a node that leads to what it was
// computed from and raises, so that asking for one is an error and never a missing term.
variable_list first_order(variable_list grads, const variable_list& sources, const char* what) {
    if (!at::GradMode::is_enabled() || !torch::autograd::compute_requires_grad(sources)) return grads;
    for (Tensor& g : grads)
        if (g.defined()) {
            g = g.detach();
            torch::autograd::set_history(
                g, std::make_shared<torch::autograd::Error>(std::string("the backward pass of ") + what +
                                                                " is not differentiable",
                                                            torch::autograd::collect_next_edges(sources)));
        }
    return grads;
}

// parameter gradients: fresh tensors, or added into the flat buffers of an optimiser
struct AffineGrads {
    Tensor dw, db;
    int accumulate = 0;
    AffineGrads(bool need_w, bool need_b, const Tensor& w_buf, const Tensor& b_buf, at::ScalarType type, int64_t C,
                const Tensor& like) {
        // (one parameter as weight and bias: its buffer would be added into from two places at once)
        const bool direct = (need_w || need_b) && (!need_w || w_buf.defined()) && (!need_b || b_buf.defined()) &&
                            !(need_w && need_b && w_buf.data_ptr() == b_buf.data_ptr());
        accumulate = direct;
        if (need_w) dw = direct ? w_buf : at::empty({C}, like.options().dtype(type));
        if (need_b) db = direct ? b_buf : at::empty({C}, like.options().dtype(type));
    }
    Tensor out(const Tensor& t) const { return accumulate ? Tensor() : t; }
};
bool usable_buffer(const Tensor& buf, const Tensor& param) {
    return !buf.defined() || (param.defined() && buf.scalar_type() == param.scalar_type() && buf.is_contiguous() &&
                              buf.numel() == param.numel() && buf.device() == param.device());
}

struct LayerNormBackward : Node {
    SavedVariable x_, w_;
    Tensor w_buf, b_buf;
    at::ScalarType ptype = at::kFloat;
    float eps = 0.f;
    std::string name() const override { return "SivLayerNormBackward"; }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        x_.reset_data();
        w_.reset_data();
    }
    variable_list apply(variable_list&& grads) override {
        require_plain(grads, "layer_norm");
        std::lock_guard<std::mutex> lock(mutex_);
        const bool need_x = task_should_compute_output(0), need_w = task_should_compute_output(1),
                   need_b = task_should_compute_output(2);
        variable_list out(3), sources = {grads[0]};
        Tensor dy = grads[0];
        if (!dy.defined() || !(need_x || need_w || need_b)) return out;
        {
            Tensor x = unpacked(x_, dy.scalar_type(), dy.sizes(), dy.device(), nullptr, true),
                   w = unpacked(w_, ptype, {rows_of(dy).C}, dy.device());
            sources.insert(sources.end(), {x, w});
            at::AutoDispatchBelowADInplaceOrView guard;
            const c10::DeviceGuard device(x.device());
            const Rows r = rows_of(x);
            const int type = type_code(x.scalar_type());
            int64_t ldx = row_stride(x, r), ldy = row_stride(dy, r);
            if (ldx < 0) { x = made_dense(x); ldx = r.C; }
            if (ldy < 0) { dy = made_dense(dy); ldy = r.C; }
            if (need_x) out[0] = empty_like_dense(x);
            const AffineGrads g(need_w, need_b, w_buf, b_buf, ptype, r.C, x);
            const Scratch ws(r, type, 1, x);
            require(lib.norm_bwd(ptr(dy), ldy, ptr(x), ldx, ptr(w), type_code(ptype), eps, ptr(out[0]), ptr(g.dw), ptr(g.db),
                                 g.accumulate, type, r.rows, r.C, ptr(ws.t), ws.bytes, stream_of(x)),
                    "siv_layer_norm_bwd");
            out[1] = g.out(g.dw);
            out[2] = g.out(g.db);
        }
        return first_order(std::move(out), sources, "layer_norm");
    }
};

struct AddLayerNormBackward : Node {
    SavedVariable s_, w_, keep_;
    Mask mask;                             // (its stored mask lives in keep_)
    Tensor w_buf, b_buf;
    at::ScalarType ptype = at::kFloat;
    float eps = 0.f;
    std::string name() const override { return "SivAddLayerNormBackward"; }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        s_.reset_data();
        w_.reset_data();
        keep_.reset_data();
    }
    variable_list apply(variable_list&& grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        const bool need_x = task_should_compute_output(0), need_r = task_should_compute_output(1),
                   need_w = task_should_compute_output(2), need_b = task_should_compute_output(3);
        variable_list out(4), sources = {grads[0], grads[1]};
        Tensor dy = grads[0], ds = grads[1];
        if (!(dy.defined() || ds.defined()) || !(need_x || need_r || need_w || need_b)) return out;
        if (dy.defined() || (need_x && mask.on)) require_plain(grads, "add_layer_norm");       // (else ds is handed on)
        {
            const Tensor& up = dy.defined() ? dy : ds;
            Tensor s = unpacked(s_, up.scalar_type(), up.sizes(), up.device(), shared_from_this()),
                   w = unpacked(w_, ptype, {rows_of(up).C}, up.device()),
                   keep = unpacked(keep_, at::kByte, up.sizes(), up.device());
            sources.insert(sources.end(), {s, w});
            at::AutoDispatchBelowADInplaceOrView guard;
            const c10::DeviceGuard device(s.device());
            const Rows r = rows_of(s);
            const int type = type_code(s.scalar_type());
            if (ds.defined() && !dense(ds)) ds = made_dense(ds);
            Mask m = mask;
            m.keep = keep;
            if (!dy.defined()) {           // only the sum went on: the norm takes no part
                if (need_x) {
                    out[0] = m.on ? empty_like_dense(s) : ds;
                    if (m.on)
                        require(lib.drop_bwd(ptr(ds), nullptr, m.stored(), m.seed, m.sid, m.epoch_ptr(), m.p, 1.f,
                                             ptr(out[0]), type, s.numel(), stream_of(s)),
                                "siv_dropout_bwd");
                }
                if (need_r) out[1] = ds;
            } else {
                if (!dense(dy)) dy = made_dense(dy);
                const bool both = !m.on && need_x && need_r;        // nothing dropped: the two gradients are one tensor
                if (need_r) out[1] = empty_like_dense(s);
                if (need_x && !both) out[0] = empty_like_dense(s);
                const AffineGrads g(need_w, need_b, w_buf, b_buf, ptype, r.C, s);
                const Scratch ws(r, type, 1, s);
                require(lib.add_bwd(ptr(dy), ptr(ds), ptr(s), m.stored(), m.seed, m.sid, m.epoch_ptr(), m.on ? m.p : 0.f,
                                    ptr(w), type_code(ptype), eps, ptr(out[0]), ptr(out[1]), ptr(g.dw), ptr(g.db),
                                    g.accumulate, type, r.rows, r.C, ptr(ws.t), ws.bytes, stream_of(s)),
                        "siv_add_layer_norm_bwd");
                if (both) out[0] = out[1];
                out[2] = g.out(g.dw);
                out[3] = g.out(g.db);
            }
        }
        out = first_order(std::move(out), sources, "add_layer_norm");
        if (!grads[0].defined()) {         // what is handed on as it came keeps its own history
            if (need_r) out[1] = grads[1];
            if (need_x && !mask.on) out[0] = grads[1];
        }
        return out;
    }
};

struct DropoutBackward : Node {
    SavedVariable x_, keep_;
    Mask mask;
    float slope = 1.f;
    std::string name() const override { return "SivDropoutBackward"; }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        x_.reset_data();
        keep_.reset_data();
    }
    variable_list apply(variable_list&& grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        const bool need_x = task_should_compute_output(0), need_r = task_should_compute_output(1);
        variable_list out(2), sources = {grads[0]};
        Tensor dy = grads[0];
        if (!dy.defined()) return out;
        if (need_x) {
            require_plain(grads, "dropout");
            Tensor x = unpacked(x_, dy.scalar_type(), dy.sizes(), dy.device()),
                   keep = unpacked(keep_, at::kByte, dy.sizes(), dy.device());
            sources.push_back(x);
            at::AutoDispatchBelowADInplaceOrView guard;
            const c10::DeviceGuard device(dy.device());
            Tensor g = dense(dy) ? dy : made_dense(dy);
            Mask m = mask;
            m.keep = keep;
            out[0] = empty_like_dense(g);
            require(lib.drop_bwd(ptr(g), ptr(x), m.stored(), m.seed, m.sid, m.epoch_ptr(), m.on ? m.p : 0.f, slope,
                                 ptr(out[0]), type_code(g.scalar_type()), g.numel(), stream_of(g)),
                    "siv_dropout_bwd");
        }
        out = first_order(std::move(out), sources, "dropout");
        if (need_r) out[1] = grads[0];     // handed on as it came, with its own history
        return out;
    }
};

template <typename... T>
bool wants_grad(const T&... t) {
    return at::GradMode::is_enabled() && torch::autograd::compute_requires_grad(t...);
}
SavedVariable saved(const Tensor& t, bool is_output = false) {
    return t.defined() ? SavedVariable(t, is_output) : SavedVariable();
}

// ---- forward: false = for the Python path ------------------------------------------------------------------------------
bool layer_norm(const Tensor& x, const Tensor& w, const Tensor& b, double eps, const Tensor& w_buf, const Tensor& b_buf,
                Tensor& y) {
    if (!plain_activation(x)) return false;
    const Rows r = rows_of(x);
    const int type = type_code(x.scalar_type()), wtype = affine_type(x, r, w, b);
    const int64_t ld = row_stride(x, r);
    if (wtype < 0 || ld < 0 || !usable_buffer(w_buf, w) || !usable_buffer(b_buf, b)) return false;
    {
        at::AutoDispatchBelowADInplaceOrView guard;
        y = empty_like_dense(x);
        if (wrapped(y)) return false;      // (inside torch.func.grad what is allocated is wrapped too)
        const Scratch ws(r, type, 0, x);
        if (lib.norm_fwd(ptr(x), ld, ptr(w), ptr(b), wtype, (float)eps, ptr(y), type, r.rows, r.C, ptr(ws.t), ws.bytes,
                         stream_of(x)))
            return false;
    }
    if (wants_grad(x, w, b)) {
        auto node = std::shared_ptr<LayerNormBackward>(new LayerNormBackward(), torch::autograd::deleteNode);
        node->set_next_edges(torch::autograd::collect_next_edges(x, w, b));
        node->x_ = saved(x);
        node->w_ = saved(w);
        node->w_buf = w_buf;
        node->b_buf = b_buf;
        node->ptype = w.defined() ? w.scalar_type() : b.defined() ? b.scalar_type() : at::kFloat;
        node->eps = (float)eps;
        torch::autograd::set_history(y, node);
    }
    return true;
}
bool add_layer_norm(const Tensor& x, const Tensor& res, const Tensor& w, const Tensor& b, double eps, const Mask& m,
                    const Tensor& w_buf, const Tensor& b_buf, Tensor& y, Tensor& s) {
    if (!plain_activation(x) || !res.defined() || !dense(x) || !same_kind(res, x) || !plain_mask(m, x)) return false;
    const Rows r = rows_of(x);
    const int type = type_code(x.scalar_type()), wtype = affine_type(x, r, w, b);
    if (wtype < 0 || !usable_buffer(w_buf, w) || !usable_buffer(b_buf, b)) return false;
    {
        at::AutoDispatchBelowADInplaceOrView guard;
        y = empty_like_dense(x);
        s = empty_like_dense(x);
        if (wrapped(y)) return false;
        const Scratch ws(r, type, 0, x);
        if (lib.add_fwd(ptr(x), ptr(res), m.stored(), m.seed, m.sid, m.epoch_ptr(), m.on ? m.p : 0.f, ptr(w), ptr(b), wtype,
                        (float)eps, ptr(s), ptr(y), type, r.rows, r.C, ptr(ws.t), ws.bytes, stream_of(x)))
            return false;
    }
    if (wants_grad(x, res, w, b)) {
        auto node = std::shared_ptr<AddLayerNormBackward>(new AddLayerNormBackward(), torch::autograd::deleteNode);
        node->set_next_edges(torch::autograd::collect_next_edges(x, res, w, b));
        torch::autograd::set_history({y, s}, node);
        node->s_ = saved(s, true);
        node->w_ = saved(w);
        node->keep_ = saved(m.keep);
        node->mask = m;
        node->mask.keep = Tensor();
        node->w_buf = w_buf;
        node->b_buf = b_buf;
        node->ptype = w.defined() ? w.scalar_type() : b.defined() ? b.scalar_type() : at::kFloat;
        node->eps = (float)eps;
    }
    return true;
}
bool dropout(const Tensor& x, const Tensor& res, const Mask& m, double slope, Tensor& out) {
    if (!plain_activation(x) || !dense(x) || (res.defined() && !same_kind(res, x)) || !plain_mask(m, x)) return false;
    {
        at::AutoDispatchBelowADInplaceOrView guard;
        out = empty_like_dense(x);
        if (wrapped(out)) return false;
        if (lib.drop_fwd(ptr(x), ptr(res), m.stored(), m.seed, m.sid, m.epoch_ptr(), m.on ? m.p : 0.f, (float)slope, ptr(out),
                         type_code(x.scalar_type()), x.numel(), stream_of(x)))
            return false;
    }
    if (wants_grad(x, res)) {
        auto node = std::shared_ptr<DropoutBackward>(new DropoutBackward(), torch::autograd::deleteNode);
        node->set_next_edges(torch::autograd::collect_next_edges(x, res));
        if ((float)slope != 1.f) node->x_ = saved(x);
        node->keep_ = saved(m.keep);
        node->mask = m;
        node->mask.keep = Tensor();
        node->slope = (float)slope;
        torch::autograd::set_history(out, node);
    }
    return true;
}

// ---- Python ------------------------------------------------------------------------------------------------------------
// Whether calls are being recorded (torch.jit.trace) or watched (a dispatch mode, make_fx's among them).  A trace would see
// the allocations made here and not the kernels that fill them, and replay uninitialised memory; of a Python function
// torch.jit.trace records the call, and make_fx is refused there.
bool recording() { return at::tracer::impl::is_dispatch_enabled() || c10::impl::dispatch_mode_enabled(); }
// a tensor of exactly torch's own types, or None (undefined); anything else: not for here.  Nor torch.func's wrappers, nor a
// tensor with a forward-mode tangent, which the nodes would lose (the Python functions refuse both).
bool tensor_arg(PyObject* o, Tensor& t) {
    if (o == Py_None) return true;
    if (!THPVariable_CheckExact(o)) return false;
    t = THPVariable_Unpack(o);
    return !wrapped(t) && !t._fw_grad(0).defined();
}
bool float_arg(PyObject* o, double& v) {
    v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) {
        PyErr_Clear();
        return false;
    }
    return true;
}
// (mask tensor or None, seed or None, stream id, epoch or None, p): four arguments from a[0] on
bool mask_args(PyObject* const* a, Mask& m) {
    double p;
    if (!tensor_arg(a[0], m.keep) || !tensor_arg(a[3], m.epoch) || !float_arg(a[4], p)) return false;
    m.p = (float)p;
    if (!(p >= 0.0 && p < 1.0)) m.p = -1.f;          // refused by plain_mask (a double just below 1 may round to 1)
    m.on = m.keep.defined();
    if (a[1] != Py_None) {
        m.on = true;
        m.seed = PyLong_AsUnsignedLongLongMask(a[1]);
        m.sid = PyLong_AsUnsignedLongLongMask(a[2]);
        if (PyErr_Occurred()) {
            PyErr_Clear();
            return false;
        }
    }
    return true;
}
#define SIV_ARGS(count)                                                                     \
    if (n != count) {                                                                       \
        PyErr_Format(PyExc_TypeError, "%d arguments expected, got %zd", count, n);          \
        return nullptr;                                                                     \
    }

PyObject* py_layer_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    SIV_ARGS(6)
    if (recording()) Py_RETURN_NONE;
    Tensor x, w, b, w_buf, b_buf, y;
    double eps;
    if (!tensor_arg(a[0], x) || !tensor_arg(a[1], w) || !tensor_arg(a[2], b) || !float_arg(a[3], eps) ||
        !tensor_arg(a[4], w_buf) || !tensor_arg(a[5], b_buf))
        Py_RETURN_NONE;
    bool done;
    {
        pybind11::gil_scoped_release nogil;
        done = layer_norm(x, w, b, eps, w_buf, b_buf, y);
    }
    if (!done) Py_RETURN_NONE;
    return THPVariable_Wrap(y);
    END_HANDLE_TH_ERRORS
}
PyObject* py_add_layer_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    SIV_ARGS(12)
    if (recording()) Py_RETURN_NONE;
    Tensor x, res, w, b, w_buf, b_buf, y, s;
    double eps;
    Mask m;
    if (!tensor_arg(a[0], x) || !tensor_arg(a[1], res) || !tensor_arg(a[2], w) || !tensor_arg(a[3], b) ||
        !float_arg(a[4], eps) || !mask_args(a + 5, m) || !tensor_arg(a[10], w_buf) || !tensor_arg(a[11], b_buf))
        Py_RETURN_NONE;
    bool done;
    {
        pybind11::gil_scoped_release nogil;
        done = add_layer_norm(x, res, w, b, eps, m, w_buf, b_buf, y, s);
    }
    if (!done) Py_RETURN_NONE;
    PyObject* out = PyTuple_New(2);
    if (!out) return nullptr;
    PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(y));
    PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(s));
    return out;
    END_HANDLE_TH_ERRORS
}
PyObject* py_dropout(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    SIV_ARGS(8)
    if (recording()) Py_RETURN_NONE;
    Tensor x, res, out;
    double slope;
    Mask m;
    if (!tensor_arg(a[0], x) || !tensor_arg(a[1], res) || !mask_args(a + 2, m) || !float_arg(a[7], slope)) Py_RETURN_NONE;
    bool done;
    {
        pybind11::gil_scoped_release nogil;
        done = dropout(x, res, m, slope, out);
    }
    if (!done) Py_RETURN_NONE;
    return THPVariable_Wrap(out);
    END_HANDLE_TH_ERRORS
}
// bind({name: address}): the entry points of the loaded libsiv
PyObject* py_bind(PyObject*, PyObject* dict) {
    HANDLE_TH_ERRORS
    auto get = [&](const char* name, auto& fn) {
        PyObject* v = PyDict_Check(dict) ? PyDict_GetItemString(dict, name) : nullptr;
        void* p = v ? PyLong_AsVoidPtr(v) : nullptr;
        TORCH_CHECK(p, "no address for ", name);
        fn = reinterpret_cast<std::remove_reference_t<decltype(fn)>>(p);
    };
    get("siv_layer_norm_workspace", lib.norm_workspace);
    get("siv_layer_norm_fwd", lib.norm_fwd);
    get("siv_layer_norm_bwd", lib.norm_bwd);
    get("siv_add_layer_norm_fwd", lib.add_fwd);
    get("siv_add_layer_norm_bwd", lib.add_bwd);
    get("siv_dropout_fwd", lib.drop_fwd);
    get("siv_dropout_bwd", lib.drop_bwd);
    get("siv_last_error", lib.last_error);
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
    {"bind", py_bind, METH_O, "bind({name: address}): entry points of the loaded libsiv"},
    {"layer_norm", (PyCFunction)(void*)py_layer_norm, METH_FASTCALL,
     "layer_norm(x, weight, bias, eps, weight_grad_buf, bias_grad_buf) -> y or None"},
    {"add_layer_norm", (PyCFunction)(void*)py_add_layer_norm, METH_FASTCALL,
     "add_layer_norm(x, residual, weight, bias, eps, mask, seed, stream_id, epoch, p, weight_grad_buf, bias_grad_buf) "
     "-> (y, s) or None"},
    {"dropout", (PyCFunction)(void*)py_dropout, METH_FASTCALL,
     "dropout(x, residual, mask, seed, stream_id, epoch, p, slope) -> out or None"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_siv_torch", "autograd nodes over libsiv", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__siv_torch(void) { return PyModule_Create(&module); }
