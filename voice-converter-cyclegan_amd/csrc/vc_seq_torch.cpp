// vc_seq_torch.cpp -- torch binding of the sequence operators (include/vc_cyclegan.h): argument checks, outputs and workspaces, autograd.
//
// A frame of a live stream is one small launch, and a training step meets these operators many times: the calls around the kernels are worth as much as
// the kernels there.  In Python one took 11 to 17 us for a single frame and 50 to 120 us for a step's two passes, beside 3 us of launch.
// The entry points are the library's own, handed over by address (bind): one copy of it is loaded, by _lib.py, which checks it against its sources.
// Host code only; no kernel and no HIP call is made here but through that library.
#include <torch/csrc/utils/pybind.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/autograd/variable.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/zeros.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/VirtualGuardImpl.h>
#include "../../include/vc_cyclegan.h"

namespace {
using at::Tensor;
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

// ---- the library -----------------------------------------------------------------------------------------------------
#define VC_ENTRIES(F) F(last_error) F(rms_norm_fwd) F(rms_norm_e4m3) F(rms_norm_bwd_work) F(rms_norm_bwd) F(causal_conv1d_fwd) F(causal_conv1d_bwd_work) \
    F(causal_conv1d_bwd) F(causal_conv1d_step) F(selective_scan_saved) F(selective_scan_fwd_work) F(selective_scan_bwd_work) F(selective_scan_fwd) \
    F(selective_scan_bwd) F(selective_scan_step)
struct Library {
#define F(n) decltype(&vc_##n) n = nullptr;
    VC_ENTRIES(F)
#undef F
} L;
PyObject* vc_error = nullptr;                  // _lib.VcError
PyObject* raw_stream_of = nullptr;             // device index -> the current stream's handle

void check(int rc, const char* what) {
    if (rc == 0) return;
    const std::string text = std::string(what) + " failed (rc=" + std::to_string(rc) + "): " + L.last_error();
    if (!PyGILState_Check()) throw std::runtime_error(text);          // in a backward pass
    PyErr_SetString(vc_error, text.c_str());
    throw py::error_already_set();
}

// ---- streams ---------------------------------------------------------------------------------------------------------
// The stream a call runs on.  A backward pass runs on its forward's (torch sees to that), so it finds the handle with the node and needs no interpreter.
struct Stream {
    c10::Stream at; void* handle;
    static c10::Stream current(const at::Device& d) { return c10::impl::VirtualGuardImpl(d.type()).getStream(d); }
    static Stream now(const at::Device& d) {
        py::gil_scoped_acquire gil;
        PyObject* i = PyLong_FromLong(d.index());
        PyObject* r = PyObject_CallFunctionObjArgs(raw_stream_of, i, nullptr);
        Py_DECREF(i);
        if (!r) throw py::error_already_set();
        void* h = (void*)PyLong_AsUnsignedLongLong(r);
        Py_DECREF(r);
        return {current(d), h};
    }
    void* of(const at::Device& d) const { return current(d) == at ? handle : now(d).handle; }
};

// ---- checks ----------------------------------------------------------------------------------------------------------
int type_code(const Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return VC_F32;
        case at::kBFloat16: return VC_BF16;
        case at::kHalf: return VC_F16;
        default: return -1;
    }
}
// what its memory alone does not tell: a lazily negated view, a tangent (these operators have reverse gradients only), another layout
void ordinary(const Tensor& t, const char* name) {
    TORCH_CHECK_VALUE(t.layout() == at::kStrided && !t.is_neg(), name, " must be a dense tensor that is not negated lazily (resolve_neg() makes one)");
    TORCH_CHECK_NOT_IMPLEMENTED(!t._fw_grad(0).defined(), name, " has a tangent: forward mode differentiation is not offered");
}
int narrow(int64_t n, const char* name) {
    TORCH_CHECK_VALUE(n >= 0 && n < (int64_t{1} << 31), n, " ", name, " are too many");
    return (int)n;
}
void activation(const Tensor& t, const char* name) {
    TORCH_CHECK_VALUE(t.is_cuda(), name, " must be a tensor on a GPU (there is no CPU path)");
    TORCH_CHECK_VALUE(type_code(t) >= 0, name, " must be float32, bfloat16 or float16, got ", t.scalar_type());
    TORCH_CHECK_VALUE(t.dim() >= 1, name, " must be [..., channels]");
    ordinary(t, name);
    narrow(t.size(-1), "channels");
}
void like(const Tensor& t, const Tensor& ref, const char* name, at::IntArrayRef shape, at::ScalarType dtype) {
    TORCH_CHECK_VALUE(t.scalar_type() == dtype && t.device() == ref.device(), name, " must be a ", dtype, " tensor on ", ref.device());
    TORCH_CHECK_VALUE(t.sizes() == shape, name, " must have shape ", shape, ", got ", t.sizes());
    ordinary(t, name);
}
void like(const OptTensor& t, const Tensor& ref, const char* name, at::IntArrayRef shape, at::ScalarType dtype) {
    if (t) like(*t, ref, name, shape, dtype);
}
bool wants_grad(std::initializer_list<const OptTensor> ts) {
    if (!at::GradMode::is_enabled()) return false;
    for (const auto& t : ts) if (t && t->requires_grad()) return true;
    return false;
}
void no_grad(const char* what, std::initializer_list<const OptTensor> ts) {
    TORCH_CHECK_VALUE(!wants_grad(ts), what, " has no gradient: call it under torch.no_grad() or on detached tensors");
}
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
Tensor plain(const OptTensor& t) { return t ? t->contiguous() : Tensor(); }
Tensor fresh(at::IntArrayRef shape, const Tensor& ref) { return at::empty(shape, ref.options().requires_grad(false)); }
Tensor fresh(at::IntArrayRef shape, const Tensor& ref, at::ScalarType dtype) { return at::empty(shape, at::TensorOptions().device(ref.device()).dtype(dtype)); }

// [..., width] as rows with one stride between them.  Copies only what cannot be seen so.
struct Rows {
    Tensor t; int64_t ld = 0;
    Rows() = default;
    explicit Rows(const Tensor& from) {
        const int64_t w = from.size(-1);
        if (from.is_contiguous()) { t = from; ld = w; return; }
        t = from.dim() == 2 ? from : from.reshape({-1, w});
        if (w > 1 && t.stride(1) != 1) t = t.contiguous();
        ld = t.size(0) > 1 ? t.stride(0) : w;
    }
    explicit Rows(const OptTensor& from) { if (from) *this = Rows(*from); }
    void* p() const { return ptr(t); }
    Rows&& within(int64_t most) && { if (ld > most && !t.is_contiguous()) { t = t.contiguous(); ld = t.size(-1); } return std::move(*this); }
};
// Widest row strides that are taken in place: below what the kernels' 32-bit offsets reach (a block of the convolution has up to 8192 rows, and up to 256
// rows where they are of 256 channels or more); rows that lie further apart are copied
int64_t conv_ld(const Tensor& x) { return x.size(-1) < 256 ? 1 << 15 : 1 << 20; }
constexpr int64_t SCAN_LD = 1 << 24;
// B or C of a scan: [..., states] or [..., groups, states] beside x [..., channels]
struct Grouped {
    Tensor t; int64_t ld = 0; int groups = 1;
    Grouped(const Tensor& from, const Tensor& x, int64_t states, const char* name) {
        TORCH_CHECK_VALUE(from.scalar_type() == x.scalar_type() && from.device() == x.device(), name, " must be a ", x.scalar_type(), " tensor on ", x.device());
        const auto lead = x.sizes().slice(0, x.dim() - 1);
        const bool one = from.dim() == x.dim();
        TORCH_CHECK_VALUE((one || from.dim() == x.dim() + 1) && from.size(-1) == states && from.sizes().slice(0, x.dim() - 1) == lead && (one || from.size(-2) > 0),
                          name, " must be ", lead, " + [groups, ", states, "] or + [", states, "], got ", from.sizes());
        ordinary(from, name);
        TORCH_CHECK_VALUE(one || from.size(-2) <= x.size(-1), name, " has more groups than there are channels");
        groups = one ? 1 : (int)from.size(-2);
        const int64_t w = groups * states;
        if (from.is_contiguous()) { t = from; ld = w; return; }
        t = from.reshape({-1, groups, states});
        if ((states > 1 && t.stride(2) != 1) || (groups > 1 && t.stride(1) != states)) t = t.contiguous();
        ld = t.size(0) > 1 ? t.stride(0) : w;
        if (ld > SCAN_LD && !t.is_contiguous()) { t = t.contiguous(); ld = w; }
    }
};

// Where a graph of a backward pass is being built, its results hang on a node that leads to all that they depend on and refuses to be run: whichever way
// a second differentiation comes, it meets an error and no missing gradient.
struct Twice : public Node {
    std::string what;
    std::string name() const override { return "CannotBeDifferentiatedTwice"; }
    variable_list apply(variable_list&&) override { throw std::runtime_error(what + " cannot be differentiated twice"); }
};
variable_list once(variable_list out, const Node& backward, const variable_list& grads, const char* what) {
    if (!at::GradMode::is_enabled()) return out;
    auto n = std::shared_ptr<Twice>(new Twice(), torch::autograd::deleteNode);
    n->what = what;
    auto edges = backward.next_edges();
    for (const auto& g : grads) if (g.defined() && g.requires_grad()) edges.push_back(torch::autograd::impl::gradient_edge(g));
    n->set_next_edges(std::move(edges));
    for (auto& o : out) if (o.defined()) { o = o.detach(); torch::autograd::set_history(o, n); }
    return out;
}
template <class N, class... Ts> std::shared_ptr<N> node_for(const Ts&... inputs) {
    auto n = std::shared_ptr<N>(new N(), torch::autograd::deleteNode);
    n->set_next_edges(torch::autograd::collect_next_edges(inputs...));
    return n;
}
Tensor or_undefined(const OptTensor& t) { return t ? *t : Tensor(); }

// ---- norm ------------------------------------------------------------------------------------------------------------
struct NormBackward : public Node {
    SavedVariable total, gamma, rstd;
    bool residual = false; at::ScalarType x_type = at::kFloat; int kind = 0, stream_kind = 0;
    std::optional<Stream> stream;
    std::string name() const override { return "RmsNormBackward"; }
    void release_variables() override { std::lock_guard<std::mutex> lock(mutex_); total.reset_data(); gamma.reset_data(); rstd.reset_data(); }
    variable_list apply(variable_list&& grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        const Tensor t = total.unpack(residual ? shared_from_this() : nullptr), g = gamma.unpack(), r = rstd.unpack();
        const bool need_x = task_should_compute_output(0), need_g = task_should_compute_output(1), need_r = residual && task_should_compute_output(2);
        Tensor dx, dres, dg;
        {
            at::NoGradGuard ng;
            const c10::DeviceGuard guard(t.device());
            const int64_t cols = t.size(-1), rows = t.numel() / cols;
            const bool one = kind == stream_kind;                     // one gradient serves both summands where they have one type
            if (need_x || (one && need_r)) dx = fresh(t.sizes(), t, x_type);
            if (need_r && !one) dres = fresh(t.sizes(), t);
            if (need_g) dg = rows ? fresh(g.sizes(), g) : at::zeros(g.sizes(), g.options());
            if (rows) {
                const Rows tr(t), dy(grads[0].defined() ? grads[0].resolve_neg() : at::zeros(t.sizes(), t.options().dtype(x_type)));
                Rows ds;
                if (residual && grads.size() > 1 && grads[1].defined()) ds = Rows(grads[1].resolve_neg());
                const Tensor gc = g.contiguous();
                Tensor work;
                const int64_t n = need_g ? L.rms_norm_bwd_work(rows, (int)cols) : 0;
                if (n) work = fresh({n}, g);
                check(L.rms_norm_bwd(dy.p(), dy.ld, ds.p(), ds.ld, tr.p(), tr.ld, (const float*)ptr(r), (const float*)ptr(gc), ptr(dx), cols, ptr(dres), cols,
                                     (float*)ptr(dg), (float*)ptr(work), n, rows, (int)cols, kind, stream_kind, stream->of(t.device())), "vc_rms_norm_bwd");
            }
            if (need_r && one) dres = dx;
            if (!need_x) dx = Tensor();
        }
        return once({dx, dg, dres}, *this, grads, "rms_norm");
    }
};
void norm_inputs(const Tensor& x, const Tensor& gamma, const OptTensor& residual, double eps) {
    activation(x, "x");
    TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) > 0, "x must be [..., channels]");
    TORCH_CHECK_VALUE(eps > 0, "eps must be positive");
    like(gamma, x, "gamma", {x.size(-1)}, at::kFloat);
    if (residual) {
        TORCH_CHECK_VALUE(residual->scalar_type() == x.scalar_type() || residual->scalar_type() == at::kFloat, "residual must be a tensor of ", x.scalar_type(), " or float32");
        like(*residual, x, "residual", x.sizes(), residual->scalar_type());
    }
}
py::object rms_norm(const Tensor& x, const Tensor& gamma, const OptTensor& residual, double eps) {
    norm_inputs(x, gamma, residual, eps);
    const bool keep = wants_grad({x, gamma, residual});
    const Stream s = Stream::now(x.device());
    const int kind = type_code(x), stream_kind = residual ? type_code(*residual) : kind;
    Tensor y, total, rstd;
    {
        at::NoGradGuard ng;
        const c10::DeviceGuard guard(x.device());
        const int64_t cols = x.size(-1), rows = x.numel() / cols;
        const Rows xr(x), rr(residual);
        const Tensor g = gamma.contiguous();
        y = fresh(x.sizes(), x);
        if (residual) total = fresh(x.sizes(), *residual);
        if (keep) rstd = fresh({rows}, gamma);
        check(L.rms_norm_fwd(xr.p(), xr.ld, rr.p(), rr.ld, (const float*)ptr(g), ptr(y), cols, ptr(total), cols, (float*)ptr(rstd), (float)eps, rows, (int)cols,
                             kind, stream_kind, s.handle), "vc_rms_norm_fwd");
    }
    if (keep) {
        auto n = node_for<NormBackward>(x, gamma, or_undefined(residual));
        n->residual = residual.has_value(); n->x_type = x.scalar_type(); n->kind = kind; n->stream_kind = stream_kind; n->stream = s;
        torch::autograd::set_history(y, n);
        if (residual) torch::autograd::set_history(total, n);
        n->total = residual ? SavedVariable(total, true) : SavedVariable(x, false);
        n->gamma = SavedVariable(gamma, false); n->rstd = SavedVariable(rstd, false);
    }
    return residual ? py::object(py::make_tuple(y, total)) : py::cast(y);
}
py::object rms_norm_e4m3(const Tensor& x, const Tensor& gamma, const OptTensor& residual, double eps, int64_t group) {
    norm_inputs(x, gamma, residual, eps);
    const int64_t cols = x.size(-1), rows = x.numel() / cols;
    TORCH_CHECK_VALUE((group == 0 || group == 32 || group == 64 || group == 128) && (group == 0 || cols % group == 0), "group must be 0, 32, 64 or 128 and divide the channels");
    no_grad("rms_norm_e4m3", {x, gamma, residual});
    at::NoGradGuard ng;
    const c10::DeviceGuard guard(x.device());
    const Rows xr(x), rr(residual);
    const Tensor g = gamma.contiguous(), q = fresh(x.sizes(), x, at::kFloat8_e4m3fn);
    auto shape = x.sizes().vec();
    shape.back() = group ? cols / group : 1;
    const Tensor scale = fresh(shape, x, at::kFloat);
    Tensor total;
    if (residual) total = fresh(x.sizes(), *residual);
    check(L.rms_norm_e4m3(xr.p(), xr.ld, rr.p(), rr.ld, (const float*)ptr(g), ptr(q), cols, (float*)ptr(scale), ptr(total), cols, (float)eps, rows, (int)cols,
                          (int)group, type_code(x), residual ? type_code(*residual) : type_code(x), Stream::now(x.device()).handle), "vc_rms_norm_e4m3");
    return residual ? py::object(py::make_tuple(q, scale, total)) : py::object(py::make_tuple(q, scale));
}

// ---- utterances ------------------------------------------------------------------------------------------------------
struct Utterances { int64_t n, rows; };
Utterances utterances(const Tensor& x, const OptTensor& offsets) {
    if (!offsets) {
        TORCH_CHECK_VALUE(x.dim() == 3, "x must be [batch, frames, channels], or [rows, channels] with seq_offsets; got ", x.sizes());
        TORCH_CHECK_VALUE(x.size(0) > 0, "x holds no utterance");
        narrow(x.size(0), "utterances");
        return {x.size(0), x.size(0) * x.size(1)};
    }
    TORCH_CHECK_VALUE(x.dim() == 2, "with seq_offsets x must be [rows, channels], got ", x.sizes());
    TORCH_CHECK_VALUE(offsets->scalar_type() == at::kInt && offsets->device() == x.device() && offsets->dim() == 1 && offsets->numel() >= 2,
                      "seq_offsets must be an int32 tensor [utterances + 1] on ", x.device());
    ordinary(*offsets, "seq_offsets");
    narrow(offsets->numel() - 1, "utterances");
    return {offsets->numel() - 1, x.size(0)};
}
void check_slots(const OptTensor& slots, int64_t rows, int64_t pool, const Tensor& ref) {
    narrow(rows, "streams"); narrow(pool, "states");
    if (slots) like(*slots, ref, "slots", {rows}, at::kInt);
    else TORCH_CHECK_VALUE(rows <= pool, rows, " frames without slots, and a state of ", pool);
}
void moved_on(const Tensor& state) { if (!state.is_inference()) state.unsafeGetTensorImpl()->bump_version(); }     // in place, and autograd is to know

// ---- convolution -----------------------------------------------------------------------------------------------------
void conv_weights(const Tensor& x, const Tensor& w, const OptTensor& bias) {
    const int64_t cols = x.size(-1);
    TORCH_CHECK_VALUE(w.dim() == 2 && w.size(0) >= 2 && w.size(0) <= 8 && w.size(1) == cols, "w must be [taps, ", cols, "] with 2 to 8 taps");
    like(w, x, "w", w.sizes(), at::kFloat);
    like(bias, x, "bias", {cols}, at::kFloat);
}
struct ConvPlan { int64_t n, rows; bool silu; };
// the fields that both passes share, and what keeps their memory
struct ConvCall {
    vc_conv1d_args a{}; Rows x; Tensor w, bias, initial, offsets;
    ConvCall(const Tensor& x_, const Tensor& w_, const OptTensor& bias_, const OptTensor& initial_, const OptTensor& offsets_, const ConvPlan& p)
        : x(Rows(x_).within(conv_ld(x_))), w(w_.contiguous()), bias(plain(bias_)), initial(plain(initial_)), offsets(plain(offsets_)) {
        a.x = x.p(); a.x_ld = x.ld; a.w = (const float*)ptr(w); a.bias = (const float*)ptr(bias); a.initial = ptr(initial); a.offsets = (const int32_t*)ptr(offsets);
        a.rows = p.rows; a.cols = (int)x_.size(-1); a.taps = (int)w.size(0); a.n_seqs = (int)p.n; a.type = type_code(x_); a.silu = p.silu; a.zero_tail = 1;
    }
};
OptTensor optional(const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }
struct ConvBackward : public Node {
    SavedVariable x, w, bias, initial, offsets; ConvPlan plan{}; std::optional<Stream> stream;
    std::string name() const override { return "CausalConv1dBackward"; }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        for (auto* v : {&x, &w, &bias, &initial, &offsets}) v->reset_data();
    }
    variable_list apply(variable_list&& grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        const Tensor xv = x.unpack(), wv = w.unpack(), bv = bias.unpack(), iv = initial.unpack(), ov = offsets.unpack();
        Tensor dx, dw, db, di;
        {
            at::NoGradGuard ng;
            const c10::DeviceGuard guard(xv.device());
            ConvCall k(xv, wv, optional(bv), optional(iv), optional(ov), plan);
            const Rows dy = Rows(grads[0].defined() ? grads[0].resolve_neg() : at::zeros(xv.sizes(), xv.options())).within(conv_ld(xv));
            const Tensor df = grads.size() > 1 && grads[1].defined() ? grads[1].resolve_neg().contiguous() : Tensor();
            if (task_should_compute_output(0)) dx = fresh(xv.sizes(), xv);
            if (task_should_compute_output(1)) dw = fresh(wv.sizes(), wv);
            if (bv.defined() && task_should_compute_output(2)) db = fresh(bv.sizes(), bv);
            if (iv.defined() && task_should_compute_output(3)) di = fresh(iv.sizes(), iv);
            k.a.dy = dy.p(); k.a.dy_ld = dy.ld; k.a.dfinal = ptr(df); k.a.dx = ptr(dx); k.a.dx_ld = k.a.cols; k.a.dw = (float*)ptr(dw); k.a.dbias = (float*)ptr(db);
            k.a.dinitial = ptr(di);
            k.a.work_floats = L.causal_conv1d_bwd_work(&k.a);
            Tensor work;
            if (k.a.work_floats > 0 && (dw.defined() || db.defined())) work = fresh({k.a.work_floats}, wv);
            k.a.work = (float*)ptr(work);
            check(L.causal_conv1d_bwd(&k.a, stream->of(xv.device())), "vc_causal_conv1d_bwd");
        }
        return once({dx, dw, db, di}, *this, grads, "causal_conv1d");
    }
};
py::object causal_conv1d(const Tensor& x, const Tensor& w, const OptTensor& bias, const OptTensor& initial, const OptTensor& offsets, bool silu, bool want_final) {
    activation(x, "x");
    const auto u = utterances(x, offsets);
    conv_weights(x, w, bias);
    if (initial) like(*initial, x, "initial_state", {u.n, w.size(0) - 1, x.size(-1)}, x.scalar_type());
    const ConvPlan plan{u.n, u.rows, silu};
    const Stream s = Stream::now(x.device());
    Tensor y, final;
    {
        at::NoGradGuard ng;
        const c10::DeviceGuard guard(x.device());
        ConvCall k(x, w, bias, initial, offsets, plan);
        y = fresh(x.sizes(), x);
        if (want_final) final = fresh({u.n, w.size(0) - 1, x.size(-1)}, x);
        k.a.y = ptr(y); k.a.y_ld = k.a.cols; k.a.final_state = ptr(final);
        check(L.causal_conv1d_fwd(&k.a, s.handle), "vc_causal_conv1d_fwd");
    }
    if (wants_grad({x, w, bias, initial})) {
        auto n = node_for<ConvBackward>(x, w, or_undefined(bias), or_undefined(initial));
        n->plan = plan; n->stream = s;
        n->x = SavedVariable(x, false); n->w = SavedVariable(w, false); n->bias = SavedVariable(or_undefined(bias), false);
        n->initial = SavedVariable(or_undefined(initial), false); n->offsets = SavedVariable(or_undefined(offsets), false);
        torch::autograd::set_history(y, n);
        if (want_final) torch::autograd::set_history(final, n);
    }
    return want_final ? py::object(py::make_tuple(y, final)) : py::cast(y);
}
Tensor causal_conv1d_step(const Tensor& x, const Tensor& state, const Tensor& w, const OptTensor& bias, const OptTensor& slots, bool silu) {
    activation(x, "x");
    TORCH_CHECK_VALUE(x.dim() == 2 && x.size(1) > 0, "x must be [streams, channels], got ", x.sizes());
    conv_weights(x, w, bias);
    TORCH_CHECK_VALUE(state.dim() == 3, "state must be [pool, taps - 1, channels]");
    like(state, x, "state", {state.size(0), w.size(0) - 1, x.size(1)}, x.scalar_type());
    TORCH_CHECK_VALUE(state.is_contiguous(), "state must be contiguous: it is moved on in place");
    no_grad("causal_conv1d_step", {x, state, w, bias});
    check_slots(slots, x.size(0), state.size(0), x);
    at::NoGradGuard ng;
    const c10::DeviceGuard guard(x.device());
    const Rows xr(x);
    const Tensor wc = w.contiguous(), bc = plain(bias), sc = plain(slots), y = fresh(x.sizes(), x);
    check(L.causal_conv1d_step(xr.p(), xr.ld, ptr(state), (const int32_t*)ptr(sc), (const float*)ptr(wc), (const float*)ptr(bc), ptr(y), x.size(1), (int)x.size(0),
                               (int)state.size(0), (int)x.size(1), (int)w.size(0), type_code(x), silu, Stream::now(x.device()).handle), "vc_causal_conv1d_step");
    moved_on(state);
    return y;
}

// ---- scan ------------------------------------------------------------------------------------------------------------
struct ScanPlan { int64_t n, rows; int max_len; bool softplus; };
void scan_inputs(const Tensor& x, const Tensor& dt, const Tensor& A, const OptTensor& D, const OptTensor& z, const OptTensor& dt_bias) {
    const int64_t cols = x.size(-1);
    like(dt, x, "dt", x.sizes(), x.scalar_type());
    like(z, x, "z", x.sizes(), x.scalar_type());
    TORCH_CHECK_VALUE(A.dim() == 2 && A.size(0) == cols && A.size(1) >= 1 && A.size(1) <= 64, "A must be [", cols, ", states] with 1 to 64 states");
    like(A, x, "A", A.sizes(), at::kFloat);
    like(D, x, "D", {cols}, at::kFloat);
    like(dt_bias, x, "dt_bias", {cols}, at::kFloat);
}
void same_groups(const Grouped& B, const Grouped& C, const Tensor& x) {
    TORCH_CHECK_VALUE(B.groups == C.groups && x.size(-1) % B.groups == 0, "B and C must have the same groups, and these divide the channels");
}
struct ScanCall {
    vc_scan_args a{}; Rows x, dt, z; Grouped B, C; Tensor A, D, dt_bias, initial, offsets;
    ScanCall(const Tensor& x_, const Tensor& dt_, const Tensor& A_, const Tensor& B_, const Tensor& C_, const OptTensor& D_, const OptTensor& z_, const OptTensor& bias_,
             const OptTensor& initial_, const OptTensor& offsets_, const ScanPlan& p)
        : x(Rows(x_).within(SCAN_LD)), dt(Rows(dt_).within(SCAN_LD)), z(Rows(z_).within(SCAN_LD)), B(B_, x_, A_.size(1), "B"), C(C_, x_, A_.size(1), "C"), A(A_.contiguous()), D(plain(D_)), dt_bias(plain(bias_)), initial(plain(initial_)),
          offsets(plain(offsets_)) {
        same_groups(B, C, x_);
        a.x = x.p(); a.dt = dt.p(); a.z = z.p(); a.B = ptr(B.t); a.C = ptr(C.t); a.A = (const float*)ptr(A); a.D = (const float*)ptr(D); a.dt_bias = (const float*)ptr(dt_bias);
        a.initial = (const float*)ptr(initial); a.offsets = (const int32_t*)ptr(offsets);
        a.x_ld = x.ld; a.dt_ld = dt.ld; a.z_ld = z.ld; a.b_ld = B.ld; a.c_ld = C.ld;
        a.rows = p.rows; a.cols = (int)A.size(0); a.states = (int)A.size(1); a.groups = B.groups; a.n_seqs = (int)p.n; a.type = type_code(x_); a.softplus = p.softplus;
        a.zero_tail = 1; a.max_len = p.max_len;
    }
};
struct ScanBackward : public Node {
    SavedVariable x, dt, A, B, C, D, z, dt_bias, initial, offsets, saved; ScanPlan plan{}; std::optional<Stream> stream;
    std::string name() const override { return "SelectiveScanBackward"; }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        for (auto* v : {&x, &dt, &A, &B, &C, &D, &z, &dt_bias, &initial, &offsets, &saved}) v->reset_data();
    }
    variable_list apply(variable_list&& grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        const Tensor xv = x.unpack(), tv = dt.unpack(), Av = A.unpack(), Bv = B.unpack(), Cv = C.unpack(), Dv = D.unpack(), zv = z.unpack(), bv = dt_bias.unpack(),
                     iv = initial.unpack(), ov = offsets.unpack(), sv = saved.unpack();
        Tensor dx, ddt, dA, dB, dC, dD, dz, db, di;
        {
            at::NoGradGuard ng;
            const c10::DeviceGuard guard(xv.device());
            ScanCall k(xv, tv, Av, Bv, Cv, optional(Dv), optional(zv), optional(bv), optional(iv), optional(ov), plan);
            const Rows dy = Rows(grads[0].defined() ? grads[0].resolve_neg() : at::zeros(xv.sizes(), xv.options())).within(SCAN_LD);
            const Tensor df = grads.size() > 1 && grads[1].defined() ? grads[1].resolve_neg().contiguous() : Tensor();
            dx = fresh(xv.sizes(), xv); ddt = fresh(tv.sizes(), xv); dB = fresh(Bv.sizes(), xv); dC = fresh(Cv.sizes(), xv); dA = fresh(Av.sizes(), Av);
            if (zv.defined()) dz = fresh(zv.sizes(), xv);
            if (Dv.defined()) dD = fresh(Dv.sizes(), Av);
            if (bv.defined()) db = fresh(bv.sizes(), Av);
            if (iv.defined()) di = fresh(iv.sizes(), Av);
            auto& a = k.a;
            a.dy = dy.p(); a.dy_ld = dy.ld; a.dfinal = (const float*)ptr(df); a.dx = ptr(dx); a.ddt = ptr(ddt); a.dz = ptr(dz); a.dB = ptr(dB); a.dC = ptr(dC);
            a.dA = (float*)ptr(dA); a.dD = (float*)ptr(dD); a.ddt_bias = (float*)ptr(db); a.dinitial = (float*)ptr(di);
            a.dx_ld = a.ddt_ld = a.dz_ld = a.cols; a.db_ld = a.dc_ld = (int64_t)a.groups * a.states;
            a.saved = (float*)ptr(sv); a.saved_floats = sv.numel();
            a.work_floats = L.selective_scan_bwd_work(&a);
            const Tensor work = fresh({std::max<int64_t>(a.work_floats, 1)}, Av);
            a.work = (float*)ptr(work);
            check(L.selective_scan_bwd(&a, stream->of(xv.device())), "vc_selective_scan_bwd");
        }
        variable_list out{dx, ddt, dA, dB, dC, dD, dz, db, di};
        for (size_t i = 0; i < out.size(); ++i) if (!task_should_compute_output(i)) out[i] = Tensor();
        return once(std::move(out), *this, grads, "selective_scan");
    }
};
py::object selective_scan(const Tensor& x, const Tensor& dt, const Tensor& A, const Tensor& B, const Tensor& C, const OptTensor& D, const OptTensor& z, const OptTensor& dt_bias,
                          const OptTensor& initial, const OptTensor& offsets, int64_t max_len, bool softplus, bool want_final) {
    activation(x, "x");
    const auto u = utterances(x, offsets);
    TORCH_CHECK_VALUE(x.size(-1) > 0, "x has no channels");
    scan_inputs(x, dt, A, D, z, dt_bias);
    if (initial) like(*initial, x, "initial_state", {u.n, A.size(0), A.size(1)}, at::kFloat);
    TORCH_CHECK_VALUE(max_len >= 0, "max_len must not be negative");
    const ScanPlan plan{u.n, u.rows, (int)std::min<int64_t>(max_len, 0x7fffffff), softplus};
    const bool keep = wants_grad({x, dt, A, B, C, D, z, dt_bias, initial});
    const Stream s = Stream::now(x.device());
    Tensor y, final, saved;
    {
        at::NoGradGuard ng;
        const c10::DeviceGuard guard(x.device());
        ScanCall k(x, dt, A, B, C, D, z, dt_bias, initial, offsets, plan);
        auto& a = k.a;
        y = fresh(x.sizes(), x);
        if (want_final) final = fresh({u.n, A.size(0), A.size(1)}, A);
        a.y = ptr(y); a.y_ld = a.cols; a.final_state = (float*)ptr(final);
        if (keep) {
            a.saved_floats = L.selective_scan_saved(&a);
            saved = fresh({std::max<int64_t>(a.saved_floats, 1)}, A);
            a.saved = (float*)ptr(saved);
        }
        a.work_floats = L.selective_scan_fwd_work(&a);
        Tensor work;
        if (a.work_floats > 0) work = fresh({a.work_floats}, A);
        a.work = (float*)ptr(work);
        check(L.selective_scan_fwd(&a, s.handle), "vc_selective_scan_fwd");
    }
    if (keep) {
        auto n = node_for<ScanBackward>(x, dt, A, B, C, or_undefined(D), or_undefined(z), or_undefined(dt_bias), or_undefined(initial));
        n->plan = plan; n->stream = s;
        n->x = SavedVariable(x, false); n->dt = SavedVariable(dt, false); n->A = SavedVariable(A, false); n->B = SavedVariable(B, false); n->C = SavedVariable(C, false);
        n->D = SavedVariable(or_undefined(D), false); n->z = SavedVariable(or_undefined(z), false); n->dt_bias = SavedVariable(or_undefined(dt_bias), false);
        n->initial = SavedVariable(or_undefined(initial), false); n->offsets = SavedVariable(or_undefined(offsets), false); n->saved = SavedVariable(saved, false);
        torch::autograd::set_history(y, n);
        if (want_final) torch::autograd::set_history(final, n);
    }
    return want_final ? py::object(py::make_tuple(y, final)) : py::cast(y);
}
Tensor selective_scan_step(const Tensor& x, const Tensor& dt, const Tensor& A, const Tensor& B, const Tensor& C, const Tensor& state, const OptTensor& D, const OptTensor& z,
                           const OptTensor& dt_bias, const OptTensor& slots, bool softplus) {
    activation(x, "x");
    TORCH_CHECK_VALUE(x.dim() == 2 && x.size(1) > 0, "x must be [streams, channels], got ", x.sizes());
    scan_inputs(x, dt, A, D, z, dt_bias);
    TORCH_CHECK_VALUE(state.dim() == 3, "state must be [pool, channels, states]");
    like(state, x, "state", {state.size(0), A.size(0), A.size(1)}, at::kFloat);
    TORCH_CHECK_VALUE(state.is_contiguous(), "state must be contiguous: it is moved on in place");
    no_grad("selective_scan_step", {x, dt, A, B, C, state, D, z, dt_bias});
    check_slots(slots, x.size(0), state.size(0), x);
    at::NoGradGuard ng;
    const c10::DeviceGuard guard(x.device());
    const Rows xr(x), tr(dt), zr(z);
    const Grouped b(B, x, A.size(1), "B"), c(C, x, A.size(1), "C");
    same_groups(b, c, x);
    const Tensor Ac = A.contiguous(), Dc = plain(D), bc = plain(dt_bias), sc = plain(slots), y = fresh(x.sizes(), x);
    check(L.selective_scan_step(xr.p(), xr.ld, tr.p(), tr.ld, zr.p(), zr.ld, ptr(b.t), b.ld, ptr(c.t), c.ld, (const float*)ptr(Ac), (const float*)ptr(Dc), (const float*)ptr(bc),
                                (float*)ptr(state), (const int32_t*)ptr(sc), ptr(y), x.size(1), (int)x.size(0), (int)state.size(0), (int)x.size(1), (int)A.size(1), b.groups,
                                type_code(x), softplus, Stream::now(x.device()).handle), "vc_selective_scan_step");
    moved_on(state);
    return y;
}
}  // namespace

#ifndef VC_BINDING_ID
#define VC_BINDING_ID "unstamped"
#endif
PYBIND11_MODULE(_seq, m) {
    m.attr("build_id") = VC_BINDING_ID;
    m.def("bind", [](const std::map<std::string, uintptr_t>& at, py::object error, py::object stream) {
#define F(n) L.n = (decltype(L.n))at.at("vc_" #n);
        VC_ENTRIES(F)
#undef F
        vc_error = error.release().ptr();
        raw_stream_of = stream.release().ptr();
    });
    m.def("rms_norm", &rms_norm);
    m.def("rms_norm_e4m3", &rms_norm_e4m3);
    m.def("causal_conv1d", &causal_conv1d);
    m.def("causal_conv1d_step", &causal_conv1d_step);
    m.def("selective_scan", &selective_scan);
    m.def("selective_scan_step", &selective_scan_step);
}
