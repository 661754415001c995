// The torch side of the feature-map and frame-sequence operators: checks of the tensors, outputs and workspaces from torch's
// allocator, torch's current stream, and the call of the C ABI (include/auditory_hip.h), in one native step -- at a few
// microseconds a kernel the same in Python took as long as the kernels.  No arithmetic.  The module holds no library of its
// own: bind() gives it the entry points that auditory_amd.capi has loaded.
#include <torch/extension.h>
#include <c10/hip/HIPStream.h>

#include <cstdint>
#include <string>
#include <tuple>

#include "auditory_hip.h"

namespace {

typedef c10::optional<at::Tensor> Maybe;
typedef at::IntArrayRef Shape;

// the entry points, and the kind of device their memory is on (the CPU for the tests' emulator)
struct Entry {
    decltype(&aud_last_error) last_error;
    decltype(&aud_group_norm_workspace_bytes) norm_bytes;
    decltype(&aud_group_norm_batch_dev) norm;
    decltype(&aud_group_norm_grad_dev) norm_grad;
    decltype(&aud_causal_conv_batch_dev) conv;
    decltype(&aud_causal_conv_workspace_bytes) conv_bytes;
    decltype(&aud_causal_conv_grad_dev) conv_grad;
    decltype(&aud_scan_workspace_bytes) scan_bytes;
    decltype(&aud_scan_kept_floats) scan_kept;
    decltype(&aud_scan_batch_dev) scan;
    decltype(&aud_scan_grad_dev) scan_grad;
    bool on_gpu = true;
} entry;

[[noreturn]] void refuse(int status, const std::string& why) {
    py::object type = py::module_::import("auditory_amd.capi").attr("AuditoryError");
    PyErr_SetObject(type.ptr(), type(status, why).ptr());
    throw py::error_already_set();
}
[[noreturn]] void bad(const std::string& why) { refuse(AUD_EINVAL, why); }

std::string shape_text(Shape s) {
    std::string t = "[";
    for (size_t i = 0; i < s.size(); ++i) t += (i ? ", " : "") + std::to_string(s[i]);
    return t + "]";
}

// Nothing here is recorded for autograd: a tensor that asks for gradients, in a call that autograd would have to record, would
// lose them without a word.
bool asks(const at::Tensor& t) { return t.defined() && t.requires_grad(); }
bool asks(const Maybe& t) { return t && asks(*t); }
template <typename... T>
void no_autograd(const T&... tensors) {
    if (at::GradMode::is_enabled() && (asks(tensors) || ...))
        bad("a tensor of this call requires grad, and the call records nothing for autograd: make it within torch.no_grad() or in "
            "the forward or backward of an autograd.Function (the gradients are a call of their own)");
}

// one call: the tensor that sets type and device, the context
struct Call {
    const at::Tensor& x;
    aud_ctx* ctx;
    int dtype;
    Call(const at::Tensor& t, uintptr_t context, const char* name, int axes, int other_axes) : x(t), ctx(reinterpret_cast<aud_ctx*>(context)) {
        if (t.is_cuda() != entry.on_gpu) bad(std::string(name) + " must be a tensor on a GPU, it is on " + t.device().str());
        switch (t.scalar_type()) {
            case at::kFloat: dtype = AUD_F32; break;
            case at::kBFloat16: dtype = AUD_BF16; break;
            case at::kHalf: dtype = AUD_F16; break;
            default: bad(std::string(name) + " must be float32, bfloat16 or float16, it is " + c10::toString(t.scalar_type()));
        }
        if (t.dim() != axes && t.dim() != other_axes)
            bad(std::string(name) + " must have " + std::to_string(axes) + " axes, it has " + std::to_string(t.dim()));
        for (int64_t n : t.sizes())
            if (n > INT32_MAX) bad(std::string(name) + " has an axis longer than 2^31 - 1: " + shape_text(t.sizes()));
    }
    bool fits(const at::Tensor& t, at::ScalarType type, Shape shape) const {
        return t.scalar_type() == type && t.sizes() == shape && t.device() == x.device();
    }
    [[noreturn]] void unfit(const char* name, at::ScalarType type, Shape shape, const char* how) const {
        bad(std::string(name) + " must be " + how + c10::toString(type) + " " + shape_text(shape) + " on " + x.device().str());
    }
    // an input of x's type whose last `tail` axes are contiguous: item and row stride
    void rows(const at::Tensor& t, const char* name, Shape shape, int tail, int64_t* item, int64_t* row) const {
        if (!fits(t, x.scalar_type(), shape)) unfit(name, x.scalar_type(), shape, "");
        int64_t want = 1;
        const int n = int(shape.size());
        for (int k = 1; k <= tail; ++k) {
            if (shape[n - k] > 1 && t.stride(n - k) != want) bad(std::string("the channels of ") + name + " must be contiguous");
            want *= shape[n - k];
        }
        *item = shape[0] > 1 ? t.stride(0) : 0;
        *row = n - tail > 1 && shape[1] > 1 ? t.stride(1) : want;
    }
    void* dense(const Maybe& t, const char* name, Shape shape) const {
        if (!t) return nullptr;
        if (!fits(*t, x.scalar_type(), shape) || !t->is_contiguous()) unfit(name, x.scalar_type(), shape, "contiguous ");
        return t->data_ptr();
    }
    float* floats(const Maybe& t, const char* name, Shape shape) const {
        if (!t) return nullptr;
        if (!fits(*t, at::kFloat, shape) || !t->is_contiguous()) unfit(name, at::kFloat, shape, "contiguous ");
        return static_cast<float*>(t->data_ptr());
    }
    int32_t* lengths(const Maybe& t, int64_t items) const {
        if (!t) return nullptr;
        if (!fits(*t, at::kInt, {items}) || !t->is_contiguous()) unfit("lengths", at::kInt, {items}, "contiguous ");
        return static_cast<int32_t*>(t->data_ptr());
    }
    at::Tensor fresh(Shape shape) const { return at::empty(shape, x.options()); }
    at::Tensor fresh_floats(Shape shape) const { return at::empty(shape, x.options().dtype(at::kFloat)); }
    at::Tensor out(const Maybe& t) const {
        if (!t) return fresh(x.sizes());
        (void)dense(t, "out", x.sizes());
        return *t;
    }
    // scratch memory: torch's allocator keeps it for this stream (and, in a capture, for this graph) until its kernels have run
    at::Tensor scratch(int64_t bytes) const { return bytes ? at::empty({bytes}, x.options().dtype(at::kByte)) : at::Tensor(); }
    void* stream() const { return entry.on_gpu ? static_cast<void*>(c10::hip::getCurrentHIPStream(x.get_device()).stream()) : nullptr; }
    void done(int rc) const {
        if (rc != AUD_OK) refuse(rc, ctx ? entry.last_error(ctx) : "no context");
    }
};
void* ptr(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
float* fptr(const at::Tensor& t) { return static_cast<float*>(ptr(t)); }
Maybe maybe(const at::Tensor& t) { return t.defined() ? Maybe(t) : Maybe(); }

// ---- group norm ----------------------------------------------------------------------------------------------------------
aud_norm_params norm_params(const Call& c, int64_t groups, int act, double eps) {
    const at::Tensor& x = c.x;
    if (groups < 1 || x.size(2) % groups)
        bad("channels (" + std::to_string(x.size(2)) + ") must be a multiple of groups (" + std::to_string(groups) + ")");
    aud_norm_params p{};
    p.dtype = c.dtype, p.act = act, p.n_items = int(x.size(0)), p.rows = int(x.size(1)), p.channels = int(x.size(2)), p.groups = int(groups);
    p.eps = float(eps);
    c.rows(x, "x", x.sizes(), 1, &p.x_item, &p.x_row);
    return p;
}
std::tuple<at::Tensor, Maybe> group_norm(uintptr_t ctx, const at::Tensor& x, int64_t groups, const Maybe& weight, const Maybe& bias, double eps,
                                         int act, const Maybe& lengths, const Maybe& out, Maybe stats, bool want_stats) {
    no_autograd(x, weight, bias, out, stats);
    const Call c(x, ctx, "x", 3, 3);
    const aud_norm_params p = norm_params(c, groups, act, eps);
    const at::Tensor y = c.out(out);
    if (!stats && want_stats) stats = c.fresh_floats({x.size(0), groups, 2});
    int64_t need = 0;
    (void)entry.norm_bytes(&p, 0, &need);
    const at::Tensor ws = c.scratch(need);
    c.done(entry.norm(c.ctx, &p, x.data_ptr(), c.floats(weight, "weight", {x.size(2)}), c.floats(bias, "bias", {x.size(2)}),
                      c.lengths(lengths, x.size(0)), y.data_ptr(), c.floats(stats, "stats", {x.size(0), groups, 2}), ptr(ws), need, c.stream()));
    return {y, stats};
}
std::tuple<at::Tensor, Maybe, Maybe> group_norm_grad(uintptr_t ctx, const at::Tensor& dy, const at::Tensor& x, const at::Tensor& stats,
                                                     int64_t groups, const Maybe& weight, const Maybe& bias, double eps, int act,
                                                     const Maybe& lengths, const Maybe& out) {
    no_autograd(dy, x, stats, weight, bias, out);
    const Call c(x, ctx, "x", 3, 3);
    aud_norm_params p = norm_params(c, groups, act, eps);
    c.rows(dy, "dy", x.sizes(), 1, &p.dy_item, &p.dy_row);
    const at::Tensor dx = c.out(out);
    at::Tensor dw, db;
    if (weight) dw = c.fresh_floats({x.size(2)});
    if (bias) db = c.fresh_floats({x.size(2)});
    int64_t need = 0;
    (void)entry.norm_bytes(&p, 1, &need);
    const at::Tensor ws = c.scratch(need);
    c.done(entry.norm_grad(c.ctx, &p, dy.data_ptr(), x.data_ptr(), c.floats(stats, "stats", {x.size(0), groups, 2}),
                           c.floats(weight, "weight", {x.size(2)}), c.floats(bias, "bias", {x.size(2)}), c.lengths(lengths, x.size(0)),
                           dx.data_ptr(), fptr(dw), fptr(db), ptr(ws), need, c.stream()));
    return {dx, maybe(dw), maybe(db)};
}

// ---- causal convolution: x [items, steps, channels], or one frame [items, channels] ---------------------------------------
aud_conv_params conv_params(const Call& c, const at::Tensor& weight, int act) {
    const at::Tensor& x = c.x;
    const int64_t channels = x.size(-1);
    if (weight.dim() != 2 || weight.size(0) != channels || weight.size(1) < 1 || weight.size(1) > 4)
        bad("weight must be [" + std::to_string(channels) + ", 1 to 4 taps]");
    aud_conv_params p{};
    p.dtype = c.dtype, p.act = act, p.n_items = int(x.size(0)), p.steps = x.dim() == 3 ? int(x.size(1)) : 1, p.channels = int(channels);
    p.taps = int(weight.size(1));
    c.rows(x, "x", x.sizes(), 1, &p.x_item, &p.x_row);
    return p;
}
at::Tensor causal_conv(uintptr_t ctx, bool one_frame, const at::Tensor& x, const at::Tensor& weight, const Maybe& bias, int act, const Maybe& state,
                       const Maybe& lengths, const Maybe& out, const Maybe& state_out) {
    no_autograd(x, weight, bias, state, out, state_out);
    const int axes = one_frame ? 2 : 3;
    const Call c(x, ctx, "x", axes, axes);
    const aud_conv_params p = conv_params(c, weight, act);
    const int64_t kept[] = {p.n_items, p.taps - 1, p.channels};
    const at::Tensor y = c.out(out);
    c.done(entry.conv(c.ctx, &p, x.data_ptr(), c.floats(weight, "weight", weight.sizes()), c.floats(bias, "bias", {p.channels}),
                      c.dense(state, "state", kept), c.lengths(lengths, p.n_items), y.data_ptr(), c.dense(state_out, "state_out", kept), c.stream()));
    return y;
}
std::tuple<at::Tensor, at::Tensor, Maybe, Maybe> causal_conv_grad(uintptr_t ctx, const at::Tensor& dy, const at::Tensor& x, const at::Tensor& weight,
                                                                  const Maybe& bias, int act, const Maybe& state, const Maybe& lengths,
                                                                  const Maybe& dstate_out, const Maybe& out) {
    no_autograd(dy, x, weight, bias, state, dstate_out, out);
    const Call c(x, ctx, "x", 3, 3);
    aud_conv_params p = conv_params(c, weight, act);
    c.rows(dy, "dy", x.sizes(), 1, &p.dy_item, &p.dy_row);
    const int64_t kept[] = {p.n_items, p.taps - 1, p.channels};
    const at::Tensor dx = c.out(out), dw = c.fresh_floats(weight.sizes());
    at::Tensor db, ds;
    if (bias) db = c.fresh_floats({p.channels});
    if (state) ds = c.fresh(kept);
    int64_t need = 0;
    (void)entry.conv_bytes(&p, &need);
    const at::Tensor ws = c.scratch(need);
    c.done(entry.conv_grad(c.ctx, &p, dy.data_ptr(), x.data_ptr(), c.floats(weight, "weight", weight.sizes()), c.floats(bias, "bias", {p.channels}),
                           c.dense(state, "state", kept), c.lengths(lengths, p.n_items), c.dense(dstate_out, "dstate_out", kept), dx.data_ptr(),
                           fptr(dw), fptr(db), ptr(ds), ptr(ws), need, c.stream()));
    return {dx, dw, maybe(db), maybe(ds)};
}

// ---- selective scan: u [items, steps, channels], B [items, steps, groups, states], or one frame without the steps ------------
struct Scan {
    Call c;
    aud_scan_params p{};
    std::vector<int64_t> vectors;  // the shape of B and C
    Scan(uintptr_t ctx, int axes, const at::Tensor& u, const at::Tensor& delta, const at::Tensor& A, const at::Tensor& B, const at::Tensor& C,
         const Maybe& z, bool softplus)
        : c(u, ctx, "u", axes, axes) {
        const int64_t channels = u.size(-1);
        if (A.dim() != 2 || A.size(0) != channels || A.size(1) < 1 || A.size(1) > 64)
            bad("A must be [" + std::to_string(channels) + ", 1 to 64 states]");
        if (B.dim() != axes + 1) bad(axes == 3 ? "B must be [items, steps, groups, states]" : "B must be [items, groups, states]");
        const int64_t groups = B.size(axes - 1);
        if (groups < 1 || channels % groups)
            bad("channels (" + std::to_string(channels) + ") must be a multiple of groups (" + std::to_string(groups) + ")");
        p.dtype = c.dtype, p.softplus = softplus, p.n_items = int(u.size(0)), p.steps = axes == 3 ? int(u.size(1)) : 1;
        p.channels = int(channels), p.groups = int(groups), p.states = int(A.size(1));
        vectors.assign(u.sizes().begin(), u.sizes().end() - 1);
        vectors.push_back(groups);
        vectors.push_back(A.size(1));
        c.rows(u, "u", u.sizes(), 1, &p.u_item, &p.u_row);
        c.rows(delta, "delta", u.sizes(), 1, &p.delta_item, &p.delta_row);
        p.z_row = p.dy_row = channels;
        if (z) c.rows(*z, "z", u.sizes(), 1, &p.z_item, &p.z_row);
        c.rows(B, "B", vectors, 2, &p.b_item, &p.b_row);
        c.rows(C, "C", vectors, 2, &p.c_item, &p.c_row);
    }
    float* floats(const Maybe& t, const char* name) const { return c.floats(t, name, {p.channels}); }
    float* state(const Maybe& t, const char* name) const { return c.floats(t, name, {p.n_items, p.channels, p.states}); }
    int64_t kept() const {
        int64_t n = 0;
        (void)entry.scan_kept(&p, &n);
        return n;
    }
    int64_t bytes(bool gradients) const {
        int64_t n = 0;
        (void)entry.scan_bytes(&p, gradients, &n);
        return n;
    }
};
std::tuple<at::Tensor, Maybe> selective_scan(uintptr_t ctx, bool one_frame, const at::Tensor& u, const at::Tensor& delta, const at::Tensor& A,
                                             const at::Tensor& B, const at::Tensor& C, const Maybe& D, const Maybe& z, const Maybe& delta_bias,
                                             bool softplus, const Maybe& state, const Maybe& lengths, const Maybe& out, const Maybe& state_out,
                                             bool keep) {
    no_autograd(u, delta, A, B, C, D, z, delta_bias, state, out, state_out);
    const Scan s(ctx, one_frame ? 2 : 3, u, delta, A, B, C, z, softplus);
    const at::Tensor y = s.c.out(out);
    at::Tensor kept;
    if (keep) kept = s.c.fresh_floats({s.kept()});
    const int64_t need = s.bytes(false);
    const at::Tensor ws = s.c.scratch(need);
    s.c.done(entry.scan(s.c.ctx, &s.p, u.data_ptr(), delta.data_ptr(), s.c.floats(A, "A", A.sizes()), B.data_ptr(), C.data_ptr(), s.floats(D, "D"),
                        z ? z->data_ptr() : nullptr, s.floats(delta_bias, "delta_bias"), s.state(state, "state"),
                        s.c.lengths(lengths, s.p.n_items), y.data_ptr(), s.state(state_out, "state_out"), fptr(kept), ptr(ws), need, s.c.stream()));
    return {y, maybe(kept)};
}
py::tuple selective_scan_grad(uintptr_t ctx, const at::Tensor& dy, const at::Tensor& u, const at::Tensor& delta, const at::Tensor& A,
                              const at::Tensor& B, const at::Tensor& C, const at::Tensor& kept, const Maybe& D, const Maybe& z,
                              const Maybe& delta_bias, bool softplus, const Maybe& state, const Maybe& lengths, const Maybe& dstate_out) {
    no_autograd(dy, u, delta, A, B, C, kept, D, z, delta_bias, state, dstate_out);
    Scan s(ctx, 3, u, delta, A, B, C, z, softplus);
    const Call& c = s.c;
    c.rows(dy, "dy", u.sizes(), 1, &s.p.dy_item, &s.p.dy_row);
    (void)s.state(state, "state");
    const at::Tensor du = c.fresh(u.sizes()), dd = c.fresh(u.sizes()), dA = c.fresh_floats(A.sizes()), dB = c.fresh(s.vectors),
                     dC = c.fresh(s.vectors);
    at::Tensor dD, dz, dbias, dstate;
    if (z) dz = c.fresh(u.sizes());
    if (D) dD = c.fresh_floats({s.p.channels});
    if (delta_bias) dbias = c.fresh_floats({s.p.channels});
    if (state) dstate = c.fresh_floats({s.p.n_items, s.p.channels, s.p.states});
    const int64_t need = s.bytes(true);
    const at::Tensor ws = c.scratch(need);
    c.done(entry.scan_grad(c.ctx, &s.p, dy.data_ptr(), u.data_ptr(), delta.data_ptr(), c.floats(A, "A", A.sizes()), B.data_ptr(), C.data_ptr(),
                           s.floats(D, "D"), z ? z->data_ptr() : nullptr, s.floats(delta_bias, "delta_bias"), c.lengths(lengths, s.p.n_items),
                           c.floats(kept, "kept", {s.kept()}), s.state(dstate_out, "dstate_out"), du.data_ptr(), dd.data_ptr(), fptr(dA),
                           dB.data_ptr(), dC.data_ptr(), fptr(dD), ptr(dz), fptr(dbias), fptr(dstate), ptr(ws), need, c.stream()));
    return py::make_tuple(du, dd, dA, dB, dC, maybe(dD), maybe(dz), maybe(dbias), maybe(dstate));
}

template <typename F>
void take(const py::dict& at, const char* name, F& f) {
    f = reinterpret_cast<F>(at[name].cast<uintptr_t>());
}
void bind(const py::dict& at, bool on_gpu) {
    take(at, "aud_last_error", entry.last_error);
    take(at, "aud_group_norm_workspace_bytes", entry.norm_bytes);
    take(at, "aud_group_norm_batch_dev", entry.norm);
    take(at, "aud_group_norm_grad_dev", entry.norm_grad);
    take(at, "aud_causal_conv_batch_dev", entry.conv);
    take(at, "aud_causal_conv_workspace_bytes", entry.conv_bytes);
    take(at, "aud_causal_conv_grad_dev", entry.conv_grad);
    take(at, "aud_scan_workspace_bytes", entry.scan_bytes);
    take(at, "aud_scan_kept_floats", entry.scan_kept);
    take(at, "aud_scan_batch_dev", entry.scan);
    take(at, "aud_scan_grad_dev", entry.scan_grad);
    entry.on_gpu = on_gpu;
}

}  // namespace

PYBIND11_MODULE(_frames, m) {
    m.def("bind", &bind);
    m.def("group_norm", &group_norm);
    m.def("group_norm_grad", &group_norm_grad);
    m.def("causal_conv", &causal_conv);
    m.def("causal_conv_grad", &causal_conv_grad);
    m.def("selective_scan", &selective_scan);
    m.def("selective_scan_grad", &selective_scan_grad);
}
