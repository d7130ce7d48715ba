// selective_scan, causal_conv, their steps and rms_norm (scan.py, norm.py) without the interpreter: argument checks, allocations and autograd nodes in C++ around the entry
// points of libvrwkv_hip.so.  As in host_ops.cpp they take the plain case and answer None to everything else: the Python functions go on by themselves.
#include <optional>
#include "host_common.h"

using namespace host;

namespace {
const at::Tensor none;

// The tensor of an argument that may be None (an undefined one then); nullptr where Python has to decide.
const at::Tensor* optional(py::handle o) { return o.is_none() ? &none : strided(o); }
std::optional<at::Tensor> given(const at::Tensor& t) { return t.defined() ? std::optional<at::Tensor>(t) : std::nullopt; }
void* pointer(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
bool on(const at::Tensor& t, const at::Tensor& like) { return !t.defined() || (t.device() == like.device() && !tangent(t)); }
bool wanted(const at::Tensor& t) { return t.defined() && t.requires_grad(); }

// rows of channels (lead dimensions, then groups or channels): what the kernels read as it lies
bool rows_fit(const at::Tensor& t, int dim) { return t.dim() == dim && t.numel() > 0 && t.stride(-1) == 1 && (dim == 2 || t.size(1) == 1 || t.stride(1) < (1 << 22)) && t.size(0) <= INT_MAX && t.size(1) <= INT_MAX; }
void row_strides(const at::Tensor& t, long long* to) {
    to[0] = t.stride(0), to[1] = t.size(1) == 1 ? 0 : t.stride(1);
    if (t.dim() == 4) to[2] = t.stride(2);
}
// (E) or (E, n) in the rows' type or fp32, contiguous
bool param_fits(const at::Tensor& t, const at::Tensor& like, int64_t E) {
    return !t.defined() || (t.dim() >= 1 && t.size(0) == E && t.is_contiguous() && (t.scalar_type() == at::kFloat || t.scalar_type() == like.scalar_type()));
}
at::Tensor like_of(const at::Tensor& t) { return at::empty(t.sizes(), t.options().requires_grad(false)); }

// Saved tensors that a hook has changed, and gradients, as the kernels take them.
at::Tensor rows_of(at::Tensor t, const at::Tensor& like) {
    TORCH_CHECK(t.defined() && t.has_storage() && t.is_cuda() && t.device() == like.device() && t.scalar_type() == like.scalar_type() && t.dim() >= 3,
                "the saved tensors and the gradient must be CUDA tensors of one type on one device");
    if (t.is_neg()) t = t.resolve_neg();
    return rows_fit(t, (int)t.dim()) ? t : t.contiguous();
}
at::Tensor own_of(const at::Tensor& t, const at::Tensor& like) {
    if (!t.defined()) return t;
    TORCH_CHECK(t.has_storage() && t.is_cuda() && t.device() == like.device(), "the saved tensors must be CUDA tensors on one device");
    return (t.is_neg() ? t.resolve_neg() : t).contiguous();
}
bool sequences_fit(const at::Tensor& x, const at::Tensor& offsets, int64_t& N) {
    N = x.size(0);
    if (!offsets.defined()) return true;
    N = offsets.numel() - 1;
    return index_fits(offsets, x) && x.size(0) == 1 && N >= 1 && N <= INT_MAX;
}
bool state_fits(const at::Tensor& t, at::ScalarType type, const at::Tensor& like, std::initializer_list<int64_t> sizes) {
    return !t.defined() || (t.scalar_type() == type && t.is_contiguous() && t.device() == like.device() && t.sizes() == at::IntArrayRef(sizes));
}
// Which of the recorded call's tensors, in their order, want a gradient: absent ones have no place in the engine's count.
struct Wanted {
    AutogradContext* ctx;
    size_t at = 0;
    bool operator()(const at::Tensor& t) { return t.defined() && ctx->needs_input_grad(at++); }
};
#define CHECK_LIBRARY(call)                                                                            \
    do {                                                                                               \
        const int rc = call;                                                                           \
        TORCH_CHECK(rc == VRWKV_OK, "vrwkv status ", rc, ": ", vrwkv_last_error());                    \
    } while (0)

// ---- the convolution -----------------------------------------------------------------------------------------------------
vrwkv_conv_args conv_args(const at::Tensor& x, const at::Tensor& w, const at::Tensor& b, const at::Tensor& state, const at::Tensor& offsets, bool silu, int64_t N) {
    vrwkv_conv_args a = {};
    a.x = x.data_ptr(), a.weight = w.data_ptr(), a.bias = pointer(b), a.state = pointer(state), a.offsets = pointer(offsets);
    row_strides(x, a.x_stride);
    a.N = (int)N, a.T = (int)x.size(1), a.E = (int)x.size(2), a.K = (int)w.size(1), a.dtype = code(x.scalar_type()), a.param_dtype = code(w.scalar_type()), a.silu = silu;
    a.offsets64 = offsets.defined() && offsets.scalar_type() == at::kLong;
    return a;
}
bool conv_fits(const at::Tensor& x, const at::Tensor& w, const at::Tensor& b, int dim) {
    const int64_t E = x.dim() == dim ? x.size(-1) : 0;
    return rows_fit(x, dim) && code(x.scalar_type()) >= 0 && w.dim() == 2 && param_fits(w, x, E) && w.size(1) >= 2 && w.size(1) <= 8 && w.device() == x.device() && E <= INT_MAX &&
           (!b.defined() || (b.dim() == 1 && param_fits(b, x, E) && b.scalar_type() == w.scalar_type() && b.device() == x.device()));
}

struct Conv : torch::autograd::Function<Conv> {
    struct Call {
        at::Tensor y, last, offsets;
        bool silu;
        int64_t N;
    };
    static tensor_list forward(AutogradContext* ctx, const Variable& x, const Variable& w, const std::optional<at::Tensor>& b, const std::optional<at::Tensor>& state, const Call* c) {
        ctx->save_for_backward({x, w, b.value_or(none), state.value_or(none), c->offsets});
        ctx->saved_data["silu"] = c->silu;
        ctx->saved_data["N"] = c->N;
        ctx->set_materialize_grads(false);
        return c->last.defined() ? tensor_list{c->y, c->last} : tensor_list{c->y};
    }
    static tensor_list backward(AutogradContext* ctx, tensor_list grads) {
        const bool recorded = at::GradMode::is_enabled();
        tensor_list out(5);
        {
            at::NoGradGuard no_grad;
            const auto saved = ctx->get_saved_variables();
            const at::Tensor x = rows_of(saved[0], saved[0]), w = own_of(saved[1], x), b = own_of(saved[2], x), state = own_of(saved[3], x), offsets = own_of(saved[4], x);
            int64_t N = 0;
            TORCH_CHECK(conv_fits(x, w, b, 3) && sequences_fit(x, offsets, N) && N == ctx->saved_data["N"].toInt() && state_fits(state, x.scalar_type(), x, {N, w.size(1) - 1, x.size(2)}),
                        "the saved tensors have other sizes or types than those of the call");
            at::Tensor gy = grads[0], glast = grads.size() > 1 ? grads[1] : at::Tensor();
            if (!gy.defined() && !glast.defined()) return out;
            Guard guard(x.device());
            gy = gy.defined() ? rows_of(gy.to(x.scalar_type()), x) : at::zeros(x.sizes(), x.options().requires_grad(false));
            if (glast.defined()) glast = own_of(glast.to(x.scalar_type()), x);
            TORCH_CHECK(gy.sizes() == x.sizes(), "the gradient must have the shape of y");
            vrwkv_conv_args a = conv_args(x, w, b, state, offsets, ctx->saved_data["silu"].toBool(), N);
            a.gy = gy.data_ptr(), a.glast = pointer(glast);
            row_strides(gy, a.gy_stride);
            Wanted want{ctx};
            want(x), want(w);
            out[0] = like_of(x), out[1] = like_of(w);
            if (want(b)) out[2] = like_of(b);
            if (want(state)) out[3] = like_of(state);
            a.dx = out[0].data_ptr(), a.dweight = out[1].data_ptr(), a.dbias = pointer(out[2]), a.dstate = pointer(out[3]);
            a.workspace_bytes = vrwkv_conv_bwd_workspace_bytes(&a);
            const at::Tensor ws = bytes(a.workspace_bytes, x);
            a.workspace = ws.data_ptr();
            CHECK_LIBRARY(vrwkv_conv_bwd(&a, stream_of(x)));
        }
        if (recorded) only_once(out);
        return out;
    }
};

// y or (y, last)
py::object result(const tensor_list& out, bool keep) {
    if (out.empty()) return py::none();
    if (!keep) return wrapped(out[0]);
    return py::make_tuple(wrapped(out[0]), wrapped(out[1]));
}

py::object causal_conv(py::handle x_, py::handle w_, py::handle b_, bool silu, py::handle state_, py::handle offsets_, bool keep) {
    if (transformed()) return py::none();
    const at::Tensor *xp = strided(x_), *wp = strided(w_), *bp = optional(b_), *sp = optional(state_), *op = optional(offsets_);
    if (!xp || !wp || !bp || !sp || !op) return py::none();
    const at::Tensor &x = *xp, &w = *wp, &b = *bp, &state = *sp, &offsets = *op;
    int64_t N = 0;
    if (!conv_fits(x, w, b, 3) || x.get_device() != c10::hip::current_device() || !on(x, x) || !on(w, x) || !on(b, x) || !on(state, x) || !sequences_fit(x, offsets, N) ||
        !state_fits(state, x.scalar_type(), x, {N, w.size(1) - 1, x.size(2)}))
        return py::none();
    tensor_list out;
    {
        py::gil_scoped_release release;
        Guard guard(x.device());
        Conv::Call c{at::empty(x.sizes(), x.options().requires_grad(false)), {}, offsets, silu, N};
        vrwkv_conv_args a = conv_args(x, w, b, state, offsets, silu, N);
        a.y = c.y.data_ptr();
        if (keep) a.last = (c.last = at::empty({N, w.size(1) - 1, x.size(2)}, x.options().requires_grad(false))).data_ptr();
        const bool done = vrwkv_conv_fwd(&a, stream_of(x)) == VRWKV_OK;
        if (done && at::GradMode::is_enabled() && (wanted(x) || wanted(w) || wanted(b) || wanted(state))) out = Conv::apply(x, w, given(b), given(state), &c);
        else if (done) out = {c.y, c.last};
    }
    return result(out, keep);
}

// What a step's pool and slots have to be: the pages, and how far apart they are.
bool pool_fits(const at::Tensor& pool, const at::Tensor& slots, const at::Tensor& like, at::ScalarType type, int64_t rows, int64_t d1, int64_t d2) {
    return pool.dim() == 3 && pool.size(0) > 0 && pool.size(0) <= INT_MAX && pool.size(1) == d1 && pool.size(2) == d2 && pool.scalar_type() == type && pool.device() == like.device() && !tangent(pool) &&
           pages_fit(pool) && (!slots.defined() || (index_fits(slots, like) && slots.numel() == rows));
}
void changed(const at::Tensor& pool) {
    if (!pool.is_inference()) pool.unsafeGetTensorImpl()->bump_version();
}

py::object causal_conv_step(py::handle x_, py::handle w_, py::handle pool_, py::handle slots_, py::handle b_, bool silu) {
    if (transformed()) return py::none();
    const at::Tensor *xp = strided(x_), *wp = strided(w_), *bp = optional(b_), *pp = strided(pool_), *sp = optional(slots_);
    if (!xp || !wp || !bp || !pp || !sp) return py::none();
    const at::Tensor &x = *xp, &w = *wp, &b = *bp, &pool = *pp, &slots = *sp;
    if (!conv_fits(x, w, b, 2) || x.get_device() != c10::hip::current_device() || !on(x, x) || !on(w, x) || !on(b, x) ||
        !pool_fits(pool, slots, x, x.scalar_type(), x.size(0), w.size(1) - 1, x.size(1)) || (at::GradMode::is_enabled() && (wanted(x) || wanted(w) || wanted(b) || wanted(pool))))
        return py::none();
    Guard guard(x.device());
    const at::Tensor y = at::empty(x.sizes(), x.options().requires_grad(false));
    vrwkv_conv_step_args a = {};
    a.x = x.data_ptr(), a.weight = w.data_ptr(), a.bias = pointer(b), a.slots = pointer(slots), a.pool = pool.data_ptr(), a.y = y.data_ptr(), a.x_stride = x.stride(0);
    a.N = (int)x.size(0), a.P = (int)pool.size(0), a.E = (int)x.size(1), a.K = (int)w.size(1), a.dtype = code(x.scalar_type()), a.param_dtype = code(w.scalar_type()), a.silu = silu;
    a.slots64 = slots.defined() && slots.scalar_type() == at::kLong;
    a.page_stride = pool.size(0) > 1 ? pool.stride(0) : pool.size(1) * pool.size(2);
    if (vrwkv_conv_step(&a, stream_of(x)) != VRWKV_OK) return py::none();
    changed(pool);
    return wrapped(y);
}

// ---- the scan ------------------------------------------------------------------------------------------------------------
// The tensors of a call, in the order of its arguments: u, delta, A, B, C, D, z, delta_bias, state.
struct ScanTensors {
    at::Tensor u, delta, A, B, C, D, z, bias, state;
    at::Tensor offsets;
    int64_t groups(int lead) const { return B.dim() == lead + 2 ? B.size(lead) : 1; }
    bool fit(int lead) const {
        const int64_t E = u.dim() == lead + 1 ? u.size(-1) : 0;
        if (!rows_fit(u, lead + 1) || code(u.scalar_type()) < 0 || E > INT_MAX || A.dim() != 2 || A.size(0) != E || A.scalar_type() != at::kFloat || !A.is_contiguous() || A.size(1) < 1 || A.size(1) > 64) return false;
        for (const at::Tensor* t : {&delta, &z})
            if (t->defined() && (t->sizes() != u.sizes() || t->scalar_type() != u.scalar_type() || !rows_fit(*t, lead + 1))) return false;
        if (B.dim() != C.dim() || (B.dim() != lead + 1 && B.dim() != lead + 2)) return false;
        for (const at::Tensor* t : {&B, &C}) {
            if (t->scalar_type() != u.scalar_type() || !rows_fit(*t, (int)B.dim()) || t->size(-1) != A.size(1) || t->size(0) != u.size(0) || (lead == 2 && t->size(1) != u.size(1)) || t->sizes() != B.sizes()) return false;
        }
        if (groups(lead) < 1 || E % groups(lead)) return false;
        for (const at::Tensor* t : {&D, &bias})
            if (t->defined() && (t->dim() != 1 || !param_fits(*t, u, E))) return false;
        for (const at::Tensor* t : {&delta, &A, &B, &C, &D, &z, &bias, &state})
            if (t->defined() && t->device() != u.device()) return false;
        return true;
    }
    bool tangents() const {
        for (const at::Tensor* t : {&u, &delta, &A, &B, &C, &D, &z, &bias, &state})
            if (t->defined() && tangent(*t)) return true;
        return false;
    }
    bool any_wanted() const {
        for (const at::Tensor* t : {&u, &delta, &A, &B, &C, &D, &z, &bias, &state})
            if (wanted(*t)) return true;
        return false;
    }
    vrwkv_scan_args args(bool softplus, int64_t N) const {
        vrwkv_scan_args a = {};
        a.u = u.data_ptr(), a.delta = delta.data_ptr(), a.A = (const float*)A.data_ptr(), a.B = B.data_ptr(), a.C = C.data_ptr(), a.D = pointer(D), a.z = pointer(z), a.delta_bias = pointer(bias);
        a.state = (const float*)pointer(state), a.offsets = pointer(offsets);
        row_strides(u, a.u_stride), row_strides(delta, a.delta_stride), row_strides(B, a.B_stride), row_strides(C, a.C_stride);
        if (z.defined()) row_strides(z, a.z_stride);
        a.N = (int)N, a.T = (int)u.size(1), a.E = (int)u.size(2), a.S = (int)A.size(1), a.G = (int)groups(2), a.dtype = code(u.scalar_type()), a.softplus = softplus;
        a.D_dtype = D.defined() ? code(D.scalar_type()) : 0, a.bias_dtype = bias.defined() ? code(bias.scalar_type()) : 0;
        a.offsets64 = offsets.defined() && offsets.scalar_type() == at::kLong;
        return a;
    }
};

struct Scan : torch::autograd::Function<Scan> {
    struct Call {
        at::Tensor y, last, kept, offsets;
        bool softplus;
        int64_t N;
    };
    typedef const std::optional<at::Tensor>& Maybe;
    static tensor_list forward(AutogradContext* ctx, const Variable& u, const Variable& delta, const Variable& A, const Variable& B, const Variable& C, Maybe D, Maybe z, Maybe bias, Maybe state, const Call* c) {
        ctx->save_for_backward({u, delta, A, B, C, D.value_or(none), z.value_or(none), bias.value_or(none), state.value_or(none), c->offsets, c->kept});
        ctx->saved_data["softplus"] = c->softplus;
        ctx->saved_data["N"] = c->N;
        ctx->set_materialize_grads(false);
        return c->last.defined() ? tensor_list{c->y, c->last} : tensor_list{c->y};
    }
    static tensor_list backward(AutogradContext* ctx, tensor_list grads) {
        const bool recorded = at::GradMode::is_enabled();
        tensor_list out(10);
        {
            at::NoGradGuard no_grad;
            const auto saved = ctx->get_saved_variables();
            const at::Tensor u = rows_of(saved[0], saved[0]);
            ScanTensors t{u, rows_of(saved[1], u), own_of(saved[2], u), rows_of(saved[3], u), rows_of(saved[4], u), own_of(saved[5], u), saved[6].defined() ? rows_of(saved[6], u) : none,
                          own_of(saved[7], u), own_of(saved[8], u), own_of(saved[9], u)};
            const at::Tensor kept = own_of(saved[10], u);
            int64_t N = 0;
            TORCH_CHECK(t.fit(2) && sequences_fit(u, t.offsets, N) && N == ctx->saved_data["N"].toInt() && state_fits(t.state, at::kFloat, u, {N, u.size(2), t.A.size(1)}),
                        "the saved tensors have other sizes or types than those of the call");
            at::Tensor gy = grads[0], glast = grads.size() > 1 ? grads[1] : at::Tensor();
            if (!gy.defined() && !glast.defined()) return out;
            Guard guard(u.device());
            vrwkv_scan_args a = t.args(ctx->saved_data["softplus"].toBool(), N);
            TORCH_CHECK(kept.scalar_type() == at::kFloat && (size_t)kept.numel() * 4 == vrwkv_scan_kept_bytes(&a), "the saved tensors have other sizes or types than those of the call");
            gy = gy.defined() ? rows_of(gy.to(u.scalar_type()), u) : at::zeros(u.sizes(), u.options().requires_grad(false));
            if (glast.defined()) glast = own_of(glast.to(at::kFloat), u);
            TORCH_CHECK(gy.sizes() == u.sizes(), "the gradient must have the shape of y");
            a.kept = (float*)kept.data_ptr(), a.gy = gy.data_ptr(), a.glast = (const float*)pointer(glast);
            row_strides(gy, a.gy_stride);
            const at::Tensor* const like[9] = {&t.u, &t.delta, &t.A, &t.B, &t.C, &t.D, &t.z, &t.bias, &t.state};
            Wanted want{ctx};
            for (int i = 0; i < 9; ++i) {
                const bool w = want(*like[i]);
                if (like[i]->defined() && (w || i < 5 || i == 6)) out[i] = like_of(*like[i]);
            }
            a.du = out[0].data_ptr(), a.ddelta = out[1].data_ptr(), a.dA = (float*)out[2].data_ptr(), a.dB = out[3].data_ptr(), a.dC = out[4].data_ptr(), a.dD = pointer(out[5]), a.dz = pointer(out[6]);
            a.dbias = pointer(out[7]), a.dstate = (float*)pointer(out[8]);
            a.workspace_bytes = vrwkv_scan_bwd_workspace_bytes(&a);
            const at::Tensor ws = bytes(a.workspace_bytes, u);
            a.workspace = ws.data_ptr();
            CHECK_LIBRARY(vrwkv_scan_bwd(&a, stream_of(u)));
        }
        if (recorded) only_once(out);
        return out;
    }
};

bool scan_tensors(py::handle u, py::handle delta, py::handle A, py::handle B, py::handle C, py::handle D, py::handle z, py::handle bias, py::handle state, py::handle offsets, ScanTensors& t) {
    const at::Tensor* p[10] = {strided(u), strided(delta), strided(A), strided(B), strided(C), optional(D), optional(z), optional(bias), optional(state), optional(offsets)};
    for (const at::Tensor* x : p)
        if (!x) return false;
    t = ScanTensors{*p[0], *p[1], *p[2], *p[3], *p[4], *p[5], *p[6], *p[7], *p[8], *p[9]};
    return true;
}

py::object selective_scan(py::handle u_, py::handle delta, py::handle A, py::handle B, py::handle C, py::handle D, py::handle z, py::handle bias, bool softplus, py::handle state, py::handle offsets, bool keep) {
    ScanTensors t;
    int64_t N = 0;
    if (transformed() || !scan_tensors(u_, delta, A, B, C, D, z, bias, state, offsets, t) || !t.fit(2) || t.u.get_device() != c10::hip::current_device() || t.tangents() ||
        !sequences_fit(t.u, t.offsets, N) || !state_fits(t.state, at::kFloat, t.u, {N, t.u.size(2), t.A.size(1)}))
        return py::none();
    tensor_list out;
    {
        py::gil_scoped_release release;
        const at::Tensor& u = t.u;
        Guard guard(u.device());
        const auto floats = u.options().dtype(at::kFloat).requires_grad(false);
        Scan::Call c{at::empty(u.sizes(), u.options().requires_grad(false)), {}, {}, t.offsets, softplus, N};
        vrwkv_scan_args a = t.args(softplus, N);
        a.y = c.y.data_ptr();
        if (keep) a.last = (float*)(c.last = at::empty({N, u.size(2), t.A.size(1)}, floats)).data_ptr();
        const bool record = at::GradMode::is_enabled() && t.any_wanted();
        if (record) a.kept = (float*)(c.kept = at::empty({(int64_t)(vrwkv_scan_kept_bytes(&a) / 4)}, floats)).data_ptr();
        at::Tensor ws;
        a.workspace_bytes = vrwkv_scan_fwd_workspace_bytes(&a);
        if (a.workspace_bytes) a.workspace = (ws = bytes(a.workspace_bytes, u)).data_ptr();
        const bool done = vrwkv_scan_fwd(&a, stream_of(u)) == VRWKV_OK;
        if (done && record) out = Scan::apply(t.u, t.delta, t.A, t.B, t.C, given(t.D), given(t.z), given(t.bias), given(t.state), &c);
        else if (done) out = {c.y, c.last};
        t = ScanTensors();                                 // (references go without the interpreter's lock)
    }
    return result(out, keep);
}

py::object selective_scan_step(py::handle u_, py::handle delta_, py::handle A_, py::handle B_, py::handle C_, py::handle pool_, py::handle slots_, py::handle D_, py::handle z_, py::handle bias_, bool softplus) {
    ScanTensors t;
    const at::Tensor *pp = strided(pool_), *sp = optional(slots_);
    if (transformed() || !pp || !sp || !scan_tensors(u_, delta_, A_, B_, C_, D_, z_, bias_, py::none(), py::none(), t) || !t.fit(1) || t.u.get_device() != c10::hip::current_device() || t.tangents()) return py::none();
    const at::Tensor &u = t.u, &pool = *pp, &slots = *sp;
    if (!pool_fits(pool, slots, u, at::kFloat, u.size(0), u.size(1), t.A.size(1)) || (at::GradMode::is_enabled() && (t.any_wanted() || wanted(pool)))) return py::none();
    Guard guard(u.device());
    const at::Tensor y = at::empty(u.sizes(), u.options().requires_grad(false));
    vrwkv_scan_step_args a = {};
    a.u = u.data_ptr(), a.delta = t.delta.data_ptr(), a.A = (const float*)t.A.data_ptr(), a.B = t.B.data_ptr(), a.C = t.C.data_ptr(), a.D = pointer(t.D), a.z = pointer(t.z), a.delta_bias = pointer(t.bias);
    a.slots = pointer(slots), a.pool = (float*)pool.data_ptr(), a.y = y.data_ptr();
    a.u_stride = u.stride(0), a.delta_stride = t.delta.stride(0), a.z_stride = t.z.defined() ? t.z.stride(0) : 0;
    a.B_stride[0] = t.B.stride(0), a.C_stride[0] = t.C.stride(0);
    if (t.B.dim() == 3) a.B_stride[1] = t.B.stride(1), a.C_stride[1] = t.C.stride(1);
    a.page_stride = pool.size(0) > 1 ? pool.stride(0) : pool.size(1) * pool.size(2);
    a.N = (int)u.size(0), a.P = (int)pool.size(0), a.E = (int)u.size(1), a.S = (int)t.A.size(1), a.G = (int)t.groups(1), a.dtype = code(u.scalar_type()), a.softplus = softplus;
    a.D_dtype = t.D.defined() ? code(t.D.scalar_type()) : 0, a.bias_dtype = t.bias.defined() ? code(t.bias.scalar_type()) : 0;
    a.slots64 = slots.defined() && slots.scalar_type() == at::kLong;
    if (vrwkv_scan_step(&a, stream_of(u)) != VRWKV_OK) return py::none();
    changed(pool);
    return wrapped(y);
}

// ---- the norm ------------------------------------------------------------------------------------------------------------
bool norm_fits(const at::Tensor& x, const at::Tensor& w, const at::Tensor& residual) {
    return x.dim() >= 1 && x.numel() > 0 && x.is_contiguous() && code(x.scalar_type()) >= 0 && w.dim() == 1 && param_fits(w, x, x.size(-1)) && w.device() == x.device() && x.size(-1) <= INT_MAX &&
           x.numel() / x.size(-1) < INT_MAX &&
           (!residual.defined() || (residual.sizes() == x.sizes() && residual.is_contiguous() && (residual.scalar_type() == x.scalar_type() || residual.scalar_type() == at::kFloat) && residual.device() == x.device()));
}
vrwkv_rmsnorm_args norm_args(const at::Tensor& w, int64_t C, int64_t rows, at::ScalarType type, at::ScalarType residual_type, double eps) {
    vrwkv_rmsnorm_args a = {};
    a.weight = w.data_ptr(), a.C = (int)C, a.rows = rows, a.eps = (float)eps, a.dtype = code(type), a.residual_dtype = code(residual_type), a.weight_dtype = code(w.scalar_type());
    a.x_stride = a.residual_stride = a.gy_stride = a.gsum_stride = C;
    return a;
}

struct Norm : torch::autograd::Function<Norm> {
    struct Call {
        at::Tensor y, r;
        double eps;
    };
    static tensor_list forward(AutogradContext* ctx, const Variable& x, const Variable& w, const std::optional<at::Tensor>& residual, const Call* c) {
        ctx->save_for_backward({residual ? c->r : x, w});
        ctx->saved_data["eps"] = c->eps;
        ctx->saved_data["type"] = (int64_t)x.scalar_type();
        ctx->saved_data["sizes"] = x.sizes().vec();
        ctx->saved_data["residual"] = residual.has_value();
        ctx->set_materialize_grads(false);
        return residual ? tensor_list{c->y, c->r} : tensor_list{c->y};
    }
    static tensor_list backward(AutogradContext* ctx, tensor_list grads) {
        const bool recorded = at::GradMode::is_enabled();
        tensor_list out(4);
        {
            at::NoGradGuard no_grad;
            const auto saved = ctx->get_saved_variables();
            const auto type = (at::ScalarType)ctx->saved_data["type"].toInt();
            const auto sizes = ctx->saved_data["sizes"].toIntVector();
            const bool has_residual = ctx->saved_data["residual"].toBool();
            TORCH_CHECK(saved[0].defined() && saved[0].is_cuda(), "the saved tensors must be CUDA tensors on one device");
            const at::Tensor r = own_of(saved[0], saved[0]), w = own_of(saved[1], r);
            const int64_t C = sizes.back();
            TORCH_CHECK(r.sizes() == at::IntArrayRef(sizes) && (r.scalar_type() == type || (has_residual && r.scalar_type() == at::kFloat)) && w.defined() && w.dim() == 1 && w.size(0) == C && code(w.scalar_type()) >= 0,
                        "the saved tensors have other sizes or types than those of the call");
            at::Tensor gy = grads[0], gr = grads.size() > 1 ? grads[1] : at::Tensor();
            if (!gy.defined() && !gr.defined()) return out;
            Guard guard(r.device());
            const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1), need_r = has_residual && ctx->needs_input_grad(2);
            if (gr.defined()) gr = own_of(gr.to(r.scalar_type()), r);
            if (!gy.defined()) {                           // the sum's gradient alone
                out[0] = gr.to(type);
                if (need_r) out[2] = gr;
                if (need_w) out[1] = at::zeros(w.sizes(), w.options().requires_grad(false));
            } else {
                gy = own_of(gy.to(type), r);
                TORCH_CHECK(gy.sizes() == r.sizes(), "the gradient must have the shape of y");
                vrwkv_rmsnorm_args a = norm_args(w, C, r.numel() / C, type, r.scalar_type(), ctx->saved_data["eps"].toDouble());
                a.sum = r.data_ptr(), a.gy = gy.data_ptr(), a.gsum = pointer(gr);
                if (need_x || !need_r) out[0] = at::empty(sizes, r.options().dtype(type).requires_grad(false));
                if (need_r) out[2] = out[0].defined() && r.scalar_type() == type ? out[0] : like_of(r);   // (one tensor for both where they are of one type, as an addition's are)
                if (need_w) out[1] = like_of(w);
                a.dx = pointer(out[0]), a.dresidual = out[2].defined() && !out[2].is_same(out[0]) ? out[2].data_ptr() : nullptr, a.dweight = pointer(out[1]);
                a.workspace_bytes = vrwkv_rmsnorm_bwd_workspace_bytes(&a);
                const at::Tensor ws = bytes(a.workspace_bytes, r);
                a.workspace = ws.data_ptr();
                CHECK_LIBRARY(vrwkv_rmsnorm_bwd(&a, stream_of(r)));
            }
        }
        if (recorded) only_once(out);
        return out;
    }
};

// rms_norm of norm.py: (y or q, scale or None, r or None)
py::object rms_norm(py::handle x_, py::handle w_, py::handle residual_, double eps, int kind) {
    if (transformed()) return py::none();
    const at::Tensor *xp = strided(x_), *wp = strided(w_), *rp = optional(residual_);
    if (!xp || !wp || !rp) return py::none();
    const at::Tensor &x = *xp, &w = *wp, &residual = *rp;
    if (!norm_fits(x, w, residual) || x.get_device() != c10::hip::current_device() || !on(x, x) || !on(w, x) || !on(residual, x)) return py::none();
    const bool record = at::GradMode::is_enabled() && (wanted(x) || wanted(w) || wanted(residual));
    if (record && kind) return py::none();
    at::Tensor scale;
    tensor_list out;
    {
        py::gil_scoped_release release;
        Guard guard(x.device());
        const int64_t C = x.size(-1);
        const auto options = x.options().requires_grad(false);
        Norm::Call c{at::empty(x.sizes(), kind ? options.dtype(kind == VRWKV_Y_E4M3 ? at::kFloat8_e4m3fn : at::kChar) : options), {}, eps};
        vrwkv_rmsnorm_args a = norm_args(w, C, x.numel() / C, x.scalar_type(), residual.defined() ? residual.scalar_type() : x.scalar_type(), eps);
        a.x = x.data_ptr(), a.residual = pointer(residual), a.y = c.y.data_ptr(), a.out_kind = kind;
        if (residual.defined()) a.sum = (c.r = like_of(residual)).data_ptr();
        if (kind) a.scale = (float*)(scale = at::empty(x.sizes().slice(0, x.dim() - 1), options.dtype(at::kFloat))).data_ptr();
        const bool done = vrwkv_rmsnorm(&a, stream_of(x)) == VRWKV_OK;
        if (done && record) out = Norm::apply(x, w, given(residual), &c);
        else if (done) out = {c.y, c.r};
    }
    if (out.empty()) return py::none();
    return py::make_tuple(wrapped(out[0]), wrapped(scale), out.size() > 1 ? wrapped(out[1]) : py::none());
}
}  // namespace

void add_scan_operators(py::module_& m) {
    m.def("causal_conv", &causal_conv);
    m.def("causal_conv_step", &causal_conv_step);
    m.def("selective_scan", &selective_scan);
    m.def("selective_scan_step", &selective_scan_step);
    m.def("rms_norm", &rms_norm);
}
