// cc1d_host_attn.cpp -- the native host path of linear attention, its decode
// step and the head norm with rotation, as cc1d_host_ssm.cpp has them for the
// scan (the same cases are taken, and NotImplemented is returned for every
// other).
#include "cc1d_host.hpp"

namespace cc1d_host {
namespace {

// entry points of the loaded library (set once by bind_attn())
struct Api {
    decltype(&cc1d_attn_fwd) fwd = nullptr;
    decltype(&cc1d_attn_workspace_floats) workspace = nullptr;
    decltype(&cc1d_attn_bwd) bwd = nullptr;
    decltype(&cc1d_attn_bwd_workspace_floats) bwd_workspace = nullptr;
    decltype(&cc1d_attn_update) update = nullptr;
    decltype(&cc1d_rotary_fwd) rotary_fwd = nullptr;
    decltype(&cc1d_rotary_bwd) rotary_bwd = nullptr;
    decltype(&cc1d_rotary_bwd_workspace_floats) rotary_workspace = nullptr;
} api;

const float* fptr(const Tensor& t) { return static_cast<const float*>(ptr(t)); }
float* fout(const Tensor& t) { return static_cast<float*>(out_ptr(t)); }
const int32_t* iptr(const Tensor& t) { return static_cast<const int32_t*>(ptr(t)); }
OptTensor opt(const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }
c10::IValue ival(const Tensor& t) { return t.defined() ? c10::IValue(t) : c10::IValue(); }
bool wants(const Tensor& t) { return t.defined() && t.requires_grad(); }
Tensor flat(const Tensor& t) { return t.defined() ? at::empty(t.sizes(), t.options()) : Tensor(); }
Tensor floats(int64_t n, const Tensor& like) { return n > 0 ? at::empty({n}, like.options().dtype(at::kFloat)) : Tensor(); }
bool states(const Tensor& t, const Tensor& q, at::IntArrayRef shape) {
    return !t.defined() || (t.scalar_type() == at::kFloat && t.device() == q.device() && shaped(t, shape));
}
bool indices(const Tensor& t, const Tensor& q) {
    return !t.defined() || (t.scalar_type() == at::kInt && t.device() == q.device() && t.dim() == 1 && t.is_contiguous());
}
// None: dk ** -0.5; NaN stands for what is neither None nor a float
double scale_of(PyObject* o, int64_t dk) {
    if (o == Py_None) return 1.0 / std::sqrt(static_cast<double>(dk));
    return PyFloat_CheckExact(o) ? PyFloat_AS_DOUBLE(o) : std::nan("");
}

PyObject* pair(Tensor a, Tensor b) {
    PyObject* t = PyTuple_New(2);
    if (t == nullptr) throw python_error();
    PyTuple_SET_ITEM(t, 0, THPVariable_Wrap(std::move(a)));
    PyTuple_SET_ITEM(t, 1, THPVariable_Wrap(std::move(b)));
    return t;
}

// q, k, v (lead.., heads, size) and g (lead.., heads): whether they fit each other
bool heads_fit(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g) {
    const int64_t n = q.dim();
    if (dtype_code(q) < 0 || v.dim() != n || g.dim() != n - 1 || q.numel() == 0 || v.numel() == 0) return false;
    for (const Tensor* t : {&k, &v, &g})
        if (!same(*t, q)) return false;
    const int64_t K = q.size(n - 2), dk = q.size(n - 1), H = v.size(n - 2), dv = v.size(n - 1);
    if (dk > CC1D_MAX_ATTN_DIM || dv > CC1D_MAX_ATTN_DIM || H % K != 0 || !shaped(k, q.sizes()) || g.size(n - 2) != H) return false;
    for (int64_t i = 0; i < n - 2; ++i)
        if (v.size(i) != q.size(i) || g.size(i) != q.size(i)) return false;
    return true;
}

// ---- linear attention ----

// states whose values lie within 2**31 of each other, as the kernels count them
Tensor near(const Tensor& t) {
    if (!t.defined() || (t.size(2) - 1) * t.stride(2) + (t.size(3) - 1) * t.stride(3) < ((int64_t)1 << 31)) return t;
    return t.contiguous();
}

struct Attn {
    Tensor q, k, v, g, cu, init;
    double scale;

    cc1d_attn_params params() const {
        cc1d_attn_params p{};
        p.q = ptr(q);
        p.k = ptr(k);
        p.v = ptr(v);
        p.g = ptr(g);
        p.cu_seqlens = iptr(cu);
        p.initial_states = fptr(init);
        p.batch = q.size(0);
        p.seqlen = q.size(1);
        p.heads = v.size(2);
        p.key_heads = q.size(2);
        p.dk = q.size(3);
        p.dv = v.size(3);
        p.num_seqs = cu.defined() ? cu.size(0) - 1 : 0;
        strides(p.q_stride, q);
        strides(p.k_stride, k);
        strides(p.v_stride, v);
        strides(p.g_stride, g);
        strides(p.initial_states_stride, init);
        p.scale = scale;
        p.dtype = dtype_code(q);
        return p;
    }
    std::array<int64_t, 4> state_shape() const {
        return {cu.defined() ? cu.size(0) - 1 : q.size(0), v.size(2), q.size(3), v.size(3)};
    }

    void forward(const Tensor& out, const Tensor& fin) const {
        RECORD_FUNCTION("causal_conv1d_amd::_attn_fwd_inplace", c10::ArrayRef<const c10::IValue>{});
        cc1d_attn_params p = params();
        p.out = out_ptr(out);
        p.final_states = fout(fin);
        const Tensor ws = floats(api.workspace(&p), q);
        p.workspace = fout(ws);
        p.workspace_floats = ws.defined() ? ws.numel() : 0;
        check(api.fwd(&p, stream_of(q)));
    }
};

struct AttnFn : public torch::autograd::Function<AttnFn> {
    static constexpr bool is_traceable = true;

    static variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v,
                                 const Tensor& g, const OptTensor& cu, const OptTensor& init, double scale, bool final_states) {
        const Tensor none;
        const Attn a{q, k, v, g, cu.value_or(none), init.value_or(none), scale};
        const Tensor out = flat(v);
        const Tensor fin = final_states ? at::empty(a.state_shape(), v.options().dtype(at::kFloat)) : none;
        a.forward(out, fin);
        ctx->save_for_backward({q, k, v, g, a.cu, a.init});
        ctx->saved_data["scale"] = scale;
        ctx->set_materialize_grads(false);
        if (final_states) return {out, fin};
        return {out};
    }

    static variable_list backward(torch::autograd::AutogradContext* ctx, const variable_list& grads) {
        const Tensor none;
        const auto s = ctx->get_saved_variables();
        const Attn a{s[0], s[1], s[2], s[3], s[4], s[5], ctx->saved_data["scale"].toDouble()};
        const Tensor dfinal = grads.size() > 1 ? near(grads[1]) : none;
        if (!grads[0].defined() && !dfinal.defined()) return {none, none, none, none, none, none, none, none};
        const c10::OptionalDeviceGuard device(a.q.device());
        const Tensor dout = grads[0].defined() ? grads[0] : at::zeros(a.v.sizes(), a.v.options());
        const Tensor dq = flat(a.q), dk = flat(a.k), dv = flat(a.v), dg = flat(a.g), dinit = flat(a.init);
        bool direct = plain_thread() && !at::GradMode::is_enabled();
        for (const Tensor& t : s) direct = direct && (!t.defined() || plain(t));
        for (const Tensor& t : {dout, dfinal}) direct = direct && (!t.defined() || plain(t));
        if (direct) {
            RECORD_FUNCTION("causal_conv1d_amd::_attn_bwd_inplace", c10::ArrayRef<const c10::IValue>{});
            cc1d_attn_bwd_params b{};
            b.fwd = a.params();
            b.dout = ptr(dout);
            b.dfinal_states = fptr(dfinal);
            b.dq = out_ptr(dq);
            b.dk = out_ptr(dk);
            b.dv = out_ptr(dv);
            b.dg = out_ptr(dg);
            b.dinitial_states = fout(dinit);
            strides(b.dout_stride, dout);
            strides(b.dfinal_states_stride, dfinal);
            const Tensor ws = floats(api.bwd_workspace(&b), a.q);
            b.workspace = fout(ws);
            b.workspace_floats = ws.defined() ? ws.numel() : 0;
            check(api.bwd(&b, stream_of(a.q)));
        } else {  // through the op: create_graph, modes, transforms, compiled autograd
            const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("causal_conv1d_amd::_attn_bwd_inplace", "");
            torch::jit::Stack stack{a.q, a.k, a.v, a.g, ival(a.cu), ival(a.init), a.scale, dout, ival(dfinal),
                                    dq, dk, dv, dg, ival(dinit)};
            op.callBoxed(&stack);
        }
        return {dq, dk, dv, dg, none, dinit, none, none};
    }
};

// linear_attn(q, k, v, g, scale, cu_seqlens, initial_states, return_final_states)
PyObject* py_attn(PyObject*, PyObject* const* o, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK(n == 8, "linear_attn takes 8 arguments");
    for (int i = 0; i < 4; ++i)
        if (!plain(o[i])) return not_implemented();
    if (!plain_or_none(o[5]) || !plain_or_none(o[6]) || !PyBool_Check(o[7]) || !plain_thread()) return not_implemented();
    Attn a{THPVariable_Unpack(o[0]), THPVariable_Unpack(o[1]), THPVariable_Unpack(o[2]), THPVariable_Unpack(o[3]),
           tensor_or_none(o[5]), tensor_or_none(o[6]), 0.0};
    const bool fin_wanted = o[7] == Py_True;
    if (a.q.dim() != 4 || !heads_fit(a.q, a.k, a.v, a.g) || !indices(a.cu, a.q)) return not_implemented();
    if (a.cu.defined() && (a.q.size(0) != 1 || a.cu.size(0) < 2)) return not_implemented();
    if (!states(a.init, a.q, a.state_shape()) || !near(a.init).is_same(a.init)) return not_implemented();
    a.scale = scale_of(o[4], a.q.size(3));
    if (std::isnan(a.scale)) return not_implemented();

    std::optional<pybind11::gil_scoped_release> unlocked(std::in_place);
    const c10::OptionalDeviceGuard device(a.q.device());
    Tensor out, fin;
    if (at::GradMode::is_enabled() && (wants(a.q) || wants(a.k) || wants(a.v) || wants(a.g) || wants(a.init))) {
        const auto r = AttnFn::apply(a.q, a.k, a.v, a.g, opt(a.cu), opt(a.init), a.scale, fin_wanted);
        out = r[0];
        if (fin_wanted) fin = r[1];
    } else {
        out = flat(a.v);
        if (fin_wanted) fin = at::empty(a.state_shape(), a.v.options().dtype(at::kFloat));
        a.forward(out, fin);
    }
    unlocked.reset();
    return fin_wanted ? pair(std::move(out), std::move(fin)) : THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// linear_attn_update(q, attn_state, k, v, g, scale, attn_state_indices)
PyObject* py_update(PyObject*, PyObject* const* o, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK(n == 7, "linear_attn_update takes 7 arguments");
    for (int i = 0; i < 5; ++i)
        if (!plain(o[i])) return not_implemented();
    if (!plain_or_none(o[6]) || !plain_thread()) return not_implemented();
    const Tensor &q = THPVariable_Unpack(o[0]), &state = THPVariable_Unpack(o[1]), &k = THPVariable_Unpack(o[2]),
                 &v = THPVariable_Unpack(o[3]), &g = THPVariable_Unpack(o[4]);
    const Tensor idx = tensor_or_none(o[6]);
    if ((q.dim() != 3 && q.dim() != 4) || state.dim() != 4 || !heads_fit(q, k, v, g) || !indices(idx, q)) return not_implemented();
    const bool timed = q.dim() == 4;
    const int64_t batch = q.size(0), H = v.size(-2), dk = q.size(-1), dv = v.size(-1);
    if (!states(state, q, {idx.defined() ? state.size(0) : batch, H, dk, dv}) || (idx.defined() && !shaped(idx, {batch})))
        return not_implemented();
    const double scale = scale_of(o[5], dk);
    if (std::isnan(scale)) return not_implemented();

    std::optional<pybind11::gil_scoped_release> unlocked(std::in_place);
    const c10::OptionalDeviceGuard device(q.device());
    Tensor out;
    {
        const at::NoGradGuard no_grad;
        out = flat(v);
    }
    cc1d_attn_update_params p{};
    p.q = ptr(q);
    p.k = ptr(k);
    p.v = ptr(v);
    p.g = ptr(g);
    p.attn_state = fout(state);
    p.attn_state_indices = iptr(idx);
    p.out = out_ptr(out);
    p.batch = batch;
    p.tokens = timed ? q.size(1) : 1;
    p.heads = H;
    p.key_heads = q.size(-2);
    p.dk = dk;
    p.dv = dv;
    p.state_rows = state.size(0);
    auto tokens = [timed](int64_t* dst, const Tensor& t) {  // (batch, [token,] ..)
        int64_t i = 0;
        for (int64_t d = 0; d < t.dim(); ++d) {
            dst[i++] = t.stride(d);
            if (d == 0 && !timed) dst[i++] = 0;
        }
    };
    tokens(p.q_stride, q);
    tokens(p.k_stride, k);
    tokens(p.v_stride, v);
    tokens(p.g_stride, g);
    strides(p.attn_state_stride, state);
    p.scale = scale;
    p.dtype = dtype_code(q);
    check(api.update(&p, stream_of(q)));
    written(state);
    unlocked.reset();
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// ---- head norm with rotation ----

struct Rotary {
    Tensor wq, wk, freq, pos;
    double eps, amplitude;
    bool interleaved;

    // (batch, seqlen, ..) strides of t, which may be (tokens, ..)
    template <int N> static void lead(int64_t (&dst)[N], const Tensor& t, bool timed) {
        int64_t i = 0;
        for (int64_t d = 0; d < t.dim(); ++d) {
            dst[i++] = t.stride(d);
            if (d == 0 && !timed) dst[i++] = 0;
        }
    }
    // of q and k alike
    cc1d_rotary_params params(const Tensor& q, const Tensor& k) const {
        cc1d_rotary_params p{};
        const bool timed = q.dim() == 4;
        p.q = ptr(q);
        p.k = ptr(k);
        p.q_weight = fptr(wq);
        p.k_weight = fptr(wk);
        p.inv_freq = fptr(freq);
        p.positions = ptr(pos);
        p.batch = q.size(0);
        p.seqlen = timed ? q.size(1) : 1;
        p.q_heads = q.size(-2);
        p.k_heads = k.size(-2);
        p.dim = q.size(-1);
        p.rotated = freq.defined() ? 2 * freq.size(0) : 0;
        lead(p.q_stride, q, timed);
        lead(p.k_stride, k, timed);
        if (pos.defined()) lead(p.positions_stride, pos, timed);
        p.positions_bytes = pos.defined() && pos.scalar_type() == at::kLong ? 8 : 4;
        p.eps = eps;
        p.amplitude = amplitude;
        p.dtype = dtype_code(q);
        p.interleaved = interleaved;
        return p;
    }
    void forward(const Tensor& q, const Tensor& k, const Tensor& qo, const Tensor& ko) const {
        RECORD_FUNCTION("causal_conv1d_amd::_rotary_fwd_inplace", c10::ArrayRef<const c10::IValue>{});
        cc1d_rotary_params p = params(q, k);
        p.q_out = out_ptr(qo);
        p.k_out = out_ptr(ko);
        check(api.rotary_fwd(&p, stream_of(q)));
    }
};

struct RotaryFn : public torch::autograd::Function<RotaryFn> {
    static constexpr bool is_traceable = true;

    static variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& q, const Tensor& k, const OptTensor& wq,
                                 const OptTensor& wk, const OptTensor& freq, const OptTensor& pos, double eps, bool interleaved,
                                 double amplitude) {
        const Tensor none;
        const Rotary r{wq.value_or(none), wk.value_or(none), freq.value_or(none), pos.value_or(none), eps, amplitude, interleaved};
        const Tensor qo = flat(q), ko = flat(k);
        r.forward(q, k, qo, ko);
        // a rotation alone needs no more than its angles
        ctx->save_for_backward({r.wq.defined() ? q : none, r.wk.defined() ? k : none, r.wq, r.wk, r.freq, r.pos});
        ctx->saved_data["eps"] = eps;
        ctx->saved_data["interleaved"] = interleaved;
        ctx->saved_data["amplitude"] = amplitude;
        return {qo, ko};
    }

    static variable_list backward(torch::autograd::AutogradContext* ctx, const variable_list& grads) {
        const Tensor none;
        const auto s = ctx->get_saved_variables();
        const Tensor &dqo = grads[0], &dko = grads[1];
        const Rotary r{s[2], s[3], s[4], s[5], ctx->saved_data["eps"].toDouble(), ctx->saved_data["amplitude"].toDouble(),
                       ctx->saved_data["interleaved"].toBool()};
        const c10::OptionalDeviceGuard device(dqo.device());
        const Tensor dq = flat(dqo), dk = flat(dko), dwq = flat(r.wq), dwk = flat(r.wk);
        bool direct = plain_thread() && !at::GradMode::is_enabled();
        for (const Tensor& t : s) direct = direct && (!t.defined() || plain(t));
        for (const Tensor& t : {dqo, dko}) direct = direct && plain(t);
        if (direct) {
            RECORD_FUNCTION("causal_conv1d_amd::_rotary_bwd_inplace", c10::ArrayRef<const c10::IValue>{});
            cc1d_rotary_bwd_params b{};
            b.fwd = r.params(s[0].defined() ? s[0] : dqo, s[1].defined() ? s[1] : dko);
            const bool timed = dqo.dim() == 4;
            b.dq_out = ptr(dqo);
            b.dk_out = ptr(dko);
            b.dq = out_ptr(dq);
            b.dk = out_ptr(dk);
            b.dq_weight = fout(dwq);
            b.dk_weight = fout(dwk);
            Rotary::lead(b.dq_out_stride, dqo, timed);
            Rotary::lead(b.dk_out_stride, dko, timed);
            const Tensor ws = floats(api.rotary_workspace(&b), dqo);
            b.workspace = fout(ws);
            b.workspace_floats = ws.defined() ? ws.numel() : 0;
            check(api.rotary_bwd(&b, stream_of(dqo)));
        } else {  // through the op, on (batch, seqlen, heads, dim)
            const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("causal_conv1d_amd::_rotary_bwd_inplace", "");
            const bool timed = dqo.dim() == 4;
            auto four = [timed](const Tensor& t) { return !t.defined() ? c10::IValue() : c10::IValue(timed ? t : t.unsqueeze(1)); };
            torch::jit::Stack stack{four(s[0]), four(s[1]), ival(r.wq), ival(r.wk), ival(r.freq), four(r.pos), r.eps,
                                    r.interleaved, r.amplitude, four(dqo), four(dko), four(dq), four(dk), ival(dwq), ival(dwk)};
            op.callBoxed(&stack);
        }
        return {dq, dk, dwq, dwk, none, none, none, none, none};
    }
};

// head_norm_rotary(q, k, q_weight, k_weight, inv_freq, positions, eps, interleaved, amplitude)
PyObject* py_rotary(PyObject*, PyObject* const* o, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK(n == 9, "head_norm_rotary takes 9 arguments");
    if (!plain(o[0]) || !plain(o[1])) return not_implemented();
    for (int i = 2; i < 6; ++i)
        if (!plain_or_none(o[i])) return not_implemented();
    if (!PyFloat_CheckExact(o[6]) || !PyBool_Check(o[7]) || !PyFloat_CheckExact(o[8]) || !plain_thread()) return not_implemented();
    const Tensor &q = THPVariable_Unpack(o[0]), &k = THPVariable_Unpack(o[1]);
    Rotary r{tensor_or_none(o[2]), tensor_or_none(o[3]), tensor_or_none(o[4]), tensor_or_none(o[5]),
             PyFloat_AS_DOUBLE(o[6]), PyFloat_AS_DOUBLE(o[8]), o[7] == Py_True};
    if (dtype_code(q) < 0 || (q.dim() != 3 && q.dim() != 4) || k.dim() != q.dim() || !same(k, q) || q.numel() == 0 || k.numel() == 0)
        return not_implemented();
    const int64_t lead = q.dim() - 2, dim = q.size(-1);
    if (dim > CC1D_MAX_ROTARY_DIM || k.size(-1) != dim) return not_implemented();
    for (int64_t i = 0; i < lead; ++i)
        if (k.size(i) != q.size(i)) return not_implemented();
    for (const Tensor* w : {&r.wq, &r.wk})
        if (w->defined() && (!states(*w, q, {dim}) || !w->is_contiguous())) return not_implemented();
    if (r.freq.defined() && (r.freq.dim() != 1 || 2 * r.freq.size(0) > dim || r.freq.scalar_type() != at::kFloat ||
                             r.freq.device() != q.device() || !r.freq.is_contiguous() || r.freq.requires_grad() ||
                             (lead == 1 && !r.pos.defined())))
        return not_implemented();
    if (r.pos.defined()) {
        if ((r.pos.scalar_type() != at::kInt && r.pos.scalar_type() != at::kLong) || r.pos.device() != q.device() || r.pos.dim() != lead)
            return not_implemented();
        for (int64_t i = 0; i < lead; ++i)
            if (r.pos.size(i) != q.size(i)) return not_implemented();
    }

    std::optional<pybind11::gil_scoped_release> unlocked(std::in_place);
    const c10::OptionalDeviceGuard device(q.device());
    Tensor qo, ko;
    if (at::GradMode::is_enabled() && (wants(q) || wants(k) || wants(r.wq) || wants(r.wk))) {
        const auto v = RotaryFn::apply(q, k, opt(r.wq), opt(r.wk), opt(r.freq), opt(r.pos), r.eps, r.interleaved, r.amplitude);
        qo = v[0];
        ko = v[1];
    } else {
        qo = flat(q);
        ko = flat(k);
        r.forward(q, k, qo, ko);
    }
    unlocked.reset();
    return pair(std::move(qo), std::move(ko));
    END_HANDLE_TH_ERRORS
}

// bind_attn(addresses of the entry points, in Api's order)
PyObject* py_bind(PyObject*, PyObject* const* o, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK(n == 8, "bind_attn takes 8 addresses");
    void* f[8];
    for (int i = 0; i < 8; ++i) {
        f[i] = PyLong_AsVoidPtr(o[i]);
        if (PyErr_Occurred()) throw python_error();
        TORCH_CHECK(f[i] != nullptr, "a null address");
    }
    api.fwd = reinterpret_cast<decltype(api.fwd)>(f[0]);
    api.workspace = reinterpret_cast<decltype(api.workspace)>(f[1]);
    api.bwd = reinterpret_cast<decltype(api.bwd)>(f[2]);
    api.bwd_workspace = reinterpret_cast<decltype(api.bwd_workspace)>(f[3]);
    api.update = reinterpret_cast<decltype(api.update)>(f[4]);
    api.rotary_fwd = reinterpret_cast<decltype(api.rotary_fwd)>(f[5]);
    api.rotary_bwd = reinterpret_cast<decltype(api.rotary_bwd)>(f[6]);
    api.rotary_workspace = reinterpret_cast<decltype(api.rotary_workspace)>(f[7]);
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

}  // namespace

PyMethodDef attn_methods[] = {
    {"bind_attn", CC1D_FAST(py_bind), "the library's entry points for linear attention and the rotation"},
    {"linear_attn", CC1D_FAST(py_attn), "linear_attn_fn's ordinary case, or NotImplemented"},
    {"linear_attn_update", CC1D_FAST(py_update), "linear_attn_update's ordinary case, or NotImplemented"},
    {"head_norm_rotary", CC1D_FAST(py_rotary), "head_norm_rotary_fn's ordinary case, or NotImplemented"},
    {nullptr, nullptr, 0, nullptr},
};

}  // namespace cc1d_host
