// cc1d_host_ssm.cpp -- the native host path of the selective scan, its decode
// step and the norm: checks, allocation, the autograd node and the launch, as
// cc1d_host.cpp has them for the convolution (the same cases are taken, and
// NotImplemented is returned for every other).
#include "cc1d_host.hpp"

namespace cc1d_host {
namespace {

// entry points of the loaded library (set once by bind_ssm())
struct Api {
    decltype(&cc1d_scan_fwd) scan_fwd = nullptr;
    decltype(&cc1d_scan_tile_floats) tile_floats = nullptr;
    decltype(&cc1d_scan_bwd) scan_bwd = nullptr;
    decltype(&cc1d_scan_bwd_workspace_floats) scan_workspace = nullptr;
    decltype(&cc1d_scan_update) scan_update = nullptr;
    decltype(&cc1d_norm_fwd) norm_fwd = nullptr;
    decltype(&cc1d_norm_bwd) norm_bwd = nullptr;
    decltype(&cc1d_norm_bwd_workspace_floats) norm_workspace = nullptr;
} api;

int64_t stride0(const Tensor& t) { return t.defined() ? t.stride(0) : 0; }
const float* fptr(const Tensor& t) { return static_cast<const float*>(ptr(t)); }
const int32_t* iptr(const Tensor& t) { return static_cast<const int32_t*>(ptr(t)); }
OptTensor opt(const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }
c10::IValue ival(const Tensor& t) { return t.defined() ? c10::IValue(t) : c10::IValue(); }
bool wants(const Tensor& t) { return t.defined() && t.requires_grad(); }

// B or C, (batch, dstate, tail..) or (batch, groups, dstate, tail..), as the ABI's four strides
void state_strides(int64_t (&dst)[4], const Tensor& t, bool grouped, bool timed) {
    int i = 0;
    dst[0] = t.stride(i++);
    dst[1] = grouped ? t.stride(i++) : 0;
    dst[2] = t.stride(i++);
    dst[3] = timed ? t.stride(i) : 0;
}

// float parameters of a scan: fp32 on u's device, of that shape
bool parameter(const Tensor& t, const Tensor& u, at::IntArrayRef shape) {
    return !t.defined() || (t.scalar_type() == at::kFloat && t.device() == u.device() && shaped(t, shape));
}
bool indices(const Tensor& t, const Tensor& u) {
    return !t.defined() || (t.scalar_type() == at::kInt && t.device() == u.device() && t.is_contiguous());
}

// ---- the scan ----

struct Scan {
    Tensor u, delta, A, B, C, D, z, bias, ids, cu, init;
    bool softplus;

    cc1d_scan_params params() const {
        cc1d_scan_params p{};
        const bool grouped = B.dim() == 4;
        p.u = ptr(u);
        p.delta = ptr(delta);
        p.z = ptr(z);
        p.A = fptr(A);
        p.B = ptr(B);
        p.C = ptr(C);
        p.D = fptr(D);
        p.delta_bias = fptr(bias);
        p.seq_idx = iptr(ids);
        p.cu_seqlens = iptr(cu);
        p.batch = u.size(0);
        p.dim = u.size(1);
        p.seqlen = u.size(2);
        p.dstate = A.size(1);
        p.groups = grouped ? B.size(1) : 1;
        p.num_seqs = cu.defined() ? cu.size(0) - 1 : 0;
        strides(p.u_stride, u);
        strides(p.delta_stride, delta);
        strides(p.z_stride, z);
        strides(p.A_stride, A);
        state_strides(p.B_stride, B, grouped, true);
        state_strides(p.C_stride, C, grouped, true);
        p.D_stride = stride0(D);
        p.delta_bias_stride = stride0(bias);
        strides(p.seq_idx_stride, ids);
        p.dtype = dtype_code(u);
        p.delta_softplus = softplus;
        return p;
    }
    int64_t sequences() const { return cu.defined() ? cu.size(0) - 1 : u.size(0); }

    void forward(const Tensor& out, const Tensor& fin, const Tensor& tiles) const {
        RECORD_FUNCTION("causal_conv1d_amd::_scan_fwd_inplace", c10::ArrayRef<const c10::IValue>{});
        cc1d_scan_params p = params();
        p.initial_states = fptr(init);
        p.out = out_ptr(out);
        p.final_states = static_cast<float*>(out_ptr(fin));
        p.tile_states = static_cast<float*>(out_ptr(tiles));
        strides(p.initial_states_stride, init);
        strides(p.out_stride, out);
        strides(p.final_states_stride, fin);
        check(api.scan_fwd(&p, stream_of(u)));
    }
};

struct ScanFn : public torch::autograd::Function<ScanFn> {
    static constexpr bool is_traceable = true;

    static variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& u, const Tensor& delta, const Tensor& A,
                                 const Tensor& B, const Tensor& C, const OptTensor& D, const OptTensor& z,
                                 const OptTensor& bias, const OptTensor& ids, const OptTensor& cu, const OptTensor& init,
                                 bool softplus, bool final_states) {
        const Tensor none;
        const Scan s{u, delta, A, B, C, D.value_or(none), z.value_or(none), bias.value_or(none), ids.value_or(none),
                     cu.value_or(none), init.value_or(none), softplus};
        const Tensor out = at::empty_like(u);
        const Tensor fin = final_states ? at::empty({s.sequences(), u.size(1), A.size(1)}, A.options()) : none;
        const cc1d_scan_params p = s.params();
        const int64_t n = api.tile_floats(&p);
        const Tensor tiles = at::empty({n > 1 ? n : 1}, A.options());
        s.forward(out, fin, tiles);
        ctx->save_for_backward({u, delta, A, B, C, s.D, s.z, s.bias, s.ids, s.cu, s.init, tiles});
        ctx->saved_data["softplus"] = softplus;
        ctx->set_materialize_grads(false);
        if (final_states) return {out, fin};
        return {out};
    }

    static variable_list backward(torch::autograd::AutogradContext* ctx, const variable_list& grads) {
        const auto v = ctx->get_saved_variables();
        const Scan s{v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7], v[8], v[9], v[10], ctx->saved_data["softplus"].toBool()};
        const Tensor& tiles = v[11];
        const c10::OptionalDeviceGuard device(s.u.device());
        const Tensor dfinal = grads.size() > 1 ? grads[1] : Tensor();
        const Tensor dout = grads[0].defined() ? match_layout(grads[0], s.u) : at::zeros_like(s.u);
        auto flat = [](const Tensor& t) { return t.defined() ? at::empty(t.sizes(), t.options()) : Tensor(); };
        const Tensor du = at::empty_like(s.u), ddelta = at::empty_like(s.delta);
        const Tensor dz = s.z.defined() ? at::empty_like(s.z) : Tensor();
        const Tensor dA = flat(s.A), dB = flat(s.B), dC = flat(s.C), dD = flat(s.D), dbias = flat(s.bias), dinit = flat(s.init);
        bool direct = plain_thread() && !at::GradMode::is_enabled();
        for (const Tensor& t : v) direct = direct && (!t.defined() || plain(t));
        for (const Tensor& t : {dout, dfinal}) direct = direct && (!t.defined() || plain(t));
        if (direct) {
            RECORD_FUNCTION("causal_conv1d_amd::_scan_bwd_inplace", c10::ArrayRef<const c10::IValue>{});
            cc1d_scan_bwd_params b{};
            b.fwd = s.params();
            b.fwd.tile_states = static_cast<float*>(out_ptr(tiles));
            b.dout = ptr(dout);
            b.dfinal_states = fptr(dfinal);
            b.du = out_ptr(du);
            b.ddelta = out_ptr(ddelta);
            b.dz = out_ptr(dz);
            b.dA = static_cast<float*>(out_ptr(dA));
            b.dB = out_ptr(dB);
            b.dC = out_ptr(dC);
            b.dD = static_cast<float*>(out_ptr(dD));
            b.ddelta_bias = static_cast<float*>(out_ptr(dbias));
            b.dinitial_states = static_cast<float*>(out_ptr(dinit));
            strides(b.dout_stride, dout);
            strides(b.dfinal_states_stride, dfinal);
            strides(b.du_stride, du);
            strides(b.ddelta_stride, ddelta);
            strides(b.dz_stride, dz);
            const int64_t n = api.scan_workspace(&b);
            const Tensor ws = at::empty({n > 1 ? n : 1}, s.A.options());
            b.workspace = ws.data_ptr<float>();
            b.workspace_floats = ws.numel();
            check(api.scan_bwd(&b, stream_of(s.u)));
        } else {  // through the op: create_graph, modes, transforms, compiled autograd
            const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("causal_conv1d_amd::_scan_bwd_inplace", "");
            const bool grouped = s.B.dim() == 4;
            auto four = [grouped](const Tensor& t) { return grouped ? t : t.unsqueeze(1); };
            torch::jit::Stack stack{s.u, s.delta, s.A, four(s.B), four(s.C), ival(s.D), ival(s.z), ival(s.bias),
                                    ival(s.ids), ival(s.cu), tiles, dout, ival(dfinal), s.softplus, du, ddelta, dA,
                                    four(dB), four(dC), ival(dD), ival(dz), ival(dbias), ival(dinit)};
            op.callBoxed(&stack);
        }
        const Tensor none;
        return {du, ddelta, dA, dB, dC, dD, dz, dbias, none, none, dinit, none, none};
    }
};

PyObject* pair(Tensor a, Tensor b) {
    PyObject* t = PyTuple_New(2);
    if (t == nullptr) throw python_error();
    PyTuple_SET_ITEM(t, 0, THPVariable_Wrap(std::move(a)));
    PyTuple_SET_ITEM(t, 1, THPVariable_Wrap(std::move(b)));
    return t;
}

// ssm_scan(u, delta, A, B, C, D, z, delta_bias, delta_softplus, seq_idx, cu_seqlens, initial_states, return_final_states)
PyObject* py_scan(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK(n == 13, "ssm_scan takes 13 arguments");
    for (int i = 0; i < 5; ++i)
        if (!plain(a[i])) return not_implemented();
    for (const int i : {5, 6, 7, 9, 10, 11})
        if (!plain_or_none(a[i])) return not_implemented();
    if (!PyBool_Check(a[8]) || !PyBool_Check(a[12]) || !plain_thread()) return not_implemented();
    const Scan s{THPVariable_Unpack(a[0]), THPVariable_Unpack(a[1]), THPVariable_Unpack(a[2]), THPVariable_Unpack(a[3]),
                 THPVariable_Unpack(a[4]), tensor_or_none(a[5]), tensor_or_none(a[6]), tensor_or_none(a[7]),
                 tensor_or_none(a[9]), tensor_or_none(a[10]), tensor_or_none(a[11]), a[8] == Py_True};
    const bool fin_wanted = a[12] == Py_True;
    if (dtype_code(s.u) < 0 || s.u.dim() != 3 || s.u.numel() == 0 || s.A.dim() != 2) return not_implemented();
    const int64_t batch = s.u.size(0), dim = s.u.size(1), L = s.u.size(2), N = s.A.size(1);
    if (N < 1 || N > CC1D_MAX_DSTATE || !same(s.delta, s.u) || !shaped(s.delta, s.u.sizes()) ||
        (s.z.defined() && (!same(s.z, s.u) || !shaped(s.z, s.u.sizes()))))
        return not_implemented();
    const bool grouped = s.B.dim() == 4;
    const int64_t G = grouped ? s.B.size(1) : 1;
    if ((s.B.dim() != 3 && !grouped) || G < 1 || dim % G != 0) return not_implemented();
    for (const Tensor* t : {&s.B, &s.C})
        if (!same(*t, s.u) || !(grouped ? shaped(*t, {batch, G, N, L}) : shaped(*t, {batch, N, L}))) return not_implemented();
    if (!parameter(s.A, s.u, {dim, N}) || !parameter(s.D, s.u, {dim}) || !parameter(s.bias, s.u, {dim}) ||
        !indices(s.ids, s.u) || !indices(s.cu, s.u))
        return not_implemented();
    if (s.ids.defined() && (s.cu.defined() || s.init.defined() || fin_wanted || !shaped(s.ids, {batch, L}))) return not_implemented();
    if (s.cu.defined() && (batch != 1 || s.cu.dim() != 1 || s.cu.size(0) < 2)) return not_implemented();
    if (!parameter(s.init, s.u, {s.sequences(), dim, N})) return not_implemented();

    std::optional<pybind11::gil_scoped_release> unlocked(std::in_place);
    const c10::OptionalDeviceGuard device(s.u.device());
    bool grad = false;
    for (const Tensor* t : {&s.u, &s.delta, &s.A, &s.B, &s.C, &s.D, &s.z, &s.bias, &s.init}) grad = grad || wants(*t);
    Tensor out, fin;
    if (grad && at::GradMode::is_enabled()) {
        const auto r = ScanFn::apply(s.u, s.delta, s.A, s.B, s.C, opt(s.D), opt(s.z), opt(s.bias), opt(s.ids), opt(s.cu),
                                     opt(s.init), s.softplus, fin_wanted);
        out = r[0];
        if (fin_wanted) fin = r[1];
    } else {
        out = at::empty_like(s.u);
        if (fin_wanted) fin = at::empty({s.sequences(), dim, N}, s.A.options());
        s.forward(out, fin, Tensor());
    }
    unlocked.reset();
    return fin_wanted ? pair(std::move(out), std::move(fin)) : THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// ssm_scan_update(u, ssm_state, delta, A, B, C, D, z, delta_bias, delta_softplus, ssm_state_indices)
PyObject* py_scan_update(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK(n == 11, "ssm_scan_update takes 11 arguments");
    for (int i = 0; i < 6; ++i)
        if (!plain(a[i])) return not_implemented();
    for (const int i : {6, 7, 8, 10})
        if (!plain_or_none(a[i])) return not_implemented();
    if (!PyBool_Check(a[9]) || !plain_thread()) return not_implemented();
    const Tensor &u = THPVariable_Unpack(a[0]), &state = THPVariable_Unpack(a[1]), &delta = THPVariable_Unpack(a[2]),
                 &A = THPVariable_Unpack(a[3]), &B = THPVariable_Unpack(a[4]), &C = THPVariable_Unpack(a[5]);
    const Tensor D = tensor_or_none(a[6]), z = tensor_or_none(a[7]), bias = tensor_or_none(a[8]), idx = tensor_or_none(a[10]);
    if (dtype_code(u) < 0 || (u.dim() != 2 && u.dim() != 3) || state.dim() != 3 || A.dim() != 2 || u.numel() == 0)
        return not_implemented();
    const bool timed = u.dim() == 3, grouped = B.dim() == u.dim() + 1;
    const int64_t batch = u.size(0), dim = u.size(1), N = A.size(1), T = timed ? u.size(2) : 1;
    const int64_t G = grouped ? B.size(1) : 1;
    if (N < 1 || N > CC1D_MAX_DSTATE || (B.dim() != u.dim() && !grouped) || G < 1 || dim % G != 0) return not_implemented();
    if (!same(delta, u) || !shaped(delta, u.sizes()) || (z.defined() && (!same(z, u) || !shaped(z, u.sizes()))))
        return not_implemented();
    for (const Tensor* t : {&B, &C}) {
        if (!same(*t, u) || t->dim() != B.dim() || t->size(0) != batch) return not_implemented();
        int i = 1;
        if (grouped && t->size(i++) != G) return not_implemented();
        if (t->size(i++) != N || (timed && t->size(i) != T)) return not_implemented();
    }
    if (!parameter(A, u, {dim, N}) || !parameter(D, u, {dim}) || !parameter(bias, u, {dim}) ||
        !parameter(state, u, {idx.defined() ? state.size(0) : batch, dim, N}) || !indices(idx, u) ||
        (idx.defined() && !shaped(idx, {batch})))
        return not_implemented();

    std::optional<pybind11::gil_scoped_release> unlocked(std::in_place);
    const c10::OptionalDeviceGuard device(u.device());
    Tensor out;
    {
        const at::NoGradGuard no_grad;
        out = at::empty_like(u);
    }
    cc1d_scan_update_params p{};
    p.u = ptr(u);
    p.delta = ptr(delta);
    p.z = ptr(z);
    p.A = fptr(A);
    p.B = ptr(B);
    p.C = ptr(C);
    p.D = fptr(D);
    p.delta_bias = fptr(bias);
    p.ssm_state = static_cast<float*>(out_ptr(state));
    p.ssm_state_indices = iptr(idx);
    p.out = out_ptr(out);
    p.batch = batch;
    p.dim = dim;
    p.seqlen = T;
    p.dstate = N;
    p.groups = G;
    p.state_rows = state.size(0);
    auto tokens = [timed](int64_t (&dst)[3], const Tensor& t) {
        for (int i = 0; i < 3; ++i) dst[i] = t.defined() && (i < 2 || timed) ? t.stride(i) : 0;
    };
    tokens(p.u_stride, u);
    tokens(p.delta_stride, delta);
    tokens(p.z_stride, z);
    tokens(p.out_stride, out);
    strides(p.A_stride, A);
    state_strides(p.B_stride, B, grouped, timed);
    state_strides(p.C_stride, C, grouped, timed);
    p.D_stride = stride0(D);
    p.delta_bias_stride = stride0(bias);
    strides(p.ssm_state_stride, state);
    p.dtype = dtype_code(u);
    p.delta_softplus = a[9] == Py_True;
    check(api.scan_update(&p, stream_of(u)));
    unlocked.reset();
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// ---- the norm ----

// The stride between rows of (..., dim), contiguous inside; -1 if they have no common one.
int64_t row_stride(const Tensor& t) {
    if (t.dim() == 2 && (t.stride(1) == 1 || t.size(1) == 1)) return t.stride(0);
    return t.is_contiguous() ? t.size(-1) : -1;
}

cc1d_norm_params norm_params(const Tensor& x, const Tensor& weight, const Tensor& residual, bool rms) {
    const Tensor& like = x.defined() ? x : residual;
    cc1d_norm_params p{};
    p.x = ptr(x);
    p.residual = ptr(residual);
    p.weight = fptr(weight);
    p.dim = like.size(-1);
    p.rows = like.numel() / p.dim;
    p.x_stride = x.defined() ? row_stride(x) : 0;
    p.residual_stride = residual.defined() ? row_stride(residual) : 0;
    p.weight_stride = weight.stride(0);
    p.rms = rms;
    return p;
}

void norm_forward(const Tensor& x, const Tensor& weight, const Tensor& bias, const Tensor& residual, double eps, bool rms,
                  const Tensor& y, const Tensor& sum, const Tensor& stats) {
    RECORD_FUNCTION("causal_conv1d_amd::_norm_fwd_inplace", c10::ArrayRef<const c10::IValue>{});
    cc1d_norm_params p = norm_params(x, weight, residual, rms);
    p.bias = fptr(bias);
    p.bias_stride = stride0(bias);
    p.y = out_ptr(y);
    p.sum = out_ptr(sum);
    p.stats = static_cast<float*>(out_ptr(stats));
    p.y_stride = p.dim;
    p.sum_stride = p.dim;
    p.eps = eps;
    p.dtype = dtype_code(x);
    p.residual_dtype = residual.defined() ? dtype_code(residual) : p.dtype;
    check(api.norm_fwd(&p, stream_of(x)));
}

struct NormFn : public torch::autograd::Function<NormFn> {
    static constexpr bool is_traceable = true;

    static variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const Tensor& weight,
                                 const OptTensor& bias_, const OptTensor& residual_, double eps, bool rms, bool both) {
        const Tensor none, bias = bias_.value_or(none), residual = residual_.value_or(none);
        const Tensor y = at::empty(x.sizes(), x.options());
        const Tensor sum = both ? at::empty(x.sizes(), residual.options()) : none;
        const Tensor stats = at::empty({x.numel() / x.size(-1), 2}, weight.options());
        norm_forward(x, weight, bias, residual, eps, rms, y, sum, stats);
        // the returned sum where it is exact, else x and the residual
        const bool exact = both && sum.scalar_type() == at::kFloat;
        ctx->save_for_backward({exact ? none : x, weight, exact ? sum : residual, stats});
        ctx->saved_data["rms"] = rms;
        ctx->saved_data["bias"] = bias.defined();
        ctx->saved_data["residual"] = residual.defined();
        ctx->saved_data["x_type"] = static_cast<int64_t>(x.scalar_type());
        ctx->set_materialize_grads(false);
        if (both) return {y, sum};
        return {y};
    }

    static variable_list backward(torch::autograd::AutogradContext* ctx, const variable_list& grads) {
        const Tensor none;
        const auto v = ctx->get_saved_variables();
        const Tensor &x = v[0], &weight = v[1], &residual = v[2], &stats = v[3];
        const Tensor& like = x.defined() ? x : residual;
        const bool rms = ctx->saved_data["rms"].toBool(), has_residual = ctx->saved_data["residual"].toBool();
        const auto type = static_cast<at::ScalarType>(ctx->saved_data["x_type"].toInt());
        Tensor dy = grads[0], dsum = grads.size() > 1 ? grads[1] : none;
        if (!dy.defined() && !dsum.defined()) return {none, none, none, none, none, none, none};
        const c10::OptionalDeviceGuard device(like.device());
        if (!dy.defined()) dy = at::zeros(like.sizes(), like.options().dtype(type));
        auto rows = [](const Tensor& t) { return !t.defined() || row_stride(t) >= 0 ? t : t.contiguous(); };
        dy = rows(dy);
        dsum = rows(dsum);
        const Tensor dx = at::empty(like.sizes(), like.options().dtype(type));
        // one tensor serves both gradients where their dtypes agree
        const bool apart = has_residual && residual.scalar_type() != type;
        const Tensor dres = apart ? at::empty(like.sizes(), residual.options()) : none;
        const Tensor dw = at::empty(weight.sizes(), weight.options());
        const Tensor db = ctx->saved_data["bias"].toBool() ? at::empty(weight.sizes(), weight.options()) : none;
        bool direct = plain_thread() && !at::GradMode::is_enabled();
        for (const Tensor& t : {x, weight, residual, stats, dy, dsum}) direct = direct && (!t.defined() || plain(t));
        if (direct) {
            RECORD_FUNCTION("causal_conv1d_amd::_norm_bwd_inplace", c10::ArrayRef<const c10::IValue>{});
            cc1d_norm_bwd_params b{};
            b.fwd = norm_params(x, weight, residual, rms);
            b.fwd.stats = static_cast<float*>(out_ptr(stats));
            b.fwd.dtype = dtype_code(dx);
            b.fwd.residual_dtype = residual.defined() ? dtype_code(residual) : b.fwd.dtype;
            b.dy = ptr(dy);
            b.dsum = ptr(dsum);
            b.dx = out_ptr(dx);
            b.dresidual = out_ptr(dres);
            b.dweight = static_cast<float*>(out_ptr(dw));
            b.dbias = static_cast<float*>(out_ptr(db));
            b.dy_stride = row_stride(dy);
            b.dsum_stride = dsum.defined() ? row_stride(dsum) : 0;
            b.dx_stride = b.dresidual_stride = b.fwd.dim;
            const int64_t n = api.norm_workspace(&b);
            const Tensor ws = at::empty({n > 1 ? n : 1}, weight.options());
            b.workspace = ws.data_ptr<float>();
            b.workspace_floats = ws.numel();
            check(api.norm_bwd(&b, stream_of(dy)));
        } else {  // through the op, on (rows, dim)
            const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("causal_conv1d_amd::_norm_bwd_inplace", "");
            auto two = [&](const Tensor& t) { return t.defined() ? c10::IValue(t.reshape({-1, like.size(-1)})) : c10::IValue(); };
            torch::jit::Stack stack{two(x), weight, two(residual), stats, rms, two(dy), two(dsum), two(dx), two(dres), dw, ival(db)};
            op.callBoxed(&stack);
        }
        return {dx, dw, db, has_residual ? (apart ? dres : dx) : none, none, none, none};
    }
};

// add_norm(x, weight, bias, residual, eps, rms, return_residual)
PyObject* py_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK(n == 7, "add_norm takes 7 arguments");
    if (!plain(a[0]) || !plain(a[1]) || !plain_or_none(a[2]) || !plain_or_none(a[3]) || !PyFloat_CheckExact(a[4]) ||
        !PyBool_Check(a[5]) || !PyBool_Check(a[6]) || !plain_thread())
        return not_implemented();
    const Tensor &x = THPVariable_Unpack(a[0]), &weight = THPVariable_Unpack(a[1]);
    const Tensor bias = tensor_or_none(a[2]), residual = tensor_or_none(a[3]);
    const double eps = PyFloat_AS_DOUBLE(a[4]);
    const bool rms = a[5] == Py_True, both = a[6] == Py_True;
    if (dtype_code(x) < 0 || x.dim() < 1 || x.numel() == 0 || (both && !residual.defined())) return not_implemented();
    const int64_t dim = x.size(-1);
    if (dim > CC1D_MAX_NORM_DIM || !parameter(weight, x, {dim}) || !parameter(bias, x, {dim}) || row_stride(x) < 0)
        return not_implemented();
    if (residual.defined() &&
        (residual.device() != x.device() || !shaped(residual, x.sizes()) || row_stride(residual) < 0 ||
         (residual.scalar_type() != x.scalar_type() && residual.scalar_type() != at::kFloat)))
        return not_implemented();

    std::optional<pybind11::gil_scoped_release> unlocked(std::in_place);
    const c10::OptionalDeviceGuard device(x.device());
    Tensor y, sum;
    if (at::GradMode::is_enabled() && (wants(x) || wants(weight) || wants(bias) || wants(residual))) {
        const auto r = NormFn::apply(x, weight, opt(bias), opt(residual), eps, rms, both);
        y = r[0];
        if (both) sum = r[1];
    } else {
        y = at::empty(x.sizes(), x.options());
        if (both) sum = at::empty(x.sizes(), residual.options());
        norm_forward(x, weight, bias, residual, eps, rms, y, sum, Tensor());
    }
    unlocked.reset();
    return both ? pair(std::move(y), std::move(sum)) : THPVariable_Wrap(std::move(y));
    END_HANDLE_TH_ERRORS
}

// bind_ssm(addresses of the entry points, in Api's order)
PyObject* py_bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK(n == 8, "bind_ssm takes 8 addresses");
    void* f[8];
    for (int i = 0; i < 8; ++i) {
        f[i] = PyLong_AsVoidPtr(a[i]);
        if (PyErr_Occurred()) throw python_error();
        TORCH_CHECK(f[i] != nullptr, "a null address");
    }
    api.scan_fwd = reinterpret_cast<decltype(api.scan_fwd)>(f[0]);
    api.tile_floats = reinterpret_cast<decltype(api.tile_floats)>(f[1]);
    api.scan_bwd = reinterpret_cast<decltype(api.scan_bwd)>(f[2]);
    api.scan_workspace = reinterpret_cast<decltype(api.scan_workspace)>(f[3]);
    api.scan_update = reinterpret_cast<decltype(api.scan_update)>(f[4]);
    api.norm_fwd = reinterpret_cast<decltype(api.norm_fwd)>(f[5]);
    api.norm_bwd = reinterpret_cast<decltype(api.norm_bwd)>(f[6]);
    api.norm_workspace = reinterpret_cast<decltype(api.norm_workspace)>(f[7]);
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

}  // namespace

PyMethodDef ssm_methods[] = {
    {"bind_ssm", CC1D_FAST(py_bind), "the library's entry points for the scan and the norm"},
    {"ssm_scan", CC1D_FAST(py_scan), "ssm_scan_fn's ordinary case, or NotImplemented"},
    {"ssm_scan_update", CC1D_FAST(py_scan_update), "ssm_scan_update's ordinary case, or NotImplemented"},
    {"add_norm", CC1D_FAST(py_norm), "add_norm_fn's ordinary case, or NotImplemented"},
    {nullptr, nullptr, 0, nullptr},
};

}  // namespace cc1d_host
