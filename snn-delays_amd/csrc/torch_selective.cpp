// Host side of the selective state-space block's operators (delrec.selective): argument checks, outputs
// and workspace from torch's caching allocator, calls of the C ABI (include/delrec.h), autograd nodes.
#include "torch_ops.h"

namespace {

// contiguous fp32 (n, s) on x's device
Tensor matrix_arg(const Tensor& m, int64_t n, int64_t s, const Tensor& x, const char* what) {
    if (!m.defined() || m.dim() != 2 || m.size(0) != n || m.size(1) != s || m.device() != x.device())
        refuse(text(what, " is ", m.defined() ? describe(m) : "None", ", expected [", n, ", ", s, "] on ", x.device()));
    return dense(m.to(at::kFloat));
}

// gradient of a (T, B, N) output, zeros where nothing used it
Tensor grad_rows(const Tensor& g, int64_t T, int64_t B, int64_t N, const at::TensorOptions& o) {
    return g.defined() ? rows_form(g) : at::zeros({1, 1, N}, o).expand({T, B, N});
}

delrec_rows step_rows(const Tensor& t) { return t.defined() ? delrec_rows{t.data_ptr(), 0, t.stride(0)} : delrec_rows{nullptr, 0, 0}; }

void written_in_place(const Tensor& t) {
    // a graph that kept the old state sees that it is gone, as after any operation in place
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// ---------------------------------------------------------------- the convolution -----------

variable_list conv_forward(const Tensor& x, const Tensor& w, const Tensor& bias, const Tensor& state, const Tensor& starts,
                           const Tensor& lengths, bool silu) {
    const c10::DeviceGuard guard(x.device());
    const int T = as_int(x.size(0)), B = as_int(x.size(1)), N = as_int(x.size(2)), W = as_int(w.size(1));
    Tensor y = at::empty({T, B, N}, x.options()), out = at::empty({B, W - 1, N}, x.options());
    delrec_causal_conv_fwd_args a{};
    a.T = T; a.B = B; a.N = N; a.W = W; a.bf16 = is_bf16(x); a.silu = silu;
    a.x = rows_of(x); a.w = fptr(w); a.bias = fptr(bias); a.state = state.defined() ? state.data_ptr() : nullptr;
    a.starts = starts_ptr(starts); a.lengths = lengths_ptr(lengths);
    a.y = rows_of(y); a.state_out = out.data_ptr();
    check(delrec_causal_conv_fwd(&a, stream_of(x)), "delrec_causal_conv_fwd");
    return {y, out};
}

struct CausalConvBackward : public KeptNode {
    std::string name() const override { return "CausalConvBackward"; }
    bool silu = false;

    variable_list apply(variable_list&& grads) override {
        const variable_list s = take();
        const Tensor &x = s[0], &w = s[1], &state = s[3];
        refuse_capture("causal_conv", x);
        once_differentiable("causal_conv");
        const c10::DeviceGuard guard(x.device());
        const int T = (int)x.size(0), B = (int)x.size(1), N = (int)x.size(2), W = (int)w.size(1);
        const auto f32 = w.options();
        const Tensor dy = grad_rows(grads[0], T, B, N, x.options()), dso = dense(grads[1]);
        Tensor dx = at::empty({T, B, N}, x.options()), dw = at::empty({N, W}, f32), db, ds;
        if (task_should_compute_output(2)) db = at::empty({N}, f32);
        if (task_should_compute_output(3)) ds = at::empty({B, W - 1, N}, x.options());
        const Tensor ws = workspace(DELREC_WS_CAUSAL_CONV_BWD, T, B, N, w, W);
        delrec_causal_conv_bwd_args a{};
        a.T = T; a.B = B; a.N = N; a.W = W; a.bf16 = is_bf16(x); a.silu = silu;
        a.x = rows_of(x); a.w = fptr(w); a.bias = fptr(s[2]); a.state = state.defined() ? state.data_ptr() : nullptr;
        a.starts = starts_ptr(s[4]); a.lengths = lengths_ptr(s[5]);
        a.dy = rows_of(dy); a.dstate_out = dso.defined() ? dso.data_ptr() : nullptr;
        a.dx = rows_of(dx); a.dstate = ds.defined() ? ds.data_ptr() : nullptr; a.dw = fptr(dw); a.db = fptr(db);
        a.workspace = ws.data_ptr(); a.workspace_bytes = (size_t)ws.numel();
        check(delrec_causal_conv_bwd(&a, stream_of(x)), "delrec_causal_conv_bwd");
        return {dx, dw, db, ds};
    }
};

Tensor conv_weight(const Tensor& w, int64_t N, const Tensor& x) {
    if (!w.defined() || w.dim() != 2 || w.size(1) < 2 || w.size(1) > 8)
        refuse(text("weight must be (N, W) with 2 <= W <= 8, got ", w.defined() ? describe(w) : "None"));
    return matrix_arg(w, N, w.size(1), x, "weight");
}

void check_conv_state(const Tensor& state, int64_t B, int64_t W, int64_t N, const Tensor& x) {
    if (state.dim() != 3 || state.size(0) != B || state.size(1) != W - 1 || state.size(2) != N || state.device() != x.device() ||
        state.scalar_type() != x.scalar_type())
        refuse(text("state is ", describe(state), ", expected [", B, ", ", W - 1, ", ", N, "] ", x.scalar_type(), " on ", x.device()));
}

py::tuple causal_conv(Tensor x, OptTensor w_, OptTensor bias_, OptTensor state_, OptTensor starts_, OptTensor lengths_, bool silu) {
    const Tensor w = given(w_), bias = given(bias_), state = given(state_);
    Tensor starts = given(starts_), lengths = given(lengths_);
    check_activation(x, "x");
    check_tangents("causal_conv", {&x, &w, &bias, &state});
    if (x.dim() != 3 || x.size(1) == 0 || x.size(2) == 0) refuse(text("x must be (T, B, N) with B, N > 0, got ", x.sizes()));
    const int64_t T = x.size(0), B = x.size(1), N = x.size(2);
    const Tensor wc = conv_weight(w, N, x), bc = vector_arg(bias, N, x, "bias");
    const int64_t W = wc.size(1);
    if (state.defined()) check_conv_state(state, B, W, N, x);
    check_masks(starts, lengths, T, B, x);
    if (T == 0) {
        // no step: the output is a tensor of the graph all the same, and its gradients are zeros
        Tensor y = x * wc.sum(1);
        if (bias.defined()) y = y + bc;
        if (state.defined()) y = y + state.sum(1);
        return py::make_tuple(y.to(x.scalar_type()), state.defined() ? state.clone() : at::zeros({B, W - 1, N}, x.options()));
    }
    if (!wanted({&x, &w, &bias, &state}))
        return pair_of(conv_forward(rows_form(x), wc.detach(), bc.defined() ? bc.detach() : bc, dense(state), starts, lengths, silu));
    auto node = make_node<CausalConvBackward>();
    node->set_next_edges(torch::autograd::collect_next_edges(x, w, bias, state));
    variable_list out;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        const Tensor xr = rows_form(x), wk = conv_weight(w, N, x), bk = vector_arg(bias, N, x, "bias"), sk = dense(state);
        out = conv_forward(xr, wk, bk, sk, starts, lengths, silu);
        node->silu = silu;
        node->keep({xr, wk, bk, sk, starts, lengths});
    }
    torch::autograd::set_history(out, node);
    return pair_of(out);
}

py::tuple conv_step(Tensor x, Tensor state, OptTensor w_, OptTensor bias_, bool silu, OptTensor out_) {
    Tensor w = given(w_), bias = given(bias_), out = given(out_);
    check_activation(x, "x");
    if (x.dim() != 2 || x.size(0) == 0 || x.size(1) == 0) refuse(text("conv_step takes x (B, N) with B, N > 0, got ", x.sizes()));
    check_tangents("conv_step", {&x, &state, &w, &bias});
    if (wanted({&x, &state, &w, &bias, &out}))
        throw std::runtime_error("conv_step has no backward pass: call it under torch.no_grad(), or causal_conv");
    const c10::DeviceGuard guard(x.device());
    const int B = as_int(x.size(0)), N = as_int(x.size(1));
    w = conv_weight(w, N, x);
    bias = vector_arg(bias, N, x, "bias");
    check_conv_state(state, B, w.size(1), N, x);
    const bool in_place = out.defined();
    if (in_place) {
        check_like(out, state, state.scalar_type(), "state_out");
        if (!out.is_contiguous() || out.is_neg()) refuse("state_out must be contiguous");
    } else {
        out = at::empty(state.sizes(), state.options());
    }
    x = rows_form(x);
    state = dense(state);
    if (in_place) check_state_out(out, "state_out", state, {&x, &w, &bias});
    const Tensor y = at::empty({B, N}, x.options());
    delrec_causal_conv_fwd_args a{};
    a.T = 1; a.B = B; a.N = N; a.W = (int)w.size(1); a.bf16 = is_bf16(x); a.silu = silu;
    a.x = step_rows(x); a.w = fptr(w); a.bias = fptr(bias); a.state = state.data_ptr(); a.y = step_rows(y); a.state_out = out.data_ptr();
    check(delrec_causal_conv_fwd(&a, stream_of(x)), "delrec_causal_conv_fwd");
    if (in_place) written_in_place(out);
    return py::make_tuple(y, out);
}

// ---------------------------------------------------------------- the recurrence ------------

struct ScanIn {
    Tensor x, dt, A, Bm, C, D, g, bias, h0, starts, lengths;
};

variable_list scan_forward(const ScanIn& s, Tensor* states) {
    const c10::DeviceGuard guard(s.x.device());
    const int T = as_int(s.x.size(0)), B = as_int(s.x.size(1)), N = as_int(s.x.size(2)), S = as_int(s.A.size(1));
    const auto f32 = s.A.options();
    Tensor y = at::empty({T, B, N}, s.x.options()), last = at::empty({B, N, S}, f32);
    delrec_selective_scan_fwd_args a{};
    if (states) {
        *states = at::empty({(T + DELREC_SELECTIVE_BLOCK - 1) / DELREC_SELECTIVE_BLOCK, B, N, S}, f32);
        a.states = fptr(*states);
    }
    const Tensor ws = workspace(DELREC_WS_SELECTIVE_FWD, T, B, N, s.x, S);
    a.T = T; a.B = B; a.N = N; a.S = S; a.bf16 = is_bf16(s.x);
    a.x = rows_of(s.x); a.dt = rows_of(s.dt); a.g = rows_of(s.g); a.Bm = rows_of(s.Bm); a.C = rows_of(s.C);
    a.A = fptr(s.A); a.D = fptr(s.D); a.dt_bias = fptr(s.bias); a.h0 = fptr(s.h0);
    a.starts = starts_ptr(s.starts); a.lengths = lengths_ptr(s.lengths);
    a.y = rows_of(y); a.h_last = fptr(last);
    a.workspace = ws.defined() ? ws.data_ptr() : nullptr;
    a.workspace_bytes = ws.defined() ? (size_t)ws.numel() : 0;
    check(delrec_selective_scan_fwd(&a, stream_of(s.x)), "delrec_selective_scan_fwd");
    return {y, last};
}

struct SelectiveScanBackward : public KeptNode {
    std::string name() const override { return "SelectiveScanBackward"; }

    variable_list apply(variable_list&& grads) override {
        const variable_list s = take();
        const Tensor &x = s[0], &A = s[2], &g = s[6], &states = s[8];
        refuse_capture("selective_scan", x);
        once_differentiable("selective_scan");
        const c10::DeviceGuard guard(x.device());
        const int T = (int)x.size(0), B = (int)x.size(1), N = (int)x.size(2), S = (int)A.size(1);
        const auto f32 = A.options(), act = x.options();
        const Tensor dy = grad_rows(grads[0], T, B, N, act), dlast = dense(grads[1]);
        Tensor dx = at::empty({T, B, N}, act), ddt = at::empty({T, B, N}, act), dg, dA, dD, dbias, dh0;
        Tensor dB = at::empty({T, B, S}, act), dC = at::empty({T, B, S}, act);
        if (task_should_compute_output(2)) dA = at::empty({N, S}, f32);
        if (task_should_compute_output(5)) dD = at::empty({N}, f32);
        if (g.defined()) dg = at::empty({T, B, N}, act);
        if (task_should_compute_output(7)) dbias = at::empty({N}, f32);
        if (task_should_compute_output(8)) dh0 = at::empty({B, N, S}, f32);
        const Tensor ws = workspace(DELREC_WS_SELECTIVE_BWD, T, B, N, x, S);
        delrec_selective_scan_bwd_args a{};
        a.T = T; a.B = B; a.N = N; a.S = S; a.bf16 = is_bf16(x);
        a.x = rows_of(x); a.dt = rows_of(s[1]); a.g = rows_of(g); a.Bm = rows_of(s[3]); a.C = rows_of(s[4]);
        a.A = fptr(A); a.D = fptr(s[5]); a.dt_bias = fptr(s[7]); a.states = fptr(states);
        a.starts = starts_ptr(s[9]); a.lengths = lengths_ptr(s[10]);
        a.dy = rows_of(dy); a.dlast = fptr(dlast); a.dx = rows_of(dx); a.ddt = rows_of(ddt); a.dg = rows_of(dg);
        a.dBm = dB.data_ptr(); a.dC = dC.data_ptr(); a.dA = fptr(dA); a.dD = fptr(dD); a.ddt_bias = fptr(dbias); a.dh0 = fptr(dh0);
        a.workspace = ws.data_ptr(); a.workspace_bytes = (size_t)ws.numel();
        check(delrec_selective_scan_bwd(&a, stream_of(x)), "delrec_selective_scan_bwd");
        return {dx, ddt, dA, dB, dC, dD, dg, dbias, dh0};
    }
};

py::tuple selective_scan(Tensor x, Tensor dt, Tensor A, Tensor Bm, Tensor C, OptTensor D_, OptTensor g_, OptTensor bias_, OptTensor h0_,
                         OptTensor starts_, OptTensor lengths_) {
    const Tensor D = given(D_), g = given(g_), bias = given(bias_), h0 = given(h0_);
    Tensor starts = given(starts_), lengths = given(lengths_);
    check_activation(x, "x");
    check_tangents("selective_scan", {&x, &dt, &A, &Bm, &C, &D, &g, &bias, &h0});
    if (x.dim() != 3 || x.size(1) == 0 || x.size(2) == 0) refuse(text("x must be (T, B, N) with B, N > 0, got ", x.sizes()));
    check_like(dt, x, x.scalar_type(), "dt");
    if (g.defined()) check_like(g, x, x.scalar_type(), "g");
    const int64_t T = x.size(0), B = x.size(1), N = x.size(2);
    if (A.dim() != 2 || A.size(1) < 1 || A.size(1) > 64) refuse(text("A must be (N, S) with 1 <= S <= 64, got ", describe(A)));
    const int64_t S = A.size(1);
    for (const auto& m : {std::make_pair(&Bm, "B"), std::make_pair(&C, "C")})
        if (m.first->dim() != 3 || m.first->size(0) != T || m.first->size(1) != B || m.first->size(2) != S ||
            m.first->device() != x.device() || m.first->scalar_type() != x.scalar_type())
            refuse(text(m.second, " is ", describe(*m.first), ", expected [", T, ", ", B, ", ", S, "] ", x.scalar_type(), " on ", x.device()));
    if (h0.defined() && (h0.dim() != 3 || h0.size(0) != B || h0.size(1) != N || h0.size(2) != S || h0.device() != x.device() ||
                         h0.scalar_type() != at::kFloat))
        refuse(text("h0 is ", describe(h0), ", expected [", B, ", ", N, ", ", S, "] Float on ", x.device()));
    check_masks(starts, lengths, T, B, x);
    auto rows = [&](ScanIn& s) {
        s = {rows_form(x), rows_form(dt), matrix_arg(A, N, S, x, "A"), rows_form(Bm), rows_form(C), vector_arg(D, N, x, "D"),
             rows_form(g), vector_arg(bias, N, x, "dt_bias"), dense(h0), starts, lengths};
    };
    if (T == 0) {
        // no step: the output is a tensor of the graph all the same, and its gradients are zeros
        Tensor y = x * dt * matrix_arg(A, N, S, x, "A").sum(1) + (Bm + C).sum(2, true);
        if (D.defined()) y = y + vector_arg(D, N, x, "D");
        if (g.defined()) y = y + g;
        if (bias.defined()) y = y + vector_arg(bias, N, x, "dt_bias");
        if (h0.defined()) y = y + h0.sum(2);
        const Tensor last = h0.defined() ? h0.clone() : at::zeros({B, N, S}, x.options().dtype(at::kFloat));
        return py::make_tuple(y.to(x.scalar_type()), last);
    }
    ScanIn s;
    if (!wanted({&x, &dt, &A, &Bm, &C, &D, &g, &bias, &h0})) {
        const at::NoGradGuard quiet;
        rows(s);
        return pair_of(scan_forward(s, nullptr));
    }
    auto node = make_node<SelectiveScanBackward>();
    node->set_next_edges(torch::autograd::collect_next_edges(x, dt, A, Bm, C, D, g, bias, h0));
    variable_list out;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        Tensor states;
        rows(s);
        out = scan_forward(s, &states);
        node->keep({s.x, s.dt, s.A, s.Bm, s.C, s.D, s.g, s.bias, states, starts, lengths});
    }
    torch::autograd::set_history(out, node);
    return pair_of(out);
}

py::tuple selective_step(Tensor x, Tensor dt, Tensor A, Tensor Bm, Tensor C, Tensor h, OptTensor D_, OptTensor g_, OptTensor bias_, OptTensor out_) {
    Tensor D = given(D_), g = given(g_), bias = given(bias_), out = given(out_);
    check_activation(x, "x");
    if (x.dim() != 2 || x.size(0) == 0 || x.size(1) == 0) refuse(text("selective_step takes x (B, N) with B, N > 0, got ", x.sizes()));
    check_like(dt, x, x.scalar_type(), "dt");
    if (g.defined()) check_like(g, x, x.scalar_type(), "g");
    check_tangents("selective_step", {&x, &dt, &A, &Bm, &C, &h, &D, &g, &bias});
    if (wanted({&x, &dt, &A, &Bm, &C, &h, &D, &g, &bias, &out}))
        throw std::runtime_error("selective_step has no backward pass: call it under torch.no_grad(), or selective_scan");
    const c10::DeviceGuard guard(x.device());
    const int B = as_int(x.size(0)), N = as_int(x.size(1));
    if (A.dim() != 2 || A.size(1) < 1 || A.size(1) > 64) refuse(text("A must be (N, S) with 1 <= S <= 64, got ", describe(A)));
    const int S = (int)A.size(1);
    A = matrix_arg(A, N, S, x, "A");
    for (const auto& m : {std::make_pair(&Bm, "B"), std::make_pair(&C, "C")})
        if (m.first->dim() != 2 || m.first->size(0) != B || m.first->size(1) != S || m.first->device() != x.device() ||
            m.first->scalar_type() != x.scalar_type())
            refuse(text(m.second, " is ", describe(*m.first), ", expected [", B, ", ", S, "] ", x.scalar_type(), " on ", x.device()));
    if (h.dim() != 3 || h.size(0) != B || h.size(1) != N || h.size(2) != S || h.device() != x.device() || h.scalar_type() != at::kFloat)
        refuse(text("h is ", describe(h), ", expected [", B, ", ", N, ", ", S, "] Float on ", x.device()));
    const bool in_place = out.defined();
    if (in_place) {
        check_like(out, h, at::kFloat, "h_out");
        if (!out.is_contiguous() || out.is_neg()) refuse("h_out must be contiguous");
    } else {
        out = at::empty(h.sizes(), h.options());
    }
    x = rows_form(x); dt = rows_form(dt); g = rows_form(g); Bm = rows_form(Bm); C = rows_form(C);
    h = dense(h);
    D = vector_arg(D, N, x, "D");
    bias = vector_arg(bias, N, x, "dt_bias");
    if (in_place) check_state_out(out, "h_out", h, {&x, &dt, &g, &A, &Bm, &C, &D, &bias});
    const Tensor y = at::empty({B, N}, x.options());
    delrec_selective_step_args a{};
    a.B = B; a.N = N; a.S = S; a.bf16 = is_bf16(x);
    a.x = step_rows(x); a.dt = step_rows(dt); a.g = step_rows(g); a.Bm = step_rows(Bm); a.C = step_rows(C);
    a.A = fptr(A); a.D = fptr(D); a.dt_bias = fptr(bias); a.h = fptr(h); a.h_out = fptr(out); a.y = y.data_ptr();
    check(delrec_selective_step(&a, stream_of(x)), "delrec_selective_step");
    if (in_place) written_in_place(out);
    return py::make_tuple(y, out);
}

}  // namespace

void bind_selective(py::module_& m) {
    m.def("causal_conv", &causal_conv, "short causal convolution (autograd)", py::arg("x"), py::arg("weight"), py::arg("bias"),
          py::arg("state"), py::arg("starts"), py::arg("lengths"), py::arg("silu"));
    m.def("conv_step", &conv_step, "one time step of the convolution", py::arg("x"), py::arg("state"), py::arg("weight"), py::arg("bias"),
          py::arg("silu"), py::arg("state_out"));
    m.def("selective_scan", &selective_scan, "selective recurrence (autograd)", py::arg("x"), py::arg("dt"), py::arg("A"), py::arg("B"),
          py::arg("C"), py::arg("D"), py::arg("g"), py::arg("dt_bias"), py::arg("h0"), py::arg("starts"), py::arg("lengths"));
    m.def("selective_step", &selective_step, "one time step of the recurrence", py::arg("x"), py::arg("dt"), py::arg("A"), py::arg("B"),
          py::arg("C"), py::arg("h"), py::arg("D"), py::arg("g"), py::arg("dt_bias"), py::arg("h_out"));
}
