// Host side of the gated-recurrence block's operators (delrec.gated, delrec.checkpoint8): argument
// checks, outputs and workspace from torch's caching allocator, calls of the C ABI
// (include/delrec.h), autograd Functions.
//
// In C++ because the smallest calls are bound by the host: a training pass of the scan at T32 B64
// N64, whose kernels take 15 us, took 235 us through Python Functions and the ctypes binding. The
// graph's nodes are torch::autograd::Node themselves: torch::autograd::Function keeps its values in
// a dictionary of boxed ones.
#include "torch_ops.h"

namespace {

// ---------------------------------------------------------------- the recurrence ------------

struct ScanKept {
    Tensor z, f;
    Packed z8, f8;
    Tensor states;
};

variable_list scan_forward(const Tensor& z, const Tensor& f, const Tensor& bias, const Tensor& h0, const Tensor& starts,
                           const Tensor& lengths, bool checkpoint, ScanKept* kept) {
    const c10::DeviceGuard guard(z.device());
    const int T = as_int(z.size(0)), B = as_int(z.size(1)), N = as_int(z.size(2));
    const auto f32 = z.options().dtype(at::kFloat);
    Tensor h = at::empty({T, B, N}, z.options()), last = at::empty({B, N}, f32);
    delrec_gated_scan_fwd_args a{};
    if (kept) {
        kept->states = at::empty({(T + DELREC_GATED_BLOCK - 1) / DELREC_GATED_BLOCK, B, N}, f32);
        a.states = fptr(kept->states);
        if (checkpoint) {
            kept->z8 = Packed((int64_t)T * B, N, z);
            kept->f8 = Packed((int64_t)T * B, N, z);
            a.z8 = kept->z8.arg();
            a.f8 = kept->f8.arg();
        } else {
            kept->z = z;
            kept->f = f;
        }
    }
    const Tensor ws = workspace(DELREC_WS_GATED_FWD, T, B, N, z);
    a.T = T; a.B = B; a.N = N; a.bf16 = is_bf16(z);
    a.z = rows_of(z); a.f = rows_of(f); a.bias = fptr(bias); a.h0 = fptr(h0);
    a.starts = starts.defined() ? (const uint8_t*)starts.data_ptr() : nullptr;
    a.lengths = lengths.defined() ? (const int64_t*)lengths.data_ptr() : nullptr;
    a.h = rows_of(h); a.h_last = fptr(last);
    a.workspace = ws.defined() ? ws.data_ptr() : nullptr;
    a.workspace_bytes = ws.defined() ? (size_t)ws.numel() : 0;
    check(delrec_gated_scan_fwd(&a, stream_of(z)), "delrec_gated_scan_fwd");
    return {h, last};
}

struct GatedScanBackward : public KeptNode {
    std::string name() const override { return "GatedScanBackward"; }
    int64_t T = 0;
    at::ScalarType type = at::kFloat;

    variable_list apply(variable_list&& grads) override {
        const variable_list s = take();
        const Tensor& states = s[7];
        refuse_capture("gated_scan", states);
        once_differentiable("gated_scan");
        const c10::DeviceGuard guard(states.device());
        const int B = (int)states.size(1), N = (int)states.size(2);
        const auto f32 = states.options();
        // an output that nothing used
        const Tensor dh = grads[0].defined() ? rows_form(grads[0]) : at::zeros({1, 1, N}, f32.dtype(type)).expand({T, B, N});
        const Tensor dlast = dense(grads[1]);
        Tensor dz = at::empty({T, B, N}, f32.dtype(type)), df = at::empty({T, B, N}, f32.dtype(type)), db, dh0;
        if (task_should_compute_output(2)) db = at::empty({N}, f32);
        if (task_should_compute_output(3)) dh0 = at::empty({B, N}, f32);
        const Tensor ws = workspace(DELREC_WS_GATED_BWD, (int)T, B, N, states);
        delrec_gated_scan_bwd_args a{};
        a.T = (int)T; a.B = B; a.N = N; a.bf16 = type == at::kBFloat16;
        a.z = rows_of(s[0]); a.f = rows_of(s[1]);
        a.z8 = Packed(s[2], s[3]).arg(); a.f8 = Packed(s[4], s[5]).arg();
        a.bias = fptr(s[6]); a.states = fptr(states);
        a.starts = s[8].defined() ? (const uint8_t*)s[8].data_ptr() : nullptr;
        a.lengths = s[9].defined() ? (const int64_t*)s[9].data_ptr() : nullptr;
        a.dh = rows_of(dh); a.dlast = fptr(dlast); a.dz = rows_of(dz); a.df = rows_of(df);
        a.db = fptr(db); a.dh0 = fptr(dh0);
        a.workspace = ws.data_ptr(); a.workspace_bytes = (size_t)ws.numel();
        check(delrec_gated_scan_bwd(&a, stream_of(states)), "delrec_gated_scan_bwd");
        return {dz, df, db, dh0};     // (the engine casts db to the bias' type)
    }
};

variable_list scan_with_graph(const Tensor& z, const Tensor& f, const Tensor& bias, const Tensor& h0, const Tensor& starts,
                              const Tensor& lengths, bool checkpoint) {
    auto node = make_node<GatedScanBackward>();
    node->set_next_edges(torch::autograd::collect_next_edges(z, f, bias, h0));
    variable_list out;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        ScanKept kept;
        const Tensor b = vector_arg(bias, z.size(2), z, "bias"), h0c = dense(h0);
        out = scan_forward(rows_form(z), rows_form(f), b, h0c, starts, lengths, checkpoint, &kept);
        node->T = z.size(0);
        node->type = z.scalar_type();
        node->keep({kept.z, kept.f, kept.z8.q, kept.z8.scale, kept.f8.q, kept.f8.scale, b, kept.states, starts, lengths});
    }
    torch::autograd::set_history(out, node);
    return out;
}

py::tuple gated_scan(Tensor z, Tensor f, OptTensor bias_, OptTensor h0_, OptTensor starts_, OptTensor lengths_, bool checkpoint) {
    const Tensor bias = given(bias_), h0 = given(h0_);
    Tensor starts = given(starts_), lengths = given(lengths_);
    check_activation(z, "z");
    check_tangents("gated_scan", {&z, &f, &bias, &h0});
    if (z.dim() != 3 || z.size(1) == 0 || z.size(2) == 0) refuse(text("z must be (T, B, N) with B, N > 0, got ", z.sizes()));
    check_like(f, z, z.scalar_type(), "f");
    const int64_t T = z.size(0), B = z.size(1), N = z.size(2);
    if (h0.defined() && (h0.dim() != 2 || h0.size(0) != B || h0.size(1) != N || h0.device() != z.device() || h0.scalar_type() != at::kFloat))
        refuse(text("h0 is ", describe(h0), ", expected [", B, ", ", N, "] Float on ", z.device()));
    check_masks(starts, lengths, T, B, z);
    if (T == 0) {
        // no step: the output is a tensor of the graph all the same, and its gradients are zeros
        Tensor h = z * f;
        if (bias.defined()) h = h + vector_arg(bias, N, z, "bias");
        if (h0.defined()) h = h + h0;
        const Tensor last = h0.defined() ? h0.clone() : at::zeros({B, N}, z.options().dtype(at::kFloat));
        return py::make_tuple(h.to(z.scalar_type()), last);
    }
    if (wanted({&z, &f, &bias, &h0})) return pair_of(scan_with_graph(z, f, bias, h0, starts, lengths, checkpoint));
    return pair_of(scan_forward(rows_form(z), rows_form(f), vector_arg(bias, N, z, "bias"), dense(h0),
                                starts, lengths, false, nullptr));
}

// ---------------------------------------------------------------- norms, gate, residual -----

struct NormKept {
    Tensor o, g, x;
    Packed o8, g8, x8;
    Tensor stats;
};

// x' (undefined without a block) and u (undefined without w2)
variable_list norm_forward(const Tensor& o, const Tensor& g, const Tensor& x, const Tensor& w, const Tensor& scale,
                           const Tensor& w2, double eps, at::IntArrayRef shape, bool checkpoint, NormKept* kept) {
    const c10::DeviceGuard guard(x.device());
    const int R0 = as_int(x.size(0)), R1 = x.dim() == 3 ? as_int(x.size(1)) : 1, N = as_int(x.size(-1));
    const int64_t rows = (int64_t)R0 * R1;
    const auto act = o.defined() ? o.options() : x.options();
    Tensor xo, u;
    if (o.defined()) xo = at::empty(shape, x.options());
    if (w2.defined()) u = at::empty(shape, act);
    delrec_norm_gate_fwd_args a{};
    if (kept) {
        kept->stats = at::empty({rows, 2}, x.options().dtype(at::kFloat));
        a.stats = fptr(kept->stats);
        if (checkpoint) {
            kept->x8 = Packed(rows, N, x);
            a.x8 = kept->x8.arg();
            if (o.defined()) {
                kept->o8 = Packed(rows, N, x);
                kept->g8 = Packed(rows, N, x);
                a.o8 = kept->o8.arg();
                a.g8 = kept->g8.arg();
            }
        } else {
            kept->o = o;
            kept->g = g;
            kept->x = x;
        }
    }
    a.R0 = R0; a.R1 = R1; a.N = N; a.bf16 = act.dtype() == at::kBFloat16; a.x_bf16 = is_bf16(x);
    a.o = rows_of(o); a.g = rows_of(g); a.x = rows_of(x); a.w = fptr(w); a.scale = fptr(scale); a.w2 = fptr(w2);
    a.eps = (float)eps;
    a.x_out = xo.defined() ? xo.data_ptr() : nullptr;
    a.u = u.defined() ? u.data_ptr() : nullptr;
    check(delrec_norm_gate_fwd(&a, stream_of(x)), "delrec_norm_gate_fwd");
    return {xo, u};
}

struct NormGateBackward : public KeptNode {
    std::string name() const override { return "NormGateBackward"; }
    std::vector<int64_t> shape;
    at::ScalarType act = at::kFloat, res = at::kFloat;
    int R0 = 0, R1 = 0;
    bool block = false;

    variable_list apply(variable_list&& grads) override {
        const variable_list s = take();
        const Tensor &w = s[9], &scale = s[10], &w2 = s[11], &stats = s[12];
        refuse_capture("norm_gate_residual", stats);
        once_differentiable("norm_gate_residual");
        const Tensor dxo = block ? rows_form(grads[0]) : Tensor();
        const Tensor du = !block ? rows_form(grads[0]) : w2.defined() ? rows_form(grads[1]) : Tensor();
        if (!dxo.defined() && !du.defined()) return variable_list(6);
        const c10::DeviceGuard guard(stats.device());
        const int N = (int)shape.back();
        const auto f32 = stats.options();
        Tensor d_o, dg, dw, ds, dw2, dx = at::empty(shape, f32.dtype(res));
        if (block) {
            d_o = at::empty(shape, f32.dtype(act));
            dg = at::empty(shape, f32.dtype(act));
            dw = at::empty({N}, f32);
            ds = at::empty({N}, f32);
        }
        if (w2.defined()) dw2 = at::empty({N}, f32);
        const Tensor ws = workspace(DELREC_WS_NORM_GATE_BWD, R0, R1, N, stats);
        delrec_norm_gate_bwd_args a{};
        a.R0 = R0; a.R1 = R1; a.N = N; a.bf16 = act == at::kBFloat16; a.x_bf16 = res == at::kBFloat16;
        a.o = rows_of(s[0]); a.g = rows_of(s[1]); a.x = rows_of(s[2]);
        a.o8 = Packed(s[3], s[4]).arg(); a.g8 = Packed(s[5], s[6]).arg(); a.x8 = Packed(s[7], s[8]).arg();
        a.w = fptr(w); a.scale = fptr(scale); a.w2 = fptr(w2); a.stats = fptr(stats);
        a.dx_out = rows_of(dxo); a.du = rows_of(du);
        a.d_o = dense_rows(d_o, R1, N); a.dg = dense_rows(dg, R1, N); a.dx = dense_rows(dx, R1, N);
        a.dw = fptr(dw); a.dscale = fptr(ds); a.dw2 = fptr(dw2);
        a.workspace = ws.data_ptr(); a.workspace_bytes = (size_t)ws.numel();
        check(delrec_norm_gate_bwd(&a, stream_of(stats)), "delrec_norm_gate_bwd");
        return {d_o, dg, dx, dw, ds, dw2};
    }
};

variable_list norm_with_graph(const Tensor& o, const Tensor& g, const Tensor& x, const Tensor& w, const Tensor& scale,
                              const Tensor& w2, double eps, bool checkpoint) {
    auto node = make_node<NormGateBackward>();
    node->set_next_edges(torch::autograd::collect_next_edges(o, g, x, w, scale, w2));
    variable_list out;
    const Tensor orow = kept_rows(o), grow = kept_rows(g), xr = kept_rows(x);
    {
        at::AutoDispatchBelowADInplaceOrView below;
        const int64_t N = x.size(-1);
        NormKept kept;
        const Tensor wc = vector_arg(w, N, x, "weight"), sc = vector_arg(scale, N, x, "scale"),
                     w2c = vector_arg(w2, N, x, o.defined() ? "next_weight" : "weight");
        for (const Tensor& t : norm_forward(orow, grow, xr, wc, sc, w2c, eps, x.sizes(), checkpoint, &kept))
            if (t.defined()) out.push_back(t);
        node->keep({kept.o, kept.g, kept.x, kept.o8.q, kept.o8.scale, kept.g8.q, kept.g8.scale, kept.x8.q, kept.x8.scale, wc,
                    sc, w2c, kept.stats});
        node->shape = x.sizes().vec();
        node->act = (o.defined() ? o : x).scalar_type();
        node->res = x.scalar_type();
        node->R0 = (int)xr.size(0);
        node->R1 = xr.dim() == 3 ? (int)xr.size(1) : 1;
        node->block = o.defined();
    }
    torch::autograd::set_history(out, node);
    return out;
}

// over one column v - e <v e> cancels to eps / x^2 of v, which 32-bit norms do not resolve
void check_width(const Tensor& x) {
    if (x.dim() == 0 || x.size(-1) < 2) refuse(text("a norm needs (..., N) tensors with N >= 2, got ", x.sizes()));
}

void check_rows(const Tensor& o, const Tensor& g, const Tensor& x, const Tensor& w, const Tensor& scale) {
    check_activation(o, "o");
    check_like(g, o, o.scalar_type(), "g");
    if (x.scalar_type() != o.scalar_type() && x.scalar_type() != at::kFloat)
        refuse(text("x must be ", o.scalar_type(), " or Float, got ", x.scalar_type()));
    check_like(x, o, x.scalar_type(), "x");
    check_width(o);
    if (!w.defined() || !scale.defined()) refuse("weight and scale are needed");
}

py::tuple norm_gate_residual(Tensor o, Tensor g, Tensor x, OptTensor w_, OptTensor scale_, OptTensor w2_, double eps, bool checkpoint) {
    const Tensor w = given(w_), scale = given(scale_), w2 = given(w2_);
    check_rows(o, g, x, w, scale);
    check_tangents("norm_gate_residual", {&o, &g, &x, &w, &scale, &w2});
    const int64_t N = x.size(-1);
    if (o.numel() == 0) {
        const Tensor y = x + (o * w * scale * g).to(x.scalar_type());
        return py::make_tuple(y, w2.defined() ? py::cast((y * w2).to(o.scalar_type())) : py::none());
    }
    if (wanted({&o, &g, &x, &w, &scale, &w2})) {
        const variable_list r = norm_with_graph(o, g, x, w, scale, w2, eps, checkpoint);
        return py::make_tuple(r[0], r.size() > 1 ? py::cast(r[1]) : py::none());
    }
    const variable_list r = norm_forward(rows_form(o), rows_form(g), rows_form(x), vector_arg(w, N, x, "weight"),
                                         vector_arg(scale, N, x, "scale"), vector_arg(w2, N, x, "next_weight"), eps, x.sizes(), false, nullptr);
    return py::make_tuple(r[0], w2.defined() ? py::cast(r[1]) : py::none());
}

Tensor rms_norm(Tensor x, OptTensor w_, double eps, bool checkpoint) {
    const Tensor w = given(w_);
    check_activation(x, "x");
    check_width(x);
    if (!w.defined()) refuse("weight is needed");
    check_tangents("rms_norm", {&x, &w});
    if (x.numel() == 0) return (x * w).to(x.scalar_type());
    if (wanted({&x, &w})) return norm_with_graph(Tensor(), Tensor(), x, Tensor(), Tensor(), w, eps, checkpoint)[0];
    return norm_forward(Tensor(), Tensor(), rows_form(x), Tensor(), Tensor(), vector_arg(w, x.size(-1), x, "weight"), eps,
                        x.sizes(), false, nullptr)[1];
}

// ---------------------------------------------------------------- residual addition, norm --

// x', u; with `pack` u8, with `stats` the rows' norms
variable_list add_norm_forward(const Tensor& x, const Tensor& y, const Tensor& w, double eps, at::IntArrayRef shape, Packed* u8, Tensor* stats) {
    const c10::DeviceGuard guard(x.device());
    const int R0 = as_int(x.size(0)), R1 = x.dim() == 3 ? as_int(x.size(1)) : 1, N = as_int(x.size(-1));
    const int64_t rows = (int64_t)R0 * R1;
    Tensor xo = at::empty(shape, x.options()), u = at::empty(shape, y.options());
    delrec_add_norm_fwd_args a{};
    if (stats) {
        *stats = at::empty({rows}, x.options().dtype(at::kFloat));
        a.stats = fptr(*stats);
    }
    if (u8) {
        *u8 = Packed(rows, N, x);
        a.u8 = u8->arg();
    }
    a.R0 = R0; a.R1 = R1; a.N = N; a.bf16 = is_bf16(y); a.x_bf16 = is_bf16(x);
    a.x = rows_of(x); a.y = rows_of(y); a.w = fptr(w); a.eps = (float)eps;
    a.x_out = xo.data_ptr(); a.u = u.data_ptr();
    check(delrec_add_norm_fwd(&a, stream_of(x)), "delrec_add_norm_fwd");
    return {xo, u};
}

struct AddNormBackward : public KeptNode {
    std::string name() const override { return "AddNormBackward"; }
    std::vector<int64_t> shape;
    at::ScalarType act = at::kFloat, res = at::kFloat;
    int R0 = 0, R1 = 0;

    variable_list apply(variable_list&& grads) override {
        const variable_list s = take();
        const Tensor &w = s[2], &stats = s[3];
        refuse_capture("add_norm", stats);
        once_differentiable("add_norm");
        const Tensor dxo = rows_form(grads[0]), du = rows_form(grads[1]);
        if (!dxo.defined() && !du.defined()) return variable_list(3);
        const c10::DeviceGuard guard(stats.device());
        const int N = (int)shape.back();
        const auto f32 = stats.options();
        Tensor dx = at::empty(shape, f32.dtype(res)), dy, dw = at::empty({N}, f32);
        if (act != res) dy = at::empty(shape, f32.dtype(act));
        const Tensor ws = workspace(DELREC_WS_ADD_NORM_BWD, R0, R1, N, stats);
        delrec_add_norm_bwd_args a{};
        a.R0 = R0; a.R1 = R1; a.N = N; a.bf16 = act == at::kBFloat16; a.x_bf16 = res == at::kBFloat16;
        a.x = rows_of(s[0]); a.y = rows_of(s[1]); a.w = fptr(w); a.stats = fptr(stats);
        if (dxo.defined()) a.dx_out = rows_of(dxo);
        if (du.defined()) a.du = rows_of(du);
        a.dx = dx.data_ptr(); a.dy = dy.defined() ? dy.data_ptr() : nullptr; a.dw = fptr(dw);
        a.workspace = ws.data_ptr(); a.workspace_bytes = (size_t)ws.numel();
        check(delrec_add_norm_bwd(&a, stream_of(stats)), "delrec_add_norm_bwd");
        return {dx, dy.defined() ? dy : dx, dw};
    }
};

py::tuple add_norm(Tensor x, Tensor y, OptTensor w_, double eps, bool pack) {
    const Tensor w = given(w_);
    check_activation(y, "y");
    if (x.scalar_type() != y.scalar_type() && x.scalar_type() != at::kFloat)
        refuse(text("x must be ", y.scalar_type(), " or Float, got ", x.scalar_type()));
    check_like(x, y, x.scalar_type(), "x");
    check_width(x);
    if (!w.defined()) refuse("weight is needed");
    check_tangents("add_norm", {&x, &y, &w});
    const int64_t N = x.size(-1);
    Packed u8;
    variable_list out;
    if (x.numel() == 0) {
        const Tensor sum = x + y.to(x.scalar_type());
        out = {sum, (sum * w).to(y.scalar_type())};
        if (pack) u8 = Packed(x.numel() / N, N, x);
    } else if (wanted({&x, &y, &w})) {
        auto node = make_node<AddNormBackward>();
        node->set_next_edges(torch::autograd::collect_next_edges(x, y, w));
        const Tensor xr = kept_rows(x), yr = kept_rows(y);
        Tensor wc, stats;
        {
            at::AutoDispatchBelowADInplaceOrView below;
            wc = vector_arg(w, N, x, "weight");
            out = add_norm_forward(xr, yr, wc, eps, x.sizes(), pack ? &u8 : nullptr, &stats);
        }
        // x' in 32 bits is the sum itself; of bf16 the addends are kept. Detached (above the autograd
        // keys, so that changes in place are noticed): the node is not to hold what holds the node.
        const bool sum = x.scalar_type() == at::kFloat;
        node->keep({sum ? kept_rows(out[0].detach()) : xr, sum ? Tensor() : yr, wc, stats});
        node->shape = x.sizes().vec();
        node->act = y.scalar_type();
        node->res = x.scalar_type();
        node->R0 = (int)xr.size(0);
        node->R1 = xr.dim() == 3 ? (int)xr.size(1) : 1;
        torch::autograd::set_history(out, node);
    } else {
        out = add_norm_forward(rows_form(x), rows_form(y), vector_arg(w, N, x, "weight"), eps, x.sizes(), pack ? &u8 : nullptr, nullptr);
    }
    return py::make_tuple(out[0], out[1], pack ? py::cast(u8.q.narrow(1, 0, N)) : py::none(), pack ? py::cast(u8.scale) : py::none());
}

// ---------------------------------------------------------------- one step, 8 bits ----------

py::tuple gated_step(Tensor z, Tensor f, Tensor g, Tensor x, Tensor h, OptTensor w_, OptTensor scale_, OptTensor w2_,
                     OptTensor bias_, double eps, OptTensor h_out_) {
    Tensor w = given(w_), scale = given(scale_), w2 = given(w2_), bias = given(bias_), h_out = given(h_out_);
    check_rows(z, g, x, w, scale);
    check_like(f, z, z.scalar_type(), "f");
    if (z.dim() != 2 || z.size(0) == 0) refuse(text("gated_step takes (B, N) tensors with B > 0, got ", z.sizes()));
    check_like(h, z, at::kFloat, "h");
    check_tangents("gated_step", {&z, &f, &g, &x, &h, &w, &scale, &w2, &bias});
    if (wanted({&z, &f, &g, &x, &h, &w, &scale, &w2, &bias, &h_out}))
        throw std::runtime_error("gated_step has no backward pass: call it under torch.no_grad(), or gated_scan and "
                                 "norm_gate_residual");
    const c10::DeviceGuard guard(z.device());
    const int B = as_int(z.size(0)), N = as_int(z.size(1));
    const bool in_place = h_out.defined();
    if (in_place) {
        check_like(h_out, h, at::kFloat, "h_out");
        if (!h_out.is_contiguous() || h_out.is_neg()) refuse("h_out must be contiguous");
    } else {
        h_out = at::empty({B, N}, h.options());
    }
    z = rows_form(z); f = rows_form(f); g = rows_form(g); x = rows_form(x);
    h = dense(h);
    w = vector_arg(w, N, z, "weight"); scale = vector_arg(scale, N, z, "scale");
    w2 = vector_arg(w2, N, z, "next_weight"); bias = vector_arg(bias, N, z, "bias");
    if (in_place) check_state_out(h_out, "h_out", h, {&z, &f, &g, &x, &w, &scale, &w2, &bias});
    const Tensor xo = at::empty({B, N}, x.options());
    Tensor u;
    if (w2.defined()) u = at::empty({B, N}, z.options());
    auto step = [](const Tensor& t) { return delrec_rows{t.data_ptr(), 0, t.stride(0)}; };
    delrec_gated_step_args a{};
    a.B = B; a.N = N; a.bf16 = is_bf16(z); a.x_bf16 = is_bf16(x);
    a.z = step(z); a.f = step(f); a.g = step(g); a.x = step(x); a.h = fptr(h); a.bias = fptr(bias);
    a.w = fptr(w); a.scale = fptr(scale); a.w2 = fptr(w2); a.eps = (float)eps;
    a.h_out = fptr(h_out); a.x_out = xo.data_ptr(); a.u = u.defined() ? u.data_ptr() : nullptr;
    check(delrec_gated_step(&a, stream_of(z)), "delrec_gated_step");
    // a graph that kept the old state sees that it is gone, as after any operation in place
    if (in_place && !h_out.is_inference()) h_out.unsafeGetTensorImpl()->bump_version();
    return py::make_tuple(xo, u.defined() ? py::cast(u) : py::none(), h_out);
}

py::tuple pack8(Tensor x) {
    check_activation(x, "x");
    if (x.dim() == 0 || x.size(-1) == 0) refuse(text("pack8 takes a (..., N) tensor with N > 0, got ", x.sizes()));
    const c10::DeviceGuard guard(x.device());
    const int64_t N = x.size(-1), rows = x.numel() / N;
    const Packed p(rows, N, x);
    if (rows) {
        const Tensor v = rows_form(x.detach());
        delrec_pack8_args a{};
        a.R0 = as_int(v.size(0)); a.R1 = v.dim() == 3 ? as_int(v.size(1)) : 1; a.N = as_int(N); a.bf16 = is_bf16(x);
        a.x = rows_of(v); a.p = p.arg();
        check(delrec_pack8(&a, stream_of(x)), "delrec_pack8");
    }
    return py::make_tuple(p.q.narrow(1, 0, N), p.scale);
}

Tensor unpack8(Tensor q, Tensor scale, std::vector<int64_t> shape, py::object dtype) {
    if (!q.is_cuda()) throw std::runtime_error(text("delrec-mi355x unpacks 8 bits with a HIP kernel on the GPU; they are on ", q.device()));
    const auto type = torch::python::detail::py_object_to_dtype(dtype);
    const int64_t groups = q.dim() == 2 ? (q.size(1) + DELREC_PACK8_GROUP - 1) / DELREC_PACK8_GROUP : 0;
    if ((type != at::kFloat && type != at::kBFloat16) || q.dim() != 2 || q.scalar_type() != at::kChar ||
        scale.dim() != 2 || scale.size(0) != q.size(0) || scale.size(1) != groups || scale.scalar_type() != at::kFloat ||
        scale.device() != q.device())
        refuse(text("not a packed tensor: q ", describe(q), ", scale ", describe(scale), ", type ", type));
    int64_t n = 1;
    for (int64_t v : shape) n *= v;
    if (n != q.numel() || shape.empty() || shape.back() != q.size(1)) refuse(text("q ", q.sizes(), " does not fill ", at::IntArrayRef(shape)));
    const c10::DeviceGuard guard(q.device());
    // copies (a tensor saved on the host and brought back) have lost the rows' pitch
    const int64_t pitch = (q.size(1) + 3) / 4 * 4;
    if (n && (q.stride(0) != pitch || (q.stride(1) != 1 && q.size(1) > 1) || (uintptr_t)q.data_ptr() % 4)) {
        const Tensor own = at::empty({q.size(0), pitch}, q.options());
        q = own.narrow(1, 0, q.size(1)).copy_(q);
    }
    scale = scale.contiguous();
    const Tensor out = at::empty(shape, q.options().dtype(type));
    if (n) {
        delrec_pack8_args a{};
        a.R0 = 1; a.R1 = as_int(q.size(0)); a.N = as_int(q.size(1)); a.bf16 = type == at::kBFloat16;
        a.x = {out.data_ptr(), 0, q.size(1)};
        a.p = Packed(q, scale).arg();
        check(delrec_unpack8(&a, stream_of(q)), "delrec_unpack8");
    }
    return out;
}

}  // namespace

void bind_gated(py::module_& m) {
    m.def("gated_scan", &gated_scan, "gated linear recurrence (autograd)", py::arg("z"), py::arg("f"), py::arg("bias"),
          py::arg("h0"), py::arg("starts"), py::arg("lengths"), py::arg("checkpoint"));
    m.def("norm_gate_residual", &norm_gate_residual, "norms, gate and residual (autograd)", py::arg("o"), py::arg("g"),
          py::arg("x"), py::arg("weight"), py::arg("scale"), py::arg("next_weight"), py::arg("eps"), py::arg("checkpoint"));
    m.def("rms_norm", &rms_norm, "norm of rows (autograd)", py::arg("x"), py::arg("weight"), py::arg("eps"), py::arg("checkpoint"));
    m.def("add_norm", &add_norm, "residual addition and norm (autograd)", py::arg("x"), py::arg("y"), py::arg("weight"), py::arg("eps"),
          py::arg("pack"));
    m.def("gated_step", &gated_step, "one time step of the block", py::arg("z"), py::arg("f"), py::arg("g"), py::arg("x"),
          py::arg("h"), py::arg("weight"), py::arg("scale"), py::arg("next_weight"), py::arg("bias"), py::arg("eps"), py::arg("h_out"));
    m.def("pack8", &pack8, "rows to 8 bits", py::arg("x"));
    m.def("unpack8", &unpack8, "the values of 8-bit rows", py::arg("q"), py::arg("scale"), py::arg("shape"), py::arg("dtype"));
}
