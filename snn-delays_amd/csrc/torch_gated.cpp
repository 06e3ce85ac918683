// Host side of the gated-recurrence block's operators (delrec.gated, delrec.checkpoint8): argument
// checks, outputs and workspace from torch's caching allocator, calls of the C ABI
// (include/delrec.h), autograd Functions.
//
// In C++ because the smallest calls are bound by the host: a training pass of the scan at T32 B64
// N64, whose kernels take 15 us, took 235 us through Python Functions and the ctypes binding. The
// graph's nodes are torch::autograd::Node themselves: torch::autograd::Function keeps its values in
// a dictionary of boxed ones.
#include <torch/extension.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>

#include <c10/hip/HIPStream.h>
#include <hip/hip_runtime.h>

#include <mutex>
#include <sstream>
#include <stdexcept>
#include <string>

#include "delrec.h"

namespace py = pybind11;

namespace {

using at::Tensor;
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;
using OptTensor = c10::optional<Tensor>;

void check(int status, const char* fn) {
    if (status != DELREC_OK)
        throw std::runtime_error(std::string(fn) + " failed: status " + std::to_string(status) + " (" +
                                 delrec_strerror(status) + ")");
}

template <class... A>
std::string text(const A&... a) {
    std::ostringstream s;
    (s << ... << a);
    return s.str();
}

std::string describe(const Tensor& t) { return text(t.sizes(), " ", t.scalar_type(), " on ", t.device()); }

[[noreturn]] void refuse(const std::string& why) { throw py::value_error(why); }

Tensor given(const OptTensor& t) { return t ? *t : Tensor(); }

bool is_bf16(const Tensor& t) { return t.scalar_type() == at::kBFloat16; }

void check_activation(const Tensor& t, const char* what) {
    if (!t.is_cuda())
        throw std::runtime_error(text("delrec-mi355x runs ", what, " with HIP kernels on the GPU; it is on ", t.device()));
    if (t.scalar_type() != at::kFloat && !is_bf16(t)) refuse(text(what, " must be fp32 or bf16, got ", t.scalar_type()));
}

void check_like(const Tensor& t, const Tensor& like, at::ScalarType type, const char* what) {
    if (!t.defined() || t.sizes() != like.sizes() || t.device() != like.device() || t.scalar_type() != type)
        refuse(text(what, " is ", t.defined() ? describe(t) : "None", ", expected ", like.sizes(), " ", type, " on ", like.device()));
}

// contiguous, and with its values in memory (the imaginary part of a conjugated tensor has their
// opposites there); undefined stays so
Tensor dense(const Tensor& t) { return t.defined() ? t.resolve_neg().contiguous() : t; }

// contiguous fp32 (n) on x's device; undefined stays so
Tensor vector_arg(const Tensor& v, int64_t n, const Tensor& x, const char* what) {
    if (!v.defined()) return v;
    if (v.dim() != 1 || v.size(0) != n || v.device() != x.device())
        refuse(text(what, " is ", describe(v), ", expected [", n, "] on ", x.device()));
    return dense(v.to(at::kFloat));
}

bool wanted(std::initializer_list<const Tensor*> ts) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor* t : ts)
        if (t->defined() && t->requires_grad()) return true;
    return false;
}

// torch's own Functions refuse inputs with a forward-mode tangent; bare nodes would drop it
void check_tangents(const char* what, std::initializer_list<const Tensor*> ts) {
    for (const Tensor* t : ts)
        if (t->defined() && t->_fw_grad(0).defined()) throw std::runtime_error(text(what, " has no forward-mode derivative"));
}

void once_differentiable(const char* what) {
    if (at::GradMode::is_enabled()) throw std::runtime_error(text(what, " has no second derivative (create_graph=True)"));
}

// Forward calls can be captured in a graph. A captured backward pass has ended the process (a
// segmentation fault in hipStreamEndCapture, cause not known): it is refused before it launches.
void refuse_capture(const char* what, const Tensor& t) {
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    if (hipStreamIsCapturing(c10::hip::getCurrentHIPStream(t.get_device()).stream(), &status) == hipSuccess &&
        status != hipStreamCaptureStatusNone)
        throw std::runtime_error(text("the backward pass of ", what, " cannot be captured in a graph"));
}

// A node of the graph: what it keeps is freed after its backward, and a second backward through it
// raises torch's own error. Under the node's mutex, since backward passes of several threads may go
// through one graph.
struct KeptNode : public Node {
    std::vector<SavedVariable> kept;
    bool released = false;
    void keep(std::initializer_list<Tensor> ts) {
        kept.reserve(ts.size());
        for (const Tensor& t : ts) kept.emplace_back(t, false);
    }
    variable_list take() {
        std::lock_guard<std::mutex> lock(mutex_);
        if (released) throw std::runtime_error(torch::autograd::ERR_BACKWARD_TWICE);
        variable_list v;
        v.reserve(kept.size());
        for (const SavedVariable& t : kept) v.push_back(t.unpack());
        return v;
    }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        kept.clear();
        released = true;
    }
};

template <class N>
std::shared_ptr<N> make_node() { return std::shared_ptr<N>(new N(), torch::autograd::deleteNode); }

// (R0, R1, N) or (R, N), the last axis contiguous; a copy only where there is no such view
Tensor rows_form(Tensor t) {
    if (!t.defined()) return t;
    t = t.resolve_neg();
    if (t.dim() == 1) t = t.unsqueeze(0);
    else if (t.dim() > 3) t = t.reshape({-1, t.size(-1)});
    return t.stride(-1) == 1 || t.size(-1) == 1 ? t : t.contiguous();
}

// The same for a tensor that the graph keeps, to be called above the autograd keys: a view taken
// there shares its tensor's version counter, and one taken below them has its own, so that a change
// in place between forward and backward would go unnoticed. Detached: no node for the view.
Tensor kept_rows(const Tensor& t) {
    if (!t.defined() || ((t.dim() == 2 || t.dim() == 3) && t.stride(-1) == 1 && !t.is_neg())) return t;
    return rows_form(t.detach());
}

delrec_rows rows_of(const Tensor& t) {
    if (!t.defined()) return {nullptr, 0, 0};
    if (t.dim() == 3) return {t.data_ptr(), t.stride(0), t.stride(1)};
    return {t.data_ptr(), t.dim() == 2 ? t.stride(0) : 0, 0};
}

// rows of a contiguous (..., N) tensor, counted as (R0, R1)
delrec_rows dense_rows(const Tensor& t, int64_t R1, int64_t N) {
    if (!t.defined()) return {nullptr, 0, 0};
    return {t.data_ptr(), R1 * N, N};
}

int as_int(int64_t v) {
    if (v > INT32_MAX) refuse(text("a size of ", v, " is past 31 bits"));
    return (int)v;
}

struct Packed {
    Tensor q, scale;
    Packed() = default;
    Packed(int64_t rows, int64_t N, const Tensor& like)
        : q(at::empty({rows, (N + 3) / 4 * 4}, like.options().dtype(at::kChar))),
          scale(at::empty({rows, (N + DELREC_PACK8_GROUP - 1) / DELREC_PACK8_GROUP}, like.options().dtype(at::kFloat))) {}
    Packed(const Tensor& q_, const Tensor& s_) : q(q_), scale(s_) {}
    delrec_packed8 arg() const {
        if (!q.defined()) return {nullptr, nullptr};
        return {(int8_t*)q.data_ptr(), (float*)scale.data_ptr()};
    }
};

float* fptr(const Tensor& t) { return t.defined() ? (float*)t.data_ptr() : nullptr; }

Tensor workspace(int kind, int T, int B, int N, const Tensor& like) {
    size_t n = 0;
    check(delrec_query_workspace(kind, T, B, N, 1, 0, &n), "delrec_query_workspace");
    return n ? at::empty({(int64_t)n}, like.options().dtype(at::kByte)) : Tensor();
}

void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

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

py::tuple pair_of(const variable_list& v) { return py::make_tuple(v[0], v[1]); }

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
    if (starts.defined()) {
        if (starts.dim() != 2 || starts.size(0) != T || starts.size(1) != B || starts.device() != z.device())
            refuse(text("starts is ", describe(starts), ", expected [", T, ", ", B, "] on ", z.device()));
        starts = starts.to(at::kBool).contiguous();
    }
    if (lengths.defined()) {
        if (lengths.dim() != 1 || lengths.size(0) != B || lengths.device() != z.device() || !at::isIntegralType(lengths.scalar_type(), false))
            refuse(text("lengths is ", describe(lengths), ", expected [", B, "] integers on ", z.device()));
        lengths = lengths.to(at::kLong).contiguous();
    }
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
    m.def("gated_step", &gated_step, "one time step of the block", py::arg("z"), py::arg("f"), py::arg("g"), py::arg("x"),
          py::arg("h"), py::arg("weight"), py::arg("scale"), py::arg("next_weight"), py::arg("bias"), py::arg("eps"), py::arg("h_out"));
    m.def("pack8", &pack8, "rows to 8 bits", py::arg("x"));
    m.def("unpack8", &unpack8, "the values of 8-bit rows", py::arg("q"), py::arg("scale"), py::arg("shape"), py::arg("dtype"));
}
