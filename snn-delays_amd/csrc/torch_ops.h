// Shared host side of the torch operators (torch_gated.cpp, torch_selective.cpp): argument checks,
// views as rows, workspace, graph nodes.
#pragma once

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

// whether t has an element in [lo, hi), from dimension `dim` on at `at`
bool touches(const char* lo, const char* hi, const Tensor& t, const char* at, int64_t dim) {
    int64_t last = 0, count = 1;
    for (int64_t d = dim; d < t.dim(); ++d) last += (t.size(d) - 1) * t.stride(d), count *= t.size(d);
    const int64_t e = (int64_t)t.element_size();
    if (at >= hi || at + (last + 1) * e <= lo) return false;
    if (last + 1 <= count) return true;               // no gaps
    for (int64_t i = 0; i < t.size(dim) && (i == 0 || t.stride(dim)); ++i)
        if (touches(lo, hi, t, at + i * t.stride(dim) * e, dim + 1)) return true;
    return false;
}

// A step writes a contiguous `out` while other workgroups still read: it is the state itself, element for
// element (each is read before it is written), or shares no memory with what the step reads.
void check_state_out(const Tensor& out, const char* what, const Tensor& state, std::initializer_list<const Tensor*> inputs) {
    const char *lo = (const char*)out.data_ptr(), *hi = lo + out.nbytes();
    auto one = [&](const Tensor& t) {
        if (t.defined() && t.numel() && touches(lo, hi, t, (const char*)t.data_ptr(), 0))
            refuse(text(what, " shares memory with an input: it must be the state itself or memory of its own"));
    };
    if (state.data_ptr() != out.data_ptr()) one(state);
    for (const Tensor* t : inputs) one(*t);
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

Tensor workspace(int kind, int T, int B, int N, const Tensor& like, int L = 1) {
    size_t n = 0;
    check(delrec_query_workspace(kind, T, B, N, L, 0, &n), "delrec_query_workspace");
    return n ? at::empty({(int64_t)n}, like.options().dtype(at::kByte)) : Tensor();
}

void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

// starts (T, B) as bools, lengths (B) as 64-bit integers
void check_masks(Tensor& starts, Tensor& lengths, int64_t T, int64_t B, const Tensor& like) {
    if (starts.defined()) {
        if (starts.dim() != 2 || starts.size(0) != T || starts.size(1) != B || starts.device() != like.device())
            refuse(text("starts is ", describe(starts), ", expected [", T, ", ", B, "] on ", like.device()));
        starts = starts.to(at::kBool).contiguous();
    }
    if (lengths.defined()) {
        if (lengths.dim() != 1 || lengths.size(0) != B || lengths.device() != like.device() || !at::isIntegralType(lengths.scalar_type(), false))
            refuse(text("lengths is ", describe(lengths), ", expected [", B, "] integers on ", like.device()));
        lengths = lengths.to(at::kLong).contiguous();
    }
}
const uint8_t* starts_ptr(const Tensor& t) { return t.defined() ? (const uint8_t*)t.data_ptr() : nullptr; }
const int64_t* lengths_ptr(const Tensor& t) { return t.defined() ? (const int64_t*)t.data_ptr() : nullptr; }

py::tuple pair_of(const variable_list& v) { return py::make_tuple(v[0], v[1]); }

}  // namespace
