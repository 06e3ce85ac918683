// extern "C" entry points of the gated-recurrence block (declared in include/delrec.h): argument
// checks and launches. Nothing here allocates device memory or synchronises the stream.
#include <hip/hip_runtime.h>

#include "kernels.h"

namespace delrec {

// rows fit 31 bits, and so do columns with room for a workgroup's stride past them
static bool sizes_ok(int R0, int R1, int N) {
    return R0 > 0 && R1 > 0 && N > 0 && N <= 0x7fffffff - 1024 && (long long)R0 * R1 <= 0x7fffffffLL &&
           (long long)R0 * R1 <= (0x7fffffffLL * 64) / N;
}

// (the last of up to 128 ranges of time ends at most as many blocks of 64 steps past T)
bool gated_scan_sizes_ok(int T, int B, int N) { return sizes_ok(T, B, N) && T <= 0x7fffffff - 128 * DELREC_GATED_BLOCK; }

// (a norm's three column sums side by side count in 32 bits)
bool norm_gate_sizes_ok(int R0, int R1, int N) { return sizes_ok(R0, R1, N) && N >= 2 && N <= 1 << 30; }

}  // namespace delrec

using namespace delrec;

namespace {

int done() { return hipGetLastError() == hipSuccess ? DELREC_OK : DELREC_ERR_LAUNCH; }

bool pair_ok(const delrec_packed8& p) { return (p.q == nullptr) == (p.scale == nullptr); }

// the norms' 8-bit forms: of o, g and x together, of x alone without a block, or none (the kernels
// go by x8)
bool eights_ok(const delrec_packed8& o8, const delrec_packed8& g8, const delrec_packed8& x8, bool block) {
    const bool others = block && x8.q;
    return pair_ok(o8) && pair_ok(g8) && pair_ok(x8) && (o8.q != nullptr) == others && (g8.q != nullptr) == others;
}

}  // namespace

extern "C" {

int delrec_gated_scan_fwd(const delrec_gated_scan_fwd_args* a, void* stream) {
    if (!a || !gated_scan_sizes_ok(a->T, a->B, a->N)) return DELREC_ERR_ARG;
    if (!a->z.data || !a->f.data || !a->h.data || !a->h_last) return DELREC_ERR_ARG;
    if (!pair_ok(a->z8) || !pair_ok(a->f8) || (a->z8.q == nullptr) != (a->f8.q == nullptr)) return DELREC_ERR_ARG;
    if (a->z8.q && !a->states) return DELREC_ERR_ARG;
    GatedScan p{};
    p.T = a->T; p.B = a->B; p.N = a->N; p.bf16 = a->bf16 != 0;
    p.z = a->z; p.f = a->f; p.bias = a->bias; p.h0 = a->h0; p.starts = a->starts; p.lengths = a->lengths;
    p.h = a->h; p.h_last = a->h_last; p.states = a->states; p.z8 = a->z8; p.f8 = a->f8;
    const size_t need = gated_fwd_ws(a->T, a->B, a->N) * sizeof(float);
    if (need && (!a->workspace || a->workspace_bytes < need)) return DELREC_ERR_WORKSPACE;
    p.ws = static_cast<float*>(a->workspace);
    launch_gated_fwd(p, static_cast<hipStream_t>(stream));
    return done();
}

int delrec_gated_scan_bwd(const delrec_gated_scan_bwd_args* a, void* stream) {
    if (!a || !gated_scan_sizes_ok(a->T, a->B, a->N)) return DELREC_ERR_ARG;
    if (!pair_ok(a->z8) || !pair_ok(a->f8) || (a->z8.q == nullptr) != (a->f8.q == nullptr)) return DELREC_ERR_ARG;
    if (!a->z8.q && (!a->z.data || !a->f.data)) return DELREC_ERR_ARG;
    if (!a->states || !a->dh.data || !a->dz.data || !a->df.data) return DELREC_ERR_ARG;
    GatedScan p{};
    p.T = a->T; p.B = a->B; p.N = a->N; p.bf16 = a->bf16 != 0;
    p.z = a->z; p.f = a->f; p.z8 = a->z8; p.f8 = a->f8; p.bias = a->bias; p.starts = a->starts; p.lengths = a->lengths;
    p.states = const_cast<float*>(a->states); p.dh = a->dh; p.dlast = a->dlast; p.dz = a->dz; p.df = a->df;
    p.db = a->db; p.dh0 = a->dh0;
    const size_t need = gated_bwd_ws(a->T, a->B, a->N) * sizeof(float);
    if (!a->workspace || a->workspace_bytes < need) return DELREC_ERR_WORKSPACE;
    p.ws = static_cast<float*>(a->workspace);
    launch_gated_bwd(p, static_cast<hipStream_t>(stream));
    return done();
}

int delrec_gated_step(const delrec_gated_step_args* a, void* stream) {
    if (!a || !norm_gate_sizes_ok(1, a->B, a->N)) return DELREC_ERR_ARG;
    if (!a->z.data || !a->f.data || !a->g.data || !a->x.data || !a->h || !a->h_out || !a->x_out) return DELREC_ERR_ARG;
    if (!a->w || !a->scale || (a->w2 && !a->u) || !(a->eps >= 0.0f)) return DELREC_ERR_ARG;
    if (!a->bf16 && a->x_bf16) return DELREC_ERR_UNSUPPORTED;
    NormGate p{};
    p.R0 = 1; p.R1 = a->B; p.N = a->N; p.bf16 = a->bf16 != 0; p.x_bf16 = a->x_bf16 != 0;
    p.z = a->z; p.f = a->f; p.g = a->g; p.x = a->x; p.h = a->h; p.bias = a->bias; p.w = a->w; p.scale = a->scale;
    p.w2 = a->w2; p.eps = a->eps; p.h_out = a->h_out; p.x_out = a->x_out; p.u = a->u;
    launch_norm_gate(p, true, static_cast<hipStream_t>(stream));
    return done();
}

int delrec_norm_gate_fwd(const delrec_norm_gate_fwd_args* a, void* stream) {
    if (!a || !norm_gate_sizes_ok(a->R0, a->R1, a->N)) return DELREC_ERR_ARG;
    const bool block = a->o.data != nullptr;
    if (!a->x.data || !(a->eps >= 0.0f) || (a->w2 && !a->u)) return DELREC_ERR_ARG;
    if (block && (!a->g.data || !a->w || !a->scale || !a->x_out)) return DELREC_ERR_ARG;
    if (!block && !a->w2) return DELREC_ERR_ARG;
    if (!eights_ok(a->o8, a->g8, a->x8, block)) return DELREC_ERR_ARG;
    if (!a->bf16 && a->x_bf16) return DELREC_ERR_UNSUPPORTED;
    NormGate p{};
    p.R0 = a->R0; p.R1 = a->R1; p.N = a->N; p.bf16 = a->bf16 != 0; p.x_bf16 = a->x_bf16 != 0;
    p.o = a->o; p.g = a->g; p.x = a->x; p.w = block ? a->w : nullptr; p.scale = a->scale; p.w2 = a->w2; p.eps = a->eps;
    p.x_out = a->x_out; p.u = a->u; p.stats = a->stats; p.o8 = a->o8; p.g8 = a->g8; p.x8 = a->x8;
    launch_norm_gate(p, true, static_cast<hipStream_t>(stream));
    return done();
}

int delrec_norm_gate_bwd(const delrec_norm_gate_bwd_args* a, void* stream) {
    if (!a || !norm_gate_sizes_ok(a->R0, a->R1, a->N)) return DELREC_ERR_ARG;
    const bool block = a->o.data || a->o8.q;
    if (!eights_ok(a->o8, a->g8, a->x8, block)) return DELREC_ERR_ARG;
    if ((!a->x.data && !a->x8.q) || !a->stats || !a->dx.data) return DELREC_ERR_ARG;
    if (!a->dx_out.data && !a->du.data) return DELREC_ERR_ARG;
    if (block && ((!a->g.data && !a->g8.q) || !a->w || !a->scale || !a->d_o.data || !a->dg.data || !a->dw || !a->dscale))
        return DELREC_ERR_ARG;
    if (!block && !a->w2) return DELREC_ERR_ARG;
    if (a->w2 && !a->dw2) return DELREC_ERR_ARG;
    if (!a->bf16 && a->x_bf16) return DELREC_ERR_UNSUPPORTED;
    NormGate p{};
    p.R0 = a->R0; p.R1 = a->R1; p.N = a->N; p.bf16 = a->bf16 != 0; p.x_bf16 = a->x_bf16 != 0;
    p.o = a->o; p.g = a->g; p.x = a->x; p.o8 = a->o8; p.g8 = a->g8; p.x8 = a->x8;
    p.w = block ? a->w : nullptr; p.scale = a->scale; p.w2 = a->w2; p.stats = const_cast<float*>(a->stats);
    p.dx_out = a->dx_out; p.du = a->du; p.d_o = a->d_o; p.dg = a->dg; p.dx = a->dx;
    p.dw = block ? a->dw : nullptr; p.dscale = block ? a->dscale : nullptr; p.dw2 = a->w2 ? a->dw2 : nullptr;
    const size_t need = norm_gate_bwd_ws((long long)a->R0 * a->R1, a->N) * sizeof(float);
    if (!a->workspace || a->workspace_bytes < need) return DELREC_ERR_WORKSPACE;
    p.part = static_cast<float*>(a->workspace);
    launch_norm_gate(p, false, static_cast<hipStream_t>(stream));
    return done();
}

static int pack_call(const delrec_pack8_args* a, bool pack, void* stream) {
    if (!a || !sizes_ok(a->R0, a->R1, a->N) || !a->x.data || !a->p.q || !a->p.scale) return DELREC_ERR_ARG;
    launch_pack8({a->R0, a->R1, a->N, a->bf16 != 0, a->x, a->p}, pack, static_cast<hipStream_t>(stream));
    return done();
}

int delrec_pack8(const delrec_pack8_args* a, void* stream) { return pack_call(a, true, stream); }
int delrec_unpack8(const delrec_pack8_args* a, void* stream) { return pack_call(a, false, stream); }

}  // extern "C"
