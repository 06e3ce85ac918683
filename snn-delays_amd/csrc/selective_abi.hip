// extern "C" entry points of the selective state-space block (declared in include/delrec.h): argument
// checks and launches. Nothing here allocates device memory or synchronises the stream.
#include <hip/hip_runtime.h>

#include "kernels.h"

namespace delrec {

// rows and steps fit 31 bits with room for a block of steps past the last, columns for a workgroup's;
// the sums over rows are counted in 64 bits
static bool sizes_ok(int T, int B, int N) {
    return T > 0 && B > 0 && N > 0 && T <= 0x7fffffff - 1024 && N <= 0x7fffffff - 1024 && (long long)T * B <= 0x7fffffffLL &&
           (long long)T * B <= (0x7fffffffLL * 64) / N;
}

bool selective_sizes_ok(int T, int B, int N, int S) { return sizes_ok(T, B, N) && S >= 1 && S <= 64; }
bool conv_sizes_ok(int T, int B, int N, int W) { return sizes_ok(T, B, N) && W >= 2 && W <= 8; }

}  // namespace delrec

using namespace delrec;

namespace {

int done() { return hipGetLastError() == hipSuccess ? DELREC_OK : DELREC_ERR_LAUNCH; }

}  // namespace

extern "C" {

int delrec_causal_conv_fwd(const delrec_causal_conv_fwd_args* a, void* stream) {
    if (!a || !conv_sizes_ok(a->T, a->B, a->N, a->W)) return DELREC_ERR_ARG;
    if (!a->x.data || !a->w || !a->y.data) return DELREC_ERR_ARG;
    if (a->state_out && a->state_out == a->state && a->T != 1) return DELREC_ERR_ARG;
    CausalConv p{};
    p.T = a->T; p.B = a->B; p.N = a->N; p.W = a->W; p.bf16 = a->bf16 != 0; p.silu = a->silu != 0;
    p.x = a->x; p.w = a->w; p.bias = a->bias; p.state = a->state; p.starts = a->starts; p.lengths = a->lengths;
    p.y = a->y; p.state_out = a->state_out;
    launch_conv(p, true, static_cast<hipStream_t>(stream));
    return done();
}

int delrec_causal_conv_bwd(const delrec_causal_conv_bwd_args* a, void* stream) {
    if (!a || !conv_sizes_ok(a->T, a->B, a->N, a->W)) return DELREC_ERR_ARG;
    if (!a->x.data || !a->w || !a->dy.data || !a->dx.data || !a->dw) return DELREC_ERR_ARG;
    CausalConv p{};
    p.T = a->T; p.B = a->B; p.N = a->N; p.W = a->W; p.bf16 = a->bf16 != 0; p.silu = a->silu != 0;
    p.x = a->x; p.w = a->w; p.bias = a->bias; p.state = a->state; p.starts = a->starts; p.lengths = a->lengths;
    p.dy = a->dy; p.dstate_out = a->dstate_out; p.dx = a->dx; p.dstate = a->dstate; p.dw = a->dw; p.db = a->db;
    const size_t need = conv_bwd_ws(a->T, a->B, a->N, a->W) * sizeof(float);
    if (!a->workspace || a->workspace_bytes < need) return DELREC_ERR_WORKSPACE;
    p.part = static_cast<float*>(a->workspace);
    launch_conv(p, false, static_cast<hipStream_t>(stream));
    return done();
}

int delrec_selective_scan_fwd(const delrec_selective_scan_fwd_args* a, void* stream) {
    if (!a || !selective_sizes_ok(a->T, a->B, a->N, a->S)) return DELREC_ERR_ARG;
    if (!a->x.data || !a->dt.data || !a->Bm.data || !a->C.data || !a->A || !a->y.data || !a->h_last) return DELREC_ERR_ARG;
    Selective p{};
    p.T = a->T; p.B = a->B; p.N = a->N; p.S = a->S; p.bf16 = a->bf16 != 0;
    p.x = a->x; p.dt = a->dt; p.g = a->g; p.Bm = a->Bm; p.C = a->C; p.A = a->A; p.D = a->D; p.dt_bias = a->dt_bias;
    p.h0 = const_cast<float*>(a->h0); p.starts = a->starts; p.lengths = a->lengths; p.y = a->y; p.h_last = a->h_last;
    p.states = a->states;
    const size_t need = selective_fwd_ws(a->T, a->B, a->N, a->S) * sizeof(float);
    if (need && (!a->workspace || a->workspace_bytes < need)) return DELREC_ERR_WORKSPACE;
    p.ws = static_cast<float*>(a->workspace);
    launch_selective_fwd(p, static_cast<hipStream_t>(stream));
    return done();
}

int delrec_selective_scan_bwd(const delrec_selective_scan_bwd_args* a, void* stream) {
    if (!a || !selective_sizes_ok(a->T, a->B, a->N, a->S)) return DELREC_ERR_ARG;
    if (!a->x.data || !a->dt.data || !a->Bm.data || !a->C.data || !a->A || !a->states || !a->dy.data) return DELREC_ERR_ARG;
    if (!a->dx.data || !a->ddt.data || !a->dBm || !a->dC || (a->g.data && !a->dg.data)) return DELREC_ERR_ARG;
    Selective p{};
    p.T = a->T; p.B = a->B; p.N = a->N; p.S = a->S; p.bf16 = a->bf16 != 0;
    p.x = a->x; p.dt = a->dt; p.g = a->g; p.Bm = a->Bm; p.C = a->C; p.A = a->A; p.D = a->D; p.dt_bias = a->dt_bias;
    p.states = const_cast<float*>(a->states); p.starts = a->starts; p.lengths = a->lengths; p.dy = a->dy; p.dlast = a->dlast;
    p.dx = a->dx; p.ddt = a->ddt; p.dg = a->dg; p.dB = a->dBm; p.dC = a->dC; p.dA = a->dA; p.dD = a->dD; p.dbias = a->ddt_bias;
    p.dh0 = a->dh0;
    const size_t need = selective_bwd_ws(a->T, a->B, a->N, a->S) * sizeof(float);
    if (!a->workspace || a->workspace_bytes < need) return DELREC_ERR_WORKSPACE;
    p.ws = static_cast<float*>(a->workspace);
    launch_selective_bwd(p, static_cast<hipStream_t>(stream));
    return done();
}

int delrec_selective_step(const delrec_selective_step_args* a, void* stream) {
    if (!a || !selective_sizes_ok(1, a->B, a->N, a->S)) return DELREC_ERR_ARG;
    if (!a->x.data || !a->dt.data || !a->Bm.data || !a->C.data || !a->A || !a->h || !a->h_out || !a->y) return DELREC_ERR_ARG;
    Selective p{};
    p.T = 1; p.B = a->B; p.N = a->N; p.S = a->S; p.bf16 = a->bf16 != 0;
    p.x = a->x; p.dt = a->dt; p.g = a->g; p.Bm = a->Bm; p.C = a->C; p.A = a->A; p.D = a->D; p.dt_bias = a->dt_bias;
    p.h0 = a->h; p.h_last = a->h_out; p.y = {a->y, 0, a->N};
    launch_selective_step(p, static_cast<hipStream_t>(stream));
    return done();
}

}  // extern "C"
