// Gated linear recurrence over (T, B, N) sequences and its reverse pass.
//     k_t = sigmoid(-(f_t + bias)), h_t = h_{t-1} + k_t (z_t - h_{t-1})
// backwards, with lam_t = dh_t + c_{t+1} and c_t = (1 - k_t) lam_t (c_T = dlast):
//     dz_t = lam_t k_t, df_t = lam_t k_t (1 - k_t) (h_{t-1} - z_t), dh0 = c_0, db = sum df.
// Both are affine in what they carry, h -> A h + S and c -> A c + S with A the product of the
// leaks 1 - k, and affine maps compose: time is cut into pieces that run side by side.
//
// A workgroup takes 64 V channels (V consecutive ones a lane) and walks time in blocks of 64
// steps, eight per wave: each wave loads its steps, composes them from nothing into (A, S), the
// waves exchange these through LDS (one barrier a block, two buffers), every wave composes those
// before it onto the block's state, and runs its steps again from there, out of registers. So z
// and f are read once and h is written once, whatever T. With too few channels to fill the GPU
// time is cut a second time, over the grid: a first launch composes each range (reading its
// inputs once more), the second starts from the composition of the ranges before it.
//
// Bound by memory where the channels fill the GPU: at T250 B128 N512 bf16 23 us forward (98 MB,
// 4.3 TB/s) and 34 backward (164 MB, 4.8 TB/s, what a large copy reaches); next, by vector issue (24
// instructions a value forward and 42 backward, two of them at a quarter of the rate; 49 and 44 with 8
// bits). A block's loads are not taken ahead of the one before: two to four workgroups a CU hide
// them, and their registers cost one of these.
//
// The forward keeps the state before every 64th step in 32 bits (1/16 byte a value and step); the
// backward starts its blocks there and recomputes the states between from z and f, which it needs
// anyway: exact in 32 bits where reading h back would bring its bf16 rounding into df, and two to
// four bytes a value less to read.
#include <algorithm>

#include "gated.h"
#include "kernels.h"

namespace delrec {

#define DELREC_GLOBAL __attribute__((address_space(1)))

namespace {

constexpr int kBlk = DELREC_GATED_BLOCK;
constexpr int kSteps = 8;                    // steps of a wave in a block
constexpr int kWaves = kBlk / kSteps;

// A start inside a piece cuts what comes before it off, also where that is infinite: the sign of A
// says so (products of leaks are never negative, and a further leak, zero too, keeps the sign).
// Only the masked forms have it.
__device__ __forceinline__ bool cut(float A) { return __float_as_int(A) < 0; }
template <bool MASK>
__device__ __forceinline__ float apply(float A, float S, float h) {
    const float r = fmaf(A, h, S);
    return MASK && cut(A) ? S : r;
}
template <bool MASK>
__device__ __forceinline__ float product(float A, float B) {
    return MASK && cut(A) && cut(B) ? -1.0f : A * B;
}

__device__ __forceinline__ int row_length(const GatedScan& p, int b) {
    if (!p.lengths) return p.T;
    const int64_t v = p.lengths[b];
    return v < 0 ? 0 : (v < p.T ? (int)v : p.T);
}

// the lane's channels: row b, columns n0 .. n0 + V - 1. The last lane of a row whose width is no
// multiple of V is moved back to end with it and repeats `skip` columns of the lane before (the
// same values, written twice). Lanes past the last row, and with 8-bit groups the lanes that fill
// a row's last group up, repeat valid columns and write nothing.
template <int V>
struct Lane {
    int b, b0, n0, skip, group;              // b0: the wave's first row; group: of the first own column
    bool on, first;                          // writes; first lane of its 8-bit group
    int i;                                   // nominal first column
    __device__ __forceinline__ Lane(const GatedScan& p, int per_row) {
        const long long c = ((long long)p.first + blockIdx.x) * 64 + (threadIdx.x & 63);
        const long long rows = c / per_row;
        b = rows < p.B ? (int)rows : p.B - 1;
        b0 = __builtin_amdgcn_readfirstlane(b);
        i = (int)(c - rows * per_row) * V;
        on = rows < p.B && i < p.N;
        first = on && i % kGroup8 == 0;
        n0 = i < p.N - V ? i : p.N - V;
        skip = on ? i - n0 : V;
        group = min(i, p.N - 1) / kGroup8;
    }
};

// A (T, B, ..) array as a lane walks it: a step's address is one base for the wave, in scalar
// registers and moved by additions, and the lane's 32-bit distance from it (checked by the
// launcher; V = 1 has 64-bit distances). A multiplication a step and access kept the scalar unit,
// which the four SIMDs share, busier than the memory.
template <class T, int V>
struct Walk {
    const char* base;
    long long pitch;
    typename std::conditional<V == 1, long long, uint32_t>::type off, here;
    uint64_t cur;
    // element (t, b, n) of `data` at t * s0 + b * s1 + n
    __device__ __forceinline__ Walk(const void* data, long long s0, long long s1, int b, int b0, int n)
        : base((const char*)data + b0 * s1 * (long long)sizeof(T)), pitch(s0 * (long long)sizeof(T)) {
        if constexpr (V == 1) off = ((b - b0) * s1 + n) * (long long)sizeof(T);
        else off = ((uint32_t)(b - b0) * (uint32_t)s1 + (uint32_t)n) * (uint32_t)sizeof(T);
    }
    __device__ __forceinline__ void seek(int t) { cur = (uint64_t)(base + t * pitch); }
    // before a run of accesses: the lane's distance anew, in the basic block that uses it (or the
    // compiler widens it once and for all and adds it to every base in vector registers)
    __device__ __forceinline__ void start() {
        here = off;
        if constexpr (V > 1) asm("" : "+v"(here));
    }
    __device__ __forceinline__ void next() { cur += pitch; }
    __device__ __forceinline__ void prev() { cur -= pitch; }
    // The base is kept apart from the lane's distance (an empty asm, or the compiler adds both into
    // 64-bit lane addresses for all steps ahead, and their registers cost a wave per SIMD).
    __device__ __forceinline__ DELREC_GLOBAL char* at() const {
        uint64_t a = cur;
        if constexpr (V > 1) {
            a = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)a) |
                (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(a >> 32)) << 32;
            asm("" : "+s"(a));
        }
        return (DELREC_GLOBAL char*)a + here;
    }
    template <class E>
    __device__ __forceinline__ E value() const { return *(const DELREC_GLOBAL E*)at(); }
    __device__ __forceinline__ Vec<T, V> load() const {
        Vec<T, V> r;
        if constexpr (V > 1) r.v = *(const DELREC_GLOBAL typename Vec<T, V>::unaligned*)at();
        else r.v = *(const DELREC_GLOBAL T*)at();
        return r;
    }
    // without the first `skip`
    __device__ __forceinline__ void store(const float* x, int skip = 0) const {
        DELREC_GLOBAL char* q = at();
        if constexpr (V > 1) {
            typename Vec<float, V>::type v;
#pragma unroll
            for (int j = 0; j < V; ++j) v[j] = x[j];
            if (skip == 0) *(DELREC_GLOBAL typename Vec<T, V>::unaligned*)q = __builtin_convertvector(v, typename Vec<T, V>::type);
            else
#pragma unroll
                for (int j = 1; j < V; ++j)
                    if (j >= skip) ((DELREC_GLOBAL T*)q)[j] = (T)x[j];
        } else if (skip == 0) {
            *(DELREC_GLOBAL T*)q = (T)x[0];
        }
    }
};

// a tensor's 8 bits and their scales, walked together
template <int V>
struct Walk8 {
    Walk<int8_t, V> q;
    Walk<float, V> scale;
    const Lane8<V>& ln;
    __device__ __forceinline__ Walk8(const delrec_packed8& p, int B, int N, int b, int b0, int group, const Lane8<V>& l)
        : q(p.q, (long long)B * pitch8(N), pitch8(N), b, b0, l.at),
          scale(p.scale, (long long)B * ((N + kGroup8 - 1) / kGroup8), (N + kGroup8 - 1) / kGroup8, b, b0, group), ln(l) {}
    __device__ __forceinline__ void seek(int t) { q.seek(t); scale.seek(t); }
    __device__ __forceinline__ void start() { q.start(); scale.start(); }
    __device__ __forceinline__ void next() { q.next(); scale.next(); }
    __device__ __forceinline__ void prev() { q.prev(); scale.prev(); }
    __device__ __forceinline__ Vec8<V> load() const {
        Vec8<V> r;
        r.q = q.template value<typename Word8<V>::type>();
        r.scale = scale.template value<float>();
        return r;
    }
    // the lane's own columns, apart from the loads: a shift next to each load is waited for there
    // (402 us instead of 245 for the backward of T1024 B64 N2048)
    __device__ __forceinline__ void own(Vec8<V>& x) const { x.q <<= ln.shift; }
    __device__ __forceinline__ void store(const float* x, bool first) const {
        float sc;
        const uint32_t word = quantise8<V>(x, ln, &sc);
        if (ln.on) *(DELREC_GLOBAL typename Word8<V>::type*)q.at() = (typename Word8<V>::type)word;
        if (first) *(DELREC_GLOBAL float*)scale.at() = sc;
    }
};

// The exchange: the waves' maps of a block in LDS, a lane's V leaks and V sums in one access. Waves
// that a short T leaves out of the launch count as maps that change nothing.
template <int V>
struct Maps {
    typedef float entry __attribute__((ext_vector_type(2 * V)));
    entry m[2][kWaves][64];
    __device__ __forceinline__ void put(int buf, int w, int lane, const float* a, const float* s) {
        entry e;
#pragma unroll
        for (int j = 0; j < V; ++j) e[j] = a[j], e[V + j] = s[j];
        m[buf][w][lane] = e;
    }
    __device__ __forceinline__ void fill_missing(int w, int nw, int lane) {
        entry e;
#pragma unroll
        for (int j = 0; j < V; ++j) e[j] = 1.0f, e[V + j] = 0.0f;
        for (int q = nw + w; q < kWaves; q += nw) m[0][q][lane] = m[1][q][lane] = e;
    }
    template <bool MASK>
    __device__ __forceinline__ entry run(int buf, int w, int lane, float* h) const {
        const entry e = m[buf][w][lane];
#pragma unroll
        for (int j = 0; j < V; ++j) h[j] = apply<MASK>(e[j], e[V + j], h[j]);
        return e;
    }
};

// The state that a range starts from: the maps of the ranges `from`, from + dir, .. (count of
// them) composed onto h by all waves together, through the exchange's first buffer.
template <int V, bool MASK>
__device__ __forceinline__ void enter_range(Maps<V>& m, const float* agg, size_t plane, size_t at, int from, int dir,
                                            int count, int w, int nw, int lane, float* h) {
    const int per = (count + nw - 1) / nw, q0 = min(w * per, count), q1 = min(q0 + per, count);
    float A[V], S[V];
#pragma unroll
    for (int j = 0; j < V; ++j) A[j] = 1.0f, S[j] = 0.0f;
    for (int q = q0; q < q1; ++q) {
        const float* a = agg + (size_t)(from + dir * q) * 2 * plane + at;
        const auto qa = vload<float, V>(a), qs = vload<float, V>(a + plane);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            S[j] = apply<MASK>(qa.get(j), qs.get(j), S[j]);
            A[j] = product<MASK>(A[j], qa.get(j));
        }
    }
    m.put(0, w, lane, A, S);
    barrier_lds();
#pragma unroll
    for (int q = 0; q < kWaves; ++q) m.template run<MASK>(0, q, lane, h);
    barrier_lds();                           // the buffer is free again
}

// A step's gates and leaks (gate_small2). f (and z, below) are vectors of any kind that get() reads,
// bias2 the bias times log2(e); off: the step is past the row's end.
template <int V, class F>
__device__ __forceinline__ void gate(const F& f, const float* bias2, bool off, float* m) {
#pragma unroll
    for (int j = 0; j < V; ++j) m[j] = off ? 0.0f : gate_small2(f.get_fma(j, kLog2e, bias2[j]));
}

// One step composed onto a piece's map (A, L), forwards (past the row's end L stays, and is not
// multiplied by the shut gate's zero: it may be infinite)
template <int V, bool MASK, class F>
__device__ __forceinline__ void step_forward(const float* m, const F& z, bool fresh, bool off, float* A, float* L) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const float from = MASK && fresh ? 0.0f : L[j], l = gate_step(m[j], from - z.get(j), from, z.get(j));
        L[j] = off ? L[j] : l;
        A[j] = MASK && fresh ? -1.0f : leak_times(m[j], A[j]);
    }
}

// and backwards, c -> a (dh + c), whose leak A is the forward map's
template <int V, bool MASK, class D>
__device__ __forceinline__ void step_backward(const float* m, const D& dh, bool fresh, bool off, float* L) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const float l = leak_times(m[j], dh.get(j) + L[j]);
        L[j] = MASK && fresh ? 0.0f : off ? L[j] : l;
    }
}
template <int V, bool MASK>
__device__ __forceinline__ void step_leak(const float* m, bool fresh, float* A) {
#pragma unroll
    for (int j = 0; j < V; ++j) A[j] = MASK && fresh ? -1.0f : leak_times(m[j], A[j]);
}

// Padding, and the steps past T of the last block. A wave whose lanes are all past their rows' ends
// loads nothing and leaves the state alone; where only some are, or some of the steps, what they
// loaded is replaced, whatever it is: z and dh by 0, and the gate itself by one that lets nothing in
// (k = 0; no value of f does that under every bias).
template <class S, int V>
__device__ __forceinline__ void blank(Vec<S, V>& x) {
    if constexpr (V > 1) {
#pragma unroll
        for (int j = 0; j < V; ++j) x.v[j] = (S)0.0f;
    } else {
        x.v = (S)0.0f;
    }
}
template <int V>
__device__ __forceinline__ void blank(Vec8<V>& x) {
    x.q = 0;
    x.scale = 0.0f;
}

// The maps of all waves applied to h in the order of DIR, what comes before this wave's own in
// `mine`. All reads are under way before the first is used.
template <int V, bool MASK, int DIR>
__device__ __forceinline__ void compose(const Maps<V>& m, int buf, int w, int lane, float* h, float* mine) {
#pragma unroll
    for (int c = 0; c < kWaves; ++c) {
        const int q = DIR > 0 ? c : kWaves - 1 - c;
        if (q == w) {
            asm volatile("");                // a branch (w is the wave's), not two selects a wave
#pragma unroll
            for (int j = 0; j < V; ++j) mine[j] = h[j];
        }
        m.template run<MASK>(buf, q, lane, h);
    }
}

}  // namespace

// (a block's loads come in two forms: without a branch between them, and with a test each where the
// last steps are past T)
#define DELREC_STEPS(s) _Pragma("unroll") for (int s = 0; s < kSteps; ++s)
#define DELREC_STEPS_BACK(s) _Pragma("unroll") for (int s = kSteps - 1; s >= 0; --s)
#define DELREC_COLS(j) _Pragma("unroll") for (int j = 0; j < V; ++j)

// PACK: z and f also to 8 bits.
template <class S, int V, bool MASK, bool PACK>
__global__ void __launch_bounds__(512, 4) gated_fwd_kernel(GatedScan p, int per_row, int range) {
    __shared__ Maps<V> maps;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), nw = blockDim.x >> 6;
    const Lane<V> ln(p, per_row);
    const int T = p.T, N = p.N, B = p.B, b = ln.b, n0 = ln.n0;
    const size_t plane = (size_t)B * N, at = (size_t)b * N + n0;
    const int ts = blockIdx.y * range, te = min(ts + range, T);
    Walk<S, V> zp(p.z.data, p.z.s0, p.z.s1, b, ln.b0, n0), fp(p.f.data, p.f.s0, p.f.s1, b, ln.b0, n0),
        yp(p.h.data, p.h.s0, p.h.s1, b, ln.b0, n0);
    Walk<uint8_t, V> sp(p.starts, B, 1, b, ln.b0, 0);
    const Lane8<V> l8(ln.i, ln.skip, ln.on, N);
    Walk8<V> z8(p.z8, B, N, b, ln.b0, ln.group, l8), f8(p.f8, B, N, b, ln.b0, ln.group, l8);
    const int len = MASK ? row_length(p, b) : T;
    float bias[V], h[V];
    DELREC_COLS(j) {
        bias[j] = p.bias ? p.bias[n0 + j] * kLog2e : 0.0f;
        h[j] = p.h0 ? p.h0[at + j] : 0.0f;
    }
    maps.fill_missing(w, nw, lane);
    if (blockIdx.y) enter_range<V, MASK>(maps, p.ws, plane, at, 0, 1, blockIdx.y, w, nw, lane, h);

    int buf = 0;
    for (int tb = ts; tb < te; tb += nw * kSteps, buf ^= 1) {
        const int t0 = tb + w * kSteps;
        if (p.states && w == 0 && ln.on) vstore<float, V>(p.states + (size_t)(tb / kBlk) * plane + at, h);
        Vec<S, V> z[kSteps], f[kSteps];
        float m[kSteps][V], A[V], L[V], g[V];
        bool fresh[kSteps];
        DELREC_COLS(j) A[j] = 1.0f, L[j] = g[j] = 0.0f;
        const bool any = MASK ? __any(t0 < len) : t0 < len, part = MASK ? !__all(t0 + kSteps <= len) : t0 + kSteps > len;
        if (!MASK || any) {
            zp.seek(t0), fp.seek(t0);
            if (MASK) sp.seek(t0);
            auto load = [&](auto full) {
                fp.start(), zp.start();
                if (MASK) sp.start();
                DELREC_STEPS(s) {
                    fresh[s] = false;
                    if (decltype(full)::value || t0 + s < T) {
                        f[s] = fp.load(), z[s] = zp.load();
                        fresh[s] = MASK && p.starts && sp.template value<uint8_t>();
                        fp.next(), zp.next();
                        if (MASK) sp.next();
                    }
                }
            };
            t0 + kSteps <= T ? load(std::true_type()) : load(std::false_type());
            if (part) DELREC_STEPS(s)
                if (t0 + s >= len) blank(z[s]), fresh[s] = false;
            DELREC_STEPS(s) {
                gate<V>(f[s], bias, t0 + s >= len, m[s]);
                step_forward<V, MASK>(m[s], z[s], fresh[s], t0 + s >= len, A, L);
            }
        }
        maps.put(buf, w, lane, A, L);
        if (PACK && any) {
            z8.seek(t0), f8.seek(t0);
            z8.start(), f8.start();
            DELREC_STEPS(s) {
                if (t0 + s < T) {
                    float v[V];
                    DELREC_COLS(j) v[j] = z[s].get(j);
                    z8.store(v, ln.first);
                    DELREC_COLS(j) v[j] = f[s].get(j);
                    f8.store(v, ln.first);
                    z8.next(), f8.next();
                }
            }
        }
        barrier_lds();
        compose<V, MASK, 1>(maps, buf, w, lane, h, g);
        if (MASK && !any) DELREC_STEPS(s) {
            blank(z[s]);
            DELREC_COLS(j) m[s][j] = 0.0f;
            fresh[s] = false;
        }
        yp.seek(t0), yp.start();
        DELREC_STEPS(s) {
            float y[V];
            DELREC_COLS(j) {
                const float from = MASK && fresh[s] ? 0.0f : g[j];
                y[j] = g[j] = gate_step(m[s][j], from - z[s].get(j), from, z[s].get(j));
            }
            if (MASK && part && t0 + s >= len) DELREC_COLS(j) y[j] = 0.0f;
            if (t0 + s < T && ln.on) yp.store(y);
            yp.next();
        }
    }
    if (w == 0 && ln.on && te == T) vstore<float, V>(p.h_last + at, h);
}

// A range's map into p.ws, each wave a run of consecutive steps on its own, composed at the end.
// BWD: the reverse map, from f and dh. PACK: f from its 8 bits.
template <class S, int V, bool MASK, bool PACK, bool BWD>
__global__ void __launch_bounds__(512, 4) gated_range_kernel(GatedScan p, int per_row, int range) {
    __shared__ Maps<V> maps;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), nw = blockDim.x >> 6;
    const Lane<V> ln(p, per_row);
    const int T = p.T, N = p.N, B = p.B, b = ln.b, n0 = ln.n0;
    const size_t plane = (size_t)B * N, at = (size_t)b * N + n0;
    const int y = blockIdx.y + (BWD ? 1 : 0);          // the last range forward, the first backward lead nowhere
    const int run = range / nw, ts = y * range + w * run;
    const delrec_rows& x = BWD ? p.dh : p.z;
    Walk<S, V> fp(p.f.data, p.f.s0, p.f.s1, b, ln.b0, n0), xp(x.data, x.s0, x.s1, b, ln.b0, n0);
    Walk<uint8_t, V> sp(p.starts, B, 1, b, ln.b0, 0);
    const Lane8<V> l8(ln.i, ln.skip, ln.on, N);
    Walk8<V> fp8(p.f8, B, N, b, ln.b0, ln.group, l8);
    const int len = MASK ? row_length(p, b) : T;
    float bias[V], A[V], L[V];
    DELREC_COLS(j) {
        bias[j] = p.bias ? p.bias[n0 + j] * kLog2e : 0.0f;
        A[j] = 1.0f;
        L[j] = 0.0f;
    }
    for (int c = 0; c < run / kSteps; ++c) {
        const int t0 = ts + (BWD ? run / kSteps - 1 - c : c) * kSteps;
        typename std::conditional<PACK, Vec8<V>, Vec<S, V>>::type f[kSteps];
        Vec<S, V> v[kSteps];
        bool fresh[kSteps];
        if (MASK ? !__any(t0 < len) : t0 >= len) continue;
        const bool part = MASK ? !__all(t0 + kSteps <= len) : t0 + kSteps > len;
        if constexpr (PACK) fp8.seek(t0);
        else fp.seek(t0);
        xp.seek(t0);
        if (MASK) sp.seek(t0);
        auto load = [&](auto full) {
            if constexpr (PACK) fp8.start();
            else fp.start();
            xp.start();
            if (MASK) sp.start();
            DELREC_STEPS(s) {
                fresh[s] = false;
                if (decltype(full)::value || t0 + s < T) {
                    if constexpr (PACK) f[s] = fp8.load(), fp8.next();
                    else f[s] = fp.load(), fp.next();
                    v[s] = xp.load(), xp.next();
                    fresh[s] = MASK && p.starts && sp.template value<uint8_t>();
                    if (MASK) sp.next();
                }
            }
        };
        t0 + kSteps <= T ? load(std::true_type()) : load(std::false_type());
        if constexpr (PACK) DELREC_STEPS(s) fp8.own(f[s]);
        if (part) DELREC_STEPS(s)
            if (t0 + s >= len) blank(v[s]), fresh[s] = false;
        DELREC_STEPS(q) {
            const int s = BWD ? kSteps - 1 - q : q;
            float m[V];
            gate<V>(f[s], bias, t0 + s >= len, m);
            if constexpr (BWD) step_backward<V, MASK>(m, v[s], fresh[s], t0 + s >= len, L), step_leak<V, MASK>(m, fresh[s], A);
            else step_forward<V, MASK>(m, v[s], fresh[s], t0 + s >= len, A, L);
        }
    }
    maps.put(0, w, lane, A, L);
    barrier_lds();
    if (w || !ln.on) return;
    DELREC_COLS(j) A[j] = 1.0f, L[j] = 0.0f;
    for (int c = 0; c < nw; ++c) {
        const int q = BWD ? nw - 1 - c : c;
        const auto e = maps.template run<MASK>(0, q, lane, L);
        DELREC_COLS(j) A[j] = product<MASK>(A[j], e[j]);
    }
    float* a = p.ws + (size_t)y * 2 * plane + at;
    vstore_own<float, V>(a, A, PACK ? ln.skip : 0);
    vstore_own<float, V>(a + plane, L, PACK ? ln.skip : 0);
}

// PACK: z and f from their 8 bits.
template <class S, int V, bool MASK, bool PACK>
__global__ void __launch_bounds__(512, 4) gated_bwd_kernel(GatedScan p, int per_row, int range, float* dbpart) {
    __shared__ Maps<V> fmap, rmap;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), nw = blockDim.x >> 6;
    const Lane<V> ln(p, per_row);
    const int T = p.T, N = p.N, B = p.B, b = ln.b, n0 = ln.n0;
    const size_t plane = (size_t)B * N, at = (size_t)b * N + n0;
    const int ts = blockIdx.y * range, te = min(ts + range, T);
    const int own = PACK ? ln.skip : 0;
    Walk<S, V> zp(p.z.data, p.z.s0, p.z.s1, b, ln.b0, n0), fp(p.f.data, p.f.s0, p.f.s1, b, ln.b0, n0),
        dhp(p.dh.data, p.dh.s0, p.dh.s1, b, ln.b0, n0), dzp(p.dz.data, p.dz.s0, p.dz.s1, b, ln.b0, n0),
        dfp(p.df.data, p.df.s0, p.df.s1, b, ln.b0, n0);
    Walk<uint8_t, V> sp(p.starts, B, 1, b, ln.b0, 0);
    const Lane8<V> l8(ln.i, ln.skip, ln.on, N);
    Walk8<V> z8(p.z8, B, N, b, ln.b0, ln.group, l8), f8(p.f8, B, N, b, ln.b0, ln.group, l8);
    const int len = MASK ? row_length(p, b) : T;
    float bias[V], c[V], db[V];
    DELREC_COLS(j) {
        bias[j] = p.bias ? p.bias[n0 + j] * kLog2e : 0.0f;
        c[j] = p.dlast ? p.dlast[at + j] : 0.0f;
        db[j] = 0.0f;
    }
    fmap.fill_missing(w, nw, lane);
    rmap.fill_missing(w, nw, lane);
    const int last = gridDim.y - 1;
    if ((int)blockIdx.y < last)
        enter_range<V, MASK>(rmap, p.ws, plane, at, last, -1, last - blockIdx.y, w, nw, lane, c);

    int buf = 0;
    for (int tb = ts + (te - 1 - ts) / (nw * kSteps) * (nw * kSteps); tb >= ts; tb -= nw * kSteps, buf ^= 1) {
        const int t0 = tb + w * kSteps;
        float m[kSteps][V], d[kSteps][V], h[V], g[V], mine[V];
        Vec<S, V> dh[kSteps];
        typename std::conditional<PACK, Vec8<V>, Vec<S, V>>::type z[kSteps];
        bool fresh[kSteps];
        const auto st = vload<float, V>(p.states + (size_t)(tb / kBlk) * plane + at);
        DELREC_COLS(j) h[j] = st.get(j), g[j] = mine[j] = 0.0f;
        const bool any = MASK ? __any(t0 < len) : t0 < len, part = MASK ? !__all(t0 + kSteps <= len) : t0 + kSteps > len;
        {
            float A[V], L[V];
            typename std::conditional<PACK, Vec8<V>, Vec<S, V>>::type f[kSteps];
            if (!MASK || any) {
                if constexpr (PACK) z8.seek(t0), f8.seek(t0);
                else zp.seek(t0), fp.seek(t0);
                dhp.seek(t0);
                if (MASK) sp.seek(t0);
                auto load = [&](auto full) {
                    if constexpr (PACK) f8.start(), z8.start();
                    else fp.start(), zp.start();
                    dhp.start();
                    if (MASK) sp.start();
                    DELREC_STEPS(s) {
                        fresh[s] = false;
                        if (decltype(full)::value || t0 + s < T) {
                            if constexpr (PACK) f[s] = f8.load(), z[s] = z8.load(), f8.next(), z8.next();
                            else f[s] = fp.load(), z[s] = zp.load(), fp.next(), zp.next();
                            dh[s] = dhp.load(), dhp.next();
                            fresh[s] = MASK && p.starts && sp.template value<uint8_t>();
                            if (MASK) sp.next();
                        }
                    }
                };
                t0 + kSteps <= T ? load(std::true_type()) : load(std::false_type());
                if constexpr (PACK) DELREC_STEPS(s) f8.own(f[s]), z8.own(z[s]);
                if (part) DELREC_STEPS(s)
                    if (t0 + s >= len) blank(z[s]), blank(dh[s]), fresh[s] = false;
            }
            DELREC_COLS(j) A[j] = 1.0f, L[j] = 0.0f;
            if (!MASK || any) DELREC_STEPS(s) {
                gate<V>(f[s], bias, t0 + s >= len, m[s]);
                step_forward<V, MASK>(m[s], z[s], fresh[s], t0 + s >= len, A, L);
            }
            fmap.put(buf, w, lane, A, L);
            DELREC_COLS(j) L[j] = 0.0f;
            if (!MASK || any) DELREC_STEPS_BACK(s) step_backward<V, MASK>(m[s], dh[s], fresh[s], t0 + s >= len, L);
            rmap.put(buf, w, lane, A, L);
        }
        barrier_lds();
        compose<V, MASK, -1>(rmap, buf, w, lane, c, g);
        // (one exchange's reads at a time: both at once are 64 registers)
        __builtin_amdgcn_sched_barrier(0);
        compose<V, MASK, 1>(fmap, buf, w, lane, h, mine);
        float blk[V];
        DELREC_COLS(j) blk[j] = 0.0f;
        if (MASK && !any) DELREC_STEPS(s) {
            blank(dh[s]), blank(z[s]);
            DELREC_COLS(j) m[s][j] = 0.0f;
            fresh[s] = false;
        }
        // d_t = h_{t-1} - z_t
        DELREC_STEPS(s) DELREC_COLS(j) {
            const float from = MASK && fresh[s] ? 0.0f : mine[j];
            d[s][j] = from - z[s].get(j);
            mine[j] = gate_step(m[s][j], d[s][j], from, z[s].get(j));
        }
        // (outside a row the gradients are zeros and the carry stays, also an infinite one)
        dzp.seek(t0 + kSteps - 1), dfp.seek(t0 + kSteps - 1);
        dzp.start(), dfp.start();
        DELREC_STEPS_BACK(s) if (MASK || t0 + s < T) {
            float oz[V], of[V];
            DELREC_COLS(j) {
                // the smaller of k lam and a lam, the larger, and k a lam
                const bool off = MASK && t0 + s >= len, leak = leak_kept(m[s][j]);
                const float lam = dh[s].get(j) + g[j], few = fabsf(m[s][j]) * lam, most = lam - few;
                oz[j] = off ? 0.0f : leak ? most : few;
                of[j] = off ? 0.0f : fmaf(-fabsf(m[s][j]), few, few) * d[s][j];
                g[j] = MASK && fresh[s] ? 0.0f : off ? lam : leak ? few : most;
                blk[j] += of[j];
            }
            if (t0 + s < T && ln.on) dzp.store(oz, own), dfp.store(of, own);
            dzp.prev(), dfp.prev();
        } else {
            dzp.prev(), dfp.prev();
        }
        // the bias sum in two levels, within a block and over blocks: one long chain of 32-bit
        // additions lost a digit at T = 16384
        DELREC_COLS(j) db[j] += blk[j];
    }
    if (w == 0 && ln.on && ts == 0 && p.dh0) vstore_own<float, V>(p.dh0 + at, c, own);
    if (!dbpart) return;
    __syncthreads();
    rmap.put(0, w, lane, db, db);
    __syncthreads();
    if (w || !ln.on) return;
    for (int q = 1; q < nw; ++q)
        DELREC_COLS(j) db[j] += rmap.m[0][q][lane][j];
    vstore_own<float, V>(dbpart + (size_t)blockIdx.y * plane + at, db, own);
}

namespace {

struct Plan {
    int V, per_row, groups, waves, range, ranges;
};

// Two columns a lane. Four have the same bytes under way in half the workgroups, and the backward's
// registers (gates, z, dh of eight steps) do not fit 128: forward and backward of T1024 B64 N2048 with
// 8 bits take 299 + 382 us with four, 312 + 291 with two, 410 + 368 with one; of T250 B128 N512 30 +
// 64, 23 + 34, 28 + 41. One for rows of one column and for offsets past 32 bits.
//
// Time over the grid where the channels give less than a workgroup a CU: each range's inputs are
// then read twice. T1000 N512 bf16, a training pass's kernels whole and in ranges: B 32 (128
// workgroups) 122 and 89 us, B 48 (192) 132 and 134, B 64 (256) 143 and 147. As many ranges as make
// one round of two workgroups a CU (T16384 B2 N700 fp32: 255 us with 22 ranges, 244 with 43, 249
// with 64). With masks twice that, since padded ranges end early (T1000 B50 N333: 188 us with 3
// ranges, 156 with 4, 141 with 6). From five blocks on, a block a range at the least: B20 N333 bf16
// whole and in ranges 27 and 29 us at T 128, 41 and 34 (and two more launches) at T 256, 48 and 37
// at T 320.
Plan gated_plan(int T, int B, int N, bool pack, bool wide, bool mask) {
    Plan q;
    q.V = N >= 2 && !wide ? 2 : 1;
    q.per_row = pack ? (N + kGroup8 - 1) / kGroup8 * (kGroup8 / q.V) : (N + q.V - 1) / q.V;
    q.groups = (int)(((long long)B * q.per_row + 63) / 64);
    q.waves = T >= kBlk ? kWaves : (T + kSteps - 1) / kSteps;
    const int blocks = (T + kBlk - 1) / kBlk;
    int want = q.groups >= 256 || blocks < 5 ? 1 : (mask ? 1024 : 512) / q.groups;
    want = std::max(1, std::min({want, 128, blocks}));
    const int per = (blocks + want - 1) / want;
    q.range = per * kBlk;
    q.ranges = (blocks + per - 1) / per;
    return q;
}

size_t map_floats(const Plan& q, int B, int N) { return q.ranges > 1 ? (size_t)q.ranges * 2 * B * N : 0; }

template <class S, int V, bool MASK, bool PACK>
void run_gated(const GatedScan& a, const Plan& q, bool fwd, hipStream_t stream) {
    GatedScan p = a;
    float* part = p.db && !fwd ? p.ws + map_floats(q, p.B, p.N) : nullptr;
    const dim3 block(64 * q.waves);
    for (long long first = 0; first < q.groups; first += kMostBlocks) {
        p.first = (int)first;
        const int groups = std::min(q.groups - p.first, kMostBlocks);
        const dim3 grid(groups, q.ranges), inner(groups, q.ranges - 1);
        if (fwd) {
            if (q.ranges > 1)
                hipLaunchKernelGGL((gated_range_kernel<S, V, MASK, false, false>), inner, block, 0, stream, p, q.per_row, q.range);
            hipLaunchKernelGGL((gated_fwd_kernel<S, V, MASK, PACK>), grid, block, 0, stream, p, q.per_row, q.range);
        } else {
            if (q.ranges > 1)
                hipLaunchKernelGGL((gated_range_kernel<S, V, MASK, PACK, true>), inner, block, 0, stream, p, q.per_row, q.range);
            hipLaunchKernelGGL((gated_bwd_kernel<S, V, MASK, PACK>), grid, block, 0, stream, p, q.per_row, q.range, part);
        }
    }
    if (part) launch_column_sums(part, (unsigned)q.ranges * p.B, p.N, p.N, p.db, nullptr, nullptr, stream);
}

template <class S, int V>
void run_gated_m(const GatedScan& p, const Plan& q, bool fwd, hipStream_t stream) {
    const bool mask = p.starts || p.lengths;
    if (p.z8.q) mask ? run_gated<S, V, true, true>(p, q, fwd, stream) : run_gated<S, V, false, true>(p, q, fwd, stream);
    else mask ? run_gated<S, V, true, false>(p, q, fwd, stream) : run_gated<S, V, false, false>(p, q, fwd, stream);
}

template <class S>
void run_gated_v(const GatedScan& p, const Plan& q, bool fwd, hipStream_t stream) {
    if (q.V == 2) run_gated_m<S, 2>(p, q, fwd, stream);
    else run_gated_m<S, 1>(p, q, fwd, stream);
}

void launch_gated(const GatedScan& p, bool fwd, hipStream_t stream) {
    // the rows that a wave's 64 V channels touch, counted generously, against 32-bit offsets
    bool wide = false;
    for (const delrec_rows* x : {&p.z, &p.f, &p.h, &p.dh, &p.dz, &p.df})
        if (x->data && (x->s1 < 0 || (256 / p.N + 2) * x->s1 + p.N > 0x7fffffffLL / 4)) wide = true;
    const Plan q = gated_plan(p.T, p.B, p.N, p.z8.q != nullptr, wide, p.starts || p.lengths);
    if (p.bf16) run_gated_v<__bf16>(p, q, fwd, stream);
    else run_gated_v<float>(p, q, fwd, stream);
}

}  // namespace

// floats of workspace, for whichever form the strides, the 8 bits and the masks ask for: the
// ranges' maps, and the ranges' bias sums
size_t gated_fwd_ws(int T, int B, int N) {
    size_t n = 0;
    for (int form = 0; form < 8; ++form) n = std::max(n, map_floats(gated_plan(T, B, N, form & 1, form & 2, form & 4), B, N));
    return n;
}
size_t gated_bwd_ws(int T, int B, int N) {
    int ranges = 1;
    for (int form = 0; form < 8; ++form) ranges = std::max(ranges, gated_plan(T, B, N, form & 1, form & 2, form & 4).ranges);
    return gated_fwd_ws(T, B, N) + (size_t)ranges * B * N;
}

void launch_gated_fwd(const GatedScan& p, hipStream_t stream) { launch_gated(p, true, stream); }
void launch_gated_bwd(const GatedScan& p, hipStream_t stream) { launch_gated(p, false, stream); }

}  // namespace delrec
