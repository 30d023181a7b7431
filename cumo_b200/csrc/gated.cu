// Gated running sums along an axis: h[t] = gate[t] * h[t-1] + x[t], and their gradients.
//
// cumsum with a coefficient per step (gate = 1 is cumsum): the state update of a gated linear recurrent layer, n = 1 being
// one new token.  With an initial state h[-1] is that state; without one h[0] = x[0], and gate[0] is not used.  Given
// g = dL/dh, the gradients are
//     dx[t] = dh[t] = g[t] + gate[t+1] * dh[t+1]         (the same recurrence, backwards in time, over the shifted gate)
//     dgate[t] = dh[t] * h[t-1]        dinitial = gate[0] * dh[0]
// so one set of kernels does both: they walk "scan steps" s = 0 .. n-1 over operands whose pointers and steps the host has
// set up (backwards: last element first, negative steps), and the gradient form multiplies by a third operand on the way out.
//
// A stretch of steps maps the state before it to the state after it by h -> A*h + B, with A the product of its gates and B
// its result from a zero state.  Stretches are folded in parallel with these pairs to find the state in front of each;
// every stretch is then walked again, from registers, starting from that state, so that each output is the formula's own
// sequence of rounded steps.  A is a product of many factors in (0, 1) as a rule: for 32-bit elements it and the
// composition are held in 64 bits, where it neither underflows in a way that could be seen in 32 bits nor loses digits.
//
// Three plans, all bound by memory traffic (3 s bytes per element forward, 5 s backward):
//   walk    a thread per run, in order: many runs, or few steps
#include "common.cuh"

namespace cb200 {

// One operand: base address of scan step 0 of run 0, byte step per scan step, byte steps of the outer dimensions.
struct GatedRuns {
    int64_t n;                       // scan steps per run
    int64_t runs;                    // number of runs
    int nd;                          // outer dimensions after merging
    int64_t shape[kMaxDim];
    // operands: 0 u (x or grad), 1 a (gate), 2 out (h or dx), 3 initial, 4 p (h one step earlier), 5 q (dgate), 6 dinitial
    int64_t step[7][kMaxDim];
    int64_t s_u, s_a, s_o, s_p, s_q;
    const char* u;
    const char* a;                   // gate of scan step 0 (never read there unless an initial state enters there)
    char* o;
    const char* init;                // may be null
    const char* p;
    char* q;
    char* dinit;                     // may be null
};

template <typename T, int V> struct alignas(sizeof(T) * V) GVec { T v[V]; };

template <typename T, int V>
__device__ __forceinline__ GVec<T, V> gld(const char* p) {
    if constexpr (sizeof(T) * V == 16) {
        GVec<T, V> r;
        *reinterpret_cast<int4*>(&r) = __ldcs(reinterpret_cast<const int4*>(p));
        return r;
    } else {
        return *reinterpret_cast<const GVec<T, V>*>(p);
    }
}
template <typename T, int V>
__device__ __forceinline__ void gst(char* p, const GVec<T, V>& v) {
    if constexpr (sizeof(T) * V == 16) __stcs(reinterpret_cast<int4*>(p), *reinterpret_cast<const int4*>(&v));
    else *reinterpret_cast<GVec<T, V>*>(p) = v;
}

__device__ __forceinline__ float gfma(float a, float b, float c) { return fmaf(a, b, c); }
__device__ __forceinline__ double gfma(double a, double b, double c) { return fma(a, b, c); }

// ---- walk: a thread per run ------------------------------------------------------------------------------------------
constexpr int kWalkAhead = 8;

template <typename T, bool GRAD>
__global__ void __launch_bounds__(kBlock)
gated_walk_kernel(const GatedRuns g) {
    for (int64_t run = (int64_t)blockIdx.x * kBlock + threadIdx.x; run < g.runs; run += (int64_t)gridDim.x * kBlock) {
        int64_t off[7];
        offsets_of<7>(run, g.nd, g.shape, g.step, off);
        const char* u = g.u + off[0];
        const char* a = g.a + off[1];
        char* o = g.o + off[2];
        const T init = g.init ? *reinterpret_cast<const T*>(g.init + off[3]) : T(0);
        const char* p = GRAD ? g.p + off[4] : nullptr;
        char* q = GRAD ? g.q + off[5] : nullptr;
        const bool enters = !GRAD && g.init;              // a state enters at scan step 0
        T h = enters ? init : T(0);
        for (int64_t s0 = 0; s0 < g.n; s0 += kWalkAhead) {
            T uu[kWalkAhead], aa[kWalkAhead], pp[kWalkAhead];
#pragma unroll
            for (int i = 0; i < kWalkAhead; ++i) {
                const int64_t s = s0 + i;
                if (s >= g.n) break;
                uu[i] = *reinterpret_cast<const T*>(u + s * g.s_u);
                aa[i] = s > 0 || enters ? *reinterpret_cast<const T*>(a + s * g.s_a) : T(0);
                if (GRAD) pp[i] = s + 1 < g.n ? *reinterpret_cast<const T*>(p + s * g.s_p) : init;
            }
#pragma unroll
            for (int i = 0; i < kWalkAhead; ++i) {
                const int64_t s = s0 + i;
                if (s >= g.n) break;
                h = s > 0 || enters ? gfma(aa[i], h, uu[i]) : uu[i];
                *reinterpret_cast<T*>(o + s * g.s_o) = h;
                if (GRAD) *reinterpret_cast<T*>(q + s * g.s_q) = s + 1 < g.n || g.init ? h * pp[i] : T(0);
            }
        }
        if (GRAD && g.dinit) *reinterpret_cast<T*>(g.dinit + off[6]) = *reinterpret_cast<const T*>(a + g.n * g.s_a) * h;
    }
}

template <typename T, bool GRAD>
static int gated_launch(GatedRuns& g) {
    if (g.n == 0 || g.runs == 0) return 0;
    // merge neighbouring outer dimensions that every operand walks evenly; drop extents of 1
    int nd = 0;
    for (int d = 0; d < g.nd; ++d) {
        if (g.shape[d] == 1) continue;
        bool even = nd > 0;
        for (int k = 0; k < 7 && even; ++k) even = g.step[k][nd - 1] == g.step[k][d] * g.shape[d];
        if (even) {
            g.shape[nd - 1] *= g.shape[d];
            for (int k = 0; k < 7; ++k) g.step[k][nd - 1] = g.step[k][d];
        } else {
            g.shape[nd] = g.shape[d];
            for (int k = 0; k < 7; ++k) g.step[k][nd] = g.step[k][d];
            ++nd;
        }
    }
    g.nd = nd;
    const unsigned grid = grid_for((g.runs + kBlock - 1) / kBlock, 8);
    gated_walk_kernel<T, GRAD><<<grid, kBlock, 0, current_stream()>>>(g);
    count_launch();
    return (int)cudaGetLastError();
}

// common part of the two entry points: outer dimensions
static bool gated_outer(GatedRuns& g, int n_outer, const size_t* shape) {
    if (n_outer < 0 || n_outer > kMaxDim) return false;
    g.nd = n_outer;
    g.runs = 1;
    for (int d = 0; d < n_outer; ++d) { g.shape[d] = (int64_t)shape[d]; g.runs *= g.shape[d]; }
    return true;
}

template <typename T>
static int gated_forward(char* x, char* gate, char* initial, char* h, ssize_t s_x, ssize_t s_gate, ssize_t s_h, uint64_t n, int n_outer,
                         const size_t* shape, const ssize_t* x_step, const ssize_t* gate_step, const ssize_t* initial_step, const ssize_t* h_step) {
    CB200_TRACE_LAUNCH();
    GatedRuns g;
    memset(&g, 0, sizeof g);
    if (!gated_outer(g, n_outer, shape)) return (int)cudaErrorInvalidValue;
    g.n = (int64_t)n;
    g.u = x; g.a = gate; g.o = h; g.init = initial;
    g.s_u = s_x; g.s_a = s_gate; g.s_o = s_h;
    for (int d = 0; d < n_outer; ++d) {
        g.step[0][d] = x_step[d]; g.step[1][d] = gate_step[d]; g.step[2][d] = h_step[d];
        if (initial) g.step[3][d] = initial_step[d];
    }
    return gated_launch<T, false>(g);
}

template <typename T>
static int gated_backward(char* grad, char* gate, char* h, char* initial, char* dx, char* dgate, char* dinitial,
                          ssize_t s_grad, ssize_t s_gate, ssize_t s_h, ssize_t s_dx, ssize_t s_dgate, uint64_t n, int n_outer, const size_t* shape,
                          const ssize_t* grad_step, const ssize_t* gate_step, const ssize_t* h_step, const ssize_t* initial_step,
                          const ssize_t* dx_step, const ssize_t* dgate_step, const ssize_t* dinitial_step) {
    CB200_TRACE_LAUNCH();
    GatedRuns g;
    memset(&g, 0, sizeof g);
    if (!gated_outer(g, n_outer, shape) || (dinitial && !initial)) return (int)cudaErrorInvalidValue;
    const int64_t last = (int64_t)n - 1;
    g.n = (int64_t)n;
    g.u = grad + last * s_grad;          g.s_u = -s_grad;
    g.a = gate + (last + 1) * s_gate;    g.s_a = -s_gate;       // scan step s uses the gate of time n - s; step 0 uses none
    g.o = dx + last * s_dx;              g.s_o = -s_dx;
    g.p = h + (last - 1) * s_h;          g.s_p = -s_h;          // ... and the state of time n - 2 - s; the last step the initial state
    g.q = dgate + last * s_dgate;        g.s_q = -s_dgate;
    g.init = initial; g.dinit = dinitial;
    for (int d = 0; d < n_outer; ++d) {
        g.step[0][d] = grad_step[d]; g.step[1][d] = gate_step[d]; g.step[2][d] = dx_step[d]; g.step[4][d] = h_step[d]; g.step[5][d] = dgate_step[d];
        if (initial) g.step[3][d] = initial_step[d];
        if (dinitial) g.step[6][d] = dinitial_step[d];
    }
    return gated_launch<T, true>(g);
}

}  // namespace cb200

#define CB200_DEF_GATED(NAME, T)                                                                                                     \
    extern "C" int cb200_##NAME##_gated_cumsum_runs_kernel_launch(                                                                   \
        char* x, char* gate, char* initial, char* h, ssize_t s_x, ssize_t s_gate, ssize_t s_h, uint64_t n, int n_outer,              \
        const size_t* shape, const ssize_t* x_step, const ssize_t* gate_step, const ssize_t* initial_step, const ssize_t* h_step) {  \
        return cb200::gated_forward<T>(x, gate, initial, h, s_x, s_gate, s_h, n, n_outer, shape, x_step, gate_step, initial_step, h_step); \
    }                                                                                                                                \
    extern "C" int cb200_##NAME##_gated_cumsum_grad_runs_kernel_launch(                                                              \
        char* grad, char* gate, char* h, char* initial, char* dx, char* dgate, char* dinitial, ssize_t s_grad, ssize_t s_gate,       \
        ssize_t s_h, ssize_t s_dx, ssize_t s_dgate, uint64_t n, int n_outer, const size_t* shape, const ssize_t* grad_step,          \
        const ssize_t* gate_step, const ssize_t* h_step, const ssize_t* initial_step, const ssize_t* dx_step,                        \
        const ssize_t* dgate_step, const ssize_t* dinitial_step) {                                                                   \
        return cb200::gated_backward<T>(grad, gate, h, initial, dx, dgate, dinitial, s_grad, s_gate, s_h, s_dx, s_dgate, n, n_outer, \
                                        shape, grad_step, gate_step, h_step, initial_step, dx_step, dgate_step, dinitial_step);      \
    }
CB200_DEF_GATED(sfloat, float)
CB200_DEF_GATED(dfloat, double)
