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
// sequence of rounded steps.  Pairs are composed in 64 bits.  Within a stretch of up to sixteen steps A and B are folded in the
// element type (a rounding per step, as the walk itself makes), A in 64 bits where the runs are contiguous; for 32-bit elements
// they are folded again in 64 bits where a product of gates comes near the ends of the range, or B leaves it: the state of the run
// may be in range all the same.  (64-bit elements have nothing wider to go to: sums from zero have to stay in their range.)
//
// Three plans, all bound by memory traffic (3 s bytes per element forward, 5 s backward):
//   walk    a thread per run (or per 16-byte group of neighbouring runs), in order: many runs, or few steps
//   strip   runs side by side in memory, too few of them to fill the GPU with a thread each: a CTA owns 32 lanes' runs, its
//           warps take stretches of eight steps, and up to eight CTAs of a cluster take turns along the run, handing their
//           stretches' (A, B) to one another through distributed shared memory
//   rows    runs that are contiguous along the axis themselves: a warp, a CTA or a cluster per run, tiles turned through
//           shared memory so that global accesses run along the axis while a thread owns consecutive steps
#include <cooperative_groups.h>

#include "split_product.cuh"
#include "tc_common.cuh"

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
    int* gave_up;                    // set when a bounded wait ran out
    int head;                        // lanes whose gate gradients are added up before they leave (0: none are)
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

// Gate modes of the packet kernels: the V runs of a lane have V neighbouring gates, or share one.
enum GateMode { kGateOwn = 0, kGateShared = 1 };

// The gradient of a gate that `head` neighbouring lanes of V runs share, in the first lane of each such group.
template <typename T, int V>
__device__ __forceinline__ T shared_sum(const GVec<T, V>& d, int head) {
    T s = d.v[0];
#pragma unroll
    for (int v = 1; v < V; ++v) s += d.v[v];
    for (int w = head >> 1; w > 0; w >>= 1) s += __shfl_xor_sync(0xffffffffu, s, w);
    return s;
}

// ---- walk: a thread per V neighbouring runs -----------------------------------------------------------------------------
// Each thread keeps U steps of loads in flight; consecutive threads own consecutive runs, so that a step is one coalesced
// access where the runs lie side by side.  Bound by memory once there are some 75000 threads.
template <typename T, int V, int GM, bool GRAD>
__global__ void __launch_bounds__(kBlock)
gated_walk_kernel(const GatedRuns g) {
    constexpr int U = V * sizeof(T) == 16 ? 4 : 8;
    constexpr int GV = GM == kGateShared ? 1 : V;
    const int64_t groups = g.runs / V, padded = (groups + 31) / 32 * 32;          // whole warps: they add up heads together
    for (int64_t group = (int64_t)blockIdx.x * kBlock + threadIdx.x; group < padded; group += (int64_t)gridDim.x * kBlock) {
        const bool live = group < groups;
        int64_t off[7];
        offsets_of<7>(live ? group * V : 0, g.nd, g.shape, g.step, off);
        const char* u = g.u + off[0];
        const char* a = g.a + off[1];
        char* o = g.o + off[2];
        const char* p = GRAD ? g.p + off[4] : nullptr;
        char* q = GRAD ? g.q + off[5] : nullptr;
        const int64_t i_step = g.nd > 0 ? g.step[3][g.nd - 1] : 0, d_step = g.nd > 0 ? g.step[6][g.nd - 1] : 0;
        T init[V], h[V];
#pragma unroll
        for (int v = 0; v < V; ++v) init[v] = g.init ? *reinterpret_cast<const T*>(g.init + off[3] + v * i_step) : T(0);
        const bool enters = !GRAD && g.init;              // a state enters at scan step 0
#pragma unroll
        for (int v = 0; v < V; ++v) h[v] = enters ? init[v] : T(0);
        for (int64_t s0 = 0; s0 < g.n; s0 += U) {
            GVec<T, V> uu[U], pp[U];
            GVec<T, GV> aa[U];
#pragma unroll
            for (int i = 0; i < U; ++i) {
                const int64_t s = s0 + i;
                if (s >= g.n) break;
                uu[i] = gld<T, V>(u + s * g.s_u);
                if (s > 0 || enters) aa[i] = gld<T, GV>(a + s * g.s_a);
                if (GRAD && s + 1 < g.n) pp[i] = gld<T, V>(p + s * g.s_p);
            }
#pragma unroll
            for (int i = 0; i < U; ++i) {
                const int64_t s = s0 + i;
                if (s >= g.n) break;
                const bool first = !(s > 0 || enters), last = s + 1 >= g.n;
                GVec<T, V> out, dg;
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    h[v] = first ? uu[i].v[v] : gfma(aa[i].v[GM == kGateShared ? 0 : v], h[v], uu[i].v[v]);
                    out.v[v] = h[v];
                    if (GRAD) dg.v[v] = !last ? h[v] * pp[i].v[v] : g.init ? h[v] * init[v] : T(0);
                }
                if (live) gst<T, V>(o + s * g.s_o, out);
                if (GRAD) {
                    if (GM == kGateShared && g.head) {
                        const T sum = shared_sum(dg, g.head);
                        if (live && (threadIdx.x & (g.head - 1)) == 0) *reinterpret_cast<T*>(q + s * g.s_q) = sum;
                    } else if (live) {
                        gst<T, V>(q + s * g.s_q, dg);
                    }
                }
            }
        }
        if (GRAD && g.dinit && live) {
            const GVec<T, GV> a0 = gld<T, GV>(a + g.n * g.s_a);
#pragma unroll
            for (int v = 0; v < V; ++v) *reinterpret_cast<T*>(g.dinit + off[6] + v * d_step) = a0.v[GM == kGateShared ? 0 : v] * h[v];
        }
    }
}

// ---- composing stretches --------------------------------------------------------------------------------------------
// The state behind a stretch, A * h + B.  Pairs are held in 64 bits and rounded once, into the state they lead to.
__device__ __forceinline__ double compose(double A, double B, double h) { return fma(A, h, B); }

// A product of finite gates stays finite and a product of non-zero gates stays non-zero: where the recurrence would carry 0
// past growing gates, or an infinity past shrinking ones, so does the pair.
__device__ __forceinline__ double gates_times(double x, double y) {
    double r = x * y;
    const int e = __double2hiint(r) & 0x7ff00000;                // 0 or subnormal; infinite or NaN: look closer
    if (e == 0 || e == 0x7ff00000) {
        if (isinf(r) && !isinf(x) && !isinf(y)) r = copysign(1.7976931348623157e308, r);
        if (r == 0.0 && x != 0.0 && y != 0.0) r = copysign(4.9406564584124654e-324, r);
    }
    return r;
}

// ---- strip: 32 lanes x V runs, time cut over warps and over the CTAs of a cluster ----------------------------------------
// A round is kStripWarps x L steps of each CTA.  Every warp loads its L steps and folds them from a zero state; warp v then
// folds the eight stretches of the lanes' run v, stores the CTA's pair into every CTA of the cluster (asynchronous stores that
// count themselves in at the receiver's mbarrier: a cluster barrier would also wait for the outputs' way to memory), and leaves
// each warp the state in front of its stretch.  The wait for the pairs is bounded.  Each thread's next steps are on their way
// (asynchronous copies into slots of shared memory that only it reads) while all this happens, and two CTAs per SM cover each
// other's exchanges.  1 x 50000 x 2048 SFloat: 287 us, 4.3 TB/s; 64 x 512 x 2048 (no cluster) 5.1 TB/s.  Time is cut over one cluster
// and no further: with few channels most SMs idle (1 x 50000 x 512 1.6 TB/s, 1 x 400000 x 64 0.23).
constexpr int kStripWarps = 8;

template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t dst, const char* src) {
    if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(BYTES) : "memory");
}

template <typename T, int V, int L, int GM, bool GRAD>
constexpr size_t strip_bytes() { return (size_t)kBlock * L * ((GRAD ? 2 : 1) * V + (GM == kGateShared ? 1 : V)) * sizeof(T); }

template <typename T, int V, int L, int GM, bool GRAD>
__global__ void __launch_bounds__(kBlock, 2)
gated_strip_kernel(const GatedRuns g, int cluster_size) {
    namespace cg = cooperative_groups;
    constexpr int W = kStripWarps;
    constexpr int GV = GM == kGateShared ? 1 : V;
    __shared__ double warp_A[W][GV][32];
    __shared__ double warp_B[W][V][32];               // a stretch's B; then the state in front of it
    extern __shared__ __align__(16) char slots[];
    using Pairs = double2[8][V][32];                  // (A, B) of every CTA of the cluster, two rounds' worth, behind the slots
    Pairs* pairs = reinterpret_cast<Pairs*>(slots + strip_bytes<T, V, L, GM, GRAD>());
    __shared__ __align__(8) uint64_t arrived[2];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    cg::cluster_group cluster = cg::this_cluster();
    const int rank = cluster_size > 1 ? (int)cluster.block_rank() : 0;
    const int64_t group = (int64_t)(blockIdx.x / cluster_size) * 32 + lane;
    const bool live = group < g.runs / V;
    int64_t off[7];
    offsets_of<7>(live ? group * V : 0, g.nd, g.shape, g.step, off);
    const char* u = g.u + off[0];
    const char* a = g.a + off[1];
    char* o = g.o + off[2];
    const char* p = GRAD ? g.p + off[4] : nullptr;
    char* q = GRAD ? g.q + off[5] : nullptr;
    const int64_t i_step = g.nd > 0 ? g.step[3][g.nd - 1] : 0, d_step = g.nd > 0 ? g.step[6][g.nd - 1] : 0;
    const bool enters = !GRAD && g.init;
    bool gave_up = false;
    double H = 0.0;                                   // warp v < V: the state of run v in front of this round (the same in every CTA)
    if (enters && warp < V) H = (double)*reinterpret_cast<const T*>(g.init + off[3] + warp * i_step);
    const int64_t per_round = (int64_t)cluster_size * W * L;
    const int64_t rounds = (g.n + per_round - 1) / per_round;
    // slots [step][thread] of u, then p, then the gate
    const GVec<T, V>* mine_u = reinterpret_cast<const GVec<T, V>*>(slots) + threadIdx.x;
    const GVec<T, V>* mine_p = mine_u + L * kBlock;
    const GVec<T, GV>* mine_a = reinterpret_cast<const GVec<T, GV>*>(slots + (size_t)kBlock * L * (GRAD ? 2 : 1) * sizeof(GVec<T, V>)) + threadIdx.x;
    const uint32_t at_u = (uint32_t)__cvta_generic_to_shared(mine_u), at_p = (uint32_t)__cvta_generic_to_shared(mine_p), at_a = (uint32_t)__cvta_generic_to_shared(mine_a);
    // Stretches inside the run take the short form of each loop: no step of theirs is the first, the last or missing.
    auto inside = [&](int64_t s0) { return (s0 > 0 || enters) && s0 + L < g.n; };
    auto fetch = [&](int64_t s0) {
        const char* ul = u + s0 * g.s_u;
        const char* al = a + s0 * g.s_a;
        const char* pl = GRAD ? p + s0 * g.s_p : nullptr;
        if (inside(s0)) {
#pragma unroll
            for (int i = 0; i < L; ++i) {
                copy_async<sizeof(T) * V>(at_u + i * kBlock * sizeof(GVec<T, V>), ul);
                copy_async<sizeof(T) * GV>(at_a + i * kBlock * sizeof(GVec<T, GV>), al);
                ul += g.s_u; al += g.s_a;
                if (GRAD) { copy_async<sizeof(T) * V>(at_p + i * kBlock * sizeof(GVec<T, V>), pl); pl += g.s_p; }
            }
        } else {
            const int steps = s0 >= g.n ? 0 : g.n - s0 < L ? (int)(g.n - s0) : L;
#pragma unroll 1
            for (int i = 0; i < steps; ++i) {
                copy_async<sizeof(T) * V>(at_u + i * kBlock * sizeof(GVec<T, V>), ul + i * g.s_u);
                if (s0 + i > 0 || enters) copy_async<sizeof(T) * GV>(at_a + i * kBlock * sizeof(GVec<T, GV>), al + i * g.s_a);
                if (GRAD && s0 + i + 1 < g.n) copy_async<sizeof(T) * V>(at_p + i * kBlock * sizeof(GVec<T, V>), pl + i * g.s_p);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    fetch((int64_t)(rank * W + warp) * L);
    if (cluster_size > 1) {
        if (threadIdx.x == 0) {
            mbar_init(&arrived[0], V);
            mbar_init(&arrived[1], V);
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
        cluster.sync();
    }
    for (int64_t round = 0; round < rounds; ++round) {
        const int64_t s0 = round * per_round + (int64_t)(rank * W + warp) * L;
        GVec<T, V> uu[L], pp[L];
        GVec<T, GV> aa[L];
        const int steps = s0 >= g.n ? 0 : g.n - s0 < L ? (int)(g.n - s0) : L;
        asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
        for (int i = 0; i < L; ++i) {
            uu[i] = mine_u[i * kBlock];
            aa[i] = mine_a[i * kBlock];
            if (GRAD) pp[i] = mine_p[i * kBlock];
        }
        // this warp's stretch from a zero state; the very first step starts from nothing, whatever its gate is
        T A[GV], B[V], least[GV];                                // (least: the smallest the product has been)
#pragma unroll
        for (int x = 0; x < GV; ++x) A[x] = least[x] = T(1);
#pragma unroll
        for (int v = 0; v < V; ++v) B[v] = T(0);
        const bool starts = s0 == 0 && !enters, whole = inside(s0);
        if (whole) {
#pragma unroll
            for (int i = 0; i < L; ++i) {
#pragma unroll
                for (int x = 0; x < GV; ++x) { A[x] *= aa[i].v[x]; least[x] = fmin(least[x], fabs(A[x])); }
#pragma unroll
                for (int v = 0; v < V; ++v) B[v] = i == 0 ? uu[i].v[v] : gfma(aa[i].v[GM == kGateShared ? 0 : v], B[v], uu[i].v[v]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < L; ++i) {
                if (i >= steps) break;
                if (i == 0 && starts) {
#pragma unroll
                    for (int v = 0; v < V; ++v) B[v] = uu[0].v[v];
                    continue;
                }
#pragma unroll
                for (int x = 0; x < GV; ++x) { A[x] *= aa[i].v[x]; least[x] = fmin(least[x], fabs(A[x])); }
#pragma unroll
                for (int v = 0; v < V; ++v) B[v] = i == 0 ? uu[i].v[v] : gfma(aa[i].v[GM == kGateShared ? 0 : v], B[v], uu[i].v[v]);
            }
        }
#pragma unroll
        for (int x = 0; x < GV; ++x) {
            double wide = (double)A[x];
            // (near) the end of what a product of gates holds, now or on the way: once more in 64 bits, with care
            if (!((double)least[x] > 1e-30 && fabs(wide) < 1e30)) {
                wide = 1.0;
#pragma unroll
                for (int i = 0; i < L; ++i)
                    if (i < steps && !(i == 0 && starts)) wide = gates_times(wide, (double)aa[i].v[x]);
            }
            warp_A[warp][x][lane] = starts ? 0.0 : wide;
        }
        T none = T(0);                                           // NaN once a B is not finite
#pragma unroll
        for (int v = 0; v < V; ++v) { warp_B[warp][v][lane] = (double)B[v]; none = gfma(B[v], T(0), none); }
        // what leaves the range from a zero state need not do so from the stretch's own: once more in 64 bits, from the slots
        if (sizeof(T) == 4 && none != T(0)) {
#pragma unroll 1
            for (int v = 0; v < V; ++v) {
                double wide = 0.0;
#pragma unroll 1
                for (int i = 0; i < steps; ++i) {
                    const double step = (double)mine_u[i * kBlock].v[v];
                    wide = i == 0 ? step : fma((double)mine_a[i * kBlock].v[GM == kGateShared ? 0 : v], wide, step);
                }
                warp_B[warp][v][lane] = wide;
            }
        }
        __syncthreads();                                         // (the slots have been read)
        if (round + 1 < rounds) fetch(s0 + per_round);
        const int buf = (int)(round & 1);
        if (warp < V) {
            const int x = GM == kGateShared ? 0 : warp;
            double wa[W], wb[W], before = H;
#pragma unroll
            for (int w = 0; w < W; ++w) { wa[w] = warp_A[w][x][lane]; wb[w] = warp_B[w][warp][lane]; }
            if (cluster_size > 1) {
                double fa = wa[0], fb = wb[0];
#pragma unroll
                for (int w = 1; w < W; ++w) { fb = compose(wa[w], wb[w], fb); fa = gates_times(fa, wa[w]); }
                const uint32_t to = smem_u32(&pairs[buf][rank][warp][lane]), bar = smem_u32(&arrived[buf]);
                if (lane == 0)
                    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"((uint32_t)(cluster_size * 32 * sizeof(double2))) : "memory");
                for (int r = 0; r < cluster_size; ++r) {
                    uint32_t there, bar_there;
                    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(to), "r"(r));
                    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(bar_there) : "r"(bar), "r"(r));
                    asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v2.b64 [%0], {%1, %2}, [%3];"
                                 ::"r"(there), "l"(__double_as_longlong(fa)), "l"(__double_as_longlong(fb)), "r"(bar_there) : "memory");
                }
                const uint32_t parity = (uint32_t)(round >> 1) & 1u;
                bool came = false;
                for (uint32_t spin = 0; spin < kSpinLimit && !came && !gave_up; ++spin) {
                    uint32_t done;
                    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                                 : "=r"(done) : "r"(bar), "r"(parity) : "memory");
                    came = done;
                    if (!came && spin > 64) __nanosleep(32);
                }
                if (!came) gave_up = true;                       // (never seen: a cluster's CTAs run together)
                __syncwarp();
#pragma unroll
                for (int r = 0; r < 8; ++r) {
                    if (r == rank) before = H;
                    if (r < cluster_size) { const double2 ab = pairs[buf][r][warp][lane]; H = compose(ab.x, ab.y, H); }
                }
            }
#pragma unroll
            for (int w = 0; w < W; ++w) {
                warp_B[w][warp][lane] = before;
                before = compose(wa[w], wb[w], before);
            }
            if (cluster_size == 1) H = before;
        }
        __syncthreads();
        T h[V];
#pragma unroll
        for (int v = 0; v < V; ++v) h[v] = (T)warp_B[warp][v][lane];
        // again, from the state in front
        char* ol = o + s0 * g.s_o;
        char* ql = GRAD ? q + s0 * g.s_q : nullptr;
        if (whole) {
#pragma unroll
            for (int i = 0; i < L; ++i) {
                GVec<T, V> out, dg;
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    h[v] = gfma(aa[i].v[GM == kGateShared ? 0 : v], h[v], uu[i].v[v]);
                    out.v[v] = h[v];
                    if (GRAD) dg.v[v] = h[v] * pp[i].v[v];
                }
                if (live) gst<T, V>(ol, out);
                ol += g.s_o;
                if (GRAD) {
                    if (GM == kGateShared && g.head) {
                        const T sum = shared_sum(dg, g.head);
                        if (live && (lane & (g.head - 1)) == 0) *reinterpret_cast<T*>(ql) = sum;
                    } else if (live) {
                        gst<T, V>(ql, dg);
                    }
                    ql += g.s_q;
                }
            }
        } else
#pragma unroll
        for (int i = 0; i < L; ++i) {
            if (i >= steps) break;
            const bool last = s0 + i + 1 >= g.n;
            GVec<T, V> out, dg;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                h[v] = i == 0 && starts ? uu[i].v[v] : gfma(aa[i].v[GM == kGateShared ? 0 : v], h[v], uu[i].v[v]);
                out.v[v] = h[v];
                if (GRAD) {
                    T prior = T(0);
                    if (!last) prior = pp[i].v[v];
                    else if (g.init) prior = *reinterpret_cast<const T*>(g.init + off[3] + v * i_step);
                    dg.v[v] = last && !g.init ? T(0) : h[v] * prior;
                }
            }
            if (live) gst<T, V>(ol + i * g.s_o, out);
            if (GRAD) {
                if (GM == kGateShared && g.head) {
                    const T sum = shared_sum(dg, g.head);
                    if (live && (lane & (g.head - 1)) == 0) *reinterpret_cast<T*>(ql + i * g.s_q) = sum;
                } else if (live) {
                    gst<T, V>(ql + i * g.s_q, dg);
                }
                if (last && g.dinit && live) {
                    const GVec<T, GV> a0 = gld<T, GV>(a + g.n * g.s_a);
#pragma unroll
                    for (int v = 0; v < V; ++v) *reinterpret_cast<T*>(g.dinit + off[6] + v * d_step) = a0.v[GM == kGateShared ? 0 : v] * h[v];
                }
            }
        }
        __syncthreads();                                         // before the next round's pairs go where these states are
    }
    if (gave_up) *reinterpret_cast<volatile int*>(g.gave_up) = 1;
    if (cluster_size > 1) cluster.sync();                        // nobody leaves while a pair may still be on its way
}

// ---- rows: runs contiguous along the axis -----------------------------------------------------------------------------------
// G threads per run (a warp, or the CTA, or the CTAs of a cluster in turns), kRowItems consecutive steps per thread.  A tile
// is copied into shared memory along the axis, padded so that threads reading their own steps hit different banks, and the
// results go back the same way.  2570 x 10000 SFloat: 101 us, 3.0 TB/s, bound by the barriers around each tile.
constexpr int kRowItems = 8;                         // (4 where a warp's run has at most 128 steps)

template <int I>
__device__ __forceinline__ int row_slot(int i) { return i + i / I; }       // one element of padding per thread

// CTAs per SM: barriers are what the tile of a whole CTA waits for, so as many as the registers allow (2570 x 10000 SFloat: 117 us
// with two, 101 with four); warps that each have a run of their own have no barriers and lose by spilling.
template <typename T, int G, bool GRAD> constexpr int rows_per_sm() { return sizeof(T) == 4 && G > 32 ? (GRAD ? 3 : 4) : 2; }

template <typename T, int G, int I, bool GRAD>
__global__ void __launch_bounds__(kBlock, rows_per_sm<T, G, GRAD>())
gated_rows_kernel(const GatedRuns g, int cluster_size) {
    namespace cg = cooperative_groups;
    constexpr int TILE = G * I, SLOTS = TILE + G, PER_CTA = kBlock / G;
    extern __shared__ __align__(16) char smem[];
    __shared__ double warp_A[kWarpsPerBlock], warp_B[kWarpsPerBlock];
    __shared__ double cta_A[2], cta_B[2];
    int buf = 0;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int me = threadIdx.x % G, slot = threadIdx.x / G;
    T* su = reinterpret_cast<T*>(smem) + (size_t)slot * SLOTS * (GRAD ? 3 : 2);
    T* sa = su + SLOTS;
    T* sp = sa + SLOTS;
    cg::cluster_group cluster = cg::this_cluster();
    const int rank = cluster_size > 1 ? (int)cluster.block_rank() : 0;
    const int64_t first = (int64_t)(blockIdx.x / cluster_size) * PER_CTA, stride = (int64_t)(gridDim.x / cluster_size) * PER_CTA;
    const bool enters = !GRAD && g.init;
    const int64_t per_round = (int64_t)cluster_size * TILE, rounds = (g.n + per_round - 1) / per_round;
    auto sync = [&]() { if (G > 32) __syncthreads(); else __syncwarp(); };
    T lu[I], la[I], lp[I];
    // the tile of a run and round, into registers: requested while the tile before it is worked on
    auto fetch = [&](int64_t run, int64_t round) {
        int64_t off[7];
        offsets_of<7>(run, g.nd, g.shape, g.step, off);
        const int64_t s0 = round * per_round + (int64_t)rank * TILE;
        const int count = s0 >= g.n ? 0 : g.n - s0 < TILE ? (int)(g.n - s0) : TILE;
        const char* u = g.u + off[0] + (s0 + me) * g.s_u;
        const char* a = g.a + off[1] + (s0 + me) * g.s_a;
        const char* p = GRAD ? g.p + off[4] + (s0 + me) * g.s_p : nullptr;
#pragma unroll
        for (int i = 0; i < I; ++i) {
            const int e = i * G + me;
            lu[i] = e < count ? ld_one<T>(u + i * G * g.s_u) : T(0);
            la[i] = e < count && (s0 + e > 0 || enters) ? ld_one<T>(a + i * G * g.s_a) : T(1);
            if (GRAD) lp[i] = e < count && s0 + e + 1 < g.n ? ld_one<T>(p + i * G * g.s_p) : T(0);
        }
    };
    if (first + slot < g.runs) fetch(first + slot, 0);
    for (int64_t base = first; base < g.runs; base += stride) {
        const int64_t run = base + slot;
        if (G <= 32 && run >= g.runs) break;                     // (a whole warp leaves; the CTA form has one run per CTA)
        int64_t off[7];
        offsets_of<7>(run, g.nd, g.shape, g.step, off);
        char* o = g.o + off[2];
        char* q = GRAD ? g.q + off[5] : nullptr;
        const T init = g.init ? *reinterpret_cast<const T*>(g.init + off[3]) : T(0);
        double H = enters ? (double)init : 0.0;
        for (int64_t round = 0; round < rounds; ++round) {
            const int64_t s0 = round * per_round + (int64_t)rank * TILE;
            const int count = s0 >= g.n ? 0 : g.n - s0 < TILE ? (int)(g.n - s0) : TILE;
#pragma unroll
            for (int i = 0; i < I; ++i) {
                const int e = row_slot<I>(i * G + me);
                su[e] = lu[i]; sa[e] = la[i];
                if (GRAD) sp[e] = s0 + i * G + me + 1 == g.n ? init : lp[i];
            }
            if (round + 1 < rounds) fetch(run, round + 1);
            else if (run + stride < g.runs) fetch(run + stride, 0);
            sync();
            // this thread's steps from a zero state
            T x[I], c[I];
            const int mine = me * (I + 1);
            double A = 1.0;
            T b = T(0);
#pragma unroll
            for (int i = 0; i < I; ++i) {
                x[i] = su[mine + i]; c[i] = sa[mine + i];
                A *= (double)c[i];
                b = i == 0 ? x[0] : gfma(c[i], b, x[i]);
            }
            if (isinf(A) || A == 0.0) {
                A = 1.0;
#pragma unroll
                for (int i = 0; i < I; ++i) A = gates_times(A, (double)c[i]);
            }
            const bool starts = s0 + me * I == 0 && !enters;     // the first step of all starts from nothing
            if (starts) A = 0.0;
            double B = (double)b;
            if (sizeof(T) == 4 && !(fabs(B) <= 3.4028235e38)) {  // (as in the strips: not from its own state, perhaps)
                B = (double)su[mine];
#pragma unroll 1
                for (int i = 1; i < I; ++i) B = fma((double)sa[mine + i], B, (double)su[mine + i]);
            }
            // pairs of this and all threads before it, within the warp
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const double pa = __shfl_up_sync(0xffffffffu, A, d), pb = __shfl_up_sync(0xffffffffu, B, d);
                if (lane >= d) { B = compose(A, B, pb); A = gates_times(A, pa); }
            }
            double before = H;
            if (G > 32) {
                if (lane == 31) { warp_A[warp] = A; warp_B[warp] = B; }
                __syncthreads();
                if (cluster_size > 1) {
                    if (threadIdx.x == 0) {
                        double fa = warp_A[0], fb = warp_B[0];
#pragma unroll
                        for (int w = 1; w < kWarpsPerBlock; ++w) { fb = compose(warp_A[w], warp_B[w], fb); fa = gates_times(fa, warp_A[w]); }
                        cta_A[buf] = fa; cta_B[buf] = fb;
                    }
                    cluster.sync();
                    for (int r = 0; r < cluster_size; ++r) {
                        if (r == rank) before = H;
                        H = compose(*cluster.map_shared_rank(&cta_A[buf], r), *cluster.map_shared_rank(&cta_B[buf], r), H);
                    }
                    buf ^= 1;                                    // (across runs too: the others may still read this one)
                    for (int w = 0; w < warp; ++w) before = compose(warp_A[w], warp_B[w], before);
                } else {
#pragma unroll
                    for (int w = 0; w < kWarpsPerBlock; ++w) {
                        if (w == warp) before = H;
                        H = compose(warp_A[w], warp_B[w], H);
                    }
                }
            } else {
                H = compose(__shfl_sync(0xffffffffu, A, 31), __shfl_sync(0xffffffffu, B, 31), H);
            }
            const double ea = __shfl_up_sync(0xffffffffu, A, 1), eb = __shfl_up_sync(0xffffffffu, B, 1);
            T h = (T)(lane > 0 ? compose(ea, eb, before) : before);
#pragma unroll
            for (int i = 0; i < I; ++i) {
                h = i == 0 && starts ? x[0] : gfma(c[i], h, x[i]);
                if (GRAD) {
                    const int64_t s = s0 + me * I + i;
                    const bool last = s + 1 == g.n;
                    sa[mine + i] = last && !g.init ? T(0) : h * sp[mine + i];
                    if (last && g.dinit) *reinterpret_cast<T*>(g.dinit + off[6]) = *reinterpret_cast<const T*>(g.a + off[1] + g.n * g.s_a) * h;
                }
                su[mine + i] = h;
            }
            sync();
#pragma unroll
            for (int i = 0; i < I; ++i) {
                const int e = i * G + me;
                if (e < count) {
                    st_one<T>(o + (s0 + e) * g.s_o, su[row_slot<I>(e)]);
                    if (GRAD) st_one<T>(q + (s0 + e) * g.s_q, sa[row_slot<I>(e)]);
                }
            }
            sync();
        }
    }
    if (cluster_size > 1) cluster.sync();
}

// ---- choice of plan -------------------------------------------------------------------------------------------------------
template <typename K>
static int launch_cluster(K kernel, const GatedRuns& g, unsigned ctas, int cluster, size_t smem) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas);
    cfg.blockDim = dim3(kBlock);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = current_stream();
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)cluster; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t rc = cudaLaunchKernelEx(&cfg, kernel, g, cluster);
    if (rc != cudaSuccess) { cudaGetLastError(); return (int)rc; }
    count_launch();
    return 0;
}

// CTAs of a cluster per strip (or row): as many as stay within two per SM, no more than the steps feed.
static int cluster_for(int64_t ctas, int64_t steps, int64_t steps_per_cta) {
    int c = 1;
    while (c < 8 && ctas * c * 2 <= (int64_t)sm_count() * 2 && steps > steps_per_cta * c) c *= 2;
    return c;
}

template <typename T, int V, int L, int GM, bool GRAD>
static int launch_strip(GatedRuns& g) {
    const int64_t strips = (g.runs / V + 31) / 32;
    const int cluster = cluster_for(strips, g.n, L * kStripWarps);
    if (strips * cluster > 0x7fffffff) return (int)cudaErrorInvalidValue;
    if (cluster > 1) {
        if (!gave_up_word(&g.gave_up)) return (int)cudaErrorMemoryAllocation;
    }
    constexpr size_t smem = strip_bytes<T, V, L, GM, GRAD>() + 2 * 8 * V * 32 * sizeof(double2);
    auto kernel = gated_strip_kernel<T, V, L, GM, GRAD>;
    if (smem > 24 * 1024) {
        const cudaError_t rc = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (rc != cudaSuccess) { cudaGetLastError(); return (int)rc; }
    }
    return launch_cluster(kernel, g, (unsigned)(strips * cluster), cluster, smem);
}

// `packet`: runs per 16 bytes that may be taken together (1: element by element)
template <typename T, int GM, bool GRAD>
static int launch_side_by_side(GatedRuns& g, int packet, int64_t shared_runs) {
    constexpr int V = 16 / sizeof(T);
    // gates shared by a whole power-of-two number of lanes: their gradients are added up in the warp
    auto heads = [&](int v) {
        const int64_t lanes = shared_runs / v;
        g.head = GRAD && shared_runs && shared_runs % v == 0 && lanes <= 32 && (lanes & (lanes - 1)) == 0 ? (int)lanes : 0;
        return !shared_runs || g.head;
    };
    if constexpr (GM == kGateOwn) {
        if (packet == 1) {
            if (shared_runs) return (int)cudaErrorNotSupported;
            if (g.runs >= (int64_t)sm_count() * 1024 || g.n <= 16) {
                gated_walk_kernel<T, 1, GM, GRAD><<<grid_for((g.runs + kBlock - 1) / kBlock, 8), kBlock, 0, current_stream()>>>(g);
                count_launch();
                return (int)cudaGetLastError();
            }
            return launch_strip<T, 1, 16, GM, GRAD>(g);
        }
    }
    const int64_t groups = g.runs / V;
    // a thread per group when that alone keeps enough loads in flight (16 bytes x 4 steps x 2 operands each, about 44 KiB per
    // SM wanted), or when there is little to cut
    if (groups >= (int64_t)sm_count() * 512 || g.n <= 16) {
        if (!heads(V)) return (int)cudaErrorNotSupported;
        gated_walk_kernel<T, V, GM, GRAD><<<grid_for((groups + kBlock - 1) / kBlock, 8), kBlock, 0, current_stream()>>>(g);
        count_launch();
        return (int)cudaGetLastError();
    }
    // strips as wide as leaves two CTAs per SM with at most eight to a cluster; the gradients hold a third operand in registers
    // and take half as many steps at a time
    if (sizeof(T) == 8 || (groups + 31) / 32 * 8 >= (int64_t)sm_count() || !heads(V / 2)) {
        if (!heads(V)) return (int)cudaErrorNotSupported;
        return launch_strip<T, V, GRAD ? 4 : 8, GM, GRAD>(g);
    }
    return launch_strip<T, V / 2, GRAD ? 8 : 16, GM, GRAD>(g);
}

template <typename T, int G, int I, bool GRAD>
static int launch_rows_of(const GatedRuns& g, int64_t rows, int cluster) {
    constexpr size_t smem = (size_t)(GRAD ? 3 : 2) * (kBlock * I + kBlock) * sizeof(T);
    auto kernel = gated_rows_kernel<T, G, I, GRAD>;
    if (smem > 48 * 1024 - 512) {
        const cudaError_t rc = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (rc != cudaSuccess) { cudaGetLastError(); return (int)rc; }
    }
    return launch_cluster(kernel, g, (unsigned)(rows * cluster), cluster, smem);
}

template <typename T, bool GRAD>
static int launch_rows(const GatedRuns& g) {
    // a warp per run where there are enough of them or a warp's tile holds most of one
    const unsigned warps = grid_for((g.runs + kWarpsPerBlock - 1) / kWarpsPerBlock, rows_per_sm<T, 32, GRAD>());
    if (g.n <= 128) return launch_rows_of<T, 32, 4, GRAD>(g, warps, 1);
    if (g.n <= 32 * kRowItems * 2 || g.runs >= (int64_t)sm_count() * 32) return launch_rows_of<T, 32, kRowItems, GRAD>(g, warps, 1);
    const int cluster = cluster_for(g.runs, g.n, (int64_t)kBlock * kRowItems);
    const int64_t most = (int64_t)sm_count() * rows_per_sm<T, kBlock, GRAD>();
    return launch_rows_of<T, kBlock, kRowItems, GRAD>(g, g.runs < most ? g.runs : most, cluster);
}

template <typename T, bool GRAD>
static int gated_launch(GatedRuns& g) {
    if (g.n == 0 || g.runs == 0) return 0;
    const int late = product_gave_up();
    if (late) return late;
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
    // Which dimension runs along memory?  Whole packets of neighbouring runs need every per-run operand contiguous and aligned
    // there (the gate may also be one for all of them).
    constexpr int ES = sizeof(T), V = 16 / ES;
    const int in = nd - 1;
    const bool shared_gate = nd > 0 && g.step[1][in] == 0;
    const int64_t shared_runs = GRAD && shared_gate && g.step[5][in] == 0 ? g.shape[in] : 0;
    for (int d = 0; GRAD && d < nd; ++d)
        if (g.step[5][d] == 0 && g.shape[d] > 1 && (d < in || !shared_runs)) return (int)cudaErrorNotSupported;     // a sum over other dimensions
    const bool side = nd > 0 && g.step[0][in] == ES && g.step[2][in] == ES && (!GRAD || (g.step[4][in] == ES && (g.step[5][in] == ES || shared_runs)));
    auto even = [&](const char* p, int k, int64_t s) {
        bool ok = aligned16(p) && mult16(s);
        for (int d = 0; d < in && ok; ++d) ok = mult16(g.step[k][d]);
        return ok;
    };
    if (side && (shared_gate || g.step[1][in] == ES) && g.shape[in] % V == 0 && even(g.u, 0, g.s_u) && even(g.o, 2, g.s_o) &&
        (shared_gate || even(g.a, 1, g.s_a)) && (!GRAD || (even(g.p, 4, g.s_p) && (shared_runs || even(g.q, 5, g.s_q)))))
        return shared_gate ? launch_side_by_side<T, kGateShared, GRAD>(g, V, shared_runs) : launch_side_by_side<T, kGateOwn, GRAD>(g, V, 0);
    const bool along = (g.s_o == ES || g.s_o == -ES) && g.n > 1;
    if (along && !side && g.n > 32) return shared_runs ? (int)cudaErrorNotSupported : launch_rows<T, GRAD>(g);
    return launch_side_by_side<T, kGateOwn, GRAD>(g, 1, shared_runs);
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
