// The linear layer y = act(x . w + bias) + residual and its gradients.
//
// z = x w + b;  y = act(z) + r.  For g = dL/dy: dz = g * act'(z), dx = dz w^T, dw = x^T dz, db = the column sums of dz (and
// dr = g itself).  All three products are contractions of two operands with arbitrary steps, so one product kernel serves
// them, and its epilogue adds the bias, keeps z where the caller wants it for the gradients, and applies the rest before the
// element leaves the registers: y is written once and z is never read back.
#include "split_product.cuh"

namespace cb200 {

// ---- the product on the CUDA cores ------------------------------------------------------------------------------------
// 64 x 64 outputs per CTA, 4 x 4 per thread, 32 (16) of K at a time through shared memory.  Lanes run along whichever axis of
// each operand is contiguous.  Every 64 of K the sums so far are put aside and new ones begun: the error of a long sum in
// 32 bits then grows with the square root of its number of pieces, not of its terms.  Bound by the FMA rate at large sizes and by
// latency at small ones.
constexpr int kPcM = 64, kPcN = 64, kPcPad = 4;

template <typename T>
__global__ void __launch_bounds__(kBlock)
product_cc_kernel(int64_t m, int64_t n, int64_t k, const Operand<T> A, const Operand<T> B, const Epilogue<T> e, int64_t tiles_n) {
    constexpr int kPcK = sizeof(T) == 4 ? 32 : 16;               // (8-byte elements: 229 against 411 us for 256 x 2048 x 2048)
    __shared__ T As[kPcK][kPcM + kPcPad];
    __shared__ T Bs[kPcK][kPcN + kPcPad];
    const int64_t i0 = (int64_t)(blockIdx.x / tiles_n) * kPcM, j0 = (int64_t)(blockIdx.x % tiles_n) * kPcN;
    const int64_t batch = blockIdx.y;
    const T* a = A.p + batch * A.batch;
    const T* b = B.p + batch * B.batch;
    const int ti = threadIdx.x / 16, tj = threadIdx.x % 16;
    const bool a_along_k = A.k == 1, b_along_k = B.k == 1;
    constexpr int PER = kPcM * kPcK / kBlock;
    T ra[PER], rb[PER], acc[4][4], aside[4][4];
#pragma unroll
    for (int x = 0; x < 4; ++x)
#pragma unroll
        for (int y = 0; y < 4; ++y) acc[x][y] = aside[x][y] = T(0);
    auto fetch = [&](int64_t k0) {
#pragma unroll
        for (int s = 0; s < PER; ++s) {
            const int f = s * kBlock + threadIdx.x;
            const int ii = a_along_k ? f / kPcK : f % kPcM, ka = a_along_k ? f % kPcK : f / kPcM;
            ra[s] = i0 + ii < m && k0 + ka < k ? a[(i0 + ii) * A.row + (k0 + ka) * A.k] : T(0);
            const int jj = b_along_k ? f / kPcK : f % kPcN, kb = b_along_k ? f % kPcK : f / kPcN;
            rb[s] = j0 + jj < n && k0 + kb < k ? b[(j0 + jj) * B.row + (k0 + kb) * B.k] : T(0);
        }
    };
    fetch(0);
    for (int64_t k0 = 0; k0 < k; k0 += kPcK) {
        __syncthreads();
#pragma unroll
        for (int s = 0; s < PER; ++s) {
            const int f = s * kBlock + threadIdx.x;
            As[a_along_k ? f % kPcK : f / kPcM][a_along_k ? f / kPcK : f % kPcM] = ra[s];
            Bs[b_along_k ? f % kPcK : f / kPcN][b_along_k ? f / kPcK : f % kPcN] = rb[s];
        }
        __syncthreads();
        if (k0 + kPcK < k) fetch(k0 + kPcK);
        const int64_t kn = k - k0 < kPcK ? k - k0 : kPcK;        // zeros behind the end would turn an infinity into NaN only against
        for (int kk = 0; kk < kn; ++kk) {                         // another operand's padding; they are not multiplied at all
            T av[4], bv[4];
#pragma unroll
            for (int x = 0; x < 4; ++x) { av[x] = As[kk][ti * 4 + x]; bv[x] = Bs[kk][tj + 16 * x]; }
#pragma unroll
            for (int x = 0; x < 4; ++x)
#pragma unroll
                for (int y = 0; y < 4; ++y) acc[x][y] = av[x] * bv[y] + acc[x][y];
        }
        if ((k0 / kPcK) % (64 / kPcK) == 64 / kPcK - 1) {
#pragma unroll
            for (int x = 0; x < 4; ++x)
#pragma unroll
                for (int y = 0; y < 4; ++y) { aside[x][y] += acc[x][y]; acc[x][y] = T(0); }
        }
    }
#pragma unroll
    for (int x = 0; x < 4; ++x)
#pragma unroll
        for (int y = 0; y < 4; ++y) {
            const int64_t i = i0 + ti * 4 + x, j = j0 + tj + 16 * y;
            if (i < m && j < n) finish(e, batch, i, j, aside[x][y] + acc[x][y]);
        }
}

template <typename T>
int launch_product_cc(int64_t m, int64_t n, int64_t k, int64_t batch, const Operand<T>& a, const Operand<T>& b, const Epilogue<T>& e, cudaStream_t st) {
    const int64_t tiles_m = (m + kPcM - 1) / kPcM, tiles_n = (n + kPcN - 1) / kPcN;
    if (tiles_m * tiles_n > 0x7fffffff || batch > 65535) return (int)cudaErrorInvalidValue;
    product_cc_kernel<T><<<dim3((unsigned)(tiles_m * tiles_n), (unsigned)batch), kBlock, 0, st>>>(m, n, k, a, b, e, tiles_n);
    count_launch();
    return (int)cudaGetLastError();
}
template int launch_product_cc<float>(int64_t, int64_t, int64_t, int64_t, const Operand<float>&, const Operand<float>&, const Epilogue<float>&, cudaStream_t);
template int launch_product_cc<double>(int64_t, int64_t, int64_t, int64_t, const Operand<double>&, const Operand<double>&, const Epilogue<double>&, cudaStream_t);

// ---- dz = grad * act'(pre), and its column sums ------------------------------------------------------------------------
// A CTA owns 32 columns and a slice of the rows: eight warps on different rows, folded through shared memory in a fixed
// order; the slices' sums are folded by a second kernel in slice order, so db is the same every run.
template <typename T>
struct Steps2 { const T* p; int64_t row, col; };

template <typename T>
__global__ void __launch_bounds__(kBlock)
dz_kernel(int64_t m, int64_t n, const Steps2<T> grad, const Steps2<T> pre, int act, T* dz, T* sums, int64_t rows_per_slice) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t j = (int64_t)blockIdx.x * 32 + lane;
    const int64_t i0 = (int64_t)blockIdx.y * rows_per_slice;
    const int64_t i1 = i0 + rows_per_slice < m ? i0 + rows_per_slice : m;
    T sum = T(0);
    if (j < n) {
        for (int64_t i = i0 + warp; i < i1; i += kWarpsPerBlock) {
            T v = grad.p[i * grad.row + j * grad.col];
            if (act != kActNone) v *= activation_slope(pre.p[i * pre.row + j * pre.col], act);
            if (dz) dz[i * n + j] = v;
            sum += v;
        }
    }
    if (!sums) return;
    __shared__ T part[kWarpsPerBlock][32];
    part[warp][lane] = sum;
    __syncthreads();
    if (warp == 0 && j < n) {
        T s = part[0][lane];
#pragma unroll
        for (int w = 1; w < kWarpsPerBlock; ++w) s += part[w][lane];
        sums[(int64_t)blockIdx.y * n + j] = s;
    }
}

template <typename T>
__global__ void __launch_bounds__(kBlock)
fold_slices_kernel(int64_t n, int slices, const T* sums, T* out) {
    const int64_t j = (int64_t)blockIdx.x * kBlock + threadIdx.x;
    if (j >= n) return;
    T s = sums[j];
    for (int k = 1; k < slices; ++k) s += sums[(int64_t)k * n + j];
    out[j] = s;
}

template <typename T>
static int launch_dz(int64_t m, int64_t n, const Steps2<T>& grad, const Steps2<T>& pre, int act, T* dz, T* db, Scratch& scratch, cudaStream_t st) {
    const int64_t strips = (n + 31) / 32;
    int64_t slices = ((int64_t)sm_count() * 8 + strips - 1) / strips;
    const int64_t most = (m + 4 * kWarpsPerBlock - 1) / (4 * kWarpsPerBlock);
    if (slices > most) slices = most;
    if (slices > 256) slices = 256;
    const int64_t per = (m + slices - 1) / slices;
    slices = (m + per - 1) / per;
    T* sums = nullptr;
    if (db) {
        sums = slices == 1 ? db : reinterpret_cast<T*>(scratch.take((size_t)slices * n * sizeof(T)));
        if (!sums) return (int)cudaErrorMemoryAllocation;
    }
    dz_kernel<T><<<dim3((unsigned)strips, (unsigned)slices), kBlock, 0, st>>>(m, n, grad, pre, act, dz, sums, per);
    count_launch();
    if (db && slices > 1) {
        fold_slices_kernel<T><<<(unsigned)((n + kBlock - 1) / kBlock), kBlock, 0, st>>>(n, (int)slices, sums, db);
        count_launch();
    }
    return (int)cudaGetLastError();
}

// ---- single precision on the tensor cores -----------------------------------------------------------------------------
// An operand of the layer split once, whichever of its axes the products contract over.
struct SplitMatrix {
    SplitSource src;
    int64_t R, C;                     // planes are [R][ld >= C]: the axis the source has contiguous runs along is the inner one
    bool swapped;                     // R, C are the matrix's columns and rows
    uint16_t* planes;
    int64_t ld;
    Marks marks;
    uint8_t *hot_row, *hot_col;       // marks of the products' outputs along the axes that the matrix keeps (each axis by one product at most)
    // as operand of a contraction over the matrix's columns (over_columns) or rows
    Planes operand(bool over_columns) const {
        Planes p;
        p.p = planes; p.batch = 1; p.ld = ld;
        p.k_major = over_columns != swapped;
        p.rows = over_columns != swapped ? R : C;
        p.k = over_columns != swapped ? C : R;
        return p;
    }
    const uint8_t* marks_of(bool over_columns) const { return over_columns != swapped ? marks.row : marks.col; }
    uint8_t* hot_of(bool over_columns) const { return over_columns != swapped ? hot_row : hot_col; }
    bool turned(bool over_columns) const { return over_columns == swapped; }
};

struct SplitSet {
    SplitMatrix x[3];
    int count = 0;
    int add(const SplitSource& s, int64_t rows, int64_t cols) {
        SplitMatrix& a = x[count];
        a.src = s; a.R = rows; a.C = cols; a.swapped = false;
        if (s.col != 1 && s.row == 1) {
            a.swapped = true;
            a.R = cols; a.C = rows;
            a.src.row = s.col; a.src.col = s.row; a.src.pre_row = s.pre_col; a.src.pre_col = s.pre_row;
        }
        a.ld = planes_ld(a.C);
        return count++;
    }
    // scratch for all of them, marks cleared by one memset, then one launch that splits them
    int split(Scratch& scratch, cudaStream_t st) {
        size_t marks = 16;
        for (int i = 0; i < count; ++i) marks += 2 * (size_t)(x[i].R + x[i].C);
        char* mk = scratch.take(marks);
        if (!mk) return (int)cudaErrorMemoryAllocation;
        const int rc = (int)cudaMemsetAsync(mk, 0, marks, st);
        if (rc) return rc;
        int* any = reinterpret_cast<int*>(mk);
        mk += 16;
        SplitJobs jobs = {};
        jobs.count = count;
        for (int i = 0; i < count; ++i) {
            SplitMatrix& a = x[i];
            a.planes = reinterpret_cast<uint16_t*>(scratch.take((size_t)3 * a.R * a.ld * 2));
            if (!a.planes) return (int)cudaErrorMemoryAllocation;
            uint8_t* at = reinterpret_cast<uint8_t*>(mk);
            a.marks = {at, at + a.R, any};
            a.hot_row = at + a.R + a.C;
            a.hot_col = a.hot_row + a.R;
            mk += 2 * (a.R + a.C);
            jobs.job[i] = {a.src, a.R, a.C, a.ld, a.planes, a.marks};
        }
        return launch_split(jobs, st);
    }
    FixJobs fixes = {};
    int product(int a, bool a_over_columns, int b, bool b_over_columns, const Epilogue<float>& e, Scratch& scratch, cudaStream_t st) {
        const Planes pa = x[a].operand(a_over_columns), pb = x[b].operand(b_over_columns);
        fixes.job[fixes.count++] = {pa.rows, pb.rows, pa.k, x[a].src, x[b].src, x[a].turned(a_over_columns), x[b].turned(b_over_columns),
                                    x[a].marks_of(a_over_columns), x[b].marks_of(b_over_columns), x[a].hot_of(a_over_columns), x[b].hot_of(b_over_columns), e};
        return launch_split_product(pa, pb, e, Hot{x[a].hot_of(a_over_columns), x[b].hot_of(b_over_columns), x[0].marks.any}, scratch, st);
    }
    // what the marks ask for, once all products are queued
    int fix(cudaStream_t st) {
        fixes.any = x[0].marks.any;
        return launch_fix_marked(fixes, st);
    }
};

static bool worth_splitting(int64_t m, int64_t n, int64_t k) {
    // (measured: 134 x 85 x 674 22 us split and 15 on the CUDA cores, 142 x 367 x 128 26 and 39)
    return m >= 32 && n >= 32 && k >= 32 && m * n * k >= (k >= 128 ? 1LL << 22 : 1LL << 24);
}

// Few rows ride along with a pass over the weights (16 to a pass).  Measured in SFloat: 64 x 1024 x 1024 26 us against 39
// split, 33 x 4096 x 4096 105 against 80, so up to 32 rows always and up to 128 while there are under 2^28 products.
static bool few_rows(int64_t m, int64_t n, int64_t k) { return k >= 16 && (m <= 32 || (m <= 128 && m * n * k <= (1LL << 28))); }

template <typename T>
static int product(int64_t m, int64_t n, int64_t k, const Operand<T>& a, const Operand<T>& b, const Epilogue<T>& e, cudaStream_t st) {
    if (few_rows(m, n, k)) return launch_product_rows<T>(m, n, k, 1, a, b, e, st);
    return launch_product_cc<T>(m, n, k, 1, a, b, e, st);
}

// ---- entry points ------------------------------------------------------------------------------------------------------
template <typename T>
static int linear(int64_t m, int64_t n, int64_t k, const T* x, ssize_t x_row, ssize_t x_col, const T* w, ssize_t w_row, ssize_t w_col,
                  const T* bias, ssize_t bias_step, const T* residual, ssize_t r_row, ssize_t r_col, int activation, T* y, T* pre) {
    CB200_TRACE_LAUNCH();
    if (m < 0 || n < 0 || k < 1 || activation < 0 || activation >= kActCount) return (int)cudaErrorInvalidValue;
    if (m == 0 || n == 0) return 0;
    const int late = product_gave_up();
    if (late) return late;
    constexpr ssize_t es = sizeof(T);
    if (x_row % es || x_col % es || w_row % es || w_col % es || bias_step % es || r_row % es || r_col % es) return (int)cudaErrorInvalidValue;
    Epilogue<T> e = {};
    e.alpha = T(1);
    e.bias = bias; e.bias_step = bias_step / es;
    e.act = activation;
    e.res = residual; e.res_row = r_row / es; e.res_col = r_col / es;
    e.y = y; e.ld = n; e.pre = pre;
    if constexpr (sizeof(T) == 4) {
        if (!few_rows(m, n, k) && worth_splitting(m, n, k)) {
            Scratch scratch(current_stream());
            SplitSet set;
            const int ix = set.add(SplitSource{x, x_row / es, x_col / es, nullptr, 0, 0, kActNone}, m, k);
            const int iw = set.add(SplitSource{w, w_row / es, w_col / es, nullptr, 0, 0, kActNone}, k, n);
            int rc = set.split(scratch, current_stream());
            if (rc == 0) rc = set.product(ix, true, iw, false, e, scratch, current_stream());
            return rc ? rc : set.fix(current_stream());
        }
    }
    const Operand<T> a = {x, x_row / es, x_col / es, 0}, b = {w, w_col / es, w_row / es, 0};
    return product<T>(m, n, k, a, b, e, current_stream());
}

template <typename T>
static int linear_grad(int64_t m, int64_t n, int64_t k, const T* grad, ssize_t g_row, ssize_t g_col, const T* x, ssize_t x_row, ssize_t x_col,
                       const T* w, ssize_t w_row, ssize_t w_col, const T* pre, ssize_t p_row, ssize_t p_col, int activation, T* dx, T* dw, T* dbias) {
    CB200_TRACE_LAUNCH();
    if (m < 0 || n < 0 || k < 1 || activation < 0 || activation >= kActCount || (activation != kActNone && !pre && m && n)) return (int)cudaErrorInvalidValue;
    constexpr ssize_t es = sizeof(T);
    if (g_row % es || g_col % es || x_row % es || x_col % es || w_row % es || w_col % es || p_row % es || p_col % es) return (int)cudaErrorInvalidValue;
    cudaStream_t st = current_stream();
    if (n == 0) return dx && m ? (int)cudaMemsetAsync(dx, 0, (size_t)m * k * es, st) : 0;
    if (m == 0) {
        cudaError_t r = cudaSuccess;
        if (dw) r = cudaMemsetAsync(dw, 0, (size_t)n * k * es, st);
        if (dbias && r == cudaSuccess) r = cudaMemsetAsync(dbias, 0, (size_t)n * es, st);
        return (int)r;
    }
    const int late = product_gave_up();
    if (late) return late;
    Scratch scratch(st);
    Steps2<T> g = {grad, g_row / es, g_col / es}, p = {pre, p_row / es, p_col / es};
    Operand<T> dz = {grad, g.row, g.col, 0};
    if constexpr (sizeof(T) == 4) {
        if ((dx || dw) && worth_splitting(m, n, k)) {
            int rc = 0;
            if (dbias) rc = launch_dz<T>(m, n, g, p, activation, nullptr, dbias, scratch, st);
            if (rc) return rc;
            SplitSet set;
            const int iz = set.add(SplitSource{grad, g.row, g.col, pre, p.row, p.col, activation}, m, n);
            const int iw = dx ? set.add(SplitSource{w, w_row / es, w_col / es, nullptr, 0, 0, kActNone}, k, n) : 0;
            const int ix = dw ? set.add(SplitSource{x, x_row / es, x_col / es, nullptr, 0, 0, kActNone}, m, k) : 0;
            rc = set.split(scratch, st);
            Epilogue<float> e = {};
            e.alpha = 1.f;
            e.y = dx; e.ld = k;
            if (rc == 0 && dx) rc = set.product(iz, true, iw, true, e, scratch, st);
            e.y = dw; e.ld = n;
            if (rc == 0 && dw) rc = set.product(ix, false, iz, false, e, scratch, st);
            return rc ? rc : set.fix(st);
        }
    }
    if (activation != kActNone || dbias) {
        T* z = nullptr;
        if (activation != kActNone && (dx || dw)) {
            z = reinterpret_cast<T*>(scratch.take((size_t)m * n * es));
            if (!z) return (int)cudaErrorMemoryAllocation;
            dz = {z, n, 1, 0};
        }
        const int rc = launch_dz<T>(m, n, g, p, activation, z, dbias, scratch, st);
        if (rc) return rc;
    }
    Epilogue<T> e = {};
    e.alpha = T(1);
    if (dx) {                                    // dx[i][c] = sum_j dz[i][j] * w[c][j]
        e.y = dx; e.ld = k;
        const Operand<T> b = {w, w_row / es, w_col / es, 0};
        const int rc = product<T>(m, k, n, dz, b, e, st);
        if (rc) return rc;
    }
    if (dw) {                                    // dw[c][j] = sum_i x[i][c] * dz[i][j]
        e.y = dw; e.ld = n;
        const Operand<T> a = {x, x_col / es, x_row / es, 0}, b = {dz.p, dz.k, dz.row, 0};
        const int rc = product<T>(k, n, m, a, b, e, st);
        if (rc) return rc;
    }
    return 0;
}

}  // namespace cb200

#define CB200_DEF_LINEAR(NAME, T)                                                                                                         \
    extern "C" int cb200_##NAME##_linear_kernel_launch(                                                                                   \
        int64_t m, int64_t n, int64_t k, const T* x, ssize_t x_row, ssize_t x_col, const T* w, ssize_t w_row, ssize_t w_col,              \
        const T* bias, ssize_t bias_step, const T* residual, ssize_t r_row, ssize_t r_col, int activation, T* y, T* pre) {                \
        return cb200::linear<T>(m, n, k, x, x_row, x_col, w, w_row, w_col, bias, bias_step, residual, r_row, r_col, activation, y, pre);  \
    }                                                                                                                                     \
    extern "C" int cb200_##NAME##_linear_grad_kernel_launch(                                                                              \
        int64_t m, int64_t n, int64_t k, const T* grad, ssize_t g_row, ssize_t g_col, const T* x, ssize_t x_row, ssize_t x_col,           \
        const T* w, ssize_t w_row, ssize_t w_col, const T* pre, ssize_t p_row, ssize_t p_col, int activation, T* dx, T* dw, T* dbias) {   \
        return cb200::linear_grad<T>(m, n, k, grad, g_row, g_col, x, x_row, x_col, w, w_row, w_col, pre, p_row, p_col, activation, dx,    \
                                     dw, dbias);                                                                                          \
    }
CB200_DEF_LINEAR(sfloat, float)
CB200_DEF_LINEAR(dfloat, double)
