// Orthogonalising matrices by Newton-Schulz products.
//
// X0 = G / (|G|_F + eps); then per step, with P = X X^T on the side with the fewer rows,
//     X <- a X + (b P + c P P) X.
// An odd polynomial of X acts on its singular values alone, so the steps drive the singular values towards the
// polynomial's fixed points and leave the singular vectors: the result is near U V^T for G = U S V^T.
// Work per step and matrix of m <= n: 2 m^2 n (P) + 2 m^3 (P P) + 2 m^2 n (the product with X).
#include "linear.cuh"

namespace cb200 {

// ---- |G|_F in 64 bits: slices of a matrix to partial sums of squares, folded in slice order ---------------------------
template <typename T>
__global__ void __launch_bounds__(kBlock)
square_sums_kernel(const Operand<T> G, int64_t m, int64_t n, int slices, double* sums) {
    const T* g = G.p + (int64_t)blockIdx.y * G.batch;
    const int64_t total = m * n;
    double s = 0;
    for (int64_t f = (int64_t)blockIdx.x * kBlock + threadIdx.x; f < total; f += (int64_t)slices * kBlock) {
        const int64_t i = f / n;
        const double v = (double)g[i * G.row + (f - i * n) * G.k];
        s += v * v;
    }
    __shared__ double part[kBlock];
    part[threadIdx.x] = s;
    __syncthreads();
    for (int w = kBlock / 2; w > 0; w >>= 1) {
        if ((int)threadIdx.x < w) part[threadIdx.x] += part[threadIdx.x + w];
        __syncthreads();
    }
    if (threadIdx.x == 0) sums[(int64_t)blockIdx.y * slices + blockIdx.x] = part[0];
}

// X0, row-major.  Sums beyond the type's range (or a NaN) make every element NaN, as the products would.
template <typename T>
__global__ void __launch_bounds__(kBlock)
scale_kernel(const Operand<T> G, int64_t m, int64_t n, int slices, const double* sums, double eps, T* x) {
    __shared__ double inv;
    if (threadIdx.x == 0) {
        double s = 0;
        for (int k = 0; k < slices; ++k) s += sums[(int64_t)blockIdx.y * slices + k];
        inv = s - s == 0 ? 1.0 / (sqrt(s) + eps) : s - s;
    }
    __syncthreads();
    const T* g = G.p + (int64_t)blockIdx.y * G.batch;
    const int64_t total = m * n;
    T* out = x + (int64_t)blockIdx.y * total;
    for (int64_t f = (int64_t)blockIdx.x * kBlock + threadIdx.x; f < total; f += (int64_t)gridDim.x * kBlock) {
        const int64_t i = f / n;
        out[f] = (T)((double)g[i * G.row + (f - i * n) * G.k] * inv);
    }
}

// out[b][j][i] = in[b][i][j] through 32 x 32 tiles in shared memory
template <typename T>
__global__ void __launch_bounds__(kBlock)
turn_kernel(int64_t m, int64_t n, int64_t tiles_n, const T* in, T* out) {
    __shared__ T tile[32][33];
    const int64_t i0 = (int64_t)(blockIdx.x / tiles_n) * 32, j0 = (int64_t)(blockIdx.x % tiles_n) * 32;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    in += (int64_t)blockIdx.y * m * n;
    out += (int64_t)blockIdx.y * m * n;
    for (int r = warp; r < 32; r += kWarpsPerBlock)
        if (i0 + r < m && j0 + lane < n) tile[r][lane] = in[(i0 + r) * n + j0 + lane];
    __syncthreads();
    for (int r = warp; r < 32; r += kWarpsPerBlock)
        if (j0 + r < n && i0 + lane < m) out[(j0 + r) * m + i0 + lane] = tile[lane][r];
}
template <typename T>
static int turn(int64_t batch, int64_t m, int64_t n, const T* in, T* out, cudaStream_t st) {
    const int64_t tm = (m + 31) / 32, tn = (n + 31) / 32;
    turn_kernel<T><<<dim3((unsigned)(tm * tn), (unsigned)batch), kBlock, 0, st>>>(m, n, tn, in, out);
    count_launch();
    return (int)cudaGetLastError();
}
// g: batch matrices of rows x columns (steps in bytes); out: the same, contiguous.  coefs: 3 numbers per step (host).
template <typename T>
static int orthogonalize(int64_t batch, int64_t rows, int64_t columns, const T* g, ssize_t g_batch, ssize_t g_row, ssize_t g_col, int steps,
                         const double* coefs, double eps, T* out) {
    CB200_TRACE_LAUNCH();
    constexpr ssize_t es = sizeof(T);
    if (batch < 0 || rows < 0 || columns < 0 || steps < 0 || (steps && !coefs) || g_batch % es || g_row % es || g_col % es || batch > 65535)
        return (int)cudaErrorInvalidValue;
    if (batch == 0 || rows == 0 || columns == 0) return 0;
    cudaStream_t st = current_stream();
    const bool tall = rows > columns;
    const int64_t m = tall ? columns : rows, n = tall ? rows : columns;
    const Operand<T> G = tall ? Operand<T>{g, g_col / es, g_row / es, g_batch / es} : Operand<T>{g, g_row / es, g_col / es, g_batch / es};
    Scratch scratch(st);
    int64_t slices = (m * n + kBlock * 8 - 1) / (kBlock * 8);
    if (slices > 256) slices = 256;
    double* sums = reinterpret_cast<double*>(scratch.take((size_t)batch * slices * sizeof(double)));
    T* x = reinterpret_cast<T*>(scratch.take((size_t)batch * m * n * es));
    T* x2 = reinterpret_cast<T*>(scratch.take((size_t)batch * m * n * es));
    T* p = reinterpret_cast<T*>(scratch.take((size_t)batch * m * m * es));
    T* q = reinterpret_cast<T*>(scratch.take((size_t)batch * m * m * es));
    if (!sums || !x || !x2 || !p || !q) return (int)cudaErrorMemoryAllocation;
    square_sums_kernel<T><<<dim3((unsigned)slices, (unsigned)batch), kBlock, 0, st>>>(G, m, n, (int)slices, sums);
    scale_kernel<T><<<dim3((unsigned)slices, (unsigned)batch), kBlock, 0, st>>>(G, m, n, (int)slices, sums, eps, x);
    count_launch(2);
    int rc = (int)cudaGetLastError();
    for (int s = 0; s < steps && rc == 0; ++s) {
        const T a = (T)coefs[3 * s], b = (T)coefs[3 * s + 1], c = (T)coefs[3 * s + 2];
        Epilogue<T> e = {};
        e.alpha = T(1); e.y = p; e.ld = m; e.y_batch = m * m;                              // P = X X^T
        rc = launch_product_cc<T>(m, m, n, batch, {x, n, 1, m * n}, {x, n, 1, m * n}, e, st);
        if (rc) break;
        e.alpha = c; e.beta = b; e.d = p; e.d_row = m; e.d_col = 1; e.d_batch = m * m; e.y = q;   // Q = b P + c P P
        rc = launch_product_cc<T>(m, m, m, batch, {p, m, 1, m * m}, {p, m, 1, m * m}, e, st);
        if (rc) break;
        e.alpha = T(1); e.beta = a; e.d = x; e.d_row = n; e.d_batch = m * n; e.y = x2; e.ld = n; e.y_batch = m * n;   // X <- a X + Q X
        rc = launch_product_cc<T>(m, n, m, batch, {q, m, 1, m * m}, {x, 1, n, m * n}, e, st);
        T* t = x; x = x2; x2 = t;
    }
    if (rc) return rc;
    // into the caller's array, turned back if the matrices were taken by their columns
    if (tall) rc = turn(batch, m, n, x, out, st);
    else rc = (int)cudaMemcpyAsync(out, x, (size_t)batch * m * n * es, cudaMemcpyDeviceToDevice, st);
    return rc;
}

}  // namespace cb200

extern "C" int cb200_sfloat_orthogonalize_kernel_launch(int64_t batch, int64_t rows, int64_t columns, const float* g, ssize_t g_batch, ssize_t g_row,
                                                        ssize_t g_col, int steps, const double* coefs, double eps, float* out) {
    return cb200::orthogonalize<float>(batch, rows, columns, g, g_batch, g_row, g_col, steps, coefs, eps, out);
}
extern "C" int cb200_dfloat_orthogonalize_kernel_launch(int64_t batch, int64_t rows, int64_t columns, const double* g, ssize_t g_batch, ssize_t g_row,
                                                        ssize_t g_col, int steps, const double* coefs, double eps, double* out) {
    return cb200::orthogonalize<double>(batch, rows, columns, g, g_batch, g_row, g_col, steps, coefs, eps, out);
}
