// Orthogonalising matrices by Newton-Schulz products.
//
// X0 = G / (|G|_F + eps); then per step, with P = X X^T on the side with the fewer rows,
//     X <- a X + (b P + c P P) X.
// An odd polynomial of X acts on its singular values alone, so the steps drive the singular values towards the
// polynomial's fixed points and leave the singular vectors: the result is near U V^T for G = U S V^T.
// Work per step and matrix of m <= n: 2 m^2 n (P) + 2 m^3 (P P) + 2 m^2 n (the product with X).
#include "split_product.cuh"

namespace cb200 {

// ---- |G|_F in 64 bits: slices of a matrix to partial sums of squares, folded in slice order ---------------------------
// (rows and columns may be exchanged for this: the caller passes the contiguous axis as columns)
// Squares of 64-bit elements above 2^500 or below 2^-500 have sums of their own, of the elements scaled by 2^-600 and 2^600.
template <typename T> constexpr int kSquareSums = sizeof(T) == 8 ? 3 : 1;
constexpr double kFarUp = 0x1p500, kFarDown = 0x1p-500, kUp = 0x1p600, kDown = 0x1p-600;

// What an element is multiplied by: (v * half) * inv * half = v / (norm + eps), half = 1 unless the norm is far from 1.
struct Inverse { double inv, half; };
template <typename T>
__device__ __forceinline__ Inverse inverse_norm(const double* s, double eps) {
    if (!(s[0] - s[0] == 0)) return {s[0] - s[0], 1.0};              // infinite or NaN: every element becomes NaN
    if constexpr (sizeof(T) == 8) {
        const double high = s[1], low = s[2];
        if (!(high - high == 0)) return {high - high, 1.0};
        if (high > 0) return {1.0 / (sqrt(high + s[0] * kDown * kDown) + eps * kDown), 0x1p-300};
        if (s[0] == 0 && low > 0 && eps < 0x1p-300) return {1.0 / (sqrt(low) + eps * kUp), 0x1p300};
        return {1.0 / (sqrt(s[0] + low * kDown * kDown) + eps), 1.0};
    }
    return {1.0 / (sqrt(s[0]) + eps), 1.0};
}

template <typename T>
__global__ void __launch_bounds__(kBlock)
square_sums_kernel(const T* g, int64_t g_batch, int64_t rows, int64_t columns, int64_t row_step, int64_t column_step, int slices, double* sums) {
    g += (int64_t)blockIdx.y * g_batch;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    constexpr int K = kSquareSums<T>;
    double s = 0, far[2] = {0, 0};
    for (int64_t i = (int64_t)blockIdx.x * kWarpsPerBlock + warp; i < rows; i += (int64_t)slices * kWarpsPerBlock) {
        const T* r = g + i * row_step;
        for (int64_t j0 = lane; j0 < columns; j0 += 32 * 8) {
            T v[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) v[u] = j0 + u * 32 < columns ? r[(j0 + u * 32) * column_step] : T(0);
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                if constexpr (K == 1) {
                    s = fma((double)v[u], (double)v[u], s);
                } else {
                    const double a = fabs((double)v[u]);
                    const bool up = !(a <= kFarUp), down = a < kFarDown;       // (a NaN counts as up)
                    const double b = up ? a * kDown : down ? a * kUp : a, sq = b * b;
                    s += up || down ? 0.0 : sq;
                    far[0] += up ? sq : 0.0;
                    far[1] += down ? sq : 0.0;
                }
            }
        }
    }
    __shared__ double part[kBlock];
#pragma unroll
    for (int c = 0; c < K; ++c) {
        part[threadIdx.x] = c == 0 ? s : far[c - 1];
        __syncthreads();
        for (int w = kBlock / 2; w > 0; w >>= 1) {
            if ((int)threadIdx.x < w) part[threadIdx.x] += part[threadIdx.x + w];
            __syncthreads();
        }
        if (threadIdx.x == 0) sums[((int64_t)blockIdx.y * slices + blockIdx.x) * K + c] = part[0];
    }
}

// X0, row-major.  An infinity or a NaN makes every element NaN, as the products would.
template <typename T>
__global__ void __launch_bounds__(kBlock)
scale_kernel(const Operand<T> G, int64_t m, int64_t n, int slices, const double* sums, double eps, T* x) {
    __shared__ Inverse by;
    constexpr int K = kSquareSums<T>;
    if (threadIdx.x == 0) {
        double s[K] = {};
        for (int k = 0; k < slices; ++k)
            for (int c = 0; c < K; ++c) s[c] += sums[((int64_t)blockIdx.y * slices + k) * K + c];
        by = inverse_norm<T>(s, eps);
    }
    __syncthreads();
    const T* g = G.p + (int64_t)blockIdx.y * G.batch;
    const int64_t total = m * n;
    T* out = x + (int64_t)blockIdx.y * total;
    for (int64_t f = (int64_t)blockIdx.x * kBlock + threadIdx.x; f < total; f += (int64_t)gridDim.x * kBlock) {
        const int64_t i = f / n;
        out[f] = (T)((double)g[i * G.row + (f - i * n) * G.k] * by.half * by.inv * by.half);
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

// ---- single precision: the iteration on planes ------------------------------------------------------------------------
// X, P and Q are held as three bfloat16 parts each, all 24 bits of a float under its own exponent: rows, columns and single
// elements that are small beside the others, and matrices that are small beside eps, keep the digits that they have in 32 bits.
// X0 as planes [plane][batch][m][ld] through 32 x 32 tiles, lanes along whichever axis of G is contiguous.
__global__ void __launch_bounds__(kBlock)
scale_planes_kernel(const Operand<float> G, int64_t m, int64_t n, int64_t tiles_n, int slices, const double* sums, double eps, uint16_t* planes,
                    int64_t ld, int64_t plane) {
    __shared__ double inv;
    __shared__ float tile[32][33];
    if (threadIdx.x < 32) {
        double s = 0;
        for (int k = threadIdx.x; k < slices; k += 32) s += sums[(int64_t)blockIdx.y * slices + k];
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (threadIdx.x == 0) inv = inverse_norm<float>(&s, eps).inv;
    }
    const int64_t i0 = (int64_t)(blockIdx.x / tiles_n) * 32, j0 = (int64_t)(blockIdx.x % tiles_n) * 32;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const float* g = G.p + (int64_t)blockIdx.y * G.batch;
    const bool down = G.row == 1 && G.k != 1;
    for (int r = warp; r < 32; r += kWarpsPerBlock) {
        const int64_t i = down ? i0 + lane : i0 + r, j = down ? j0 + r : j0 + lane;
        const float v = i < m && j < n ? g[i * G.row + j * G.k] : 0.f;
        if (down) tile[lane][r] = v; else tile[r][lane] = v;
    }
    __syncthreads();
    uint16_t* out = planes + (int64_t)blockIdx.y * m * ld;
    for (int r = warp; r < 32; r += kWarpsPerBlock) {
        const int64_t i = i0 + r, j = j0 + lane;
        if (i >= m || j >= n) continue;
        uint32_t a, b, c;
        split3_all((float)((double)tile[r][lane] * inv), a, b, c);
        out[i * ld + j] = (uint16_t)a;
        out[plane + i * ld + j] = (uint16_t)b;
        out[2 * plane + i * ld + j] = (uint16_t)c;
    }
}

// out[b][i][j] (or [j][i]) = the sum of the parts
__global__ void __launch_bounds__(kBlock)
join_planes_kernel(int64_t m, int64_t n, int64_t tiles_n, const uint16_t* planes, int64_t ld, int64_t plane, bool tall, float* out) {
    __shared__ float tile[32][33];
    const int64_t i0 = (int64_t)(blockIdx.x / tiles_n) * 32, j0 = (int64_t)(blockIdx.x % tiles_n) * 32;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint16_t* in = planes + (int64_t)blockIdx.y * m * ld;
    out += (int64_t)blockIdx.y * m * n;
    for (int r = warp; r < 32; r += kWarpsPerBlock) {
        const int64_t i = i0 + r, j = j0 + lane;
        if (i < m && j < n) {
            const uint16_t* p = in + i * ld + j;
            const float v = bf16_at(p[0]) + (bf16_at(p[plane]) + bf16_at(p[2 * plane]));
            if (tall) tile[r][lane] = v; else out[i * n + j] = v;
        }
    }
    if (!tall) return;
    __syncthreads();
    for (int r = warp; r < 32; r += kWarpsPerBlock)
        if (j0 + r < n && i0 + lane < m) out[(j0 + r) * m + i0 + lane] = tile[lane][r];
}

static int orthogonalize_split(int64_t batch, int64_t m, int64_t n, bool tall, const Operand<float>& G, int steps, const double* coefs, double eps, int slices,
                               const double* sums, float* out, Scratch& scratch, cudaStream_t st) {
    const int64_t ldx = planes_ld(n), ldp = planes_ld(m), px = batch * m * ldx, pp = batch * m * ldp;
    uint16_t* x = reinterpret_cast<uint16_t*>(scratch.take((size_t)px * 6));
    uint16_t* x2 = reinterpret_cast<uint16_t*>(scratch.take((size_t)px * 6));
    uint16_t* p = reinterpret_cast<uint16_t*>(scratch.take((size_t)pp * 6));
    uint16_t* q = reinterpret_cast<uint16_t*>(scratch.take((size_t)pp * 6));
    if (!x || !x2 || !p || !q) return (int)cudaErrorMemoryAllocation;
    const int64_t tm = (m + 31) / 32, tn = (n + 31) / 32;
    if (tm * tn > 0x7fffffff) return (int)cudaErrorInvalidValue;
    const dim3 grid((unsigned)(tm * tn), (unsigned)batch);
    scale_planes_kernel<<<grid, kBlock, 0, st>>>(G, m, n, tn, slices, sums, eps, x, ldx, px);
    count_launch();
    int rc = (int)cudaGetLastError();
    for (int s = 0; s < steps && rc == 0; ++s) {
        const float a = (float)coefs[3 * s], b = (float)coefs[3 * s + 1], c = (float)coefs[3 * s + 2];
        const Planes X = {x, m, n, batch, ldx, true}, Xn = {x, n, m, batch, ldx, false}, P = {p, m, m, batch, ldp, true}, Q = {q, m, m, batch, ldp, true};
        PlaneEpilogue e = {};
        e.alpha = 1.f; e.out = p; e.ld = ldp; e.plane = pp; e.batch_step = m * ldp;              // P = X X^T
        rc = launch_split_product(X, X, e, true, st);
        if (rc) break;
        e.alpha = c; e.beta = b; e.d = p; e.out = q;                                             // Q = b P + c P P
        rc = launch_split_product(P, P, e, true, st);
        if (rc) break;
        e.alpha = 1.f; e.beta = a; e.d = x; e.out = x2; e.ld = ldx; e.plane = px; e.batch_step = m * ldx;      // X <- a X + Q X
        rc = launch_split_product(Q, Xn, e, false, st);
        uint16_t* t = x; x = x2; x2 = t;
    }
    if (rc) return rc;
    join_planes_kernel<<<grid, kBlock, 0, st>>>(m, n, tn, x, ldx, px, tall, out);
    count_launch();
    return (int)cudaGetLastError();
}

// g: batch matrices of rows x columns (steps in bytes); out: the same, contiguous.  coefs: 3 numbers per step (host).
template <typename T>
static int orthogonalize(int64_t batch, int64_t rows, int64_t columns, const T* g, ssize_t g_batch, ssize_t g_row, ssize_t g_col, int steps,
                         const double* coefs, double eps, T* out) {
    CB200_TRACE_LAUNCH();
    constexpr ssize_t es = sizeof(T);
    if (batch < 0 || rows < 0 || columns < 0 || steps < 0 || (steps && !coefs) || g_batch % es || g_row % es || g_col % es)
        return (int)cudaErrorInvalidValue;
    if (batch == 0 || rows == 0 || columns == 0) return 0;
    const int late = product_gave_up();
    if (late) return late;
    constexpr int64_t kMostBatch = 32768;                       // (grids count the matrices in 16 bits)
    if (batch > kMostBatch) {
        for (int64_t b = 0; b < batch; b += kMostBatch) {
            const int rc = orthogonalize<T>(batch - b < kMostBatch ? batch - b : kMostBatch, rows, columns, g + b * (g_batch / es), g_batch, g_row, g_col, steps,
                                            coefs, eps, out + b * rows * columns);
            if (rc) return rc;
        }
        return 0;
    }
    cudaStream_t st = current_stream();
    const bool tall = rows > columns;
    const int64_t m = tall ? columns : rows, n = tall ? rows : columns;
    const Operand<T> G = tall ? Operand<T>{g, g_col / es, g_row / es, g_batch / es} : Operand<T>{g, g_row / es, g_col / es, g_batch / es};
    Scratch scratch(st);
    const bool along_k = G.k == 1 || G.row != 1;
    const int64_t sr = along_k ? m : n, sc_ = along_k ? n : m;
    int64_t slices = (sr + kWarpsPerBlock - 1) / kWarpsPerBlock;
    const int64_t enough = ((int64_t)sm_count() * 4 + batch - 1) / batch;
    if (slices > enough) slices = enough;
    if (slices > 256) slices = 256;
    double* sums = reinterpret_cast<double*>(scratch.take((size_t)batch * slices * kSquareSums<T> * sizeof(double)));
    if (!sums) return (int)cudaErrorMemoryAllocation;
    square_sums_kernel<T><<<dim3((unsigned)slices, (unsigned)batch), kBlock, 0, st>>>(G.p, G.batch, sr, sc_, along_k ? G.row : G.k, along_k ? G.k : G.row,
                                                                                  (int)slices, sums);
    count_launch();
    if constexpr (sizeof(T) == 4) {
        // Few rows with long sums: a product on planes has one or a few tiles then, each with the whole of K before it, while the
        // row products cut P's sums over clusters and cost little arithmetic.  Five steps in us, on planes and on the CUDA cores:
        // 64 x 256 149 and 187, 128 x 1024 244 and 255, 128 x 2048 352 and 260, 128 x 16384 1914 and 582, 33 x 30000 3370 and 582;
        // with more of them the arithmetic counts, 64 of 32 x 2000 632 and 561, 8 of 128 x 2048 409 and 578.  (Errors are alike.)
        const bool few = m < 16 || (m <= 128 && n >= 9 * m && batch * m * m <= 65536);
        if (!few) return orthogonalize_split(batch, m, n, tall, G, steps, coefs, eps, (int)slices, sums, out, scratch, st);
    }
    T* x = reinterpret_cast<T*>(scratch.take((size_t)batch * m * n * es));
    T* x2 = reinterpret_cast<T*>(scratch.take((size_t)batch * m * n * es));
    T* p = reinterpret_cast<T*>(scratch.take((size_t)batch * m * m * es));
    T* q = reinterpret_cast<T*>(scratch.take((size_t)batch * m * m * es));
    if (!x || !x2 || !p || !q) return (int)cudaErrorMemoryAllocation;
    scale_kernel<T><<<dim3(256u, (unsigned)batch), kBlock, 0, st>>>(G, m, n, (int)slices, sums, eps, x);
    count_launch();
    int rc = (int)cudaGetLastError();
    for (int s = 0; s < steps && rc == 0; ++s) {
        const T a = (T)coefs[3 * s], b = (T)coefs[3 * s + 1], c = (T)coefs[3 * s + 2];
        Epilogue<T> e = {};
        e.alpha = T(1); e.y = p; e.ld = m; e.y_batch = m * m;                              // P = X X^T
        rc = m <= 128 && n >= 64 ? launch_product_rows<T>(m, m, n, batch, {x, n, 1, m * n}, {x, n, 1, m * n}, e, st)
                                 : launch_product_cc<T>(m, m, n, batch, {x, n, 1, m * n}, {x, n, 1, m * n}, e, st);
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
