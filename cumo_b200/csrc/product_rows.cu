// Products with few rows: y[i][j] = sum_k A(i, k) * B(j, k) for m up to a few dozen (one token, a few sequences' tokens).
//
// Bound by reading B (the weights) once: sizeof(T) bytes per element against 2 m operations, so up to about 16 rows the
// CUDA cores' FMAs keep up with memory and no tensor core is needed.  All rows of A (in tiles of MT) ride along with one
// pass over B: a CTA holds a piece of A in shared memory and MT x (columns of a lane) sums in registers.
//   columns   B contiguous along j: a lane owns V neighbouring columns, a CTA a strip of 32 V; its eight warps take every
//             eighth k
//   dots      B contiguous along k: a warp owns C columns, its lanes run along k in packets, a shuffle adds them up
// K is cut over the CTAs of a cluster too, until the loads in flight cover the memory's latency; their sums meet in
// distributed shared memory and are added in CTA order, so that the result is the same every run, and the epilogue is applied
// by whichever CTA finishes an output: one launch, nothing goes through global memory twice.
#include "linear.cuh"

#include <cooperative_groups.h>

namespace cb200 {

constexpr int kRowsChunk = 512;                     // k per piece of A

// Adds the cluster's partial sums red[MT][cols] in CTA order and finishes this CTA's share of the outputs.
template <typename T, int MT>
__device__ __forceinline__ void finish_rows(T* red, int cols, int cluster_size, int64_t batch, int64_t i0, int64_t j0, int64_t m, int64_t n,
                                            const Epilogue<T>& e) {
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    if (cluster_size > 1) cluster.sync();
    else __syncthreads();
    const int rank = cluster_size > 1 ? (int)cluster.block_rank() : 0;
    for (int f = rank * kBlock + threadIdx.x; f < MT * cols; f += cluster_size * kBlock) {
        const int64_t i = i0 + f / cols, j = j0 + f % cols;
        if (i >= m || j >= n) continue;
        T s = T(0);
        if (cluster_size > 1) {
            T part[8];
#pragma unroll
            for (int r = 0; r < 8; ++r) if (r < cluster_size) part[r] = *cluster.map_shared_rank(red + f, r);
#pragma unroll
            for (int r = 0; r < 8; ++r) if (r < cluster_size) s = r == 0 ? part[0] : s + part[r];
        } else {
            s = red[f];
        }
        finish(e, batch, i, j, s);
    }
    if (cluster_size > 1) cluster.sync();                        // nobody leaves while its sums may still be read
}

template <typename T, int MT>
__device__ __forceinline__ void load_piece(T* xs, const Operand<T>& A, int64_t i0, int64_t m, int64_t k0, int kn) {
    for (int f = threadIdx.x; f < MT * kn; f += kBlock) {
        const int r = f / kn, c = f - r * kn;
        xs[c * MT + r] = i0 + r < m ? A.p[(i0 + r) * A.row + (k0 + c) * A.k] : T(0);
    }
}

template <typename T, int N> struct alignas(sizeof(T) * N > 16 ? 16 : sizeof(T) * N) RowVec { T v[N]; };

template <typename T, int MT, bool PACKETS>
__global__ void __launch_bounds__(kBlock)
rows_by_columns_kernel(int64_t m, int64_t n, int64_t k, Operand<T> A, Operand<T> B, const Epilogue<T> e, int cluster_size, int64_t strips) {
    constexpr int V = 16 / sizeof(T), COLS = 32 * V, U = 8;
    extern __shared__ __align__(16) char smem[];
    T* xs = reinterpret_cast<T*>(smem);                          // [k of the piece][MT]
    T* part = reinterpret_cast<T*>(smem);                        // [8 warps][MT][COLS], after the last piece
    T* red = part + kWarpsPerBlock * MT * COLS;                  // [MT][COLS]
    A.p += (int64_t)blockIdx.y * A.batch;
    B.p += (int64_t)blockIdx.y * B.batch;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int rank = blockIdx.x % cluster_size;
    const int64_t unit = blockIdx.x / cluster_size, j0 = (unit % strips) * COLS, i0 = (unit / strips) * MT;
    const int64_t per = (k + cluster_size - 1) / cluster_size, k_begin = rank * per, k_end = k_begin + per < k ? k_begin + per : k;
    T acc[MT][V];
#pragma unroll
    for (int r = 0; r < MT; ++r)
#pragma unroll
        for (int v = 0; v < V; ++v) acc[r][v] = T(0);
    const int64_t jv = j0 + lane * V;
    const bool whole = PACKETS && jv + V <= n;
    const T* b = B.p + (whole ? jv : 0) * B.row;
    for (int64_t k0 = k_begin; k0 < k_end; k0 += kRowsChunk) {
        const int kn = k_end - k0 < kRowsChunk ? (int)(k_end - k0) : kRowsChunk;
        __syncthreads();
        load_piece<T, MT>(xs, A, i0, m, k0, kn);
        __syncthreads();
        for (int c0 = warp; c0 < kn; c0 += kWarpsPerBlock * U) {
            T w[U][V];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int c = c0 + u * kWarpsPerBlock;
                if (PACKETS) {
                    if (c < kn && whole) {
                        const Pack<T> q = ld_pack<T>(b + (k0 + c) * B.k);
#pragma unroll
                        for (int v = 0; v < V; ++v) w[u][v] = q.v[v];
                    }
                } else {
#pragma unroll
                    for (int v = 0; v < V; ++v) {
                        const int64_t j = j0 + lane + 32 * v;
                        w[u][v] = c < kn && j < n ? ld_one<T>(B.p + j * B.row + (k0 + c) * B.k) : T(0);
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int c = c0 + u * kWarpsPerBlock;
                if (c >= kn) break;
                constexpr int P = MT * sizeof(T) >= 16 ? 16 / sizeof(T) : MT;
#pragma unroll
                for (int r = 0; r < MT; r += P) {
                    const RowVec<T, P> x = *reinterpret_cast<const RowVec<T, P>*>(xs + c * MT + r);
#pragma unroll
                    for (int p = 0; p < P; ++p)
#pragma unroll
                        for (int v = 0; v < V; ++v) acc[r + p][v] = x.v[p] * w[u][v] + acc[r + p][v];
                }
            }
        }
    }
    __syncthreads();
    const bool mine = !PACKETS || whole;
#pragma unroll
    for (int r = 0; r < MT; ++r)
#pragma unroll
        for (int v = 0; v < V; ++v)
            if (mine) part[(warp * MT + r) * COLS + (PACKETS ? lane * V + v : lane + 32 * v)] = acc[r][v];
    __syncthreads();
    for (int f = threadIdx.x; f < MT * COLS; f += kBlock) {
        T s = part[f];
#pragma unroll
        for (int w = 1; w < kWarpsPerBlock; ++w) s += part[w * MT * COLS + f];
        red[f] = s;
    }
    finish_rows<T, MT>(red, COLS, cluster_size, blockIdx.y, i0, j0, m, n, e);
}

template <typename T, int MT, int C, bool PACKETS>
__global__ void __launch_bounds__(kBlock)
rows_by_dots_kernel(int64_t m, int64_t n, int64_t k, Operand<T> A, Operand<T> B, const Epilogue<T> e, int cluster_size, int64_t strips) {
    constexpr int V = PACKETS ? 16 / sizeof(T) : 1, COLS = kWarpsPerBlock * C, SPAN = 32 * V;
    extern __shared__ __align__(16) char smem[];
    T* xs = reinterpret_cast<T*>(smem);                          // [MT][k of the piece]
    __shared__ T red[MT * COLS];
    A.p += (int64_t)blockIdx.y * A.batch;
    B.p += (int64_t)blockIdx.y * B.batch;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int rank = blockIdx.x % cluster_size;
    const int64_t unit = blockIdx.x / cluster_size, j0 = (unit % strips) * COLS, i0 = (unit / strips) * MT;
    int64_t per = (k + cluster_size - 1) / cluster_size;
    per = (per + 3) / 4 * 4;                                     // pieces start on packets
    const int64_t k_begin = rank * per < k ? rank * per : k, k_end = k_begin + per < k ? k_begin + per : k;
    T acc[MT][C];
#pragma unroll
    for (int r = 0; r < MT; ++r)
#pragma unroll
        for (int c = 0; c < C; ++c) acc[r][c] = T(0);
    const T* b[C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int64_t j = j0 + warp * C + c;
        b[c] = B.p + (j < n ? j : n - 1) * B.row;                // a column past the end repeats the last one; it is not stored
    }
    for (int64_t k0 = k_begin; k0 < k_end; k0 += kRowsChunk) {
        const int kn = k_end - k0 < kRowsChunk ? (int)(k_end - k0) : kRowsChunk;
        __syncthreads();
        for (int f = threadIdx.x; f < MT * kRowsChunk; f += kBlock) {
            const int r = f / kRowsChunk, c = f % kRowsChunk;
            xs[f] = i0 + r < m && c < kn ? A.p[(i0 + r) * A.row + (k0 + c) * A.k] : T(0);
        }
        __syncthreads();
        constexpr int U = 2;
        for (int c0 = 0; c0 < kn; c0 += SPAN * U) {
            T w[U][C][V];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int at = c0 + u * SPAN + lane * V;
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    if (PACKETS && at + V <= kn) {
                        const Pack<T> q = ld_pack<T>(b[c] + k0 + at);
#pragma unroll
                        for (int v = 0; v < V; ++v) w[u][c][v] = q.v[v];
                    } else {
#pragma unroll
                        for (int v = 0; v < V; ++v) w[u][c][v] = at + v < kn ? ld_one<T>(b[c] + (k0 + at + v) * B.k) : T(0);
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int at = c0 + u * SPAN + lane * V;
                if (at >= kn) break;
#pragma unroll
                for (int r = 0; r < MT; ++r) {
                    const RowVec<T, V> x = *reinterpret_cast<const RowVec<T, V>*>(xs + r * kRowsChunk + at);
#pragma unroll
                    for (int v = 0; v < V; ++v) {
                        if (at + v >= kn) break;                 // (what lies behind the end may be anything in B's place)
#pragma unroll
                        for (int c = 0; c < C; ++c) acc[r][c] = x.v[v] * w[u][c][v] + acc[r][c];
                    }
                }
            }
        }
    }
#pragma unroll
    for (int r = 0; r < MT; ++r)
#pragma unroll
        for (int c = 0; c < C; ++c) {
            T s = acc[r][c];
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
            if (lane == 0) red[r * COLS + warp * C + c] = s;
        }
    finish_rows<T, MT>(red, COLS, cluster_size, blockIdx.y, i0, j0, m, n, e);
}

template <typename T, typename K>
static int launch_rows_kernel(K kernel, int64_t m, int64_t n, int64_t k, int64_t batch, const Operand<T>& a, const Operand<T>& b, const Epilogue<T>& e, int mt, int cols,
                              size_t smem, cudaStream_t st) {
    const int64_t strips = (n + cols - 1) / cols, units = strips * ((m + mt - 1) / mt);
    int cluster = 1;                                             // up to two or three CTAs per SM (256 on 148 for 1 x 4096 x 4096), each with at least 64 of K
    while (cluster < 8 && units * batch * cluster < (int64_t)sm_count() * 2 && k > 64 * cluster) cluster *= 2;
    if (units * cluster > 0x7fffffff || batch > 65535) return (int)cudaErrorInvalidValue;
    if (smem > 40 * 1024) {
        const cudaError_t rc = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (rc != cudaSuccess) { cudaGetLastError(); return (int)rc; }
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(units * cluster), (unsigned)batch);
    cfg.blockDim = dim3(kBlock);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)cluster; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t rc = cudaLaunchKernelEx(&cfg, kernel, m, n, k, a, b, e, cluster, strips);
    if (rc != cudaSuccess) { cudaGetLastError(); return (int)rc; }
    count_launch();
    return 0;
}

template <typename T, int MT>
static int launch_rows_of(int64_t m, int64_t n, int64_t k, int64_t batch, const Operand<T>& a, const Operand<T>& b, const Epilogue<T>& e, cudaStream_t st) {
    constexpr int V = 16 / sizeof(T);
    if (b.k == 1 && b.row != 1) {
        constexpr int C = MT >= 8 ? 4 : 2;
        const bool packets = aligned16(b.p) && b.row % V == 0;
        constexpr size_t smem = (size_t)MT * kRowsChunk * sizeof(T);
        if (packets) return launch_rows_kernel<T>(rows_by_dots_kernel<T, MT, C, true>, m, n, k, batch, a, b, e, MT, kWarpsPerBlock * C, smem, st);
        return launch_rows_kernel<T>(rows_by_dots_kernel<T, MT, C, false>, m, n, k, batch, a, b, e, MT, kWarpsPerBlock * C, smem, st);
    }
    constexpr size_t piece = (size_t)MT * kRowsChunk * sizeof(T), sums = (size_t)(kWarpsPerBlock + 1) * MT * 32 * V * sizeof(T);
    constexpr size_t smem = piece > sums ? piece : sums;
    const bool packets = b.row == 1 && aligned16(b.p) && b.k % V == 0 && n % V == 0;
    if (packets) return launch_rows_kernel<T>(rows_by_columns_kernel<T, MT, true>, m, n, k, batch, a, b, e, MT, 32 * V, smem, st);
    return launch_rows_kernel<T>(rows_by_columns_kernel<T, MT, false>, m, n, k, batch, a, b, e, MT, 32 * V, smem, st);
}

template <typename T>
int launch_product_rows(int64_t m, int64_t n, int64_t k, int64_t batch, const Operand<T>& a, const Operand<T>& b, const Epilogue<T>& e, cudaStream_t st) {
    if (m == 1) return launch_rows_of<T, 1>(m, n, k, batch, a, b, e, st);
    if (m == 2) return launch_rows_of<T, 2>(m, n, k, batch, a, b, e, st);
    if (m <= 4) return launch_rows_of<T, 4>(m, n, k, batch, a, b, e, st);
    if (m <= 8 || sizeof(T) == 8) return launch_rows_of<T, 8>(m, n, k, batch, a, b, e, st);
    if constexpr (sizeof(T) == 4) return launch_rows_of<T, 16>(m, n, k, batch, a, b, e, st);
    return (int)cudaErrorInvalidValue;
}
template int launch_product_rows<float>(int64_t, int64_t, int64_t, int64_t, const Operand<float>&, const Operand<float>&, const Epilogue<float>&, cudaStream_t);
template int launch_product_rows<double>(int64_t, int64_t, int64_t, int64_t, const Operand<double>&, const Operand<double>&, const Epilogue<double>&, cudaStream_t);

}  // namespace cb200
