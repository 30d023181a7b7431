// Pieces shared by the kernels behind linalg.linear, linear_grad and orthogonalize: the epilogue of a product, the
// activations with their derivatives, and scratch memory that a captured graph may keep.
#pragma once

#include "common.cuh"

namespace cb200 {

// Order is ABI (cb200_<T>_linear_kernel_launch).
enum Activation { kActNone = 0, kActRelu, kActSilu, kActGelu, kActGeluTanh, kActSigmoid, kActTanh, kActCount };

__device__ __forceinline__ float a_exp(float x) { return expf(x); }
__device__ __forceinline__ double a_exp(double x) { return exp(x); }
__device__ __forceinline__ float a_erfc(float x) { return erfcf(x); }
__device__ __forceinline__ double a_erfc(double x) { return erfc(x); }
__device__ __forceinline__ float a_tanh(float x) { return tanhf(x); }
__device__ __forceinline__ double a_tanh(double x) { return tanh(x); }

constexpr double kSqrtHalf = 0.70710678118654752440, kTwoRootTwoOverPi = 1.59576912160573071176, kInvRootTwoPi = 0.39894228040143267794;
constexpr double kGeluCubic = 0.044715;

// gelu is z * Phi(z) with Phi from erfc, which keeps its digits in the lower tail where 1 + erf cancels; the tanh form of
// gelu is z times the logistic function of twice tanh's argument, the same value with one exponential.
template <typename T>
__device__ __forceinline__ T activate(T z, int act) {
    switch (act) {
        case kActRelu: return z > T(0) ? z : (z == z ? T(0) : z);
        case kActSilu: return z / (T(1) + a_exp(-z));
        case kActGelu: return T(0.5) * z * a_erfc(-z * T(kSqrtHalf));
        case kActGeluTanh: return z / (T(1) + a_exp(-T(kTwoRootTwoOverPi) * (z + T(kGeluCubic) * z * z * z)));
        case kActSigmoid: return T(1) / (T(1) + a_exp(-z));
        case kActTanh: return a_tanh(z);
        default: return z;
    }
}

template <typename T>
__device__ __forceinline__ T activation_slope(T z, int act) {
    switch (act) {
        case kActRelu: return z > T(0) ? T(1) : (z == z ? T(0) : z);
        case kActSilu: { const T p = T(1) / (T(1) + a_exp(-z)); return p * (T(1) + z * (T(1) - p)); }
        case kActGelu: return T(0.5) * a_erfc(-z * T(kSqrtHalf)) + z * a_exp(T(-0.5) * z * z) * T(kInvRootTwoPi);
        case kActGeluTanh: {
            const T p = T(1) / (T(1) + a_exp(-T(kTwoRootTwoOverPi) * (z + T(kGeluCubic) * z * z * z)));
            const T q = p * (T(1) - p);                                   // 0 far out, where z * z may have overflowed
            return q == T(0) ? p : p + z * q * T(kTwoRootTwoOverPi) * (T(1) + T(3 * kGeluCubic) * z * z);
        }
        case kActSigmoid: { const T p = T(1) / (T(1) + a_exp(-z)); return p * (T(1) - p); }
        case kActTanh: { const T t = a_tanh(z); return T(1) - t * t; }
        default: return T(1);
    }
}

// What happens to an element of a product on its way out: z = alpha * acc + beta * d + bias[column]; pre = z;
// y = act(z) + residual.  Steps in elements; y and pre are row-major with ld elements per row.
template <typename T>
struct Epilogue {
    T alpha, beta;
    const T* d; int64_t d_row, d_col, d_batch;
    const T* bias; int64_t bias_step;
    int act;
    const T* res; int64_t res_row, res_col;
    T* y; int64_t ld, y_batch;
    T* pre;
};

template <typename T>
__device__ __forceinline__ void finish(const Epilogue<T>& e, int64_t batch, int64_t i, int64_t j, T acc) {
    T z = e.alpha == T(1) ? acc : e.alpha * acc;
    if (e.d) z += e.beta * e.d[batch * e.d_batch + i * e.d_row + j * e.d_col];
    if (e.bias) z += e.bias[j * e.bias_step];
    const int64_t at = batch * e.y_batch + i * e.ld + j;
    if (e.pre) e.pre[at] = z;
    T y = e.act == kActNone ? z : activate(z, e.act);
    if (e.res) y += e.res[i * e.res_row + j * e.res_col];
    e.y[at] = y;
}

// Operand of a product: element (row, k) at p[batch * b + row * r + k * c].
template <typename T>
struct Operand { const T* p; int64_t row, k, batch; };

// The product on the CUDA cores: any steps, any sizes, both types.  C[i][j] = sum_k A(i, k) * B(j, k).
template <typename T>
int launch_product_cc(int64_t m, int64_t n, int64_t k, int64_t batch, const Operand<T>& a, const Operand<T>& b, const Epilogue<T>& e, cudaStream_t st);

// The same with few rows, where reading B once is what it costs: m up to a few dozen, any steps.
template <typename T>
int launch_product_rows(int64_t m, int64_t n, int64_t k, int64_t batch, const Operand<T>& a, const Operand<T>& b, const Epilogue<T>& e, cudaStream_t st);

// Scratch of one call.  Outside a capture it comes from the pool callback and goes back to it when the call returns (the
// next taker queues behind on the same stream).  Inside a capture it is an allocation node of the graph itself: two graphs
// never share it, nor does an eager call that runs while one of them replays.
struct Scratch {
    explicit Scratch(cudaStream_t stream) : st(stream) {
        cudaStreamCaptureStatus c = cudaStreamCaptureStatusNone;
        if (cudaStreamIsCapturing(st, &c) != cudaSuccess) { cudaGetLastError(); c = cudaStreamCaptureStatusNone; }
        captured = c == cudaStreamCaptureStatusActive;
    }
    ~Scratch() {
        for (int i = 0; i < count; ++i) {
            if (captured) cudaFreeAsync(blocks[i], st);
            else cumo_cuda_runtime_free(blocks[i]);
        }
    }
    Scratch(const Scratch&) = delete;
    Scratch& operator=(const Scratch&) = delete;
    char* take(size_t bytes) {
        if (count == kMost) return nullptr;
        void* p = nullptr;
        if (captured) { if (cudaMallocAsync(&p, bytes ? bytes : 1, st) != cudaSuccess) { cudaGetLastError(); p = nullptr; } }
        else p = cumo_cuda_runtime_malloc(bytes);
        if (p) blocks[count++] = static_cast<char*>(p);
        return static_cast<char*>(p);
    }
    static constexpr int kMost = 16;
    cudaStream_t st;
    bool captured;
    char* blocks[kMost];
    int count = 0;
};

}  // namespace cb200
