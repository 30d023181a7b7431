// Single-precision products on the 16-bit tensor cores: operands held as three 16-bit parts ("planes") each.
//
// A float is the sum of three bfloat16 numbers to its last bit (8 + 8 + 8 bits, the float's own exponent range).  With
// a = a1 + a2 + a3, b alike,
//     a b = a1 b1 + (a1 b2 + a2 b1) + (a2 b2 + a1 b3 + a3 b1) + terms of 2^-24 a b and below,
// six bfloat16 products.  (Two half-precision parts would take three, but hold 22 bits only of numbers within 2^16 of the largest
// under a common power of two: rows of a matrix that are small beside the others would lose theirs.)  Products of two 16-bit
// numbers are exact in the tensor core; what it adds them into is 32 bits wide but truncates, an error that leans one way and
// grows with the number of additions (2e-8 of the accumulator each, measured).  So the large products a1 b1 have an
// accumulator of their own, which takes 64 to 256 of K -- four to 16 additions -- before it is added into registers with
// ordinary rounded additions; what truncation does to the accumulator of the small products is 2^-8 of that and less.
#pragma once

#include "linear.cuh"

#include <cuda_bf16.h>

namespace cb200 {

constexpr int kParts = 3;

// a = a1 + a2 + a3 with each part the bfloat16 nearest to what the parts before it leave: 8 bits each, so that three hold
// all 24.  (Parts under 2^-126 lose bits: products of operands that are all under 2^-112 do, 6e-7 off at 2^-114, 9e-6 at 2^-118.)
// What rounds to infinity in the first part has no such parts: false, and zeros.
__device__ __forceinline__ bool split3(float v, uint32_t& a, uint32_t& b, uint32_t& c) {
    const bool fine = (__float_as_uint(v) & 0x7fffffffu) < 0x7f7f8000u;
    if (!fine) v = 0.f;
    const __nv_bfloat16 x = __float2bfloat16_rn(v);
    const float r = v - __bfloat162float(x);
    const __nv_bfloat16 y = __float2bfloat16_rn(r);
    const __nv_bfloat16 z = __float2bfloat16_rn(r - __bfloat162float(y));
    a = __bfloat16_as_ushort(x); b = __bfloat16_as_ushort(y); c = __bfloat16_as_ushort(z);
    return fine;
}
// Two numbers' parts side by side in 32 bits each; `none` becomes NaN if one of them has no parts.
__device__ __forceinline__ void split3_pair(float u, float v, uint32_t& a, uint32_t& b, uint32_t& c, float& none) {
    auto pack = [](float lo, float hi) { const __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi); return *reinterpret_cast<const uint32_t*>(&p); };
    a = pack(u, v);
    float r = u - __uint_as_float(a << 16), s = v - __uint_as_float(a & 0xffff0000u);
    none = fmaf(r, 0.f, fmaf(s, 0.f, none));
    b = pack(r, s);
    r -= __uint_as_float(b << 16);
    s -= __uint_as_float(b & 0xffff0000u);
    c = pack(r, s);
}
// One number for which there is no leaving out: infinities and NaN are their own first part, and what only rounds to infinity is cut off.
__device__ __forceinline__ void split3_all(float v, uint32_t& a, uint32_t& b, uint32_t& c) {
    if (split3(v, a, b, c)) return;
    const uint32_t bits = __float_as_uint(v), mag = bits & 0x7fffffffu;
    a = (bits >> 16) | (mag > 0x7f800000u ? 0x40u : 0u);
    if (mag >= 0x7f800000u) return;
    const float r = v - __uint_as_float(bits & 0xffff0000u);
    const __nv_bfloat16 y = __float2bfloat16_rn(r);
    b = __bfloat16_as_ushort(y);
    c = __bfloat16_as_ushort(__float2bfloat16_rn(r - __bfloat162float(y)));
}
__device__ __forceinline__ float bf16_at(uint32_t bits) { return __uint_as_float(bits << 16); }

// A matrix of `rows` x `k` (per batch entry) as planes in global memory.  k_major: rows of k contiguous elements, ld apart;
// otherwise k rows of `rows` contiguous elements.  Plane p of batch entry b starts at (p * batch + b) * rows_or_k * ld.
struct Planes {
    uint16_t* p;
    int64_t rows, k, batch, ld;
    bool k_major;
    int64_t outer() const { return k_major ? rows : k; }
    int64_t inner() const { return k_major ? k : rows; }
};
inline int64_t planes_ld(int64_t inner) { return (inner + 7) / 8 * 8; }

// Out of a product of planes into planes (orthogonalisation): alpha * acc + beta * d.
struct PlaneEpilogue {
    float alpha, beta;
    const uint16_t* d;                  // planes of the same shape as the output, or null
    uint16_t* out;
    int64_t ld, plane;                  // elements per row; elements from one plane to the next
    int64_t batch_step;
};

// Where outputs beyond the range are marked: rows and columns of the result (see Marks).
struct Hot { uint8_t* row; uint8_t* col; int* any; };

// C = A . B^T (per batch entry), contraction over k; the result leaves through `e` (float) or `pe` (planes).  Returns a
// cudaError_t; cudaErrorNotSupported when tensor maps cannot be had, in which case nothing was launched.
// Outputs beyond the range are marked in `hot`.
int launch_split_product(const Planes& a, const Planes& b, const Epilogue<float>& e, const Hot& hot, Scratch& scratch, cudaStream_t st);
// `symmetric` says that the result is (A = B, or A and B symmetric and equal, and d symmetric): about half the tiles are computed.
int launch_split_product(const Planes& a, const Planes& b, const PlaneEpilogue& e, bool symmetric, cudaStream_t st);

// Elements that have no parts (infinities, NaN, what bfloat16 rounds to infinity) are left out of the planes and marked by
// row and by column; fix_marked() then computes the outputs they touch from the operands themselves.  So it does for outputs
// that leave the range as sums of parts: there, and just below its end, the parts' products may overflow to either side of what
// they add up to.  Those are marked by row and column of the result (`hot`); where a marked row and a marked column cross, the
// output is computed again.
struct Marks {
    uint8_t* row;
    uint8_t* col;
    int* any;
};

// v(i, j) = p[i * row + j * col], times act'(pre(i, j)) when act is not kActNone.
struct SplitSource {
    const float* p; int64_t row, col;
    const float* pre; int64_t pre_row, pre_col;
    int act;
};

// R x C sources as three bfloat16 planes each, [plane][R][ld]; up to three in one launch.
struct SplitJob {
    SplitSource s;
    int64_t R, C, ld;
    uint16_t* planes;
    Marks marks;
};
struct SplitJobs { SplitJob job[3]; int count; };
int launch_split(const SplitJobs& jobs, cudaStream_t st);

// Outputs i, j with a[i] or b[j] marked, or hot_row[i] and hot_col[j], in float from the operands: element (row, k) of A at
// (row, k) of `a`, or (k, row) if a_turned; B alike.  Returns at once on the device when nothing was marked.  Up to two products in one launch.
struct FixJob {
    int64_t m, n, k;
    SplitSource a, b;
    bool a_turned, b_turned;
    const uint8_t* a_marks;
    const uint8_t* b_marks;
    const uint8_t* hot_row;
    const uint8_t* hot_col;
    Epilogue<float> e;
};
struct FixJobs { FixJob job[2]; int count; const int* any; };
int launch_fix_marked(const FixJobs& jobs, cudaStream_t st);

// 0, or cudaErrorLaunchTimeout once a bounded wait inside a product has run out on this device (see cb200_product_status).
int product_gave_up();
// The word behind it, and its address on the current device; null when it cannot be had.
int* gave_up_word(int** dev);

}  // namespace cb200
