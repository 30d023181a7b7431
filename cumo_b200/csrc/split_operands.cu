// Operands of the tensor-core product: floats into bfloat16 planes, and the outputs that infinities and NaN reach.
#include "split_product.cuh"

#include <cuda_bf16.h>

namespace cb200 {

// a = a1 + a2 + a3 with each part the bfloat16 nearest to what the parts before it leave: 8 bits each, so that three hold
// all 24 (parts under 2^-126 are lost, which only operands under 2^-102 have).  What rounds to infinity in the first part has
// no such parts.
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

__device__ __forceinline__ float source_at(const SplitSource& s, int64_t i, int64_t j) {
    float v = s.p[i * s.row + j * s.col];
    if (s.act != kActNone) v *= activation_slope(s.pre[i * s.pre_row + j * s.pre_col], s.act);
    return v;
}

// A thread takes eight neighbouring columns: two 16-byte loads where the source allows it, one 16-byte store per plane.
// Bound by memory: 4 bytes read and 6 written per element (8 read with an activation's slope).
template <bool VEC>
__global__ void __launch_bounds__(kBlock)
split_kernel(const SplitSource s, int64_t R, int64_t C, uint16_t* planes, int64_t ld, const Marks marks) {
    const int64_t groups = ld / 8, total = R * groups;
    const int64_t plane = R * ld;
    for (int64_t f = (int64_t)blockIdx.x * kBlock + threadIdx.x; f < total; f += (int64_t)gridDim.x * kBlock) {
        const int64_t i = f / groups, j = (f - i * groups) * 8;
        float v[8];
        if (VEC && j + 8 <= C) {
            const float4* p = reinterpret_cast<const float4*>(s.p + i * s.row + j);
            const float4 x = __ldg(p), y = __ldg(p + 1);
            v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w; v[4] = y.x; v[5] = y.y; v[6] = y.z; v[7] = y.w;
            if (s.act != kActNone) {
                const float4* q = reinterpret_cast<const float4*>(s.pre + i * s.pre_row + j);
                const float4 a = __ldg(q), b = __ldg(q + 1);
                const float z[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] *= activation_slope(z[e], s.act);
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = j + e < C ? source_at(s, i, j + e) : 0.f;
        }
        uint32_t out[3][4];
        bool fine = true;
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            uint32_t a0, b0, c0, a1, b1, c1;
            const bool f0 = split3(v[e], a0, b0, c0), f1 = split3(v[e + 1], a1, b1, c1);
            fine = fine && f0 && f1;
            out[0][e / 2] = a0 | a1 << 16; out[1][e / 2] = b0 | b1 << 16; out[2][e / 2] = c0 | c1 << 16;
        }
#pragma unroll
        for (int p = 0; p < 3; ++p) *reinterpret_cast<uint4*>(planes + p * plane + i * ld + j) = make_uint4(out[p][0], out[p][1], out[p][2], out[p][3]);
        if (!fine) {
            *marks.any = 1;
            marks.row[i] = 1;
            for (int e = 0; e < 8; ++e)
                if (j + e < C && (__float_as_uint(v[e]) & 0x7fffffffu) >= 0x7f7f8000u) marks.col[j + e] = 1;
        }
    }
}

int launch_split(const SplitSource& s, int64_t R, int64_t C, uint16_t* planes, int64_t ld, const Marks& marks, cudaStream_t st) {
    const bool vec = s.col == 1 && aligned16(s.p) && s.row % 4 == 0 &&
                     (s.act == kActNone || (s.pre_col == 1 && aligned16(s.pre) && s.pre_row % 4 == 0));
    const unsigned grid = grid_for((R * (ld / 8) + kBlock - 1) / kBlock, 16);
    if (vec) split_kernel<true><<<grid, kBlock, 0, st>>>(s, R, C, planes, ld, marks);
    else split_kernel<false><<<grid, kBlock, 0, st>>>(s, R, C, planes, ld, marks);
    count_launch();
    return (int)cudaGetLastError();
}

__global__ void __launch_bounds__(kBlock)
fix_marked_kernel(int64_t m, int64_t n, int64_t k, const SplitSource a, bool a_turned, const uint8_t* a_marks, const SplitSource b, bool b_turned,
                  const uint8_t* b_marks, const int* any, const Epilogue<float> e) {
    if (*any == 0) return;
    const int64_t total = m * n;
    for (int64_t f = (int64_t)blockIdx.x * kBlock + threadIdx.x; f < total; f += (int64_t)gridDim.x * kBlock) {
        const int64_t i = f / n, j = f - i * n;
        if (!a_marks[i] && !b_marks[j]) continue;
        float acc = 0.f;
        for (int64_t c = 0; c < k; ++c) acc = fmaf(a_turned ? source_at(a, c, i) : source_at(a, i, c), b_turned ? source_at(b, c, j) : source_at(b, j, c), acc);
        finish(e, 0, i, j, acc);
    }
}

int launch_fix_marked(int64_t m, int64_t n, int64_t k, const SplitSource& a, bool a_turned, const uint8_t* a_marks, const SplitSource& b, bool b_turned,
                      const uint8_t* b_marks, const int* any, const Epilogue<float>& e, cudaStream_t st) {
    fix_marked_kernel<<<grid_for((m * n + kBlock - 1) / kBlock, 4), kBlock, 0, st>>>(m, n, k, a, a_turned, a_marks, b, b_turned, b_marks, any, e);
    count_launch();
    return (int)cudaGetLastError();
}

}  // namespace cb200
