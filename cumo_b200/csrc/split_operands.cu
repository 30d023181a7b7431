// Operands of the tensor-core product: floats into bfloat16 planes, and the outputs that infinities and NaN reach.
#include "split_product.cuh"

namespace cb200 {

__device__ __forceinline__ float source_at(const SplitSource& s, int64_t i, int64_t j) {
    float v = s.p[i * s.row + j * s.col];
    if (s.act != kActNone) v *= activation_slope(s.pre[i * s.pre_row + j * s.pre_col], s.act);
    return v;
}

// A thread takes eight neighbouring columns: two 16-byte loads where the source allows it, one 16-byte store per plane.
// Bound by memory: 4 bytes read and 6 written per element (8 read with an activation's slope); 4096 x 4096 35 us, 4.8 TB/s.
__global__ void __launch_bounds__(kBlock)
split_kernel(const SplitJobs jobs) {
    pdl_trigger();                                               // the product behind sets itself up meanwhile
    const SplitJob& job = jobs.job[blockIdx.y];
    const SplitSource& s = job.s;
    const int64_t C = job.C, ld = job.ld, groups = ld / 8, total = job.R * groups, plane = job.R * ld;
    uint16_t* planes = job.planes;
    const bool vec = s.col == 1 && (reinterpret_cast<uintptr_t>(s.p) & 15) == 0 && s.row % 4 == 0 &&
                     (s.act == kActNone || (s.pre_col == 1 && (reinterpret_cast<uintptr_t>(s.pre) & 15) == 0 && s.pre_row % 4 == 0));
    for (int64_t f = (int64_t)blockIdx.x * kBlock + threadIdx.x; f < total; f += (int64_t)gridDim.x * kBlock) {
        const int64_t i = total < 0x7fffffff ? (int64_t)((uint32_t)f / (uint32_t)groups) : f / groups, j = (f - i * groups) * 8;
        float v[8];
        if (vec && j + 8 <= C) {
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
            *job.marks.any = 1;
            job.marks.row[i] = 1;
            for (int e = 0; e < 8; ++e)
                if (j + e < C && (__float_as_uint(v[e]) & 0x7fffffffu) >= 0x7f7f8000u) job.marks.col[j + e] = 1;
        }
    }
}

int launch_split(const SplitJobs& jobs, cudaStream_t st) {
    int64_t most = 0;
    for (int i = 0; i < jobs.count; ++i) { const int64_t t = jobs.job[i].R * (jobs.job[i].ld / 8); most = t > most ? t : most; }
    split_kernel<<<dim3(grid_for((most + kBlock - 1) / kBlock, 16), (unsigned)jobs.count), kBlock, 0, st>>>(jobs);
    count_launch();
    return (int)cudaGetLastError();
}

__global__ void __launch_bounds__(kBlock)
fix_marked_kernel(const FixJobs jobs) {
    pdl_wait();                                                  // launched while the product in front of it still runs
    if (*jobs.any == 0) return;
    const FixJob& x = jobs.job[blockIdx.y];
    const int64_t total = x.m * x.n;
    for (int64_t f = (int64_t)blockIdx.x * kBlock + threadIdx.x; f < total; f += (int64_t)gridDim.x * kBlock) {
        const int64_t i = f / x.n, j = f - i * x.n;
        if (!x.a_marks[i] && !x.b_marks[j] && !(x.hot_row[i] && x.hot_col[j])) continue;
        float acc = 0.f;
        for (int64_t c = 0; c < x.k && acc == acc; ++c)          // (a NaN stays)
            acc = fmaf(x.a_turned ? source_at(x.a, c, i) : source_at(x.a, i, c), x.b_turned ? source_at(x.b, c, j) : source_at(x.b, j, c), acc);
        finish(x.e, 0, i, j, acc);
    }
}

int launch_fix_marked(const FixJobs& jobs, cudaStream_t st) {
    int64_t most = 0;
    for (int i = 0; i < jobs.count; ++i) { const int64_t t = jobs.job[i].m * jobs.job[i].n; most = t > most ? t : most; }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid_for((most + kBlock - 1) / kBlock, 2), (unsigned)jobs.count);
    cfg.blockDim = dim3(kBlock);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t rc = cudaLaunchKernelEx(&cfg, fix_marked_kernel, jobs);
    if (rc != cudaSuccess) { cudaGetLastError(); return (int)rc; }
    count_launch();
    return 0;
}

}  // namespace cb200
