// The tensor-core product of split operands (split_product.cuh says what the parts are): tcgen05 with tensor-memory
// accumulators, operands brought by the tensor memory accelerator.
//
// Roles of the 12 warps of a CTA:
//   warp 0      one thread issues the TMA loads of a K-block (64 elements of K, all planes of both operands) into a ring of
//               128-byte-swizzled stages
//   warp 1      allocates tensor memory; one thread issues the tcgen05.mma's, the large products (first part x first part)
//               into one accumulator, all the small ones into another
//   warps 2, 3  idle; this warpgroup gives most of its registers to the others
//   warps 4..11 epilogue: after every chunk of K-blocks they add the large products' accumulator to registers (two take turns
//               where tensor memory has room, else the next block's small products run meanwhile); at the end of a tile the
//               small ones follow and the sums pass through a small shared-memory tile per warp, so that global memory is read
//               and written along rows
// What bounds it: at 8192^3 3257 cycles per K-block of 3072 tensor cycles (counted in the issuing thread), 4.4 ms, the power limit
// (1480 TFLOP/s of bf16 products).  At 4096^3 503 us, the tensor pipe 88 % busy, 632 MB read from memory and 4.2 GB through L2;
// into planes 571 us and 74 %: writing a tile takes longer than the first chunk of the next one hides.  Reading an accumulator
// takes some 57 bytes per cycle, which is why a chunk is as long as truncation allows.  A 128 x 64 tile's K-block takes about 2500
// cycles of 1152 tensor cycles (8 x 256 x 1024 against x 256); what it waits for has not been established.
// With CG = 2 two CTAs of a cluster share a 256 x 256 tile: each loads its 128 rows of A and its half of B, the first CTA
// issues the instructions for both.  Shared memory feeds 64 bytes per cycle to the tensor cores then, instead of the 128 of
// a 128 x 128 tile (its limit), and each operand byte loaded is used twice as often.  Small problems take 128-row tiles of one
// CTA, 128 or 64 columns wide.  Every wait is bounded; when one runs out the kernel raises a word in host memory that the next
// call finds.
#include "split_product.cuh"
#include "tc_common.cuh"
#include "tile_tma.cuh"

#include <atomic>
#include <mutex>

namespace cb200 {

constexpr int kSpThreads = 384;                 // a warpgroup for loads and products, two for the epilogue
constexpr int kSpKB = 64;                       // K per stage: one 128-byte swizzle row of 16-bit elements
constexpr int kSpStageCols = 33;                // epilogue tile: 32 x 32 floats, rows padded by one

template <int CG, int BN>
struct SplitShape {
    static constexpr int kBRows = BN / CG;                               // rows of B a CTA loads
    static constexpr int kABytes = 128 * 128, kBBytes = kBRows * 128;    // per plane
    static constexpr int kStageBytes = kParts * (kABytes + kBBytes);
    static constexpr int kEpilogueBytes = 8 * 32 * kSpStageCols * 4;
    static constexpr int kStages = (232448 - 1024 - kEpilogueBytes) / kStageBytes < 4 ? (232448 - 1024 - kEpilogueBytes) / kStageBytes : 4;
    static constexpr int kMains = BN == 256 ? 1 : 2;                     // accumulators of large products, taking turns where there is room
    static constexpr uint32_t kTmemCols = BN == 64 ? 256 : 512;          // kMains + 1 accumulators of BN columns, a power of two
    static constexpr size_t kSmem = (size_t)kStages * kStageBytes + kEpilogueBytes + 256;
    static_assert(kStages >= 2, "two stages at least");
};

struct SplitArgs {
    int64_t m, n;
    int kblocks, chunk;                         // K-blocks; how many of them the large products' accumulator takes
    int64_t tiles_m, tiles_n, n_tiles;          // n_tiles counts all batch entries
    int64_t batch;
    int a_k_major, b_k_major;
    int splits, per_split;                      // K cut into so many pieces of so many K-blocks, each to an output of its own
    int symmetric;                              // square tiles on and above the diagonal; what lies above is written to both sides
    uint32_t idesc;
    int* gave_up;
};

__device__ __forceinline__ uint32_t cluster_rank() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ void cluster_sync_all() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t in_cta(uint32_t saddr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(saddr), "r"(rank));
    return r;
}

template <int CG>
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x0, int x1, int x2) {
    if constexpr (CG == 1)
        asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
                     ::"r"(dst), "l"(map), "r"(bar), "r"(x0), "r"(x1), "r"(x2) : "memory");
    else
        asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
                     ::"r"(dst), "l"(map), "r"(bar), "r"(x0), "r"(x1), "r"(x2) : "memory");
}

template <int CG>
__device__ __forceinline__ void split_commit(uint64_t* bar) {
    if constexpr (CG == 1)
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
    else
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                     ::"r"(smem_u32(bar)), "h"((uint16_t)3) : "memory");
}

// Bounded waits that let the hardware hold the thread until the phase ends (at most 2 microseconds a try: half a second in all):
// an accumulator's turn is under a microsecond, and the sleeping poll of tc_common.cuh wakes too late for it.
constexpr uint32_t kTries = 1u << 18;
template <bool PAIR>
__device__ __forceinline__ bool split_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
    const uint32_t addr = smem_u32(bar);
    for (uint32_t t = 0; t < kTries; ++t) {
        uint32_t done;
        if constexpr (PAIR)                                      // barriers that the other CTA of the pair arrives at
            asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, %3;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                         : "=r"(done) : "r"(addr), "r"(parity), "r"(2000u) : "memory");
        else
            asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                         : "=r"(done) : "r"(addr), "r"(parity), "r"(2000u) : "memory");
        if (done) return true;
        if ((t & 63u) == 63u && *abort_flag) return false;
    }
    *abort_flag = 1;
    return false;
}

// ---- issuing the products -----------------------------------------------------------------------------------------------
// One thread issues them all, so what it computes per instruction is time the tensor cores wait (measured: building both
// 64-bit descriptors each time made every instruction take 130 to 190 cycles, whatever its shape).  A descriptor's upper half is
// constant and its lower half a stage's base plus an offset known at compile time: the layouts are template arguments.
//   K-major: rows of 128 bytes, 16 of K are 32 bytes on.  MN-major: 8 rows of k (1024 bytes) per group, 16 of K are 2048
//   bytes on, the next 64 elements of the row axis 8192 (the leading byte offset, in the lower half).
constexpr uint32_t kDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);      // stride byte offset, version, 128-byte swizzle
template <bool K_MAJOR>
__device__ __forceinline__ uint32_t desc_low(uint32_t saddr) { return ((saddr & 0x3ffffu) >> 4) | ((K_MAJOR ? 1u : 8192u >> 4) << 16); }

template <int CG, bool FRESH>
__device__ __forceinline__ void mma_f16(uint32_t d_tmem, uint32_t a_low, uint32_t b_low, uint32_t idesc) {
    const uint64_t da = (uint64_t)kDescHigh << 32 | a_low, db = (uint64_t)kDescHigh << 32 | b_low;
    if constexpr (CG == 1)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                     ::"r"(d_tmem), "l"(da), "l"(db), "r"(idesc), "n"(FRESH ? 0 : 1) : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                     ::"r"(d_tmem), "l"(da), "l"(db), "r"(idesc), "n"(FRESH ? 0 : 1) : "memory");
}

// The large product of a stage (MAIN) or all its small ones, 64 of K; FRESH: the first instruction starts the accumulator anew.
template <int CG, int A_BYTES, int B_BYTES, bool AK, bool BK, bool MAIN, bool FRESH>
__device__ __forceinline__ void issue_stage(uint32_t sa, uint32_t sb, uint32_t d_tmem, uint32_t idesc) {
    constexpr int kTerms = 6;
    constexpr int ta[kTerms] = {2, 0, 1, 1, 0, 0};
    constexpr int tb[kTerms] = {0, 2, 1, 0, 1, 0};
    const uint32_t a0 = desc_low<AK>(sa), b0 = desc_low<BK>(sb);
#pragma unroll
    for (int term = MAIN ? kTerms - 1 : 0; term < (MAIN ? kTerms : kTerms - 1); ++term)
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
            const uint32_t a = a0 + ((ta[term] * A_BYTES + ks * (AK ? 32 : 2048)) >> 4), b = b0 + ((tb[term] * B_BYTES + ks * (BK ? 32 : 2048)) >> 4);
            if (FRESH && term == (MAIN ? kTerms - 1 : 0) && ks == 0) mma_f16<CG, true>(d_tmem, a, b, idesc);
            else mma_f16<CG, false>(d_tmem, a, b, idesc);
        }
}
template <int CG, int A_BYTES, int B_BYTES, bool MAIN, bool FRESH>
__device__ __forceinline__ void issue(int layout, uint32_t sa, uint32_t sb, uint32_t d_tmem, uint32_t idesc) {
    switch (layout) {                                            // bit 0: A K-major, bit 1: B K-major
        case 0: issue_stage<CG, A_BYTES, B_BYTES, false, false, MAIN, FRESH>(sa, sb, d_tmem, idesc); break;
        case 1: issue_stage<CG, A_BYTES, B_BYTES, true, false, MAIN, FRESH>(sa, sb, d_tmem, idesc); break;
        case 2: issue_stage<CG, A_BYTES, B_BYTES, false, true, MAIN, FRESH>(sa, sb, d_tmem, idesc); break;
        default: issue_stage<CG, A_BYTES, B_BYTES, true, true, MAIN, FRESH>(sa, sb, d_tmem, idesc); break;
    }
}

// Marks a piece of the result that holds a number beyond the range (out of line: hardly ever called, and code in the way costs
// its fetching).
__device__ __noinline__ void mark_piece(const Hot hot, int64_t i0, int rows, int64_t j0, int cols) {
    for (int r = 0; r < rows; ++r) hot.row[i0 + r] = 1;
    for (int c = 0; c < cols; ++c) hot.col[j0 + c] = 1;
    *hot.any = 1;
}

// Out: how a finished 32-row x 32-column piece leaves shared memory.  Loads are issued ahead of the stores that they might
// alias, several 16-byte packets per lane; rows of the piece are padded by one float, which keeps every access below free of
// bank conflicts.  The float form:
struct FloatOut {
    static constexpr bool kIterated = false;
    Epilogue<float> e;
    Hot hot;                           // (a piece of K that leaves the range marks what it is added to)
    bool packets;                      // y (and residual) take 16-byte accesses
    struct Ahead {};
    __device__ __forceinline__ void ahead(Ahead&, int, int64_t, int64_t, int64_t, int64_t, int64_t) const {}
    __device__ __forceinline__ void piece(float* tile, int lane, int64_t batch, int64_t i0, int64_t j0, int64_t m, int64_t n, bool, Ahead&) const {
        const int rows = m - i0 < 32 ? (int)(m - i0) : 32;
        float none = 0.f;                                         // NaN once a sum is not finite, then the whole piece is marked
        const int64_t y0 = batch * e.y_batch + i0 * e.ld + j0;
        const bool whole = packets && rows == 32 && j0 + 32 <= n;
        if (e.bias || e.pre || e.act != kActNone) {
            const int64_t j = j0 + lane;
            if (j < n) {
                const float bias = e.bias ? e.bias[j * e.bias_step] : 0.f;
                float* pre = e.pre ? e.pre + y0 + lane : nullptr;
                float* t = tile + lane;
#pragma unroll 2
                for (int r = 0; r < rows; ++r, t += kSpStageCols) {
                    float z = *t;
                    none = fmaf(z, 0.f, none);
                    if (e.bias) z += bias;
                    if (pre) { *pre = z; pre += e.ld; }
                    if (e.act != kActNone) z = activate(z, e.act);
                    *t = z;
                }
            }
            __syncwarp();
        }
        if (whole) {
            const int r0 = lane >> 3, c0 = (lane & 7) * 4;
#pragma unroll 1
            for (int h = 0; h < 32; h += 16) {
                float4 res[4];
                if (e.res)
#pragma unroll
                    for (int q = 0; q < 4; ++q) res[q] = __ldcs(reinterpret_cast<const float4*>(e.res + (i0 + h + q * 4 + r0) * e.res_row + j0 + c0));
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int r = h + q * 4 + r0;
                    const float* t = tile + r * kSpStageCols + c0;
                    float4 v = make_float4(t[0], t[1], t[2], t[3]);
                    none = fmaf((v.x + v.y) + (v.z + v.w), 0.f, none);
                    if (e.res) { v.x += res[q].x; v.y += res[q].y; v.z += res[q].z; v.w += res[q].w; }
                    *reinterpret_cast<float4*>(e.y + y0 + r * e.ld + c0) = v;
                }
            }
            if (none != 0.f) mark_piece(hot, i0, rows, j0, 32);
            return;
        }
        if (j0 + lane >= n) return;
        // one column per lane, eight rows in flight
        float* y = e.y + y0 + lane;
        const float* res = e.res ? e.res + i0 * e.res_row + (j0 + lane) * e.res_col : nullptr;
#pragma unroll 1
        for (int h = 0; h < rows; h += 8) {
            float v[8], w[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                v[q] = tile[(h + q) * kSpStageCols + lane];
                none = fmaf(v[q], 0.f, none);
                w[q] = res && h + q < rows ? res[q * e.res_row] : 0.f;
            }
            if (res) res += 8 * e.res_row;
#pragma unroll
            for (int q = 0; q < 8; ++q)
                if (h + q < rows) y[q * e.ld] = e.res ? v[q] + w[q] : v[q];
            y += 8 * e.ld;
        }
        if (none != 0.f) mark_piece(hot, i0, rows, j0, n - j0 < 32 ? (int)(n - j0) : 32);
    }
};

// ... and the form that leaves as planes (ld is a multiple of 8, so packets are always aligned; columns between n and ld are
// padding that nothing reads).
struct PlaneOut {
    static constexpr bool kIterated = true;      // its results go into further products
    PlaneEpilogue e;
    struct Ahead { uint4 part[kParts]; };
    // eight rows of the piece's part of d, requested before they are needed
    __device__ __forceinline__ void ahead(Ahead& d, int lane, int64_t batch, int64_t i0, int64_t j0, int64_t m, int64_t) const {
        const int r0 = lane >> 2, c0 = (lane & 3) * 8;
        if (!e.d || j0 + c0 >= e.ld || i0 + r0 >= m) return;
        const uint16_t* p = e.d + batch * e.batch_step + (i0 + r0) * e.ld + j0 + c0;
#pragma unroll
        for (int q = 0; q < kParts; ++q) d.part[q] = *reinterpret_cast<const uint4*>(p + q * e.plane);
    }
    __device__ __forceinline__ void piece(float* tile, int lane, int64_t batch, int64_t i0, int64_t j0, int64_t m, int64_t n, bool mirror, Ahead& d) const {
        const int r0 = lane >> 2, c0 = (lane & 3) * 8;
        const int64_t at0 = batch * e.batch_step + (i0 + r0) * e.ld + j0 + c0;
        const bool here = j0 + c0 < e.ld;
#pragma unroll 1
        for (int q = 0; q < 4; ++q) {
            const bool live = here && i0 + q * 8 + r0 < m;
            float* t = tile + (q * 8 + r0) * kSpStageCols + c0;
            Ahead cur = d;
            if (q < 3) ahead(d, lane, batch, i0 + (q + 1) * 8, j0, m, n);
            float v[8];
            if (live) {
#pragma unroll
                for (int x = 0; x < 8; ++x) v[x] = t[x] * e.alpha;
                if (e.d) {
                    const uint32_t* part[kParts];
#pragma unroll
                    for (int w = 0; w < kParts; ++w) part[w] = reinterpret_cast<const uint32_t*>(&cur.part[w]);
#pragma unroll
                    for (int x = 0; x < 4; ++x) {                // smallest part first: the sum is the number itself
                        float lo = bf16_at(part[kParts - 1][x]), hi = __uint_as_float(part[kParts - 1][x] & 0xffff0000u);
#pragma unroll
                        for (int w = kParts - 2; w >= 0; --w) { lo += bf16_at(part[w][x]); hi += __uint_as_float(part[w][x] & 0xffff0000u); }
                        v[2 * x] = fmaf(e.beta, lo, v[2 * x]);
                        v[2 * x + 1] = fmaf(e.beta, hi, v[2 * x + 1]);
                    }
                }
            }
            if (!live) continue;
            store(v, at0 + q * 8 * e.ld);
            if (mirror)
#pragma unroll
                for (int x = 0; x < 8; ++x) t[x] = v[x];
        }
        if (!mirror) return;
        __syncwarp();
        // the same piece turned: row j0 + r, columns i0 + c ..
#pragma unroll 1
        for (int r = r0; r < 32; r += 8) {
            if (j0 + r >= n || i0 + c0 >= e.ld) continue;
            float v[8];
#pragma unroll
            for (int x = 0; x < 8; ++x) v[x] = tile[(c0 + x) * kSpStageCols + r];
            store(v, batch * e.batch_step + (j0 + r) * e.ld + i0 + c0);
        }
    }
    __device__ __forceinline__ void store(const float (&v)[8], int64_t at) const {
        uint32_t out[kParts][4];
        float none = 0.f;                                        // NaN once a number has no parts
#pragma unroll
        for (int x = 0; x < 4; ++x) split3_pair(v[2 * x], v[2 * x + 1], out[0][x], out[1][x], out[2][x], none);
        if (none != 0.f) {
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                uint32_t a0, b0, c0, a1, b1, c1;
                split3_all(v[2 * x], a0, b0, c0);
                split3_all(v[2 * x + 1], a1, b1, c1);
                out[0][x] = a0 | a1 << 16; out[1][x] = b0 | b1 << 16; out[2][x] = c0 | c1 << 16;
            }
        }
#pragma unroll
        for (int w = 0; w < kParts; ++w) *reinterpret_cast<uint4*>(e.out + at + w * e.plane) = make_uint4(out[w][0], out[w][1], out[w][2], out[w][3]);
    }
};

template <int CG, int BN, typename Out>
__global__ void __launch_bounds__(kSpThreads, 1)
split_product_kernel(const SplitArgs g, const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const Out out) {
    using S = SplitShape<CG, BN>;
    extern __shared__ __align__(1024) char smem_raw[];
    char* base = smem_raw;
    float* pieces = reinterpret_cast<float*>(base + S::kStages * S::kStageBytes);
    uint64_t* bars = reinterpret_cast<uint64_t*>(base + S::kStages * S::kStageBytes + S::kEpilogueBytes);
    uint64_t* full = bars;                          // [4] TMA -> MMA
    uint64_t* empty = bars + 4;                     // [4] MMA -> TMA
    uint64_t* main_full = bars + 8;                 // [2] MMA -> epilogue
    uint64_t* main_empty = bars + 10;               // [2] epilogue -> MMA, 8 warps of each CTA
    uint64_t* cross_full = bars + 12;
    uint64_t* cross_empty = bars + 13;
    uint64_t* drain = bars + 14;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 15);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t rank = CG == 2 ? cluster_rank() : 0;
    const bool misplaced = (smem_u32(base) & 1023u) != 0;       // the same in every CTA; nothing is launched into it then
    if (tid == 32) {                                            // the first loads do not wait for their descriptors then
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_a) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_b) : "memory");
    }
    if (tid == 0) {
        for (int i = 0; i < 4; ++i) { mbar_init(full + i, 1); mbar_init(empty + i, 1); }
        for (int i = 0; i < 2; ++i) { mbar_init(main_full + i, 1); mbar_init(main_empty + i, 8 * CG); }
        mbar_init(cross_full, 1);
        mbar_init(cross_empty, 8 * CG);
        mbar_init(drain, 1);
        abort_flag[0] = misplaced ? 1 : 0;
        abort_flag[1] = 0;                                       // never set: what the last waits poll
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    if (warp == 1) {
        if constexpr (CG == 1) {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(S::kTmemCols) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(S::kTmemCols) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if constexpr (CG == 2) cluster_sync_all();                   // the peer's barriers exist before anything arrives at them
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem_base = *tmem_slot;
    // Launched while the kernel in front of it may still run (so that launch and set-up cost nothing between the products of a
    // chain): from here on its results are read, and the kernel behind may be launched in turn.
    pdl_wait();
    pdl_trigger();

    const int64_t cluster = blockIdx.x / CG, clusters = gridDim.x / CG;
    const int64_t my_tiles = misplaced || cluster >= g.n_tiles ? 0 : (g.n_tiles - cluster + clusters - 1) / clusters;
    // bands of eight tile rows, walked column by column: the tiles in flight share rows of A and columns of B in L2
    auto tile_of = [&](int64_t t, int64_t* batch, int64_t* i0, int64_t* j0, int* piece) {
        int64_t f = cluster + t * clusters;
        *piece = (int)(f % g.splits);
        f /= g.splits;
        const int64_t per = g.symmetric ? g.tiles_m * (g.tiles_m + 1) / 2 : g.tiles_m * g.tiles_n;
        *batch = f / per;
        f -= *batch * per;
        if (g.symmetric) {                                       // column by column: tile column c holds rows 0 .. c
            int64_t c = (int64_t)((sqrtf(8.f * (float)f + 1.f) - 1.f) * 0.5f);
            while (c * (c + 1) / 2 > f) --c;
            while ((c + 1) * (c + 2) / 2 <= f) ++c;
            *j0 = c * BN;
            *i0 = (f - c * (c + 1) / 2) * (128 * CG) + rank * 128;
            return;
        }
        const int64_t band = f / (8 * g.tiles_n);
        const int64_t height = g.tiles_m - band * 8 < 8 ? g.tiles_m - band * 8 : 8;
        f -= band * 8 * g.tiles_n;
        *j0 = (f / height) * BN;
        *i0 = (band * 8 + f % height) * (128 * CG) + rank * 128;
    };

    // 384 threads of 168 registers: 128 keep 56 each, which leaves 224 for each of the other 256 (56 + 2 * 224 = 3 * 168)
    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        if (warp == 0) {
            // ---- loads ------------------------------------------------------------------------------
            if (lane == 0) {
                uint32_t it = 0;
                bool ok = true;
                for (int64_t t = 0; t < my_tiles && ok; ++t) {
                    int64_t batch, i0, j0;
                    int piece;
                    tile_of(t, &batch, &i0, &j0, &piece);
                    j0 += rank * S::kBRows;
                    const int end = (piece + 1) * g.per_split < g.kblocks ? (piece + 1) * g.per_split : g.kblocks;
                    for (int kb = piece * g.per_split; kb < end; ++kb, ++it) {
                        const uint32_t slot = it % S::kStages;
                        if (!split_wait<false>(empty + slot, ((it / S::kStages) & 1u) ^ 1u, abort_flag)) { ok = false; break; }
                        if (rank == 0) mbar_expect_tx(full + slot, (uint32_t)(S::kStageBytes * CG));
                        const uint32_t bar = CG == 2 ? in_cta(smem_u32(full + slot), 0) : smem_u32(full + slot);
                        uint32_t dst = smem_u32(base + slot * S::kStageBytes);
                        const int k0 = kb * kSpKB;
#pragma unroll
                        for (int p = 0; p < kParts; ++p) {
                            const int z = (int)(p * g.batch + batch);
                            if (g.a_k_major) tma_load_3d<CG>(dst, &map_a, bar, k0, (int)i0, z);
                            else { tma_load_3d<CG>(dst, &map_a, bar, (int)i0, k0, z); tma_load_3d<CG>(dst + 8192, &map_a, bar, (int)i0 + 64, k0, z); }
                            dst += S::kABytes;
                        }
#pragma unroll
                        for (int p = 0; p < kParts; ++p) {
                            const int z = (int)(p * g.batch + batch);
                            if (g.b_k_major) tma_load_3d<CG>(dst, &map_b, bar, k0, (int)j0, z);
                            else {
#pragma unroll
                                for (int h = 0; h < S::kBRows / 64; ++h) tma_load_3d<CG>(dst + h * 8192, &map_b, bar, (int)j0 + h * 64, k0, z);
                            }
                            dst += S::kBBytes;
                        }
                    }
                }
                if (!ok) for (int i = 0; i < 1000; ++i) __nanosleep(1000);      // gave up: copies still in flight land before the CTA leaves
            }
            __syncwarp();
        } else if (warp == 1) {
            // ---- products ---------------------------------------------------------------------------
            if (lane == 0 && rank == 0) {
                uint32_t it = 0, item = 0;
                bool ok = true;
                const int layout = (g.a_k_major ? 1 : 0) | (g.b_k_major ? 2 : 0);
                for (int64_t t = 0; t < my_tiles && ok; ++t) {
                    const int piece = (int)((cluster + t * clusters) % g.splits);
                    const int begin = piece * g.per_split, end = (piece + 1) * g.per_split < g.kblocks ? (piece + 1) * g.per_split : g.kblocks;
                    int in_chunk = 0;
                    for (int kb = begin; kb < end; ++kb, ++it) {
                        const uint32_t slot = it % S::kStages;
                        if (!split_wait<false>(full + slot, (it / S::kStages) & 1u, abort_flag)) { ok = false; break; }
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                        const uint32_t sa = smem_u32(base + slot * S::kStageBytes), sb = sa + kParts * S::kABytes;
                        // a tile's first block starts with the large products, whose accumulator the epilogue hands back first
                        constexpr uint32_t kCross = S::kMains * BN;
                        const uint32_t which = item % S::kMains, turn = item / S::kMains;
                        if (kb > begin) issue<CG, S::kABytes, S::kBBytes, false, false>(layout, sa, sb, tmem_base + kCross, g.idesc);
                        if (in_chunk == 0) {
                            if (!split_wait<CG == 2>(main_empty + which, (turn & 1u) ^ 1u, abort_flag)) { ok = false; break; }
                            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                        }
                        if (in_chunk == 0) issue<CG, S::kABytes, S::kBBytes, true, true>(layout, sa, sb, tmem_base + which * BN, g.idesc);
                        else issue<CG, S::kABytes, S::kBBytes, true, false>(layout, sa, sb, tmem_base + which * BN, g.idesc);
                        if (kb == begin) {
                            if (!split_wait<CG == 2>(cross_empty, ((uint32_t)t & 1u) ^ 1u, abort_flag)) { ok = false; break; }
                            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                            issue<CG, S::kABytes, S::kBBytes, false, true>(layout, sa, sb, tmem_base + kCross, g.idesc);
                        }
                        split_commit<CG>(empty + slot);
                        if (++in_chunk == g.chunk || kb + 1 == end) { split_commit<CG>(main_full + which); in_chunk = 0; ++item; }
                    }
                    if (ok) split_commit<CG>(cross_full);
                }
                // what was issued finishes before tensor memory is freed, whatever happened above
                if constexpr (CG == 1) asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(drain)) : "memory");
                else asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(drain)) : "memory");
                split_wait<false>(drain, 0u, abort_flag + 1);
            }
            __syncwarp();
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
        // ---- epilogue ---------------------------------------------------------------------------
        const int ew = warp - 4;                                   // 0..7
        const uint32_t quarter = (uint32_t)(warp & 3);             // the 32 lanes of tensor memory this warp may read
        const int half = ew >> 2;                                  // which half of the columns
        constexpr int kCols = BN / 2;
        float* piece = pieces + ew * 32 * kSpStageCols;
        float sum[kCols];
        uint32_t item = 0;
        bool ok = true;
        for (int64_t t = 0; t < my_tiles && ok; ++t) {
            int64_t batch, i0, j0;
            int part;
            tile_of(t, &batch, &i0, &j0, &part);
            const int blocks = (part + 1) * g.per_split < g.kblocks ? g.per_split : g.kblocks - part * g.per_split;
            const uint32_t chunks = (uint32_t)((blocks + g.chunk - 1) / g.chunk);
#pragma unroll
            for (int x = 0; x < kCols; ++x) sum[x] = 0.f;
            const int64_t row0 = i0 + (int64_t)quarter * 32, col0 = j0 + half * kCols, in = g.splits > 1 ? part : batch;
            typename Out::Ahead ahead;
            if (row0 < g.m) out.ahead(ahead, lane, in, row0, col0, g.m, g.n);
            // the chunks of large products, then the small ones
#pragma unroll 1
            for (uint32_t c = 0; c <= chunks; ++c) {
                const bool cross = c == chunks;
                const uint32_t which = item % S::kMains, turn = item / S::kMains;
                uint64_t* bar = cross ? cross_full : main_full + which;
                if (!__all_sync(0xffffffffu, split_wait<false>(bar, (cross ? (uint32_t)t : turn) & 1u, abort_flag))) { ok = false; break; }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint32_t taddr = tmem_base + (cross ? S::kMains : which) * (uint32_t)BN + (uint32_t)(half * kCols) + ((quarter * 32u) << 16);
                // 16 columns are added while the next 16 are on their way
                uint32_t ra[16], rb[16];
                tmem_ld16(taddr, ra);
                tmem_ld_wait(ra);
#pragma unroll
                for (int q = 0; q < kCols / 16; q += 2) {
                    tmem_ld16(taddr + (q + 1) * 16u, rb);
#pragma unroll
                    for (int x = 0; x < 16; ++x) sum[q * 16 + x] += __uint_as_float(ra[x]);
                    tmem_ld_wait(rb);
                    if (q + 2 < kCols / 16) tmem_ld16(taddr + (q + 2) * 16u, ra);
#pragma unroll
                    for (int x = 0; x < 16; ++x) sum[q * 16 + 16 + x] += __uint_as_float(rb[x]);
                    if (q + 2 < kCols / 16) tmem_ld_wait(ra);
                }
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) {
                    uint64_t* back = cross ? cross_empty : main_empty + which;
                    if constexpr (CG == 1) mbar_arrive(back);
                    else asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(in_cta(smem_u32(back), 0)) : "memory");
                }
                if (!cross) ++item;
            }
            if (!ok) break;
            // (one copy of the code that writes a piece: run once per piece, it costs the fetching of its instructions)
#pragma unroll 1
            for (int q = 0; q < kCols / 32; ++q) {
#pragma unroll
                for (int w = 0; w < kCols / 32; ++w)
                    if (w == q) {
#pragma unroll
                        for (int x = 0; x < 32; ++x) piece[lane * kSpStageCols + x] = sum[w * 32 + x];
                    }
                __syncwarp();
                if (row0 < g.m) {
                    out.piece(piece, lane, in, row0, col0 + q * 32, g.m, g.n, g.symmetric && i0 / (128 * CG) != j0 / BN, ahead);
                    if (q + 1 < kCols / 32) out.ahead(ahead, lane, in, row0, col0 + (q + 1) * 32, g.m, g.n);
                }
                __syncwarp();
            }
        }
    }

    // ---- wind-down: everyone meets here, also after a bounded wait ran out ----------------------
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if constexpr (CG == 2) cluster_sync_all();                     // neither CTA leaves while the other may still arrive at its barriers
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (warp == 1) {
        if constexpr (CG == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(S::kTmemCols) : "memory");
        else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(S::kTmemCols) : "memory");
    }
    if ((abort_flag[0] | abort_flag[1]) && tid == 0) *reinterpret_cast<volatile int*>(g.gave_up) = 1;
}

// ---- host ---------------------------------------------------------------------------------------------------------------
// One word of mapped host memory per process that a kernel sets when a bounded wait ran out; read without synchronising.
static std::atomic<int*> word_on_host{nullptr};
int* gave_up_word(int** dev) {
    static std::mutex mu;
    int* host = word_on_host.load(std::memory_order_acquire);
    static int* on_device[64] = {};
    int d = 0;
    if (dev && cudaGetDevice(&d) != cudaSuccess) return nullptr;
    if (d < 0 || d >= 64) return nullptr;
    if (host && !dev) return host;
    std::lock_guard<std::mutex> lock(mu);
    host = word_on_host.load(std::memory_order_acquire);
    if (!host || !on_device[d]) {
        cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;       // the first call may come during a capture
        cudaThreadExchangeStreamCaptureMode(&mode);
        void* p = host;
        cudaError_t rc = cudaSuccess;
        if (!host) rc = cudaHostAlloc(&p, sizeof(int), cudaHostAllocMapped | cudaHostAllocPortable);
        if (rc == cudaSuccess && !host) { host = static_cast<int*>(p); *host = 0; word_on_host.store(host, std::memory_order_release); }
        void* q = nullptr;
        if (rc == cudaSuccess && dev) rc = cudaHostGetDevicePointer(&q, host, 0);
        cudaThreadExchangeStreamCaptureMode(&mode);
        if (rc != cudaSuccess) { cudaGetLastError(); return nullptr; }
        if (dev) on_device[d] = static_cast<int*>(q);
    }
    if (dev) *dev = on_device[d];
    return host;
}

int product_gave_up() {
    const int* w = word_on_host.load(std::memory_order_acquire);     // (none yet: nothing that waits has been launched)
    return w && *const_cast<const volatile int*>(w) ? (int)cudaErrorLaunchTimeout : 0;
}

static bool planes_map(CUtensorMap* map, const Planes& x, int box_rows) {
    TensorMapEncodeFn enc = tensor_map_encoder();
    if (!enc || !aligned16(x.p) || x.ld % 8 != 0) return false;
    if (x.inner() > (1LL << 31) - 1024 || x.outer() > (1LL << 31) - 1024 || kParts * x.batch > 0x7fffffff) return false;
    cuuint64_t dim[3] = {(cuuint64_t)x.inner(), (cuuint64_t)x.outer(), (cuuint64_t)(kParts * x.batch)};
    cuuint64_t stride[2] = {(cuuint64_t)x.ld * 2, (cuuint64_t)(x.outer() * x.ld * 2)};
    cuuint32_t box[3] = {64, (cuuint32_t)(x.k_major ? box_rows : kSpKB), 1};
    cuuint32_t estr[3] = {1, 1, 1};
    return enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, x.p, dim, stride, box, estr,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

static std::atomic<unsigned long long> launched_tiles[3][2];         // 256, 128, 64 columns; whole, one side of the diagonal

template <int CG, int BN, typename Out>
static int launch_shape(const Planes& a, const Planes& b, const Out& out, bool symmetric, int splits, cudaStream_t st) {
    using S = SplitShape<CG, BN>;
    SplitArgs g;
    memset(&g, 0, sizeof g);
    g.m = a.rows; g.n = b.rows; g.batch = a.batch;
    g.kblocks = (int)((a.k + kSpKB - 1) / kSpKB);
    g.tiles_m = (a.rows + 128 * CG - 1) / (128 * CG);
    g.tiles_n = (b.rows + BN - 1) / BN;
// K-blocks to an accumulator: four, a fraction of a rounding of what a single layer's product is good to.  Products whose
    // errors add up over an iteration take fewer where tiles are narrow, because there are few: reading an accumulator costs little
    // there and hides behind the other one.
    g.chunk = !Out::kIterated || (BN == 256 && g.kblocks > 4) ? 4 : BN == 128 && g.kblocks > 16 ? 2 : 1;
    g.symmetric = symmetric && BN == 128 * CG;
    g.per_split = (g.kblocks + splits - 1) / splits;
    g.splits = (g.kblocks + g.per_split - 1) / g.per_split;             // no piece is empty
    g.n_tiles = g.splits * (g.symmetric ? g.tiles_m * (g.tiles_m + 1) / 2 : g.tiles_m * g.tiles_n) * a.batch;
    g.a_k_major = a.k_major; g.b_k_major = b.k_major;
    g.idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((a.k_major ? 0u : 1u) << 15) | ((b.k_major ? 0u : 1u) << 16) | ((uint32_t)(BN >> 3) << 17) |
              ((uint32_t)((128 * CG) >> 4) << 24);
    if (!gave_up_word(&g.gave_up)) return (int)cudaErrorMemoryAllocation;
    CUtensorMap ma, mb;
    if (!planes_map(&ma, a, 128) || !planes_map(&mb, b, S::kBRows)) return (int)cudaErrorNotSupported;
    auto kernel = split_product_kernel<CG, BN, Out>;
    static std::mutex mu;
    static bool ready[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64) return (int)cudaErrorInvalidDevice;
    {
        std::lock_guard<std::mutex> lock(mu);
        if (!ready[dev]) {
            const cudaError_t rc = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::kSmem);
            if (rc != cudaSuccess) { cudaGetLastError(); return (int)rc; }
            ready[dev] = true;
        }
    }
    const int64_t slots = sm_count() / CG;
    const unsigned grid = (unsigned)((g.n_tiles < slots ? g.n_tiles : slots) * CG);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(kSpThreads);
    cfg.dynamicSmemBytes = S::kSmem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = CG; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = CG == 1 ? 1 : 2;
    const cudaError_t rc = cudaLaunchKernelEx(&cfg, kernel, g, ma, mb, out);
    if (rc != cudaSuccess) { cudaGetLastError(); return (int)rc; }
    count_launch();
    launched_tiles[BN == 256 ? 0 : BN == 128 ? 1 : 2][g.symmetric ? 1 : 0].fetch_add(1, std::memory_order_relaxed);
    return 0;
}

// The tile and the number of pieces K is cut into are those with the least estimated cycles: rounds over the SMs x K-blocks of
// a piece x instructions x cycles per instruction -- measured at 4096^3, a 256 x 256 pair takes the tensor cores' 128, a
// 128 x 128 tile 95 and a 128 x 64 tile 70, the latter two on twice as many slots -- plus, with pieces, writing and adding up
// their results (about 2500 bytes per cycle) and one more launch.
struct Shape { int tile, splits; };

static Shape choose_shape(const Planes& a, const Planes& b, bool symmetric, int most_splits) {
    const int64_t sms = sm_count(), kblocks = (a.k + kSpKB - 1) / kSpKB;
    const int64_t tm[3] = {256, 128, 128}, tn[3] = {256, 128, 64}, cycles[3] = {128, 95, 70}, slots[3] = {sms / 2, sms, sms};
    Shape best = {0, 1};
    int64_t least = INT64_MAX;
    for (int t = 0; t < 3; ++t) {
        const int64_t across = (a.rows + tm[t] - 1) / tm[t];
        const int64_t tiles = (symmetric && tm[t] == tn[t] ? across * (across + 1) / 2 : across * ((b.rows + tn[t] - 1) / tn[t])) * a.batch;
        for (int s = 1; s <= most_splits && (s == 1 || kblocks / s >= 2); ++s) {
            const int64_t rounds = (tiles * s + slots[t] - 1) / slots[t];
            int64_t cost = rounds * ((kblocks + s - 1) / s * 24 * cycles[t] + 3000);
            if (s > 1) cost += 6000 + (int64_t)(s + 1) * a.rows * b.rows * 4 / 2500;
            if (cost < least) { least = cost; best = {t, s}; }
        }
    }
    return best;
}

template <typename Out>
static int launch_any(const Planes& a, const Planes& b, const Out& out, bool symmetric, Shape shape, cudaStream_t st) {
    if (a.k != b.k || a.batch != b.batch || a.k < 1 || (symmetric && a.rows != b.rows)) return (int)cudaErrorInvalidValue;
    if (shape.tile == 0) return launch_shape<2, 256, Out>(a, b, out, symmetric, shape.splits, st);
    if (shape.tile == 1) return launch_shape<1, 128, Out>(a, b, out, symmetric, shape.splits, st);
    return launch_shape<1, 64, Out>(a, b, out, symmetric, shape.splits, st);
}

// The pieces' results added in order, and the epilogue.
__global__ void __launch_bounds__(kBlock)
join_pieces_kernel(int64_t m, int64_t n, int splits, const float* pieces, const Epilogue<float> e) {
    const int64_t total = m * n;
    for (int64_t f = (int64_t)blockIdx.x * kBlock + threadIdx.x; f < total; f += (int64_t)gridDim.x * kBlock) {
        float part[8];
#pragma unroll
        for (int s = 0; s < 8; ++s) if (s < splits) part[s] = pieces[s * total + f];
        float z = part[0];
#pragma unroll
        for (int s = 1; s < 8; ++s) if (s < splits) z += part[s];
        const int64_t i = f / n;
        finish(e, 0, i, f - i * n, z);
    }
}

int launch_split_product(const Planes& a, const Planes& b, const Epilogue<float>& e, const Hot& hot, Scratch& scratch, cudaStream_t st) {
    if (e.alpha != 1.0f || e.d || a.batch != 1) return (int)cudaErrorInvalidValue;
    Shape shape = choose_shape(a, b, false, 8);
    Epilogue<float> way = e;
    float* pieces = nullptr;
    if (shape.splits > 1) {
        const int64_t kblocks = (a.k + kSpKB - 1) / kSpKB, per = (kblocks + shape.splits - 1) / shape.splits;
        shape.splits = (int)((kblocks + per - 1) / per);
        pieces = reinterpret_cast<float*>(scratch.take((size_t)shape.splits * a.rows * b.rows * sizeof(float)));
        if (!pieces) return (int)cudaErrorMemoryAllocation;
        way = Epilogue<float>{};
        way.alpha = 1.f; way.y = pieces; way.ld = b.rows; way.y_batch = a.rows * b.rows;
    }
    const FloatOut out = {way, hot, way.ld % 4 == 0 && aligned16(way.y) && way.y_batch % 4 == 0 &&
                                   (!way.res || (way.res_col == 1 && way.res_row % 4 == 0 && aligned16(way.res)))};
    int rc = launch_any(a, b, out, false, shape, st);
    if (rc || shape.splits == 1) return rc;
    join_pieces_kernel<<<grid_for((a.rows * b.rows + kBlock - 1) / kBlock, 8), kBlock, 0, st>>>(a.rows, b.rows, shape.splits, pieces, e);
    count_launch();
    return (int)cudaGetLastError();
}
int launch_split_product(const Planes& a, const Planes& b, const PlaneEpilogue& e, bool symmetric, cudaStream_t st) {
    const PlaneOut out = {e};
    return launch_any(a, b, out, symmetric, choose_shape(a, b, symmetric, 1), st);
}

}  // namespace cb200

// As if a bounded wait had run out: for a program that tests what it does then.
extern "C" int cb200_product_status_set(void) {
    int* w = cb200::gave_up_word(nullptr);
    if (!w) return -1;
    *const_cast<volatile int*>(w) = 1;
    return 0;
}

// 0: no bounded wait of the tensor-core product or the recurrence has run out in this process since the last call; 1: one did, and results since
// then are not valid; -1: the word could not be read.  Synchronises the device; clears the word.
extern "C" int cb200_product_status(void) {
    int* w = cb200::gave_up_word(nullptr);
    if (!w || cudaDeviceSynchronize() != cudaSuccess) return -1;
    const int v = *const_cast<volatile int*>(w);
    *const_cast<volatile int*>(w) = 0;
    return v;
}

// Launches of the product in this process whose tiles are 256 (two CTAs), 128 or 64 columns wide; of those the ones that compute
// one side of a symmetric result, or the others.
extern "C" unsigned long long cb200_split_product_launches(int columns, int symmetric) {
    return cb200::launched_tiles[columns == 256 ? 0 : columns == 128 ? 1 : 2][symmetric ? 1 : 0].load(std::memory_order_relaxed);
}
