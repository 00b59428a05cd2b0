// Elementwise kernels of the operators, bound by HBM: the activation gradient with the
// bias gradient, and the copy of operands that TMA cannot address.
#pragma once

#include <cuda.h>
#include <cstdint>

#include "ptx.cuh"
#include "tc_ops.cuh"

namespace b200 {

// ---------------------------------------------------------------- operand copy
constexpr int RP_THREADS = 256;

// One matrix to copy: rows x cols -> rows x pitch, by `units` units of a block each.
struct RepackJob {
    const uint8_t *src;
    uint8_t *dst;
    int64_t rows, cols, pitch, units;
    int log_lanes;      // threads per row: a power of two, at most the block
};

inline RepackJob repack_job(const void *src, void *dst, int64_t rows, int64_t cols, int64_t pitch, int elem)
{
    const int64_t chunks = pitch * elem / 16;
    int log_lanes = 0;
    while ((1 << log_lanes) < RP_THREADS && (int64_t{1} << log_lanes) < chunks)
        ++log_lanes;
    const int64_t per_block = RP_THREADS >> log_lanes, lanes = int64_t{1} << log_lanes;
    const int64_t units = (rows + per_block - 1) / per_block * ((chunks + lanes - 1) / lanes);
    return {static_cast<const uint8_t *>(src), static_cast<uint8_t *>(dst), rows, cols, pitch, units, log_lanes};
}

// rows x cols of ELEM-byte elements at any element alignment -> rows x pitch with pitch a
// multiple of 16 bytes, zero in the added columns.  Each thread writes 16-byte chunks; a
// source that starts between two 4-byte words is read as a half word, three words and a
// half word and shifted into place, so that nothing outside the matrix is read.
// Up to two matrices in one launch.
template <int ELEM>
__global__ void __launch_bounds__(RP_THREADS) repack_kernel(const RepackJob job0, const RepackJob job1)
{
    constexpr int kPer = 16 / ELEM;
    wait_for_prior_grid();
    allow_next_grid();
    for (int64_t at = blockIdx.x; at < job0.units + job1.units; at += gridDim.x) {
        const RepackJob &job = at < job0.units ? job0 : job1;
        const int64_t u = at < job0.units ? at : at - job0.units;
        const int64_t cols = job.cols, pitch = job.pitch;
        const int lanes = 1 << job.log_lanes;
        const int64_t chunks = pitch / kPer, segments = (chunks + lanes - 1) >> job.log_lanes;
        const int64_t block_row = u / segments;
        const int64_t row = block_row * (RP_THREADS >> job.log_lanes) + (threadIdx.x >> job.log_lanes);
        const int64_t c = (u - block_row * segments) * lanes + (threadIdx.x & (lanes - 1));
        if (row >= job.rows || c >= chunks)
            continue;
        const uint8_t *from = job.src + (row * cols + c * kPer) * ELEM;
        uint4 q;
        if ((c + 1) * kPer <= cols) {
            if (ELEM == 2 && (reinterpret_cast<uintptr_t>(from) & 2u)) {
                const uint32_t w0 = *reinterpret_cast<const uint16_t *>(from);
                const uint32_t w1 = *reinterpret_cast<const uint32_t *>(from + 2);
                const uint32_t w2 = *reinterpret_cast<const uint32_t *>(from + 6);
                const uint32_t w3 = *reinterpret_cast<const uint32_t *>(from + 10);
                const uint32_t w4 = *reinterpret_cast<const uint16_t *>(from + 14);
                q.x = w0 | (w1 << 16);
                q.y = (w1 >> 16) | (w2 << 16);
                q.z = (w2 >> 16) | (w3 << 16);
                q.w = (w3 >> 16) | (w4 << 16);
            } else {
                q.x = reinterpret_cast<const uint32_t *>(from)[0];
                q.y = reinterpret_cast<const uint32_t *>(from)[1];
                q.z = reinterpret_cast<const uint32_t *>(from)[2];
                q.w = reinterpret_cast<const uint32_t *>(from)[3];
            }
        } else {
            uint32_t words[4] = {};
#pragma unroll
            for (int e = 0; e < kPer; ++e)
                if (c * kPer + e < cols) {
                    if constexpr (ELEM == 2)
                        words[e / 2] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t *>(from)[e]) << (16 * (e & 1));
                    else
                        words[e] = reinterpret_cast<const uint32_t *>(from)[e];
                }
            q = make_uint4(words[0], words[1], words[2], words[3]);
        }
        *reinterpret_cast<uint4 *>(job.dst + (row * pitch + c * kPer) * ELEM) = q;
    }
}

// ---------------------------------------------------------------- activation and bias gradient
constexpr int AG_THREADS = 256;
constexpr int AG_COLS = 256;      // columns per block: 32 lanes x 8
constexpr int AG_ROWS = 2;        // rows a thread has in flight
constexpr int AG_CLUSTER = 8;     // row chunks whose sums are joined in one cluster

struct ActGradParams {
    const void *dout, *preact;    // m x n; preact null without an activation
    int preact_half;
    void *dz;                     // m x n, or null: the bias gradient alone
    long long dz_pitch;           // elements; rows start on 16 bytes
    float *partial;               // [clusters of row chunks][n] when there are several, else null
    void *dbias;                  // null, or written directly when there is one cluster
    int dbias_half;
    int m, n, rows_per_chunk, activation;
    int vec;                      // rows of dout and preact start on 16 bytes
};

// dz = dout * act'(z) in the input format, and the column sums of the unrounded FP32
// values: each thread takes 8 columns and every eighth row of its block's chunk, two rows
// in flight; a block's eight warps join through its shared memory and the blocks of a
// cluster (along y) through each other's, both in a fixed order.
template <int FMT>
__global__ void __launch_bounds__(AG_THREADS) act_grad_kernel(const ActGradParams p)
{
    using Type = OpType<FMT>;
    using T = typename Type::T;
    __shared__ float sums[8][AG_COLS];
    __shared__ __align__(16) float block_sums[AG_COLS];
    wait_for_prior_grid();
    allow_next_grid();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int col0 = static_cast<int>(blockIdx.x) * AG_COLS + lane * 8;
    const long long row_begin = static_cast<long long>(blockIdx.y) * p.rows_per_chunk;
    const int row_end = static_cast<int>(min(static_cast<long long>(p.m), row_begin + p.rows_per_chunk));
    const bool vec = p.vec && col0 + 8 <= p.n;
    float sum[8] = {};
    auto read = [&](const void *src, bool half, int row, float (&x)[8]) {
        const long long at = static_cast<long long>(row) * p.n + col0;
        if (vec && half) {
            if constexpr (FMT != kOpTF32) {
                const uint4 q = *reinterpret_cast<const uint4 *>(static_cast<const T *>(src) + at);
                const T *h = reinterpret_cast<const T *>(&q);
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    x[e] = Type::to(h[e]);
            }
        } else if (vec) {
            const float4 q0 = reinterpret_cast<const float4 *>(static_cast<const float *>(src) + at)[0];
            const float4 q1 = reinterpret_cast<const float4 *>(static_cast<const float *>(src) + at)[1];
            x[0] = q0.x, x[1] = q0.y, x[2] = q0.z, x[3] = q0.w;
            x[4] = q1.x, x[5] = q1.y, x[6] = q1.z, x[7] = q1.w;
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                x[e] = col0 + e < p.n ? (half ? Type::to(static_cast<const T *>(src)[at + e])
                                              : static_cast<const float *>(src)[at + e])
                                      : 0.0f;
        }
    };
    op_with_activation(p.preact ? p.activation : kActNone, [&](auto act) {
        constexpr int ACT = decltype(act)::value;
        if (col0 >= p.n)
            return;
        for (int row = static_cast<int>(row_begin) + warp; row < row_end; row += 8 * AG_ROWS) {
            float d[AG_ROWS][8], z[AG_ROWS][8];
#pragma unroll
            for (int i = 0; i < AG_ROWS; ++i)
                if (row + 8 * i < row_end) {
                    read(p.dout, FMT != kOpTF32, row + 8 * i, d[i]);
                    if (ACT != kActNone)
                        read(p.preact, p.preact_half != 0, row + 8 * i, z[i]);
                }
#pragma unroll
            for (int i = 0; i < AG_ROWS; ++i) {
                if (row + 8 * i >= row_end)
                    break;
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                    float2 dz = make_float2(d[i][e], d[i][e + 1]);
                    if (ACT != kActNone)
                        dz = __fmul2_rn(dz, op_activation_slope<ACT>(make_float2(z[i][e], z[i][e + 1])));
                    d[i][e] = dz.x;
                    d[i][e + 1] = dz.y;
                    sum[e] += dz.x;
                    sum[e + 1] += dz.y;
                }
                if (p.dz) {
                    T *dst = static_cast<T *>(p.dz) + (row + 8 * i) * p.dz_pitch + col0;
                    if (col0 + 8 <= p.dz_pitch) {       // rows are padded to 16 bytes
                        if constexpr (FMT == kOpTF32) {
                            reinterpret_cast<float4 *>(dst)[0] = make_float4(d[i][0], d[i][1], d[i][2], d[i][3]);
                            reinterpret_cast<float4 *>(dst)[1] = make_float4(d[i][4], d[i][5], d[i][6], d[i][7]);
                        } else {
                            *reinterpret_cast<uint4 *>(dst) =
                                make_uint4(Type::pack(d[i][0], d[i][1]), Type::pack(d[i][2], d[i][3]),
                                           Type::pack(d[i][4], d[i][5]), Type::pack(d[i][6], d[i][7]));
                        }
                    } else {
                        for (int e = 0; e < 8 && col0 + e < p.dz_pitch; ++e)
                            dst[e] = Type::from(d[i][e]);
                    }
                }
            }
        }
    });
    if (!p.dbias)
        return;      // the same for the whole cluster
#pragma unroll
    for (int e = 0; e < 8; ++e)
        sums[warp][lane * 8 + e] = sum[e];
    __syncthreads();
    float total = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i)
        total += sums[i][threadIdx.x];
    block_sums[threadIdx.x] = total;
    // The cluster's first block adds its blocks' sums in order.
    cluster_sync_all();
    uint32_t blocks;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(blocks));
    const int col = static_cast<int>(blockIdx.x) * AG_COLS + threadIdx.x;
    if (cluster_cta_rank() == 0 && col < p.n) {
        total = 0.0f;
        for (uint32_t j = 0; j < blocks; ++j)
            total += __uint_as_float(ld_shared_cluster_u32(map_to_cta(smem_addr(block_sums + threadIdx.x), j)));
        if (p.partial)
            p.partial[static_cast<long long>(blockIdx.y / blocks) * p.n + col] = total;
        else if (p.dbias_half)
            static_cast<T *>(p.dbias)[col] = Type::from(total);
        else
            static_cast<float *>(p.dbias)[col] = total;
    }
    cluster_sync_all();      // no block leaves while its sums are read
}

// dbias = the clusters' partial sums, added in order.
template <int FMT>
__global__ void __launch_bounds__(256) bias_grad_kernel(const float *partial, int count, int n, void *dbias,
                                                        int dbias_half)
{
    using Type = OpType<FMT>;
    using T = typename Type::T;
    wait_for_prior_grid();
    allow_next_grid();
    const int col = static_cast<int>(blockIdx.x) * 256 + threadIdx.x;
    if (col >= n)
        return;
    float total = 0.0f;
#pragma unroll 8
    for (int i = 0; i < count; ++i)
        total += partial[static_cast<long long>(i) * n + col];
    if (dbias_half)
        static_cast<T *>(dbias)[col] = Type::from(total);
    else
        static_cast<float *>(dbias)[col] = total;
}

} // namespace b200
