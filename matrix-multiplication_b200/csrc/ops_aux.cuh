// The elementwise half of the epilogue product's backward pass: the activation gradient
// with the bias gradient, bound by HBM.
#pragma once

#include <cuda.h>
#include <cstdint>

#include "ptx.cuh"
#include "tc_ops.cuh"

namespace b200 {

// ---------------------------------------------------------------- activation and bias gradient
constexpr int AG_THREADS = 256;
constexpr int AG_COLS = 256;      // columns per block: 32 lanes x 8

struct ActGradParams {
    const void *dout, *preact;    // m x n; preact null without an activation
    int preact_half;
    void *dz;                     // m x n, or null: the bias gradient alone
    long long dz_pitch;           // elements; a multiple of 8 (16-bit) or 4 (FP32) when vec
    float *partial;               // [row chunks][n] or null
    void *dbias;                  // written directly when there is one row chunk
    int dbias_half;
    int m, n, rows_per_chunk, activation;
    int vec;                      // rows of dout and preact start on 16 bytes
};

// dz = dout * act'(z) in the input format, and per block the column sums of the
// unrounded FP32 values over its rows (each thread 8 columns, every eighth row; the
// eight warps join through shared memory in a fixed order).
template <int FMT>
__global__ void __launch_bounds__(AG_THREADS) act_grad_kernel(const ActGradParams p)
{
    using Type = OpType<FMT>;
    using T = typename Type::T;
    __shared__ float sums[8][AG_COLS];
    wait_for_prior_grid();
    allow_next_grid();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int col0 = static_cast<int>(blockIdx.x) * AG_COLS + lane * 8;
    const long long row_begin = static_cast<long long>(blockIdx.y) * p.rows_per_chunk;
    const int row_end = static_cast<int>(min(static_cast<long long>(p.m), row_begin + p.rows_per_chunk));
    const bool vec = p.vec && col0 + 8 <= p.n;
    float sum[8] = {};
    for (int row = static_cast<int>(row_begin) + warp; row < row_end; row += 8) {
        if (col0 >= p.n)
            break;
        const long long at = static_cast<long long>(row) * p.n + col0;
        const long long dz_at = static_cast<long long>(row) * p.dz_pitch + col0;
        float d[8], z[8];
        auto read = [&](const void *src, bool half, float (&x)[8]) {
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
        read(p.dout, FMT != kOpTF32, d);
        if (p.preact) {
            read(p.preact, p.preact_half != 0, z);
#pragma unroll
            for (int e = 0; e < 8; ++e)
                d[e] *= op_activation_slope(z[e], p.activation);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e)
            sum[e] += d[e];
        if (p.dz) {
            T *dst = static_cast<T *>(p.dz) + dz_at;
            if (col0 + 8 <= p.dz_pitch) {       // the scratch copy's rows are padded to 16 bytes
                if constexpr (FMT == kOpTF32) {
                    reinterpret_cast<float4 *>(dst)[0] = make_float4(d[0], d[1], d[2], d[3]);
                    reinterpret_cast<float4 *>(dst)[1] = make_float4(d[4], d[5], d[6], d[7]);
                } else {
                    *reinterpret_cast<uint4 *>(dst) = make_uint4(Type::pack(d[0], d[1]), Type::pack(d[2], d[3]),
                                                                 Type::pack(d[4], d[5]), Type::pack(d[6], d[7]));
                }
            } else {
                for (int e = 0; e < 8 && col0 + e < p.dz_pitch; ++e)
                    dst[e] = Type::from(d[e]);
            }
        }
    }
    if (!p.partial && !p.dbias)
        return;
#pragma unroll
    for (int e = 0; e < 8; ++e)
        sums[warp][lane * 8 + e] = sum[e];
    __syncthreads();
    const int col = static_cast<int>(blockIdx.x) * AG_COLS + threadIdx.x;
    if (col < p.n) {
        float total = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            total += sums[i][threadIdx.x];
        if (p.partial)
            p.partial[static_cast<long long>(blockIdx.y) * p.n + col] = total;
        else if (p.dbias_half)
            static_cast<T *>(p.dbias)[col] = Type::from(total);
        else
            static_cast<float *>(p.dbias)[col] = total;
    }
}

// dbias = the row chunks' partial sums, added in order.
template <int FMT>
__global__ void __launch_bounds__(256) bias_grad_kernel(const float *partial, int chunks, int n, void *dbias,
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
    for (int i = 0; i < chunks; ++i)
        total += partial[static_cast<long long>(i) * n + col];
    if (dbias_half)
        static_cast<T *>(dbias)[col] = Type::from(total);
    else
        static_cast<float *>(dbias)[col] = total;
}

} // namespace b200
