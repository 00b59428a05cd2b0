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
// multiple of 16 bytes, zero in the added columns; each thread writes 16-byte chunks.
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
            q = load_16_bytes<ELEM>(from);
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
constexpr int AG_COLS = 64;       // columns per block: 8 lanes x 8, so that a warp covers four rows
constexpr int AG_PASS = 32;       // rows of one pass of a block
constexpr int AG_ROWS = 4;        // rows a thread has in flight
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

// dz = dout * act'(z) in the input format, which both products that read it need (an FP32
// dz would take two of each, for its high and its low part; as it is, da and db are off by
// about the square root of two of their own rounding), and the column sums of the unrounded
// FP32 values: each thread takes 8 columns and every 32nd row of its block's chunk, four rows in
// flight; a block's 32 row positions join through its shared memory and the blocks of a
// cluster (along y) through each other's, both in a fixed order.  Bound by HBM: two reads
// and a write.
template <int FMT>
__global__ void __launch_bounds__(AG_THREADS, 4) act_grad_kernel(const ActGradParams p)
{
    using Type = OpType<FMT>;
    using T = typename Type::T;
    __shared__ float sums[AG_PASS][AG_COLS + 1];
    __shared__ float block_sums[AG_COLS];
    wait_for_prior_grid();
    allow_next_grid();
    const int place = threadIdx.x >> 3;            // row within a pass
    const int local = (threadIdx.x & 7) * 8;       // first column within the block
    const int col0 = static_cast<int>(blockIdx.x) * AG_COLS + local;
    const int64_t row_begin = static_cast<int64_t>(blockIdx.y) * p.rows_per_chunk;
    const int row_end = static_cast<int>(min(static_cast<int64_t>(p.m), row_begin + p.rows_per_chunk));
    const bool whole = col0 + 8 <= p.n;
    float sum[8] = {};
    auto widen = [&](const uint4 &q, float (&x)[8]) {
        if constexpr (FMT != kOpTF32) {
            const T *h = reinterpret_cast<const T *>(&q);
#pragma unroll
            for (int e = 0; e < 8; ++e)
                x[e] = Type::to(h[e]);
        }
    };
    auto read = [&](const void *src, bool half, int row, float (&x)[8]) {
        const int64_t at = static_cast<int64_t>(row) * p.n + col0;
        if (!whole) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                x[e] = col0 + e < p.n ? (half ? Type::to(static_cast<const T *>(src)[at + e])
                                              : static_cast<const float *>(src)[at + e])
                                      : 0.0f;
        } else if (half) {
            const uint8_t *from = static_cast<const uint8_t *>(src) + at * 2;
            widen(p.vec ? *reinterpret_cast<const uint4 *>(from) : load_16_bytes<2>(from), x);
        } else {
            const uint8_t *from = static_cast<const uint8_t *>(src) + at * 4;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint4 q = p.vec ? reinterpret_cast<const uint4 *>(from)[h] : load_16_bytes<4>(from + 16 * h);
                x[4 * h] = __uint_as_float(q.x);
                x[4 * h + 1] = __uint_as_float(q.y);
                x[4 * h + 2] = __uint_as_float(q.z);
                x[4 * h + 3] = __uint_as_float(q.w);
            }
        }
    };
    op_with_activation(p.preact ? p.activation : kActNone, [&](auto act) {
        constexpr int ACT = decltype(act)::value;
        if (col0 >= p.n)
            return;
        // dz of 8 columns of a row: summed, and stored rounded.
        auto finish = [&](int row, float (&d)[8], float (&z)[8]) {
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                float2 dz = make_float2(d[e], d[e + 1]);
                if (ACT != kActNone)
                    dz = __fmul2_rn(dz, op_activation_slope<ACT>(make_float2(z[e], z[e + 1])));
                d[e] = dz.x;
                d[e + 1] = dz.y;
                sum[e] += dz.x;
                sum[e + 1] += dz.y;
            }
            if (p.dz) {
                T *dst = static_cast<T *>(p.dz) + row * p.dz_pitch + col0;
                // Rows in scratch are padded to 128 bytes: 8 columns always fit.
                if constexpr (FMT == kOpTF32) {
                    reinterpret_cast<float4 *>(dst)[0] = make_float4(d[0], d[1], d[2], d[3]);
                    reinterpret_cast<float4 *>(dst)[1] = make_float4(d[4], d[5], d[6], d[7]);
                } else {
                    *reinterpret_cast<uint4 *>(dst) = make_uint4(Type::pack(d[0], d[1]), Type::pack(d[2], d[3]),
                                                                 Type::pack(d[4], d[5]), Type::pack(d[6], d[7]));
                }
            }
        };
        int row = static_cast<int>(row_begin) + place;
        if (FMT != kOpTF32 && whole && p.vec && (ACT == kActNone || p.preact_half)) {
            // All loads of AG_ROWS rows before the first use: with a branch around each load a
            // thread waited for one at a time (4096 x 14336: 132 us against 97 us).
            for (; row + AG_PASS * (AG_ROWS - 1) < row_end; row += AG_PASS * AG_ROWS) {
                uint4 dq[AG_ROWS], zq[AG_ROWS];
#pragma unroll
                for (int i = 0; i < AG_ROWS; ++i) {
                    const int64_t at = static_cast<int64_t>(row + AG_PASS * i) * p.n + col0;
                    dq[i] = *reinterpret_cast<const uint4 *>(static_cast<const T *>(p.dout) + at);
                    if (ACT != kActNone)
                        zq[i] = *reinterpret_cast<const uint4 *>(static_cast<const T *>(p.preact) + at);
                }
#pragma unroll
                for (int i = 0; i < AG_ROWS; ++i) {
                    float d[8], z[8];
                    widen(dq[i], d);
                    if (ACT != kActNone)
                        widen(zq[i], z);
                    finish(row + AG_PASS * i, d, z);
                }
            }
        }
        for (; row < row_end; row += AG_PASS) {
            float d[8], z[8];
            read(p.dout, FMT != kOpTF32, row, d);
            if (ACT != kActNone)
                read(p.preact, p.preact_half != 0, row, z);
            finish(row, d, z);
        }
    });
    if (!p.dbias)
        return;      // the same for the whole cluster
#pragma unroll
    for (int e = 0; e < 8; ++e)
        sums[place][local + e] = sum[e];
    __syncthreads();
    if (threadIdx.x < AG_COLS) {
        float total = 0.0f;
#pragma unroll
        for (int i = 0; i < AG_PASS; ++i)
            total += sums[i][threadIdx.x];
        block_sums[threadIdx.x] = total;
    }
    // The cluster's first block adds its blocks' sums in order.
    cluster_sync_all();
    uint32_t blocks;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(blocks));
    const int col = static_cast<int>(blockIdx.x) * AG_COLS + threadIdx.x;
    if (cluster_cta_rank() == 0 && threadIdx.x < AG_COLS && col < p.n) {
        float total = 0.0f;
        for (uint32_t j = 0; j < blocks; ++j)
            total += __uint_as_float(ld_shared_cluster_u32(map_to_cta(smem_addr(block_sums + threadIdx.x), j)));
        if (p.partial)
            p.partial[static_cast<int64_t>(blockIdx.y / blocks) * p.n + col] = total;
        else if (p.dbias_half)
            static_cast<T *>(p.dbias)[col] = Type::from(total);
        else
            static_cast<float *>(p.dbias)[col] = total;
    }
    cluster_sync_all();      // no block leaves while its sums are read
}

// ---------------------------------------------------------------- chunks of K
struct ChunkSumParams {
    const float *chunks;          // count slabs of rows x cols, pitch a multiple of 4
    int count, rows, cols;
    int64_t slab, pitch;
    const float *base;            // null, or FP32 to add (pitch base_pitch)
    int64_t base_pitch;
    void *out;
    int64_t out_pitch;
    int out_half, vec;            // vec: out's and base's rows start on 16 bytes
};

// out = base + the chunks' products, added in order; four columns a thread.  Bound by the
// chunks' bytes, which are in L2.
template <int FMT>
__global__ void __launch_bounds__(256) chunk_sum_kernel(const ChunkSumParams p)
{
    using Type = OpType<FMT>;
    using T = typename Type::T;
    wait_for_prior_grid();
    allow_next_grid();
    const int quads = (p.cols + 3) / 4;
    const int64_t total = static_cast<int64_t>(p.rows) * quads;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < total;
         i += static_cast<int64_t>(gridDim.x) * 256) {
        const int row = static_cast<int>(i / quads), col = static_cast<int>(i - static_cast<int64_t>(row) * quads) * 4;
        const int count = min(4, p.cols - col);
        float v[4] = {};
        if (p.base) {
            const float *b = p.base + row * p.base_pitch + col;
            for (int e = 0; e < count; ++e)
                v[e] = b[e];
        }
        const float *x = p.chunks + row * p.pitch + col;
#pragma unroll 8
        for (int j = 0; j < p.count; ++j) {
            const float4 q = *reinterpret_cast<const float4 *>(x + j * p.slab);
            v[0] += q.x;
            v[1] += q.y;
            v[2] += q.z;
            v[3] += q.w;
        }
        if (p.out_half) {
            T *to = static_cast<T *>(p.out) + row * p.out_pitch + col;
            if (p.vec && count == 4 && FMT != kOpTF32)
                *reinterpret_cast<uint2 *>(to) = make_uint2(Type::pack(v[0], v[1]), Type::pack(v[2], v[3]));
            else
                for (int e = 0; e < count; ++e)
                    to[e] = Type::from(v[e]);
        } else {
            float *to = static_cast<float *>(p.out) + row * p.out_pitch + col;
            if (p.vec && count == 4)
                *reinterpret_cast<float4 *>(to) = make_float4(v[0], v[1], v[2], v[3]);
            else
                for (int e = 0; e < count; ++e)
                    to[e] = v[e];
        }
    }
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
