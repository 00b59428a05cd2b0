// The operators' kernels as seen from the host code (ops.cu): one translation unit per
// input format (ops_f16.cu, ops_bf16.cu, ops_tf32.cu) instantiates them.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include "ops_aux.cuh"
#include "tc_ops.cuh"

namespace b200 {

// How a product's operands are stored: A.B, A.B^T, A^T.B of row-major matrices.
enum OpLayout : int { kNN = 0, kNT = 1, kTN = 2 };

// Tiles: a CTA pair's 256 x 256, one CTA's 128 x 128 or 128 x 64, or, transposed, 128
// columns x 16 / 32 / 64 / 128 rows.
enum OpTileKind : int { kPair256 = 0, kSingle128 = 1, kSingle64 = 2, kSwap16 = 3, kSwap32 = 4, kSwap64 = 5, kSwap128 = 6 };

struct OpLaunch {
    CUtensorMap map_a{}, map_b{}, map_c{}, map_z{};
    OpParams p{};
    int layout = kNN, tile = kPair256, epilogue = kEpiStore;
    int grid = 1;       // CTAs, or tiles when splits > 1
    int splits = 1;     // K splits: clusters of that many CTAs along z (single-CTA tiles)
};

struct OpKernels {
    cudaError_t (*setup)();     // kernel attributes; once per context
    cudaError_t (*product)(const OpLaunch &launch, cudaStream_t stream);
    cudaError_t (*act_grad)(const ActGradParams &params, dim3 grid, int cluster, cudaStream_t stream);
    cudaError_t (*bias_grad)(const float *partial, int count, int n, void *dbias, int dbias_half, cudaStream_t stream);
    cudaError_t (*repack)(const RepackJob &job0, const RepackJob &job1, int sms, cudaStream_t stream);
    cudaError_t (*chunk_sum)(const ChunkSumParams &params, int sms, cudaStream_t stream);
};

extern const OpKernels kOpKernelsF16, kOpKernelsBF16, kOpKernelsTF32;

} // namespace b200
