// Host side shared by the library's translation units: the per-device context, the
// error convention (0/1 with "operation: detail"), tensor-map encoding,
// stream-ordered scratch and launches with programmatic stream serialisation.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>
#include <cstdio>
#include <mutex>
#include <utility>

#include "pack.cuh"
#include "ptx.cuh"

namespace b200 {

using EncodeTiledFn = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                   const cuuint64_t *, const cuuint32_t *, const cuuint32_t *,
                                   CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                                   CUtensorMapFloatOOBfill);

struct Context {
    int device = 0;
    int major = 0;
    int minor = 0;
    // What the tensor-core launches may use: the device's SMs, or fewer after
    // matmul_set_sm_limit (the device_* fields keep the device's own values).
    int sm_count = 0;
    int max_pairs = 0;        // co-resident 2-CTA clusters of the pair kernel
    int max_split_ctas[4] = {}; // co-resident CTAs of the single-CTA kernel in (1,1,S) clusters, S = 1,2,4,8
    int device_sm_count = 0;
    int device_max_pairs = 0;
    int device_max_split_ctas[4] = {};
    int ffma_resident[2] = {}; // resident blocks per SM of each aligned FFMA tile
    EncodeTiledFn encode = nullptr;
    cudaMemPool_t pool = nullptr;
    // Device address of g_noalloc_scratch in this context's device, looked up by
    // the context's first matmul_launch_noalloc call with the device current (in
    // host code the symbol itself is a host-side stand-in, never a device
    // address).  Kept per context, so a context created after a device reset
    // looks it up again in the reloaded module.
    std::mutex noalloc_mutex;
    void *noalloc_scratch = nullptr;
    // Limit of the bounded waits that depend on another warp's progress
    // (matmul_set_wait_limit); 0 = the default.
    unsigned long long wait_limit_ns = 0;
    unsigned int *status = nullptr;   // device address of the status word (matmul_device_status)
    // Whether the operators' kernels of a format have their attributes in this context's device
    // (setup_operators).
    std::mutex operators_mutex;
    std::atomic<bool> operators_ready[3] = {};
};

inline unsigned long long wait_limit(const Context *ctx)
{
    return ctx->wait_limit_ns ? ctx->wait_limit_ns : kWaitLimitNs;
}

inline void clear_error(char *error, size_t error_size)
{
    if (error && error_size)
        error[0] = '\0';
}

inline int fail(char *error, size_t error_size, const char *operation, const char *detail)
{
    if (error && error_size)
        std::snprintf(error, error_size, "%s: %s", operation, detail);
    return 1;
}

inline int fail_cuda(char *error, size_t error_size, const char *operation, cudaError_t status)
{
    const char *detail = cudaGetErrorString(status);
    cudaGetLastError();
    return fail(error, error_size, operation, detail);
}

inline bool aligned16(const void *p)
{
    return (reinterpret_cast<uintptr_t>(p) & 15u) == 0;
}

inline int64_t round_up(int64_t x, int64_t to)
{
    return (x + to - 1) / to * to;
}

inline bool encode_2d(const Context *ctx, CUtensorMap *map, CUtensorMapDataType type, const void *base, uint64_t inner,
               uint64_t outer, uint64_t row_bytes, uint32_t box_inner, uint32_t box_outer,
               CUtensorMapSwizzle swizzle = CU_TENSOR_MAP_SWIZZLE_128B)
{
    const cuuint64_t dims[2] = {inner, outer};
    const cuuint64_t strides[1] = {row_bytes};
    const cuuint32_t box[2] = {box_inner, box_outer};
    const cuuint32_t elem_strides[2] = {1, 1};
    const CUresult r = ctx->encode(map, type, 2, const_cast<void *>(base), dims, strides, box, elem_strides,
                                   CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                                   CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS;
}

// Stream-ordered scratch: from the context's pool outside capture, as a graph
// allocation node inside capture.  Freed on the same stream after use.
inline cudaError_t scratch_alloc(Context *ctx, void **ptr, size_t bytes, cudaStream_t stream)
{
    cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
    cudaError_t st = cudaStreamIsCapturing(stream, &capture);
    if (st != cudaSuccess)
        return st;
    if (capture == cudaStreamCaptureStatusActive || ctx->pool == nullptr)
        return cudaMallocAsync(ptr, bytes, stream);
    return cudaMallocFromPoolAsync(ptr, bytes, ctx->pool, stream);
}

// Launch with programmatic stream serialisation: the kernel may start while the
// previous kernel on the stream finishes; our kernels run their prologue and
// then wait (griddepcontrol.wait) before touching global memory.
template <typename... Params, typename... Args>
cudaError_t launch_pdl(void (*kernel)(Params...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream,
                       Args &&...args)
{
    cudaLaunchConfig_t config{};
    config.gridDim = grid;
    config.blockDim = block;
    config.dynamicSmemBytes = smem;
    config.stream = stream;
    cudaLaunchAttribute attribute{};
    attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute.val.programmaticStreamSerializationAllowed = 1;
    config.attrs = &attribute;
    config.numAttrs = 1;
    return cudaLaunchKernelEx(&config, kernel, std::forward<Args>(args)...);
}

// launch_pdl with clusters of (1, 1, cluster_z) CTAs (cluster_z divides grid.z).
template <typename... Params, typename... Args>
cudaError_t launch_pdl_cluster_z(void (*kernel)(Params...), dim3 grid, dim3 block, size_t smem, unsigned int cluster_z,
                                 cudaStream_t stream, Args &&...args)
{
    cudaLaunchConfig_t config{};
    config.gridDim = grid;
    config.blockDim = block;
    config.dynamicSmemBytes = smem;
    config.stream = stream;
    cudaLaunchAttribute attributes[2]{};
    attributes[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attributes[0].val.programmaticStreamSerializationAllowed = 1;
    attributes[1].id = cudaLaunchAttributeClusterDimension;
    attributes[1].val.clusterDim.x = 1;
    attributes[1].val.clusterDim.y = 1;
    attributes[1].val.clusterDim.z = cluster_z;
    config.attrs = attributes;
    config.numAttrs = cluster_z > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&config, kernel, std::forward<Args>(args)...);
}

// Operands TMA cannot read in place (base not 16-byte aligned, or a row pitch
// that is not a multiple of 16 bytes), repacked into 16-byte aligned scratch in
// one launch (an operand with `direct` set is skipped).  TF32 operands are copied
// as FP32 words: the TMA loads round them.
template <typename T>
cudaError_t pack_operands(const Context *ctx, const void *a, bool a_direct, void *a_dst, int64_t m, int64_t k,
                          int64_t lda, const void *b, bool b_direct, void *b_dst, int64_t n, int64_t ldb,
                          cudaStream_t stream)
{
    if (a_direct && b_direct)
        return cudaSuccess;
    const PackJob<T> ja{static_cast<const T *>(a), static_cast<T *>(a_dst), a_direct ? 0 : m, k, lda};
    const PackJob<T> jb{static_cast<const T *>(b), static_cast<T *>(b_dst), b_direct ? 0 : k, n, ldb};
    const int64_t cap = 4LL * ctx->sm_count;
    auto blocks_for = [&](const PackJob<T> &j) {
        const int64_t blocks = (j.rows * j.ld + 255) / 256;
        return blocks < 1 ? int64_t{1} : blocks > cap ? cap : blocks;
    };
    const int64_t a_blocks = blocks_for(ja), b_blocks = blocks_for(jb);
    return launch_pdl(pack_pair_kernel<T>, dim3(static_cast<unsigned int>(a_blocks + b_blocks)), dim3(256), 0,
                      stream, ja, jb, static_cast<int>(a_blocks));
}

} // namespace b200
