// Instantiates the operators' kernels for one input format (see ops.cuh).
#pragma once

#include "context.cuh"
#include "ops.cuh"

namespace b200 {

template <int FMT>
struct OpInstances {
    using T = typename OpType<FMT>::T;
    static constexpr bool kHalf = FMT != kOpTF32;

    // Calls f(kernel, CTAs per tile, threads, shared memory) and shared memory for the kernel of a launch.
    template <int CTAS, int BN, bool A_MN, bool B_MN, int EPI, bool DIRECT = false, typename F>
    static cudaError_t with(F &&f)
    {
        using Tile = OpTile<CTAS, BN, DIRECT>;
        return f(&op_kernel<FMT, CTAS, BN, A_MN, B_MN, EPI, DIRECT>, CTAS, Tile::kThreads, Tile::kSmem);
    }
    // Kernels that load B themselves (chosen by direct_pays).
    template <typename F>
    static cudaError_t with_direct(int tile, int epilogue, F &&f)
    {
        if constexpr (kHalf) {
            if (epilogue == kEpiLse && tile == kSingle128)
                return with<1, 128, false, true, kEpiLse, true>(f);
            if (epilogue == kEpiStoreT && tile == kSwap16)
                return with<1, 16, true, false, kEpiStoreT, true>(f);
            if (epilogue == kEpiStoreT && tile == kSwap32)
                return with<1, 32, true, false, kEpiStoreT, true>(f);
            if (epilogue == kEpiStoreT && tile == kSwap64)
                return with<1, 64, true, false, kEpiStoreT, true>(f);
        }
        return cudaErrorInvalidValue;
    }
    template <bool A_MN, bool B_MN, int EPI, typename F>
    static cudaError_t with_tile(int tile, F &&f)
    {
        switch (tile) {
        case kPair256: return with<2, 256, A_MN, B_MN, EPI>(f);
        case kSingle128: return with<1, 128, A_MN, B_MN, EPI>(f);
        case kSingle64: return with<1, 64, A_MN, B_MN, EPI>(f);
        }
        return cudaErrorInvalidValue;
    }
    template <typename F>
    static cudaError_t with_kernel(int layout, int tile, int epilogue, F &&f)
    {
        if (epilogue == kEpiStoreT) {
            switch (tile) {
            case kSwap16: return with<1, 16, true, false, kEpiStoreT>(f);
            case kSwap32: return with<1, 32, true, false, kEpiStoreT>(f);
            case kSwap64: return with<1, 64, true, false, kEpiStoreT>(f);
            case kSwap128: return with<1, 128, true, false, kEpiStoreT>(f);
            }
            return cudaErrorInvalidValue;
        }
        if (epilogue == kEpiStore)
            return layout == kNN   ? with_tile<false, true, kEpiStore>(tile, f)
                   : layout == kNT ? with_tile<false, false, kEpiStore>(tile, f)
                                   : with_tile<true, true, kEpiStore>(tile, f);
        if (layout != kNN)
            return cudaErrorInvalidValue;
        if (epilogue == kEpiLse)
            return with_tile<false, true, kEpiLse>(tile, f);
        if constexpr (FMT != kOpF16)      // probabilities fall below FP16's range
            return with_tile<false, true, kEpiSoftmaxGrad>(tile, f);
        return cudaErrorInvalidValue;
    }

    static cudaError_t setup()
    {
        auto set = [](auto kernel, int, int, int smem) {
            return cudaFuncSetAttribute(reinterpret_cast<const void *>(kernel),
                                        cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        };
        cudaError_t st = cudaSuccess;
        for (int tile = kPair256; tile <= kSingle64 && st == cudaSuccess; ++tile) {
            for (int layout = kNN; layout <= kTN && st == cudaSuccess; ++layout)
                st = with_kernel(layout, tile, kEpiStore, set);
            if (st == cudaSuccess)
                st = with_kernel(kNN, tile, kEpiLse, set);
            if (st == cudaSuccess && FMT != kOpF16)
                st = with_kernel(kNN, tile, kEpiSoftmaxGrad, set);
        }
        for (int tile = kSwap16; tile <= kSwap128 && st == cudaSuccess; ++tile)
            st = with_kernel(kNN, tile, kEpiStoreT, set);
        if (kHalf) {
            for (int tile = kSwap16; tile <= kSwap64 && st == cudaSuccess; ++tile)
                st = with_direct(tile, kEpiStoreT, set);
            if (st == cudaSuccess)
                st = with_direct(kSingle128, kEpiLse, set);
        }
        return st;
    }

    static cudaError_t product(const OpLaunch &l, cudaStream_t stream)
    {
        auto launch = [&](auto kernel, int ctas, int threads, int smem) {
            cudaLaunchConfig_t config{};
            config.gridDim = dim3(static_cast<unsigned int>(l.grid), 1, static_cast<unsigned int>(l.splits));
            config.blockDim = dim3(static_cast<unsigned int>(threads));
            config.dynamicSmemBytes = static_cast<size_t>(smem);
            config.stream = stream;
            cudaLaunchAttribute attributes[2]{};
            attributes[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
            attributes[0].val.programmaticStreamSerializationAllowed = 1;
            attributes[1].id = cudaLaunchAttributeClusterDimension;
            attributes[1].val.clusterDim.x = static_cast<unsigned int>(ctas);
            attributes[1].val.clusterDim.y = 1;
            attributes[1].val.clusterDim.z = static_cast<unsigned int>(l.splits);
            config.attrs = attributes;
            config.numAttrs = ctas > 1 || l.splits > 1 ? 2 : 1;
            return cudaLaunchKernelEx(&config, kernel, l.map_a, l.map_b, l.map_c, l.map_z, l.p);
        };
        return l.p.direct ? with_direct(l.tile, l.epilogue, launch) : with_kernel(l.layout, l.tile, l.epilogue, launch);
    }

    static cudaError_t act_grad(const ActGradParams &params, dim3 grid, int cluster, cudaStream_t stream)
    {
        cudaLaunchConfig_t config{};
        config.gridDim = grid;
        config.blockDim = dim3(AG_THREADS);
        config.stream = stream;
        cudaLaunchAttribute attributes[2]{};
        attributes[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attributes[0].val.programmaticStreamSerializationAllowed = 1;
        attributes[1].id = cudaLaunchAttributeClusterDimension;
        attributes[1].val.clusterDim.x = 1;
        attributes[1].val.clusterDim.y = static_cast<unsigned int>(cluster);
        attributes[1].val.clusterDim.z = 1;
        config.attrs = attributes;
        config.numAttrs = 2;
        return cudaLaunchKernelEx(&config, act_grad_kernel<FMT>, params);
    }

    static cudaError_t bias_grad(const float *partial, int count, int n, void *dbias, int dbias_half,
                                 cudaStream_t stream)
    {
        return launch_pdl(bias_grad_kernel<FMT>, dim3(static_cast<unsigned int>((n + 255) / 256)), dim3(256), 0, stream,
                          partial, count, n, dbias, dbias_half);
    }

    static cudaError_t repack(const RepackJob &job0, const RepackJob &job1, int sms, cudaStream_t stream)
    {
        const int64_t units = job0.units + job1.units, cap = 32LL * sms;
        return launch_pdl(repack_kernel<static_cast<int>(sizeof(T))>,
                          dim3(static_cast<unsigned int>(units < cap ? units : cap)), dim3(RP_THREADS), 0, stream, job0,
                          job1);
    }

    static cudaError_t chunk_sum(const ChunkSumParams &params, int sms, cudaStream_t stream)
    {
        const int64_t blocks = (static_cast<int64_t>(params.rows) * ((params.cols + 3) / 4) + 255) / 256, cap = 8LL * sms;
        return launch_pdl(chunk_sum_kernel<FMT>, dim3(static_cast<unsigned int>(blocks < cap ? blocks : cap)), dim3(256), 0,
                          stream, params);
    }

    static constexpr OpKernels kTable{setup, product, act_grad, bias_grad, repack, chunk_sum};
};

} // namespace b200
