// Small kernels around the operators' products (tc_ops.cuh): the tile plan of grouped
// products and the join of the loss's per-tile maxima and sums.  Both are bound by
// launch latency.  Included by ops.cu alone.
#pragma once

#include <cuda.h>
#include <cstdint>

#include "ptx.cuh"
#include "tc_ops.cuh"

namespace b200 {

// ---------------------------------------------------------------- plan of a grouped product
constexpr int GP_THREADS = 256;
constexpr int GP_WARPS = GP_THREADS / 32;

struct GroupPlanParams {
    const void *offsets;      // groups + 1 row offsets
    int offsets64;
    int groups, rows;
    int tile_rows;            // rows mode: rows per tile; 0: one entry per group (ragged-K mode)
    int maps;                 // tensor maps per group (0, 1 or 2)
    int *count;               // number of row tiles
    OpRowTile *tiles;
    CUtensorMap *group_maps;  // [groups][maps]
    // Ragged-K mode: the first tile of each of `units` CTAs or pairs (and the end).
    int units;
    int *unit_first;
    long long tiles_per_group;
    int k_block;              // rows per K block
};

// A tile's epilogue in K blocks, for the shares of ragged-K mode.  Too little for a tile of an empty group, which
// takes as long as one of a small group: the stores of either (about 5000 cycles a pair).  Units whose share
// lies in empty groups finish last (32 groups of 256 rows on average, four of them empty, 2048 x 1408 outputs:
// 181000 cycles, 112000 on average).
constexpr int GP_EPILOGUE_BLOCKS = 6;

// Group g's rows are [max(offsets[0..g]), max(offsets[0..g+1])) clipped to
// [0, rows], so that whatever the offsets hold, groups are disjoint, in order and in
// range.  Rows mode writes ceil(rows of g / tile_rows) entries per group, in order, one
// thread a group; ragged-K mode one entry per group (`unused` = K blocks and epilogues of a
// tile of each group before it, summed) and each unit's share: consecutive tiles of about
// the same total weight, so that a unit meets few groups (each costs it two tensor-map
// fences before its loads can start: with tiles dealt out in turn, 64 groups of 256 rows
// took 420 us on 2048 x 2816 outputs).  Each group's tensor maps are the templates with the
// row extent cut at the group's end.  Every block computes the ends; block 0 writes the
// tables, all blocks share the maps.
__global__ void __launch_bounds__(GP_THREADS) group_plan_kernel(const __grid_constant__ CUtensorMap map0,
                                                                const __grid_constant__ CUtensorMap map1,
                                                                const __grid_constant__ CUtensorMap map2,
                                                                const __grid_constant__ GroupPlanParams first_plan,
                                                                const __grid_constant__ GroupPlanParams second_plan)
{
    // Blocks of the second row make the second plan (a backward pass has two), with map2 alone.
    const GroupPlanParams &p = blockIdx.y ? second_plan : first_plan;
    __shared__ int warp_max[GP_WARPS], warp_sum[GP_WARPS];
    __shared__ int carry_max, carry_sum;
    __shared__ int ends[GP_THREADS];
    __shared__ __align__(128) uint8_t map_s[GP_WARPS][128];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    wait_for_prior_grid();
    allow_next_grid();
    auto offset = [&](int i) {
        const long long v = p.offsets64 ? static_cast<const long long *>(p.offsets)[i]
                                        : static_cast<long long>(static_cast<const int *>(p.offsets)[i]);
        return static_cast<int>(v < 0 ? 0 : v > p.rows ? p.rows : v);
    };
    if (threadIdx.x == 0) {
        carry_max = offset(0);
        carry_sum = 0;
    }
    __syncthreads();
    for (int g0 = 0; g0 < p.groups; g0 += GP_THREADS) {
        const int g = g0 + threadIdx.x;
        // Running maximum of the ends.
        int end = g < p.groups ? offset(g + 1) : 0;
        for (int d = 1; d < 32; d <<= 1) {
            const int o = __shfl_up_sync(0xffffffffu, end, d);
            if (lane >= d)
                end = max(end, o);
        }
        if (lane == 31)
            warp_max[warp] = end;
        __syncthreads();
        int before = carry_max;
        for (int i = 0; i < warp; ++i)
            before = max(before, warp_max[i]);
        end = max(end, before);
        ends[threadIdx.x] = end;
        __syncthreads();
        const int begin = threadIdx.x ? ends[threadIdx.x - 1] : carry_max;
        const int count = g >= p.groups    ? 0
                          : p.tile_rows ? (end - begin + p.tile_rows - 1) / p.tile_rows
                                        : (end - begin + p.k_block - 1) / p.k_block + GP_EPILOGUE_BLOCKS;
        // Running sum of the tile counts.
        int sum = count;
        for (int d = 1; d < 32; d <<= 1) {
            const int o = __shfl_up_sync(0xffffffffu, sum, d);
            if (lane >= d)
                sum += o;
        }
        if (lane == 31)
            warp_sum[warp] = sum;
        __syncthreads();
        int first = carry_sum + sum - count;
        for (int i = 0; i < warp; ++i)
            first += warp_sum[i];
        if (g < p.groups && blockIdx.x == 0) {
            if (p.tile_rows) {
                for (int i = 0; i < count; ++i)
                    p.tiles[first + i] = OpRowTile{g, begin + i * p.tile_rows, end, 0};
            } else {
                p.tiles[g] = OpRowTile{g, begin, end, first};
            }
        }
        // Tensor maps of this chunk's groups, one warp each.
        for (int i = warp + GP_WARPS * static_cast<int>(blockIdx.x);
             i < GP_THREADS * p.maps && g0 + i / p.maps < p.groups; i += GP_WARPS * static_cast<int>(gridDim.x)) {
            const uint32_t s = smem_addr(map_s[warp]);
            const int local = i / p.maps;
            const uint32_t *src = reinterpret_cast<const uint32_t *>(blockIdx.y               ? &map2
                                                                    : i - local * p.maps ? &map1
                                                                                         : &map0);
            reinterpret_cast<uint32_t *>(map_s[warp])[lane] = src[lane];
            __syncwarp();
            if (lane == 0) {
                const uint32_t extent = static_cast<uint32_t>(max(ends[local], 1));
                asm volatile("tensormap.replace.tile.global_dim.shared::cta.b1024.b32 [%0], 1, %1;" ::"l"(
                                 static_cast<uint64_t>(s)),
                             "r"(extent)
                             : "memory");
            }
            __syncwarp();
            asm volatile(
                "tensormap.cp_fenceproxy.global.shared::cta.tensormap::generic.release.gpu.sync.aligned "
                "[%0], [%1], 128;" ::"l"(reinterpret_cast<uint64_t>(p.group_maps + static_cast<int64_t>(g0) * p.maps + i)),
                "r"(s)
                : "memory");
            __syncwarp();
        }
        __syncthreads();
        if (threadIdx.x == GP_THREADS - 1) {
            carry_max = end;
            carry_sum = first + count;
        }
        __syncthreads();
    }
    if (blockIdx.x != 0)
        return;
    if (p.tile_rows) {
        if (threadIdx.x == 0)
            *p.count = carry_sum;
        return;
    }
    // Unit u starts at the first tile at or past u / units of all tiles' weight.
    for (int u = threadIdx.x; u <= p.units; u += GP_THREADS) {
        const long long total = carry_sum * p.tiles_per_group;
        const long long target = total / p.units * u + total % p.units * u / p.units;
        int lo = 0, hi = p.groups;          // the last group that starts at or before the target
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (p.tiles[mid].unused * p.tiles_per_group <= target)
                lo = mid;
            else
                hi = mid;
        }
        const int before = p.tiles[lo].unused;
        const int weight = (lo + 1 < p.groups ? p.tiles[lo + 1].unused : carry_sum) - before;
        const long long local = (target - before * p.tiles_per_group + weight - 1) / weight;
        p.unit_first[u] = static_cast<int>(lo * p.tiles_per_group + min(local, p.tiles_per_group));
    }
}

// ---------------------------------------------------------------- loss
constexpr int LJ_WARPS = 32;

// lse = log sum exp over the column ranges' (maximum, sum) pairs, loss = lse - the label's
// logit.  A block takes 32 rows, each warp every 32nd range: the maximum
// first, then the sums scaled to it (loads and exponentials without a chain through
// them), joined over the warps in a fixed order.  A range's sum is NaN where a logit was.
__global__ void __launch_bounds__(32 * LJ_WARPS) loss_join_kernel(const float2 *partial, int ranges,
                                                                  const float *label_logit, float *loss, float *lse,
                                                                  const OpParams p)
{
    __shared__ float tops[LJ_WARPS][32], sums[LJ_WARPS][32];
    wait_for_prior_grid();
    allow_next_grid();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int row = static_cast<int>(blockIdx.x) * 32 + lane;
    const float2 *column = partial + min(row, p.m - 1);
    float top = -INFINITY;
#pragma unroll 4
    for (int i = warp; i < ranges; i += LJ_WARPS)
        top = fmaxf(top, column[static_cast<long long>(i) * p.m].x);
    tops[warp][lane] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < LJ_WARPS; ++i)
        top = fmaxf(top, tops[i][lane]);
    const bool far = op_far(top);
    const float origin = far ? op_far_origin(top) : op_origin(top);
    float sum = 0.0f;
#pragma unroll 4
    for (int i = warp; i < ranges; i += LJ_WARPS) {
        const float2 v = column[static_cast<long long>(i) * p.m];
        sum += v.y * exp2f(far ? (v.x - origin) * kLog2E : __fmul_rn(v.x, kLog2E) - origin);
    }
    sums[warp][lane] = sum;
    __syncthreads();
    if (warp == 0 && row < p.m) {
        sum = 0.0f;
#pragma unroll
        for (int i = 0; i < LJ_WARPS; ++i)
            sum += sums[i][lane];
        // Far from zero the logarithm of the sum is below half a step of the maximum: the loss takes
        // the maximum's distance from the label's logit first.
        constexpr float kLn2 = 0.69314718055994531f;
        const float rest = log2f(sum), total = far ? top + rest * kLn2 : (origin + rest) * kLn2;
        const int label = op_label(p, row);
        lse[row] = total;
        if (label < 0)
            loss[row] = label == -1 ? 0.0f : __int_as_float(0x7fc00000);
        else
            loss[row] = far ? (top - label_logit[row]) + rest * kLn2 : total - label_logit[row];
    }
}

} // namespace b200
