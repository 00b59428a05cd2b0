// Tensor-core product with a fused epilogue, the main loop of the operators next to
// matmul_launch (ops.cu): D = Aop * Bop, FP32 accumulation in tensor memory, where
//
//   * either operand may be stored with its K index contiguous ("K-major") or its
//     M/N index contiguous ("MN-major"), so A.B, A.B^T and A^T.B of row-major
//     matrices are read in place;
//   * the rows may belong to groups (experts) of any size, each with its own B:
//     - rows mode: a row tile lies in one group, whose table entry names the group,
//       its first row and the end of its rows;
//     - ragged-K mode (gradient of B): one product per group over the group's rows.
//       Operand tensor maps of that group end at its last row, so TMA fills the
//       rest of a K block with zeros and no value of a neighbour enters a sum;
//   * a long K may be cut into chunks whose FP32 products are added up by a second
//     kernel (few output tiles, as in the gradient of a few rows through a vocabulary);
//   * the epilogue applies bias, activation and residual, reduces each row to a
//     maximum and a sum of exponentials (loss), or turns logits into gradients.
//
// Roles, rings, bounded waits and the pair protocol are those of tc2_gemm.cuh (CTAS
// = 2: one 256 x BN tile per CTA pair, each CTA staging half of either operand) and
// tc_gemm.cuh (CTAS = 1: 128 x BN).  Operand maps are four-dimensional (inner, rows,
// column block, group): a coordinate past a group's own K rows reads zeros, not the next
// group.  An MN-major operand whose columns are whole 128-byte blocks is one load per
// stage.  A 16-bit weight that TMA cannot address may be loaded by extra warps (DIRECT).
//
// Measured choices stand at the host's plan (ops.cu).
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cstdint>
#include <type_traits>

#include "ptx.cuh"

namespace b200 {

enum OpFormat : int { kOpF16 = 0, kOpBF16 = 1, kOpTF32 = 2 };
enum OpEpilogue : int {
    kEpiStore = 0,      // out = act(D + bias) + residual, D's rows are out's rows
    kEpiStoreT = 1,     // the same, D's rows are out's columns (few rows: they take the MMA's N side)
    kEpiLse = 2,        // per row: maximum and sum of exponentials of this tile's columns, label's logit
    kEpiSoftmaxGrad = 3 // out = (exp(D - lse) - [column == label]) * grad
};
enum OpActivation : int { kActNone = 0, kActRelu = 1, kActGelu = 2, kActGeluTanh = 3, kActSilu = 4 };
enum OpGrouping : int { kUngrouped = 0, kGroupedRows = 1, kGroupedK = 2, kChunkedK = 3 };

// Status bits of the device status word (matmul_device_status).
enum : unsigned int { kOpLoadTimeout = 1u, kOpMmaTimeout = 2u, kOpEpilogueTimeout = 4u, kOpDrainTimeout = 8u };

constexpr int OP_BM = 128;                    // M rows per CTA (TMEM lanes)
constexpr int OP_ROW_BYTES = 128;             // one swizzle row: K depth of a stage (K-major)
constexpr int OP_A_STAGE = OP_BM * OP_ROW_BYTES;
constexpr int OP_BOX = 128 * 128;             // epilogue box: 128 rows x 128 bytes
constexpr int OP_BAR_BYTES = 512;

// Geometry of a tile of BN N columns on one CTA or a pair, with two accumulators.  Tiles
// of 128 columns and more have two epilogue warpgroups, each with half of the columns:
// one warpgroup needs longer for an activation and two outputs than the MMAs of a
// 4096-deep 256 x 256 tile (4096 x 4096 x 14336 BF16 with gelu, bias and pre-activation:
// 609 us with one, 496 us with two).  A 256 x 512 pair tile (one accumulator, freed half
// by half, as in tc2_gemm.cuh) was built and taken out: once one elected thread issued the
// instructions it was ahead of 256 x 256 by 1 % at most, where its count of tiles fits the
// pairs better.
//
// DIRECT: B (16-bit, 128 columns a tile) has rows that start on any element, which TMA
// cannot address.  Two more warps fetch the aligned 16-byte pieces that a K block's rows lie
// in through kRaw buffers, eight more shift them into the place where TMA would have
// written them.  For few rows of A, whose products are too short to hide a copy of B behind
// (direct_pays).  Bound by the shifting: 2 to 4 TB/s of B where TMA reads an aligned one at
// 5.
template <int CTAS, int BN, bool DIRECT = false>
struct OpTile {
    static constexpr int kBCols = BN / CTAS;                   // N columns staged per CTA
    static constexpr int kBStage = kBCols * OP_ROW_BYTES;
    static constexpr int kStages = DIRECT ? 3 : kBCols >= 128 ? 5 : 8;
    static constexpr int kGroups = BN >= 128 ? 2 : 1;          // epilogue warpgroups
    static constexpr int kFirstEpi = kGroups == 2 ? 4 : 2;     // first epilogue warp (after TMA, MMA, two idle ones)
    static constexpr int kFirstLoader = kFirstEpi + 4 * kGroups;
    static constexpr int kFetchers = DIRECT ? 2 : 0, kShifters = DIRECT ? 8 : 0;   // warps
    static constexpr int kThreads = 32 * (kFirstLoader + kFetchers + kShifters);
    static constexpr int kRaw = DIRECT ? (BN >= 128 ? 7 : 8) : 0;
    static constexpr int kRawPitch = 17 * 16;                  // a row's 128 16-bit columns at any skew
    static constexpr int kRawBytes = 64 * kRawPitch;
    static constexpr int kBoxes = 2;                           // boxes per epilogue warpgroup
    static constexpr int kEpiBytes = DIRECT ? 0 : kBoxes * kGroups * OP_BOX;   // none in these epilogues
    static constexpr int kBiasBytes = BN * 4 < 256 ? 256 : BN * 4;
    static constexpr int kSmem = 1024 + kStages * (OP_A_STAGE + kBStage) + kEpiBytes + OP_BAR_BYTES + kBiasBytes +
                                 kRaw * kRawBytes;
    static constexpr uint32_t kTmemColumns = 2 * BN < 32 ? 32 : 2 * BN;   // two accumulators
    static_assert(kSmem <= 227 * 1024, "tile exceeds shared memory");
};

// A row tile of a grouped product: group, first row, end of the group's rows.
struct OpRowTile {
    int group, row0, row_end, unused;
};

// One lane of a converged warp.  The roles that issue TMA and tensor-core instructions
// branch on this rather than on a lane number, so that the compiler knows that a single
// thread holds their operands.
__device__ __forceinline__ bool op_elect_one()
{
    uint32_t elected;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "elect.sync _|p, 0xffffffff;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(elected));
    return elected != 0;
}

// Division by a divisor the host knows (Granlund and Montgomery's multiply-and-shift for
// 32-bit numbers): quotients of numbers below 2^31.
struct OpDivisor {
    uint32_t magic, shift;
    int value;
};

__device__ __forceinline__ int op_divide(int x, const OpDivisor &d)
{
    const uint32_t t = __umulhi(d.magic, static_cast<uint32_t>(x));
    return d.value == 1 ? x : static_cast<int>((t + ((static_cast<uint32_t>(x) - t) >> 1)) >> d.shift);
}

struct OpParams {
    int m, n;                 // rows and columns of the output (of one group in ragged-K mode)
    int num_m_blocks, num_n_blocks, num_k_blocks;   // M- and N-side tiles of D, K blocks
    int num_tiles;
    int full_tiles;           // pairs: from here on two indices name the column halves of one tile
    int log_raster;           // log2 of the M-side tiles per raster group
    OpDivisor per_raster;     // raster x N-side tiles (transposed epilogue: M-side tiles)
    OpDivisor per_group;      // ragged-K and chunked-K modes: tiles of one group or chunk
    int chunk_blocks;         // chunked-K mode: K blocks per chunk
    uint32_t stage_tx;        // bytes that the TMA loads of a K block bring
    const void *direct;       // DIRECT: B (K x n, rows without padding)
    int k;                    // DIRECT: its rows
    int grouping;             // OpGrouping
    int a_blocked, b_blocked; // MN-major operands: 1 when their map sees blocks of 128 bytes of columns
    const int *row_tile_count;        // rows mode: number of row tiles (device)
    const OpRowTile *row_tiles;       // rows mode: table of row tiles; ragged-K mode: one entry per group
    const CUtensorMap *group_maps;    // rows mode: out's map per group; ragged-K mode: Aop's and Bop's
    const int *unit_first;            // ragged-K mode: the first tile of each CTA or pair, and the end
    int groups;
    // kEpiStore / kEpiStoreT / kEpiSoftmaxGrad
    void *out;
    long long out_pitch, out_slab;    // elements between rows / between groups' outputs
    int out_half;                     // 1: the 16-bit input format, 0: FP32
    int out_tma;                      // 1: TMA can write out, and its rows and the residual's start on 16 bytes
    void *preact;                     // D + bias before the activation, or null
    long long preact_pitch;
    int preact_half, preact_tma;
    const void *residual;             // null, or added after the activation (pitch out_pitch)
    int residual_half;
    int residual_tma;                 // 1: TMA brings it (map_z; out's format, no pre-activation)
    const void *bias;                 // n values or null
    int bias_half;
    int activation;
    // kEpiLse / kEpiSoftmaxGrad
    const void *labels;
    int labels64;
    int column0;                      // vocabulary index of column 0
    long long ignore;
    long long classes;                // vocabulary size: labels outside [0, classes) that are not `ignore` give NaN
    float2 *partial;                  // [n tiles x epilogue groups][m]: maximum logit, sum of exponentials from it
    float *label_logit;               // [m]
    const float *lse, *grad;          // [m]
    unsigned int *status;
    unsigned long long wait_limit_ns;
};

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const void *map, uint32_t bar, int x, int y, int z, int w)
{
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z), "r"(w)
        : "memory");
}

// The load of a CTA pair: `bar` may be the other CTA's barrier.
__device__ __forceinline__ void tma_load_4d_pair(uint32_t dst, const void *map, uint32_t bar, int x, int y, int z, int w)
{
    asm volatile(
        "cp.async.bulk.tensor.4d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z), "r"(w)
        : "memory");
}

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const void *map, uint32_t bar, int x, int y, int z)
{
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z)
        : "memory");
}

__device__ __forceinline__ void tma_store_3d(const void *map, uint32_t src, int x, int y, int z)
{
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(
                     reinterpret_cast<uint64_t>(map)),
                 "r"(src), "r"(x), "r"(y), "r"(z)
                 : "memory");
}

// Arrives on an mbarrier of a CTA of this cluster with CTA-scope release: what the
// arrival reports is that this warp's TMEM loads have completed (tcgen05.wait::ld).  A
// cluster-scope release also waits for the stores this thread has under way, 1700 of the
// 7100 cycles of a 256 x 256 tile with K = 256.
__device__ __forceinline__ void mbar_arrive_remote(uint32_t cluster_addr)
{
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}

// 64 consecutive FP32 columns of this thread's TMEM lane, waited for in the same asm block.
__device__ __forceinline__ void tmem_load_64cols(uint32_t taddr, float (&v)[64])
{
    uint32_t(&u)[64] = reinterpret_cast<uint32_t(&)[64]>(v);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x64.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, "
        "%32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, "
        "%48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63}, [%64];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]),
          "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15]), "=r"(u[16]),
          "=r"(u[17]), "=r"(u[18]), "=r"(u[19]), "=r"(u[20]), "=r"(u[21]), "=r"(u[22]), "=r"(u[23]), "=r"(u[24]),
          "=r"(u[25]), "=r"(u[26]), "=r"(u[27]), "=r"(u[28]), "=r"(u[29]), "=r"(u[30]), "=r"(u[31]), "=r"(u[32]),
          "=r"(u[33]), "=r"(u[34]), "=r"(u[35]), "=r"(u[36]), "=r"(u[37]), "=r"(u[38]), "=r"(u[39]), "=r"(u[40]),
          "=r"(u[41]), "=r"(u[42]), "=r"(u[43]), "=r"(u[44]), "=r"(u[45]), "=r"(u[46]), "=r"(u[47]), "=r"(u[48]),
          "=r"(u[49]), "=r"(u[50]), "=r"(u[51]), "=r"(u[52]), "=r"(u[53]), "=r"(u[54]), "=r"(u[55]), "=r"(u[56]),
          "=r"(u[57]), "=r"(u[58]), "=r"(u[59]), "=r"(u[60]), "=r"(u[61]), "=r"(u[62]), "=r"(u[63])
        : "r"(taddr)
        : "memory");
}

// A tensor map written by an earlier kernel is read through the tensor-map proxy.
__device__ __forceinline__ void tensormap_acquire(const void *map)
{
    asm volatile("fence.proxy.tensormap::generic.acquire.gpu [%0], 128;" ::"l"(reinterpret_cast<uint64_t>(map))
                 : "memory");
}

template <int FMT>
struct OpType;
template <>
struct OpType<kOpF16> {
    using T = __half;
    static __device__ __forceinline__ float to(T x) { return __half2float(x); }
    static __device__ __forceinline__ T from(float x) { return __float2half_rn(x); }
    static __device__ __forceinline__ uint32_t pack(float lo, float hi)
    {
        const __half2 v = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<const uint32_t *>(&v);
    }
};
template <>
struct OpType<kOpBF16> {
    using T = __nv_bfloat16;
    static __device__ __forceinline__ float to(T x) { return __bfloat162float(x); }
    static __device__ __forceinline__ T from(float x) { return __float2bfloat16_rn(x); }
    static __device__ __forceinline__ uint32_t pack(float lo, float hi)
    {
        const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t *>(&v);
    }
};
template <>
struct OpType<kOpTF32> {
    using T = float;
    static __device__ __forceinline__ float to(T x) { return x; }
    static __device__ __forceinline__ T from(float x) { return x; }
    static __device__ __forceinline__ uint32_t pack(float, float) { return 0u; }   // no 16-bit form
};

// 2^x by the hardware's approximation (relative error below 2^-22; results below the
// smallest normal number are zero).
__device__ __forceinline__ float op_exp2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// 1 / x by the hardware's approximation (1 ulp; zero for results below the smallest normal
// number).
__device__ __forceinline__ float op_reciprocal(float x)
{
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// The normal distribution function, Phi(-a) = exp(-a^2 / 2) t q(t) with t = 1 / (1 + 0.3 a), a = |z|: the form of
// Hastings's approximations of erf (Abramowitz and Stegun, Handbook of Mathematical Functions, 7.1.26), with a
// polynomial q of degree 7 fitted here for the least relative error over 0 <= a <= 14 (1.5e-7).  In FP32
// the lower tail is off by 6e-7 of itself near 0, 9e-7 at z = -3 and 1.5e-6 at -5 (the exponent's rounding), where
// 7.1.26 itself, whose error is small against 1, was off by 7e-7, 5e-5 and 1.6e-3.  Two values at a time: the
// polynomial and products are packed FP32 instructions, half the instructions of erff.  `e` receives
// exp(-z^2 / 2).
__device__ __forceinline__ float2 op_normal_cdf(float2 z, float2 &e)
{
    constexpr float kQ[] = {0.11962930f, 0.12075395f, 0.099913500f, 0.12856160f,
                            -0.053683590f, 0.20635344f, -0.15720305f, 0.035674766f};
    const float2 a = make_float2(fabsf(z.x), fabsf(z.y));
    const float2 d = __ffma2_rn(make_float2(0.3f, 0.3f), a, make_float2(1.0f, 1.0f));
    const float2 t = make_float2(op_reciprocal(d.x), op_reciprocal(d.y));
    const float2 x = __fmul2_rn(__fmul2_rn(a, make_float2(-0.72134752f, -0.72134752f)), a);   // -z^2 / 2 log2 e
    e = make_float2(op_exp2(x.x), op_exp2(x.y));
    float2 q = make_float2(kQ[7], kQ[7]);
#pragma unroll
    for (int i = 6; i >= 0; --i)
        q = __ffma2_rn(t, q, make_float2(kQ[i], kQ[i]));
    const float2 tail = __fmul2_rn(__fmul2_rn(t, q), e);       // Phi(-a)
    return make_float2(z.x < 0.0f ? tail.x : 1.0f - tail.x, z.y < 0.0f ? tail.y : 1.0f - tail.y);
}

// act(z) of two values in FP32.  relu keeps NaN; gelu_tanh uses 0.5 (1 + tanh u) = 1 / (1
// + exp(-2u)).
template <int ACT>
__device__ __forceinline__ float2 op_activation(float2 z)
{
    if constexpr (ACT == kActRelu)
        return make_float2(z.x < 0.0f ? 0.0f : z.x, z.y < 0.0f ? 0.0f : z.y);
    if constexpr (ACT == kActGelu) {
        float2 e;
        return __fmul2_rn(z, op_normal_cdf(z, e));
    }
    if constexpr (ACT == kActGeluTanh) {
        // -2 u log2 e = z (-2.3022082 - 0.10294324 z^2)
        const float2 p = __ffma2_rn(__fmul2_rn(z, z), make_float2(-0.10294324f, -0.10294324f),
                                    make_float2(-2.3022082f, -2.3022082f));
        const float2 x = __fmul2_rn(z, p);
        return make_float2(z.x * op_reciprocal(1.0f + op_exp2(x.x)), z.y * op_reciprocal(1.0f + op_exp2(x.y)));
    }
    if constexpr (ACT == kActSilu) {
        const float2 x = __fmul2_rn(z, make_float2(-1.44269504f, -1.44269504f));
        return make_float2(z.x * op_reciprocal(1.0f + op_exp2(x.x)), z.y * op_reciprocal(1.0f + op_exp2(x.y)));
    }
    return z;
}

// act'(z) of two values in FP32.
template <int ACT>
__device__ __forceinline__ float2 op_activation_slope(float2 z)
{
    const float2 one = make_float2(1.0f, 1.0f);
    if constexpr (ACT == kActRelu)
        return make_float2(z.x > 0.0f ? 1.0f : 0.0f, z.y > 0.0f ? 1.0f : 0.0f);
    if constexpr (ACT == kActGelu) {
        float2 e;
        const float2 cdf = op_normal_cdf(z, e);
        return __ffma2_rn(__fmul2_rn(z, make_float2(0.39894228f, 0.39894228f)), e, cdf);
    }
    if constexpr (ACT == kActGeluTanh) {
        // Beyond 64 the slope is 0 or 1 to all its bits: |z| is held there, since z^2 could be infinite. NaN
        // comes through x.
        const float2 a = make_float2(fminf(fabsf(z.x), 64.0f), fminf(fabsf(z.y), 64.0f));
        const float2 zz = __fmul2_rn(a, a);
        const float2 x = __fmul2_rn(z, __ffma2_rn(zz, make_float2(-0.10294324f, -0.10294324f),
                                                  make_float2(-2.3022082f, -2.3022082f)));
        const float2 s = make_float2(op_reciprocal(1.0f + op_exp2(x.x)), op_reciprocal(1.0f + op_exp2(x.y)));
        const float2 du = __ffma2_rn(zz, make_float2(0.21406446f, 0.21406446f), make_float2(1.59576912f, 1.59576912f));
        const float2 rest = __ffma2_rn(make_float2(-s.x, -s.y), s, s);         // s (1 - s)
        return __ffma2_rn(__fmul2_rn(make_float2(copysignf(a.x, z.x), copysignf(a.y, z.y)), rest), du, s);
    }
    if constexpr (ACT == kActSilu) {
        const float2 x = __fmul2_rn(z, make_float2(-1.44269504f, -1.44269504f));
        const float2 s = make_float2(op_reciprocal(1.0f + op_exp2(x.x)), op_reciprocal(1.0f + op_exp2(x.y)));
        const float2 rest = __ffma2_rn(make_float2(-s.x, -s.y), s, s);
        return __ffma2_rn(z, rest, s);
    }
    return one;
}

// The activation of N values (N even).
template <int ACT, int N>
__device__ __forceinline__ void op_activate(float (&v)[N])
{
#pragma unroll
    for (int j = 0; j < N; j += 2) {
        const float2 y = op_activation<ACT>(make_float2(v[j], v[j + 1]));
        v[j] = y.x;
        v[j + 1] = y.y;
    }
}

// Calls f with the activation as a constant, so that loops over it hold no branch (with
// the branch inside, 4096 x 4096 x 14336 BF16 with silu took 577 us, 386 us without it).
template <typename F>
__device__ __forceinline__ void op_with_activation(int act, F &&f)
{
    switch (act) {
    case kActRelu: f(std::integral_constant<int, kActRelu>{}); break;
    case kActGelu: f(std::integral_constant<int, kActGelu>{}); break;
    case kActGeluTanh: f(std::integral_constant<int, kActGeluTanh>{}); break;
    case kActSilu: f(std::integral_constant<int, kActSilu>{}); break;
    default: f(std::integral_constant<int, kActNone>{}); break;
    }
}

// A row's label: its column, -1 for an ignored row, -2 for a label outside the vocabulary.
__device__ __forceinline__ int op_label(const OpParams &p, int row)
{
    const long long y = p.labels64 ? static_cast<const long long *>(p.labels)[row]
                                   : static_cast<long long>(static_cast<const int *>(p.labels)[row]);
    if (y == p.ignore)
        return -1;
    return y >= 0 && y < p.classes ? static_cast<int>(y) : -2;
}

// Exponentials of logits are taken in base 2, exp(z - top) = 2^(z log2 e - origin) with origin = top log2 e: one
// FMA a logit, and the origin's rounding is in every term and in the result alike.  From 2^126 on a maximum is
// far: its origin may be infinite, so the maximum is taken off first, exp(z - top) = 2^((z - top) log2 e).
// Such logits are those of columns masked with the format's lowest value (or -infinity, from which nothing is
// taken off).  An origin below -2^127 is held there, where its terms are zero.
constexpr float kLog2E = 1.44269504f;

__device__ __forceinline__ bool op_far(float top)
{
    return fabsf(top) > 0x1p126f;
}

__device__ __forceinline__ float op_origin(float top)
{
    return fmaxf(__fmul_rn(top, kLog2E), -0x1p127f);
}

__device__ __forceinline__ float op_far_origin(float top)
{
    return top == -INFINITY ? 0.0f : top;
}

// Where a tile of D lies: M-side and N-side origin, group, K blocks and K origin, and
// the end of the output rows it may write.
struct OpWhere {
    int m0, n0, group, nkb, k0, row_end;
    int n_block;
    int cols;          // columns of the tile: BN, or half of it
};

template <int CTAS, int BN, bool SWAP>
__device__ __forceinline__ OpWhere op_where(int tile, int row_tile_count, int bk, const OpParams &p)
{
    constexpr int kBM = OP_BM * CTAS;
    OpWhere w;
    int half = 0;
    w.cols = BN;
    if (CTAS == 2 && tile >= p.full_tiles) {
        half = (tile - p.full_tiles) & 1;
        tile = p.full_tiles + ((tile - p.full_tiles) >> 1);
        w.cols = BN / 2;
    }
    int local = tile;
    w.group = 0;
    w.k0 = 0;
    w.nkb = p.num_k_blocks;
    w.row_end = p.m;
    if (p.grouping == kGroupedK) {
        w.group = op_divide(tile, p.per_group);
        local = tile - w.group * p.per_group.value;
        const OpRowTile t = p.row_tiles[w.group];
        w.k0 = t.row0;
        w.nkb = (t.row_end - t.row0 + bk - 1) / bk;
    } else if (p.grouping == kChunkedK) {
        w.group = op_divide(tile, p.per_group);
        local = tile - w.group * p.per_group.value;
        const int first = w.group * p.chunk_blocks;
        w.k0 = first * bk;
        w.nkb = min(p.chunk_blocks, p.num_k_blocks - first);
    }
    int mb, nb;
    if constexpr (SWAP) {       // all M-side tiles (columns) of a row tile, then the next
        nb = op_divide(local, p.per_raster);
        mb = local - nb * p.per_raster.value;
    } else {
        // Raster groups of 2^log_raster M-side tiles, so that the CTAs at work share panels in L2.
        const int blocks_m = p.grouping == kGroupedRows ? row_tile_count : p.num_m_blocks;
        const int rg = op_divide(local, p.per_raster);
        const int first = rg << p.log_raster;
        const int in_group = local - rg * p.per_raster.value;
        const int rows = blocks_m - first;
        if (rows >> p.log_raster) {
            nb = in_group >> p.log_raster;
            mb = first + (in_group & ((1 << p.log_raster) - 1));
        } else {
            nb = in_group / rows;
            mb = first + in_group - nb * rows;
        }
    }
    w.m0 = mb * kBM;
    w.n0 = nb * BN + half * (BN / 2);
    w.n_block = nb;
    if (p.grouping == kGroupedRows) {
        const OpRowTile t = p.row_tiles[SWAP ? nb : mb];
        w.group = t.group;
        w.row_end = t.row_end;
        (SWAP ? w.n0 : w.m0) = t.row0;
    }
    return w;
}

// 16 bytes from an address aligned to ELEM bytes: words where it starts on 4 bytes, else a
// half word, three words and a half word shifted into place, so that nothing outside the
// 16 bytes is read.
template <int ELEM>
__device__ __forceinline__ uint4 load_16_bytes(const uint8_t *from)
{
    uint4 q;
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
    return q;
}

// 16 bytes that start `skew` (even) bytes into lo, the rest from hi.
__device__ __forceinline__ uint4 skewed_16_bytes(const uint4 &lo, const uint4 &hi, uint32_t skew)
{
    uint32_t w0 = lo.x, w1 = lo.y, w2 = lo.z, w3 = lo.w, w4 = hi.x, w5 = hi.y, w6 = hi.z;
    if (skew & 8) {
        w0 = w2;
        w1 = w3;
        w2 = w4;
        w3 = w5;
        w4 = w6;
        w5 = hi.w;
    }
    if (skew & 4) {
        w0 = w1;
        w1 = w2;
        w2 = w3;
        w3 = w4;
        w4 = w5;
    }
    const uint32_t bits = 8 * (skew & 3);
    return make_uint4(__funnelshift_r(w0, w1, bits), __funnelshift_r(w1, w2, bits), __funnelshift_r(w2, w3, bits),
                      __funnelshift_r(w3, w4, bits));
}

// The aligned 16 bytes at `at`; what lies outside [begin, end) is not read and zero.
__device__ __forceinline__ uint4 load_16_within(uintptr_t at, uintptr_t begin, uintptr_t end)
{
    if (at >= begin && at + 16 <= end)
        return *reinterpret_cast<const uint4 *>(at);
    uint32_t words[4] = {};
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (at + 2 * e >= begin && at + 2 * e + 2 <= end)
            words[e / 2] |= static_cast<uint32_t>(*reinterpret_cast<const uint16_t *>(at + 2 * e)) << (16 * (e & 1));
    return make_uint4(words[0], words[1], words[2], words[3]);
}

template <int FMT, int CTAS, int BN, bool A_MN, bool B_MN, int EPI, bool DIRECT = false>
__global__ void __launch_bounds__(OpTile<CTAS, BN, DIRECT>::kThreads, 1)
op_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
          const __grid_constant__ CUtensorMap map_c, const __grid_constant__ CUtensorMap map_z,
          const __grid_constant__ OpParams p)
{
    using Tile = OpTile<CTAS, BN, DIRECT>;
    using Type = OpType<FMT>;
    using T = typename Type::T;
    constexpr bool kPair = CTAS == 2;
    constexpr bool kSwap = EPI == kEpiStoreT;
    constexpr bool kTF32 = FMT == kOpTF32;
    constexpr int kThreads = Tile::kThreads;
    constexpr int kFirstLoader = Tile::kFirstLoader;
    constexpr int kElem = kTF32 ? 4 : 2;
    constexpr int kBK = OP_ROW_BYTES / kElem;             // K elements per stage (64 or 32)
    constexpr int kMmaK = 32 / kElem;
    constexpr int kMmasPerStage = kBK / kMmaK;            // 4
    constexpr int kBox = OP_ROW_BYTES / kElem;            // M/N elements per MN-major box
    constexpr uint32_t kBoxBytes = kBK * OP_ROW_BYTES;    // one MN-major box
    constexpr int kStages = Tile::kStages;
    constexpr int kBStage = Tile::kBStage;
    constexpr int kBCols = Tile::kBCols;
    constexpr int kGroups = Tile::kGroups;
    constexpr int kBoxes = Tile::kBoxes;
    constexpr bool kSplittable = CTAS == 1 && (EPI == kEpiStore || EPI == kEpiStoreT);
    constexpr int kGroupCols = BN / kGroups;              // D columns per epilogue warpgroup
    constexpr uint32_t kIdescHalfN = static_cast<uint32_t>((BN / 2) >> 3) << 17;
    // FP32 accumulator, formats, A MN-major (bit 15), B MN-major (bit 16), N >> 3, M >> 4.
    constexpr uint32_t kIdesc = (1u << 4) | (static_cast<uint32_t>(FMT) << 7) | (static_cast<uint32_t>(FMT) << 10) |
                                ((A_MN ? 1u : 0u) << 15) | ((B_MN ? 1u : 0u) << 16) |
                                (static_cast<uint32_t>(BN >> 3) << 17) |
                                (static_cast<uint32_t>((OP_BM * CTAS) >> 4) << 24);
    static_assert(!B_MN || kBCols % kBox == 0, "whole MN-major boxes");
    static_assert(!kPair || !kSwap, "the transposed epilogue runs on single CTAs");
    static_assert(!DIRECT || (!kPair && !kTF32 && (kSwap || (B_MN && BN == 128))), "128 columns of B per CTA");

    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_addr(smem_raw);
    const uint32_t base = (raw + 1023u) & ~1023u;
    const uint32_t s_a = base;
    const uint32_t s_b = s_a + kStages * OP_A_STAGE;
    const uint32_t s_epi = s_b + kStages * kBStage;
    const uint32_t s_bar = s_epi + Tile::kEpiBytes;
    const uint32_t s_bias = s_bar + OP_BAR_BYTES;
    auto full_bar = [&](int s) { return s_bar + 8u * s; };
    auto empty_bar = [&](int s) { return s_bar + 8u * (kStages + s); };
    auto accf_bar = [&](int i) { return s_bar + 8u * (2 * kStages + i); };
    auto acce_bar = [&](int i) { return s_bar + 8u * (2 * kStages + 2 + i); };
    const uint32_t drain_bar = s_bar + 8u * (2 * kStages + 4);
    const uint32_t tmem_slot = s_bar + 8u * (2 * kStages + 5);
    const uint32_t recv_bar = s_bar + 8u * (2 * kStages + 6);   // split K: partial rows received
    auto direct_bar = [&](int s) { return s_bar + 8u * (2 * kStages + 12 + s); };     // DIRECT: B's part of a stage
    auto raw_full_bar = [&](int i) { return s_bar + 8u * (3 * kStages + 12 + i); };   // its buffers on the way there
    auto raw_empty_bar = [&](int i) { return s_bar + 8u * (3 * kStages + 12 + Tile::kRaw + i); };
    static_assert(8 * (3 * kStages + 12 + 2 * Tile::kRaw) <= OP_BAR_BYTES && kGroups * kBoxes <= 4, "barriers fit");
    const uint32_t fail_flag = s_bar + 8u * (2 * kStages + 7);  // split K: 1 once a progress wait of this CTA ran out
    volatile uint32_t *fail_flag_ptr = reinterpret_cast<volatile uint32_t *>(smem_raw + (fail_flag - raw));
    uint32_t *tmem_slot_ptr = reinterpret_cast<uint32_t *>(smem_raw + (tmem_slot - raw));
    float *bias_s = reinterpret_cast<float *>(smem_raw + (s_bias - raw));

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const uint32_t rank = kPair ? cluster_cta_rank() : 0u;
    const bool leader = rank == 0;
    const int unit = static_cast<int>(blockIdx.x) / CTAS;       // this CTA's or pair's first tile
    const int units = static_cast<int>(gridDim.x) / CTAS;
    // Split K (clusters of S CTAs along z, one tile per cluster, ungrouped): CTA z runs K
    // blocks [z * ceil(nk / S), (z + 1) * ceil(nk / S)).
    const int splits = kSplittable ? static_cast<int>(gridDim.z) : 1;
    const int kb_per_split = (p.num_k_blocks + splits - 1) / splits;
    const int kb_begin = splits > 1 ? min(static_cast<int>(blockIdx.z) * kb_per_split, p.num_k_blocks) : 0;
    auto kb_end = [&](int nkb) { return splits > 1 ? min(nkb, kb_begin + kb_per_split) : nkb; };

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(full_bar(s), 1);
            mbar_init(empty_bar(s), 1);
            if constexpr (DIRECT)
                mbar_init(direct_bar(s), Tile::kShifters / 2);
        }
        for (int i = 0; i < Tile::kRaw; ++i) {
            mbar_init(raw_full_bar(i), 32 * Tile::kFetchers);
            mbar_init(raw_empty_bar(i), Tile::kShifters / 2);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(accf_bar(i), 1);
            mbar_init(acce_bar(i), 4 * CTAS * kGroups);
        }
        mbar_init(drain_bar, 1);
        mbar_init(recv_bar, 1);
        for (int i = 0; i < kGroups * Tile::kBoxes; ++i)
            mbar_init(s_bar + 8u * (2 * kStages + 8 + i), 1);
        *fail_flag_ptr = 0u;
        fence_mbarrier_init();
    }
    if (warp == 0 && lane == 0) {
        if constexpr (!DIRECT || !kSwap)
            tma_prefetch_map(&map_a);
        if constexpr (!DIRECT || kSwap)
            tma_prefetch_map(&map_b);
    }
    if (warp == 1) {
        if constexpr (kPair) {
            tmem_alloc_pair(tmem_slot, Tile::kTmemColumns);
            tmem_relinquish_pair();
        } else {
            tmem_alloc(tmem_slot, Tile::kTmemColumns);
            tmem_relinquish();
        }
    }
    tc_fence_before();
    if constexpr (kPair)
        cluster_sync_all();        // both CTAs' barriers exist before either signals the other
    else
        __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *reinterpret_cast<volatile uint32_t *>(tmem_slot_ptr);
    wait_for_prior_grid();
    allow_next_grid();

    auto load_bias = [&](int col) {
        return p.bias_half ? Type::to(static_cast<const T *>(p.bias)[col]) : static_cast<const float *>(p.bias)[col];
    };
    // The epilogue of `count` elements (row + i * row_step, col + i * col_step), i < N, from
    // D + bias, with plain loads and stores.
    auto store_elements = [&](auto &v, int count, int row, int col, int row_step, int col_step) {
        constexpr int N = std::extent<std::remove_reference_t<decltype(v)>>::value;
        const long long at = row * p.out_pitch + col, step = row_step * p.out_pitch + col_step;
        if (p.preact) {
            const long long z_at = row * p.preact_pitch + col, z_step = row_step * p.preact_pitch + col_step;
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (i < count) {
                    if (p.preact_half)
                        static_cast<T *>(p.preact)[z_at + i * z_step] = Type::from(v[i]);
                    else
                        static_cast<float *>(p.preact)[z_at + i * z_step] = v[i];
                }
        }
        op_with_activation(p.activation, [&](auto act) {
            op_activate<decltype(act)::value>(v);
        });
        if (p.residual) {
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (i < count)
                    v[i] += p.residual_half ? Type::to(static_cast<const T *>(p.residual)[at + i * step])
                                            : static_cast<const float *>(p.residual)[at + i * step];
        }
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (i < count) {
                if (p.out_half)
                    static_cast<T *>(p.out)[at + i * step] = Type::from(v[i]);
                else
                    static_cast<float *>(p.out)[at + i * step] = v[i];
            }
    };

    // NaN over rows x cols elements of the outputs, clipped, one warp per row.
    auto nan_elements = [&](const OpWhere &w, int first_row, int rows, int first_col, int cols, int warp_index,
                            int warps, int lane_index) {
        const float nan = __int_as_float(0x7fc00000);
        const int row_end = min(w.row_end, first_row + rows), col_end = min(p.n, first_col + cols);
        for (int row = first_row + warp_index; row < row_end; row += warps)
            for (int col = first_col + lane_index; col < col_end; col += 32) {
                const long long at = (p.grouping >= kGroupedK ? w.group : 0) * p.out_slab + row * p.out_pitch + col;
                if (p.out_half)
                    static_cast<T *>(p.out)[at] = Type::from(nan);
                else
                    static_cast<float *>(p.out)[at] = nan;
                if (EPI != kEpiSoftmaxGrad && p.preact) {
                    const long long z_at = row * p.preact_pitch + col;
                    if (p.preact_half)
                        static_cast<T *>(p.preact)[z_at] = Type::from(nan);
                    else
                        static_cast<float *>(p.preact)[z_at] = nan;
                }
            }
    };

    const int row_tile_count = p.grouping == kGroupedRows ? *p.row_tile_count : 0;
    const int num_tiles = p.grouping == kGroupedRows ? row_tile_count * (kSwap ? p.num_m_blocks : p.num_n_blocks)
                                                     : p.num_tiles;
    // Tiles are dealt out in turn; in ragged-K mode each unit has consecutive ones.
    const bool in_turn = p.grouping != kGroupedK;
    const int tile_first = in_turn ? unit : p.unit_first[unit];
    const int tile_end = in_turn ? num_tiles : p.unit_first[unit + 1];
    const int tile_step = in_turn ? units : 1;

    if (warp == 0) {
        // ------------------------------------------------------------ producer
        if (op_elect_one()) {
            int stage = 0;
            uint32_t phase = 0, filled = 0, fill_parity = 0;
            bool ok = true;
            int acquired = -1;     // ragged-K mode: the group whose maps this thread has acquired
            const uint32_t leader_full0 = kPair ? map_to_cta(full_bar(0), 0) : full_bar(0);
            for (int tile = tile_first; ok && tile < tile_end; tile += tile_step) {
                const OpWhere w = op_where<CTAS, BN, kSwap>(tile, row_tile_count, kBK, p);
                const void *ma = &map_a, *mb = &map_b;
                int za = 0, zb = 0;
                if (p.grouping == kGroupedK) {
                    ma = p.group_maps + 2 * w.group;
                    mb = p.group_maps + 2 * w.group + 1;
                    if (acquired != w.group) {
                        tensormap_acquire(ma);
                        tensormap_acquire(mb);
                        acquired = w.group;
                    }
                } else if (p.grouping == kGroupedRows) {
                    (kSwap ? za : zb) = w.group;
                }
                int am = w.m0 + static_cast<int>(rank) * OP_BM;
                // Half a pair's tile past its group's rows: a coordinate past the matrix reads zeros, no
                // memory, where the next group's rows would cost loads and power for nothing.
                if (!A_MN && p.grouping == kGroupedRows && !kSwap && am >= w.row_end)
                    am = p.m;
                // Half a tile's columns are the first halves of the same boxes.
                const int bn = w.n0 + static_cast<int>(rank) * (w.cols / CTAS);
                for (int kb = kb_begin; kb < kb_end(w.nkb); ++kb) {
                    // In a pair this wait keeps the fixed limit: both CTAs then stop at the
                    // same stage and the leader's drain covers every copy of either.
                    if (!mbar_wait(empty_bar(stage), phase ^ 1u, kPair ? kWaitLimitNs : p.wait_limit_ns)) {
                        atomicOr(p.status, kOpLoadTimeout);
                        ok = false;
                        break;
                    }
                    const uint32_t fb = leader_full0 + 8u * stage;
                    if (leader)
                        mbar_arrive_expect_tx(full_bar(stage), p.stage_tx);
                    const int k = w.k0 + kb * kBK;
                    auto load = [&](uint32_t dst, const void *map, int x, int y, int block, int z) {
                        if constexpr (kPair)
                            tma_load_4d_pair(dst, map, fb, x, y, block, z);
                        else
                            tma_load_4d(dst, map, fb, x, y, block, z);
                    };
                    // `cols` M/N columns from `mn` on, as MN-major boxes: one load, or one per box.
                    auto load_mn = [&](uint32_t dst, const void *map, bool blocked, int mn, int cols, int z) {
                        if (blocked) {
                            load(dst, map, 0, k, mn / kBox, z);
                        } else {
                            for (int j = 0; j < cols / kBox; ++j)
                                load(dst + j * kBoxBytes, map, mn + j * kBox, k, 0, z);
                        }
                    };
                    const uint32_t sa = s_a + stage * OP_A_STAGE, sb = s_b + stage * kBStage;
                    if constexpr (DIRECT && kSwap)
                        ;
                    else if constexpr (A_MN)
                        load_mn(sa, ma, p.a_blocked != 0, am, OP_BM, za);
                    else
                        load(sa, ma, k, am, 0, za);
                    if constexpr (DIRECT && !kSwap)
                        ;
                    else if constexpr (B_MN)
                        load_mn(sb, mb, p.b_blocked != 0, bn, kBCols, zb);
                    else
                        load(sb, mb, k, bn, 0, zb);
                    filled |= 1u << stage;
                    fill_parity = (fill_parity & ~(1u << stage)) | (phase << stage);
                    if (++stage == kStages) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
            }
            // Every issued copy lands before a CTA can exit.
            if (leader)
                for (int s = 0; s < kStages; ++s)
                    if ((filled >> s) & 1u)
                        if (!mbar_wait(full_bar(s), (fill_parity >> s) & 1u))
                            atomicOr(p.status, kOpDrainTimeout);
        }
        __syncwarp();
    } else if (warp == 1) {
        // ------------------------------------------------------------ MMA issuer (a pair's leader)
        if (leader && op_elect_one()) {
            int stage = 0;
            uint32_t phase = 0;
            const uint64_t a_desc0 = A_MN ? smem_desc_mn<kTF32>(s_a, kBoxBytes) : smem_desc_sw128(s_a, 16, 1024);
            const uint64_t b_desc0 = B_MN ? smem_desc_mn<kTF32>(s_b, kBoxBytes) : smem_desc_sw128(s_b, 16, 1024);
            constexpr uint64_t kAStep = A_MN ? (kMmaK * OP_ROW_BYTES) >> 4 : 32 >> 4;
            constexpr uint64_t kBStep = B_MN ? (kMmaK * OP_ROW_BYTES) >> 4 : 32 >> 4;
            auto commit = [&](uint32_t bar) {
                if constexpr (kPair)
                    tc_commit_pair_both(bar, 3);
                else
                    tc_commit(bar);
            };
            auto arrive_both = [&](uint32_t bar) {
                if constexpr (kPair) {
                    mbar_arrive_cluster(map_to_cta(bar, 0));
                    mbar_arrive_cluster(map_to_cta(bar, 1));
                } else {
                    mbar_arrive(bar);
                }
            };
            int acc = 0;
            uint32_t acc_phase = 0;
            bool ok = true;
            for (int tile = tile_first; ok && tile < tile_end; tile += tile_step) {
                const OpWhere w = op_where<CTAS, BN, kSwap>(tile, row_tile_count, kBK, p);
                if (!mbar_wait(acce_bar(acc), acc_phase ^ 1u, p.wait_limit_ns)) {
                    atomicOr(p.status, kOpMmaTimeout);
                    break;
                }
                tc_fence_after();
                const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(acc * BN);
                const uint32_t idesc = kPair && w.cols != BN ? kIdesc - kIdescHalfN : kIdesc;     // half the N
                const int nkb = kb_end(w.nkb);
                for (int kb = kb_begin; kb < nkb; ++kb) {
                    bool here = mbar_wait(full_bar(stage), phase, p.wait_limit_ns);
                    if constexpr (DIRECT)
                        here = here && mbar_wait(direct_bar(stage), phase, p.wait_limit_ns);
                    if (!here) {
                        atomicOr(p.status, kOpMmaTimeout);
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint64_t a_desc = a_desc0 + static_cast<uint64_t>(stage) * (OP_A_STAGE >> 4);
                    const uint64_t b_desc = b_desc0 + static_cast<uint64_t>(stage) * (kBStage >> 4);
#pragma unroll
                    for (int kk = 0; kk < kMmasPerStage; ++kk) {
                        const uint32_t accumulate = kb != kb_begin || kk != 0 ? 1u : 0u;
                        if constexpr (kPair)
                            tc_mma_pair<kTF32>(d_tmem, a_desc + kk * kAStep, b_desc + kk * kBStep, idesc, accumulate);
                        else
                            tc_mma<kTF32>(d_tmem, a_desc + kk * kAStep, b_desc + kk * kBStep, idesc, accumulate);
                    }
                    commit(empty_bar(stage));
                    if (++stage == kStages) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
                if (!ok)
                    break;
                if (nkb > kb_begin) {
                    commit(accf_bar(acc));
                } else {          // no K block (an empty group or split): a zero sum, nothing to wait for
                    arrive_both(accf_bar(acc));
                }
                if (++acc == 2) {
                    acc = 0;
                    acc_phase ^= 1u;
                }
            }
            // Every MMA issued above completes before TMEM is released.
            if constexpr (kPair)
                tc_commit_pair(drain_bar);
            else
                tc_commit(drain_bar);
            if (!mbar_wait(drain_bar, 0))
                atomicOr(p.status, kOpDrainTimeout);
        }
        __syncwarp();
    } else if (DIRECT && warp >= kFirstLoader) {
        // ------------------------------------------------------------ B without TMA
        // Some warps fetch, others shift: threads that did both (copy, shift, fence.proxy.async) took
        // 1900 cycles a K block however many were in flight (product 8 x 4096 x 14337: 55 us, 37 so).
        if constexpr (DIRECT) {
            constexpr int kRaw = Tile::kRaw, kPieces = 17 * 64;
            constexpr int kFetching = 32 * Tile::kFetchers, kShifting = 16 * Tile::kShifters;    // threads per K block
            const uint32_t s_raw = s_bias + Tile::kBiasBytes;
            const uintptr_t begin = reinterpret_cast<uintptr_t>(p.direct);
            const uintptr_t row_bytes = static_cast<uintptr_t>(p.n) * 2;
            const int kb_last = kb_end(p.num_k_blocks);
            int buffer = 0;
            uint32_t buffer_phase = 0;
            bool ok = true;
            if (warp < kFirstLoader + Tile::kFetchers) {
                const int thread = static_cast<int>(threadIdx.x) - 32 * kFirstLoader;
                const uintptr_t end = begin + static_cast<uintptr_t>(p.k) * row_bytes;
                // 64 rows, and 128 columns, are multiples of 16 bytes: a thread's pieces lie alike in every K
                // block of every tile.
                constexpr int kMine = (kPieces + kFetching - 1) / kFetching;
                uintptr_t source[kMine];
                uint32_t place[kMine];
#pragma unroll
                for (int j = 0; j < kMine; ++j) {
                    const int at = min(thread + j * kFetching, kPieces - 1), row = at / 17, piece = at - row * 17;
                    source[j] = ((begin + row * row_bytes) & ~uintptr_t{15}) + 16 * piece;
                    place[j] = s_raw + row * Tile::kRawPitch + piece * 16;
                }
                for (int tile = tile_first; ok && tile < tile_end; tile += tile_step) {
                    const OpWhere w = op_where<CTAS, BN, kSwap>(tile, row_tile_count, kBK, p);
                    const int column = kSwap ? w.m0 : w.n0;
                    for (int kb = kb_begin; kb < kb_last; ++kb) {
                        if (!mbar_wait(raw_empty_bar(buffer), buffer_phase ^ 1u, p.wait_limit_ns)) {
                            atomicOr(p.status, kOpLoadTimeout);
                            ok = false;
                            break;
                        }
                        const uintptr_t block = static_cast<uintptr_t>(kb) * kBK * row_bytes + static_cast<uintptr_t>(column) * 2;
                        const uint32_t to = buffer * Tile::kRawBytes;
                        const int rows = min(64, p.k - kb * kBK);
                        // Away from both ends of the matrix every piece is whole, or behind the last row.
                        if (block >= 16 && begin + block + (rows - 1) * row_bytes + 17 * 16 <= end) {
#pragma unroll
                            for (int j = 0; j < kMine; ++j) {
                                const int at = thread + j * kFetching;
                                if (j == kMine - 1 && at >= kPieces)
                                    break;
                                const bool inside = rows == 64 || at < 17 * rows;
                                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(place[j] + to),
                                             "l"(inside ? source[j] + block : begin & ~uintptr_t{15}), "r"(inside ? 16 : 0)
                                             : "memory");
                            }
                            asm volatile("cp.async.mbarrier.arrive.noinc.shared.b64 [%0];" ::"r"(raw_full_bar(buffer))
                                         : "memory");
                        } else {
#pragma unroll 1
                            for (int i = thread; i < kPieces; i += kFetching) {
                                const int row = i / 17, piece = i - row * 17;
                                const uintptr_t at = ((begin + row * row_bytes) & ~uintptr_t{15}) + 16 * piece + block;
                                const uint32_t dst = s_raw + to + row * Tile::kRawPitch + piece * 16;
                                if (kb * kBK + row < p.k && at >= begin && at + 16 <= end) {
                                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(at) : "memory");
                                } else {
                                    const uint4 v = kb * kBK + row < p.k ? load_16_within(at, begin, end)
                                                                         : make_uint4(0u, 0u, 0u, 0u);
                                    st_shared_v4(dst, v.x, v.y, v.z, v.w);
                                }
                            }
                            asm volatile("cp.async.wait_all;" ::: "memory");
                            mbar_arrive(raw_full_bar(buffer));
                        }
                        if (++buffer == kRaw) {
                            buffer = 0;
                            buffer_phase ^= 1u;
                        }
                    }
                }
                asm volatile("cp.async.wait_all;" ::: "memory");
            } else {
                // Two sets of warps take K blocks in turn.
                const int shifter = static_cast<int>(threadIdx.x) - 32 * (kFirstLoader + Tile::kFetchers);
                const int thread = shifter % kShifting, set = shifter / kShifting;
                int turn = 0;
                const uint32_t skew = static_cast<uint32_t>(begin + (thread >> 4) * row_bytes) & 15u;
                int stage = 0;
                uint32_t phase = 0;
                for (int tile = tile_first; ok && tile < tile_end; tile += tile_step) {
                    for (int kb = kb_begin; kb < kb_last; ++kb) {
                        const bool mine = turn == set;
                        turn ^= 1;
                        if (mine) {
                            int ready = 0;
                            if (lane == 0)
                                ready = mbar_wait(empty_bar(stage), phase ^ 1u, p.wait_limit_ns) &&
                                                mbar_wait(raw_full_bar(buffer), buffer_phase, p.wait_limit_ns)
                                            ? 1
                                            : 0;
                            ready = __shfl_sync(0xffffffffu, ready, 0);
                            // Every thread waits by itself for what it reads (this one is complete).
                            if (!ready || !mbar_wait(raw_full_bar(buffer), buffer_phase, p.wait_limit_ns)) {
                                if (lane == 0)
                                    atomicOr(p.status, kOpLoadTimeout);
                                ok = false;
                                break;
                            }
                            const uint32_t from = s_raw + buffer * Tile::kRawBytes;
                            const uint32_t to = kSwap ? s_a + stage * OP_A_STAGE : s_b + stage * kBStage;
#pragma unroll
                            for (int i0 = 0; i0 < 64 * 16 / kShifting; i0 += 4) {
                                uint4 lo[4], hi[4];
#pragma unroll
                                for (int i = 0; i < 4; ++i) {
                                    const int at = thread + (i0 + i) * kShifting, row = at >> 4, piece = at & 15;
                                    const uint32_t src = from + row * Tile::kRawPitch + piece * 16;
                                    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                                                 : "=r"(lo[i].x), "=r"(lo[i].y), "=r"(lo[i].z), "=r"(lo[i].w)
                                                 : "r"(src));
                                    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                                                 : "=r"(hi[i].x), "=r"(hi[i].y), "=r"(hi[i].z), "=r"(hi[i].w)
                                                 : "r"(src + 16));
                                }
#pragma unroll
                                for (int i = 0; i < 4; ++i) {
                                    const int at = thread + (i0 + i) * kShifting, row = at >> 4, piece = at & 15;
                                    const uint4 v = skewed_16_bytes(lo[i], hi[i], skew);
                                    st_shared_v4(to + (piece >> 3) * kBoxBytes + row * OP_ROW_BYTES +
                                                     (((piece & 7) ^ (row & 7)) << 4),
                                                 v.x, v.y, v.z, v.w);
                                }
                            }
                            fence_proxy_async_shared();      // the tensor core reads these stores
                            __syncwarp();
                            if (lane == 0) {
                                mbar_arrive(direct_bar(stage));
                                mbar_arrive(raw_empty_bar(buffer));
                            }
                        }
                        if (++buffer == kRaw) {
                            buffer = 0;
                            buffer_phase ^= 1u;
                        }
                        if (++stage == kStages) {
                            stage = 0;
                            phase ^= 1u;
                        }
                    }
                }
            }
        }
    } else if (warp >= Tile::kFirstEpi) {
        // ------------------------------------------------------------ epilogue
        const int quarter = warp & 3;                 // TMEM lanes 32 * quarter .. +31
        const int r = quarter * 32 + lane;
        const int group = (warp - Tile::kFirstEpi) >> 2;   // epilogue warpgroup: D columns group * kGroupCols ..
        const int gthread = static_cast<int>(threadIdx.x) - 32 * Tile::kFirstEpi - 128 * group;
        // One thread of the warpgroup issues and waits for its TMA stores: the same lane at
        // every election (elect.sync is deterministic for a mask).
        const bool issuer_warp = gthread < 32;
        const bool issuer = issuer_warp && op_elect_one();
        const uint32_t s_box = s_epi + group * kBoxes * OP_BOX;
        // A warpgroup's own part whatever a tile's width is: the warpgroups do not wait for each other, so
        // one may be at the half tile after the other's whole one.
        float *group_bias = bias_s + group * kGroupCols;
        auto epilogue_sync = [&]() { asm volatile("bar.sync %0, 128;" ::"r"(1 + group) : "memory"); };
        // 1 only if every thread of the warpgroup passes 1.
        auto epilogue_all = [&](int ok) {
            uint32_t all;
            asm volatile(
                "{\n\t.reg .pred p, q;\n\t"
                "setp.ne.u32 p, %1, 0;\n\t"
                "bar.red.and.pred q, %2, 128, p;\n\t"
                "selp.u32 %0, 1, 0, q;\n\t}"
                : "=r"(all)
                : "r"(static_cast<uint32_t>(ok)), "r"(1 + group)
                : "memory");
            return static_cast<int>(all);
        };
        int acc = 0;
        uint32_t acc_phase = 0, stores = 0;
        int failed_tile = -1;
        int acquired = -1;
        // Residual boxes: loads issued and used, the parity of each box's next load, and boxes of
        // the current tile already stored.
        uint32_t res_issued = 0, res_used = 0, res_parity = 0, box_done = 0;
        auto res_bar = [&](uint32_t b) { return s_bar + 8u * (2 * kStages + 8 + group * kBoxes + b); };
        // Releases the accumulator after this warp's last read of it.
        auto release = [&]() {
            const uint32_t bar = acce_bar(acc);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if constexpr (kPair)
                    mbar_arrive_remote(map_to_cta(bar, 0));
                else
                    mbar_arrive(bar);
            }
        };
        for (int tile = tile_first; tile < tile_end; tile += tile_step) {
            const OpWhere w = op_where<CTAS, BN, kSwap>(tile, row_tile_count, kBK, p);
            const int row0 = w.m0 + static_cast<int>(rank) * OP_BM;     // D's first row in this CTA
            const int group_cols = kPair ? w.cols / kGroups : kGroupCols;
            const int gcol = group * group_cols;
            const uint32_t t_row = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) +
                                   static_cast<uint32_t>(acc * BN + gcol);
            if constexpr (EPI == kEpiStore) {
                if (p.bias) {       // the tile's bias, read once into shared memory
                    epilogue_sync();
                    for (int c = gthread; c < group_cols; c += 128) {
                        const int col = w.n0 + gcol + c;
                        float b = 0.0f;
                        if (col < p.n)
                            b = load_bias(col);
                        group_bias[c] = b;
                    }
                    epilogue_sync();
                }
            }
            // Per-row values of the loss epilogues.
            int label = -1;
            float row_lse = 0.0f, row_grad = 0.0f;
            if constexpr (EPI == kEpiLse || EPI == kEpiSoftmaxGrad) {
                if (row0 + r < p.m) {
                    label = op_label(p, row0 + r);
                    if constexpr (EPI == kEpiSoftmaxGrad) {
                        row_lse = p.lse[row0 + r];
                        row_grad = p.grad[row0 + r];
                    }
                }
            }
            // Residual by TMA: box u of this tile (32 FP32 or 64 16-bit columns) is loaded into the
            // shared-memory box that its result will leave from, one box ahead.
            const int box_cols = p.out_half ? 64 : 32;
            auto fetch = [&](int u) {
                const int col0 = w.n0 + gcol + u * box_cols;
                if (u * box_cols >= group_cols || col0 >= p.n || row0 >= w.row_end)
                    return;
                const uint32_t b = (stores + static_cast<uint32_t>(u) - box_done) % kBoxes;
                if (issuer_warp && op_elect_one()) {
                    bulk_wait_group_read<0>();      // the stores that last read the boxes
                    mbar_arrive_expect_tx(res_bar(b), OP_BOX);
                    tma_load_3d(s_box + b * OP_BOX, &map_z, res_bar(b), col0, row0, 0);
                }
                __syncwarp();
                ++res_issued;
            };
            box_done = 0;
            if constexpr (EPI == kEpiStore)
                if (p.residual_tma && splits == 1)
                    fetch(0);
            int ok = 1;
            if (issuer) {     // one thread polls, the others wait at the barrier
                // The tile's whole K loop: a microsecond a K block on top of the default limit (the longest
                // sums take 2^26 of them).
                const int blocks = max(kb_end(w.nkb) - kb_begin, 0);
                const uint64_t limit = p.wait_limit_ns < kWaitLimitNs ? p.wait_limit_ns : kWaitLimitNs + 1000ull * blocks;
                ok = mbar_wait(accf_bar(acc), acc_phase, limit) ? 1 : 0;
            }
            ok = epilogue_all(ok);
            if (!ok) {
                if (issuer) {
                    atomicOr(p.status, kOpEpilogueTimeout);
                    *fail_flag_ptr = 1u;
                }
                failed_tile = tile;
                break;
            }
            tc_fence_after();
            if (splits > 1)
                break;     // one tile; its partial sums are exchanged below

            if constexpr (EPI == kEpiStore || EPI == kEpiSoftmaxGrad) {
                const void *mc = &map_c;
                if (p.grouping == kGroupedRows && p.out_tma && row0 + OP_BM > w.row_end && row0 < w.row_end) {
                    // Rows of the next group in this tile: the group's own map clips them.
                    mc = p.group_maps + w.group;
                    if (issuer && acquired != w.group) {
                        tensormap_acquire(mc);
                        acquired = w.group;
                    }
                }
                const int zc = p.grouping >= kGroupedK ? w.group : 0;
                // Puts 128 bytes of this thread's row into a box of 128 rows.
                auto fill = [&](uint32_t box, const uint32_t (&words)[32]) {
                    const uint32_t row_addr = box + r * 128;
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        st_shared_v4(row_addr + ((j ^ (r & 7)) << 4), words[4 * j], words[4 * j + 1], words[4 * j + 2],
                                     words[4 * j + 3]);
                };
                // A box of 32 FP32 or 64 16-bit columns, stored by TMA.
                auto emit = [&](const uint32_t (&words)[32], const void *map, int z, int col0) {
                    const uint32_t box = s_box + stores % kBoxes * OP_BOX;
                    if (issuer)
                        bulk_wait_group_read<kBoxes - 1>();      // the store that last read this box
                    epilogue_sync();
                    fill(box, words);
                    fence_proxy_async_shared();
                    epilogue_sync();
                    __syncwarp();
                    if (issuer_warp && op_elect_one()) {
                        tma_store_3d(map, box, col0, row0, z);
                        bulk_commit_group();
                    }
                    __syncwarp();
                    ++stores;
                };
                // The same with the residual already in the box: each thread adds its own row to `v`,
                // puts the result in its place and the box is stored.  False where the residual did not come in
                // time: the box is not stored, and its loads are left to the drain below.
                auto emit_residual = [&](auto &v, const void *map, int col0) {
                    constexpr bool kShiftingBox = std::extent<std::remove_reference_t<decltype(v)>>::value == 64;
                    const uint32_t b = stores % kBoxes;
                    fetch(static_cast<int>(box_done) + 1);
                    const bool here = mbar_wait(res_bar(b), (res_parity >> b) & 1u, p.wait_limit_ns);
                    if (here) {
                        const uint32_t row_addr = s_box + b * OP_BOX + r * 128;
                        uint32_t words[32];
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const uint4 q =
                                *reinterpret_cast<const uint4 *>(smem_raw + (row_addr + ((j ^ (r & 7)) << 4) - raw));
                            if constexpr (kShiftingBox) {
                                const T *h = reinterpret_cast<const T *>(&q);
#pragma unroll
                                for (int e = 0; e < 4; ++e)
                                    words[4 * j + e] = Type::pack(v[8 * j + 2 * e] + Type::to(h[2 * e]),
                                                                  v[8 * j + 2 * e + 1] + Type::to(h[2 * e + 1]));
                            } else {
                                words[4 * j] = __float_as_uint(v[4 * j] + __uint_as_float(q.x));
                                words[4 * j + 1] = __float_as_uint(v[4 * j + 1] + __uint_as_float(q.y));
                                words[4 * j + 2] = __float_as_uint(v[4 * j + 2] + __uint_as_float(q.z));
                                words[4 * j + 3] = __float_as_uint(v[4 * j + 3] + __uint_as_float(q.w));
                            }
                        }
                        fill(s_box + b * OP_BOX, words);
                        fence_proxy_async_shared();
                    }
                    if (!epilogue_all(here ? 1 : 0))
                        return false;
                    res_parity ^= 1u << b;
                    ++res_used;
                    __syncwarp();
                    if (issuer_warp && op_elect_one()) {
                        tma_store_3d(map, s_box + b * OP_BOX, col0, row0, 0);
                        bulk_commit_group();
                    }
                    __syncwarp();
                    ++stores;
                    ++box_done;
                    return true;
                };
                // 128 bytes of each row, 32 FP32 or 64 16-bit columns, at any element alignment, without
                // TMA.  Each warp puts its own 32 rows into the boxes' memory at a pitch of 33 words,
                // then eight lanes take a row: a lane moves one 16-byte chunk that is aligned in memory
                // (words from shared memory, shifted by half a word where the row starts on an odd
                // element), and the up to 15 bytes at either end go element by element.  No bank
                // conflicts either way.  (One row per instruction with 4-byte words took 13000 cycles
                // for a 128 x 128 tile of 16-bit outputs.)
                auto emit_unaligned = [&](const uint32_t (&words)[32], bool half, void *dst, long long at0,
                                          long long pitch, int col0) {
                    if (p.out_tma | p.preact_tma) {       // the other output's boxes leave by TMA
                        if (issuer)
                            bulk_wait_group_read<0>();
                        epilogue_sync();
                    }
                    uint32_t *area = reinterpret_cast<uint32_t *>(smem_raw + (s_box - raw));
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        area[r * 33 + i] = words[i];
                    __syncwarp();
                    const int log_elem = half ? 1 : 2, per = 16 >> log_elem;
                    const int cols = min(128 >> log_elem, p.n - col0), rows = min(OP_BM, w.row_end - row0);
                    const int place = lane & 7, row_first = quarter * 32 + (lane >> 3);
                    uint8_t *base_row = static_cast<uint8_t *>(dst) + ((at0 + (row0 + row_first) * pitch + col0) << log_elem);
                    const long long row_step = (4 * pitch) << log_elem;
#pragma unroll 4
                    for (int it = 0; it < 8; ++it) {
                        const int rr = row_first + 4 * it;
                        uint8_t *to = base_row + it * row_step;
                        if (rr >= rows)
                            continue;
                        const uint32_t *row = area + rr * 33;
                        const int head = min(static_cast<int>((0u - static_cast<uint32_t>(reinterpret_cast<uintptr_t>(to))) & 15u) >> log_elem, cols);
                        const int whole = (cols - head) >> (4 - log_elem);        // aligned 16-byte chunks
                        const int ends = cols - (whole << (4 - log_elem));
                        if (place < whole) {
                            const int first = head + place * per;
                            uint4 q;
                            if (half) {
                                const uint32_t *x = row + (first >> 1);
                                const int shift = (first & 1) * 16;
                                q.x = __funnelshift_r(x[0], x[1], shift);
                                q.y = __funnelshift_r(x[1], x[2], shift);
                                q.z = __funnelshift_r(x[2], x[3], shift);
                                q.w = __funnelshift_r(x[3], x[4], shift);
                            } else {
                                const uint32_t *x = row + first;
                                q = make_uint4(x[0], x[1], x[2], x[3]);
                            }
                            *reinterpret_cast<uint4 *>(to + (first << log_elem)) = q;
                        }
                        // At most 8 elements, one a lane, but in the last columns of the matrix.
                        auto end_element = [&](int e) {
                            const int c = e < head ? e : e + (whole << (4 - log_elem));
                            if (half)
                                reinterpret_cast<uint16_t *>(to)[c] = reinterpret_cast<const uint16_t *>(row)[c];
                            else
                                reinterpret_cast<uint32_t *>(to)[c] = row[c];
                        };
                        if (place < ends)
                            end_element(place);
                        if (place + 8 < ends)
                            end_element(place + 8);
                    }
                    __syncwarp();
                };
                // Adds a residual that TMA cannot bring: eight lanes read a row, and each thread finds its own
                // in the memory that emit_unaligned uses after it (2048 x 256 x 4101 BF16 with gelu: 68 us
                // when the stores added it row by row, 35 us so).
                auto add_unaligned = [&](float (&v)[64], int col0) {
                    if (p.preact_tma) {
                        if (issuer)
                            bulk_wait_group_read<0>();
                        epilogue_sync();
                    }
                    uint32_t *area = reinterpret_cast<uint32_t *>(smem_raw + (s_box - raw));
                    const bool half = p.residual_half != 0;
                    const int log_elem = half ? 1 : 2, per = 16 >> log_elem;
                    const int rows = min(OP_BM, w.row_end - row0), place = lane & 7, row_first = quarter * 32 + (lane >> 3);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int first = col0 + 32 * h;
                        if (first >= p.n || (half && h))
                            break;
                        const int cols = min(128 >> log_elem, p.n - first) - place * per;     // from this lane's on
                        const uint8_t *base = static_cast<const uint8_t *>(p.residual) +
                                              (((row0 + row_first) * p.out_pitch + first + place * per) << log_elem);
                        const long long row_step = (4 * p.out_pitch) << log_elem;
#pragma unroll
                        for (int it0 = 0; it0 < 8; it0 += 4) {
                            uint4 q[4];
#pragma unroll
                            for (int it = 0; it < 4; ++it) {
                                const uint8_t *from = base + (it0 + it) * row_step;
                                q[it] = make_uint4(0u, 0u, 0u, 0u);
                                if (row_first + 4 * (it0 + it) >= rows)
                                    continue;
                                if (cols >= per) {
                                    q[it] = half ? load_16_bytes<2>(from) : load_16_bytes<4>(from);
                                } else {
                                    uint32_t words[4] = {};
#pragma unroll
                                    for (int e = 0; e < 8; ++e)
                                        if (e < cols) {
                                            if (half)
                                                words[e / 2] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t *>(from)[e])
                                                                << (16 * (e & 1));
                                            else if (e < 4)
                                                words[e & 3] = reinterpret_cast<const uint32_t *>(from)[e];
                                        }
                                    q[it] = make_uint4(words[0], words[1], words[2], words[3]);
                                }
                            }
#pragma unroll
                            for (int it = 0; it < 4; ++it) {
                                uint32_t *to = area + (row_first + 4 * (it0 + it)) * 33 + place * 4;
                                to[0] = q[it].x;
                                to[1] = q[it].y;
                                to[2] = q[it].z;
                                to[3] = q[it].w;
                            }
                        }
                        __syncwarp();
                        if (half) {
                            if constexpr (!kTF32) {
#pragma unroll
                                for (int i = 0; i < 32; ++i) {
                                    const uint32_t word = area[r * 33 + i];
                                    const T *x = reinterpret_cast<const T *>(&word);
                                    v[2 * i] += Type::to(x[0]);
                                    v[2 * i + 1] += Type::to(x[1]);
                                }
                            }
                        } else {
#pragma unroll
                            for (int i = 0; i < 32; ++i)
                                v[32 * h + i] += __uint_as_float(area[r * 33 + i]);
                        }
                        __syncwarp();
                    }
                };
                auto emit_columns = [&](const float (&v)[64], const void *map, int z, bool tma, bool half, void *dst,
                                        long long at0, long long pitch, int col0) {
                    uint32_t words[32];
                    if (half) {
#pragma unroll
                        for (int j = 0; j < 32; ++j)
                            words[j] = Type::pack(v[2 * j], v[2 * j + 1]);
                        if (tma)
                            emit(words, map, z, col0);
                        else
                            emit_unaligned(words, true, dst, at0, pitch, col0);
                    } else {
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            if (col0 + 32 * h >= p.n)
                                break;
#pragma unroll
                            for (int j = 0; j < 32; ++j)
                                words[j] = __float_as_uint(v[32 * h + j]);
                            if (tma)
                                emit(words, map, z, col0 + 32 * h);
                            else
                                emit_unaligned(words, false, dst, at0, pitch, col0 + 32 * h);
                        }
                    }
                };
                // 64 columns of this thread's row: epilogue arithmetic and stores.  False, for the whole
                // warpgroup, where a residual did not come in time.
                auto process = [&](float (&v)[64], int step) {
                    const int col0 = w.n0 + gcol + step * 64;
                    if (col0 >= p.n || row0 >= w.row_end)      // the same for all four warps
                        return true;
                    if constexpr (EPI == kEpiSoftmaxGrad) {
                        // dz = (exp(z - lse) - [column == label]) grad, rounded to the input format because
                        // both products that read it take operands of that format (an FP32 dz would take
                        // two of each, for its high and its low part); the gradients are off by about the
                        // square root of two of their own rounding.  The exponential is taken 2^24 times too
                        // large and grad as much too small, so that only their product, not the
                        // hardware's exponential, falls below the normal numbers.  An ignored row's
                        // gradient is zero whatever its logits are.
                        if (label == -1) {
#pragma unroll
                            for (int j = 0; j < 64; ++j)
                                v[j] = 0.0f;
                        } else {
                            const float scale = (label == -2 ? __int_as_float(0x7fc00000) : row_grad) * 0x1p-24f;
                            const float2 shift = make_float2(-row_lse, -row_lse), scale2 = make_float2(scale, scale);
#pragma unroll
                            for (int j = 0; j < 64; j += 2) {
                                const float2 d = __fadd2_rn(make_float2(v[j], v[j + 1]), shift);
                                const float2 t = __ffma2_rn(d, make_float2(1.44269504f, 1.44269504f), make_float2(24.0f, 24.0f));
                                const float2 q = __fmul2_rn(make_float2(op_exp2(t.x), op_exp2(t.y)), scale2);
                                v[j] = q.x;
                                v[j + 1] = q.y;
                            }
                            const int hit = label - p.column0 - col0;
                            if (hit >= 0 && hit < 64) {
#pragma unroll
                                for (int j = 0; j < 64; ++j)
                                    v[j] -= j == hit ? row_grad : 0.0f;
                            }
                        }
                    } else {
                        if (p.bias) {
                            const float4 *b4 = reinterpret_cast<const float4 *>(group_bias + step * 64);
#pragma unroll
                            for (int j = 0; j < 16; ++j) {
                                const float4 b = b4[j];
                                v[4 * j] += b.x;
                                v[4 * j + 1] += b.y;
                                v[4 * j + 2] += b.z;
                                v[4 * j + 3] += b.w;
                            }
                        }
                        if (p.preact)
                            emit_columns(v, &map_z, 0, p.preact_tma != 0, p.preact_half != 0, p.preact, 0,
                                         p.preact_pitch, col0);
                        op_with_activation(p.activation, [&](auto act) {
                            op_activate<decltype(act)::value>(v);
                        });
                        if (p.residual_tma) {
                            if (p.out_half) {
                                if constexpr (!kTF32)
                                    return emit_residual(v, mc, col0);
                            } else {
                                return emit_residual(reinterpret_cast<float(&)[32]>(v[0]), mc, col0) &&
                                       (col0 + 32 >= p.n ||
                                        emit_residual(reinterpret_cast<float(&)[32]>(v[32]), mc, col0 + 32));
                            }
                        }
                        // Where TMA writes out but does not bring the residual (a pre-activation takes its
                        // boxes, or it has another format), each thread reads its own row of it.
                        if (p.residual && !p.out_tma)
                            add_unaligned(v, col0);
                        else if (p.residual && row0 + r < w.row_end) {
                            const long long at = (row0 + r) * p.out_pitch + col0;
                            if (col0 + 64 <= p.n) {
                                if (p.residual_half) {
                                    if constexpr (!kTF32) {
                                        const uint4 *src = reinterpret_cast<const uint4 *>(static_cast<const T *>(p.residual) + at);
#pragma unroll
                                        for (int j = 0; j < 8; ++j) {
                                            const uint4 q = src[j];
                                            const T *h = reinterpret_cast<const T *>(&q);
#pragma unroll
                                            for (int e = 0; e < 8; ++e)
                                                v[8 * j + e] += Type::to(h[e]);
                                        }
                                    }
                                } else {
                                    const float4 *src = reinterpret_cast<const float4 *>(static_cast<const float *>(p.residual) + at);
#pragma unroll
                                    for (int j = 0; j < 16; ++j) {
                                        const float4 q = src[j];
                                        v[4 * j] += q.x;
                                        v[4 * j + 1] += q.y;
                                        v[4 * j + 2] += q.z;
                                        v[4 * j + 3] += q.w;
                                    }
                                }
                            } else {
#pragma unroll
                                for (int j = 0; j < 64; ++j)
                                    if (col0 + j < p.n)
                                        v[j] += p.residual_half ? Type::to(static_cast<const T *>(p.residual)[at + j])
                                                                : static_cast<const float *>(p.residual)[at + j];
                            }
                        }
                    }
                    emit_columns(v, mc, zc, p.out_tma != 0, p.out_half != 0, p.out, zc * p.out_slab, p.out_pitch, col0);
                    return true;
                };
                auto load = [&](float (&v)[64], int step) {
                    if (w.nkb > 0) {
                        tmem_load_64cols(t_row + step * 64, v);
                    } else {
#pragma unroll
                        for (int j = 0; j < 64; ++j)
                            v[j] = 0.0f;
                    }
                };
                bool stored = true;
#pragma unroll 1
                for (int step = 0; stored && step < group_cols / 64; ++step) {
                    float v[64];
                    load(v, step);
                    if (step == group_cols / 64 - 1)
                        release();
                    stored = process(v, step);
                }
                if (!stored) {
                    if (issuer)
                        atomicOr(p.status, kOpEpilogueTimeout);
                    failed_tile = tile;
                    break;
                }
            } else if constexpr (EPI == kEpiStoreT) {
                // D's rows are output columns: one lane per column, one store of 32 consecutive
                // elements per output row and warp.
                const int col = row0 + r;
                const float b = p.bias && col < p.n ? load_bias(col) : 0.0f;
#pragma unroll 1
                for (int chunk = 0; chunk < kGroupCols / 16; ++chunk) {
                    uint32_t u[16];
                    tmem_load_16cols(t_row + chunk * 16, u);
                    if (chunk == kGroupCols / 16 - 1)
                        release();
                    const int first = w.n0 + gcol + chunk * 16;
                    const int rows = min(16, w.row_end - first);
                    if (col >= p.n || rows <= 0)
                        continue;
                    float v[16];
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                        v[j] = __uint_as_float(u[j]) + b;
                    store_elements(v, rows, first, col, 1, 0);
                }
            } else {
                // One pass: running maximum and sum of exponentials, in base 2, of this row's
                // columns in the tile; columns past the vocabulary count as -infinity.
                float top = -INFINITY, origin = -0x1p127f, sum = 0.0f;
                bool held = true;
                const int row = row0 + r;
                const int chunks = min(kGroupCols / 32, (p.n - w.n0 - gcol + 31) / 32);   // below 1: none in the matrix
#pragma unroll 1
                for (int chunk = 0; chunk < chunks; ++chunk) {
                    uint32_t u[32];
                    tmem_load_32cols(t_row + chunk * 32, u);
                    const int col0 = w.n0 + gcol + chunk * 32;
                    const int hit = label - col0;
                    if (label >= 0 && hit >= 0 && hit < 32) {
                        float z = 0.0f;
#pragma unroll
                        for (int j = 0; j < 32; ++j)
                            z = j == hit ? __uint_as_float(u[j]) : z;
                        p.label_logit[row] = z;
                    }
                    float x[32], chunk_top = -INFINITY;
#pragma unroll
                    for (int j = 0; j < 32; ++j)
                        x[j] = __uint_as_float(u[j]);
                    if (col0 + 32 > p.n) {
#pragma unroll
                        for (int j = 0; j < 32; ++j)
                            x[j] = col0 + j < p.n ? x[j] : -INFINITY;
                    }
#pragma unroll
                    for (int j = 0; j < 32; ++j)
                        chunk_top = fmaxf(chunk_top, x[j]);
                    top = fmaxf(top, chunk_top);
                    // (Lanes past the matrix may hold anything.)
                    if (chunk == chunks - 1 && !__any_sync(0xffffffffu, op_far(top) && row < p.m)) {
                        release();
                        held = false;
                    }
                    // A row whose logits are all -infinity so far adds nothing; NaN is carried by the sum.
                    const float next_origin = op_origin(top);
                    sum *= op_exp2(origin - next_origin);
                    origin = next_origin;
                    const float2 scale = make_float2(kLog2E, kLog2E), minus = make_float2(-origin, -origin);
                    float2 chain[2] = {};
#pragma unroll
                    for (int j = 0; j < 32; j += 2) {
                        const float2 t = __ffma2_rn(make_float2(x[j], x[j + 1]), scale, minus);
                        chain[(j >> 1) & 1] = __fadd2_rn(chain[(j >> 1) & 1], make_float2(op_exp2(t.x), op_exp2(t.y)));
                    }
                    sum += (chain[0].x + chain[0].y) + (chain[1].x + chain[1].y);
                }
                if (held) {
                    // Rows with a far maximum take a second pass from it; the others keep their sums, so that
                    // no row's result depends on another row.
                    const float from = op_far_origin(top);
                    float far_sum = 0.0f;
#pragma unroll 1
                    for (int c = 0; c < 2 * chunks; ++c) {
                        uint32_t u[16];
                        tmem_load_16cols(t_row + c * 16, u);
                        const int cols = p.n - w.n0 - gcol - c * 16;
#pragma unroll
                        for (int j = 0; j < 16; ++j)
                            far_sum += j < cols ? op_exp2((__uint_as_float(u[j]) - from) * kLog2E) : 0.0f;
                    }
                    if (op_far(top))
                        sum = far_sum;
                    release();
                }
                if (row < p.m)
                    p.partial[static_cast<long long>(w.n_block * kGroups + group) * p.m + row] = make_float2(top, sum);
            }
            if (++acc == 2) {
                acc = 0;
                acc_phase ^= 1u;
            }
        }
        // Residual boxes that were fetched and not used (an accumulator or a residual that did not
        // come in time) land before the CTA can exit.
        for (; res_used != res_issued; ++res_used) {
            const uint32_t b = (stores + res_issued - res_used - 1) % kBoxes;
            if (!mbar_wait(res_bar(b), (res_parity >> b) & 1u))
                atomicOr(p.status, kOpDrainTimeout);
        }
        if (issuer) {
            if (failed_tile >= 0)
                bulk_wait_group<0>();      // the stored boxes are in memory before the NaN below
            else
                bulk_wait_group_read<0>();
        }
        __syncwarp();
        if (failed_tile >= 0 && splits == 1) {
            // NaN over what this CTA did not finish, so that no later step reads stale values.
            epilogue_sync();
            for (int tile = failed_tile; tile < tile_end; tile += tile_step) {
                const OpWhere w = op_where<CTAS, BN, kSwap>(tile, row_tile_count, kBK, p);
                const int row0 = w.m0 + static_cast<int>(rank) * OP_BM;
                if constexpr (EPI == kEpiLse) {
                    if (row0 + r < p.m)
                        p.partial[static_cast<long long>(w.n_block * kGroups + group) * p.m + row0 + r] =
                            make_float2(__int_as_float(0x7fc00000), __int_as_float(0x7fc00000));
                } else {
                    const int group_cols = kPair ? w.cols / kGroups : kGroupCols;
                    const int first = w.n0 + group * group_cols;
                    nan_elements(w, kSwap ? first : row0, kSwap ? group_cols : OP_BM, kSwap ? row0 : first,
                                 kSwap ? OP_BM : group_cols, quarter, 4, lane);
                }
            }
        }
    }

    if constexpr (kSplittable) {
        constexpr uint32_t kPitch = BN * 4;                          // a D row of FP32 partial sums
        constexpr uint32_t kPartialBytes = OP_BM * kPitch;
        constexpr int kSwizzle = BN / 4 - 1 < 7 ? BN / 4 - 1 : 7;    // 16-byte chunks XOR row
        static_assert(kPartialBytes + 7 * (kPartialBytes / 8) <= kStages * (OP_A_STAGE + kBStage),
                      "the partial and seven received slices fit the ring");
        if (splits > 1) {
            // D rows [j * rows, (j + 1) * rows) of the tile are summed by CTA j.  Every CTA writes its
            // accumulator into its own idle ring, the bulk-copy engine sends each row slice to
            // its owner, and the owner adds the slices in the order 0 .. S-1.
            const int rows = OP_BM / splits;
            const uint32_t slice_bytes = static_cast<uint32_t>(rows) * kPitch;
            const int z = static_cast<int>(blockIdx.z);
            if (threadIdx.x == 0)
                mbar_arrive_expect_tx(recv_bar, static_cast<uint32_t>(splits - 1) * slice_bytes);
            cluster_sync_all();     // every CTA of the cluster is past its main loop: rings idle
            // A CTA whose progress wait ran out has no valid partial: NaN from all of them.
            uint32_t any_failed = 0;
            for (int j = 0; j < splits; ++j)
                any_failed |= ld_shared_cluster_u32(map_to_cta(fail_flag, static_cast<uint32_t>(j)));
            if (warp >= Tile::kFirstEpi && warp < kFirstLoader) {
                const int quarter = warp & 3, r = quarter * 32 + lane;
                const int first = ((warp - Tile::kFirstEpi) >> 2) * kGroupCols;
                const uint32_t row_addr = s_a + static_cast<uint32_t>(r) * kPitch;
                const uint32_t t_row = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
#pragma unroll 1
                for (int chunk = first / 16; chunk < (first + kGroupCols) / 16; ++chunk) {
                    uint32_t v[16];
                    if (kb_begin < kb_end(p.num_k_blocks)) {
                        tmem_load_16cols(t_row + chunk * 16, v);
                    } else {
#pragma unroll
                        for (int j = 0; j < 16; ++j)
                            v[j] = 0u;
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        st_shared_v4(row_addr + (((chunk * 4 + j) ^ (r & kSwizzle)) << 4), v[4 * j], v[4 * j + 1],
                                     v[4 * j + 2], v[4 * j + 3]);
                }
                fence_proxy_async_shared();     // the bulk copies below read these stores
            }
            __syncthreads();
            if (threadIdx.x == 0) {
                for (int j = 0; j < splits; ++j) {
                    if (j == z)
                        continue;
                    const uint32_t slot = static_cast<uint32_t>(z < j ? z : z - 1);
                    bulk_copy_to_cluster(map_to_cta(s_a + kPartialBytes + slot * slice_bytes, static_cast<uint32_t>(j)),
                                         s_a + static_cast<uint32_t>(j) * slice_bytes, slice_bytes,
                                         map_to_cta(recv_bar, static_cast<uint32_t>(j)));
                }
            }
            int received = 1;
            if (lane == 0)
                received = mbar_wait(recv_bar, 0) ? 1 : 0;
            received = __shfl_sync(0xffffffffu, received, 0);
            if (!received && lane == 0)
                atomicOr(p.status, kOpDrainTimeout);
            const OpWhere w = op_where<CTAS, BN, kSwap>(unit, row_tile_count, kBK, p);
            const int first_row = w.m0 + z * rows;        // D's rows of this CTA
            if (any_failed || !received) {
                nan_elements(w, kSwap ? w.n0 : first_row, kSwap ? BN : rows, kSwap ? first_row : w.n0, kSwap ? rows : BN,
                             warp, kThreads / 32, lane);
            } else {
                const uint8_t *ring = smem_raw + (s_a - raw);
                for (int idx = threadIdx.x; idx < rows * (BN / 4); idx += kThreads) {
                    // Neighbouring threads take neighbouring output columns.
                    const int rl = kSwap ? idx % rows : idx / (BN / 4), q = kSwap ? idx / rows : idx % (BN / 4);
                    const int r = z * rows + rl;
                    const uint32_t offset = static_cast<uint32_t>(rl) * kPitch +
                                            (static_cast<uint32_t>(q ^ (r & kSwizzle)) << 4);
                    float v[4] = {};
#pragma unroll
                    for (int src = 0; src < 8; ++src) {
                        if (src < splits) {
                            const uint32_t at = src == z ? static_cast<uint32_t>(z) * slice_bytes
                                                         : kPartialBytes + static_cast<uint32_t>(src < z ? src : src - 1) *
                                                                               slice_bytes;
                            const float4 x = *reinterpret_cast<const float4 *>(ring + at + offset);
                            v[0] += x.x;
                            v[1] += x.y;
                            v[2] += x.z;
                            v[3] += x.w;
                        }
                    }
                    const int d_row = first_row + rl, d_col = w.n0 + q * 4;
                    if constexpr (kSwap) {
                        const float b = p.bias && d_row < p.n ? load_bias(d_row) : 0.0f;
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            v[i] += b;
                        if (d_row < p.n && d_col < w.row_end)
                            store_elements(v, min(4, w.row_end - d_col), d_col, d_row, 1, 0);
                    } else if (d_row < w.row_end && d_col < p.n) {
                        const int count = min(4, p.n - d_col);
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (p.bias && i < count)
                                v[i] += load_bias(d_col + i);
                        store_elements(v, count, d_row, d_col, 0, 1);
                    }
                }
            }
            // No CTA leaves while a copy into it (or out of it) may be in flight.
            cluster_sync_all();
        }
    }

    // No CTA (of a pair) releases TMEM before the last MMA and every epilogue are done.
    tc_fence_before();
    if constexpr (kPair)
        cluster_sync_all();
    else
        __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        if constexpr (kPair)
            tmem_dealloc_pair(tmem_base, Tile::kTmemColumns);
        else
            tmem_dealloc(tmem_base, Tile::kTmemColumns);
    }
}

} // namespace b200
