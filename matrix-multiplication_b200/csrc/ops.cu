// C-ABI of the operators next to matmul_launch: the product with bias, activation and
// residual in its epilogue, products grouped by expert, and softmax cross entropy over
// a large vocabulary, each with its gradient.  Declarations and contracts:
// include/b200_matmul.h; kernels: tc_ops.cuh, ops_aux.cuh.
#include <algorithm>
#include <cmath>
#include <cstring>
#include <initializer_list>

#include "context.cuh"
#include "ops.cuh"
#include "ops_plan.cuh"

namespace {

using namespace b200;

constexpr int kTf32 = 1, kFp16 = 2, kBf16 = 3;     // precision ids of the ABI
constexpr int kMaxSize = 0x7fffffff - 1023;        // a tile past the end still has int coordinates
// The plan kernel adds up row tiles (rows / 16 + groups at most) or K blocks and epilogues (rows / 32 +
// (1 + GP_EPILOGUE_BLOCKS) groups at most) of all groups as ints.
constexpr int kMaxGroups = 1 << 28;
static_assert(kMaxSize / 32 + int64_t{kMaxGroups} * (1 + GP_EPILOGUE_BLOCKS) <= 0x7fffffff &&
                  kMaxSize / 16 + int64_t{kMaxGroups} <= 0x7fffffff,
              "a plan's sums fit an int");

// Makes a device current for a call and puts the caller's back.
struct DeviceScope {
    int previous = -1;
    cudaError_t status;
    explicit DeviceScope(int device)
    {
        status = cudaGetDevice(&previous);
        if (status == cudaSuccess && previous != device)
            status = cudaSetDevice(device);
        else if (status == cudaSuccess)
            previous = -1;
    }
    ~DeviceScope()
    {
        if (previous >= 0)
            cudaSetDevice(previous);
    }
};

const OpKernels &kernels_of(int precision)
{
    return precision == kTf32 ? kOpKernelsTF32 : precision == kFp16 ? kOpKernelsF16 : kOpKernelsBF16;
}

int element(int precision)
{
    return precision == kTf32 ? 4 : 2;
}

CUtensorMapDataType operand_type(int precision)
{
    return precision == kTf32   ? CU_TENSOR_MAP_DATA_TYPE_TFLOAT32
           : precision == kFp16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
}

// A row-major matrix, or `groups` of them `slab` elements apart.
struct Matrix {
    const void *ptr = nullptr;
    int64_t rows = 0, cols = 0, pitch = 0;
    int64_t groups = 1, slab = 0;
    int64_t skipped = 0;     // columns of the rows before `ptr` (a piece of a matrix)
};

// One call: its context, format, stream and stream-ordered scratch.  Scratch is asked
// for with reserve() first, taken by one allocation, and given back to the stream when
// the call returns, after everything it enqueued.
struct Call {
    Context *ctx;
    int precision;
    cudaStream_t stream;
    const char *name;
    char *error;
    size_t error_size;
    uint8_t *scratch = nullptr;
    size_t scratch_bytes = 0;

    ~Call()
    {
        if (scratch) {
            DeviceScope device(ctx->device);     // a default stream is the current device's
            cudaFreeAsync(scratch, stream);
        }
    }
    int failed(const char *detail) { return fail(error, error_size, name, detail); }
    int failed(cudaError_t st) { return fail_cuda(error, error_size, name, st); }
    const OpKernels &kernels() const { return kernels_of(precision); }
    int elem() const { return element(precision); }

    size_t reserve(size_t bytes)
    {
        const size_t at = scratch_bytes;
        scratch_bytes += (bytes + 255) / 256 * 256;
        return at;
    }
    int allocate()
    {
        if (!scratch_bytes)
            return 0;
        void *ptr = nullptr;
        const cudaError_t st = scratch_alloc(ctx, &ptr, scratch_bytes, stream);
        if (st != cudaSuccess)
            return fail_cuda(error, error_size, name, st);
        scratch = static_cast<uint8_t *>(ptr);
        return 0;
    }
};

bool tma_addressable(const void *ptr, int64_t cols, int elem)
{
    return aligned16(ptr) && cols * elem % 16 == 0;
}

// An operand that TMA can address: the caller's matrix, or its copy in scratch with rows
// padded to 128 bytes (unaligned bases and row pitches).
struct Operand {
    Matrix source;
    Matrix ready;
    bool direct = true;
    size_t at = 0;

    void plan(Call &c, const void *ptr, int64_t rows, int64_t cols, int64_t groups = 1)
    {
        source = Matrix{ptr, rows, cols, cols, groups, rows * cols};
        direct = tma_addressable(ptr, cols, c.elem());
        ready = source;
        if (!direct) {
            ready.pitch = round_up(cols, OP_ROW_BYTES / c.elem());
            ready.slab = rows * ready.pitch;
            at = c.reserve(static_cast<size_t>(groups * ready.slab * c.elem()));
        }
    }
    RepackJob job(Call &c)
    {
        ready.ptr = c.scratch + at;
        return repack_job(source.ptr, c.scratch + at, source.rows * source.groups, source.cols, ready.pitch, c.elem());
    }
};

// Copies the operands that need it, two to a launch.
int prepare_operands(Call &c, std::initializer_list<Operand *> operands)
{
    RepackJob jobs[4]{};
    int count = 0;
    for (Operand *o : operands)
        if (o->source.ptr && !o->direct)
            jobs[count++] = o->job(c);
    for (int i = 0; i < count; i += 2) {
        const cudaError_t st = c.kernels().repack(jobs[i], i + 1 < count ? jobs[i + 1] : RepackJob{}, c.ctx->sm_count,
                                                  c.stream);
        if (st != cudaSuccess)
            return c.failed(st);
    }
    return 0;
}

bool encode_3d(const Context *ctx, CUtensorMap *map, CUtensorMapDataType type, const Matrix &m, int elem,
               uint32_t box_inner, uint32_t box_rows, CUtensorMapSwizzle swizzle)
{
    const cuuint64_t dims[3] = {static_cast<cuuint64_t>(m.cols), static_cast<cuuint64_t>(m.rows),
                                static_cast<cuuint64_t>(m.groups)};
    const cuuint64_t row = static_cast<cuuint64_t>(m.pitch) * elem;
    const cuuint64_t slab = m.groups > 1 ? static_cast<cuuint64_t>(m.slab) * elem : row * m.rows;
    const cuuint64_t strides[2] = {row, slab};
    const cuuint32_t box[3] = {box_inner, box_rows, 1};
    const cuuint32_t steps[3] = {1, 1, 1};
    return ctx->encode(map, type, 3, const_cast<void *>(m.ptr), dims, strides, box, steps,
                       CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                       CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Whether an MN-major operand's columns are whole 128-byte blocks in memory (up to the row
// pitch, which a copy in scratch has to spare).
bool whole_blocks(const Call &c, const Matrix &m)
{
    const int64_t block = OP_ROW_BYTES / c.elem();
    return m.skipped + round_up(m.cols, block) <= m.pitch;
}

// An operand's map: K-major tiles are boxes of 128 bytes of K x `extent` rows; MN-major
// tiles are boxes of 128 bytes of M/N x one K block of rows, `extent` columns of them in
// one load where the columns are whole blocks (then the map's inner dimension is a block,
// its third the blocks of a row).
bool operand_map(const Call &c, CUtensorMap *map, const Matrix &m, bool mn_major, int extent)
{
    const uint32_t inner = static_cast<uint32_t>(OP_ROW_BYTES / c.elem());
    const bool blocked = mn_major && whole_blocks(c, m);
    const CUtensorMapSwizzle swizzle = mn_major && c.precision == kTf32 ? CU_TENSOR_MAP_SWIZZLE_128B_ATOM_32B
                                                                        : CU_TENSOR_MAP_SWIZZLE_128B;
    const cuuint64_t blocks = static_cast<cuuint64_t>((m.cols + inner - 1) / inner);
    const cuuint64_t dims[4] = {blocked ? inner : static_cast<cuuint64_t>(m.cols), static_cast<cuuint64_t>(m.rows),
                                blocked ? blocks : 1, static_cast<cuuint64_t>(m.groups)};
    const cuuint64_t row = static_cast<cuuint64_t>(m.pitch) * c.elem();
    const cuuint64_t slab = m.groups > 1 ? static_cast<cuuint64_t>(m.slab) * c.elem() : row * m.rows;
    const cuuint64_t strides[3] = {row, blocked ? OP_ROW_BYTES : slab, slab};
    const cuuint32_t box[4] = {inner, mn_major ? inner : static_cast<cuuint32_t>(extent),
                               blocked ? static_cast<cuuint32_t>(extent) / inner : 1, 1};
    const cuuint32_t steps[4] = {1, 1, 1, 1};
    return c.ctx->encode(map, operand_type(c.precision), 4, const_cast<void *>(m.ptr), dims, strides, box, steps,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Whether TMA can write an output, and its map (boxes of 128 rows x 128 bytes).
bool output_tma(const Matrix &m, int elem)
{
    return aligned16(m.ptr) && m.pitch * elem % 16 == 0 && (m.groups == 1 || m.slab * elem % 16 == 0);
}

bool output_map(const Call &c, CUtensorMap *map, const Matrix &m, bool half)
{
    const CUtensorMapDataType type = half ? operand_type(c.precision) : CU_TENSOR_MAP_DATA_TYPE_FLOAT32;
    return encode_3d(c.ctx, map, type, m, half ? 2 : 4, half ? 64 : 32, 128, CU_TENSOR_MAP_SWIZZLE_128B);
}

struct TileShape {
    int ctas, bm, bn;     // CTAs per tile, D's rows and columns per tile
};
constexpr TileShape kTileShapes[] = {{2, 256, 256}, {1, 128, 128}, {1, 128, 64}, {1, 128, 16},
                                     {1, 128, 32},  {1, 128, 64},  {1, 128, 128}};

// Column ranges of a tile that the loss reduces on its own: one per epilogue warpgroup.
int loss_parts(int tile)
{
    return kTileShapes[tile].bn >= 128 ? 2 : 1;
}

bool is_swap(int tile)
{
    return tile >= kSwap16;
}

// What the choice of a tile knows of a product: sizes, K blocks of 128 bytes, groups, bytes
// read and written per output element, whether TMA writes the output, and whether the
// epilogue can take partial sums (K splits) and run transposed.
struct TileProblem {
    int64_t m, n, k_blocks, groups = 1;
    int bytes_out = 2;
    bool out_tma = true, splittable = false, transposable = false, ragged_k = false;
    bool exponentials = false;     // the loss: an exponential of every element
    bool half_tiles = true;        // not in its forward pass
};

// Estimated cycles of a tile kind with K split S ways.  A K block costs the most of its MMA
// time (2 cycles a column, 140 at least), its operand bytes into one SM at 70 B/cycle and
// all running CTAs' bytes out of L2 at 9.3 KB/cycle; a tile's epilogue adds the kind's own
// cycles, more where rows are stored without TMA, and a tile costs no less than its stores
// (a pair's 5050 cycles, one CTA's 128 x 128 2960 for BF16, measured with K = 256).  A split
// adds its exchange.  The constants are fitted to 1170 times of every kind and split over 95
// BF16 products of 33 to 2048 rows (10 % rms; the kind chosen is 0.3 % slower than the
// fastest on average, 7 % at worst).
double tile_cycles(const Context *ctx, int tile, int splits, const TileProblem &q)
{
    constexpr double kEpilogue[] = {4400.0, 1100.0, 1140.0, 810.0, 800.0, 1170.0, 1170.0};
    constexpr double kRowStores[] = {6000.0, 2000.0, 1000.0, 200.0, 400.0, 800.0, 1700.0};
    constexpr double kFloor[] = {2500.0, 1480.0, 900.0, 0.0, 0.0, 0.0, 0.0};
    constexpr double kExponentials[] = {6300.0, 4300.0, 3050.0, 0.0, 0.0, 0.0, 0.0};
    const TileShape &t = kTileShapes[tile];
    const bool swap = is_swap(tile);
    const int64_t side_m = swap ? q.n : q.m, side_n = swap ? q.m : q.n;
    const double tiles = static_cast<double>((side_m + t.bm - 1) / t.bm * ((side_n + t.bn - 1) / t.bn) * q.groups);
    const double units = t.ctas == 2 ? ctx->max_pairs : ctx->sm_count;
    const double active = splits > 1 ? tiles * splits : t.ctas * std::min(tiles, units);
    double rounds = splits > 1 ? 1.0 : std::max(1.0, std::ceil(tiles / units));
    // A pair's short last round runs as half tiles (enqueue).
    if (t.ctas == 2 && q.groups == 1 && q.half_tiles && std::fmod(tiles, units) > 0.0 && std::fmod(tiles, units) <= units / 2)
        rounds = std::floor(tiles / units) + 0.6;
    const double bytes = static_cast<double>(OP_BM + t.bn / t.ctas) * OP_ROW_BYTES;
    const double k_cycles = std::max({2.0 * t.bn, 140.0, bytes / 70.0, active * bytes / 9300.0});
    const double epilogue = kEpilogue[tile] + (q.out_tma ? 0.0 : kRowStores[tile]);
    double tile_time = std::ceil(static_cast<double>(q.k_blocks) / splits) * k_cycles + epilogue;
    // In ragged-K mode one CTA's tile also waits for its group's tables and tensor maps, which a
    // pair's longer tile hides (32 groups of 256 rows, 2048 x 1408 outputs: 4800 cycles a
    // 128 x 128 tile, 3000 ungrouped; 80 us in pairs, 107 us without).
    if (q.ragged_k && t.ctas == 1)
        tile_time += 1800.0;
    // The loss's epilogues take as long whatever K is (forward, 1024 x 50304 with K = 64: 37, 49
    // and 68 us on the three kinds; K = 256 52 us with one CTA, 39 in pairs).
    tile_time = std::max(tile_time, q.exponentials ? kExponentials[tile] : kFloor[tile] * q.bytes_out);
    return rounds * tile_time +
           (splits > 1 ? 3700.0 + 0.093 * static_cast<double>(splits - 1) / splits * OP_BM * t.bn * 4.0 : 0.0);
}

struct TileChoice {
    int tile, splits;
    int chunks = 1;      // K chunks added up by a second kernel (GradientProduct)
};

// Whether K blocks split S ways leave every CTA some and fit the device in one wave.
bool can_split(const Context *ctx, int log_splits, int64_t tiles, int64_t k_blocks)
{
    const int64_t splits = int64_t{1} << log_splits, per = (k_blocks + splits - 1) / splits;
    return tiles * splits <= ctx->max_split_ctas[log_splits] && (splits - 1) * per < k_blocks;
}

// The tile kind and K split with the fewest estimated cycles.  Transposed kinds are
// considered for up to 64 rows, and where one wave holds all their tiles: their stores go
// element by element (2048 x 256 x 45056 with a residual took 1236 us on 128 x 128 tiles
// transposed, 146 us not).
TileChoice choose_tile(const Context *ctx, const TileProblem &q)
{
    TileChoice best{kSingle64, 1};
    double best_cycles = 0.0;
    for (int tile = kPair256; tile <= (q.transposable ? kSwap128 : kSingle64); ++tile) {
        const TileShape &t = kTileShapes[tile];
        const bool swap = is_swap(tile);
        if (t.ctas == 2 && (ctx->max_pairs < 1 || q.m <= OP_BM))
            continue;
        const int64_t side_m = swap ? q.n : q.m, side_n = swap ? q.m : q.n;
        const int64_t tiles = (side_m + t.bm - 1) / t.bm * ((side_n + t.bn - 1) / t.bn) * q.groups;
        if (swap && q.m > 64 && tiles > ctx->sm_count)
            continue;
        for (int i = 0; i < (q.splittable && t.ctas == 1 ? 4 : 1); ++i) {
            if (i > 0 && !can_split(ctx, i, tiles, q.k_blocks))
                continue;
            const double cycles = tile_cycles(ctx, tile, 1 << i, q);
            if (best_cycles == 0.0 || cycles < best_cycles) {
                best = {tile, 1 << i};
                best_cycles = cycles;
            }
        }
    }
    return best;
}

// Whether a kernel had better load by itself a B that TMA cannot address (OpTile's DIRECT;
// one tile of rows, 16-bit) than read a copy: it takes about 860 cycles more for a K block,
// the copy what its bytes take in L2 and HBM (BF16, copied and direct: product 1 x 1024 x 50257
// 56.5 and 29.6 us, 64 x 2048 x 18949 50.0 and 39.5, 32 x 300 x 9999 9.1 and 10.5; loss
// 1 x 1024 x 50257 76 and 40, 128 x 1024 x 50257 73 and 46, 3 x 2000 x 777 15.6 and 25).
bool direct_pays(const Context *ctx, int precision, const TileProblem &q, const TileChoice &choice, int epilogue)
{
    if (precision == kTf32 || (epilogue == kEpiLse ? choice.tile != kSingle128 || q.m > OP_BM
                                                   : !is_swap(choice.tile) || choice.tile == kSwap128 ||
                                                         q.m > kTileShapes[choice.tile].bn))
        return false;
    const int64_t tiles = (q.n + OP_BM - 1) / OP_BM, per = (q.k_blocks + choice.splits - 1) / choice.splits;
    const int64_t rounds = choice.splits > 1 ? 1 : (tiles + ctx->sm_count - 1) / ctx->sm_count;
    const double copied = 2.0 * static_cast<double>(q.k_blocks * OP_ROW_BYTES) * static_cast<double>(q.n);
    return 1500.0 + 860.0 * static_cast<double>(rounds * per) < copied / 2700.0;
}

// A product with everything but its tile-dependent parts: operands as stored, sizes, and
// in `launch` the epilogue's parameters.
struct Product {
    Matrix a, b;             // kNN: M x K, K x N;  kNT: M x K, N x K;  kTN: K x M, K x N
    int64_t m = 0, n = 0, k = 0;
    OpLaunch launch;
    void set_tile(const TileChoice &choice)
    {
        launch.tile = choice.tile;
        launch.splits = choice.splits;
    }
};

// Exact quotients by a positive divisor on the device (op_divide).
OpDivisor divisor(int64_t value)
{
    int bits = 0;
    while ((int64_t{1} << bits) < value)
        ++bits;
    const uint64_t magic = (((uint64_t{1} << bits) - static_cast<uint64_t>(value)) << 32) / static_cast<uint64_t>(value) + 1;
    return {static_cast<uint32_t>(magic), static_cast<uint32_t>(bits > 0 ? bits - 1 : 0), static_cast<int>(value)};
}

int enqueue(Call &c, Product &q)
{
    OpLaunch &l = q.launch;
    const TileShape &t = kTileShapes[l.tile];
    const bool swap = is_swap(l.tile);
    const bool a_mn = l.layout == kTN, b_mn = l.layout != kNT;
    const int b_cols = t.bn / t.ctas;     // Bop columns per CTA
    l.p.a_blocked = whole_blocks(c, swap ? q.b : q.a) ? 1 : 0;
    l.p.b_blocked = whole_blocks(c, q.b) ? 1 : 0;
    // Where one tile holds all rows of A, its box holds them alone: TMA writes zeros for rows
    // past the matrix more slowly than it reads rows, and what the shared memory holds there
    // instead enters only rows of D that are not stored (the loss of 1 x 1024 x 50257, BF16: 76 -> 67 us).
    const int most = swap ? b_cols : OP_BM;
    const int box_rows = a_mn || q.m > most ? most : static_cast<int>(round_up(q.m, 8));
    l.p.stage_tx = static_cast<uint32_t>(OP_ROW_BYTES * (t.ctas * (OP_BM + b_cols) - t.ctas * (most - box_rows)));
    bool ok;
    if (l.p.direct) {     // B is loaded without TMA
        l.p.k = static_cast<int>(q.k);
        l.p.stage_tx = static_cast<uint32_t>(OP_ROW_BYTES * box_rows);
        ok = operand_map(c, swap ? &l.map_b : &l.map_a, q.a, false, box_rows);
    } else if (swap)     // D = B^T A^T: B's columns on the M side, A's rows on the N side
        ok = operand_map(c, &l.map_a, q.b, true, OP_BM) && operand_map(c, &l.map_b, q.a, false, box_rows);
    else
        ok = operand_map(c, &l.map_a, q.a, a_mn, box_rows) && operand_map(c, &l.map_b, q.b, b_mn, b_cols);
    if (!ok) {
        cudaGetLastError();
        return c.failed("cuTensorMapEncodeTiled rejected an operand");
    }
    OpParams &p = l.p;
    p.m = static_cast<int>(q.m);
    p.n = static_cast<int>(q.n);
    const int64_t side_m = swap ? q.n : q.m, side_n = swap ? q.m : q.n;
    p.num_m_blocks = static_cast<int>((side_m + t.bm - 1) / t.bm);
    p.num_n_blocks = static_cast<int>((side_n + t.bn - 1) / t.bn);
    const int bk = OP_ROW_BYTES / c.elem();
    p.num_k_blocks = static_cast<int>((q.k + bk - 1) / bk);
    int64_t tiles = static_cast<int64_t>(p.num_m_blocks) * p.num_n_blocks;
    if (p.grouping == kGroupedK || p.grouping == kChunkedK)
        tiles *= p.groups;
    else if (p.grouping == kGroupedRows)     // at most this many; the plan on the device has the number
        tiles = (q.m / (swap ? t.bn : t.bm) + std::min<int64_t>(p.groups, q.m)) *
                (swap ? p.num_m_blocks : p.num_n_blocks);
    if (tiles > 0x7fffffff)
        return c.failed("too many output tiles");
    p.num_tiles = static_cast<int>(tiles);
    p.log_raster = t.ctas == 2 ? 3 : 4;
    const int64_t per_raster = swap ? p.num_m_blocks : static_cast<int64_t>(p.num_n_blocks) << p.log_raster;
    const int64_t per_group = static_cast<int64_t>(p.num_m_blocks) * p.num_n_blocks;
    p.per_raster = divisor(std::min<int64_t>(per_raster, 0x7fffffff));
    p.per_group = divisor(std::min<int64_t>(per_group, 0x7fffffff));
    // A last round that leaves half of the pairs without a tile runs as half tiles on twice as
    // many of them (4096 x 14336 . 14336 x 4096: 256 tiles on 74 pairs, 3.5 rounds in place
    // of 4).
    p.full_tiles = p.num_tiles;
    if (l.tile == kPair256 && p.grouping == kUngrouped && l.epilogue != kEpiLse) {
        const int rest = p.num_tiles % c.ctx->max_pairs;
        if (2 * rest <= c.ctx->max_pairs) {
            p.full_tiles = p.num_tiles - rest;
            p.num_tiles += rest;
            tiles = p.num_tiles;
        }
    }
    p.status = c.ctx->status;
    p.wait_limit_ns = wait_limit(c.ctx);
    const int64_t units = t.ctas == 2 ? c.ctx->max_pairs : c.ctx->sm_count;
    l.grid = l.splits > 1 ? static_cast<int>(tiles) : static_cast<int>(std::min(tiles, units)) * t.ctas;
    const cudaError_t st = c.kernels().product(l, c.stream);
    return st == cudaSuccess ? 0 : c.failed(st);
}

// Gives a product's epilogue its residual (rows as the output's), after set_output and the
// pre-activation.
int set_residual(Call &c, OpLaunch &l, const Matrix &residual, bool half)
{
    OpParams &p = l.p;
    p.residual = residual.ptr;
    p.residual_half = half ? 1 : 0;
    p.residual_tma = p.out_tma && !p.preact && p.residual_half == p.out_half && !is_swap(l.tile) && l.splits == 1 ? 1 : 0;
    if (p.residual_tma && !output_map(c, &l.map_z, residual, half)) {
        cudaGetLastError();
        return c.failed("cuTensorMapEncodeTiled rejected the residual");
    }
    return 0;
}

// Points a product's epilogue at an output matrix.
int set_output(Call &c, OpLaunch &l, const Matrix &out, bool half)
{
    OpParams &p = l.p;
    p.out = const_cast<void *>(out.ptr);
    p.out_pitch = out.pitch;
    p.out_slab = out.slab;
    p.out_half = half ? 1 : 0;
    p.out_tma = output_tma(out, half ? 2 : 4) ? 1 : 0;
    if (p.out_tma && !output_map(c, &l.map_c, out, half)) {
        cudaGetLastError();
        return c.failed("cuTensorMapEncodeTiled rejected an output");
    }
    return 0;
}

// A product whose epilogue only stores, possibly added to an FP32 matrix: the gradients.
// Where there are few output tiles and K is long, K is cut into chunks over all SMs.
struct GradientProduct {
    static constexpr int64_t kChunkBytes = 64 << 20;     // the chunks' products stay in L2
    int layout = kNN;
    int64_t m = 0, n = 0, k = 0;
    TileChoice choice{kSingle64, 1};
    size_t at = 0;

    // Before the call's scratch is allocated.  `base`: an FP32 matrix is added.
    void plan(Call &c, int product_layout, int64_t rows, int64_t cols, int64_t depth, const Matrix &out, bool half,
              bool base = false)
    {
        layout = product_layout;
        m = rows;
        n = cols;
        k = depth;
        const int64_t bk = OP_ROW_BYTES / c.elem(), k_blocks = (k + bk - 1) / bk;
        const int out_bytes = half ? 2 : 4;
        TileProblem q{m, n, k_blocks, 1, out_bytes + (base ? 4 : 0), output_tma(out, out_bytes), true};
        choice = choose_tile(c.ctx, q);
        // Chunks cost their FP32 products, written and read once more through L2, and a launch of about
        // 8000 cycles; the estimate knows nothing of operands that HBM limits, so a gain below 8 % is
        // not taken (BF16 da: 302 x 20352 . 20352 x 1920 51.9 -> 41.6 us, 1024 x 30000 . 30000 x 512
        // 50.3 -> 39.5; 27 x 64 x 113300 with its loss's other kernels 91 -> 65).
        double best = 0.92 * tile_cycles(c.ctx, choice.tile, choice.splits, q);
        q.bytes_out = 4;
        q.out_tma = true;
        for (int chunks : {2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64}) {
            if (k_blocks < 4 * chunks || chunks * m * round_up(n, 4) * 4 > kChunkBytes)
                break;
            q.k_blocks = (k_blocks + chunks - 1) / chunks;
            if ((chunks - 1) * q.k_blocks >= k_blocks)
                continue;        // the last chunk would be empty
            q.groups = chunks;
            for (int tile : {kPair256, kSingle128, kSingle64}) {
                if (tile == kPair256 && (c.ctx->max_pairs < 1 || m <= OP_BM))
                    continue;
                const double cycles = tile_cycles(c.ctx, tile, 1, q) + 8000.0 +
                                      static_cast<double>(chunks) * static_cast<double>(m * n) * 8.0 / 4000.0;
                if (cycles < best) {
                    best = cycles;
                    choice = {tile, 1, chunks};
                }
            }
        }
        if (choice.chunks > 1)
            at = c.reserve(static_cast<size_t>(choice.chunks) * m * round_up(n, 4) * sizeof(float));
    }

    // a and b as stored for the layout; depth may be below the planned one (a last piece).
    int run(Call &c, const Matrix &a, const Matrix &b, int64_t depth, const Matrix &out, bool half, const Matrix *base = nullptr)
    {
        Product q;
        q.a = a;
        q.b = b;
        q.m = m;
        q.n = n;
        q.k = depth;
        q.launch.layout = layout;
        q.set_tile(choice);
        const int64_t bk = OP_ROW_BYTES / c.elem(), k_blocks = (depth + bk - 1) / bk;
        int64_t per = (k_blocks + choice.chunks - 1) / choice.chunks;
        const int chunks = static_cast<int>((k_blocks + per - 1) / per);
        if (choice.chunks == 1) {
            if (set_output(c, q.launch, out, half))
                return 1;
            if (base) {
                if (!output_tma(*base, 4))
                    q.launch.p.out_tma = 0;
                if (set_residual(c, q.launch, *base, false))
                    return 1;
            }
            return enqueue(c, q);
        }
        const int64_t pitch = round_up(n, 4);
        const Matrix sums{c.scratch + at, m, n, pitch, chunks, m * pitch};
        OpParams &p = q.launch.p;
        p.grouping = kChunkedK;
        p.groups = chunks;
        p.chunk_blocks = static_cast<int>(per);
        if (set_output(c, q.launch, sums, false) || enqueue(c, q))
            return 1;
        ChunkSumParams g{};
        g.chunks = static_cast<const float *>(sums.ptr);
        g.count = chunks;
        g.rows = static_cast<int>(m);
        g.cols = static_cast<int>(n);
        g.slab = sums.slab;
        g.pitch = pitch;
        g.base = base ? static_cast<const float *>(base->ptr) : nullptr;
        g.base_pitch = base ? base->pitch : 0;
        g.out = const_cast<void *>(out.ptr);
        g.out_pitch = out.pitch;
        g.out_half = half ? 1 : 0;
        g.vec = output_tma(out, half ? 2 : 4) ? 1 : 0;
        const cudaError_t st = c.kernels().chunk_sum(g, c.ctx->sm_count, c.stream);
        return st == cudaSuccess ? 0 : c.failed(st);
    }
};

// ---------------------------------------------------------------- argument checks
int check_call(void *opaque, int precision, const char *name, char *error, size_t error_size)
{
    clear_error(error, error_size);
    if (!opaque)
        return fail(error, error_size, name, "context is null");
    if (precision != kTf32 && precision != kFp16 && precision != kBf16)
        return fail(error, error_size, name, "the precision must be 1 (tf32), 2 (fp16) or 3 (bf16)");
    return 0;
}

int check_sizes(Call &c, std::initializer_list<int> sizes)
{
    for (int size : sizes) {
        if (size <= 0)
            return c.failed("dimensions must be positive");
        if (size > kMaxSize)
            return c.failed("dimensions must be at most 2147482624");
    }
    return 0;
}

bool misaligned(const void *ptr, int bytes)
{
    return reinterpret_cast<uintptr_t>(ptr) % static_cast<uintptr_t>(bytes) != 0;
}

bool aligned_to(std::initializer_list<std::pair<const void *, int>> pointers)
{
    for (const auto &p : pointers)
        if (p.first && misaligned(p.first, p.second))
            return false;
    return true;
}

// Sets the attributes of a format's kernels by its first call, with the device current: it loads
// them, about half a millisecond each, which programs that call no operator need not pay for
// (matmul_create with all of them: 32 ms, 5 ms without).
cudaError_t setup_operators(Call &c)
{
    std::atomic<bool> &ready = c.ctx->operators_ready[c.precision - kTf32];
    if (ready.load(std::memory_order_acquire))
        return cudaSuccess;
    std::lock_guard<std::mutex> lock(c.ctx->operators_mutex);
    const cudaError_t st = c.kernels().setup();
    if (st == cudaSuccess)
        ready.store(true, std::memory_order_release);
    return st;
}

// Makes the call's device current, and its kernels ready.
struct CallScope : DeviceScope {
    explicit CallScope(Call &c) : DeviceScope(c.ctx->device)
    {
        if (status == cudaSuccess)
            status = setup_operators(c);
    }
};

} // namespace

extern "C" int matmul_epilogue(void *opaque, int precision, const void *a, const void *b, const void *bias,
                               int bias_fp32, int activation, const void *residual, void *out, int out_fp32,
                               void *preact, int preact_fp32, int m, int k, int n, void *stream, char *error,
                               size_t error_size)
{
    const char *name = "matmul_epilogue";
    if (check_call(opaque, precision, name, error, error_size))
        return 1;
    Call c{static_cast<Context *>(opaque), precision, static_cast<cudaStream_t>(stream), name, error, error_size};
    if (!a || !b || !out)
        return c.failed("matrix pointer is null");
    if (check_sizes(c, {m, k, n}))
        return 1;
    if (activation < kActNone || activation > kActSilu)
        return c.failed("unknown activation");
    const int e = c.elem();
    const bool out_half = e == 2 && !out_fp32, preact_half = e == 2 && !preact_fp32, bias_half = e == 2 && !bias_fp32;
    if (!aligned_to({{a, e}, {b, e}, {out, out_half ? 2 : 4}, {residual, out_half ? 2 : 4},
                     {preact, preact_half ? 2 : 4}, {bias, bias_half ? 2 : 4}}))
        return c.failed("a pointer is not aligned to its element size");
    CallScope device(c);
    if (device.status != cudaSuccess)
        return c.failed(device.status);
    Product q;
    OpLaunch &l = q.launch;
    const int bk = OP_ROW_BYTES / e;
    const int64_t k_blocks = (static_cast<int64_t>(k) + bk - 1) / bk;
    const int bytes_out = (out_half ? 2 : 4) * (residual ? 2 : 1) + (preact ? (preact_half ? 2 : 4) : 0);
    const Matrix mo{out, m, n, n};
    const bool out_tma = output_tma(mo, out_half ? 2 : 4) && (!residual || aligned16(residual));
    const TileProblem problem{m, n, k_blocks, 1, bytes_out, out_tma, true, true};
    const TileChoice choice = choose_tile(c.ctx, problem);
    l.tile = choice.tile;
    l.splits = choice.splits;
    l.epilogue = is_swap(choice.tile) ? kEpiStoreT : kEpiStore;
    Operand oa, ob;
    oa.plan(c, a, m, k);
    if (!tma_addressable(b, n, e) && direct_pays(c.ctx, precision, problem, choice, l.epilogue))
        l.p.direct = b;
    else
        ob.plan(c, b, k, n);
    if (c.allocate() || prepare_operands(c, {&oa, &ob}))
        return 1;
    q.a = oa.ready;
    q.b = ob.ready;
    q.m = m;
    q.n = n;
    q.k = k;
    if (set_output(c, l, mo, out_half))
        return 1;
    OpParams &p = l.p;
    p.bias = bias;
    p.bias_half = bias_half ? 1 : 0;
    p.activation = activation;
    p.out_tma = out_tma ? 1 : 0;
    if (preact) {
        const Matrix mz{preact, m, n, n};
        p.preact = preact;
        p.preact_pitch = mz.pitch;
        p.preact_half = preact_half ? 1 : 0;
        p.preact_tma = output_tma(mz, preact_half ? 2 : 4) ? 1 : 0;
        if (p.preact_tma && !output_map(c, &l.map_z, mz, preact_half)) {
            cudaGetLastError();
            return c.failed("cuTensorMapEncodeTiled rejected an output");
        }
    }
    if (residual && set_residual(c, l, Matrix{residual, m, n, n}, out_half))
        return 1;
    return enqueue(c, q);
}

namespace {

// dz = dout * act'(preact) into `dz` (pitch dz_pitch; null without an activation) and
// dbias, the column sums, through `partial` ([chunks][n]) when there are several chunks.
struct ActGradPlan {
    int chunks = 1, rows_per_chunk = 0, cluster = 1, clusters = 1;
    void choose(const Context *ctx, int m, int n)
    {
        // Eight row chunks of at least 32 rows, a cluster whose blocks add up their sums; where
        // the columns are few and the rows many, several clusters and a second kernel.
        const int64_t column_blocks = (static_cast<int64_t>(n) + AG_COLS - 1) / AG_COLS;
        const int64_t most = std::max<int64_t>(1, m / 32);
        const int64_t fill = std::max<int64_t>(1, 4LL * ctx->sm_count / (column_blocks * AG_CLUSTER));
        const int64_t all = std::min<int64_t>((m + 2047LL) / 2048, fill);
        const int64_t wanted = most >= AG_CLUSTER ? AG_CLUSTER * std::min(all, most / AG_CLUSTER) : most;
        cluster = static_cast<int>(std::min<int64_t>(wanted, AG_CLUSTER));
        clusters = static_cast<int>(wanted / cluster);
        chunks = static_cast<int>(wanted);
        rows_per_chunk = static_cast<int>((m + wanted - 1) / wanted);
    }
};

} // namespace

extern "C" int matmul_epilogue_backward(void *opaque, int precision, const void *dout, const void *a, const void *b,
                                        const void *preact, int preact_fp32, int activation, void *da, int da_fp32,
                                        void *db, int db_fp32, void *dbias, int dbias_fp32, int m, int k, int n,
                                        void *stream, char *error, size_t error_size)
{
    const char *name = "matmul_epilogue_backward";
    if (check_call(opaque, precision, name, error, error_size))
        return 1;
    Call c{static_cast<Context *>(opaque), precision, static_cast<cudaStream_t>(stream), name, error, error_size};
    if (!dout || (da && !b) || (db && !a) || (activation != kActNone && !preact))
        return c.failed("matrix pointer is null");
    if (!da && !db && !dbias)
        return c.failed("no gradient is asked for");
    if (check_sizes(c, {m, k, n}))
        return 1;
    if (activation < kActNone || activation > kActSilu)
        return c.failed("unknown activation");
    const int e = c.elem();
    const bool da_half = e == 2 && !da_fp32, db_half = e == 2 && !db_fp32, dbias_half = e == 2 && !dbias_fp32;
    const bool preact_half = e == 2 && !preact_fp32;
    if (!aligned_to({{dout, e}, {a, e}, {b, e}, {preact, preact_half ? 2 : 4}, {da, da_half ? 2 : 4},
                     {db, db_half ? 2 : 4}, {dbias, dbias_half ? 2 : 4}}))
        return c.failed("a pointer is not aligned to its element size");
    CallScope device(c);
    if (device.status != cudaSuccess)
        return c.failed(device.status);

    const bool own_dz = activation != kActNone && (da || db);
    Operand oa, ob, od;
    if (db)
        oa.plan(c, a, m, k);
    if (da)
        ob.plan(c, b, k, n);
    size_t dz_at = 0;
    const int64_t dz_pitch = round_up(n, OP_ROW_BYTES / e);
    if (own_dz)
        dz_at = c.reserve(static_cast<size_t>(m * dz_pitch * e));
    else if (da || db)
        od.plan(c, dout, m, n);
    const Matrix ma{da, m, k, k}, mb{db, k, n, n};
    GradientProduct pa, pb;
    if (da)
        pa.plan(c, kNT, m, k, n, ma, da_half);
    if (db)
        pb.plan(c, kTN, k, n, m, mb, db_half);
    ActGradPlan plan;
    plan.choose(c.ctx, m, n);
    size_t partial_at = 0;
    const bool partial = dbias && plan.clusters > 1;
    if (partial)
        partial_at = c.reserve(static_cast<size_t>(plan.clusters) * n * sizeof(float));
    if (c.allocate() || prepare_operands(c, {&oa, &ob, &od}))
        return 1;

    if (own_dz || dbias) {
        ActGradParams g{};
        g.dout = dout;
        g.preact = activation != kActNone ? preact : nullptr;
        g.preact_half = preact_half ? 1 : 0;
        g.dz = own_dz ? c.scratch + dz_at : nullptr;
        g.dz_pitch = dz_pitch;
        g.partial = partial ? reinterpret_cast<float *>(c.scratch + partial_at) : nullptr;
        g.dbias = dbias;
        g.dbias_half = dbias_half ? 1 : 0;
        g.m = m;
        g.n = n;
        g.rows_per_chunk = plan.rows_per_chunk;
        g.activation = activation;
        g.vec = aligned16(dout) && static_cast<int64_t>(n) * e % 16 == 0 && (!g.preact || aligned16(preact)) &&
                (!g.preact || static_cast<int64_t>(n) * (preact_half ? 2 : 4) % 16 == 0);
        cudaError_t st = c.kernels().act_grad(g, dim3(static_cast<unsigned int>((n + AG_COLS - 1) / AG_COLS),
                                                      static_cast<unsigned int>(plan.chunks)),
                                              plan.cluster, c.stream);
        if (st == cudaSuccess && partial)
            st = c.kernels().bias_grad(g.partial, plan.clusters, n, dbias, g.dbias_half, c.stream);
        if (st != cudaSuccess)
            return c.failed(st);
    }
    const Matrix dz = own_dz ? Matrix{c.scratch + dz_at, m, n, dz_pitch} : od.ready;
    if (da && pa.run(c, dz, ob.ready, n, ma, da_half))
        return 1;
    if (db && pb.run(c, oa.ready, dz, m, mb, db_half))
        return 1;
    return 0;
}

namespace {

// The device-side plan of a grouped product in scratch: row tiles (or group bounds) and
// the groups' tensor maps.
struct GroupPlan {
    int tile_rows = 0, maps = 0;
    size_t maps_at = 0, tiles_at = 0, count_at = 0, units_at = 0;
    int units = 0;

    // tile_rows 0: ragged-K mode.
    void plan(Call &c, int groups, int rows, int tile, int map_count)
    {
        tile_rows = tile;
        maps = map_count;
        const int64_t entries = tile ? rows / tile + std::min(groups, rows) : groups;
        maps_at = c.reserve(static_cast<size_t>(groups) * std::max(maps, 1) * sizeof(CUtensorMap));
        tiles_at = c.reserve(static_cast<size_t>(entries) * sizeof(OpRowTile));
        count_at = c.reserve(sizeof(int));
        units_at = c.reserve(static_cast<size_t>(c.ctx->sm_count + 1) * sizeof(int));
    }
    // The plan kernel's parameters, and what the product reads of its results.
    // `tiles_per_group`, `max_units`: ragged-K mode's tiles and the CTAs or pairs that share them.
    GroupPlanParams fill(Call &c, const void *offsets, int offsets64, int groups, int rows, OpParams &p,
                         int64_t tiles_per_group = 0, int64_t max_units = 0) const
    {
        GroupPlanParams g{};
        if (!tile_rows) {
            g.units = static_cast<int>(std::min(tiles_per_group * groups, max_units));
            g.unit_first = reinterpret_cast<int *>(c.scratch + units_at);
            g.tiles_per_group = tiles_per_group;
            g.k_block = OP_ROW_BYTES / c.elem();
            p.unit_first = g.unit_first;
        }
        g.offsets = offsets;
        g.offsets64 = offsets64;
        g.groups = groups;
        g.rows = rows;
        g.tile_rows = tile_rows;
        g.maps = maps;
        g.count = reinterpret_cast<int *>(c.scratch + count_at);
        g.tiles = reinterpret_cast<OpRowTile *>(c.scratch + tiles_at);
        g.group_maps = reinterpret_cast<CUtensorMap *>(c.scratch + maps_at);
        p.grouping = tile_rows ? kGroupedRows : kGroupedK;
        p.groups = groups;
        p.row_tile_count = g.count;
        p.row_tiles = g.tiles;
        p.group_maps = g.group_maps;
        return g;
    }
};

// One launch for one plan, or for a backward pass's two (`second` with map2 alone).
int enqueue_plans(Call &c, const CUtensorMap &map0, const CUtensorMap &map1, const CUtensorMap &map2,
                  const GroupPlanParams &first, const GroupPlanParams *second)
{
    // One warp per tensor map, up to sixteen blocks.
    const int maps = std::max(first.groups * first.maps, second ? second->groups * second->maps : 0);
    const dim3 grid(static_cast<unsigned int>(std::min(16, std::max(1, maps / GP_WARPS))), second ? 2 : 1);
    const cudaError_t st = launch_pdl(group_plan_kernel, grid, dim3(GP_THREADS), 0, c.stream, map0, map1, map2, first,
                                      second ? *second : first);
    return st == cudaSuccess ? 0 : c.failed(st);
}

int check_groups(Call &c, int groups, int rows, int k, int n, const void *offsets, int offsets64)
{
    if (check_sizes(c, {rows, k, n, groups}))
        return 1;
    if (groups > kMaxGroups)
        return c.failed("groups must be at most 268435456");
    if (!offsets)
        return c.failed("offsets pointer is null");
    if (misaligned(offsets, offsets64 ? 8 : 4))
        return c.failed("a pointer is not aligned to its element size");
    return 0;
}

// Rows per tile follow the mean group: with few rows they take the MMA's N side (16 to 128
// wide) and the weight's columns its M side, so that a tile wastes little (64 groups, 2048 x
// 2816 BF16: mean 50 rows 100 us on 64-row transposed tiles, 118 us on pairs; mean
// 100 rows 124 us on 128-row ones, 129 us on pairs; mean 200 rows 198 and 163 us).  Larger
// groups go by the cycles of a mean group.  The loads themselves are known on the device
// alone, so a group of many times the mean runs on its narrow tiles and reads its weight once
// for each (4096 rows over 64 experts, 2048 x 2816: 122 us evenly spread, 151 with half of the
// rows in one expert, 179 with nine tenths; 8192 over 512, 1024 x 1024: 168, 213 and 254).
int choose_grouped_tile(const Context *ctx, int64_t rows, int64_t groups, int64_t n, int64_t k_blocks, int bytes_out,
                        bool out_tma)
{
    const int64_t mean = (rows + groups - 1) / groups;
    if (mean <= 16)
        return kSwap16;
    if (mean <= 32)
        return kSwap32;
    if (mean <= 64)
        return kSwap64;
    if (mean <= 128)
        return kSwap128;
    return choose_tile(ctx, {mean, n, k_blocks, groups, bytes_out, out_tma, false, true}).tile;
}

} // namespace

extern "C" int matmul_grouped(void *opaque, int precision, const void *a, const void *b, const void *offsets,
                              int offsets64, int groups, void *out, int out_fp32, int rows, int k, int n, void *stream,
                              char *error, size_t error_size)
{
    const char *name = "matmul_grouped";
    if (check_call(opaque, precision, name, error, error_size))
        return 1;
    Call c{static_cast<Context *>(opaque), precision, static_cast<cudaStream_t>(stream), name, error, error_size};
    if (!a || !b || !out)
        return c.failed("matrix pointer is null");
    if (check_groups(c, groups, rows, k, n, offsets, offsets64))
        return 1;
    const int e = c.elem();
    const bool half = e == 2 && !out_fp32;
    if (!aligned_to({{a, e}, {b, e}, {out, half ? 2 : 4}}))
        return c.failed("a pointer is not aligned to its element size");
    CallScope device(c);
    if (device.status != cudaSuccess)
        return c.failed(device.status);
    const int64_t bk = OP_ROW_BYTES / e;
    Product q;
    OpLaunch &l = q.launch;
    const Matrix mo{out, rows, n, n};
    l.tile = choose_grouped_tile(c.ctx, rows, groups, n, (k + bk - 1) / bk, half ? 2 : 4, output_tma(mo, half ? 2 : 4));
    const bool swap = is_swap(l.tile);
    l.epilogue = swap ? kEpiStoreT : kEpiStore;
    Operand oa, ob;
    oa.plan(c, a, rows, k);
    ob.plan(c, b, k, n, groups);
    GroupPlan plan;
    plan.plan(c, groups, rows, swap ? kTileShapes[l.tile].bn : kTileShapes[l.tile].bm,
              !swap && output_tma(mo, half ? 2 : 4) ? 1 : 0);
    if (c.allocate() || prepare_operands(c, {&oa, &ob}))
        return 1;
    q.a = oa.ready;
    q.b = ob.ready;
    q.m = rows;
    q.n = n;
    q.k = k;
    if (set_output(c, l, mo, half))
        return 1;
    const GroupPlanParams g = plan.fill(c, offsets, offsets64, groups, rows, l.p);
    return enqueue_plans(c, l.map_c, l.map_c, l.map_c, g, nullptr) || enqueue(c, q) ? 1 : 0;
}

extern "C" int matmul_grouped_backward(void *opaque, int precision, const void *dout, const void *a, const void *b,
                                       const void *offsets, int offsets64, int groups, void *da, int da_fp32, void *db,
                                       int db_fp32, int rows, int k, int n, void *stream, char *error,
                                       size_t error_size)
{
    const char *name = "matmul_grouped_backward";
    if (check_call(opaque, precision, name, error, error_size))
        return 1;
    Call c{static_cast<Context *>(opaque), precision, static_cast<cudaStream_t>(stream), name, error, error_size};
    if (!dout || (da && !b) || (db && !a))
        return c.failed("matrix pointer is null");
    if (!da && !db)
        return c.failed("no gradient is asked for");
    if (check_groups(c, groups, rows, k, n, offsets, offsets64))
        return 1;
    const int e = c.elem();
    const bool da_half = e == 2 && !da_fp32, db_half = e == 2 && !db_fp32;
    if (!aligned_to({{dout, e}, {a, e}, {b, e}, {da, da_half ? 2 : 4}, {db, db_half ? 2 : 4}}))
        return c.failed("a pointer is not aligned to its element size");
    CallScope device(c);
    if (device.status != cudaSuccess)
        return c.failed(device.status);
    const int64_t bk = OP_ROW_BYTES / e;
    Operand oa, ob, od;
    od.plan(c, dout, rows, n);
    GroupPlan rows_plan, k_plan;
    Product qa, qb;
    const Matrix ma{da, rows, k, k};
    if (da) {
        ob.plan(c, b, k, n, groups);
        const int64_t mean = (rows + groups - 1) / groups;
        qa.launch.layout = kNT;
        qa.launch.tile = choose_tile(c.ctx, {mean, k, (n + bk - 1) / bk, groups, da_half ? 2 : 4,
                                           output_tma(ma, da_half ? 2 : 4)}).tile;
        rows_plan.plan(c, groups, rows, kTileShapes[qa.launch.tile].bm, output_tma(ma, da_half ? 2 : 4) ? 1 : 0);
    }
    const Matrix mb{db, k, n, n, groups, static_cast<int64_t>(k) * n};
    if (db) {
        oa.plan(c, a, rows, k);
        const int64_t mean = (rows + groups - 1) / groups;
        qb.launch.layout = kTN;
        qb.launch.tile = choose_tile(c.ctx, {k, n, (mean + bk - 1) / bk, groups, db_half ? 2 : 4,
                                           output_tma(mb, db_half ? 2 : 4), false, false,
                                           true}).tile;
        k_plan.plan(c, groups, rows, 0, 2);
    }
    if (c.allocate() || prepare_operands(c, {&od, &ob, &oa}))
        return 1;
    // The plans first, both in one launch, then the two products.
    GroupPlanParams ga{}, gb{};
    CUtensorMap map0{}, map1{};
    if (da) {
        qa.a = od.ready;
        qa.b = ob.ready;
        qa.m = rows;
        qa.n = k;
        qa.k = n;
        if (set_output(c, qa.launch, ma, da_half))
            return 1;
        ga = rows_plan.fill(c, offsets, offsets64, groups, rows, qa.launch.p);
    }
    if (db) {
        qb.a = oa.ready;
        qb.b = od.ready;
        qb.m = k;
        qb.n = n;
        qb.k = rows;
        const TileShape &t = kTileShapes[qb.launch.tile];
        if (!operand_map(c, &map0, qb.a, true, OP_BM) ||
            !operand_map(c, &map1, qb.b, true, t.bn / t.ctas)) {
            cudaGetLastError();
            return c.failed("cuTensorMapEncodeTiled rejected an operand");
        }
        if (set_output(c, qb.launch, mb, db_half))
            return 1;
        gb = k_plan.fill(c, offsets, offsets64, groups, rows, qb.launch.p,
                         ((k + t.bm - 1) / t.bm) * ((static_cast<int64_t>(n) + t.bn - 1) / t.bn),
                         t.ctas == 2 ? c.ctx->max_pairs : c.ctx->sm_count);
    }
    const CUtensorMap &map_da = qa.launch.map_c;
    if (db ? enqueue_plans(c, map0, map1, map_da, gb, da ? &ga : nullptr)
           : enqueue_plans(c, map_da, map_da, map_da, ga, nullptr))
        return 1;
    if ((da && enqueue(c, qa)) || (db && enqueue(c, qb)))
        return 1;
    return 0;
}

namespace {

int check_loss(Call &c, int m, int k, int v, const void *labels, int labels64)
{
    if (check_sizes(c, {m, k, v}))
        return 1;
    if (!labels)
        return c.failed("labels pointer is null");
    if (misaligned(labels, labels64 ? 8 : 4))
        return c.failed("a pointer is not aligned to its element size");
    return 0;
}

} // namespace

extern "C" int matmul_cross_entropy(void *opaque, int precision, const void *hidden, const void *weight,
                                    const void *labels, int labels64, long long ignore_index, float *loss, float *lse,
                                    int m, int k, int v, void *stream, char *error, size_t error_size)
{
    const char *name = "matmul_cross_entropy";
    if (check_call(opaque, precision, name, error, error_size))
        return 1;
    Call c{static_cast<Context *>(opaque), precision, static_cast<cudaStream_t>(stream), name, error, error_size};
    if (!hidden || !weight || !loss || !lse)
        return c.failed("pointer is null");
    if (check_loss(c, m, k, v, labels, labels64))
        return 1;
    const int e = c.elem();
    if (!aligned_to({{hidden, e}, {weight, e}, {loss, 4}, {lse, 4}}))
        return c.failed("a pointer is not aligned to its element size");
    CallScope device(c);
    if (device.status != cudaSuccess)
        return c.failed(device.status);
    const int64_t bk = OP_ROW_BYTES / e;
    Product q;
    OpLaunch &l = q.launch;
    l.epilogue = kEpiLse;
    TileProblem problem{m, v, (k + bk - 1) / bk};
    problem.exponentials = true;
    problem.half_tiles = false;
    l.tile = choose_tile(c.ctx, problem).tile;
    if (!tma_addressable(weight, v, e) && direct_pays(c.ctx, precision, problem, {kSingle128, 1}, kEpiLse)) {
        l.tile = kSingle128;
        l.p.direct = weight;
    }
    // One (maximum, sum) per row and column range of a tile.
    const int tiles = (v + kTileShapes[l.tile].bn - 1) / kTileShapes[l.tile].bn * loss_parts(l.tile);
    Operand oh, ow;
    oh.plan(c, hidden, m, k);
    if (!l.p.direct)
        ow.plan(c, weight, k, v);
    const size_t partial_at = c.reserve(static_cast<size_t>(tiles) * m * sizeof(float2));
    const size_t logit_at = c.reserve(static_cast<size_t>(m) * sizeof(float));
    if (c.allocate() || prepare_operands(c, {&oh, &ow}))
        return 1;
    q.a = oh.ready;
    q.b = ow.ready;
    q.m = m;
    q.n = v;
    q.k = k;
    OpParams &p = l.p;
    p.labels = labels;
    p.labels64 = labels64;
    p.ignore = ignore_index;
    p.classes = v;
    p.partial = reinterpret_cast<float2 *>(c.scratch + partial_at);
    p.label_logit = reinterpret_cast<float *>(c.scratch + logit_at);
    if (enqueue(c, q))
        return 1;
    const cudaError_t st = launch_pdl(loss_join_kernel, dim3(static_cast<unsigned int>((m + 31) / 32)),
                                      dim3(32 * LJ_WARPS), 0,
                                      c.stream, static_cast<const float2 *>(p.partial), tiles,
                                      static_cast<const float *>(p.label_logit), loss, lse, p);
    return st == cudaSuccess ? 0 : c.failed(st);
}

extern "C" int matmul_cross_entropy_backward(void *opaque, int precision, const float *grad, const void *hidden,
                                             const void *weight, const void *labels, int labels64,
                                             long long ignore_index, const float *lse, void *dhidden, int dhidden_fp32,
                                             void *dweight, int dweight_fp32, int m, int k, int v, void *stream,
                                             char *error, size_t error_size)
{
    const char *name = "matmul_cross_entropy_backward";
    if (check_call(opaque, precision, name, error, error_size))
        return 1;
    Call c{static_cast<Context *>(opaque), precision, static_cast<cudaStream_t>(stream), name, error, error_size};
    if (precision == kFp16)
        return c.failed("the gradient of each logit is held in the input format, and fp16 cannot hold the small ones; "
                        "use bf16 or tf32");
    if (!grad || !hidden || !weight || !lse)
        return c.failed("pointer is null");
    if (!dhidden && !dweight)
        return c.failed("no gradient is asked for");
    if (check_loss(c, m, k, v, labels, labels64))
        return 1;
    const int e = c.elem();
    const bool dh_half = e == 2 && !dhidden_fp32, dw_half = e == 2 && !dweight_fp32;
    if (!aligned_to({{hidden, e}, {weight, e}, {grad, 4}, {lse, 4}, {dhidden, dh_half ? 2 : 4}, {dweight, dw_half ? 2 : 4}}))
        return c.failed("a pointer is not aligned to its element size");
    CallScope device(c);
    if (device.status != cudaSuccess)
        return c.failed(device.status);
    const int64_t bk = OP_ROW_BYTES / e;
    // Vocabulary pieces: the logits' gradients of one piece (m x width, input format) take at
    // most 64 MB, so that the two products that read them find them in L2, but a piece has
    // 4096 columns at least (fewer would make dhidden's sum over the pieces dear): from 8193
    // BF16 or 4097 TF32 rows on its scratch is 8 or 16 KB a row, and L2 holds a part of it.
    constexpr int64_t kPieceBytes = int64_t{64} << 20;
    int64_t width = kPieceBytes / (static_cast<int64_t>(m) * e) / 256 * 256;
    width = std::max<int64_t>(width, 4096);
    width = std::min<int64_t>(width, round_up(v, 256));
    const int64_t pieces = (v + width - 1) / width;
    Operand oh, ow;
    oh.plan(c, hidden, m, k);
    ow.plan(c, weight, k, v);
    const size_t dz_at = c.reserve(static_cast<size_t>(m) * width * e);
    // dH is summed over the pieces in FP32: in the output itself where it is FP32.
    const bool own_sum = dhidden && dh_half && pieces > 1;
    const size_t sum_at = own_sum ? c.reserve(static_cast<size_t>(m) * k * sizeof(float)) : 0;
    const Matrix dh{dhidden, m, k, k};
    GradientProduct ph, pw;
    if (dhidden)
        ph.plan(c, kNT, m, k, width, dh, dh_half && !own_sum, pieces > 1);
    if (dweight)
        pw.plan(c, kTN, k, width, m, Matrix{dweight, k, width, v}, dw_half);
    if (c.allocate() || prepare_operands(c, {&oh, &ow}))
        return 1;
    const Matrix sum = own_sum ? Matrix{c.scratch + sum_at, m, k, k} : dh;
    for (int64_t piece = 0; piece < pieces; ++piece) {
        const int64_t v0 = piece * width, cols = std::min<int64_t>(width, v - v0);
        const Matrix w{static_cast<const uint8_t *>(ow.ready.ptr) + v0 * e, k, cols, ow.ready.pitch, 1, 0, v0};
        const Matrix dz{c.scratch + dz_at, m, cols, width};
        {
            Product q;
            q.a = oh.ready;
            q.b = w;
            q.m = m;
            q.n = cols;
            q.k = k;
            q.launch.epilogue = kEpiSoftmaxGrad;
            TileProblem problem{m, cols, (k + bk - 1) / bk, 1, e};
            problem.exponentials = true;
            q.launch.tile = choose_tile(c.ctx, problem).tile;
            OpParams &p = q.launch.p;
            p.labels = labels;
            p.labels64 = labels64;
            p.ignore = ignore_index;
            p.classes = v;
            p.column0 = static_cast<int>(v0);
            p.lse = lse;
            p.grad = grad;
            if (set_output(c, q.launch, dz, e == 2) || enqueue(c, q))
                return 1;
        }
        if (dhidden) {
            const bool last = piece == pieces - 1;
            if (ph.run(c, dz, w, cols, last ? dh : sum, last && dh_half, piece > 0 ? &sum : nullptr))
                return 1;
        }
        if (dweight) {
            const Matrix dw{static_cast<uint8_t *>(dweight) + v0 * (dw_half ? 2 : 4), k, cols, v};
            pw.n = cols;
            if (pw.run(c, oh.ready, dz, m, dw, dw_half))
                return 1;
        }
    }
    return 0;
}
