// Orthogonalised updates by Newton-Schulz products.  Every matrix G of a batch becomes U p(p(..p(S / |G|)..)) V^T, where G = U S V^T
// and p(s) = a s + b s^3 + c s^5 acts on each singular value: with |G| the Frobenius norm
//     X = G / |G|;   `steps` times:  A = X X^T,  B = b A + c A A,  X = a X + B X
// in the orientation with fewer rows than columns.  A zero matrix gives zeros.
//
// The products are fp16 with fp32 sums on the tensor cores, of operands in two halves: hi hi + hi lo + lo hi (lo lo would be 2^-22 of
// it).  X, A and B are such pairs in memory, too.  One half would be a third of the tensor work (32 x 1024 x 1024: 1.07 ms), but small
// singular values are carried by the term a X and grow by a factor a in every step, and so does what a rounding leaves in directions
// that X does not have: with 16 bits of X results were 2e-2 off where the spectrum falls off as 1/k^2, with X in two halves and operands
// of one 1e-3 for flat spectra, 6e-3 where two rows hold everything and up to 2e-2 for one direction.  All fp16 values are scaled by
// powers of two that keep them below 65504 for every X the coefficients can reach (orthogonalize_in_range).
#include "orth.cuh"
#include "pair_ptx.cuh"
#include <cuda.h>
#include <algorithm>
#include <cmath>

namespace ts2 {

static constexpr float SX = ORTH_SX, SA = ORTH_SA, SB = ORTH_SB, MAX_X = ORTH_MAX_X, MAX_B = ORTH_MAX_B;
constexpr int PT = 256, BK = 64, HALF = 128 * 128; // HALF: a CTA's part of the first operand, one K block
// ---- G -> X ---------------------------------------------------------------------------------------------
// partial sums of squares in fp64: no input over- or underflows, and nothing is lost over 2^40 terms
template <class T>
__global__ void __launch_bounds__(256) orth_sum2_kernel(const T *__restrict__ g, long long ld, long long stride, int rows, int cols, bool vec,
                                                        double *part)
{
    grid_dep_wait();
    __shared__ double warps[8];
    g += blockIdx.y * stride;
    const int pieces = (cols + 7) / 8;
    const long long total = (long long)rows * pieces;
    double sum = 0.;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
        const int r = (int)(i / pieces), c = (int)(i - (long long)r * pieces) * 8;
        float v[8];
        orth_load8(g + r * ld, c, cols, vec, v);
#pragma unroll
        for (int j = 0; j < 8; ++j)
            sum = fma((double)v[j], (double)v[j], sum);
    }
    sum = warp_sum(sum);
    if ((threadIdx.x & 31) == 0)
        warps[threadIdx.x >> 5] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 8; ++w)
            sum += warps[w];
        part[blockIdx.y * gridDim.x + blockIdx.x] = sum;
    }
}

// 64 x 64 of X [n][m] (padded to np x mp with zeros) from G, transposed where G has more rows than columns
template <class T, bool TALL>
__global__ void __launch_bounds__(256) orth_load_kernel(const T *__restrict__ g, long long ld, long long stride, int rows, int cols, bool vec,
                                                        const double *part, int n_part, int np, int mp, __half *hi, __half *lo)
{
    grid_dep_wait();
    __shared__ double norm;
    __shared__ float tile[TALL ? 64 : 1][65];
    const int b = blockIdx.z, i0 = blockIdx.y * 64, j0 = blockIdx.x * 64, q = threadIdx.x >> 3, c8 = (threadIdx.x & 7) * 8;
    g += b * stride;
    float v[2][8];
#pragma unroll
    for (int h = 0; h < 2; ++h) { // 32 rows of G at a time
        const int r = (TALL ? j0 : i0) + q + 32 * h;
        if (r < rows)
            orth_load8(g + r * ld, (TALL ? i0 : j0) + c8, cols, vec, v[h]);
        else
#pragma unroll
            for (int j = 0; j < 8; ++j)
                v[h][j] = 0.f;
    }
    if (threadIdx.x < 32) {
        double sum = 0.;
        for (int i = threadIdx.x; i < n_part; i += 32)
            sum += part[b * n_part + i];
        sum = warp_sum(sum);
        if (threadIdx.x == 0)
            norm = sum == 0. ? 0. : SX / sqrt(sum);
    }
    if (TALL) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int j = 0; j < 8; ++j)
                tile[q + 32 * h][c8 + j] = v[h][j];
    }
    __syncthreads();
    // fp32 holds the scale unless G is all but denormal; then the product is made in fp64
    const double scale = norm;
    const bool small = !(scale < 1e30);
    const float scale32 = (float)scale;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int i = q + 32 * h;
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            x[j] = TALL ? tile[c8 + j][i] : v[h][j];
            x[j] = small ? (float)(x[j] * scale) : x[j] * scale32;
        }
        const size_t at = ((size_t)b * np + i0 + i) * mp + j0 + c8;
        orth_split8(x, *(uint4 *)(hi + at), *(uint4 *)(lo + at));
    }
}

// ---- the products ----------------------------------------------------------------------------------------------------
// Pairs of CTAs on tiles of 256 x 256 or 256 x 128 (as in gemm_pair.cu), one launch for a product of every matrix of the batch.
//   SQUARE  A = X X^T     POLY  B = b A + c A A     both operands K-contiguous; symmetric, so only tiles on and above the diagonal are
//                         computed, and what is above it leaves a second time as its transpose
//   UPDATE  X = a X + B X   B is K-contiguous (it is its own transpose), X is contiguous along N; writes a second pair of arrays, since
//                         other tiles still read the first
//   LAST    UPDATE of the last step: writes the result
//   PARTIAL a K range of SQUARE or POLY in fp32, for outputs of few tiles; orth_join_kernel adds the ranges
// A pair of arrays is one tensor of 2 x batch matrices, the low halves behind the high ones.  A slot of the ring holds the high or the low
// halves of a K block; the products of a block begin with its first slot and free both.  Residual inputs are read row by row and
// handed out to the threads, which have a row of 32 each, through shared memory; results leave from there as blocks of 32 x 32 by TMA.
enum Form { SQUARE, POLY, UPDATE, PARTIAL, LAST };
constexpr bool updates(int form) { return form == UPDATE || form == LAST; }
constexpr int STAGES = 5, EPI_WARPS = 8, THREADS = 64 + 32 * EPI_WARPS;
// an epilogue warp's shared memory: blocks of 32 x 32, high and low halves of the residual input and then of the output, and of what is
// mirrored
constexpr int BLOCK = 2048, WARP_BYTES = 4 * BLOCK, STG_OFF = STAGES * 2 * HALF, BAR_OFF = STG_OFF + EPI_WARPS * WARP_BYTES,
              SMEM = BAR_OFF + 1024 + 1024;
static_assert(SMEM <= 232448, "shared memory budget");

struct ProductArgs {
    int n, cols;         // rows and columns of the output (of every matrix)
    int tiles, col_tiles; // a matrix's tiles; UPDATE: in col_tiles columns
    int units, k_blocks, splits, kb_per_split;
    float alpha, beta; // POLY: alpha acc + beta A; UPDATE: alpha acc + beta X; else alpha acc
    float *part;       // PARTIAL: [matrix][tile][split][256][256]
    const __half *res; // A, or X: the high halves, the low ones res_low elements behind them
    size_t res_low;
    int batch; // the low halves of matrix i are matrix batch + i of a pair
    // LAST
    __nv_bfloat16 *out;
    long long ld_out, out_stride;
    int out_rows, out_cols;
    float out_scale;
    bool tall, vec_out;
    int32_t *status;
};
struct ProductUnit {
    int matrix, row, col, kb0, kb1, index;
};
// the r-th tile on or above the diagonal of a square of tiles, column by column
__device__ __forceinline__ void upper_tile(int r, int &row, int &col)
{
    col = (int)((sqrtf(8.f * r + 1.f) - 1.f) * 0.5f);
    while (col * (col + 1) / 2 > r)
        --col;
    while ((col + 1) * (col + 2) / 2 <= r)
        ++col;
    row = r - col * (col + 1) / 2;
}
template <int FORM, int PN>
__device__ __forceinline__ ProductUnit product_unit(const ProductArgs &p, int u)
{
    ProductUnit t;
    const int tile = u / p.splits, split = u - tile * p.splits;
    t.index = u;
    t.matrix = tile / p.tiles;
    const int r = tile - t.matrix * p.tiles;
    if (updates(FORM))
        t.row = r / p.col_tiles, t.col = r - t.row * p.col_tiles;
    else if (PN == PT) {
        upper_tile(r, t.row, t.col);
    } else { // p.col_tiles - 2 row of them in a row of tiles
        int i = r;
        for (t.row = 0; i >= p.col_tiles - 2 * t.row; ++t.row)
            i -= p.col_tiles - 2 * t.row;
        t.col = 2 * t.row + i;
    }
    t.row *= PT, t.col *= PN;
    t.kb0 = split * p.kb_per_split;
    t.kb1 = min(p.k_blocks, t.kb0 + p.kb_per_split);
    return t;
}

// PN: columns of a tile.  tmA, tmB: boxes of 128 rows x 64 (tmB of UPDATE, LAST and PN = 128: 64 rows x 64); tmC: the output, boxes of
// 32 rows x 32, 64-byte swizzle
template <int FORM, int PN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS, 1)
    orth_product_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const __grid_constant__ CUtensorMap tmC,
                        const ProductArgs p)
{
    constexpr int STAGE = HALF + PN * 64, PART = PN / 2; // bytes; columns of an epilogue warp
    constexpr bool RES = FORM == POLY || updates(FORM); // there is a residual input
    extern __shared__ uint8_t orth_smem[];
    uint8_t *smem = (uint8_t *)(((uintptr_t)orth_smem + 1023) & ~(uintptr_t)1023); // the same offset in both CTAs
    uint64_t *bars = (uint64_t *)(smem + BAR_OFF);
    const uint32_t full0 = smem_u32(bars), empty0 = smem_u32(bars + STAGES), tfull0 = smem_u32(bars + 2 * STAGES),
                   tempty0 = smem_u32(bars + 2 * STAGES + 2), drain = smem_u32(bars + 2 * STAGES + 4);
    uint32_t *tmem_slot = (uint32_t *)(bars + 2 * STAGES + 5);
    volatile int *abort_flag = (volatile int *)(tmem_slot + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();
    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(full0 + 8 * s, 1);
            mbar_init(empty0 + 8 * s, 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(tfull0 + 8 * a, 1);
            mbar_init(tempty0 + 8 * a, 2 * EPI_WARPS); // the leader's counts the epilogue warps of both CTAs
        }
        mbar_init(drain, 1);
        *abort_flag = 0;
        fence_barrier_init();
        prefetch_tmap(&tmA);
        prefetch_tmap(&tmB);
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync(); // both CTAs' barriers exist
    tc_fence_after();
    grid_dep_wait();
    const uint32_t tmem_base = *tmem_slot;
    const int first = (int)blockIdx.x >> 1, step = (int)gridDim.x >> 1;

    if (warp == 0) {
        // TMA producer of the CTA's halves; all copies of a stage complete on the leader's barrier
        if (lane == 0) {
            int stage = 0, issued = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int u = first; u < p.units && ok; u += step) {
                const ProductUnit un = product_unit<FORM, PN>(p, u);
                const int am = un.row + (int)rank * 128, bn = un.col + (int)rank * (PN / 2);
                for (int i = 2 * un.kb0; i < 2 * un.kb1; ++i) { // the high, then the low halves of a K block
                    const int kb = i >> 1, matrix = un.matrix + (i & 1 ? p.batch : 0);
                    if (!mbar_wait(empty0 + 8 * stage, phase ^ 1, abort_flag)) {
                        ok = false;
                        break;
                    }
                    const uint32_t fb = map_to_leader(full0 + 8 * stage);
                    if (rank == 0)
                        mbar_arrive_expect_tx(full0 + 8 * stage, 2 * STAGE);
                    const uint32_t sa = smem_u32(smem + stage * STAGE), sb = sa + HALF;
                    tma_load_3d_pair(sa, &tmA, fb, kb * BK, am, matrix);
                    if constexpr (updates(FORM)) {
                        tma_load_3d_pair(sb, &tmB, fb, bn, kb * BK, matrix);
                        if (PN == PT)
                            tma_load_3d_pair(sb + BK * 128, &tmB, fb, bn + 64, kb * BK, matrix);
                    } else {
                        tma_load_3d_pair(sb, &tmB, fb, kb * BK, bn, matrix);
                    }
                    ++issued;
                    if (++stage == STAGES) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
            }
            if (!ok && rank == 0) { // copies in flight land (a bounded wait) before the CTA may leave
                int s = stage;
                uint32_t ph = phase;
                for (int i = 0; i < min(issued, STAGES); ++i) {
                    if (--s < 0) {
                        s = STAGES - 1;
                        ph ^= 1;
                    }
                    const long long t0 = clock64();
                    while (!mbar_try_wait(full0 + 8 * s, ph) && clock64() - t0 < 200000000ll) {
                    }
                }
            }
        }
    } else if (warp == 1) {
        // MMA issuer (leader)
        if (lane == 0 && rank == 0) {
            constexpr uint32_t idesc = (1u << 4) | ((updates(FORM) ? 1u : 0u) << 16) | ((uint32_t)(PN >> 3) << 17) | ((uint32_t)(PT >> 4) << 24);
            int stage = 0, acc = 0;
            uint32_t phase = 0, acc_phase = 0;
            bool ok = true;
            for (int u = first; u < p.units && ok; u += step) {
                const ProductUnit un = product_unit<FORM, PN>(p, u);
                if (!mbar_wait(tempty0 + 8 * acc, acc_phase ^ 1, abort_flag))
                    break;
                tc_fence_after();
                const uint32_t tmem_d = tmem_base + acc * PT;
                const auto multiply = [&](int left, int right, bool clear) { // of the operands in these slots
                    const uint32_t a = smem_u32(smem + left * STAGE), b = smem_u32(smem + right * STAGE) + HALF;
                    const uint64_t adesc = umma_smem_desc(a, 16, 1024), bdesc = umma_smem_desc(b, updates(FORM) ? BK * 128 : 16, 1024);
                    constexpr uint64_t a_step = 2, b_step = updates(FORM) ? (16 * 128) >> 4 : 2; // 16 of K, in 16-byte units
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        umma_pair<1>(tmem_d, adesc + k * a_step, bdesc + k * b_step, idesc, !clear || k > 0 ? 1u : 0u);
                };
                int high = 0; // the slot of the block's high halves
                for (int i = 2 * un.kb0; i < 2 * un.kb1; ++i) {
                    if (!mbar_wait(full0 + 8 * stage, phase, abort_flag)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    if (i & 1) {
                        multiply(high, stage, false);
                        multiply(stage, high, false);
                        commit_both(empty0 + 8 * high);
                        commit_both(empty0 + 8 * stage);
                    } else {
                        multiply(stage, stage, i == 2 * un.kb0);
                        high = stage;
                    }
                    if (++stage == STAGES) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
                if (ok)
                    commit_both(tfull0 + 8 * acc);
                acc ^= 1;
                if (acc == 0)
                    acc_phase ^= 1;
            }
            commit_own(drain); // every MMA issued so far has completed once this arrives
            const long long t0 = clock64();
            while (!mbar_try_wait(drain, 0) && clock64() - t0 < 1500000000ll) {
            }
        }
    } else {
        // epilogue: a warp takes 32 rows x PART columns in blocks of 32 x 32, thread = row
        const int quarter = warp & 3, ew = warp - 2, part = ew >> 2;
        uint8_t *const high = smem + STG_OFF + ew * WARP_BYTES, *const low = high + BLOCK, *const mirrored = low + BLOCK;
        const int sw = (lane >> 1) & 3; // the 64-byte swizzle of the thread's row
        uint32_t column[4];             // of the thread in a mirrored row; the swizzle of rows 8 i + 2 j and the one behind is j
#pragma unroll
        for (int j = 0; j < 4; ++j)
            column[j] = smem_u32(mirrored) + (((lane >> 3) ^ j) << 4) + (lane & 7) * 2;
        int acc = 0;
        uint32_t acc_phase = 0;
        for (int u = first; u < p.units; u += step) {
            const ProductUnit un = product_unit<FORM, PN>(p, u);
            const uint32_t taddr = tmem_base + ((uint32_t)(quarter * 32) << 16) + acc * PT + part * PART;
            const int row0 = un.row + (int)rank * 128 + quarter * 32, col0 = un.col + part * PART;
            const auto there = [&](int c) { return row0 < p.n && col0 + c * 32 < p.cols; }; // multiples of 32: a block is there or not
            uint4 rows[2][4]; // of the next block of the residual input, high and low halves: 4 lanes a row, 8 rows at a time
            const auto fetch = [&](int c) {
                if constexpr (RES) {
                    if (!there(c))
                        return;
                    const __half *from = p.res + ((size_t)un.matrix * p.n + row0 + (lane >> 2)) * p.cols + col0 + c * 32 + (lane & 3) * 8;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        rows[0][i] = *(const uint4 *)(from + (size_t)(8 * i) * p.cols);
                        rows[1][i] = *(const uint4 *)(from + p.res_low + (size_t)(8 * i) * p.cols);
                    }
                }
            };
            fetch(0);
            if (!__all_sync(0xffffffffu, mbar_wait(tfull0 + 8 * acc, acc_phase, abort_flag)))
                break;
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < PART / 32; ++c) {
                uint32_t r[32];
                __syncwarp(); // lane 0 comes from its stores
                tmem_ld32(taddr + c * 32, r);
                tmem_ld_wait();
                if (c == PART / 32 - 1) { // the accumulator is read: the next tile may have it
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0)
                        mbar_arrive_cluster(map_to_leader(tempty0 + 8 * acc));
                }
                if constexpr (FORM != PARTIAL && FORM != LAST) {
                    if (lane == 0)
                        bulk_wait_read<0>(); // the stores of the block before have read what lies here
                    __syncwarp();
                }
                if constexpr (RES) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int at = (8 * i + (lane >> 2)) * 64 + (((lane & 3) ^ (lane >> 3 & 3)) << 4);
                        *(uint4 *)(high + at) = rows[0][i];
                        *(uint4 *)(low + at) = rows[1][i];
                    }
                    __syncwarp();
                    if (c + 1 < PART / 32)
                        fetch(c + 1);
                }
                // 8 columns of the thread's row: alpha times the accumulator, and beta times the residual input
                const auto eight = [&](int i, float (&v)[8]) {
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        v[j] = p.alpha * __uint_as_float(r[8 * i + j]);
                    if constexpr (RES) {
                        const int at = lane * 64 + ((i ^ sw) << 4);
                        float x[8];
                        orth_join8(*(const uint4 *)(high + at), *(const uint4 *)(low + at), x);
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            v[j] = fmaf(p.beta, x[j], v[j]);
                    }
                };
                const int col = col0 + c * 32;
                if constexpr (FORM == PARTIAL) {
                    // through shared memory, so that 8 lanes write 128 bytes of a row
                    __syncwarp();
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        *(uint4 *)(high + lane * 128 + ((i ^ (lane & 7)) << 4)) = make_uint4(r[4 * i], r[4 * i + 1], r[4 * i + 2], r[4 * i + 3]);
                    __syncwarp();
                    float *to = p.part + ((size_t)un.index * PT + (row0 - un.row)) * PT + (col - un.col);
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int at = i * 4 + (lane >> 3), q = lane & 7;
                        *(uint4 *)(to + (size_t)at * PT + q * 4) = *(const uint4 *)(high + at * 128 + ((q ^ (at & 7)) << 4));
                    }
                } else if constexpr (FORM == LAST) {
                    const int i0 = row0 + lane; // X's row: (tall) a column of the result, 32 neighbours a store
                    __nv_bfloat16 *out = p.out + un.matrix * p.out_stride;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float v[8];
                        eight(i, v);
                        __nv_bfloat162 o[4];
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            o[j] = __floats2bfloat162_rn(v[2 * j] * p.out_scale, v[2 * j + 1] * p.out_scale);
                        if (p.tall) {
#pragma unroll
                            for (int j = 0; j < 8; ++j)
                                if (i0 < p.out_cols && col + 8 * i + j < p.out_rows)
                                    out[(long long)(col + 8 * i + j) * p.ld_out + i0] = j & 1 ? __high2bfloat16(o[j / 2]) : __low2bfloat16(o[j / 2]);
                        } else {
                            *(uint4 *)(mirrored + lane * 128 + ((((c & 1) * 4 + i) ^ (lane & 7)) << 4)) =
                                make_uint4(*(uint32_t *)&o[0], *(uint32_t *)&o[1], *(uint32_t *)&o[2], *(uint32_t *)&o[3]);
                        }
                    }
                    if (!p.tall && c & 1) { // 32 rows x 64 by rows
                        __syncwarp();
                        const int left = col - 32, right = min(p.out_cols - left, 64);
                        if (p.vec_out) {
#pragma unroll
                            for (int i = 0; i < 8; ++i) {
                                const int at = i * 4 + (lane >> 3), q = lane & 7;
                                const uint4 eight = *(const uint4 *)(mirrored + at * 128 + ((q ^ (at & 7)) << 4));
                                __nv_bfloat16 *to = out + (long long)(row0 + at) * p.ld_out + left + q * 8;
                                if (row0 + at >= p.out_rows)
                                    continue;
                                if (q * 8 + 8 <= right)
                                    *(uint4 *)to = eight;
                                else
#pragma unroll
                                    for (int j = 0; j < 8; ++j)
                                        if (q * 8 + j < right)
                                            to[j] = ((const __nv_bfloat16 *)&eight)[j];
                            }
                        } else {
                            for (int at = 0; at < 32 && row0 + at < p.out_rows; ++at)
#pragma unroll
                                for (int h = 0; h < 2; ++h) {
                                    const int k = h * 32 + lane;
                                    if (k < right)
                                        out[(long long)(row0 + at) * p.ld_out + left + k] =
                                            *(const __nv_bfloat16 *)(mirrored + at * 128 + (((k >> 3) ^ (at & 7)) << 4) + (k & 7) * 2);
                                }
                        }
                        __syncwarp();
                    }
                } else {
                    const bool mirror = FORM != UPDATE && un.col >= un.row + PT;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float v[8];
                        eight(i, v);
                        uint4 h, l;
                        orth_split8(v, h, l);
                        const int at = lane * 64 + ((i ^ sw) << 4); // in the place of the thread's residual input
                        *(uint4 *)(high + at) = h;
                        *(uint4 *)(low + at) = l;
                        if (mirror) {
                            // element (column, row) of the transpose: a column's 32 rows are the 64 bytes of one row there
                            const uint32_t hw[4] = {h.x, h.y, h.z, h.w}, lw[4] = {l.x, l.y, l.z, l.w};
#pragma unroll
                            for (int j = 0; j < 8; ++j) {
                                const uint32_t to = column[j >> 1] + (8 * i + j) * 64;
                                asm volatile("st.shared.u16 [%0], %1;" ::"r"(to), "h"((uint16_t)(hw[j >> 1] >> 16 * (j & 1))) : "memory");
                                asm volatile("st.shared.u16 [%0], %1;" ::"r"(to + BLOCK), "h"((uint16_t)(lw[j >> 1] >> 16 * (j & 1))) : "memory");
                            }
                        }
                    }
                    fence_proxy_async();
                    __syncwarp();
                    if (lane == 0) {
                        if (there(c)) {
                            tma_store_3d(&tmC, smem_u32(high), col, row0, un.matrix);
                            tma_store_3d(&tmC, smem_u32(low), col, row0, un.matrix + p.batch);
                            if (mirror) {
                                tma_store_3d(&tmC, smem_u32(mirrored), row0, col, un.matrix);
                                tma_store_3d(&tmC, smem_u32(mirrored + BLOCK), row0, col, un.matrix + p.batch);
                            }
                        }
                        bulk_commit();
                    }
                }
            }
            acc ^= 1;
            if (acc == 0)
                acc_phase ^= 1;
        }
        if (lane == 0)
            bulk_wait_read<0>(); // the blocks must outlive the stores that read them
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync(); // nothing of the peer refers to this CTA any more
    if (warp == 1)
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512u) : "memory");
    if (threadIdx.x == 0 && *abort_flag)
        atomicOr(p.status, TS2_STATUS_WAIT_TIMEOUT);
}

// The K ranges of SQUARE or (with a) POLY added in their order; 64 x 64 of a tile per block
__global__ void __launch_bounds__(256) orth_join_kernel(const float *__restrict__ part, const ProductArgs p, bool poly, __half *out, size_t out_low)
{
    grid_dep_wait();
    __shared__ float tile[64][65];
    const int q = threadIdx.x >> 3, c8 = (threadIdx.x & 7) * 8;
    int row, col;
    upper_tile(blockIdx.y, row, col);
    const bool mirror = row != col;
    const int i0 = (blockIdx.x >> 2) * 64, j0 = (blockIdx.x & 3) * 64;
    row = row * PT + i0, col = col * PT + j0;
    if (row >= p.n || col >= p.n)
        return;
    part += ((size_t)blockIdx.z * p.tiles + blockIdx.y) * p.splits * PT * PT;
    out += (size_t)blockIdx.z * p.n * p.n;
    const __half *a = p.res + (size_t)blockIdx.z * p.n * p.n; // poly
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int i = q + 32 * h;
        float sum[8] = {};
        for (int s = 0; s < p.splits; ++s) {
            const float4 *from = (const float4 *)(part + ((size_t)s * PT + i0 + i) * PT + j0 + c8);
            const float4 x = from[0], y = from[1];
            sum[0] += x.x, sum[1] += x.y, sum[2] += x.z, sum[3] += x.w, sum[4] += y.x, sum[5] += y.y, sum[6] += y.z, sum[7] += y.w;
        }
        const size_t at = (size_t)(row + i) * p.n + col + c8;
        float old[8] = {};
        if (poly)
            orth_join8(*(const uint4 *)(a + at), *(const uint4 *)(a + p.res_low + at), old);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            sum[j] = fmaf(p.beta, old[j], p.alpha * sum[j]);
            tile[i][c8 + j] = sum[j];
        }
        orth_split8(sum, *(uint4 *)(out + at), *(uint4 *)(out + out_low + at));
    }
    if (!mirror)
        return;
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int i = q + 32 * h;
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j)
            v[j] = tile[c8 + j][i];
        const size_t at = (size_t)(col + i) * p.n + row + c8;
        orth_split8(v, *(uint4 *)(out + at), *(uint4 *)(out + out_low + at));
    }
}

// ---- host ------------------------------------------------------------------------------------------------------------
// largest |a s + b s^3 + c s^5| over [0, top]: at the end or where the derivative a + 3 b q + 5 c q^2, q = s^2, is zero
static double poly_max(double a, double b, double c, double top)
{
    const auto p = [&](double s) { return std::fabs(s * (a + s * s * (b + s * s * c))); };
    double most = p(top);
    const double disc = 9 * b * b - 20 * a * c;
    if (disc >= 0) {
        const double t = -0.5 * (3 * b + std::copysign(std::sqrt(disc), b)); // no difference of near numbers, however small c is
        for (const double q : {t / (5 * c), a / t})
            if (q > 0 && q < top * top)
                most = std::max(most, p(std::sqrt(q)));
    }
    return most;
}
bool orthogonalize_in_range(const float coef[3], int steps)
{
    double x = 1.;
    for (int k = 0; k < steps; ++k) {
        x *= 1.02; // the roundings of a step move a singular value by less
        const double q = x * x, b = coef[1], c = coef[2];
        double most = std::fabs(b * q + c * q * q);
        if (c && -b / (2 * c) > 0 && -b / (2 * c) < q)
            most = std::max(most, b * b / (4 * std::fabs(c)));
        if (!(x <= MAX_X) || !(most <= MAX_B))
            return false;
        x = poly_max(coef[0], b, c, x);
    }
    return x * 1.02 <= MAX_X;
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                                  const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
// [batch][rows][cols] halves; box: `wide` elements (64: 128-byte swizzle, 32: 64-byte) x `high` rows
static int half_map(CUtensorMap *tm, const void *base, int64_t cols, int64_t rows, int64_t batch, int wide, int high)
{
    static const EncodeTiledFn encode = [] {
        void *f = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess)
            f = nullptr;
        return (EncodeTiledFn)f;
    }();
    if (!encode)
        return fail(TS2_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
    const cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)batch};
    const cuuint64_t strides[2] = {(cuuint64_t)cols * 2, (cuuint64_t)(cols * rows * 2)};
    const cuuint32_t box[3] = {(cuuint32_t)wide, (cuuint32_t)high, 1}, estr[3] = {1, 1, 1};
    const CUresult r = encode(tm, CU_TENSOR_MAP_DATA_TYPE_UINT16, 3, const_cast<void *>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              wide == 32 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? TS2_OK : fail(TS2_ERR_CUDA, "cuTensorMapEncodeTiled failed with code %d", (int)r);
}

template <int FORM, int PN = PT>
static int product(const Ctx &c, const CUtensorMap &A, const CUtensorMap &B, const CUtensorMap &C, const ProductArgs &p)
{
    static std::atomic<unsigned> ready{0}; // a bit a device: it has been told how much shared memory the kernel takes
    const unsigned bit = 1u << (c.device & 15);
    if (!(ready.load() & bit)) {
        TS2_CUDA(cudaFuncSetAttribute((const void *)orth_product_kernel<FORM, PN>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM));
        ready.fetch_or(bit);
    }
    const int pairs = std::min(sm_count(c.device) / 2, p.units);
    TS2_LAUNCH((orth_product_kernel<FORM, PN>), 2 * pairs, THREADS, SMEM, c.stream, A, B, C, p);
    return TS2_OK;
}

// K ranges of a symmetric product: the number with the least estimated time, in K blocks of a whole tile (0.8 us each).  Halves of few tiles
// (see `few`) take 0.9 a block; ranges leave fp32 and are joined by another launch, 2.5 and their bytes more than such an epilogue.
// SQUARE, us of a call with whole tiles, halves, 2 and 4 ranges: 1024 x 1024 332, 306, 292, 278; 2000 x 2000 572, 539, 513, 526; 512 x 512
// 235, 212, 209, 203; 3 x 1000 x 333 246, 233, 217, 204; SQUARE and POLY of 3000 x 3001 whole 1500, 2 ranges 1413.
static int choose_splits(int pairs, int64_t tiles, int k_blocks)
{
    double best = 2 * tiles <= pairs ? 0.9 * k_blocks + 1 : (double)ceil_div(tiles, pairs) * (k_blocks + 1) + 2;
    int splits = 1;
    for (int s = 2; s <= 64 && s <= k_blocks; ++s) {
        const int per = (int)ceil_div(k_blocks, s), used = (int)ceil_div(k_blocks, per);
        const double cost = (double)ceil_div(tiles * s, pairs) * (per + 1) + 3.5 + 0.1 * tiles * s + 0.1 * s;
        if (used == s && cost < best)
            best = cost, splits = s;
    }
    return splits;
}

template <class T>
static int orthogonalize_typed(const Ctx &c, const T *g, int64_t ld, int64_t stride, int batch, int rows, int cols, const float coef[3], int steps,
                               float out_scale, __nv_bfloat16 *out, int64_t ld_out, int64_t out_stride)
{
    const bool tall = rows > cols;
    const int n = std::min(rows, cols), m = std::max(rows, cols), np = (int)ceil_div(n, 64) * 64, mp = (int)ceil_div(m, 64) * 64;
    const int pairs = sm_count(c.device) / 2;
    const int n_part = (int)std::max<int64_t>(1, std::min<int64_t>(ceil_div((int64_t)rows * cols, 8192), std::max(1, 4 * sm_count(c.device) / batch)));
    const int nt = (int)ceil_div(np, PT), mt = (int)ceil_div(mp, PT), upper = nt * (nt + 1) / 2;
    const size_t x = (size_t)batch * np * mp, a = (size_t)batch * np * np;
    const int split1 = choose_splits(pairs, (int64_t)batch * upper, mp / BK), split2 = choose_splits(pairs, (int64_t)batch * upper, np / BK);
    const int most = std::max(split1, split2);
    const size_t part_bytes = most > 1 ? (size_t)batch * upper * most * PT * PT * 4 : 0;
    Scratch s(c, part_bytes + x * 8 + a * 8 + (size_t)batch * n_part * 8);
    if (s.rc != TS2_OK)
        return s.rc;
    // pairs: the low halves behind the high ones
    float *part = (float *)s.p;
    __half *X[2] = {(__half *)((uint8_t *)s.p + part_bytes), (__half *)((uint8_t *)s.p + part_bytes) + 2 * x}, *A = X[1] + 2 * x, *B = A + 2 * a;
    double *sums = (double *)(B + 2 * a);

    const bool vec = ((uintptr_t)g | (uintptr_t)(ld * sizeof(T)) | (uintptr_t)(stride * sizeof(T))) % 16 == 0;
    TS2_LAUNCH((orth_sum2_kernel<T>), dim3(n_part, batch), 256, 0, c.stream, g, ld, stride, rows, cols, vec, sums);
    const dim3 blocks(mp / 64, np / 64, batch);
    if (tall)
        TS2_LAUNCH((orth_load_kernel<T, true>), blocks, 256, 0, c.stream, g, ld, stride, rows, cols, vec, sums, n_part, np, mp, X[0], X[0] + x);
    else
        TS2_LAUNCH((orth_load_kernel<T, false>), blocks, 256, 0, c.stream, g, ld, stride, rows, cols, vec, sums, n_part, np, mp, X[0], X[0] + x);
    CUtensorMap x_rows[2], x_cols[2], x_block[2], a_rows, a_half, a_block, b_rows, b_block; // x_cols, a_half: boxes of 64 rows x 64
    int rc = TS2_OK;
    for (int i = 0; i < 2 && rc == TS2_OK; ++i) {
        rc = half_map(&x_rows[i], X[i], mp, np, 2 * batch, 64, 128);
        if (rc == TS2_OK)
            rc = half_map(&x_cols[i], X[i], mp, np, 2 * batch, 64, 64);
        if (rc == TS2_OK)
            rc = half_map(&x_block[i], X[i], mp, np, 2 * batch, 32, 32);
    }
    if (rc != TS2_OK || (rc = half_map(&a_rows, A, np, np, 2 * batch, 64, 128)) || (rc = half_map(&a_half, A, np, np, 2 * batch, 64, 64)) ||
        (rc = half_map(&a_block, A, np, np, 2 * batch, 32, 32)) || (rc = half_map(&b_rows, B, np, np, 2 * batch, 64, 128)) ||
        (rc = half_map(&b_block, B, np, np, 2 * batch, 32, 32)))
        return rc;
    ProductArgs p = {};
    p.status = device_status_word(c.device);
    if (!p.status)
        return fail(TS2_ERR_CUDA, "no device status word");
    p.n = np;
    p.batch = batch;
    p.part = part;
    // Tiles of 256 x 128 where those of 256 x 256 would leave half of the device without any: half the products and half the epilogue
    // each, and more SMs at work.  4 x 130 x 140 184 -> 144 us, 8 x 200 x 264 207 -> 159, 400 x 500 262 -> 207; from 38 tiles on narrow
    // ones would come in a second round.  Outputs of so few tiles that K is divided keep whole tiles.
    const auto few = [&](int64_t tiles) { return 2 * tiles <= pairs; };
    const auto symmetric = [&](bool poly, int k, int splits, const CUtensorMap &in, const CUtensorMap &in_half, const CUtensorMap &to, __half *dst) {
        p.cols = np, p.tiles = upper, p.col_tiles = 0;
        p.k_blocks = k / BK, p.splits = splits, p.kb_per_split = (int)ceil_div(p.k_blocks, splits), p.units = batch * upper * splits;
        if (splits == 1 && few(batch * upper)) {
            p.col_tiles = (int)ceil_div(np, 128), p.tiles = 0;
            for (int r = 0; r < nt; ++r)
                p.tiles += std::max(0, p.col_tiles - 2 * r);
            p.units = batch * p.tiles;
            return poly ? product<POLY, 128>(c, in, in_half, to, p) : product<SQUARE, 128>(c, in, in_half, to, p);
        }
        if (splits == 1)
            return poly ? product<POLY>(c, in, in, to, p) : product<SQUARE>(c, in, in, to, p);
        if (int e = product<PARTIAL>(c, in, in, to, p))
            return e;
        TS2_LAUNCH(orth_join_kernel, dim3(16, upper, batch), 256, 0, c.stream, part, p, poly, dst, a);
        return TS2_OK;
    };
    for (int k = 0; k < steps; ++k) {
        const int now = k & 1;
        p.alpha = SA / (SX * SX), p.beta = 0.f;
        if ((rc = symmetric(false, mp, split1, x_rows[now], x_cols[now], a_block, A)))
            return rc;
        p.alpha = SB * coef[2] / (SA * SA), p.beta = SB * coef[1] / SA, p.res = A, p.res_low = a;
        if ((rc = symmetric(true, np, split2, a_rows, a_half, b_block, B)))
            return rc;
        p.alpha = 1.f / SB, p.beta = coef[0], p.res = X[now], p.res_low = x;
        p.cols = mp, p.tiles = nt * mt, p.col_tiles = mt, p.k_blocks = np / BK, p.splits = 1, p.kb_per_split = p.k_blocks, p.units = batch * nt * mt;
        if (k == steps - 1) {
            p.out = out, p.ld_out = ld_out, p.out_stride = out_stride, p.out_rows = rows, p.out_cols = cols, p.out_scale = out_scale / SX, p.tall = tall;
            p.vec_out = ((uintptr_t)out | (uintptr_t)(ld_out * 2) | (uintptr_t)(out_stride * 2)) % 16 == 0;
        }
        if (few(p.units)) {
            p.col_tiles = (int)ceil_div(mp, 128), p.tiles = nt * p.col_tiles, p.units = batch * p.tiles;
            rc = k < steps - 1 ? product<UPDATE, 128>(c, b_rows, x_cols[now], x_block[now ^ 1], p)
                               : product<LAST, 128>(c, b_rows, x_cols[now], x_block[now ^ 1], p);
        } else {
            rc = k < steps - 1 ? product<UPDATE>(c, b_rows, x_cols[now], x_block[now ^ 1], p)
                               : product<LAST>(c, b_rows, x_cols[now], x_block[now ^ 1], p);
        }
        if (rc != TS2_OK)
            return rc;
    }
    return TS2_OK;
}

int orthogonalize(const Ctx &c, int type, const void *g, int64_t ld, int64_t stride, int batch, int rows, int cols, const float coef[3], int steps,
                  float out_scale, void *out, int64_t ld_out, int64_t out_stride)
{
    if (orth_chip_ranks(rows, cols))
        return orth_chip(c, type, g, ld, stride, batch, rows, cols, coef, steps, out_scale, out, ld_out, out_stride);
    __nv_bfloat16 *o = (__nv_bfloat16 *)out;
    switch (type) {
    case TS2_OUT_F32: return orthogonalize_typed(c, (const float *)g, ld, stride, batch, rows, cols, coef, steps, out_scale, o, ld_out, out_stride);
    case TS2_OUT_F16: return orthogonalize_typed(c, (const __half *)g, ld, stride, batch, rows, cols, coef, steps, out_scale, o, ld_out, out_stride);
    case TS2_OUT_BF16:
        return orthogonalize_typed(c, (const __nv_bfloat16 *)g, ld, stride, batch, rows, cols, coef, steps, out_scale, o, ld_out, out_stride);
    default: return fail(TS2_ERR_INVALID_ARG, "orthogonalize: unknown type %d", type);
    }
}

} // namespace ts2
