// Orthogonalised updates (kernels_orth.cu has the formula and its scaling) of matrices with at most 128 rows or columns, in one launch
// and without memory in between: a cluster holds a matrix.  Each CTA has the 128 rows (padded with zeros) of up to 256 columns of X:
// as fp32 in tensor memory, thread = row, and as two fp16 halves in shared memory, the operands of the products
//     A = X X^T   (the CTAs' parts are added through distributed shared memory, each 128 / cluster rows for all)
//     B = b A + c A A   (every CTA for itself, in the place of A)      X = a X + B X
// Operands in one fp16 half each would take a third of the tensor work (128 x 256: 34 us instead of 53), but results of few directions or
// few rows were up to 2e-2 off: the rounding of X meets the large entries of B, and what it leaves in directions that X does not have
// grows by a factor a in every step.  With two halves every matrix is within 1e-4.
// A chain of small products: its latency is the bound, 9 us a step (4 of them tensor work at two chunks of columns), 10 us to bring G in
// and normalise it, and with more than one CTA the exchange of A, 5 - 8 us a step.  64 x 64: 38 us, 128 x 256: 53, 128 x 4000 on a cluster
// of 16: 112.
#include "kernels.cuh"
#include "orth.cuh"
#include "pair_ptx.cuh"
#include <algorithm>

namespace ts2 {

namespace {

constexpr int THREADS = 256, MAX_CHUNKS = 2, MAX_CLUSTER = 16;
constexpr int BLK = 128 * 128;   // 128 rows x 64 columns of fp16, 128-byte swizzle
constexpr int PART = 2 * BLK;    // 128 x 128 of fp16
// X's chunks, high half and low half each; behind them A, then B, alike.  The staging area of 128 x 128 fp32 is the same memory: it
// is used while there is neither (G on its way in, the CTAs' parts of A, the result on its way out).
constexpr int A_OFF = MAX_CHUNKS * 2 * PART, END_OFF = A_OFF + 2 * PART;
constexpr int SMEM = END_OFF + 128 + 1024;
static_assert(SMEM <= 232448 && 2 * PART == 128 * 128 * 4, "shared memory budget");
constexpr uint32_t WORK = MAX_CHUNKS * 128; // tensor-memory columns of the products at hand; X's chunks lie before them

struct ChipArgs {
    const void *g;
    long long ld, stride;
    int rows, cols, chunks; // chunks: of 128 columns of X in a CTA
    int steps;
    float a, b, c, out_scale;
    __nv_bfloat16 *out;
    long long ld_out, out_stride;
    bool vec, vec_out;
    int32_t *status;
};

__device__ __forceinline__ unsigned cluster_size()
{
    unsigned r;
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}
// 16-byte piece c (0 .. 15) of row r of 128 columns of fp16, as two swizzled blocks
__device__ __forceinline__ uint32_t piece(int r, int c) { return (uint32_t)((c >> 3) * BLK + r * 128 + (((c & 7) ^ (r & 7)) << 4)); }

// fp32 staging of 128 x 128: where 4 elements of row r from column c (a multiple of 4) on lie, so that neither 8 rows nor 8 pieces of a
// row, nor every eighth row, meet in a bank
__device__ __forceinline__ int staged(int r, int c) { return r * 128 + (((c >> 2) ^ ((r ^ (r >> 3)) & 7)) << 2); }

// 32 values as two halves to the columns [32 j, +32) of the thread's row
__device__ __forceinline__ void put_halves(uint8_t *base, int row, int j, const float (&v)[32])
{
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float e[8] = {v[8 * i], v[8 * i + 1], v[8 * i + 2], v[8 * i + 3], v[8 * i + 4], v[8 * i + 5], v[8 * i + 6], v[8 * i + 7]};
        uint4 hi, lo;
        orth_split8(e, hi, lo);
        *(uint4 *)(base + piece(row, 4 * j + i)) = hi;
        *(uint4 *)(base + PART + piece(row, 4 * j + i)) = lo;
    }
}

template <class T, bool TALL>
__global__ void __launch_bounds__(THREADS, 1) orth_chip_kernel(const ChipArgs p)
{
    extern __shared__ uint8_t chip_smem[];
    uint8_t *smem = (uint8_t *)(((uintptr_t)chip_smem + 1023) & ~(uintptr_t)1023); // the same offset in every CTA of a cluster
    float *stage = (float *)(smem + A_OFF);
    uint64_t *bar_at = (uint64_t *)(smem + END_OFF);
    uint32_t *tmem_slot = (uint32_t *)(bar_at + 1);
    volatile int *abort_flag = (volatile int *)(tmem_slot + 1);
    double *sums = (double *)(smem + END_OFF + 32); // a warp's, the CTA's
    const uint32_t bar = smem_u32(bar_at);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, quarter = warp & 3, half = warp >> 2;
    const unsigned rank = cluster_rank(), ranks = cluster_size();
    if (threadIdx.x == 0) {
        mbar_init(bar, 1);
        *abort_flag = 0;
        fence_barrier_init();
    }
    if (warp == 1) { // a warp that no branch has split
        tmem_alloc(smem_u32(tmem_slot), 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    if (ranks > 1)
        cluster_sync(); // all CTAs have started: their shared memory can be used
    tc_fence_after();
    grid_dep_wait();
    const uint32_t tmem = *tmem_slot, lane_base = tmem + ((uint32_t)(quarter * 32) << 16) + half * 64; // the thread's row, its half of 128 columns
    const int row = quarter * 32 + lane, matrix = blockIdx.x / ranks;
    const int j0 = (int)rank * p.chunks * 128;
    const T *g = (const T *)p.g + matrix * p.stride;
    // (accesses of tensor memory are a warp's: lanes that come from branches of their own meet first)
    const auto load32 = [&](uint32_t column, float (&v)[32]) {
        uint32_t r[32];
        __syncwarp();
        tmem_ld32(lane_base + column, r);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 32; ++i)
            v[i] = __uint_as_float(r[i]);
    };
    const auto load64 = [&](uint32_t column, float (&v)[2][32]) { // the thread's half of 128 columns; tmem_ld_wait is the caller's
        uint32_t(&r)[2][32] = (uint32_t(&)[2][32])v;
        __syncwarp();
        tmem_ld32(lane_base + column, r[0]);
        tmem_ld32(lane_base + column + 32, r[1]);
    };
    const auto store32 = [&](uint32_t column, const float (&v)[32]) {
        uint32_t r[32];
#pragma unroll
        for (int i = 0; i < 32; ++i)
            r[i] = __float_as_uint(v[i]);
        __syncwarp();
        tmem_st32(lane_base + column, r);
    };

    const auto staged32 = [&](int column, float (&v)[32]) { // of the thread's row
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float4 f = *(const float4 *)(stage + staged(row, column + 4 * i));
            v[4 * i] = f.x, v[4 * i + 1] = f.y, v[4 * i + 2] = f.z, v[4 * i + 3] = f.w;
        }
    };
    const auto stage32 = [&](int column, const float (&v)[32]) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            *(float4 *)(stage + staged(row, column + 4 * i)) = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
    };

    // ---- G -> X, unscaled, and its sum of squares (fp64: nothing over- or underflows) ----
    double sum = 0.;
    for (int q = 0; q < p.chunks; ++q) {
        const int j = j0 + q * 128, part = threadIdx.x >> 4, c8 = (threadIdx.x & 15) * 8;
        float v[8][8]; // all loads of a chunk are on their way together
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int r = (TALL ? j : 0) + part + 16 * k; // of G
            if (r < p.rows)
                orth_load8(g + r * p.ld, (TALL ? 0 : j) + c8, p.cols, p.vec, v[k]);
            else
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    v[k][i] = 0.f;
        }
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (TALL) {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    stage[staged(c8 + i, (part + 16 * k) & ~3) + (part & 3)] = v[k][i];
            } else {
#pragma unroll
                for (int i = 0; i < 8; i += 4)
                    *(float4 *)(stage + staged(part + 16 * k, c8 + i)) = make_float4(v[k][i], v[k][i + 1], v[k][i + 2], v[k][i + 3]);
            }
        __syncthreads();
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float v[32], most = 0.f;
            staged32(half * 64 + h * 32, v);
#pragma unroll
            for (int i = 0; i < 32; ++i)
                most = fmaxf(most, fabsf(v[i]));
            if (most > 1e-12f && most < 1e15f) { // 32 squares that fp32 holds; a NaN among them makes the sum one
                float four[4] = {};
#pragma unroll
                for (int i = 0; i < 32; ++i)
                    four[i & 3] = fmaf(v[i], v[i], four[i & 3]);
                sum += (double)((four[0] + four[1]) + (four[2] + four[3]));
            } else {
#pragma unroll
                for (int i = 0; i < 32; ++i)
                    sum = fma((double)v[i], (double)v[i], sum);
            }
            store32(q * 128 + h * 32, v);
        }
        __syncthreads();
    }
    tmem_st_wait();
    sum = warp_sum(sum);
    if (lane == 0)
        sums[warp] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        sum = sums[0];
        for (int w = 1; w < THREADS / 32; ++w)
            sum += sums[w];
        sums[8] = sum;
    }
    if (ranks > 1)
        cluster_sync();
    else
        __syncthreads();
    sum = sums[8];
    if (ranks > 1) {
        sum = 0.;
        for (unsigned r = 0; r < ranks; ++r) {
            double s;
            asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(s) : "r"(map_to_rank(smem_u32(sums + 8), r)) : "memory");
            sum += s;
        }
    }
    {
        const double scale = sum == 0. ? 0. : (double)ORTH_SX / sqrt(sum);
        const bool small = !(scale < 1e30); // G is all but denormal, or not finite
        const float scale32 = (float)scale;
        for (int q = 0; q < p.chunks; ++q)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float v[32];
                load32(q * 128 + h * 32, v);
#pragma unroll
                for (int i = 0; i < 32; ++i)
                    v[i] = small ? (float)(v[i] * scale) : v[i] * scale32;
                store32(q * 128 + h * 32, v);
                put_halves(smem + q * 2 * PART, row, half * 2 + h, v);
            }
    }

    // ---- steps ----
    uint32_t phase = 0;
    bool alive = true; // of the whole CTA: no wait has given up
    // The operands in shared memory are complete and the product's columns are free: one thread issues, all wait for the product.
    // After a wait that gave up nothing is multiplied any more, but the CTA keeps its appointments with the rest of the cluster.
    const auto product = [&](auto &&issue) {
        fence_proxy_async();
        tmem_st_wait();
        tc_fence_before();
        __syncthreads();
        tc_fence_after();
        if (alive) {
            if (threadIdx.x == 0) {
                issue();
                tc_commit(bar);
            }
            const bool done = mbar_wait(bar, phase, abort_flag);
            if (!done && threadIdx.x == 0) { // what was issued may still end (a bounded wait): it uses shared and tensor memory
                const long long t0 = clock64();
                while (!mbar_try_wait(bar, phase) && clock64() - t0 < 1500000000ll) {
                }
            }
            alive = __syncthreads_and(done); // warps are whole again, too: what reads tensor memory wants them so
            phase ^= 1;
        }
        tc_fence_after();
    };
    const uint32_t x_at = smem_u32(smem), a_at = smem_u32(smem + A_OFF), work = tmem + WORK;
    constexpr uint32_t IDESC = umma_idesc_f16(128, false, false), IDESC_MN = umma_idesc_f16(128, false, true);
    // A product of operands in two halves: low times high, high times low, high times high (low times low is 2^-22 of it).  The small
    // ones come first, while the sum that they are added to is small.
    const auto halves = [&](auto &&one) {
        one(PART, 0, true);
        one(0, PART, false);
        one(0, 0, false);
    };
    for (int step = 0; step < p.steps; ++step) {
        product([&] { // A = X X^T
            halves([&](int left, int right, bool clear) {
                for (int b = 0; b < 2 * p.chunks; ++b) {
                    const uint32_t at = x_at + (b >> 1) * 2 * PART + (b & 1) * BLK;
                    umma_f16_x4(work, umma_smem_desc(at + left, 16, 1024), umma_smem_desc(at + right, 16, 1024), IDESC, !clear || b > 0, 2, 2);
                }
            });
        });
        constexpr float ALPHA = ORTH_SA / (ORTH_SX * ORTH_SX);
        float w2[2][32];
        load64(WORK, w2);
        tmem_ld_wait();
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float(&v)[32] = w2[h];
#pragma unroll
            for (int i = 0; i < 32; ++i)
                v[i] *= ALPHA;
            if (ranks == 1) {
                put_halves(smem + A_OFF, row, half * 2 + h, v);
            } else {
                stage32(half * 64 + h * 32, v);
            }
        }
        if (ranks > 1) {
            cluster_sync();
            const int rows_each = 128 / (int)ranks;
            uint4 hi[4], lo[4]; // this CTA's 8-column pieces of A: 2048 / ranks of them
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int i = threadIdx.x + q * THREADS;
                if (i >= rows_each * 16)
                    break;
                const int r = (int)rank * rows_each + (i >> 4), c = i & 15;
                const uint32_t at[2] = {smem_u32(stage + staged(r, c * 8)), smem_u32(stage + staged(r, c * 8 + 4))};
                float v[8] = {};
                for (unsigned k0 = 0; k0 < ranks; k0 += 2) { // in their order, two CTAs' loads at a time
                    float4 f[2][2];
#pragma unroll
                    for (int k = 0; k < 2; ++k)
#pragma unroll
                        for (int e = 0; e < 2; ++e)
                            asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                                         : "=f"(f[k][e].x), "=f"(f[k][e].y), "=f"(f[k][e].z), "=f"(f[k][e].w)
                                         : "r"(map_to_rank(at[e], k0 + k))
                                         : "memory");
#pragma unroll
                    for (int k = 0; k < 2; ++k)
#pragma unroll
                        for (int e = 0; e < 2; ++e)
                            v[4 * e] += f[k][e].x, v[4 * e + 1] += f[k][e].y, v[4 * e + 2] += f[k][e].z, v[4 * e + 3] += f[k][e].w;
                }
                orth_split8(v, hi[q], lo[q]);
            }
            cluster_sync(); // the parts have been read everywhere: A may take their place
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int i = threadIdx.x + q * THREADS;
                if (i >= rows_each * 16)
                    break;
                const uint32_t at = a_at + piece((int)rank * rows_each + (i >> 4), i & 15);
                for (unsigned k = 0; k < ranks; ++k) {
                    const uint32_t to = map_to_rank(at, k);
                    asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to), "r"(hi[q].x), "r"(hi[q].y), "r"(hi[q].z),
                                 "r"(hi[q].w)
                                 : "memory");
                    asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to + PART), "r"(lo[q].x), "r"(lo[q].y), "r"(lo[q].z),
                                 "r"(lo[q].w)
                                 : "memory");
                }
            }
            cluster_sync();
        }
        product([&] { // A A
            halves([&](int left, int right, bool clear) {
                for (int b = 0; b < 2; ++b)
                    umma_f16_x4(work, umma_smem_desc(a_at + left + b * BLK, 16, 1024), umma_smem_desc(a_at + right + b * BLK, 16, 1024), IDESC,
                                !clear || b > 0, 2, 2);
            });
        });
        const float kb = ORTH_SB * p.b / ORTH_SA, kc = ORTH_SB * p.c / (ORTH_SA * ORTH_SA);
        load64(WORK, w2);
        tmem_ld_wait();
#pragma unroll
        for (int h = 0; h < 2; ++h) { // a thread's values of B take the place of its values of A
            float(&v)[32] = w2[h];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint8_t *at = smem + A_OFF + piece(row, (half * 2 + h) * 4 + i);
                float f[8];
                orth_join8(*(const uint4 *)at, *(const uint4 *)(at + PART), f);
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    v[8 * i + k] = fmaf(kb, f[k], kc * v[8 * i + k]);
            }
            put_halves(smem + A_OFF, row, half * 2 + h, v);
        }
        const bool last = step == p.steps - 1;
        product([&] { // B X, 128 columns a chunk
            for (int q = 0; q < p.chunks; ++q)
                halves([&](int left, int right, bool clear) {
                    const uint64_t x = umma_smem_desc(x_at + q * 2 * PART + right, BLK, 1024);
                    for (int b = 0; b < 2; ++b)
                        umma_f16_x4(work + q * 128, umma_smem_desc(a_at + left + b * BLK, 16, 1024), x + (uint64_t)(b * 4 * (16 * 128 >> 4)), IDESC_MN,
                                    !clear || b > 0, 2, 16 * 128 >> 4);
                });
        });
        for (int q = 0; q < p.chunks; ++q) {
            if (last && q)
                __syncthreads(); // the staging of the chunk before has been read
            float x2[2][32];
            load64(WORK + q * 128, w2);
            load64(q * 128, x2);
            tmem_ld_wait();
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float(&v)[32] = w2[h];
                const float(&x)[32] = x2[h];
#pragma unroll
                for (int i = 0; i < 32; ++i)
                    v[i] = fmaf(p.a, x[i], v[i] * (1.f / ORTH_SB));
                if (last) {
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        v[i] *= p.out_scale / ORTH_SX;
                    stage32(half * 64 + h * 32, v);
                } else {
                    store32(q * 128 + h * 32, v);
                    put_halves(smem + q * 2 * PART, row, half * 2 + h, v);
                }
            }
            if (!last)
                continue;
            // X -> out, by rows of out
            __syncthreads();
            const int j = j0 + q * 128, part = threadIdx.x >> 4, c8 = (threadIdx.x & 15) * 8;
            __nv_bfloat16 *out = p.out + matrix * p.out_stride;
            for (int k = 0; k < 8; ++k) {
                const int r = (TALL ? j : 0) + part + 16 * k, c = (TALL ? 0 : j) + c8;
                if (r >= p.rows || c >= p.cols)
                    continue;
                alignas(16) __nv_bfloat16 o[8];
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    o[i] = __float2bfloat16_rn(TALL ? stage[staged(c8 + i, (part + 16 * k) & ~3) + (part & 3)]
                                                    : stage[staged(part + 16 * k, c8 + (i & 4)) + (i & 3)]);
                if (p.vec_out && c + 8 <= p.cols) {
                    *(uint4 *)(out + r * p.ld_out + c) = *(uint4 *)o;
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (c + i < p.cols)
                            out[r * p.ld_out + c + i] = o[i];
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (ranks > 1)
        cluster_sync(); // nobody uses another CTA's shared memory any more
    if (warp == 1)
        tmem_dealloc(tmem, 512);
    if (threadIdx.x == 0 && *abort_flag)
        atomicOr(p.status, TS2_STATUS_WAIT_TIMEOUT);
}

template <class T, bool TALL>
int launch(const Ctx &c, const ChipArgs &p, int batch, int ranks)
{
    static std::atomic<unsigned> ready{0}; // a bit a device
    const unsigned bit = 1u << (c.device & 15);
    const auto kern = orth_chip_kernel<T, TALL>;
    if (!(ready.load() & bit)) {
        TS2_CUDA(cudaFuncSetAttribute((const void *)kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM));
        TS2_CUDA(cudaFuncSetAttribute((const void *)kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        ready.fetch_or(bit);
    }
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = ranks;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = batch * ranks;
    cfg.blockDim = THREADS;
    cfg.dynamicSmemBytes = SMEM;
    cfg.stream = c.stream;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    g_launch_count.fetch_add(1, std::memory_order_relaxed);
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, p);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return fail(TS2_ERR_CUDA, "kernel launch failed: %s (%s:%d)", cudaGetErrorString(e), __FILE__, __LINE__);
    }
    return TS2_OK;
}

} // namespace

// CTAs of the cluster that holds a matrix, 0: it does not fit
int orth_chip_ranks(int rows, int cols)
{
    if (std::min(rows, cols) > 128)
        return 0;
    const int64_t chunks = ceil_div(std::max(rows, cols), 128);
    // as few as hold it: more CTAs with fewer chunks each save less than the exchange of A costs (128 x 256 in one 53 us, 100 x 384 in
    // two 76)
    for (int ranks = 1; ranks <= MAX_CLUSTER; ranks *= 2)
        if (chunks <= (int64_t)ranks * MAX_CHUNKS)
            return ranks;
    return 0;
}

int orth_chip(const Ctx &c, int type, const void *g, int64_t ld, int64_t stride, int batch, int rows, int cols, const float coef[3], int steps,
              float out_scale, void *out, int64_t ld_out, int64_t out_stride)
{
    const int ranks = orth_chip_ranks(rows, cols), es = type == TS2_OUT_F32 ? 4 : 2;
    ChipArgs p = {};
    p.g = g, p.ld = ld, p.stride = stride, p.rows = rows, p.cols = cols;
    p.chunks = (int)ceil_div(ceil_div(std::max(rows, cols), 128), ranks);
    p.steps = steps, p.a = coef[0], p.b = coef[1], p.c = coef[2], p.out_scale = out_scale;
    p.out = (__nv_bfloat16 *)out, p.ld_out = ld_out, p.out_stride = out_stride;
    p.vec = ((uintptr_t)g | (uintptr_t)(ld * es) | (uintptr_t)(stride * es)) % 16 == 0;
    p.vec_out = ((uintptr_t)out | (uintptr_t)(ld_out * 2) | (uintptr_t)(out_stride * 2)) % 16 == 0;
    p.status = device_status_word(c.device);
    if (!p.status)
        return fail(TS2_ERR_CUDA, "no device status word");
    const bool tall = rows > cols;
    switch (type) {
    case TS2_OUT_F32: return tall ? launch<float, true>(c, p, batch, ranks) : launch<float, false>(c, p, batch, ranks);
    case TS2_OUT_F16: return tall ? launch<__half, true>(c, p, batch, ranks) : launch<__half, false>(c, p, batch, ranks);
    default: return tall ? launch<__nv_bfloat16, true>(c, p, batch, ranks) : launch<__nv_bfloat16, false>(c, p, batch, ranks);
    }
}

} // namespace ts2
