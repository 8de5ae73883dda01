// A dense layer, z = x W^T + bias, y = act(z) + residual, and its backward pass: dz = dy act'(z), dx = dz W, dw = dz^T x, dbias = sum_t dz.
//
// The three products are one kernel: pairs of CTAs (tcgen05 with cta_group::2) on tiles of 256 x 256 or 256 x 128 of the output, operands by TMA from where they
// lie, either contiguous along K (x, W and dz in the forward product and dx) or along the output's rows or columns (W in dx; dz and x in
// dw).  fp16 or bf16 operands, fp32 sums in tensor memory, two accumulators so that a tile's epilogue runs beside the next tile's products.  The
// epilogue adds the bias, takes the activation and adds the residual in fp32, rounds once, and sends blocks of 32 rows x 128 bytes by TMA.
// Large products are bound by the tensor pipe (under the part's power limit), small ones by the latency of a launch and the first loads.  Outputs of few tiles are
// divided along K: partial tiles in fp32, added in their order by a second launch that runs the epilogue.  dw and dx are one launch: the units that take longer are
// dealt out first, and the others even out what those leave.
// Rows that TMA cannot address (a base or a pitch that is no multiple of 16 bytes) are copied to a pitch that it can.
//
// One by one, 32768 x 2048 x 8192: without activation 742 us (1.48 PFLOP/s), with GELU and z 816; both gradients 1480 to 1515 (1.45 to 1.49 PFLOP/s).  In a row the part's power limit takes
// the clock to 1.3 GHz: 853 to 881 us without activation where a library product of the same operands takes 834.  A tile takes 18.5 k clocks, of which 16.8 k are
// products and the ring waits 2.6 k for copies; five stages are what fits beside two blocks of staging a warp (four stages and three blocks 2 % slower).  Sums over
// a K of 256 or less are bound by the epilogue, 9 k clocks a tile.
#include "elem_types.cuh"
#include "kernels.cuh"
#include "pair_ptx.cuh"
#include <cuda.h>
#include <algorithm>

namespace ts2 {

namespace {

constexpr int PM = 256, BK = 64, BAND = 8,  HALF = 128 * BK * 2; // HALF: a CTA's 128 rows of an operand, one K block, bytes
constexpr int STAGES = 5, EPI_WARPS = 8, THREADS = 64 + 32 * EPI_WARPS;
constexpr int BLOCK = 4096, SLOTS = 2; // an epilogue warp's blocks of 32 rows x 128 bytes on their way out
constexpr int STG_OFF = STAGES * 2 * HALF, BAR_OFF = STG_OFF + EPI_WARPS * SLOTS * BLOCK, SMEM = BAR_OFF + 256 + 1024;
static_assert(SMEM <= 232448, "shared memory budget");
enum { KIND_PARTIAL = 16 }; // beside TS2_OUT_*: fp32 partial tiles

struct LinearArgs {
    int m, n; // rows and columns of the output
    int m_tiles, n_tiles, units, k_blocks, splits, kb_per_split;
    int kind, act;
    bool a_mn; // the first operand is contiguous along the output's rows
    const float *bias;
    const void *res;
    int64_t res_ld;
    void *y, *z;
    int64_t y_ld, z_ld;
    bool y_tma, z_tma, res_vec, bias_vec; // what 16-byte accesses can reach
    bool ends_whole;                      // a row of y and z is a multiple of 16 bytes
    float *part;
};
// The units of up to two products dealt out to pairs: those of the first one after the other to all pairs in turn.  Where they do not come out even, pairs that got
// one less take `extra` units of the second each, about as long as one of the first; the rest goes to all pairs in turn.
struct Deal {
    int units[2], uneven, extra, early; // uneven: pairs with one more of the first; early: units of the second for those with one less
    // sums of columns that the epilogue's warps add up before their first tile is there: [blocks][n] -> out
    const float *sums;
    float *sums_out;
    int sums_n, sums_blocks;
    int32_t *status;
};
// the i-th unit of a pair: false behind the last one
__device__ __forceinline__ bool unit_at(const Deal &d, int pair, int pairs, int i, int &which, int &unit)
{
    which = 0, unit = pair + i * pairs;
    if (unit < d.units[0])
        return true;
    which = 1;
    int j = i - (d.units[0] - pair + pairs - 1) / pairs;
    if (pair >= d.uneven && d.extra) {
        unit = pair - d.uneven + j * (pairs - d.uneven);
        if (j < d.extra)
            return unit < d.early;
        j -= d.extra;
    }
    unit = d.early + pair + j * pairs;
    return unit < d.units[1];
}
struct Unit {
    int row, col, kb0, kb1;
};
// Units go through the output in bands of BAND rows of tiles, column by column, so that the tiles at work at a time share rows and columns of the operands in
// the L2; the K ranges of a tile are neighbours.
template <int PN>
__device__ __forceinline__ Unit unit_of(const LinearArgs &p, int u)
{
    const int tile = u / p.splits, split = u - tile * p.splits, band = tile / (BAND * p.n_tiles), rest = tile - band * BAND * p.n_tiles;
    const int high = min(BAND, p.m_tiles - band * BAND), col = rest / high;
    Unit t;
    t.row = (band * BAND + rest - col * high) * PM;
    t.col = col * PN;
    t.kb0 = split * p.kb_per_split;
    t.kb1 = min(p.k_blocks, t.kb0 + p.kb_per_split);
    return t;
}

// ---- activations ----------------------------------------------------------------------------------------------------------
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }
__device__ __forceinline__ float2 minus_abs(float2 z) { return make_float2(-fabsf(z.x), -fabsf(z.y)); }
// zero below -87.3, where z sigmoid(z) is below 2^-119
__device__ __forceinline__ float2 sigmoid(float2 z) { return rcp(add2(ex2(mul2(z, both(-1.44269504f))), both(1.f))); }
// 1 - Phi(|z|) = e g with e = exp(-z^2 / 2) and g = t P(t), t = 1 / (1 + 0.2575 |z|).  P: a fit of degree 6 for |z| up to 14, by a linear program over 1500 Chebyshev nodes in t that
// bounds the absolute error near zero and the relative one in the tail, whose values a 16-bit result keeps.  In fp32 it is off by 2.2e-7 at most, and of itself by
// 2e-6 at 3, 3e-6 at 6, 1e-5 at 13 (what e's exponent is rounded by); half a step of fp16 is 4.9e-4.  Beyond 13.2 e is 0.
__device__ __forceinline__ void normal_tail(float2 z, float2 minus_z, float2 &g, float2 &e)
{
    const float2 t = rcp(fma2(minus_z, both(-0.257499993f), both(1.f)));
    e = ex2(mul2(mul2(z, z), both(-0.72134752f)));
    float2 q = fma2(t, both(-0.0768212900f), both(0.251779079f));
    q = fma2(t, q, both(-0.136068970f));
    q = fma2(t, q, both(0.185658634f));
    q = fma2(t, q, both(0.0655971989f));
    q = fma2(t, q, both(0.107425064f));
    q = fma2(t, q, both(0.102430306f));
    g = mul2(t, q);
}
template <int ACT>
__device__ __forceinline__ float2 activation(float2 z)
{
    if (ACT == TS2_ACT_RELU)
        return make_float2(z.x < 0.f ? 0.f : z.x, z.y < 0.f ? 0.f : z.y); // a NaN stays one
    if (ACT == TS2_ACT_GELU) { // z Phi(z) = max(z, 0) - |z| (1 - Phi(|z|)), the last term 0 far out
        const float2 m = minus_abs(z);
        float2 g, e;
        normal_tail(z, m, g, e);
        return fma2(make_float2(fmaxf(m.x, -64.f), fmaxf(m.y, -64.f)), mul2(g, e), make_float2(fmaxf(z.x, 0.f), fmaxf(z.y, 0.f)));
    }
    if (ACT == TS2_ACT_SILU)
        return mul2(z, sigmoid(z));
    return z;
}
template <int ACT>
__device__ __forceinline__ float2 activation_slope(float2 z)
{
    if (ACT == TS2_ACT_RELU)
        return make_float2(z.x > 0.f ? 1.f : 0.f, z.y > 0.f ? 1.f : 0.f);
    if (ACT == TS2_ACT_GELU) { // Phi(z) + z phi(z): e (g - |z| / sqrt(2 pi)) at -|z|, where nothing cancels but at the zero itself, and one minus that at |z|
        const float2 m = minus_abs(z);
        float2 g, e;
        normal_tail(z, m, g, e);
        const float2 low = mul2(e, fma2(make_float2(fmaxf(m.x, -64.f), fmaxf(m.y, -64.f)), both(0.39894228f), g));
        return make_float2(z.x < 0.f ? low.x : 1.f - low.x, z.y < 0.f ? low.y : 1.f - low.y);
    }
    if (ACT == TS2_ACT_SILU) {
        const float2 s = sigmoid(z);
        return mul2(s, fma2(z, fma2(s, both(-1.f), both(1.f)), both(1.f)));
    }
    return both(1.f);
}
template <int ACT, int N>
__device__ __forceinline__ void activate_all(float (&v)[N])
{
#pragma unroll
    for (int i = 0; i < N; i += 2) {
        const float2 y = activation<ACT>(make_float2(v[i], i + 1 < N ? v[i + 1 < N ? i + 1 : i] : 0.f));
        v[i] = y.x;
        if (i + 1 < N)
            v[i + 1 < N ? i + 1 : i] = y.y;
    }
}
template <int N>
__device__ __forceinline__ void activate(int act, float (&v)[N])
{
    switch (act) {
    case TS2_ACT_RELU: activate_all<TS2_ACT_RELU>(v); break;
    case TS2_ACT_GELU: activate_all<TS2_ACT_GELU>(v); break;
    case TS2_ACT_SILU: activate_all<TS2_ACT_SILU>(v); break;
    default: break;
    }
}
template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi)
{
    if (BF16) {
        const __nv_bfloat162 r = __floats2bfloat162_rn(lo, hi);
        return *(const uint32_t *)&r;
    }
    const __half2 r = sat_half2(lo, hi);
    return *(const uint32_t *)&r;
}
// without saturation: infinite beyond the type's range
template <bool BF16>
__device__ __forceinline__ uint32_t pack2_open(float lo, float hi)
{
    if (BF16)
        return pack2<true>(lo, hi);
    const __half2 r = __floats2half2_rn(lo, hi);
    return *(const uint32_t *)&r;
}
template <bool BF16>
__device__ __forceinline__ float2 unpack2(uint32_t v)
{
    return BF16 ? __bfloat1622float2(*(const __nv_bfloat162 *)&v) : __half22float2(*(const __half2 *)&v);
}
template <bool BF16>
__device__ __forceinline__ float widen16(uint16_t v)
{
    return unpack2<BF16>(v).x;
}

__device__ __forceinline__ void st_shared(uint32_t at, uint4 v)
{
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ uint4 ld_shared(uint32_t at)
{
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ float ld_shared_f32(uint32_t at)
{
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ uint16_t ld_shared_u16(uint32_t at)
{
    uint16_t v;
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ void tma_add_2d(const void *tmap, uint32_t src, int c0, int c1)
{
    asm volatile("cp.reduce.async.bulk.tensor.2d.global.shared::cta.add.bulk_group [%0, {%2, %3}], [%1];" ::"l"(tmap), "r"(src), "r"(c0), "r"(c1)
                 : "memory");
}

// ---- the product ----------------------------------------------------------------------------------------------------------
// BACK: up to two products, the second operand contiguous along the output's columns instead of along K, the first along its rows where its a_mn says so; else
// one, both operands contiguous along K.  A, B: boxes of 64 along K x 128 (B of PN = 128: 64) rows, or of 64 rows or columns x 64 along K; Y, Z: blocks of 32
// rows x 128 bytes; all 128-byte swizzle
struct LinearMaps {
    CUtensorMap A[2], B[2], Y[2], Z;
};
template <bool BACK, int PN, bool BF16>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS, 1)
    linear_product_kernel(const __grid_constant__ LinearMaps maps, const __grid_constant__ LinearArgs arg0, const __grid_constant__ LinearArgs arg1,
                          const __grid_constant__ Deal deal)
{
    constexpr bool B_MN = BACK;
    constexpr int PART = PN / 2, STAGE = HALF + PART * BK * 2;
    extern __shared__ uint8_t linear_smem[];
    uint8_t *smem = (uint8_t *)(((uintptr_t)linear_smem + 1023) & ~(uintptr_t)1023); // the same offset in both CTAs
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
        prefetch_tmap(&maps.A[0]);
        prefetch_tmap(&maps.B[0]);
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
    const int pair = (int)blockIdx.x >> 1, pairs = (int)gridDim.x >> 1;
    int which = 0, u = 0; // the unit at work
    const auto args = [&]() -> const LinearArgs & { return BACK && which ? arg1 : arg0; };

    if (warp == 0) {
        // TMA producer of the CTA's halves; all copies of a stage complete on the leader's barrier
        if (lane == 0) {
            int stage = 0, issued = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int i = 0; ok && unit_at(deal, pair, pairs, i, which, u); ++i) {
                const Unit un = unit_of<PN>(args(), u);
                const bool a_mn = BACK && args().a_mn;
                const CUtensorMap *tmA = &maps.A[BACK ? which : 0], *tmB = &maps.B[BACK ? which : 0];
                const int am = un.row + (int)rank * 128, bn = un.col + (int)rank * PART;
                for (int kb = un.kb0; kb < un.kb1; ++kb) {
                    if (!mbar_wait(empty0 + 8 * stage, phase ^ 1, abort_flag)) {
                        ok = false;
                        break;
                    }
                    const uint32_t fb = map_to_leader(full0 + 8 * stage);
                    if (rank == 0)
                        mbar_arrive_expect_tx(full0 + 8 * stage, 2 * STAGE);
                    const uint32_t sa = smem_u32(smem + stage * STAGE), sb = sa + HALF;
                    if (a_mn) {
                        tma_load_2d_pair(sa, tmA, fb, am, kb * BK);
                        tma_load_2d_pair(sa + BK * 128, tmA, fb, am + 64, kb * BK);
                    } else {
                        tma_load_2d_pair(sa, tmA, fb, kb * BK, am);
                    }
                    if constexpr (B_MN) {
#pragma unroll
                        for (int j = 0; j < PART / 64; ++j)
                            tma_load_2d_pair(sb + j * BK * 128, tmB, fb, bn + 64 * j, kb * BK);
                    } else {
                        tma_load_2d_pair(sb, tmB, fb, kb * BK, bn);
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
            constexpr uint32_t idesc0 = (1u << 4) | (BF16 ? (1u << 7) | (1u << 10) : 0u) | ((B_MN ? 1u : 0u) << 16) | ((uint32_t)(PN >> 3) << 17) |
                                        ((uint32_t)(PM >> 4) << 24);
            int stage = 0, acc = 0;
            uint32_t phase = 0, acc_phase = 0;
            bool ok = true;
            for (int i = 0; ok && unit_at(deal, pair, pairs, i, which, u); ++i) {
                const Unit un = unit_of<PN>(args(), u);
                const bool a_mn = BACK && args().a_mn;
                const uint32_t idesc = idesc0 | (a_mn ? 1u << 15 : 0u), a_step = a_mn ? (16 * 128) >> 4 : 2; // 16 of K, in 16-byte units
                if (!mbar_wait(tempty0 + 8 * acc, acc_phase ^ 1, abort_flag))
                    break;
                tc_fence_after();
                const uint32_t tmem_d = tmem_base + acc * PN;
                for (int kb = un.kb0; kb < un.kb1; ++kb) {
                    if (!mbar_wait(full0 + 8 * stage, phase, abort_flag)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t a = smem_u32(smem + stage * STAGE), b = a + HALF;
                    const uint64_t adesc = umma_smem_desc(a, a_mn ? BK * 128 : 16, 1024), bdesc = umma_smem_desc(b, B_MN ? BK * 128 : 16, 1024);
                    constexpr uint32_t b_step = B_MN ? (16 * 128) >> 4 : 2;
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        umma_pair<1>(tmem_d, adesc + (uint64_t)(k * a_step), bdesc + (uint64_t)(k * b_step), idesc, kb > un.kb0 || k > 0 ? 1u : 0u);
                    commit_both(empty0 + 8 * stage);
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
        // epilogue: a warp takes 32 rows x PART columns, 32 columns at a time, thread = row
        const int quarter = warp & 3, ew = warp - 2, part = ew >> 2;
        const uint32_t slots = smem_u32(smem) + STG_OFF + ew * SLOTS * BLOCK;
        int slot = 0, acc = 0;
        uint32_t acc_phase = 0;
        // the next block; the store that last used it, two blocks before, has read it (a block for z is taken while y's has not left)
        const auto take = [&](bool second) {
            const uint32_t b = slots + slot * BLOCK;
            slot = slot == SLOTS - 1 ? 0 : slot + 1;
            if (lane == 0) {
                if (second)
                    bulk_wait_read<SLOTS - 2>();
                else
                    bulk_wait_read<SLOTS - 1>();
            }
            __syncwarp();
            return b;
        };
        const auto piece = [&](uint32_t block, int row, int q) { return block + row * 128 + ((q ^ (row & 7)) << 4); };
        if (BACK && deal.sums_out) // no tile is there for a while
            for (int at = ((int)blockIdx.x * EPI_WARPS + ew) * 32 + lane; at < deal.sums_n; at += (int)gridDim.x * EPI_WARPS * 32) {
                float sum = 0.f;
#pragma unroll 4
                for (int i = 0; i < deal.sums_blocks; ++i)
                    sum += deal.sums[(int64_t)i * deal.sums_n + at];
                deal.sums_out[at] = sum;
            }
        for (int i = 0; unit_at(deal, pair, pairs, i, which, u); ++i) {
            const LinearArgs &p = args();
            const CUtensorMap *tmY = &maps.Y[BACK ? which : 0];
            const bool halves = p.kind == TS2_OUT_F16 || p.kind == TS2_OUT_BF16;
            const Unit un = unit_of<PN>(p, u);
            const uint32_t taddr = tmem_base + ((uint32_t)(quarter * 32) << 16) + acc * PN + part * PART;
            const int row0 = un.row + (int)rank * 128 + quarter * 32, col0 = un.col + part * PART;
            if (p.res && row0 + lane < p.m) { // the residual into the L2 while the tile is multiplied
                const uint16_t *from = (const uint16_t *)p.res + (row0 + lane) * p.res_ld;
#pragma unroll
                for (int k = 0; k < PART; k += 64)
                    if (col0 + k < p.n)
                        asm volatile("prefetch.global.L2 [%0];" ::"l"(from + col0 + k));
            }
            if (p.bias && col0 + 4 * lane < p.n) { // and the bias into the L1
                float ignored;
                asm volatile("ld.global.ca.f32 %0, [%1];" : "=f"(ignored) : "l"(p.bias + col0 + 4 * lane));
            }
            uint4 ahead[2][4]; // of the next two times 32 columns of the residual: 4 lanes a row, 8 rows at a time
            const auto fetch = [&](int col, uint4 (&rows)[4]) {
                if (!p.res || col >= p.n)
                    return;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int row = row0 + 8 * i + (lane >> 2), at = col + (lane & 3) * 8;
                    const uint16_t *from = (const uint16_t *)p.res + row * p.res_ld + at;
                    rows[i] = make_uint4(0, 0, 0, 0);
                    if (row >= p.m)
                        continue;
                    if (p.res_vec && at + 8 <= p.n) {
                        rows[i] = *(const uint4 *)from;
                    } else {
                        uint32_t w[4] = {};
#pragma unroll
                        for (int k = 0; k < 8; ++k)
                            w[k >> 1] |= at + k < p.n ? (uint32_t)from[k] << (16 * (k & 1)) : 0u;
                        rows[i] = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                }
            };
            fetch(col0, ahead[0]);
            fetch(col0 + 32, ahead[1]);
            if (!__all_sync(0xffffffffu, mbar_wait(tfull0 + 8 * acc, acc_phase, abort_flag)))
                break;
            tc_fence_after();
            uint32_t yb = 0, zb = 0;
#pragma unroll 1
            for (int c2 = 0; c2 < PART / 32; c2 += 2)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int c = c2 + half, col = col0 + c * 32; // 16-bit results fill half of a block's rows
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
                if (row0 >= p.m || col0 >= p.n)
                    continue;
                float v[32];
#pragma unroll
                for (int i = 0; i < 32; ++i)
                    v[i] = __uint_as_float(r[i]);
                if (!halves) {
                    yb = take(false);
#pragma unroll
                    for (int q = 0; q < 8; ++q)
                        st_shared(piece(yb, lane, q), make_uint4(r[4 * q], r[4 * q + 1], r[4 * q + 2], r[4 * q + 3]));
                } else {
                    if (!half) {
                        yb = take(false);
                        if (p.z)
                            zb = take(true);
                    }
                    if (p.res) {
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            st_shared(piece(yb, 8 * i + (lane >> 2), 4 * half + (lane & 3)), ahead[half][i]);
                        __syncwarp();
                        if (c + 2 < PART / 32)
                            fetch(col + 64, ahead[half]);
                    }
                    if (p.bias) {
                        if (p.bias_vec && col + 32 <= p.n) {
#pragma unroll
                            for (int i = 0; i < 8; ++i) {
                                const float4 b = *(const float4 *)(p.bias + col + 4 * i);
                                v[4 * i] += b.x, v[4 * i + 1] += b.y, v[4 * i + 2] += b.z, v[4 * i + 3] += b.w;
                            }
                        } else {
#pragma unroll
                            for (int i = 0; i < 32; ++i)
                                if (col + i < p.n)
                                    v[i] += p.bias[col + i];
                        }
                    }
                    if (p.z) {
#pragma unroll
                        for (int q = 0; q < 4; ++q)
                            st_shared(piece(zb, lane, 4 * half + q),
                                      make_uint4(pack2<BF16>(v[8 * q], v[8 * q + 1]), pack2<BF16>(v[8 * q + 2], v[8 * q + 3]),
                                                 pack2<BF16>(v[8 * q + 4], v[8 * q + 5]), pack2<BF16>(v[8 * q + 6], v[8 * q + 7])));
                    }
                    activate(p.act, v);
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const uint32_t at = piece(yb, lane, 4 * half + q);
                        if (p.res) {
                            const uint4 raw = ld_shared(at);
                            const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                const float2 f = unpack2<BF16>(w[k]);
                                v[8 * q + 2 * k] += f.x, v[8 * q + 2 * k + 1] += f.y;
                            }
                        }
                        st_shared(at, make_uint4(pack2<BF16>(v[8 * q], v[8 * q + 1]), pack2<BF16>(v[8 * q + 2], v[8 * q + 3]),
                                                 pack2<BF16>(v[8 * q + 4], v[8 * q + 5]), pack2<BF16>(v[8 * q + 6], v[8 * q + 7])));
                    }
                    if (!half)
                        continue;
                }
                const int left = halves ? col - 32 : col; // of the block
                // a store by TMA is cut off at the last 16 bytes that hold some of the row, not at its last element
                const bool whole = p.ends_whole || left + (halves ? 64 : 32) <= p.n, y_tma = p.y_tma && whole, z_tma = p.z_tma && whole;
                fence_proxy_async();
                __syncwarp();
                if (y_tma && lane == 0 && left < p.n) {
                    if (p.kind == KIND_PARTIAL)
                        tma_store_2d(tmY, yb, left - un.col, u * PM + row0 - un.row);
                    else if (p.kind == TS2_OUT_F32_ADD)
                        tma_add_2d(tmY, yb, left, row0);
                    else
                        tma_store_2d(tmY, yb, left, row0);
                }
                if (lane == 0)
                    bulk_commit(); // a group for every block taken, with or without a store
                if (halves && p.z) {
                    if (z_tma && lane == 0 && left < p.n)
                        tma_store_2d(&maps.Z, zb, left, row0);
                    if (lane == 0)
                        bulk_commit();
                }
                // Rows that TMA cannot address: 8 lanes a row, each the 16 bytes behind the first 16-byte boundary that are its, put together from two
                // neighbouring pieces; what lies before that boundary and behind the last one element by element.
                const auto by_rows = [&](uint32_t block, uint16_t *base, int64_t ld) {
                    const int there = min(64, p.n - left), q = lane & 7; // there: elements of a row, not always above 0
#pragma unroll 2
                    for (int i = 0; i < 8; ++i) {
                        const int r = i * 4 + (lane >> 3);
                        uint16_t *to = base + (row0 + r) * ld + left;
                        const int head = -((int)(uintptr_t)to >> 1) & 7, whole = max(0, there - head) >> 3, behind = head + 8 * whole + q;
                        if (row0 + r >= p.m)
                            continue;
                        const auto element = [&](int e) { return ld_shared_u16(piece(block, r, e >> 3) + (e & 7) * 2); };
                        if (q < whole) {
                            const uint4 x = ld_shared(piece(block, r, q)), y = head ? ld_shared(piece(block, r, q + 1)) : x;
                            uint32_t w[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
                            for (int k = 0; k < 6; ++k)
                                w[k] = head & 4 ? w[k + 2] : w[k];
#pragma unroll
                            for (int k = 0; k < 5; ++k)
                                w[k] = head & 2 ? w[k + 1] : w[k];
#pragma unroll
                            for (int k = 0; k < 4; ++k)
                                w[k] = __funnelshift_r(w[k], w[k + 1], head & 1 ? 16 : 0);
                            *(uint4 *)(to + head + 8 * q) = make_uint4(w[0], w[1], w[2], w[3]);
                        }
                        if (q < head && q < there)
                            to[q] = element(q);
                        if (behind < there)
                            to[behind] = element(behind);
                    }
                };
                if (!y_tma) {
                    if (halves) {
                        by_rows(yb, (uint16_t *)p.y, p.y_ld);
                    } else {
                        for (int i = 0; i < 32 && row0 + i < p.m; ++i)
                            if (left + lane < p.n) {
                                float *to = (float *)p.y + (row0 + i) * p.y_ld + left + lane;
                                const float now = ld_shared_f32(piece(yb, i, lane >> 2) + (lane & 3) * 4);
                                *to = p.kind == TS2_OUT_F32_ADD ? *to + now : now;
                            }
                    }
                }
                if (halves && p.z && !z_tma)
                    by_rows(zb, (uint16_t *)p.z, p.z_ld);
                __syncwarp();
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
        atomicOr(deal.status, TS2_STATUS_WAIT_TIMEOUT);
}

// The K ranges of a product added in their order, and its epilogue: 4 columns a thread
template <int PN, bool BF16>
__global__ void __launch_bounds__(256) linear_join_kernel(const LinearArgs p, int kind)
{
    grid_dep_wait();
    const int quads = (p.n + 3) / 4;
    const int64_t total = (int64_t)p.m * quads;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int row = (int)(i / quads), col = (int)(i - (int64_t)row * quads) * 4;
        const int band = row / (BAND * PM), high = min(BAND, p.m_tiles - band * BAND);
        const int tile = band * BAND * p.n_tiles + col / PN * high + row / PM - band * BAND;
        const float *from = p.part + ((int64_t)tile * p.splits * PM + row % PM) * PN + col % PN;
        float v[4] = {};
        for (int s = 0; s < p.splits; ++s) {
            const float4 x = *(const float4 *)(from + (int64_t)s * PM * PN);
            v[0] += x.x, v[1] += x.y, v[2] += x.z, v[3] += x.w;
        }
        if (kind == TS2_OUT_F32 || kind == TS2_OUT_F32_ADD) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (col + k < p.n) {
                    float *to = (float *)p.y + row * p.y_ld + col + k;
                    *to = kind == TS2_OUT_F32_ADD ? *to + v[k] : v[k];
                }
            continue;
        }
        const auto store = [&](void *base, int64_t ld, bool vec) {
            const uint32_t a = pack2<BF16>(v[0], v[1]), b = pack2<BF16>(v[2], v[3]);
            uint16_t *to = (uint16_t *)base + row * ld + col;
            if (vec && col + 4 <= p.n) {
                *(uint2 *)to = make_uint2(a, b);
            } else {
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (col + k < p.n)
                        to[k] = (uint16_t)((k & 2 ? b : a) >> (16 * (k & 1)));
            }
        };
        if (p.bias) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (col + k < p.n)
                    v[k] += p.bias[col + k];
        }
        if (p.z)
            store(p.z, p.z_ld, p.z_tma);
        activate(p.act, v);
        if (p.res) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (col + k < p.n)
                    v[k] += widen16<BF16>(((const uint16_t *)p.res)[row * p.res_ld + col + k]);
        }
        store(p.y, p.y_ld, p.y_tma);
    }
}

// ---- a few tokens --------------------------------------------------------------------------------------------------------
// Bound by reading W once.  A CTA takes 16 rows of W; its 8 warps, and those of the up to 8 CTAs of a cluster where W has few rows, divide K.  A lane reads 8
// neighbours of two rows of W and of the tokens' x; four lanes' pieces are 32 of K, and as both operands come in the same order they are the fragments of two
// m16n8k16 products as they lie in the registers.  Sums are added in the order of the warps and CTAs.
constexpr int FEW_WARPS = 8;
// Blocks of 32 of K on their way at a time: more of them, or more warps an SM with fewer registers.  us for 2048 x 8192 with 2 and 4: 1 token 8.5, 9.4; 16 tokens
// 12.9, 12.0; 32 tokens 16.3, 21.2.
constexpr int few_batch(int nt) { return nt == 2 ? 4 : 2; }
struct FewArgs {
    int T, n, m; // tokens, columns of x and W, rows of W
    const uint16_t *x, *w, *res;
    int64_t x_ld, w_ld, res_ld, y_ld, z_ld;
    const float *bias;
    uint16_t *y, *z;
    int act, ranks;
};
template <bool BF16>
__device__ __forceinline__ void mma16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    if (BF16)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// 8 neighbours of a row from column k on, zeros behind the last one and where the row is not there
template <bool VEC>
__device__ __forceinline__ uint4 eight_of(const uint16_t *row, int k, int n, bool there)
{
    if (VEC && there && k + 8 <= n)
        return *(const uint4 *)(row + k);
    uint32_t v[4] = {};
    if (there)
#pragma unroll
        for (int i = 0; i < 8; ++i)
            v[i >> 1] |= k + i < n ? (uint32_t)row[k + i] << (16 * (i & 1)) : 0u;
    return make_uint4(v[0], v[1], v[2], v[3]);
}
// NT: tokens in eights
template <int NT, bool BF16, bool VEC>
__global__ void __launch_bounds__(32 * FEW_WARPS, NT == 1 ? 4 : 1) linear_few_kernel(const FewArgs p)
{
    constexpr int BATCH = few_batch(NT);
    __shared__ float part[FEW_WARPS][8 * NT][17], sums[8 * NT][17];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
    const uint32_t rank = p.ranks > 1 ? cluster_rank() : 0;
    const int row0 = (int)(blockIdx.x / p.ranks) * 16, blocks = (p.n + 31) / 32, workers = p.ranks * FEW_WARPS, mine = (int)rank * FEW_WARPS + warp;
    const int kb0 = (int)((int64_t)blocks * mine / workers), kb1 = (int)((int64_t)blocks * (mine + 1) / workers);
    grid_dep_wait();
    const uint16_t *wa = p.w + (int64_t)(row0 + g) * p.w_ld, *wb = wa + 8 * p.w_ld;
    const bool a_there = row0 + g < p.m, b_there = row0 + g + 8 < p.m;
    float c[NT][4] = {};
#pragma unroll 1
    for (int kb = kb0; kb < kb1; kb += BATCH) {
        uint4 a[BATCH], b[BATCH], x[BATCH][NT];
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
            const int k = (kb + i) * 32 + q * 8;
            const bool in = kb + i < kb1;
            a[i] = eight_of<VEC>(wa, k, p.n, in && a_there);
            b[i] = eight_of<VEC>(wb, k, p.n, in && b_there);
#pragma unroll
            for (int t = 0; t < NT; ++t)
                x[i][t] = eight_of<VEC>(p.x + (int64_t)(8 * t + g) * p.x_ld, k, p.n, in && 8 * t + g < p.T);
        }
#pragma unroll
        for (int i = 0; i < BATCH; ++i)
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                mma16<BF16>(c[t], a[i].x, b[i].x, a[i].y, b[i].y, x[i][t].x, x[i][t].y);
                mma16<BF16>(c[t], a[i].z, b[i].z, a[i].w, b[i].w, x[i][t].z, x[i][t].w);
            }
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        part[warp][8 * t + 2 * q][g] = c[t][0], part[warp][8 * t + 2 * q + 1][g] = c[t][1];
        part[warp][8 * t + 2 * q][g + 8] = c[t][2], part[warp][8 * t + 2 * q + 1][g + 8] = c[t][3];
    }
    __syncthreads();
    const int row = threadIdx.x & 15;
    for (int t = threadIdx.x >> 4; t < 8 * NT; t += 2 * FEW_WARPS) {
        float s = 0.f;
#pragma unroll
        for (int k = 0; k < FEW_WARPS; ++k)
            s += part[k][t][row];
        sums[t][row] = s;
    }
    if (p.ranks > 1)
        cluster_sync(); // every CTA's sums are there
    if (rank == 0) {
        for (int t = threadIdx.x >> 4; t < p.T; t += 2 * FEW_WARPS) {
            float v[1] = {sums[t][row]}; // this thread's own, the other CTAs' by their order
            for (int k = 1; k < p.ranks; ++k) {
                float other;
                asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(other) : "r"(map_to_rank(smem_u32(&sums[t][row]), k)) : "memory");
                v[0] += other;
            }
            const int at = row0 + row;
            if (at >= p.m)
                continue;
            if (p.bias)
                v[0] += p.bias[at];
            if (p.z)
                p.z[t * p.z_ld + at] = (uint16_t)pack2<BF16>(v[0], 0.f);
            activate(p.act, v);
            if (p.res)
                v[0] += widen16<BF16>(p.res[t * p.res_ld + at]);
            p.y[t * p.y_ld + at] = (uint16_t)pack2<BF16>(v[0], 0.f);
        }
    }
    if (p.ranks > 1)
        cluster_sync(); // nobody reads this CTA's sums any more
}

// ---- dz and its column sums; rows at another pitch --------------------------------------------------------------------------
// rows of 16-bit elements to a pitch that TMA can address
struct PitchJob {
    const uint16_t *from;
    uint16_t *to;
    int64_t from_ld, to_ld, rows;
    int cols;
};
struct PitchJobs {
    PitchJob job[2];
    int64_t items[2]; // pieces of rows
    int n;
};
// A block of the first `layers` takes 128 columns and rows b, b + layers, ... of 16: dz = dy act'(z) rounded to 16 bits, without saturation (dz null: not wanted), and the sums of
// the unrounded dz over its rows (sums null: not wanted).  Bound by reading dy and z and writing dz (32768 x 8192 with GELU 312 us, 5.2 TB/s).  Where 16-byte accesses are not possible (VEC false) a lane has pairs of
// columns that are 16 pairs apart, so that neighbouring lanes read neighbouring 4-byte words.  The layers behind copy rows.
template <int ACT, bool BF16, bool VEC>
__global__ void __launch_bounds__(256) linear_dz_kernel(const uint16_t *__restrict__ dy, int64_t dy_ld, const uint16_t *__restrict__ z, int64_t z_ld,
                                                        int64_t T, int n, int layers, uint16_t *dz, int64_t dz_ld, float *sums, const PitchJobs jobs)
{
    grid_dep_wait();
    if ((int)blockIdx.y >= layers) {
        const int64_t worker = ((int64_t)(blockIdx.y - layers) * gridDim.x + blockIdx.x) * 8 + (threadIdx.x >> 5), workers = (int64_t)(gridDim.y - layers) * gridDim.x * 8;
        for (int64_t all = worker; all < jobs.items[0] + jobs.items[1]; all += workers) {
            const bool second = all >= jobs.items[0];
            const PitchJob &j = second ? jobs.job[1] : jobs.job[0];
            const int64_t item = all - (second ? jobs.items[0] : 0);
            const int words = (j.cols + 1) / 2, pieces = (words + 255) / 256; // 256 words of a row at a time
            const int64_t r = pieces == 1 ? item : item / pieces;
            const int begin = (int)(item - r * pieces) * 256 + (threadIdx.x & 31);
            // 4-byte words that hold an element of the row; where it begins with the upper half of one, halves of neighbours
            const uint16_t *row = j.from + r * j.from_ld;
            const bool odd = (uintptr_t)row & 2;
            const uint32_t *from = (const uint32_t *)(row - odd);
            uint32_t *to = (uint32_t *)(j.to + r * j.to_ld); // 16-byte aligned, with room for a multiple of 8
            const int last = (j.cols + odd - 1) / 2;
            uint32_t w[9]; // all loads before the first store; w[8]: the word behind the piece, in lane 0
#pragma unroll
            for (int k = 0; k < 8; ++k)
                w[k] = begin + k * 32 < words ? from[begin + k * 32] : 0u;
            if (odd) { // the word behind the row's last one may be needed, and no other
                const int lane = threadIdx.x & 31;
                w[8] = lane == 0 && begin + 256 <= last ? from[begin + 256] : 0u;
                const uint32_t end = words <= last && words > begin - lane && words <= begin - lane + 256 ? from[words] : 0u;
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const uint32_t beside = __shfl_down_sync(0xffffffffu, w[k], 1), first = __shfl_sync(0xffffffffu, w[k + 1], 0);
                    uint32_t next = lane == 31 ? first : beside;
                    if (begin + k * 32 + 1 == words)
                        next = end;
                    w[k] = w[k] >> 16 | next << 16;
                }
            }
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (begin + k * 32 < words)
                    to[begin + k * 32] = w[k];
        }
        return;
    }
    __shared__ float part[16][132];
    const int sub = threadIdx.x & 15, line = threadIdx.x >> 4, col0 = blockIdx.x * 128;
    const auto column = [&](int k) { return col0 + (VEC ? sub * 8 + k : 2 * (sub + 16 * (k >> 1)) + (k & 1)); };
    const bool full = col0 + 128 <= n;
    float2 acc[4] = {};
    const auto read = [&](const uint16_t *row, uint32_t (&v)[4]) {
        if (VEC && column(0) + 8 <= n) {
            const uint4 q = *(const uint4 *)(row + column(0));
            v[0] = q.x, v[1] = q.y, v[2] = q.z, v[3] = q.w;
        } else if (!VEC && full) { // words that hold an element of the row; halves of neighbours where it begins with the upper half of one
            const bool odd = (uintptr_t)row & 2;
            const uint32_t *words = (const uint32_t *)(row - odd) + col0 / 2 + sub;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                v[k] = words[16 * k];
                if (odd)
                    v[k] = v[k] >> 16 | words[16 * k + 1] << 16;
            }
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k)
                v[k] = (column(2 * k) < n ? (uint32_t)row[column(2 * k)] : 0u) | (column(2 * k + 1) < n ? (uint32_t)row[column(2 * k + 1)] << 16 : 0u);
        }
    };
#pragma unroll 2
    for (int64_t t = (int64_t)blockIdx.y * 16 + line; t < T; t += (int64_t)layers * 16) {
        uint32_t a[4], b[4], o[4];
        read(dy + t * dy_ld, a);
        if (ACT != TS2_ACT_NONE)
            read(z + t * z_ld, b);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            float2 d = unpack2<BF16>(a[k]);
            if (ACT != TS2_ACT_NONE)
                d = mul2(d, activation_slope<ACT>(unpack2<BF16>(b[k])));
            acc[k] = add2(acc[k], d);
            o[k] = pack2_open<BF16>(d.x, d.y); // dw shows a gradient that left the range
        }
        if (!dz)
            continue;
        uint16_t *to = dz + t * dz_ld;
        if (VEC) {
            if (column(0) < n) // the pitch is a multiple of 8
                *(uint4 *)(to + column(0)) = make_uint4(o[0], o[1], o[2], o[3]);
        } else if (full) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
                *(uint32_t *)(to + column(2 * k)) = o[k];
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (column(k) < n)
                    to[column(k)] = (uint16_t)(o[k >> 1] >> (16 * (k & 1)));
        }
    }
    if (!sums)
        return;
#pragma unroll
    for (int k = 0; k < 8; ++k)
        part[line][column(k) - col0] = k & 1 ? acc[k >> 1].y : acc[k >> 1].x;
    __syncthreads();
    if (threadIdx.x < 128 && col0 + (int)threadIdx.x < n) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i)
            s += part[i][threadIdx.x];
        sums[(int64_t)blockIdx.y * n + col0 + threadIdx.x] = s;
    }
}
__global__ void __launch_bounds__(128) linear_sum_kernel(const float *__restrict__ sums, int n, int blocks, float *out)
{
    grid_dep_wait();
    const int col = blockIdx.x * 128 + threadIdx.x;
    if (col >= n)
        return;
    float s = 0.f;
#pragma unroll 4
    for (int b = 0; b < blocks; ++b)
        s += sums[(int64_t)b * n + col];
    out[col] = s;
}

// ---- host ------------------------------------------------------------------------------------------------------------------
typedef CUresult (*EncodeTiledFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                                  const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
// [rows][cols] of 2- or 4-byte elements; boxes of 128 bytes x `high` rows, 128-byte swizzle
int linear_map(CUtensorMap *tm, const void *base, int size, int64_t cols, int64_t rows, int64_t ld, int high)
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
    const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)(ld * size)};
    const cuuint32_t box[2] = {(cuuint32_t)(128 / size), (cuuint32_t)high}, estr[2] = {1, 1};
    const CUresult r = encode(tm, size == 2 ? CU_TENSOR_MAP_DATA_TYPE_UINT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 2, const_cast<void *>(base), dims, strides,
                              box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? TS2_OK : fail(TS2_ERR_CUDA, "cuTensorMapEncodeTiled failed with code %d", (int)r);
}
bool tma_ok(const void *base, int64_t ld, int size) { return (uintptr_t)base % 16 == 0 && ld * size % 16 == 0; }

// an operand: rows of 16-bit elements, where they lie or as a job copies them to a pitch that TMA can address
struct Operand {
    const void *p = nullptr;
    int64_t rows = 0, ld = 0;
    int cols = 0;
    Scratch copy;
    int rc = TS2_OK;
    Operand(const Ctx &c, const void *from, int64_t from_ld, int64_t rows_, int cols_, PitchJobs &jobs)
        : p(from), rows(rows_), ld(from_ld), cols(cols_), copy(c, !from || tma_ok(from, from_ld, 2) ? 0 : (size_t)rows_ * ceil_div(cols_, 8) * 16), rc(copy.rc)
    {
        if (!copy.p)
            return;
        p = copy.p, ld = ceil_div(cols, 8) * 8;
        jobs.items[jobs.n] = rows * ceil_div((cols + 1) / 2, 256);
        jobs.job[jobs.n++] = {(const uint16_t *)from, (uint16_t *)copy.p, from_ld, ld, rows, cols};
    }
};
template <int ACT, bool BF16>
int prepare(const Ctx &c, const void *dy, int64_t dy_ld, const void *z, int64_t z_ld, int64_t T, int n, int layers, void *dz, int64_t dz_ld, float *sums,
            const PitchJobs &jobs)
{
    const bool vec = tma_ok(dy, dy_ld, 2) && (ACT == TS2_ACT_NONE || tma_ok(z, z_ld, 2));
    const int strips = layers ? (int)ceil_div(n, 128) : 4 * sm_count(c.device);
    const dim3 grid(strips, layers + (int)ceil_div(std::min<int64_t>(ceil_div(jobs.items[0] + jobs.items[1], 8), 8 * sm_count(c.device)), strips));
    if (vec)
        TS2_LAUNCH((linear_dz_kernel<ACT, BF16, true>), grid, 256, 0, c.stream, (const uint16_t *)dy, dy_ld, (const uint16_t *)z, z_ld, T, n, layers,
                   (uint16_t *)dz, dz_ld, sums, jobs);
    else
        TS2_LAUNCH((linear_dz_kernel<ACT, BF16, false>), grid, 256, 0, c.stream, (const uint16_t *)dy, dy_ld, (const uint16_t *)z, z_ld, T, n, layers,
                   (uint16_t *)dz, dz_ld, sums, jobs);
    return TS2_OK;
}

// a product: operands and what its epilogue does; m = 0: none
struct Product {
    const Operand *a = nullptr, *b = nullptr;
    int64_t K = 0;
    LinearArgs p = {};
};
// How products are divided: tiles of 256 x PN, and the first one's K into ranges.  Times in K blocks of a whole tile, 0.33 us with its copies: a unit takes its
// blocks and 4 more for its start and its epilogue, tiles of half the width 0.75 of that (32768 x 2048 x 8192 742 us, with those 1100); joining takes a launch, 10, and 0.1 for every range of a tile.
struct Plan {
    int pn, splits;
};
// Bytes of partial tiles.  Large outputs gain less from K ranges than one part in 40, and their partials would have to be mapped in each call: dw of 18048 x 24224 over
// 222160 tokens 217 ms without ranges, 219 with two and 3.5 GB of partials.
constexpr double MOST_PARTIALS = SCRATCH_KEEP_BYTES / 2;
Plan plan_of(int pairs, const Product *products, int n)
{
    Plan plan = {256, 1};
    double best = 1e30;
    for (const int pn : {256, 128}) {
        const double width = pn == 256 ? 1. : 0.75;
        const auto tiles = [&](const Product &q) { return (double)(ceil_div(q.p.m, PM) * ceil_div(q.p.n, pn)); };
        const auto blocks = [&](const Product &q) { return ceil_div(q.K, BK); };
        const double rest = n > 1 ? tiles(products[1]) * (blocks(products[1]) + 4.) : 0.;
        for (int s = 1; s <= 64 && s <= blocks(products[0]); ++s) {
            const int64_t per = ceil_div(blocks(products[0]), s);
            if (ceil_div(blocks(products[0]), per) != s)
                continue;
            const double units = tiles(products[0]) * s, unit = per + 4.;
            if (s > 1 && units * PM * pn * 4 > MOST_PARTIALS)
                continue;
            // alone in whole rounds; with a second product that evens them out, by the sum
            double cost = n > 1 && rest > 0. ? std::max((units * unit + rest) / pairs, unit) + 0.5 * (blocks(products[1]) + 4.)
                                             : (double)ceil_div((int64_t)units, pairs) * unit;
            cost = width * cost + (s > 1 ? 10. + 0.1 * width * units : 0.);
            if (cost < best)
                best = cost, plan = {pn, s};
        }
    }
    return plan;
}

template <bool BACK, int PN, bool BF16>
int run_products(const Ctx &c, const Product *products, int n, int splits, Deal deal)
{
    static std::atomic<unsigned> ready{0}; // a bit a device: it has been told how much shared memory the kernel takes
    const unsigned bit = 1u << (c.device & 15);
    if (!(ready.load() & bit)) {
        TS2_CUDA(cudaFuncSetAttribute((const void *)linear_product_kernel<BACK, PN, BF16>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM));
        ready.fetch_or(bit);
    }
    const int pairs = sm_count(c.device) / 2;
    deal.status = device_status_word(c.device);
    if (!deal.status)
        return fail(TS2_ERR_CUDA, "no device status word");
    LinearMaps maps = {};
    LinearArgs args[2] = {}, join = {};
    Scratch part(c, splits > 1 ? (size_t)ceil_div(products[0].p.m, PM) * ceil_div(products[0].p.n, PN) * splits * PM * PN * 4 : 0);
    int rc = part.rc;
    for (int i = 0; i < n && rc == TS2_OK; ++i) {
        const Product &q = products[i];
        LinearArgs &p = args[i];
        p = q.p;
        p.m_tiles = (int)ceil_div(p.m, PM), p.n_tiles = (int)ceil_div(p.n, PN), p.k_blocks = (int)ceil_div(q.K, BK);
        p.splits = i == 0 ? splits : 1, p.kb_per_split = (int)ceil_div(p.k_blocks, p.splits), p.units = p.m_tiles * p.n_tiles * p.splits;
        deal.units[i] = p.units;
        const int size = p.kind == TS2_OUT_F32 || p.kind == TS2_OUT_F32_ADD ? 4 : 2;
        p.y_tma = tma_ok(p.y, p.y_ld, size), p.z_tma = tma_ok(p.z, p.z_ld, 2), p.res_vec = tma_ok(p.res, p.res_ld, 2), p.bias_vec = (uintptr_t)p.bias % 16 == 0;
        p.ends_whole = (int64_t)p.n * size % 16 == 0;
        rc = linear_map(&maps.A[i], q.a->p, 2, q.a->cols, q.a->rows, q.a->ld, p.a_mn ? BK : 128);
        if (rc == TS2_OK)
            rc = linear_map(&maps.B[i], q.b->p, 2, q.b->cols, q.b->rows, q.b->ld, BACK ? BK : PN / 2);
        if (p.splits > 1) {
            p.part = (float *)part.p, join = p;
            p.kind = KIND_PARTIAL, p.y_tma = p.ends_whole = true, p.res = nullptr, p.z = nullptr, p.bias = nullptr;
            if (rc == TS2_OK)
                rc = linear_map(&maps.Y[i], part.p, 4, PN, (int64_t)p.units * PM, PN, 32);
        } else {
            if (rc == TS2_OK && p.y_tma)
                rc = linear_map(&maps.Y[i], p.y, size, p.n, p.m, p.y_ld, 32);
            if (rc == TS2_OK && p.z && p.z_tma)
                rc = linear_map(&maps.Z, p.z, 2, p.n, p.m, p.z_ld, 32);
        }
    }
    if (rc != TS2_OK)
        return rc;
    const int used = std::min(pairs, deal.units[0] + deal.units[1]);
    deal.uneven = deal.units[0] % used;
    if (deal.uneven && deal.units[1]) {
        deal.extra = std::max(1, (int)((args[0].kb_per_split + 4. ) / (args[1].k_blocks + 4.) + 0.5));
        deal.early = std::min(deal.units[1], deal.extra * (used - deal.uneven));
    }
    TS2_LAUNCH((linear_product_kernel<BACK, PN, BF16>), 2 * used, THREADS, SMEM, c.stream, maps, args[0], args[1], deal);
    if (splits > 1)
        TS2_LAUNCH((linear_join_kernel<PN, BF16>), (int)std::min<int64_t>(ceil_div((int64_t)join.m * ceil_div(join.n, 4), 256), 8 * sm_count(c.device)), 256, 0,
                   c.stream, join, join.kind);
    return TS2_OK;
}
template <bool BACK>
int run_products(const Ctx &c, bool bf16, const Product *products, int n, const Deal &deal)
{
    const Plan plan = plan_of(sm_count(c.device) / 2, products, n);
    if (plan.pn == 128)
        return bf16 ? run_products<BACK, 128, true>(c, products, n, plan.splits, deal) : run_products<BACK, 128, false>(c, products, n, plan.splits, deal);
    return bf16 ? run_products<BACK, 256, true>(c, products, n, plan.splits, deal) : run_products<BACK, 256, false>(c, products, n, plan.splits, deal);
}

// Tokens that take the form for a few.  us by it and by tiles: 32 x 2048 x 8192 16.3, 19.2; 32 x 768 x 768 3.7, 10.1; 32 x 8192 x 2048 20.3, 19.5; beyond, what
// the tokens' own reads cost grows with them.
constexpr int FEW_TOKENS = 32;
template <int NT, bool BF16, bool VEC>
int few(const Ctx &c, const FewArgs &p)
{
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = p.ranks, attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(ceil_div(p.m, 16) * p.ranks));
    cfg.blockDim = 32 * FEW_WARPS;
    cfg.stream = c.stream;
    cfg.attrs = attr;
    cfg.numAttrs = p.ranks > 1 ? 2 : 1;
    g_launch_count.fetch_add(1, std::memory_order_relaxed);
    if (const cudaError_t e = cudaLaunchKernelEx(&cfg, linear_few_kernel<NT, BF16, VEC>, p); e != cudaSuccess) {
        cudaGetLastError();
        return fail(TS2_ERR_CUDA, "kernel launch failed: %s (%s:%d)", cudaGetErrorString(e), __FILE__, __LINE__);
    }
    return TS2_OK;
}
template <int NT>
int few(const Ctx &c, bool bf16, bool vec, const FewArgs &p)
{
    return bf16 ? vec ? few<NT, true, true>(c, p) : few<NT, true, false>(c, p) : vec ? few<NT, false, true>(c, p) : few<NT, false, false>(c, p);
}

} // namespace

int linear_forward(const Ctx &c, const LinearShape &s, const void *x, int64_t x_ld, const void *w, int64_t w_ld, const float *bias, const void *residual,
                   int64_t residual_ld, void *y, int64_t y_ld, void *z, int64_t z_ld)
{
    if (s.T == 0)
        return TS2_OK;
    if (s.T <= FEW_TOKENS) {
        FewArgs f = {(int)s.T, s.in, s.out, (const uint16_t *)x, (const uint16_t *)w, (const uint16_t *)residual, x_ld, w_ld, residual_ld, y_ld, z_ld, bias,
                     (uint16_t *)y, (uint16_t *)z, s.act, 1};
        // CTAs for two an SM, each warp with 128 of K at least
        while (f.ranks < 8 && ceil_div(s.out, 16) * f.ranks < 2 * sm_count(c.device) && s.in >= 2 * f.ranks * FEW_WARPS * 4 * 32)
            f.ranks *= 2;
        const bool vec = tma_ok(x, x_ld, 2) && tma_ok(w, w_ld, 2);
        const auto form = s.T <= 8 ? few<1> : s.T <= 16 ? few<2> : few<4>;
        return form(c, s.type == TS2_OUT_BF16, vec, f);
    }
    PitchJobs jobs = {};
    const Operand a(c, x, x_ld, s.T, s.in, jobs), b(c, w, w_ld, s.out, s.in, jobs);
    if (a.rc != TS2_OK || b.rc != TS2_OK)
        return a.rc != TS2_OK ? a.rc : b.rc;
    if (jobs.n)
        if (const int rc = prepare<TS2_ACT_NONE, false>(c, nullptr, 0, nullptr, 0, 0, 0, 0, nullptr, 0, nullptr, jobs))
            return rc;
    Product q;
    q.a = &a, q.b = &b, q.K = s.in;
    LinearArgs &p = q.p;
    p.m = (int)s.T, p.n = s.out, p.kind = s.type, p.act = s.act, p.bias = bias;
    p.res = residual, p.res_ld = residual_ld, p.y = y, p.y_ld = y_ld, p.z = z, p.z_ld = z_ld;
    return run_products<false>(c, s.type == TS2_OUT_BF16, &q, 1, {});
}

int linear_backward(const Ctx &c, const LinearShape &s, const void *dy, int64_t dy_ld, const void *z, int64_t z_ld, const void *x, int64_t x_ld,
                    const void *w, int64_t w_ld, void *dx, int64_t dx_ld, int dw_kind, void *dw, int64_t dw_ld, float *dbias)
{
    const bool bf16 = s.type == TS2_OUT_BF16, products = dx || dw;
    if (s.T == 0) {
        if (dw && dw_kind != TS2_OUT_F32_ADD) {
            const size_t size = dw_kind == TS2_OUT_F32 ? 4 : 2;
            TS2_CUDA(cudaMemset2DAsync(dw, dw_ld * size, 0, s.in * size, s.out, c.stream));
        }
        if (dbias)
            TS2_CUDA(cudaMemsetAsync(dbias, 0, (size_t)s.out * 4, c.stream));
        return TS2_OK;
    }
    // dz where it differs from dy, the sums of its columns, and operands at another pitch
    const bool own_dz = s.act != TS2_ACT_NONE && products;
    const int layers = own_dz || dbias ? (int)std::max<int64_t>(1, std::min<int64_t>(ceil_div(s.T, 64), 8 * sm_count(c.device) / ceil_div(s.out, 128))) : 0;
    const int64_t own_ld = ceil_div(s.out, 8) * 8;
    const Scratch dz(c, own_dz ? (size_t)s.T * own_ld * 2 : 0), sums(c, dbias ? (size_t)layers * s.out * 4 : 0);
    PitchJobs jobs = {}, first = {};
    const Operand b(c, dx ? w : nullptr, w_ld, s.out, s.in, jobs), a(c, dw ? x : nullptr, x_ld, s.T, s.in, jobs),
        d(c, own_dz ? dz.p : products ? dy : nullptr, own_dz ? own_ld : dy_ld, s.T, s.out, first);
    for (const int rc : {dz.rc, sums.rc, a.rc, b.rc, d.rc})
        if (rc != TS2_OK)
            return rc;
    if (layers || jobs.n) {
        using F = int (*)(const Ctx &, const void *, int64_t, const void *, int64_t, int64_t, int, int, void *, int64_t, float *, const PitchJobs &);
        static const F forms[4][2] = {{prepare<TS2_ACT_NONE, false>, prepare<TS2_ACT_NONE, true>},
                                      {prepare<TS2_ACT_RELU, false>, prepare<TS2_ACT_RELU, true>},
                                      {prepare<TS2_ACT_GELU, false>, prepare<TS2_ACT_GELU, true>},
                                      {prepare<TS2_ACT_SILU, false>, prepare<TS2_ACT_SILU, true>}};
        if (const int rc = forms[s.act][bf16](c, dy, dy_ld, z, z_ld, s.T, s.out, layers, dz.p, own_ld, (float *)sums.p, jobs))
            return rc;
    }
    if (first.n) // dy itself
        if (const int rc = prepare<TS2_ACT_NONE, false>(c, nullptr, 0, nullptr, 0, 0, 0, 0, nullptr, 0, nullptr, first))
            return rc;
    if (!products) {
        if (dbias)
            TS2_LAUNCH(linear_sum_kernel, (int)ceil_div(s.out, 128), 128, 0, c.stream, (const float *)sums.p, s.out, layers, dbias);
        return TS2_OK;
    }
    // the product with the longer sums first: its units are the long ones, or are divided
    Product of_w, of_x, q[2];
    of_w.a = &d, of_w.b = &a, of_w.K = s.T;
    of_w.p.m = s.out, of_w.p.n = s.in, of_w.p.a_mn = true, of_w.p.kind = dw_kind, of_w.p.y = dw, of_w.p.y_ld = dw_ld;
    of_x.a = &d, of_x.b = &b, of_x.K = s.out;
    of_x.p.m = (int)s.T, of_x.p.n = s.in, of_x.p.kind = s.type, of_x.p.y = dx, of_x.p.y_ld = dx_ld;
    const int n = (dx ? 1 : 0) + (dw ? 1 : 0);
    const bool w_first = dw && (!dx || s.T >= s.out);
    q[0] = w_first ? of_w : of_x, q[1] = w_first ? of_x : of_w;
    Deal deal = {};
    if (dbias)
        deal.sums = (const float *)sums.p, deal.sums_out = dbias, deal.sums_n = s.out, deal.sums_blocks = layers;
    return run_products<true>(c, bf16, q, n, deal);
}

} // namespace ts2
