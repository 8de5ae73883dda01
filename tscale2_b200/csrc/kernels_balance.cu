// The load-balance term of a mixture-of-experts router and its gradient.  With p[t] = softmax(logits[t]), N tokens that count,
// C[e] choices of expert e among theirs and k choices a token:
//     loss = E / (k N) sum_e C[e] P[e],   P[e] = 1 / N sum_t p[t][e]     (1 where every expert gets the same)
//     d loss / d logits[t][e] = E / (k N^2) p[t][e] (C[e] - sum_j C[j] p[t][j])
// The counts have no gradient.  The routing weights are exp((l - lmax) / 2), so p is their square, normalised.
//
// G lanes share a row, each with its 16-byte pieces of it, so a warp reads 32 / G rows at a time, the next ones while it works on
// these; the softmax is a maximum and a sum over G lanes.  Logits are read once forward, and read once and written once
// backward: memory bandwidth bounds large calls, the latency of a launch small ones.  The column sums stay in registers until a
// block's rows are done; the blocks of a cluster join theirs through distributed shared memory, so that a small call is one
// launch and a large one leaves a partial result per cluster to a second.  All sums have a fixed order; counts are integers, so
// that the order of their atomics does not matter.
#include "kernels.cuh"
#include "pair_ptx.cuh"
#include <algorithm>

namespace ts2 {

static constexpr int THREADS = 256, WARPS = THREADS / 32;                // backward
static constexpr int SUM_THREADS = 512, SUM_WARPS = SUM_THREADS / 32;    // forward
static constexpr int MAX_EXPERTS = MOE_BALANCE_MAX_EXPERTS, CLUSTER = 8, MAX_CLUSTERS = 32;

template <class T>
__device__ __forceinline__ float widen(T v) { return (float)v; }
template <class T>
__device__ __forceinline__ T narrow(float v);
template <>
__device__ __forceinline__ float narrow<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half narrow<__half>(float v) { return __low2half(sat_half2(v, v)); }
template <>
__device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <class T, int VEC>
struct alignas(VEC * sizeof(T)) Piece {
    T v[VEC];
};

// Columns of a lane: piece i holds columns (i G + lane of the group) VEC ...
template <class T, int VEC, int G, int N>
struct Row {
    static constexpr int VALUES = VEC * N, PIECE = VEC % 4 ? 1 : 4; // PIECE: neighbouring columns that are 16 bytes of fp32
    float v[VALUES];

    static __device__ __forceinline__ int column(int i) { return ((i / VEC) * G + (int)(threadIdx.x & (G - 1))) * VEC + i % VEC; }
    // the lane's pieces of the row as they lie in memory; E = 0: nothing is read.  VEC > 1: E is a multiple of it
    struct Raw {
        Piece<T, VEC> p[N];
        __device__ __forceinline__ void load(const T *row, int E)
        {
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (column(i * VEC) < E)
                    p[i] = *(const Piece<T, VEC> *)(row + column(i * VEC));
        }
    };
    __device__ __forceinline__ void widen_from(const Raw &raw, int E)
    {
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int j = 0; j < VEC; ++j)
                v[i * VEC + j] = column(i * VEC) < E ? widen(raw.p[i].v[j]) : -INFINITY;
    }
    __device__ __forceinline__ void store(T *row, int E, bool add) const
    {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int c = column(i * VEC);
            if (c >= E)
                continue;
            Piece<T, VEC> p;
            if (add)
                p = *(const Piece<T, VEC> *)(row + c);
#pragma unroll
            for (int j = 0; j < VEC; ++j)
                p.v[j] = narrow<T>(add ? widen(p.v[j]) + v[i * VEC + j] : v[i * VEC + j]);
            *(Piece<T, VEC> *)(row + c) = p;
        }
    }
    // A row that is -inf throughout has no probabilities: zeros.  The maximum drops a NaN, the exponential of it does not.
    __device__ __forceinline__ void softmax()
    {
        float m = -INFINITY, sum = 0.f;
#pragma unroll
        for (int i = 0; i < VALUES; ++i)
            m = fmaxf(m, v[i]);
#pragma unroll
        for (int o = G / 2; o > 0; o >>= 1)
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        const float ref = m == -INFINITY ? 0.f : m; // the difference first: it may be of the lowest finite values
#pragma unroll
        for (int i = 0; i < VALUES; ++i) {
            asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(v[i]) : "f"((v[i] - ref) * 1.4426950408889634f));
            sum += v[i];
        }
#pragma unroll
        for (int o = G / 2; o > 0; o >>= 1)
            sum += __shfl_xor_sync(0xffffffffu, sum, o);
        const float r = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
        for (int i = 0; i < VALUES; ++i)
            v[i] *= r;
    }
};

struct BalanceArgs {
    const void *logits;
    long long ld, T;
    int E, selected;
    const int *ids;
    const uint8_t *mask;
    long long rows_per_block;
    // forward
    float *part_prob; // [clusters][E]
    int *part_count;  // [clusters][E + 1], the last one: rows that count
    int *counts;
    float *prob, *loss;
    // backward
    const float *dloss;
    float scale;
    void *dlogits;
    long long ld_d;
    int add;
};

// this CTA's shared-memory address `p`, in CTA `rank` of the cluster
template <class V>
__device__ __forceinline__ uint32_t in_rank(const V *p, unsigned rank) { return map_to_rank(smem_u32(p), rank); }
__device__ __forceinline__ float ld_float(uint32_t a)
{
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ int ld_int(uint32_t a)
{
    int v;
    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
    return v;
}

// 1 / N, and what sum_e C[e] P[e] is multiplied by: found while other things are on their way
struct BalanceUnit {
    double mean, loss;
    __device__ __forceinline__ BalanceUnit(int tokens, int E, int selected)
    {
        mean = tokens ? 1. / tokens : 0.;
        loss = mean * E / selected;
    }
};

// Two blocks an SM, but where a lane has more than 16 columns (65536 x 512 bf16 41 us; with one, and 32 clusters for which there is no room
// at once, 69).  That spills 48 bytes a thread for 512 columns of 16 bits, and 32 single columns a lane (1024 without alignment) 148.
template <class T, int VEC, int G, int N>
__global__ void __cluster_dims__(CLUSTER, 1, 1) __launch_bounds__(SUM_THREADS, VEC * N <= 16 ? 2 : 1) balance_sums_kernel(const BalanceArgs p)
{
    grid_dep_wait();
    using R = Row<T, VEC, G, N>;
    constexpr int ROWS = 32 / G, WIDTH = VEC * G * N < MAX_EXPERTS ? VEC * G * N : MAX_EXPERTS; // columns there is room for
    constexpr int PARTS = WIDTH <= 512 ? SUM_WARPS : SUM_WARPS / 2; // warps that leave their sums side by side
    __shared__ __align__(16) float sums[PARTS][WIDTH];
    __shared__ int count[MAX_EXPERTS + 1];
    __shared__ double terms[CLUSTER], warp_terms[SUM_WARPS];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, E = p.E;
    for (int e = threadIdx.x; e <= E; e += SUM_THREADS)
        count[e] = 0;
    __syncthreads();
    // the block's rows, counted from 0; what is read ahead of them: logits (of rows that do not count, too: waiting for the mask
    // would cost more), mask and each lane's first choice
    constexpr int STEP = SUM_WARPS * ROWS;
    const long long t_begin = blockIdx.x * p.rows_per_block;
    const int rows = (int)max(0ll, min(p.rows_per_block, p.T - t_begin)), own = warp * ROWS + lane / G, choice_row = lane / p.selected;
    const T *from = (const T *)p.logits + (t_begin + own) * p.ld;
    const uint8_t *mask = p.mask ? p.mask + t_begin + own : nullptr;
    const int *ids = p.ids + (t_begin + warp * ROWS) * p.selected + lane;
    const long long step_from = STEP * p.ld;
    float acc[R::VALUES];
#pragma unroll
    for (int i = 0; i < R::VALUES; ++i)
        acc[i] = 0.f;
    typename R::Raw raw;
    bool on;
    int id = -1;
    const auto fetch = [&](int r) { // r: the warp's first row
        const bool there = r + lane / G < rows;
        raw.load(from, there ? E : 0);
        on = there && (!mask || *mask);
        id = choice_row < ROWS && r + choice_row < rows ? *ids : -1;
        from += step_from, ids += STEP * p.selected;
        if (mask)
            mask += STEP;
    };
    fetch(warp * ROWS);
    for (int r = warp * ROWS; r < rows; r += STEP) {
        R row;
        const bool now = on;
        row.widen_from(raw, now ? E : 0);
        const unsigned m = __ballot_sync(0xffffffffu, now && (lane & (G - 1)) == 0);
        const int e = id;
        const int *more = ids - STEP * p.selected; // of these rows
        fetch(r + STEP);
        if (lane == 0 && m)
            atomicAdd(&count[E], __popc(m));
        if ((m >> ((choice_row * G) & 31) & 1) && e >= 0 && e < E)
            atomicAdd(&count[e], 1);
        for (int i = lane + 32; i < ROWS * p.selected; i += 32) { // what 32 lanes do not hold
            more += 32;
            const int at = i / p.selected;
            if (m >> at * G & 1) {
                const int f = *more;
                if (f >= 0 && f < E)
                    atomicAdd(&count[f], 1);
            }
        }
        row.softmax();
        if (now) {
#pragma unroll
            for (int i = 0; i < R::VALUES; ++i)
                acc[i] += row.v[i];
        }
    }
#pragma unroll
    for (int i = 0; i < R::VALUES; ++i)
#pragma unroll
        for (int o = G; o < 32; o <<= 1)
            acc[i] += __shfl_xor_sync(0xffffffffu, acc[i], o);
    const auto leave = [&](bool add) {
        if (lane < G)
#pragma unroll
            for (int i = 0; i < R::VALUES; i += R::PIECE) {
                float *to = &sums[warp % PARTS][R::column(i)];
                if constexpr (R::PIECE == 4) {
                    const float4 old = add ? *(const float4 *)to : make_float4(0.f, 0.f, 0.f, 0.f);
                    *(float4 *)to = make_float4(old.x + acc[i], old.y + acc[i + 1], old.z + acc[i + 2], old.w + acc[i + 3]);
                } else {
                    *to = add ? *to + acc[i] : acc[i];
                }
            }
    };
    if (warp < PARTS)
        leave(false);
    __syncthreads();
    if (PARTS < SUM_WARPS) {
        if (warp >= PARTS)
            leave(true);
        __syncthreads();
    }
    for (int e = threadIdx.x; e < E; e += SUM_THREADS) {
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < PARTS; ++w)
            sum += sums[w][e];
        sums[0][e] = sum;
    }
    // every CTA joins the columns rank, rank + 8, .. of the cluster
    cluster_sync();
    const unsigned rank = cluster_rank();
    const bool alone = gridDim.x == CLUSTER;
    int tokens = 0;
#pragma unroll
    for (int r = 0; r < CLUSTER; ++r)
        tokens += ld_int(in_rank(&count[E], r));
    const BalanceUnit unit(tokens, E, p.selected);
    double loss = 0.;
    const size_t cluster = blockIdx.x / CLUSTER;
    for (int e = (int)rank + CLUSTER * threadIdx.x; e < E; e += CLUSTER * SUM_THREADS) {
        double sum = 0.;
        int n = 0;
#pragma unroll
        for (int r = 0; r < CLUSTER; ++r) {
            sum += ld_float(in_rank(&sums[0][e], r));
            n += ld_int(in_rank(&count[e], r));
        }
        if (alone) {
            const double mean = sum * unit.mean;
            p.prob[e] = (float)mean;
            p.counts[e] = n;
            loss += mean * n;
        } else {
            p.part_prob[cluster * E + e] = (float)sum;
            p.part_count[cluster * (E + 1) + e] = n;
        }
    }
    if (rank == 0 && threadIdx.x == 0)
        *(alone ? &p.counts[E] : &p.part_count[cluster * (E + 1) + E]) = tokens;
    if (alone) {
        loss = warp_sum(loss);
        if (lane == 0)
            warp_terms[warp] = loss;
        __syncthreads();
        if (warp == 0)
            loss = warp_sum(lane < SUM_WARPS ? warp_terms[lane] : 0.);
        if (threadIdx.x == 0) {
            asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(in_rank(&terms[rank], 0)), "d"(loss) : "memory");
        }
    }
    cluster_sync(); // nobody reads a CTA's shared memory any more; the terms of the loss are there
    if (alone && rank == 0 && threadIdx.x == 0) {
#pragma unroll
        for (int r = 1; r < CLUSTER; ++r)
            loss += terms[r];
        *p.loss = (float)(loss * unit.loss);
    }
}

// One block: the clusters' sums.  `parts` threads a column, a part of the clusters each; a thread's loads are on their way together and
// a warp's are neighbours: 2 us behind a large launch (with a warp a column and a lane a cluster it grew to 20)
__global__ void __launch_bounds__(1024) balance_finish_kernel(const BalanceArgs p, int clusters, int width, int parts)
{
    grid_dep_wait();
    __shared__ double sums[1024], terms[32];
    __shared__ int counts[1024];
    const int E = p.E, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, e = threadIdx.x % width, part = threadIdx.x / width;
    const int tokens = __reduce_add_sync(0xffffffffu, lane < clusters ? p.part_count[(size_t)lane * (E + 1) + E] : 0);
    const BalanceUnit unit(tokens, E, p.selected);
    double sum = 0.;
    int n = 0;
    for (int c = part; c < clusters; c += 8 * parts) {
        float v[8];
        int k[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const bool in = c + i * parts < clusters && e < E;
            v[i] = in ? p.part_prob[(size_t)(c + i * parts) * E + e] : 0.f;
            k[i] = in ? p.part_count[(size_t)(c + i * parts) * (E + 1) + e] : 0;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
            sum += v[i], n += k[i];
    }
    sums[threadIdx.x] = sum, counts[threadIdx.x] = n;
    __syncthreads();
    double loss = 0.;
    if (threadIdx.x < E) { // part 0
        for (int i = 1; i < parts; ++i)
            sum += sums[i * width + e], n += counts[i * width + e];
        const double mean = sum * unit.mean;
        p.prob[e] = (float)mean, p.counts[e] = n;
        loss = mean * n;
    }
    loss = warp_sum(loss);
    if (lane == 0)
        terms[warp] = loss;
    __syncthreads();
    if (warp == 0)
        loss = warp_sum(lane < (int)blockDim.x / 32 ? terms[lane] : 0.);
    if (threadIdx.x == 0) {
        *p.loss = (float)(loss * unit.loss);
        p.counts[E] = tokens;
    }
}

// The counts enter as their distance from an even share: a constant in all C[e] falls out of the gradient, and the difference
// loses no digits where the load is nearly even.
template <class T, int VEC, int G, int N>
__global__ void __launch_bounds__(THREADS) balance_backward_kernel(const BalanceArgs p)
{
    grid_dep_wait();
    using R = Row<T, VEC, G, N>;
    constexpr int ROWS = 32 / G;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, E = p.E;
    long long t = ((long long)blockIdx.x * WARPS + warp) * ROWS + lane / G;
    const long long step = (long long)gridDim.x * WARPS * ROWS, step_from = step * p.ld, step_to = step * p.ld_d;
    const T *from = (const T *)p.logits + t * p.ld;
    T *to = (T *)p.dlogits + t * p.ld_d;
    typename R::Raw raw;
    bool on_next;
    const auto fetch = [&](long long t) {
        raw.load(from, t < p.T ? E : 0);
        on_next = t < p.T && (!p.mask || p.mask[t]);
        from += step_from;
    };
    fetch(t);
    const double tokens = p.counts[E];
    const double even = tokens * p.selected / E;
    const double unit = tokens > 0 ? (p.dloss ? (double)*p.dloss : 1.) * p.scale * E / (p.selected * tokens * tokens) : 0.;
    float f[R::VALUES];
#pragma unroll
    for (int i = 0; i < R::VALUES; ++i)
        f[i] = R::column(i) < E ? (float)((p.counts[R::column(i)] - even) * unit) : 0.f;
    for (; t - lane / G < p.T; t += step, to += step_to) { // a warp together
        const bool on = on_next;
        R row;
        row.widen_from(raw, on ? E : 0);
        fetch(t + step);
        row.softmax();
        float dot = 0.f;
#pragma unroll
        for (int i = 0; i < R::VALUES; ++i)
            dot = fmaf(row.v[i], f[i], dot);
#pragma unroll
        for (int o = G / 2; o > 0; o >>= 1)
            dot += __shfl_xor_sync(0xffffffffu, dot, o);
#pragma unroll
        for (int i = 0; i < R::VALUES; ++i)
            row.v[i] = on ? row.v[i] * (f[i] - dot) : 0.f;
        if (t < p.T && (on || !p.add)) // a row that does not count has no gradient: zeros, or nothing added
            row.store(to, E, p.add && on);
    }
}

// ---- launches --------------------------------------------------------------------------------------------------------
template <class T, int VEC, int G, int N>
static int launch(const Ctx &c, BalanceArgs &p, bool backward)
{
    if (backward) {
        // blocks a device holds, each of which reads the counts first: 2 an SM where a lane has several pieces (16384 x 512 bf16 11.2 us, with 4
        // 13.0), 4 where it has one (65536 x 128 10.9 us, with 2 12.6)
        const int rows = 32 / G * WARPS, cap = sm_count(c.device) * (N > 1 ? 2 : 4);
        TS2_LAUNCH((balance_backward_kernel<T, VEC, G, N>), (unsigned)std::max<int64_t>(1, std::min<int64_t>(cap, ceil_div(p.T, rows))), THREADS, 0,
                   c.stream, p);
        return TS2_OK;
    }
    // One cluster for up to four rounds of its warps, and then as many as the device holds at once: a second launch is 2 us, a round half
    // of one (x 64 bf16, us with one cluster and with several: 2048 rows, 4 rounds 6.4 and 6.7; 4096, 8 rounds 8.8 and 7.0; 2048 x 512,
    // 16 rounds 24.1 and 12.0)
    const int64_t round = (int64_t)32 / G * SUM_WARPS, clusters_wanted = ceil_div(p.T, round * CLUSTER);
    const int clusters = clusters_wanted <= 4 ? 1 : (int)std::min<int64_t>(clusters_wanted, VEC * N <= 16 ? MAX_CLUSTERS : MAX_CLUSTERS / 2);
    p.rows_per_block = ceil_div(ceil_div(p.T, (int64_t)clusters * CLUSTER), 32 / G) * (32 / G);
    if (clusters == 1) {
        TS2_LAUNCH((balance_sums_kernel<T, VEC, G, N>), CLUSTER, SUM_THREADS, 0, c.stream, p);
        return TS2_OK;
    }
    void *scratch;
    if (int rc = scratch_alloc(c.device, (size_t)clusters * (2 * p.E + 1) * 4, c.stream, &scratch))
        return rc;
    p.part_prob = (float *)scratch;
    p.part_count = (int *)scratch + (size_t)clusters * p.E;
    const auto work = [&] {
        TS2_LAUNCH((balance_sums_kernel<T, VEC, G, N>), clusters * CLUSTER, SUM_THREADS, 0, c.stream, p);
        const int width = (int)ceil_div(p.E, 32) * 32, parts = std::min(8, 1024 / width);
        TS2_LAUNCH(balance_finish_kernel, 1, width * parts, 0, c.stream, p, clusters, width, parts);
        return TS2_OK;
    };
    const int rc = work();
    scratch_free(c.stream, scratch);
    return rc;
}

// pieces of VEC elements, and as few lanes to a row as hold it with one piece each
template <class T, int VEC>
static int by_width(const Ctx &c, BalanceArgs &p, bool backward)
{
    const int pieces = (p.E + VEC - 1) / VEC;
    if (pieces <= 2)
        return launch<T, VEC, 2, 1>(c, p, backward);
    if (pieces <= 4)
        return launch<T, VEC, 4, 1>(c, p, backward);
    if (pieces <= 8)
        return launch<T, VEC, 8, 1>(c, p, backward);
    if (pieces <= 16)
        return launch<T, VEC, 16, 1>(c, p, backward);
    if (pieces <= 32)
        return launch<T, VEC, 32, 1>(c, p, backward);
    if (pieces <= 64)
        return launch<T, VEC, 32, 2>(c, p, backward);
    if constexpr (VEC <= 8)
        if (pieces <= 128)
            return launch<T, VEC, 32, 4>(c, p, backward);
    if constexpr (VEC <= 4)
        if (pieces <= 256)
            return launch<T, VEC, 32, 8>(c, p, backward);
    if constexpr (VEC == 1)
        return launch<T, VEC, 32, 32>(c, p, backward);
    return fail(TS2_ERR_UNSUPPORTED, "moe balance: %d experts", p.E);
}

template <class T>
static int by_type(const Ctx &c, BalanceArgs &p, bool backward)
{
    constexpr int VEC = 16 / sizeof(T);
    const bool pieces = p.E % VEC == 0 && p.ld % VEC == 0 && (uintptr_t)p.logits % 16 == 0 &&
                        (!backward || (p.ld_d % VEC == 0 && (uintptr_t)p.dlogits % 16 == 0));
    return pieces ? by_width<T, VEC>(c, p, backward) : by_width<T, 1>(c, p, backward);
}

static int run(const Ctx &c, int type, BalanceArgs &p, bool backward)
{
    switch (type) {
    case TS2_OUT_F32: return by_type<float>(c, p, backward);
    case TS2_OUT_F16: return by_type<__half>(c, p, backward);
    case TS2_OUT_BF16: return by_type<__nv_bfloat16>(c, p, backward);
    default: return fail(TS2_ERR_INVALID_ARG, "moe balance: unknown type %d", type);
    }
}

int moe_balance_forward(const Ctx &c, int type, const void *logits, int64_t ld, int64_t T, int E, int selected, const int *ids,
                        const uint8_t *mask, int *counts, float *prob, float *loss)
{
    BalanceArgs p = {};
    p.logits = logits, p.ld = ld, p.T = T, p.E = E, p.selected = selected, p.ids = ids, p.mask = mask;
    p.counts = counts, p.prob = prob, p.loss = loss;
    return run(c, type, p, false);
}

int moe_balance_backward(const Ctx &c, int type, const void *logits, int64_t ld, int64_t T, int E, int selected, const uint8_t *mask,
                         const int *counts, const float *dloss, float scale, void *dlogits, int64_t ld_d, bool add)
{
    BalanceArgs p = {};
    p.logits = logits, p.ld = ld, p.T = T, p.E = E, p.selected = selected, p.mask = mask;
    p.counts = const_cast<int *>(counts), p.dloss = dloss, p.scale = scale, p.dlogits = dlogits, p.ld_d = ld_d, p.add = add;
    return run(c, type, p, true);
}

} // namespace ts2
