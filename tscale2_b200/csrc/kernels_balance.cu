// The load-balance term of a mixture-of-experts router and its gradient.  With p[t] = softmax(logits[t]), N tokens that count,
// C[e] choices of expert e among theirs and k choices a token:
//     loss = E / (k N) sum_e C[e] P[e],   P[e] = 1 / N sum_t p[t][e]     (1 where every expert gets the same)
//     d loss / d logits[t][e] = E / (k N^2) p[t][e] (C[e] - sum_j C[j] p[t][j])
// The counts have no gradient.  The routing weights are exp((l - lmax) / 2), so p is their square, normalised.
//
// G lanes share a row, each with its 16-byte pieces of it, so a warp reads 32 / G rows at a time; the softmax is a maximum and a
// sum over G lanes.  Logits are read once forward, and read once and written once backward: memory bandwidth bounds large calls,
// the latency of a launch small ones.  The column sums stay in registers until a block's rows are done and are joined in a fixed
// order; counts are integers, so that the order of their atomics does not matter.
#include "kernels.cuh"
#include <algorithm>

namespace ts2 {

static constexpr int THREADS = 256, WARPS = THREADS / 32;
static constexpr int MAX_EXPERTS = 1024;

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
    static constexpr int VALUES = VEC * N;
    float v[VALUES];

    static __device__ __forceinline__ int column(int i) { return ((i / VEC) * G + (int)(threadIdx.x & (G - 1))) * VEC + i % VEC; }
    __device__ __forceinline__ void load(const T *row, int E)
    {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int c = column(i * VEC);
            if (c < E) { // VEC > 1: E is a multiple of it
                const Piece<T, VEC> p = *(const Piece<T, VEC> *)(row + c);
#pragma unroll
                for (int j = 0; j < VEC; ++j)
                    v[i * VEC + j] = widen(p.v[j]);
            } else {
#pragma unroll
                for (int j = 0; j < VEC; ++j)
                    v[i * VEC + j] = -INFINITY;
            }
        }
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
        const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int i = 0; i < VALUES; ++i)
            sum += v[i] = expf(v[i] - ref);
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
    float *part_prob; // [blocks][E]
    int *part_count;  // [blocks][E + 1], the last one: rows that count
    int *counts;
    float *prob, *loss;
    // backward
    const float *dloss;
    float scale;
    void *dlogits;
    long long ld_d;
    int add;
};

template <class T, int VEC, int G, int N>
__global__ void __launch_bounds__(THREADS) balance_sums_kernel(const BalanceArgs p)
{
    grid_dep_wait();
    using R = Row<T, VEC, G, N>;
    constexpr int ROWS = 32 / G;
    __shared__ float sums[MAX_EXPERTS];
    __shared__ int count[MAX_EXPERTS + 1];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, E = p.E;
    for (int e = threadIdx.x; e <= E; e += THREADS)
        count[e] = 0;
    __syncthreads();
    const long long t_begin = blockIdx.x * p.rows_per_block, t_end = min(p.T, t_begin + p.rows_per_block);
    float acc[R::VALUES];
#pragma unroll
    for (int i = 0; i < R::VALUES; ++i)
        acc[i] = 0.f;
    for (long long base = t_begin + warp * ROWS; base < t_end; base += WARPS * ROWS) {
        const long long t = base + lane / G;
        R row;
        const bool on = t < t_end && (!p.mask || p.mask[t]);
        row.load((const T *)p.logits + t * p.ld, on ? E : 0);
        row.softmax();
        if (on) {
#pragma unroll
            for (int i = 0; i < R::VALUES; ++i)
                acc[i] += row.v[i];
        }
        const unsigned m = __ballot_sync(0xffffffffu, on && (lane & (G - 1)) == 0);
        if (lane == 0 && m)
            atomicAdd(&count[E], __popc(m));
    }
    for (long long i = t_begin * p.selected + threadIdx.x; i < t_end * p.selected; i += THREADS) {
        const int e = p.ids[i];
        if (e >= 0 && e < E && (!p.mask || p.mask[i / p.selected]))
            atomicAdd(&count[e], 1);
    }
#pragma unroll
    for (int i = 0; i < R::VALUES; ++i)
#pragma unroll
        for (int o = G; o < 32; o <<= 1)
            acc[i] += __shfl_xor_sync(0xffffffffu, acc[i], o);
    for (int w = 0; w < WARPS; ++w) { // warp by warp: a fixed order
        if (warp == w && lane < G) {
#pragma unroll
            for (int i = 0; i < R::VALUES; ++i) {
                const int c = R::column(i);
                if (c < E)
                    sums[c] = w ? sums[c] + acc[i] : acc[i];
            }
        }
        __syncthreads();
    }
    for (int e = threadIdx.x; e < E; e += THREADS)
        p.part_prob[(size_t)blockIdx.x * E + e] = sums[e];
    for (int e = threadIdx.x; e <= E; e += THREADS)
        p.part_count[(size_t)blockIdx.x * (E + 1) + e] = count[e];
}

// one block: the blocks' sums, in their order
__global__ void __launch_bounds__(MAX_EXPERTS) balance_finish_kernel(const BalanceArgs p, int blocks)
{
    grid_dep_wait();
    __shared__ int total;
    __shared__ double terms[32];
    const int E = p.E, e = threadIdx.x, lane = e & 31, warp = e >> 5;
    if (warp == 0) {
        int n = 0;
        for (int b = lane; b < blocks; b += 32)
            n += p.part_count[(size_t)b * (E + 1) + E];
        n = __reduce_add_sync(0xffffffffu, n);
        if (lane == 0)
            total = n, p.counts[E] = n;
    }
    double sum = 0.;
    int n = 0;
    if (e < E) {
        for (int b = 0; b < blocks; ++b) {
            sum += p.part_prob[(size_t)b * E + e];
            n += p.part_count[(size_t)b * (E + 1) + e];
        }
        p.counts[e] = n;
    }
    __syncthreads();
    const double tokens = total;
    const double mean = total ? sum / tokens : 0.;
    if (e < E)
        p.prob[e] = (float)mean;
    double term = total ? mean * n * E / (tokens * p.selected) : 0.;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        term += __shfl_xor_sync(0xffffffffu, term, o);
    if (lane == 0)
        terms[warp] = term;
    __syncthreads();
    if (e == 0) {
        for (int w = 1; w < (int)blockDim.x / 32; ++w)
            term += terms[w];
        *p.loss = (float)term;
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
    const double tokens = p.counts[E];
    const double even = tokens * p.selected / E;
    const double unit = tokens > 0 ? (p.dloss ? (double)*p.dloss : 1.) * p.scale * E / (p.selected * tokens * tokens) : 0.;
    float f[R::VALUES];
#pragma unroll
    for (int i = 0; i < R::VALUES; ++i)
        f[i] = R::column(i) < E ? (float)((p.counts[R::column(i)] - even) * unit) : 0.f;
    for (long long base = ((long long)blockIdx.x * WARPS + warp) * ROWS; base < p.T; base += (long long)gridDim.x * WARPS * ROWS) {
        const long long t = base + lane / G;
        const bool on = t < p.T && (!p.mask || p.mask[t]);
        R row;
        row.load((const T *)p.logits + t * p.ld, on ? E : 0);
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
            row.store((T *)p.dlogits + t * p.ld_d, E, p.add && on);
    }
}

// ---- launches --------------------------------------------------------------------------------------------------------
template <class T, int VEC, int G, int N>
static int launch(const Ctx &c, BalanceArgs &p, bool backward)
{
    const int rows = 32 / G * WARPS, cap = sm_count(c.device) * 4;
    if (backward) {
        TS2_LAUNCH((balance_backward_kernel<T, VEC, G, N>), (unsigned)std::max<int64_t>(1, std::min<int64_t>(cap, ceil_div(p.T, rows))), THREADS, 0,
                   c.stream, p);
        return TS2_OK;
    }
    p.rows_per_block = std::max<int64_t>(rows, ceil_div(ceil_div(p.T, cap), rows) * rows);
    const int blocks = (int)std::max<int64_t>(1, ceil_div(p.T, p.rows_per_block));
    void *scratch;
    if (int rc = scratch_alloc(c.device, (size_t)blocks * (2 * p.E + 1) * 4, c.stream, &scratch))
        return rc;
    p.part_prob = (float *)scratch;
    p.part_count = (int *)scratch + (size_t)blocks * p.E;
    const auto work = [&] {
        TS2_LAUNCH((balance_sums_kernel<T, VEC, G, N>), blocks, THREADS, 0, c.stream, p);
        TS2_LAUNCH(balance_finish_kernel, 1, (p.E + 31) / 32 * 32, 0, c.stream, p, blocks);
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
    if (p.E < 1 || p.E > MAX_EXPERTS)
        return fail(TS2_ERR_UNSUPPORTED, "moe balance: need 1 <= experts <= %d (got %d)", MAX_EXPERTS, p.E);
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
