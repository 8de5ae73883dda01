// Choice of experts from a router's logits and the gradient of the weights.  Per token, l the logits,
//     s = softmax(l) or sigmoid(l),   key = s + bias
// the largest keys (of the best groups) are chosen, and their weights are scale * s or scale * s / (sum of the chosen s).  Back, with the choices
// given, d = the gradient of the weights, w = the weights over scale,
//     softmax              dl[e] = scale (d[e] w[e] - s[e] sum_j d[j] w[j])         (d[e] w[e] only where e was chosen)
//     softmax, renormalised  dl[e] = scale w[e] (d[e] - sum_j d[j] w[j])            for chosen e
//     sigmoid              dl[e] = scale d[e] s[e] (1 - s[e])
//     sigmoid, renormalised  dl[e] = scale w[e] (1 - s[e]) (d[e] - sum_j d[j] w[j])
// A warp takes a row.
#include "elem_types.cuh"
#include "kernels.cuh"
#include <algorithm>

namespace ts2 {

static constexpr int WARPS = 8, THREADS = 32 * WARPS;
static constexpr unsigned FULL = 0xffffffffu;

__device__ __forceinline__ double warp_max(double v)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        v = fmax(v, __shfl_xor_sync(FULL, v, o));
    return v;
}
// over the warp: the largest key, the lowest index among equal ones; -1 where all are -inf
__device__ __forceinline__ int warp_best(double key, int at)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const double k = __shfl_xor_sync(FULL, key, o);
        const int i = __shfl_xor_sync(FULL, at, o);
        if (k > key || (k == key && i < at))
            key = k, at = i;
    }
    return key == -INFINITY ? -1 : at;
}
// the weights of a token's choices, lane j has choice j (id < 0: none): over scale; s: the scores
__device__ __forceinline__ float choice_weight(bool softmax, bool renormalize, bool made, float l, float row_max, float row_sum, float &s)
{
    float w;
    if (softmax) {
        s = made ? expf(l - row_max) / row_sum : 0.f;
        if (!renormalize)
            return s;
        const float top = warp_max(made ? l : -INFINITY);
        w = made ? expf(l - top) : 0.f;
    } else {
        // sigmoid(l) = exp(min(l, 0)) / (1 + exp(-|l|)): nothing underflows that matters to the quotient
        const float low = fminf(l, 0.f), rest = 1.f / (1.f + expf(-fabsf(l)));
        s = made ? expf(low) * rest : 0.f;
        if (!renormalize)
            return s;
        const float top = warp_max(made ? low : -INFINITY);
        w = made ? expf(low - top) * rest : 0.f;
    }
    const float sum = warp_sum(w);
    return sum > 0.f ? w / sum : 0.f;
}

template <class T>
__global__ void __launch_bounds__(THREADS) route_forward_kernel(const T *__restrict__ logits, int64_t ld, RouteShape p, const float *__restrict__ bias,
                                                                int groups, int kept, int group_top, const uint8_t *__restrict__ mask, int *ids, float *weights)
{
    grid_dep_wait();
    extern __shared__ double route_keys[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, E = p.E, per = E / groups;
    double *key = route_keys + warp * E;
    const bool softmax = p.score == TS2_SCORE_SOFTMAX;
    for (int64_t t = (int64_t)blockIdx.x * WARPS + warp; t < p.T; t += (int64_t)gridDim.x * WARPS) {
        const T *row = logits + t * ld;
        const bool on = !mask || mask[t];
        float top = -INFINITY, sum = 1.f;
        double top64 = 0., sum64 = 1.;
        bool bad = false;
        if (softmax) {
            sum = 0.f, sum64 = 0.;
            for (int c = lane; c < E; c += 32) {
                const float l = widen(row[c]);
                bad |= !(l < INFINITY);
                top = fmaxf(top, l);
            }
            top = warp_max(top);
            if (top == -INFINITY)
                top = 0.f;
            top64 = top;
            for (int c = lane; c < E; c += 32) {
                const float l = widen(row[c]);
                sum += expf(l - top);
                sum64 += exp((double)l - top64);
            }
            sum = warp_sum(sum), sum64 = warp_sum(sum64);
            bad = __any_sync(FULL, bad);
        }
        const auto out = [&](float l) { return bad || !on || l == -INFINITY || !(l == l); };
        for (int c = lane; c < E; c += 32) {
            const float l = widen(row[c]);
            double k = softmax ? exp((double)l - top64) / sum64 : 1. / (1. + exp(-(double)l));
            if (bias)
                k += bias[c];
            key[c] = out(l) || !(k == k) ? -INFINITY : k;
        }
        __syncwarp();
        unsigned keep = FULL; // groups that experts are taken from
        if (groups > 1) {
            double best = -INFINITY, second = -INFINITY;
            if (lane < groups)
                for (int c = lane * per; c < (lane + 1) * per; ++c) {
                    second = fmax(second, fmin(best, key[c]));
                    best = fmax(best, key[c]);
                }
            double rank = group_top == 2 ? best + second : best;
            if (!(rank == rank))
                rank = -INFINITY;
            keep = 0;
            for (int k = 0; k < kept; ++k) {
                const int g = warp_best(rank, lane);
                if (g < 0)
                    break;
                keep |= 1u << g;
                if (lane == g)
                    rank = -INFINITY;
            }
        }
        __syncwarp();
        for (int c = lane; c < E; c += 32) {
            if (!(keep >> (groups > 1 ? c / per : 0) & 1))
                key[c] = -INFINITY;
            else if (!bias && key[c] > -INFINITY)
                key[c] = widen(row[c]);
        }
        __syncwarp();
        int id = -1; // lane j: choice j
        for (int j = 0; j < p.selected; ++j) {
            double best = -INFINITY;
            int at = E;
            for (int c = lane; c < E; c += 32)
                if (key[c] > best)
                    best = key[c], at = c;
            at = warp_best(best, at);
            if (at < 0)
                break;
            if (lane == j)
                id = at;
            __syncwarp();
            if (lane == 0)
                key[at] = -INFINITY;
            __syncwarp();
        }
        float s;
        const float w = choice_weight(softmax, p.renormalize, id >= 0, id >= 0 ? widen(row[id]) : 0.f, top, sum, s);
        if (lane < p.selected) {
            ids[t * p.selected + lane] = id;
            weights[t * p.selected + lane] = p.scale * w;
        }
        __syncwarp();
    }
}

template <class T>
__global__ void __launch_bounds__(THREADS) route_backward_kernel(const T *__restrict__ logits, int64_t ld, RouteShape p, const uint8_t *__restrict__ mask,
                                                                 const int *__restrict__ ids, const float *__restrict__ dweights, T *dlogits, int64_t ld_d, bool add)
{
    grid_dep_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, E = p.E;
    const bool softmax = p.score == TS2_SCORE_SOFTMAX, dense = softmax && !p.renormalize;
    for (int64_t t = (int64_t)blockIdx.x * WARPS + warp; t < p.T; t += (int64_t)gridDim.x * WARPS) {
        const T *row = logits + t * ld;
        const bool on = !mask || mask[t];
        const int id = on && lane < p.selected ? ids[t * p.selected + lane] : -1;
        const bool made = id >= 0 && id < E;
        const float d = made ? dweights[t * p.selected + lane] : 0.f;
        const bool any = __any_sync(FULL, made);
        float top = -INFINITY, sum = 0.f;
        if (dense && any) {
            for (int c = lane; c < E; c += 32)
                top = fmaxf(top, widen(row[c]));
            top = warp_max(top);
            if (top == -INFINITY)
                top = 0.f;
            for (int c = lane; c < E; c += 32)
                sum += expf(widen(row[c]) - top);
            sum = warp_sum(sum);
        }
        float s;
        const float w = choice_weight(softmax, p.renormalize, made, made ? widen(row[id]) : 0.f, top, sum, s);
        const float dot = warp_sum(d * w);
        float g = d * w; // of the choice's logit, over scale
        if (p.renormalize)
            g = w * (d - dot) * (softmax ? 1.f : 1.f - s);
        else if (!softmax)
            g *= 1.f - s;
        for (int c = lane; c < (E + 31) / 32 * 32; c += 32) {
            float v = 0.f;
            for (int j = 0; j < p.selected; ++j) {
                const int e = __shfl_sync(FULL, made ? id : -1, j);
                const float x = __shfl_sync(FULL, g, j);
                v += e == c ? x : 0.f;
            }
            if (c >= E)
                continue;
            if (dense && any)
                v -= dot * (expf(widen(row[c]) - top) / sum);
            v *= p.scale;
            T *to = dlogits + t * ld_d + c;
            *to = narrow<T>(add ? widen(*to) + v : v);
        }
        __syncwarp();
    }
}

// ---- host ------------------------------------------------------------------------------------------------------------
static int blocks_for(const Ctx &c, int64_t T) { return (int)std::max<int64_t>(1, std::min<int64_t>(ceil_div(T, WARPS), 8 * sm_count(c.device))); }

template <class T>
static int forward(const Ctx &c, const RouteShape &s, const void *logits, int64_t ld, const float *bias, int groups, int kept, int group_top,
                   const uint8_t *mask, int *ids, float *weights)
{
    const size_t smem = (size_t)WARPS * s.E * 8;
    TS2_CUDA(cudaFuncSetAttribute((const void *)route_forward_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, WARPS * MOE_ROUTE_MAX_EXPERTS * 8));
    TS2_LAUNCH((route_forward_kernel<T>), blocks_for(c, s.T), THREADS, smem, c.stream, (const T *)logits, ld, s, bias, groups, kept, group_top, mask, ids,
               weights);
    return TS2_OK;
}
template <class T>
static int backward(const Ctx &c, const RouteShape &s, const void *logits, int64_t ld, const uint8_t *mask, const int *ids, const float *dweights,
                    void *dlogits, int64_t ld_d, bool add)
{
    TS2_LAUNCH((route_backward_kernel<T>), blocks_for(c, s.T), THREADS, 0, c.stream, (const T *)logits, ld, s, mask, ids, dweights, (T *)dlogits, ld_d, add);
    return TS2_OK;
}

int moe_route_forward(const Ctx &c, const RouteShape &s, const void *logits, int64_t ld, const float *bias, int groups, int groups_kept, int group_top,
                      const uint8_t *mask, int *ids, float *weights)
{
    if (s.T == 0)
        return TS2_OK;
    const auto f = s.type == TS2_OUT_F32 ? forward<float> : s.type == TS2_OUT_F16 ? forward<__half> : forward<__nv_bfloat16>;
    return f(c, s, logits, ld, bias, groups, groups_kept, group_top, mask, ids, weights);
}
int moe_route_backward(const Ctx &c, const RouteShape &s, const void *logits, int64_t ld, const uint8_t *mask, const int *ids, const float *dweights,
                       void *dlogits, int64_t dlogits_ld, bool add)
{
    if (s.T == 0)
        return TS2_OK;
    const auto f = s.type == TS2_OUT_F32 ? backward<float> : s.type == TS2_OUT_F16 ? backward<__half> : backward<__nv_bfloat16>;
    return f(c, s, logits, ld, mask, ids, dweights, dlogits, dlogits_ld, add);
}

} // namespace ts2
