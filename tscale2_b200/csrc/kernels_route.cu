// Choice of experts from a router's logits and the gradient of the weights.  Per token, l the logits,
//     s = softmax(l) or sigmoid(l),   key = s + bias
// the largest keys (of the best groups) are chosen, and their weights are scale * s or scale * s / (sum of the chosen s).  Back, with the choices
// given, d = the gradient of the weights, w = the weights over scale,
//     softmax              dl[e] = scale (d[e] w[e] - s[e] sum_j d[j] w[j])         (d[e] w[e] only where e was chosen)
//     softmax, renormalised  dl[e] = scale w[e] (d[e] - sum_j d[j] w[j])            for chosen e
//     sigmoid              dl[e] = scale d[e] s[e] (1 - s[e])
//     sigmoid, renormalised  dl[e] = scale w[e] (1 - s[e]) (d[e] - sum_j d[j] w[j])
//
// A warp takes 4 rows (8 of up to 128 experts).  They come in a row at a time in pieces of 8 columns a lane, and their keys and every piece's largest key go to
// shared memory.  Then 4 or 8 lanes have a row, each the largest keys of some neighbouring pieces in registers: a choice is a maximum over those and over the
// lanes, and only the piece that it came from is looked at again, by all of them.  Bound by instructions, 540 a row of 256 sigmoid scores with a bias, in groups and
// 8 choices (of 224 for the row itself, 72 for its keys, 105 for groups, 20 for a choice), at 2.1 a clock of an SM with 39 % of its warps: 35.6 us for 32768 rows,
// whose bytes take 3; 18.3 us for 65537 rows of 128, 4 choices, whose bytes take 2.9.
//
// Keys are fp32 first.  They order as exact ones would where they differ by more than fp32 can be wrong, so a row in which two choices, the last choice and the
// next key, or two groups at the border are nearer than that is done once more in fp64 by the whole warp.  A group's rank of two keys is off by what those are
// rounded by, which is not small where a large bias and one of the other sign cancel, so a rank carries the size of its keys.  Without a bias (and with groups
// ranked by one key) the logits themselves are the keys, and exact.
#include "elem_types.cuh"
#include "kernels.cuh"
#include <algorithm>
#include <type_traits>

namespace ts2 {

static constexpr int THREADS = 128;
static constexpr unsigned FULL = 0xffffffffu;

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

struct Choice { // what the forward pass needs beside a RouteShape
    const float *bias;
    int groups, kept, group_top;
};

// One row by the whole warp, its keys in fp64: any row, and slow
template <class T>
__device__ __noinline__ void route_row_exactly(const T *__restrict__ row, const RouteShape &p, const Choice &c, double *key, int *ids, float *weights)
{
    const int lane = threadIdx.x & 31, E = p.E, per = E / c.groups;
    const bool softmax = p.score == TS2_SCORE_SOFTMAX;
    float top = -INFINITY, sum = 0.f;
    double sum64 = 0.;
    bool bad = false;
    if (softmax) {
        for (int e = lane; e < E; e += 32) {
            const float l = widen(row[e]);
            bad |= !(l < INFINITY);
            top = fmaxf(top, l);
        }
        bad = __any_sync(FULL, bad);
        top = warp_max(top);
        if (top == -INFINITY)
            top = 0.f;
        for (int e = lane; e < E; e += 32)
            sum64 += exp((double)widen(row[e]) - (double)top);
        sum64 = warp_sum(sum64);
        sum = (float)sum64;
    }
    for (int e = lane; e < E; e += 32) {
        const double l = widen(row[e]);
        double k = softmax ? exp(l - (double)top) / sum64 : 1. / (1. + exp(-l));
        if (c.bias)
            k += c.bias[e];
        key[e] = bad || l == -INFINITY || !(k == k) ? -INFINITY : k;
    }
    __syncwarp();
    unsigned keep = FULL; // groups that experts are taken from
    if (c.groups > 1) {
        double best = -INFINITY, second = -INFINITY;
        if (lane < c.groups)
            for (int e = lane * per; e < (lane + 1) * per; ++e) {
                second = fmax(second, fmin(best, key[e]));
                best = fmax(best, key[e]);
            }
        double rank = c.group_top == 2 ? best + second : best;
        if (!(rank == rank))
            rank = -INFINITY;
        keep = 0;
        for (int k = 0; k < c.kept; ++k) {
            const int g = warp_best(rank, lane);
            if (g < 0)
                break;
            keep |= 1u << g;
            if (lane == g)
                rank = -INFINITY;
        }
    }
    __syncwarp();
    for (int e = lane; e < E; e += 32) {
        if (!(keep >> (c.groups > 1 ? e / per : 0) & 1))
            key[e] = -INFINITY;
        else if (!c.bias && key[e] > -INFINITY)
            key[e] = widen(row[e]);
    }
    __syncwarp();
    int id = -1; // lane j: choice j
    for (int j = 0; j < p.selected; ++j) {
        double best = -INFINITY;
        int at = E;
        for (int e = lane; e < E; e += 32)
            if (key[e] > best)
                best = key[e], at = e;
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
        ids[lane] = id;
        weights[lane] = p.scale * w;
    }
    __syncwarp();
}

// Shared memory of a warp, in 4-byte words: keys of ROWS rows (a pitch that keeps the rows' pieces in different banks), the largest and the second key of
// their pieces, the groups' ranks and the sizes of the keys in them, choices and what they weigh, and of the softmax the row's maximum and its sum's reciprocal.
__host__ __device__ constexpr int key_pitch(int pieces) { return (pieces + 3) / 4 * 32 + 4; }
__host__ __device__ constexpr int piece_pitch(int most) { return most + 4; } // most: pieces that a row may have
__host__ __device__ constexpr int warp_words(int rows, int pieces, int most, bool second, int groups, int selected)
{
    return (rows * (key_pitch(pieces) + piece_pitch(most) * (second ? 2 : 1) + (groups > 1 ? 2 * groups : 0) + 2 * (selected + 1) + 2) + 3) / 4 * 4;
}

// eight neighbours from column e on as they lie in memory, -inf behind the last one and where there is nothing to read
template <class T>
struct Eight {
    static constexpr int PER = 16 / sizeof(T);
    Piece<T, PER> q[8 / PER];
    __device__ __forceinline__ void load(const T *row, int e, int E, bool vec, bool there)
    {
        if (vec && there && e + 8 <= E) {
#pragma unroll
            for (int i = 0; i < 8 / PER; ++i)
                q[i] = *(const Piece<T, PER> *)(row + e + i * PER);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                q[i / PER].v[i % PER] = there && e + i < E ? row[e + i] : narrow_infinity();
        }
    }
    static __device__ __forceinline__ T narrow_infinity()
    {
        if constexpr (sizeof(T) == 4)
            return -INFINITY;
        else if constexpr (std::is_same<T, __half>::value)
            return __ushort_as_half(0xfc00);
        else
            return __ushort_as_bfloat16(0xff80);
    }
    __device__ __forceinline__ void widen_to(float (&v)[8]) const
    {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            v[i] = widen(q[i / PER].v[i % PER]);
    }
};
// over the `width` neighbouring lanes that share a row
__device__ __forceinline__ float max_over(float v, int width)
{
#pragma unroll
    for (int o = width / 2; o > 0; o >>= 1)
        v = fmaxf(v, __shfl_xor_sync(FULL, v, o));
    return v;
}
__device__ __forceinline__ float sum_over(float v, int width)
{
#pragma unroll
    for (int o = width / 2; o > 0; o >>= 1)
        v += __shfl_xor_sync(FULL, v, o);
    return v;
}
__device__ __forceinline__ float max8(const float (&v)[8])
{
    return fmaxf(fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])), fmaxf(fmaxf(v[4], v[5]), fmaxf(v[6], v[7])));
}

// the largest and the second of eight
__device__ __forceinline__ void two_of(const float (&v)[8], float &best, float &next)
{
    float a[4], b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        a[i] = fmaxf(v[2 * i], v[2 * i + 1]), b[i] = fminf(v[2 * i], v[2 * i + 1]);
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
        b[i] = fmaxf(fminf(a[i], a[i + 1]), fmaxf(b[i], b[i + 1]));
        a[i] = fmaxf(a[i], a[i + 1]);
    }
    best = fmaxf(a[0], a[2]), next = fmaxf(fminf(a[0], a[2]), fmaxf(b[0], b[2]));
}

// half the sum of two keys, which does not overflow where both are fp32's lowest or largest value; -inf where one of them is none
__device__ __forceinline__ float half_sum(float best, float next) { return next > -INFINITY ? fmaf(0.5f, best, 0.5f * next) : -INFINITY; }

// L: lanes that share a row while choices are made; NB: pieces of 8 columns that each of them has (E <= 8 L NB)
template <class T, int L, int NB>
__global__ void __launch_bounds__(THREADS, NB <= 4 ? 8 : NB * L == 32 ? 5 : 4) route_forward_kernel(const T *__restrict__ logits, int64_t ld, bool vec, const RouteShape p, const Choice c,
                                                                const uint8_t *__restrict__ mask, int *ids, float *weights)
{
    grid_dep_wait();
    // WIDTH: lanes that share a row while it comes in, HELD pieces each, STEP passes at a time
    constexpr int ROWS = 32 / L, MOST = L * NB, WIDTH = MOST >= 32 ? 32 : MOST, HELD = MOST / WIDTH, PASSES = ROWS * WIDTH / 32, STEP = PASSES < 8 / HELD ? PASSES : 8 / HELD;
    extern __shared__ __align__(16) float route_smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, E = p.E, pieces = (E + 7) / 8, per = E / c.groups;
    // groups of 8, 16 .. 256 neighbours are ranked while they come in, others from what lies in shared memory
    const bool two = c.groups > 1 && c.group_top == 2, coming = HELD == 1 && per >= 8 && (per & (per - 1)) == 0, kept_second = two && !coming;
    constexpr int pp = piece_pitch(MOST);
    const int pitch = key_pitch(pieces), slots = p.selected + 1, group_pieces = per >> 3, shift = coming ? 31 - __clz(group_pieces) : 0;
    float *keys = route_smem + warp * warp_words(ROWS, pieces, MOST, kept_second, c.groups, p.selected), *first = keys + ROWS * pitch, *second = first + ROWS * pp,
          *ranks = second + (kept_second ? ROWS * pp : 0), *sizes = ranks + (c.groups > 1 ? ROWS * c.groups : 0), *chosen = sizes + (c.groups > 1 ? ROWS * c.groups : 0),
          *row_max = chosen + ROWS * slots,
          *row_inv = row_max + ROWS;
    int *chosen_id = (int *)(row_inv + ROWS);
    const int64_t t0 = ((int64_t)blockIdx.x * (THREADS / 32) + warp) * ROWS;
    if (t0 >= p.T)
        return;
    const bool softmax = p.score == TS2_SCORE_SOFTMAX, by_logit = !c.bias && (c.groups == 1 || c.group_top == 1), stats = softmax && !(by_logit && p.renormalize);
    const int at = lane & (WIDTH - 1), sub = lane / WIDTH;
    float bias[HELD][8]; // of the lane's columns
#pragma unroll
    for (int h = 0; h < HELD; ++h)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int e = (at + 32 * h) * 8 + i;
            bias[h][i] = c.bias && e < E ? c.bias[e] : 0.f;
        }
    // rows come in
#pragma unroll 1
    for (int pass0 = 0; pass0 < PASSES; pass0 += STEP) {
        Eight<T> raw[STEP][HELD];
        bool on[STEP];
#pragma unroll
        for (int s = 0; s < STEP; ++s) {
            const int64_t t = t0 + (pass0 + s) * (32 / WIDTH) + sub;
            on[s] = t < p.T && (!mask || mask[t]);
#pragma unroll
            for (int h = 0; h < HELD; ++h)
                raw[s][h].load(logits + t * ld, (at + 32 * h) * 8, E, vec, on[s] && at + 32 * h < pieces);
        }
#pragma unroll
        for (int s = 0; s < STEP; ++s) {
            const int r = (pass0 + s) * (32 / WIDTH) + sub;
            float v[HELD][8];
            float top = 0.f, inv = 1.f;
            bool bad = !on[s];
#pragma unroll
            for (int h = 0; h < HELD; ++h)
                raw[s][h].widen_to(v[h]);
            if (stats) {
                top = max8(v[0]);
#pragma unroll
                for (int h = 1; h < HELD; ++h)
                    top = fmaxf(top, max8(v[h]));
                top = max_over(top, WIDTH);
                top = top == -INFINITY ? 0.f : top;
                float sum = 0.f;
#pragma unroll
                for (int h = 0; h < HELD; ++h)
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        sum += ex2((v[h][i] - top) * 1.44269504f); // a NaN, and infinity minus itself, end here
                sum = sum_over(sum, WIDTH);
                bad |= !(sum == sum);
                inv = 1.f / sum;
                if (at == 0)
                    row_max[r] = top, row_inv[r] = inv;
            } else if (softmax) {
                bool wrong = false;
#pragma unroll
                for (int h = 0; h < HELD; ++h)
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        wrong |= !(v[h][i] < INFINITY);
                const unsigned lanes = WIDTH == 32 ? FULL : ((1u << (WIDTH & 31)) - 1) << (sub * WIDTH);
                bad |= (__ballot_sync(FULL, wrong) & lanes) != 0;
            }
#pragma unroll
            for (int h = 0; h < HELD; ++h) {
                const int piece = at + 32 * h;
                float k[8];
                if (by_logit) {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        k[i] = fmaxf(v[h][i], -INFINITY); // a NaN is none
                } else {
                    if (softmax) {
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            k[i] = ex2((v[h][i] - top) * 1.44269504f) * inv;
                    } else {
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            k[i] = rcp(1.f + ex2(v[h][i] * -1.44269504f));
                    }
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        k[i] = fmaxf(k[i] + bias[h][i], -INFINITY);
                    const float least = fminf(fminf(fminf(v[h][0], v[h][1]), fminf(v[h][2], v[h][3])), fminf(fminf(v[h][4], v[h][5]), fminf(v[h][6], v[h][7])));
                    if (least == -INFINITY)
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            k[i] = v[h][i] == -INFINITY ? -INFINITY : k[i];
                }
                if (bad)
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        k[i] = -INFINITY;
                float best, next = 0.f;
                if (two)
                    two_of(k, best, next);
                else
                    best = max8(k);
                if (piece < pieces) {
                    float4 *to = (float4 *)(keys + r * pitch + piece * 8);
                    to[0] = make_float4(k[0], k[1], k[2], k[3]);
                    to[1] = make_float4(k[4], k[5], k[6], k[7]);
                }
                { // -inf where there is none
                    first[r * pp + piece] = best;
                    if (kept_second)
                        second[r * pp + piece] = next;
                }
                if (c.groups > 1 && coming) { // over the lanes of a group
                    for (int o = 1; o < group_pieces; o *= 2) {
                        const float a = __shfl_xor_sync(FULL, best, o);
                        if (two)
                            next = fmaxf(fminf(best, a), fmaxf(next, __shfl_xor_sync(FULL, next, o)));
                        best = fmaxf(best, a);
                    }
                    if (piece < pieces && (piece & (group_pieces - 1)) == 0) {
                        ranks[r * c.groups + (piece >> shift)] = two ? half_sum(best, next) : best;
                        sizes[r * c.groups + (piece >> shift)] = two ? half_sum(fabsf(best), fabsf(next)) : fabsf(best);
                    }
                }
            }
        }
    }
    __syncwarp();

    // L lanes a row from here on
    const int r = lane / L, l = lane % L;
    const int64_t t = t0 + r;
    float *my_keys = keys + r * pitch, *my_first = first + r * pp, *my_second = second + r * pp, *my_ranks = ranks + r * c.groups, *my_sizes = sizes + r * c.groups, *my_chosen = chosen + r * slots;
    int *my_id = chosen_id + r * slots;
    const float unit = !by_logit && softmax ? row_inv[r] * 0x1p-18f : 0x1p-19f; // two scores are off by less together
    const auto near = [&](float a, float b) { return !(a - b > unit + 0x1p-22f * (fabsf(a) + fabsf(b))); };
    bool unsure = false;
    unsigned dropped = 0; // groups whose experts are not to be taken
    if (c.groups > 1) {
        if (!coming) {
            for (int g = l; g < c.groups; g += L) {
                float best = -INFINITY, next = -INFINITY;
                const auto take = [&](float k) {
                    next = fmaxf(next, fminf(best, k));
                    best = fmaxf(best, k);
                };
                if (per % 8 == 0) { // a group is whole pieces
                    for (int i = g * group_pieces; i < (g + 1) * group_pieces; ++i) {
                        if (two)
                            next = fmaxf(next, my_second[i]);
                        take(my_first[i]);
                    }
                } else {
                    for (int e = g * per; e < (g + 1) * per; ++e)
                        take(my_keys[e]);
                }
                my_ranks[g] = two ? half_sum(best, next) : best;
                my_sizes[g] = two ? half_sum(fabsf(best), fabsf(next)) : fabsf(best);
            }
            __syncwarp();
        }
        float worst_kept = INFINITY, best_left = -INFINITY; // as far down and up as they may be: scores, and the roundings of keys and sum
        for (int g = l; g < c.groups; g += L) {
            const float mine = my_ranks[g];
            int before = 0;
            for (int h = 0; h < c.groups; ++h) {
                const float other = my_ranks[h];
                before += other > mine || (other == mine && h < g) ? 1 : 0;
            }
            const float off = mine < INFINITY ? 0.5f * unit + 0x1p-21f * my_sizes[g] : 0.f;
            if (before < c.kept && mine > -INFINITY) {
                worst_kept = fminf(worst_kept, mine - off);
            } else {
                best_left = mine > -INFINITY ? fmaxf(best_left, mine + off) : best_left;
                dropped |= 1u << g;
            }
        }
        worst_kept = -max_over(-worst_kept, L), best_left = max_over(best_left, L);
#pragma unroll
        for (int o = L / 2; o > 0; o >>= 1)
            dropped |= __shfl_xor_sync(FULL, dropped, o);
        unsure = !by_logit && best_left > -INFINITY && !(worst_kept > best_left);
        if (per % 8) { // pieces across groups: what is left of them
            for (int i = l; i < pieces; i += L) {
                float best = -INFINITY;
                for (int e = i * 8; e < min(E, i * 8 + 8); ++e) {
                    if (dropped >> (e / per) & 1)
                        my_keys[e] = -INFINITY;
                    best = fmaxf(best, my_keys[e]);
                }
                my_first[i] = best;
            }
            dropped = 0;
        }
        __syncwarp();
    }
    float held[NB];
#pragma unroll
    for (int i = 0; i < NB; ++i) {
        const int piece = l * NB + i; // neighbours
        held[i] = my_first[piece];
        if (dropped) {
            const int g = coming ? piece >> shift : piece / group_pieces;
            held[i] = piece < pieces && (dropped >> g & 1) ? -INFINITY : held[i];
        }
    }
    const int rounds = p.selected + (by_logit ? 0 : 1); // the first key that is not chosen, for its distance
#pragma unroll 1
    for (int j = 0; j < rounds; ++j) {
        float mine = held[0];
#pragma unroll
        for (int i = 1; i < NB; ++i)
            mine = fmaxf(mine, held[i]);
        const float best = max_over(mine, L);
        // the first lane with this key, and the first of its pieces
        const int owner = __ffs(__ballot_sync(FULL, mine == best) >> (lane & ~(L - 1)) & ((1u << L) - 1)) - 1;
        int at_i = 0;
#pragma unroll
        for (int i = NB - 1; i >= 0; --i)
            at_i = held[i] == best ? i : at_i;
        at_i = __shfl_sync(FULL, at_i, owner, L);
        const int piece = owner * NB + at_i;
        const bool found = best > -INFINITY;
        // the lanes look at the piece together: its first element with this key, and the largest of the others
        constexpr int EACH = 8 / L;
        float k[EACH];
        int i0 = 8;
#pragma unroll
        for (int i = 0; i < EACH; ++i)
            k[i] = my_keys[piece * 8 + l * EACH + i];
        if constexpr (EACH == 1) {
            i0 = __ffs(__ballot_sync(FULL, k[0] == best) >> (lane & ~(L - 1)) & ((1u << L) - 1)) - 1;
        } else {
#pragma unroll
            for (int i = EACH - 1; i >= 0; --i)
                i0 = k[i] == best ? l * EACH + i : i0;
#pragma unroll
            for (int o = L / 2; o > 0; o >>= 1)
                i0 = min(i0, __shfl_xor_sync(FULL, i0, o));
        }
        float rest = -INFINITY;
#pragma unroll
        for (int i = 0; i < EACH; ++i)
            rest = l * EACH + i == i0 ? rest : fmaxf(rest, k[i]);
        rest = max_over(rest, L);
        if (found && l == owner) {
#pragma unroll
            for (int i = 0; i < NB; ++i)
                held[i] = i == at_i ? rest : held[i];
            my_keys[piece * 8 + i0] = -INFINITY;
        }
        if (l == 0)
            my_id[j] = found ? piece * 8 + i0 : -1, my_chosen[j] = best;
        __syncwarp(); // the key is gone for all lanes
    }
    __syncwarp();

    // weights: a lane has every L-th choice
    const bool here = t < p.T;
    const T *row = logits + t * ld;
    constexpr int MINE = MOE_ROUTE_MAX_SELECTED / L;
    float v[MINE], top = -INFINITY, total = 0.f;
#pragma unroll
    for (int i = 0; i < MINE; ++i) {
        const int j = i * L + l, id = here && j < p.selected ? my_id[j] : -1;
        v[i] = id >= 0 ? widen(row[id]) : -INFINITY;
        top = fmaxf(top, softmax ? v[i] : fminf(v[i], 0.f));
        if (!by_logit && id >= 0) {
            const int next = my_id[j + 1];
            if (next >= 0 && near(my_chosen[j], my_chosen[j + 1])) // equal logits and biases are equal keys, whose order is known
                unsure |= j == p.selected - 1 || v[i] != widen(row[next]) || (c.bias && c.bias[id] != c.bias[next]);
        }
        if (i * L + L >= p.selected)
            break;
    }
    top = max_over(top, L);
    const float ref = p.renormalize ? top : softmax ? row_max[r] : 0.f;
#pragma unroll
    for (int i = 0; i < MINE; ++i) {
        // sigmoid(v) = exp(min(v, 0)) / (1 + exp(-|v|)): nothing underflows that matters to a quotient
        const float w = softmax ? ex2((v[i] - ref) * 1.44269504f) : ex2((fminf(v[i], 0.f) - ref) * 1.44269504f) * rcp(1.f + ex2(fabsf(v[i]) * -1.44269504f));
        v[i] = v[i] > -INFINITY ? w : 0.f;
        total += v[i];
        if (i * L + L >= p.selected)
            break;
    }
    total = sum_over(total, L);
    const float factor = p.scale * (p.renormalize ? (total > 0.f ? 1.f / total : 0.f) : softmax ? row_inv[r] : 1.f);
#pragma unroll
    for (int i = 0; i < MINE; ++i) {
        const int j = i * L + l;
        if (here && j < p.selected) {
            ids[t * p.selected + j] = my_id[j];
            weights[t * p.selected + j] = v[i] > 0.f ? v[i] * factor : 0.f;
        }
        if (i * L + L >= p.selected)
            break;
    }
    unsigned again = __ballot_sync(FULL, unsure && here);
    while (again) {
        const int i = (__ffs(again) - 1) / L;
        again &= ~(((1u << L) - 1) << (L * i));
        __syncwarp();
        route_row_exactly(logits + (t0 + i) * ld, p, c, (double *)keys, ids + (t0 + i) * p.selected, weights + (t0 + i) * p.selected);
    }
}

// Gradients of a warp's rows are put together in shared memory, zeros but for the choices, and leave a row at a time in pieces of 8 columns a lane; with a softmax
// over all experts (DENSE) every column has its share, of logits that stay in registers from the softmax to there.  L, NB: as above.
__host__ __device__ constexpr int backward_words(int rows, int pieces) { return rows * (key_pitch(pieces) + 3) / 4 * 4 + 4; }
template <class T, int L, int NB, bool DENSE>
__global__ void __launch_bounds__(THREADS) route_backward_kernel(const T *__restrict__ logits, int64_t ld, bool vec, const RouteShape p,
                                                                 const uint8_t *__restrict__ mask, const int *__restrict__ ids,
                                                                 const float *__restrict__ dweights, T *dlogits, int64_t ld_d, bool vec_d, bool add)
{
    grid_dep_wait();
    constexpr int ROWS = 32 / L, MOST = L * NB, WIDTH = MOST >= 32 ? 32 : MOST, HELD = MOST / WIDTH, PASSES = ROWS * WIDTH / 32;
    extern __shared__ __align__(16) float route_smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, E = p.E, pieces = (E + 7) / 8, pitch = key_pitch(pieces);
    float *grads = route_smem + warp * backward_words(ROWS, pieces), *row_max = grads + ROWS * pitch, *row_inv = row_max + ROWS, *row_dot = row_inv + ROWS;
    const int64_t t0 = ((int64_t)blockIdx.x * (THREADS / 32) + warp) * ROWS;
    if (t0 >= p.T)
        return;
    const bool softmax = p.score == TS2_SCORE_SOFTMAX;
    const int at = lane & (WIDTH - 1), sub = lane / WIDTH;

    Eight<T> raw[DENSE ? PASSES : 1][DENSE ? HELD : 1];
    if constexpr (DENSE) {
#pragma unroll
        for (int s = 0; s < PASSES; ++s) {
            const int64_t t = t0 + s * (32 / WIDTH) + sub;
            const bool on = t < p.T && (!mask || mask[t]);
#pragma unroll
            for (int h = 0; h < HELD; ++h)
                raw[s][h].load(logits + t * ld, (at + 32 * h) * 8, E, vec, on && at + 32 * h < pieces);
        }
    }
    for (int i = lane; i < ROWS * pitch / 4; i += 32)
        ((float4 *)grads)[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    if constexpr (DENSE) {
#pragma unroll
        for (int s = 0; s < PASSES; ++s) {
            float v[8], top = -INFINITY, sum = 0.f;
#pragma unroll
            for (int h = 0; h < HELD; ++h) {
                raw[s][h].widen_to(v);
                top = fmaxf(top, max8(v));
            }
            top = max_over(top, WIDTH);
            top = top == -INFINITY ? 0.f : top;
#pragma unroll
            for (int h = 0; h < HELD; ++h) {
                raw[s][h].widen_to(v);
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    sum += ex2((v[i] - top) * 1.44269504f);
            }
            sum = sum_over(sum, WIDTH);
            const int r = s * (32 / WIDTH) + sub;
            if (at == 0)
                row_max[r] = top, row_inv[r] = 1.f / sum;
        }
    }
    __syncwarp();

    { // the gradients of the choices' logits over scale; L lanes a row, every L-th choice each
        const int r = lane / L, l = lane % L;
        const int64_t t = t0 + r;
        const bool here = t < p.T && (!mask || mask[t]);
        const T *row = logits + t * ld;
        constexpr int MINE = MOE_ROUTE_MAX_SELECTED / L;
        int id[MINE];
        float v[MINE], d[MINE], top = -INFINITY, total = 0.f, dot = 0.f;
#pragma unroll
        for (int i = 0; i < MINE; ++i) {
            const int j = i * L + l;
            id[i] = here && j < p.selected ? ids[t * p.selected + j] : -1;
            if (id[i] >= E)
                id[i] = -1;
            v[i] = 0.f, d[i] = 0.f;
            if (id[i] >= 0)
                v[i] = widen(row[id[i]]), d[i] = dweights[t * p.selected + j], top = fmaxf(top, softmax ? v[i] : fminf(v[i], 0.f));
            if (i * L + L >= p.selected)
                break;
        }
        if (p.renormalize)
            top = max_over(top, L);
        const float ref = p.renormalize ? top : softmax ? row_max[r] : 0.f;
        float w[MINE];
#pragma unroll
        for (int i = 0; i < MINE; ++i) {
            w[i] = softmax ? ex2((v[i] - ref) * 1.44269504f) : ex2((fminf(v[i], 0.f) - ref) * 1.44269504f) * rcp(1.f + ex2(fabsf(v[i]) * -1.44269504f));
            w[i] = id[i] >= 0 ? w[i] : 0.f;
            total += w[i], dot = fmaf(w[i], d[i], dot);
            if (i * L + L >= p.selected)
                break;
        }
        total = sum_over(total, L), dot = sum_over(dot, L);
        const bool any = total > 0.f; // a choice was made (or weighs nothing)
        const float factor = p.renormalize ? (any ? 1.f / total : 0.f) : softmax ? row_inv[r] : 1.f;
        dot = any ? dot * factor : 0.f;
        if (l == 0)
            row_dot[r] = dot;
#pragma unroll
        for (int i = 0; i < MINE; ++i) {
            // 1 - sigmoid(v) = sigmoid(-v), without cancellation
            const float rest = softmax ? 1.f : ex2(fmaxf(v[i], 0.f) * -1.44269504f) * rcp(1.f + ex2(fabsf(v[i]) * -1.44269504f));
            const float g = w[i] * factor * (p.renormalize ? d[i] - dot : d[i]) * rest;
            // one lane after the other: a caller's ids may name an expert twice
#pragma unroll
            for (int k = 0; k < L; ++k) {
                if (l == k && id[i] >= 0)
                    grads[r * pitch + id[i]] += g;
                __syncwarp();
            }
            if (i * L + L >= p.selected)
                break;
        }
    }
    __syncwarp();

#pragma unroll
    for (int s = 0; s < PASSES; ++s) {
        const int r = s * (32 / WIDTH) + sub;
        const int64_t t = t0 + r;
        if (t >= p.T)
            continue;
        const float ref = DENSE ? row_max[r] : 0.f, share = DENSE && row_dot[r] != 0.f ? row_dot[r] * row_inv[r] : 0.f;
#pragma unroll
        for (int h = 0; h < HELD; ++h) {
            const int i = at + 32 * h;
            if (i >= pieces)
                continue;
            const float4 a = *(const float4 *)(grads + r * pitch + i * 8), b = *(const float4 *)(grads + r * pitch + i * 8 + 4);
            float v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
            if (DENSE && share != 0.f) {
                float x[8];
                raw[DENSE ? s : 0][DENSE ? h : 0].widen_to(x);
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    v[k] = fmaf(-share, ex2((x[k] - ref) * 1.44269504f), v[k]);
            }
            T *to = dlogits + t * ld_d + i * 8;
            const bool whole = vec_d && i * 8 + 8 <= E;
            constexpr int PER = 16 / sizeof(T);
#pragma unroll
            for (int j = 0; j < 8 / PER; ++j) {
                Piece<T, PER> q;
                if (add) {
                    if (whole)
                        q = *(const Piece<T, PER> *)(to + j * PER);
                    else
#pragma unroll
                        for (int k = 0; k < PER; ++k)
                            if (i * 8 + j * PER + k < E)
                                q.v[k] = to[j * PER + k];
                }
#pragma unroll
                for (int k = 0; k < PER; ++k)
                    q.v[k] = narrow<T>(add ? fmaf(p.scale, v[j * PER + k], widen(q.v[k])) : p.scale * v[j * PER + k]);
                if (whole)
                    *(Piece<T, PER> *)(to + j * PER) = q;
                else
#pragma unroll
                    for (int k = 0; k < PER; ++k)
                        if (i * 8 + j * PER + k < E)
                            to[j * PER + k] = q.v[k];
            }
        }
    }
}

// ---- host ------------------------------------------------------------------------------------------------------------
template <class T, int L, int NB>
static int forward(const Ctx &c, const RouteShape &s, const void *logits, int64_t ld, const Choice &choice, const uint8_t *mask, int *ids, float *weights)
{
    const int warps = THREADS / 32;
    constexpr int most = warps * warp_words(32 / L, L * NB, L * NB, true, MOE_ROUTE_MAX_GROUPS, MOE_ROUTE_MAX_SELECTED) * 4;
    static_assert(most <= 232448, "shared memory budget");
    static std::atomic<unsigned> ready{0}; // a bit a device: it has been told how much shared memory the kernel takes
    const unsigned bit = 1u << (c.device & 15);
    if (!(ready.load() & bit)) {
        TS2_CUDA(cudaFuncSetAttribute((const void *)route_forward_kernel<T, L, NB>, cudaFuncAttributeMaxDynamicSharedMemorySize, most));
        ready.fetch_or(bit);
    }
    const bool vec = (uintptr_t)logits % 16 == 0 && ld * sizeof(T) % 16 == 0;
    const int per = s.E / choice.groups;
    const bool coming = L * NB <= 32 && per >= 8 && (per & (per - 1)) == 0; // as in the kernel
    const size_t smem = (size_t)warps * warp_words(32 / L, (s.E + 7) / 8, L * NB, choice.groups > 1 && choice.group_top == 2 && !coming, choice.groups, s.selected) * 4;
    TS2_LAUNCH((route_forward_kernel<T, L, NB>), (unsigned)ceil_div(s.T, warps * (32 / L)), THREADS, smem, c.stream, (const T *)logits, ld, vec, s, choice, mask, ids,
               weights);
    return TS2_OK;
}
template <class T>
static int forward(const Ctx &c, const RouteShape &s, const void *logits, int64_t ld, const Choice &choice, const uint8_t *mask, int *ids, float *weights)
{
    // 4 lanes a row take fewer instructions, 8 two times the warps.  Up to 128 experts 4 are faster (65537 x 128 18.3 against 20.9 us), beyond 8 (32768 x 256
    // in groups 35.6 against 39.2); for the gradient, whose row has little to do, 8 are from 33 experts on (65537 x 128 22.8 against 27.4, 32768 x 256 8.9
    // against 10.4).
    const auto f = s.E <= 32    ? forward<T, 4, 1>
                   : s.E <= 64  ? forward<T, 4, 2>
                   : s.E <= 128 ? forward<T, 4, 4>
                   : s.E <= 256 ? forward<T, 8, 4>
                   : s.E <= 512 ? forward<T, 8, 8>
                                : forward<T, 8, 16>;
    return f(c, s, logits, ld, choice, mask, ids, weights);
}
template <class T, int L, int NB, bool DENSE>
static int backward(const Ctx &c, const RouteShape &s, const void *logits, int64_t ld, const uint8_t *mask, const int *ids, const float *dweights,
                    void *dlogits, int64_t ld_d, bool add)
{
    const int warps = THREADS / 32;
    static std::atomic<unsigned> ready{0}; // as above
    const unsigned bit = 1u << (c.device & 15);
    if (!(ready.load() & bit)) {
        TS2_CUDA(cudaFuncSetAttribute((const void *)route_backward_kernel<T, L, NB, DENSE>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      warps * backward_words(32 / L, L * NB) * 4));
        ready.fetch_or(bit);
    }
    const auto aligned = [](const void *p, int64_t pitch) { return (uintptr_t)p % 16 == 0 && pitch * sizeof(T) % 16 == 0; };
    TS2_LAUNCH((route_backward_kernel<T, L, NB, DENSE>), (unsigned)ceil_div(s.T, warps * (32 / L)), THREADS, (size_t)warps * backward_words(32 / L, (s.E + 7) / 8) * 4, c.stream,
               (const T *)logits, ld, aligned(logits, ld), s, mask, ids, dweights, (T *)dlogits, ld_d, aligned(dlogits, ld_d), add);
    return TS2_OK;
}
template <class T, bool DENSE>
static int backward(const Ctx &c, const RouteShape &s, const void *logits, int64_t ld, const uint8_t *mask, const int *ids, const float *dweights,
                    void *dlogits, int64_t ld_d, bool add)
{
    const auto f = s.E <= 32    ? backward<T, 4, 1, DENSE>
                   : s.E <= 64  ? backward<T, 8, 1, DENSE>
                   : s.E <= 128 ? backward<T, 8, 2, DENSE>
                   : s.E <= 256 ? backward<T, 8, 4, DENSE>
                   : s.E <= 512 ? backward<T, 8, 8, DENSE>
                                : backward<T, 8, 16, DENSE>;
    return f(c, s, logits, ld, mask, ids, dweights, dlogits, ld_d, add);
}
template <class T>
static int backward(const Ctx &c, const RouteShape &s, const void *logits, int64_t ld, const uint8_t *mask, const int *ids, const float *dweights,
                    void *dlogits, int64_t ld_d, bool add)
{
    return s.score == TS2_SCORE_SOFTMAX && !s.renormalize ? backward<T, true>(c, s, logits, ld, mask, ids, dweights, dlogits, ld_d, add)
                                                          : backward<T, false>(c, s, logits, ld, mask, ids, dweights, dlogits, ld_d, add);
}

int moe_route_forward(const Ctx &c, const RouteShape &s, const void *logits, int64_t ld, const float *bias, int groups, int groups_kept, int group_top,
                      const uint8_t *mask, int *ids, float *weights)
{
    if (s.T == 0)
        return TS2_OK;
    const auto f = s.type == TS2_OUT_F32 ? forward<float> : s.type == TS2_OUT_F16 ? forward<__half> : forward<__nv_bfloat16>;
    return f(c, s, logits, ld, {bias, groups, groups_kept, group_top}, mask, ids, weights);
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
