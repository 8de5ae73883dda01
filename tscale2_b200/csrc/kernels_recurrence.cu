// The gated linear recurrence over packed sequences and its backward pass: per channel and sequence
//     h[t] = a[t] h[t-1] + (1 - a[t]) x[t],   a = 1 / (1 + exp(-gate)),   h before the first node: h0 or zero
//     e[t] = dh[t] + a[t+1] e[t+1] (dh_last beyond the last node),   dx = (1 - a) e,   dgate = a (1 - a) (h[t-1] - x) e,   dh0 = a e
// The decay is held as a logit: 16 bits are too coarse for a decay next to one, and 1 - a comes from the logit without
// cancellation.  States and decays are fp32 in registers, whatever the type of the arrays.
//
// A recurrence of this form is a scan over maps h -> A h + B, which compose; so the nodes are cut into groups of S consecutive
// ones.  A warp owns a group of 64 channels (two a lane), folds it into one map in registers, leaves the map in shared memory,
// and once the maps of the groups before it are there goes over its registers again with the state that enters the group.
// gate and x are read once and h is written once: memory bandwidth is the bound.  The order of every sum is fixed.
#include "kernels.cuh"

namespace ts2 {

static constexpr int WARPS = 8;
static constexpr int THREADS = WARPS * 32;
static constexpr int STRIP = 64; // channels a block carries through time, two a lane

// ---- two neighbouring channels as they lie in memory -----------------------------------------------------------------
template <class T>
struct Two;
template <>
struct Two<float> {
    using Raw = float2;
    static __device__ __forceinline__ float2 get(Raw r) { return r; }
    static __device__ __forceinline__ Raw put(float2 v) { return v; }
    static __device__ __forceinline__ Raw join(float a, float b) { return make_float2(a, b); }
};
template <>
struct Two<__half> {
    using Raw = __half2;
    static __device__ __forceinline__ float2 get(Raw r) { return __half22float2(r); }
    static __device__ __forceinline__ Raw put(float2 v) { return sat_half2(v.x, v.y); }
    static __device__ __forceinline__ Raw join(__half a, __half b) { return __halves2half2(a, b); }
};
template <>
struct Two<__nv_bfloat16> {
    using Raw = __nv_bfloat162;
    static __device__ __forceinline__ float2 get(Raw r) { return __bfloat1622float2(r); }
    static __device__ __forceinline__ Raw put(float2 v) { return __float22bfloat162_rn(v); }
    static __device__ __forceinline__ Raw join(__nv_bfloat16 a, __nv_bfloat16 b) { return __halves2bfloat162(a, b); }
};

// VEC: pairs are aligned, so that one access takes both channels; else one access each.  n: how many of the two exist
template <class T, bool VEC>
__device__ __forceinline__ typename Two<T>::Raw load_two(const T *p, int n)
{
    if (VEC)
        return n ? *(const typename Two<T>::Raw *)p : Two<T>::put(make_float2(0.f, 0.f));
    const T zero = T(0.f);
    return Two<T>::join(n > 0 ? p[0] : zero, n > 1 ? p[1] : zero);
}
template <class T, bool VEC>
__device__ __forceinline__ void store_two(T *p, int n, float2 v)
{
    const typename Two<T>::Raw r = Two<T>::put(v);
    if (VEC) {
        if (n)
            *(typename Two<T>::Raw *)p = r;
    } else {
        if (n > 0)
            p[0] = r.x;
        if (n > 1)
            p[1] = r.y;
    }
}
__device__ __forceinline__ float2 load_state(const float *p, int n) { return make_float2(n > 0 ? p[0] : 0.f, n > 1 ? p[1] : 0.f); }
__device__ __forceinline__ void store_state(float *p, int n, float2 v)
{
    if (n > 0)
        p[0] = v.x;
    if (n > 1)
        p[1] = v.y;
}

// a = 1 / (1 + exp(-g)) and 1 - a, each to fp32's relative accuracy.  The exponent stops at 126, where a is 1e-38 and 1 - a is
// 1: beyond it exp(-g) would be infinite and 1 - a = exp(-g) a not a number.  A NaN stays one.
__device__ __forceinline__ void decay(float g, float &a, float &keep)
{
    float t = -1.4426950408889634f * g;
    asm("min.NaN.f32 %0, %0, 0f42FC0000;" : "+f"(t)); // 126
    float e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
    a = r;
    keep = e * r;
}

// ---- where sequences start and end -----------------------------------------------------------------------------------
// number of entries ptr[0 .. n) that lie below t (ptr ascending), by the whole warp: 32 probes a round
__device__ __forceinline__ int entries_below(const int *__restrict__ ptr, int n, int t)
{
    const int lane = threadIdx.x & 31;
    int lo = 0, hi = n; // the answer lies in [lo, hi]
    while (hi > lo) {
        const int step = (hi - lo + 31) / 32;
        const long long at = (long long)lo + (long long)(lane + 1) * step - 1;
        const int below = __popc(__ballot_sync(0xffffffffu, at < hi && ptr[at] < t));
        const long long from = (long long)lo + (long long)below * step;
        if (step == 1)
            return (int)(from < hi ? from : hi);
        lo = (int)(from < hi ? from : hi);
        hi = (int)min((long long)hi, from + step - 1);
    }
    return lo;
}

// The borders among the nodes [t0, t0 + S) that lie in [begin, end), S <= 16: bit s of starts: a sequence starts at node t0 + s;
// of ends: one ends there
struct Borders {
    unsigned starts, ends;
};
template <int S>
__device__ __forceinline__ Borders find_borders(const int *__restrict__ ptr, int n_ptr, int t0, int begin, int end)
{
    const int lane = threadIdx.x & 31;
    unsigned at = 0; // bit s: some sequence starts at t0 + s, another ends before it
    if (ptr) {
        for (int i = entries_below(ptr, n_ptr, t0); i < n_ptr; i += 32) { // once, but where more than 31 sequences are empty
            const int d = i + lane < n_ptr ? ptr[i + lane] - t0 : S + 1;
            at |= __reduce_or_sync(0xffffffffu, d >= 0 && d <= S ? 1u << d : 0u);
            if (__any_sync(0xffffffffu, d > S))
                break;
        }
    } else {
        at = (begin >= t0 && begin <= t0 + S ? 1u << (begin - t0) : 0u) | (end >= t0 && end <= t0 + S ? 1u << (end - t0) : 0u);
    }
    unsigned in = (1u << S) - 1; // nodes of the range
    if (t0 + S > end)
        in &= t0 < end ? (1u << (end - t0)) - 1 : 0u;
    if (t0 < begin)
        in = t0 + S > begin ? in & ~((1u << (begin - t0)) - 1) : 0u;
    return {at & in, at >> 1 & in};
}
// the sequence that holds node t (whole warp)
__device__ __forceinline__ int sequence_of(const int *__restrict__ ptr, int n_seq, int t)
{
    if (!ptr)
        return 0;
    return max(0, min(n_seq - 1, entries_below(ptr, n_seq + 1, t + 1) - 1));
}

struct ScanArgs {
    const void *gate, *x;
    long long gate_ld, x_ld;
    int T, D, n_seq;
    const int *ptr; // null: one sequence over all T nodes
    const float *h0;
    // forward
    void *h;
    long long h_ld;
    float *h_last;
    // backward: h is read
    const void *dh;
    long long dh_ld;
    const float *dh_last;
    void *dgate, *dx;
    long long dgate_ld, dx_ld;
    float *dh0;
};

// nodes [begin, end) that belong to a sequence; a table that does not ascend inside [0, T] changes which, not that they lie in [0, T)
__device__ __forceinline__ void scan_range(const ScanArgs &p, int &begin, int &end)
{
    begin = 0, end = p.T;
    if (p.ptr) {
        begin = max(0, min(p.T, p.ptr[0]));
        end = max(begin, min(p.T, p.ptr[p.n_seq]));
    }
}
// what an empty sequence passes on: its state before is its state after (and the same of the gradients)
__device__ __forceinline__ void pass_empty(const ScanArgs &p, const float *from, float *to, int c0, int n)
{
    const int lane = threadIdx.x & 31;
    if (!to || !p.ptr) {
        if (to && p.T == 0)
            store_state(to + c0, n, from ? load_state(from + c0, n) : make_float2(0.f, 0.f));
        return;
    }
    for (int s0 = 32 * (threadIdx.x >> 5); s0 < p.n_seq; s0 += THREADS) {
        const int s = s0 + lane;
        unsigned m = __ballot_sync(0xffffffffu, s < p.n_seq && p.ptr[s + 1] <= p.ptr[s]);
        for (; m; m &= m - 1) {
            const size_t at = (size_t)(s0 + __ffs(m) - 1) * p.D + c0;
            store_state(to + at, n, from ? load_state(from + at, n) : make_float2(0.f, 0.f));
        }
    }
}

// a map h -> A h + B of two channels; cut: a sequence starts inside, what was before has no part in it (A is not used then:
// zero times an infinity of the sequence before would be a NaN of this one)
__device__ __forceinline__ float2 apply(float4 map, bool cut, float2 h)
{
    return cut ? make_float2(map.z, map.w) : make_float2(fmaf(map.x, h.x, map.z), fmaf(map.y, h.y, map.w));
}

// One block carries 64 channels through all nodes, WARPS * S of them at a time.  The next tile's values are on their way while
// this one's are worked on.
template <class T, int S, bool VEC>
__global__ void __launch_bounds__(THREADS, 2) recurrence_forward_kernel(const ScanArgs p)
{
    grid_dep_wait();
    __shared__ float4 maps[2][WARPS][32];
    __shared__ int cuts[2][WARPS];
    using Raw = typename Two<T>::Raw;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int c0 = blockIdx.x * STRIP + 2 * lane, n = max(0, min(2, p.D - c0));
    const T *gate = (const T *)p.gate + c0, *x = (const T *)p.x + c0;
    T *h_out = (T *)p.h + c0;
    pass_empty(p, p.h0, p.h_last, c0, n);
    int begin, end;
    scan_range(p, begin, end);

    Raw rg[S], rx[S];
    auto fetch = [&](int t0) {
#pragma unroll
        for (int s = 0; s < S; ++s) {
            const int m = t0 + s < end ? n : 0;
            rg[s] = load_two<T, VEC>(gate + (t0 + s) * p.gate_ld, m);
            rx[s] = load_two<T, VEC>(x + (t0 + s) * p.x_ld, m);
        }
    };
    float2 state = make_float2(0.f, 0.f); // behind the tiles so far, the same in every warp
    int t0 = begin + warp * S, buf = 0;
    fetch(t0);
    for (int base = begin; base < end; base += WARPS * S, t0 += WARPS * S, buf ^= 1) {
        const Borders b = find_borders<S>(p.ptr, p.n_seq + 1, t0, begin, end);
        float2 a[S], u[S];
        float4 map = make_float4(1.f, 1.f, 0.f, 0.f);
#pragma unroll
        for (int s = 0; s < S; ++s) {
            const float2 g = Two<T>::get(rg[s]), v = Two<T>::get(rx[s]);
            float k0, k1;
            decay(g.x, a[s].x, k0);
            decay(g.y, a[s].y, k1);
            u[s] = make_float2(k0 * v.x, k1 * v.y);
            if (t0 + s >= end)
                a[s] = make_float2(1.f, 1.f), u[s] = make_float2(0.f, 0.f);
            if (b.starts >> s & 1) {
                if (p.h0) {
                    const float2 h = load_state(p.h0 + (size_t)sequence_of(p.ptr, p.n_seq, t0 + s) * p.D + c0, n);
                    u[s].x = fmaf(a[s].x, h.x, u[s].x), u[s].y = fmaf(a[s].y, h.y, u[s].y);
                }
                map.z = u[s].x, map.w = u[s].y;
            } else {
                map.z = fmaf(a[s].x, map.z, u[s].x), map.w = fmaf(a[s].y, map.w, u[s].y);
            }
            map.x *= a[s].x, map.y *= a[s].y;
        }
        if (t0 + WARPS * S < end)
            fetch(t0 + WARPS * S);
        maps[buf][warp][lane] = map;
        if (lane == 0)
            cuts[buf][warp] = b.starts != 0;
        __syncthreads(); // once a tile: the other buffer's readers have passed it, too
        float2 h = make_float2(0.f, 0.f);
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            if (w == warp)
                h = state;
            state = apply(maps[buf][w][lane], cuts[buf][w], state);
        }
#pragma unroll
        for (int s = 0; s < S; ++s) {
            if (t0 + s >= end)
                break;
            if (b.starts >> s & 1)
                h = make_float2(u[s].x, u[s].y);
            else
                h = make_float2(fmaf(a[s].x, h.x, u[s].x), fmaf(a[s].y, h.y, u[s].y));
            store_two<T, VEC>(h_out + (t0 + s) * p.h_ld, n, h);
            if (p.h_last && (b.ends >> s & 1))
                store_state(p.h_last + (size_t)sequence_of(p.ptr, p.n_seq, t0 + s) * p.D + c0, n, h);
        }
    }
}

// The same from the last node to the first: what a node passes on is f[t] = a[t] e[t], e[t] = dh[t] + f[t+1], cut where a sequence ends
template <class T, int S, bool VEC>
__global__ void __launch_bounds__(THREADS, 2) recurrence_backward_kernel(const ScanArgs p)
{
    grid_dep_wait();
    __shared__ float4 maps[2][WARPS][32];
    __shared__ int cuts[2][WARPS];
    using Raw = typename Two<T>::Raw;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int c0 = blockIdx.x * STRIP + 2 * lane, n = max(0, min(2, p.D - c0));
    const T *gate = (const T *)p.gate + c0, *x = (const T *)p.x + c0, *h = (const T *)p.h + c0, *dh = (const T *)p.dh + c0;
    T *dgate = (T *)p.dgate + c0, *dx = (T *)p.dx + c0;
    pass_empty(p, p.dh_last, p.dh0, c0, n);
    int begin, end;
    scan_range(p, begin, end);

    Raw rg[S], rx[S], rh[S], rd[S];
    auto fetch = [&](int t0) { // the state before the group's first node is the last one of another group
#pragma unroll
        for (int s = 0; s < S; ++s) {
            const int t = t0 + s, m = t >= begin && t < end ? n : 0;
            rg[s] = load_two<T, VEC>(gate + t * p.gate_ld, m);
            rx[s] = load_two<T, VEC>(x + t * p.x_ld, m);
            rh[s] = load_two<T, VEC>(h + (t - 1) * p.h_ld, t > begin ? m : 0);
            rd[s] = load_two<T, VEC>(dh + t * p.dh_ld, m);
        }
    };
    float2 state = make_float2(0.f, 0.f); // what the tiles so far pass on
    int t0 = end - (warp + 1) * S, buf = 0;
    fetch(t0);
    for (int base = end; base > begin; base -= WARPS * S, t0 -= WARPS * S, buf ^= 1) {
        const Borders b = find_borders<S>(p.ptr, p.n_seq + 1, t0, begin, end);
        float2 a[S], k[S], d[S], w[S]; // w = h[t-1] - x[t]
        float4 map = make_float4(1.f, 1.f, 0.f, 0.f);
#pragma unroll
        for (int s = S - 1; s >= 0; --s) {
            const float2 g = Two<T>::get(rg[s]), v = Two<T>::get(rx[s]);
            float2 hb = Two<T>::get(rh[s]);
            d[s] = Two<T>::get(rd[s]);
            decay(g.x, a[s].x, k[s].x);
            decay(g.y, a[s].y, k[s].y);
            if (b.starts >> s & 1)
                hb = p.h0 ? load_state(p.h0 + (size_t)sequence_of(p.ptr, p.n_seq, t0 + s) * p.D + c0, n) : make_float2(0.f, 0.f);
            w[s] = make_float2(hb.x - v.x, hb.y - v.y);
            if (t0 + s < begin)
                a[s] = make_float2(1.f, 1.f), d[s] = make_float2(0.f, 0.f);
            if (b.ends >> s & 1) {
                if (p.dh_last) {
                    const float2 l = load_state(p.dh_last + (size_t)sequence_of(p.ptr, p.n_seq, t0 + s) * p.D + c0, n);
                    d[s].x += l.x, d[s].y += l.y;
                }
                map.z = a[s].x * d[s].x, map.w = a[s].y * d[s].y;
            } else {
                map.z = a[s].x * (map.z + d[s].x), map.w = a[s].y * (map.w + d[s].y);
            }
            map.x *= a[s].x, map.y *= a[s].y;
        }
        if (base - WARPS * S > begin)
            fetch(t0 - WARPS * S);
        maps[buf][warp][lane] = map;
        if (lane == 0)
            cuts[buf][warp] = b.ends != 0;
        __syncthreads();
        float2 f = make_float2(0.f, 0.f);
#pragma unroll
        for (int i = 0; i < WARPS; ++i) {
            if (i == warp)
                f = state;
            state = apply(maps[buf][i][lane], cuts[buf][i], state);
        }
#pragma unroll
        for (int s = S - 1; s >= 0; --s) {
            const int t = t0 + s;
            if (t < begin)
                break;
            const bool cut = b.ends >> s & 1;
            const float2 e = make_float2(cut ? d[s].x : d[s].x + f.x, cut ? d[s].y : d[s].y + f.y);
            f = make_float2(a[s].x * e.x, a[s].y * e.y);
            const float2 ke = make_float2(k[s].x * e.x, k[s].y * e.y);
            store_two<T, VEC>(dx + t * p.dx_ld, n, ke);
            store_two<T, VEC>(dgate + t * p.dgate_ld, n, make_float2(a[s].x * ke.x * w[s].x, a[s].y * ke.y * w[s].y));
            if (p.dh0 && (b.starts >> s & 1))
                store_state(p.dh0 + (size_t)sequence_of(p.ptr, p.n_seq, t) * p.D + c0, n, f);
        }
    }
}

template <class T, int S_FORWARD, int S_BACKWARD>
static int launch(const Ctx &c, const ScanArgs &p, bool backward, bool vec)
{
    const dim3 grid((unsigned)ceil_div(p.D, STRIP));
    if (backward) {
        if (vec)
            TS2_LAUNCH((recurrence_backward_kernel<T, S_BACKWARD, true>), grid, THREADS, 0, c.stream, p);
        else
            TS2_LAUNCH((recurrence_backward_kernel<T, S_BACKWARD, false>), grid, THREADS, 0, c.stream, p);
    } else {
        if (vec)
            TS2_LAUNCH((recurrence_forward_kernel<T, S_FORWARD, true>), grid, THREADS, 0, c.stream, p);
        else
            TS2_LAUNCH((recurrence_forward_kernel<T, S_FORWARD, false>), grid, THREADS, 0, c.stream, p);
    }
    return TS2_OK;
}

static int run(const Ctx &c, int type, const ScanArgs &p, bool backward)
{
    // both channels of a pair in one access: even pitches, bases aligned to a pair
    const uintptr_t pair = type == TS2_OUT_F32 ? 8 : 4;
    const long long odd = (p.gate_ld | p.x_ld | p.h_ld | p.D | (backward ? p.dh_ld | p.dgate_ld | p.dx_ld : 0)) & 1;
    const uintptr_t at = (uintptr_t)p.gate | (uintptr_t)p.x | (uintptr_t)p.h | (backward ? (uintptr_t)p.dh | (uintptr_t)p.dgate | (uintptr_t)p.dx : 0);
    const bool vec = !odd && at % pair == 0;
    switch (type) {
    case TS2_OUT_F32: return launch<float, 8, 4>(c, p, backward, vec);
    case TS2_OUT_F16: return launch<__half, 16, 8>(c, p, backward, vec);
    case TS2_OUT_BF16: return launch<__nv_bfloat16, 16, 8>(c, p, backward, vec);
    default: return fail(TS2_ERR_INVALID_ARG, "recurrence: unknown type %d", type);
    }
}

int recurrence_forward(const Ctx &c, int type, const void *gate, int64_t gate_ld, const void *x, int64_t x_ld, int T, int D, int n_seq,
                       const int *seq_ptr, const float *h0, void *h, int64_t h_ld, float *h_last)
{
    ScanArgs p = {};
    p.gate = gate, p.gate_ld = gate_ld, p.x = x, p.x_ld = x_ld, p.T = T, p.D = D, p.n_seq = n_seq, p.ptr = seq_ptr, p.h0 = h0;
    p.h = h, p.h_ld = h_ld, p.h_last = h_last;
    return run(c, type, p, false);
}

int recurrence_backward(const Ctx &c, int type, const void *gate, int64_t gate_ld, const void *x, int64_t x_ld, const void *h, int64_t h_ld,
                        int T, int D, int n_seq, const int *seq_ptr, const float *h0, const void *dh, int64_t dh_ld, const float *dh_last,
                        void *dgate, int64_t dgate_ld, void *dx, int64_t dx_ld, float *dh0)
{
    ScanArgs p = {};
    p.gate = gate, p.gate_ld = gate_ld, p.x = x, p.x_ld = x_ld, p.T = T, p.D = D, p.n_seq = n_seq, p.ptr = seq_ptr, p.h0 = h0;
    p.h = const_cast<void *>(h), p.h_ld = h_ld, p.dh = dh, p.dh_ld = dh_ld, p.dh_last = dh_last;
    p.dgate = dgate, p.dgate_ld = dgate_ld, p.dx = dx, p.dx_ld = dx_ld, p.dh0 = dh0;
    return run(c, type, p, true);
}

} // namespace ts2
