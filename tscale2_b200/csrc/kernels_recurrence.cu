// The gated linear recurrence over packed sequences and its backward pass: per channel and sequence
//     h[t] = a[t] h[t-1] + (1 - a[t]) x[t],   a = 1 / (1 + exp(-gate)),   h before the first node: h0 or zero
//     e[t] = dh[t] + a[t+1] e[t+1] (dh_last beyond the last node),   dx = (1 - a) e,   dgate = a (1 - a) (h[t-1] - x) e,   dh0 = a e
// The decay is held as a logit: 16 bits are too coarse for a decay next to one, and 1 - a comes from the logit without
// cancellation.  States and decays are fp32 in registers, whatever the type of the arrays.
//
// A recurrence of this form is a scan over maps h -> A h + B, which compose.  A block carries a strip of 64 channels (two a lane)
// through a segment of the nodes, a tile of them at a time: each of its warps folds a group of S consecutive nodes into one map in
// registers, leaves the map in shared memory, and once the maps of the groups before it are there goes over its registers again
// with the state that enters the group.  Long arrays are cut into segments that blocks work on side by side: a first launch finds
// what each segment does to the state that enters it, from the last start of a sequence in it on.  The bound is memory
// bandwidth (gate and x in, h out), for 16-bit arrays nearly the issue slots, too (23 instructions an element, two of them in
// the unit of exponentials and reciprocals).  The order of every sum is fixed.
#include "kernels.cuh"
#include <algorithm>
#include <climits>

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

// VEC: pairs are aligned, so that one access takes both channels; else one access each
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
// the channels of a lane: c0 and c0 + 1, n of which exist
struct Lane {
    int strip, c0, n;
    __device__ __forceinline__ explicit Lane(int D)
    {
        strip = blockIdx.y * STRIP;
        c0 = strip + 2 * (threadIdx.x & 31);
        n = max(0, min(2, D - c0));
    }
};
__device__ __forceinline__ float2 load_state(const float *p, int n) { return make_float2(n > 0 ? p[0] : 0.f, n > 1 ? p[1] : 0.f); }
__device__ __forceinline__ void store_state(float *p, int n, float2 v)
{
    if (n > 0)
        p[0] = v.x;
    if (n > 1)
        p[1] = v.y;
}

// both channels in one instruction
__device__ __forceinline__ float2 mul2(float2 a, float2 b)
{
    float2 r;
    asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b)
{
    float2 r;
    asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c)
{
    float2 r;
    asm("{\n\t.reg .b64 x, y, z, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\tfma.rn.f32x2 w, x, y, z;\n\t"
        "mov.b64 {%0, %1}, w;\n\t}"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return r;
}
// a = 1 / (1 + exp(-g)) and 1 - a, both with a small relative error (the product with log2 e is rounded: |g| 2^-24, and the three
// instructions' own) however near to one the other is.  The exponent stops at 126, where a is 1e-38 and 1 - a is 1: beyond it exp(-g)
// would be infinite and 1 - a = exp(-g) a not a number.  A NaN stays one.
__device__ __forceinline__ void decay(float2 g, float2 &a, float2 &keep)
{
    float2 e = mul2(g, make_float2(-1.4426950408889634f, -1.4426950408889634f));
    asm("min.NaN.f32 %0, %0, 0f42FC0000;" : "+f"(e.x)); // 126
    asm("min.NaN.f32 %0, %0, 0f42FC0000;" : "+f"(e.y));
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(e.x));
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(e.y));
    a = add2(e, make_float2(1.f, 1.f));
    asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(a.x));
    asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(a.y));
    keep = mul2(e, a);
}

// ---- where sequences start and end -----------------------------------------------------------------------------------
__device__ __forceinline__ int ceil_div_dev(int a, int b) { return (a + b - 1) / b; }
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

// The borders among the nodes [t0, t0 + S) that lie in the segment [lo, hi) of [begin, end), S <= 16: bit s of starts: a sequence starts at node t0 + s;
// of ends: one ends there.  below, above: the nearest entries of the table below t0 and above t0 + S: between them nothing has
// to be looked for again.
struct Borders {
    unsigned starts, ends;
    int below, above;
};
template <int S>
__device__ __forceinline__ Borders find_borders(const int *__restrict__ ptr, int n_ptr, int t0, int begin, int end, int lo, int hi)
{
    const int lane = threadIdx.x & 31;
    unsigned at = 0; // bit s: some sequence starts at t0 + s, another ends before it
    Borders b = {0u, 0u, -1, INT_MAX};
    if (ptr) {
        const int first = entries_below(ptr, n_ptr, t0);
        if (first > 0)
            b.below = ptr[first - 1];
        for (int i = first; i < n_ptr; i += 32) { // once, but where more than 31 sequences are empty
            const int v = i + lane < n_ptr ? ptr[i + lane] : INT_MAX;
            const bool inside = v >= t0 && v <= t0 + S;
            at |= __reduce_or_sync(0xffffffffu, inside ? 1u << (v - t0) : 0u);
            if (__any_sync(0xffffffffu, v > t0 + S)) {
                b.above = __reduce_min_sync(0xffffffffu, v > t0 + S ? v : INT_MAX);
                break;
            }
        }
    } else {
        at = (begin >= t0 && begin <= t0 + S ? 1u << (begin - t0) : 0u) | (end >= t0 && end <= t0 + S ? 1u << (end - t0) : 0u);
        b.below = begin < t0 ? begin : -1, b.above = end > t0 + S ? end : INT_MAX;
    }
    unsigned in = (1u << S) - 1; // nodes of the segment
    if (t0 + S > hi)
        in &= t0 < hi ? (1u << (hi - t0)) - 1 : 0u;
    if (t0 < lo)
        in = t0 + S > lo ? in & ~((1u << (lo - t0)) - 1) : 0u;
    b.starts = at & in, b.ends = at >> 1 & in;
    return b;
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
    int gate_ld, x_ld;
    int T, D, n_seq;
    const int *ptr; // null: one sequence over all T nodes
    const float *h0;
    // forward
    void *h;
    int h_ld;
    float *h_last;
    // backward: h is read
    const void *dh;
    int dh_ld;
    const float *dh_last;
    void *dgate, *dx;
    int dgate_ld, dx_ld;
    float *dh0;
    int segments, subs; // parts of the nodes that blocks work on side by side; parts of a segment of which each has a map
    float4 *maps;       // [strips][segments][subs][32]: what a part does to the state that enters it
};

// nodes [begin, end) that belong to a sequence.  A table that does not ascend inside [0, T] changes which nodes these are, not
// that they lie in [0, T).
__device__ __forceinline__ void scan_range(const ScanArgs &p, int &begin, int &end)
{
    begin = 0, end = p.T;
    if (p.ptr) {
        begin = max(0, min(p.T, p.ptr[0]));
        end = max(begin, min(p.T, p.ptr[p.n_seq]));
    }
}
// of those, the first one of segment k
__device__ __forceinline__ int segment_start(const ScanArgs &p, int k, int begin, int end)
{
    return begin + (int)((long long)(end - begin) * k / p.segments);
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

// ---- tiles on their way in -------------------------------------------------------------------------------------------
// One row range of an array, as a lane's copies see it
template <class T>
struct Source {
    const T *base; // the strip's first channel
    int ld, shift; // rows t + shift
};
// A warp's group of the next tiles, S rows of N arrays each.  COPY bytes at a time go by cp.async into STAGES slots of shared memory
// that are the warp's own, so that it waits for nobody else's copies; a row out of [begin, end) is another row of it.
// COPY < a pair (16-bit arrays without the alignment): the values of one tile ahead wait in registers.
// No branches between the loads: with a branch each load waited for the one before (65536 x 768 bf16: 400 us, without 114).
template <class T, int S, int N, int COPY>
struct Feed {
    static constexpr int STAGES = 3, ROW = STRIP * sizeof(T), GROUP = S * N * ROW, BYTES = STAGES * WARPS * GROUP;
    uint32_t at; // shared memory: the warp's slot of stage 0
    int lane;
    __device__ __forceinline__ Feed(uint8_t *smem) : at(smem_u32(smem) + (threadIdx.x >> 5) * GROUP), lane(threadIdx.x & 31) {}
    __device__ __forceinline__ uint32_t slot(int stage) const { return at + stage * (WARPS * GROUP); }
    static __device__ __forceinline__ void copy(uint32_t to, const T *from)
    {
        if constexpr (COPY == 16)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
        else
            asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(to), "l"(from), "n"(COPY) : "memory");
    }
    __device__ __forceinline__ void issue(int stage, const Source<T> (&src)[N], int t0, int begin, int end, int channels)
    {
        constexpr int PER_ROW = ROW / COPY, ROWS = PER_ROW >= 32 ? 1 : 32 / PER_ROW, REST = PER_ROW >= 32 ? PER_ROW / 32 : 1;
        const int r0 = lane / PER_ROW, c0 = (lane % PER_ROW) * (COPY / (int)sizeof(T));
        const uint32_t to = slot(stage) + r0 * ROW + c0 * (int)sizeof(T);
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int k = 0; k < REST; ++k) {
                const int c = c0 + 32 * k * (COPY / (int)sizeof(T)), first = t0 + r0 + src[i].shift;
                const T *column = src[i].base + (c < channels ? c : 0);
#pragma unroll
                for (int s = 0; s < S; s += ROWS)
                    copy(to + (i * S + s) * ROW + 32 * k * COPY, column + (long long)max(begin, min(first + s, end - 1)) * src[i].ld);
            }
    }
    __device__ __forceinline__ void commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
    // the oldest of the STAGES - 1 tiles on their way is there
    __device__ __forceinline__ void wait()
    {
        asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
        __syncwarp();
    }
    __device__ __forceinline__ float2 take(int stage, int i, int s) const
    {
        typename Two<T>::Raw r;
        if constexpr (sizeof(T) == 4)
            asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(r.x), "=f"(r.y) : "r"(slot(stage) + (i * S + s) * ROW + lane * 8) : "memory");
        else
            asm volatile("ld.shared.u32 %0, [%1];" : "=r"(*(uint32_t *)&r) : "r"(slot(stage) + (i * S + s) * ROW + lane * 4) : "memory");
        return Two<T>::get(r);
    }
};
template <class T, int S, int N>
struct Feed<T, S, N, 2> {
    static constexpr int STAGES = 2, BYTES = 0;
    T lo[N][S], hi[N][S], lo_now[N][S], hi_now[N][S];
    int c;
    __device__ __forceinline__ Feed(uint8_t *) : c(2 * (threadIdx.x & 31)) {}
    __device__ __forceinline__ void issue(int, const Source<T> (&src)[N], int t0, int begin, int end, int channels)
    {
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int s = 0; s < S; ++s) {
                const long long t = max(begin, min(t0 + s + src[i].shift, end - 1));
                const T *p = src[i].base + t * src[i].ld;
                lo[i][s] = p[c < channels ? c : 0];
                hi[i][s] = p[c + 1 < channels ? c + 1 : 0];
            }
    }
    __device__ __forceinline__ void commit() {}
    __device__ __forceinline__ void wait() // what came in becomes this tile's
    {
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int s = 0; s < S; ++s)
                lo_now[i][s] = lo[i][s], hi_now[i][s] = hi[i][s];
    }
    __device__ __forceinline__ float2 take(int, int i, int s) const { return Two<T>::get(Two<T>::join(lo_now[i][s], hi_now[i][s])); }
};

// Two channels' maps h -> A h + B as (A, A, B, B).  A sequence that starts inside makes the first A negative (a decay never is):
// what was before has no part in it, and zero times an infinity of the sequence before would be a NaN of this one.  Where no map
// has a start inside, which is known for all of them at once, the simple forms do.
constexpr float CUT = -1.f;
__device__ __forceinline__ float2 apply_plain(float4 map, float2 h) { return fma2(make_float2(map.x, map.y), h, make_float2(map.z, map.w)); }
__device__ __forceinline__ float2 apply(float4 map, float2 h) { return map.x < 0.f ? make_float2(map.z, map.w) : apply_plain(map, h); }
// first `m`, then `n`
__device__ __forceinline__ float4 join_plain(float4 m, float4 n)
{
    const float2 a = mul2(make_float2(m.x, m.y), make_float2(n.x, n.y)), b = apply_plain(n, make_float2(m.z, m.w));
    return make_float4(a.x, a.y, b.x, b.y);
}
__device__ __forceinline__ float4 join(float4 m, float4 n)
{
    const float2 b = apply(n, make_float2(m.z, m.w));
    return make_float4(m.x < 0.f || n.x < 0.f ? CUT : m.x * n.x, m.y * n.y, b.x, b.y);
}

// the maps of WARPS warps, in two buffers
struct ScanShared {
    float4 maps[2][WARPS][32];
};
// From a warp's map to the state that enters it, and `state` on to behind the tile, in the order of the recurrence
__device__ __forceinline__ float2 enter(ScanShared &sh, int buf, float4 map, float2 &state)
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    sh.maps[buf][warp][lane] = map;
    __syncthreads(); // once a tile: the other buffer's readers have passed it, too
    float2 h = make_float2(0.f, 0.f);
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
        if (w == warp)
            h = state;
        state = apply(sh.maps[buf][w][lane], state);
    }
    return h;
}
// The state that enters segment k: the maps of the segments before it (backward: behind it), a part of them by each warp
template <bool BACKWARD>
__device__ __forceinline__ float2 segment_state(const ScanArgs &p, ScanShared &sh, int k)
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int n = (BACKWARD ? p.segments - 1 - k : k) * p.subs, last = p.segments * p.subs - 1;
    float2 state = make_float2(0.f, 0.f);
    if (n == 0)
        return state;
    const float4 *maps = p.maps + (size_t)blockIdx.y * (last + 1) * 32 + lane;
    const int part = (n + WARPS - 1) / WARPS;
    float4 all = make_float4(1.f, 1.f, 0.f, 0.f);
    for (int i = warp * part; i < min(n, (warp + 1) * part); i += 8) {
        float4 m[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int at = min(i + j, n - 1);
            m[j] = maps[(size_t)(BACKWARD ? last - at : at) * 32];
        }
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (i + j < min(n, (warp + 1) * part))
                all = join(all, m[j]);
    }
    enter(sh, 1, all, state); // the first tile's buffer is the other one
    return state;
}

// ---- what a segment does to a state ----------------------------------------------------------------------------------
// The state leaves a segment as the map of what follows the last start in it (backward: precedes the first end in it).  These
// nodes, which are all or few of the segment's, are shared by `subs` blocks, and a block's by its warps.
template <class T, int S, int COPY, bool BACKWARD>
__global__ void __launch_bounds__(THREADS, 2) recurrence_maps_kernel(const ScanArgs p)
{
    grid_dep_wait();
    extern __shared__ __align__(16) uint8_t ring[];
    __shared__ ScanShared sh;
    using In = Feed<T, S, 2, COPY>;
    In in(ring);
    const Lane ch(p.D);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, at = blockIdx.x + (BACKWARD ? p.subs : 0), seg = at / p.subs, sub = at % p.subs;
    int begin, end;
    scan_range(p, begin, end);
    const int s_lo = segment_start(p, seg, begin, end), s_hi = segment_start(p, seg + 1, begin, end);
    // where the nodes begin (backward: end) that matter to the segment, and whether that is a border
    int from = BACKWARD ? s_hi : s_lo;
    bool border = !p.ptr && s_lo < s_hi && (BACKWARD ? s_hi == end : s_lo == begin);
    if (p.ptr) {
        const int i = BACKWARD ? entries_below(p.ptr, p.n_seq + 1, s_lo + 1) : entries_below(p.ptr, p.n_seq + 1, s_hi) - 1;
        const int v = i >= 0 && i <= p.n_seq ? p.ptr[i] : -1;
        border = BACKWARD ? v > s_lo && v <= s_hi : v >= s_lo && v < s_hi;
        if (border)
            from = v;
    }
    // this block's part of them
    const int all_lo = BACKWARD ? s_lo : from, need = BACKWARD ? from - s_lo : s_hi - from;
    const int lo = all_lo + (int)((long long)need * sub / p.subs), hi = all_lo + (int)((long long)need * (sub + 1) / p.subs);
    int seq = -1; // of the border, if it is in this block's part
    if (border && lo < hi && (BACKWARD ? from == hi : from == lo))
        seq = sequence_of(p.ptr, p.n_seq, BACKWARD ? from - 1 : from);
    const int part = ceil_div_dev(hi - lo, WARPS * S) * S;
    // this warp's nodes, from the one that the recurrence reaches first
    const int first = BACKWARD ? hi - warp * part : lo + warp * part, n = max(0, min(part, BACKWARD ? first - lo : hi - first));
    const Source<T> src[2] = {{(const T *)p.gate + ch.strip, p.gate_ld, 0},
                              {(const T *)(BACKWARD ? p.dh : p.x) + ch.strip, BACKWARD ? p.dh_ld : p.x_ld, 0}};
    const int channels = p.D - ch.strip;
    const auto group = [&](int i) { return BACKWARD ? first - i - S : first + i; };
    float2 A = make_float2(1.f, 1.f), B = make_float2(0.f, 0.f);
    const float *states = BACKWARD ? p.dh_last : p.h0;
    if (warp == 0 && seq >= 0 && states)
        B = load_state(states + (size_t)seq * p.D + ch.c0, ch.n);
    int stage = 0;
#pragma unroll
    for (int i = 0; i < In::STAGES - 1; ++i) {
        if (i * S < n)
            in.issue(i, src, group(i * S), begin, end, channels);
        in.commit();
    }
    for (int i = 0; i < n; i += S, stage = stage + 1 == In::STAGES ? 0 : stage + 1) {
        in.wait();
        if (i + (In::STAGES - 1) * S < n)
            in.issue(stage ? stage - 1 : In::STAGES - 1, src, group(i + (In::STAGES - 1) * S), begin, end, channels);
        in.commit();
        float2 a[S], u[S];
#pragma unroll
        for (int s = 0; s < S; ++s) {
            float2 keep;
            decay(in.take(stage, 0, s), a[s], keep);
            u[s] = in.take(stage, 1, s);
            if (!BACKWARD)
                u[s] = mul2(keep, u[s]);
        }
        if (i + S <= n) {
#pragma unroll
            for (int s = 0; s < S; ++s) {
                const int r = BACKWARD ? S - 1 - s : s;
                A = mul2(A, a[r]);
                B = BACKWARD ? mul2(a[r], add2(B, u[r])) : fma2(a[r], B, u[r]);
            }
        } else {
#pragma unroll
            for (int s = 0; s < S; ++s) {
                const int r = BACKWARD ? S - 1 - s : s;
                if (i + s < n) {
                    A = mul2(A, a[r]);
                    B = BACKWARD ? mul2(a[r], add2(B, u[r])) : fma2(a[r], B, u[r]);
                }
            }
        }
    }
    sh.maps[0][warp][lane] = make_float4(warp == 0 && seq >= 0 ? CUT : A.x, A.y, B.x, B.y);
    __syncthreads();
    if (warp == 0) {
        float4 all = sh.maps[0][0][lane];
#pragma unroll
        for (int w = 1; w < WARPS; ++w)
            all = join(all, sh.maps[0][w][lane]);
        p.maps[((size_t)blockIdx.y * p.segments * p.subs + at) * 32 + lane] = all;
    }
}

// ---- the passes ------------------------------------------------------------------------------------------------------
// A block carries 64 channels through the nodes of a segment, WARPS * S of them at a time.  The next tiles' values are on their way
// while this one's are worked on.  Groups without a border take a path without questions.
template <class T, int S, int COPY>
__global__ void __launch_bounds__(THREADS, 2) recurrence_forward_kernel(const ScanArgs p)
{
    grid_dep_wait();
    extern __shared__ __align__(16) uint8_t ring[];
    __shared__ ScanShared sh;
    using In = Feed<T, S, 2, COPY>;
    constexpr bool VEC = COPY >= 2 * (int)sizeof(T);
    In in(ring);
    const Lane ch(p.D);
    const int warp = threadIdx.x >> 5;
    if (blockIdx.x == 0)
        pass_empty(p, p.h0, p.h_last, ch.c0, ch.n);
    int begin, end;
    scan_range(p, begin, end);
    const int lo = segment_start(p, blockIdx.x, begin, end), hi = segment_start(p, blockIdx.x + 1, begin, end);
    const Source<T> src[2] = {{(const T *)p.gate + ch.strip, p.gate_ld, 0}, {(const T *)p.x + ch.strip, p.x_ld, 0}};
    const int span = WARPS * S, channels = p.D - ch.strip;
    int t0 = lo + warp * S, above = 0, stage = 0, buf = 0;
#pragma unroll
    for (int i = 0; i < In::STAGES - 1; ++i) {
        if (lo + i * span < hi)
            in.issue(i, src, t0 + i * span, begin, end, channels);
        in.commit();
    }
    float2 state = segment_state<false>(p, sh, blockIdx.x); // behind the tiles so far, the same in every warp
    for (int base = lo; base < hi; base += span, t0 += span, buf ^= 1, stage = stage + 1 == In::STAGES ? 0 : stage + 1) {
        in.wait();
        if (base + (In::STAGES - 1) * span < hi) // into the slot that the tile before left
            in.issue(stage ? stage - 1 : In::STAGES - 1, src, t0 + (In::STAGES - 1) * span, begin, end, channels);
        in.commit();
        float2 a[S], u[S];
#pragma unroll
        for (int s = 0; s < S; ++s) {
            const float2 g = in.take(stage, 0, s), v = in.take(stage, 1, s);
            float2 keep;
            decay(g, a[s], keep);
            u[s] = mul2(keep, v);
        }
        const bool plain = t0 > begin && t0 + S < min(hi, above);
        float2 A = make_float2(1.f, 1.f), B = make_float2(0.f, 0.f);
        unsigned starts = 0, ends = 0;
        if (plain) {
#pragma unroll
            for (int s = 0; s < S; ++s) {
                A = mul2(A, a[s]);
                B = fma2(a[s], B, u[s]);
            }
        } else {
            const Borders b = find_borders<S>(p.ptr, p.n_seq + 1, t0, begin, end, lo, hi);
            starts = b.starts, ends = b.ends, above = b.above;
            for (unsigned m = p.h0 ? starts : 0; m; m &= m - 1) {
                const int at = __ffs(m) - 1;
                const float2 h = load_state(p.h0 + (size_t)sequence_of(p.ptr, p.n_seq, t0 + at) * p.D + ch.c0, ch.n);
#pragma unroll
                for (int s = 0; s < S; ++s)
                    if (s == at)
                        u[s] = fma2(a[s], h, u[s]);
            }
#pragma unroll
            for (int s = 0; s < S; ++s) {
                if (t0 + s >= hi)
                    a[s] = make_float2(1.f, 1.f), u[s] = make_float2(0.f, 0.f);
                A = mul2(A, a[s]);
                B = starts >> s & 1 ? u[s] : fma2(a[s], B, u[s]);
            }
        }
        float2 h = enter(sh, buf, make_float4(starts ? CUT : A.x, A.y, B.x, B.y), state);
        T *out = (T *)p.h + ch.c0 + (long long)t0 * p.h_ld;
        if (plain) {
#pragma unroll
            for (int s = 0; s < S; ++s) {
                h = fma2(a[s], h, u[s]);
                store_two<T, VEC>(out, ch.n, h);
                out += p.h_ld;
            }
        } else {
#pragma unroll
            for (int s = 0; s < S; ++s) {
                if (!(starts >> s & 1))
                    u[s] = fma2(a[s], h, u[s]);
                h = u[s];
                if (t0 + s < hi)
                    store_two<T, VEC>(out, ch.n, h);
                out += p.h_ld;
            }
            for (unsigned m = p.h_last ? ends : 0; m; m &= m - 1) {
                const int at = __ffs(m) - 1;
#pragma unroll
                for (int s = 0; s < S; ++s)
                    if (s == at)
                        h = u[s];
                store_state(p.h_last + (size_t)sequence_of(p.ptr, p.n_seq, t0 + at) * p.D + ch.c0, ch.n, h);
            }
        }
    }
}

// The same from the last node to the first: what a node passes on is f[t] = a[t] e[t], e[t] = dh[t] + f[t+1], cut where a sequence ends
template <class T, int S, int COPY>
__global__ void __launch_bounds__(THREADS, 2) recurrence_backward_kernel(const ScanArgs p)
{
    grid_dep_wait();
    extern __shared__ __align__(16) uint8_t ring[];
    __shared__ ScanShared sh;
    using In = Feed<T, S, 4, COPY>;
    constexpr bool VEC = COPY >= 2 * (int)sizeof(T);
    In in(ring);
    const Lane ch(p.D);
    const int warp = threadIdx.x >> 5;
    if (blockIdx.x == 0)
        pass_empty(p, p.dh_last, p.dh0, ch.c0, ch.n);
    int begin, end;
    scan_range(p, begin, end);
    const int lo = segment_start(p, blockIdx.x, begin, end), hi = segment_start(p, blockIdx.x + 1, begin, end);
    // the state before a group's first node is the last one of another group
    const Source<T> src[4] = {{(const T *)p.gate + ch.strip, p.gate_ld, 0}, {(const T *)p.x + ch.strip, p.x_ld, 0},
                              {(const T *)p.h + ch.strip, p.h_ld, -1}, {(const T *)p.dh + ch.strip, p.dh_ld, 0}};
    const int span = WARPS * S, channels = p.D - ch.strip;
    int t0 = hi - (warp + 1) * S, below = INT_MAX, stage = 0, buf = 0;
#pragma unroll
    for (int i = 0; i < In::STAGES - 1; ++i) {
        if (hi - i * span > lo)
            in.issue(i, src, t0 - i * span, begin, end, channels);
        in.commit();
    }
    float2 state = segment_state<true>(p, sh, blockIdx.x); // what the tiles so far pass on
    for (int base = hi; base > lo; base -= span, t0 -= span, buf ^= 1, stage = stage + 1 == In::STAGES ? 0 : stage + 1) {
        in.wait();
        if (base - (In::STAGES - 1) * span > lo) // into the slot that the tile before left
            in.issue(stage ? stage - 1 : In::STAGES - 1, src, t0 - (In::STAGES - 1) * span, begin, end, channels);
        in.commit();
        float2 a[S], k[S], d[S], w[S]; // w = h[t-1] - x[t]
#pragma unroll
        for (int s = 0; s < S; ++s) {
            const float2 g = in.take(stage, 0, s), v = in.take(stage, 1, s), before = in.take(stage, 2, s);
            d[s] = in.take(stage, 3, s);
            decay(g, a[s], k[s]);
            w[s] = make_float2(before.x - v.x, before.y - v.y);
        }
        const bool plain = t0 >= lo && t0 > max(begin, below) && t0 + S < end;
        float2 A = make_float2(1.f, 1.f), B = make_float2(0.f, 0.f);
        unsigned starts = 0, ends = 0;
        if (plain) {
#pragma unroll
            for (int s = S - 1; s >= 0; --s) {
                A = mul2(A, a[s]);
                B = mul2(a[s], add2(B, d[s]));
            }
        } else {
            const Borders b = find_borders<S>(p.ptr, p.n_seq + 1, t0, begin, end, lo, hi);
            starts = b.starts, ends = b.ends, below = b.below;
            for (unsigned m = starts; m; m &= m - 1) {
                const int at = __ffs(m) - 1;
                float2 h = make_float2(0.f, 0.f);
                if (p.h0)
                    h = load_state(p.h0 + (size_t)sequence_of(p.ptr, p.n_seq, t0 + at) * p.D + ch.c0, ch.n);
#pragma unroll
                for (int s = 0; s < S; ++s)
                    if (s == at) {
                        const float2 v = in.take(stage, 1, s);
                        w[s] = make_float2(h.x - v.x, h.y - v.y);
                    }
            }
            for (unsigned m = p.dh_last ? ends : 0; m; m &= m - 1) {
                const int at = __ffs(m) - 1;
                const float2 l = load_state(p.dh_last + (size_t)sequence_of(p.ptr, p.n_seq, t0 + at) * p.D + ch.c0, ch.n);
#pragma unroll
                for (int s = 0; s < S; ++s)
                    if (s == at)
                        d[s] = make_float2(d[s].x + l.x, d[s].y + l.y);
            }
#pragma unroll
            for (int s = S - 1; s >= 0; --s) {
                if (t0 + s < lo)
                    a[s] = make_float2(1.f, 1.f), d[s] = make_float2(0.f, 0.f);
                A = mul2(A, a[s]);
                B = mul2(a[s], ends >> s & 1 ? d[s] : add2(B, d[s]));
            }
        }
        float2 f = enter(sh, buf, make_float4(ends ? CUT : A.x, A.y, B.x, B.y), state);
        T *dx = (T *)p.dx + ch.c0 + (long long)(t0 + S - 1) * p.dx_ld, *dgate = (T *)p.dgate + ch.c0 + (long long)(t0 + S - 1) * p.dgate_ld;
        if (plain) {
#pragma unroll
            for (int s = S - 1; s >= 0; --s) {
                const float2 e = add2(d[s], f), ke = mul2(k[s], e);
                f = mul2(a[s], e);
                store_two<T, VEC>(dx, ch.n, ke);
                store_two<T, VEC>(dgate, ch.n, mul2(mul2(a[s], ke), w[s]));
                dx -= p.dx_ld, dgate -= p.dgate_ld;
            }
        } else {
#pragma unroll
            for (int s = S - 1; s >= 0; --s) {
                const float2 e = ends >> s & 1 ? d[s] : add2(d[s], f), ke = mul2(k[s], e);
                f = mul2(a[s], e);
                if (t0 + s >= lo) {
                    store_two<T, VEC>(dx, ch.n, ke);
                    store_two<T, VEC>(dgate, ch.n, mul2(mul2(a[s], ke), w[s]));
                }
                dx -= p.dx_ld, dgate -= p.dgate_ld;
                d[s] = f;
            }
            for (unsigned m = p.dh0 ? starts : 0; m; m &= m - 1) {
                const int at = __ffs(m) - 1;
#pragma unroll
                for (int s = 0; s < S; ++s)
                    if (s == at)
                        f = d[s];
                store_state(p.dh0 + (size_t)sequence_of(p.ptr, p.n_seq, t0 + at) * p.D + ch.c0, ch.n, f);
            }
        }
    }
}

template <class In>
static int launch(const Ctx &c, void (*kern)(ScanArgs), dim3 grid, const ScanArgs &p, std::atomic<unsigned> &ready)
{
    const unsigned bit = 1u << (c.device & 15); // the device has been told how much shared memory the kernel takes
    if (!(ready.load() & bit)) {
        TS2_CUDA(cudaFuncSetAttribute((const void *)kern, cudaFuncAttributeMaxDynamicSharedMemorySize, In::BYTES));
        ready.fetch_or(bit);
    }
    TS2_LAUNCH(kern, grid, THREADS, In::BYTES, c.stream, p);
    return TS2_OK;
}
template <class T, int S, int COPY, bool BACKWARD>
static int passes(const Ctx &c, ScanArgs &p)
{
    static std::atomic<unsigned> ready[2];
    const int strips = (int)ceil_div(p.D, STRIP);
    // As many blocks as the device holds at once, with two tiles each: then every segment's maps have to be there first, which
    // reads gate and x (dh) a second time from the L2 or from memory (32768 x 512 fp32, one sequence, us: 1 segment 532, 12: 80,
    // 36: 57; 5001 x 333 fp16 backward 199, 31, 20).  Up to six tiles one after the other are faster than two launches.
    const int64_t tiles = ceil_div(p.T, WARPS * S);
    p.segments = tiles <= 6 ? 1 : (int)std::max<int64_t>(1, std::min<int64_t>(2 * sm_count(c.device) / strips, tiles / 2));
    // two blocks share the nodes that a segment's map needs, which are all or few (64 sequences, 65536 x 768 bf16: 98 -> 91 us)
    p.subs = tiles / p.segments >= 4 ? 2 : 1;
    void *scratch = nullptr;
    if (p.segments > 1) {
        if (int rc = scratch_alloc(c.device, (size_t)strips * p.segments * p.subs * 512, c.stream, &scratch))
            return rc;
        p.maps = (float4 *)scratch;
    }
    const auto work = [&] {
        if (p.segments > 1)
            if (int rc = launch<Feed<T, S, 2, COPY>>(c, recurrence_maps_kernel<T, S, COPY, BACKWARD>, dim3((p.segments - 1) * p.subs, strips), p, ready[0]))
                return rc;
        if constexpr (BACKWARD)
            return launch<Feed<T, S, 4, COPY>>(c, recurrence_backward_kernel<T, S, COPY>, dim3(p.segments, strips), p, ready[1]);
        else
            return launch<Feed<T, S, 2, COPY>>(c, recurrence_forward_kernel<T, S, COPY>, dim3(p.segments, strips), p, ready[1]);
    };
    const int rc = work();
    if (scratch)
        scratch_free(c.stream, scratch);
    return rc;
}
template <class T, int S_FORWARD, int S_BACKWARD, int COPY>
static int by_direction(const Ctx &c, ScanArgs &p, bool backward)
{
    return backward ? passes<T, S_BACKWARD, COPY, true>(c, p) : passes<T, S_FORWARD, COPY, false>(c, p);
}

static int run(const Ctx &c, int type, ScanArgs &p, bool backward)
{
    // what all rows begin on a multiple of: 16 bytes, a pair or an element
    const int es = type == TS2_OUT_F32 ? 4 : 2;
    const uintptr_t at = (uintptr_t)p.gate | (uintptr_t)p.x | (uintptr_t)p.h | (backward ? (uintptr_t)p.dh | (uintptr_t)p.dgate | (uintptr_t)p.dx : 0);
    const unsigned pitch = (unsigned)(p.gate_ld | p.x_ld | p.h_ld | p.D | (backward ? p.dh_ld | p.dgate_ld | p.dx_ld : 0)) * es;
    const unsigned align = (unsigned)at | pitch;
    const bool wide = align % 16 == 0, pair = align % (2 * es) == 0;
    switch (type) {
    case TS2_OUT_F32: return wide ? by_direction<float, 8, 4, 16>(c, p, backward) : pair ? by_direction<float, 8, 4, 8>(c, p, backward) : by_direction<float, 8, 4, 4>(c, p, backward);
    case TS2_OUT_F16: return wide ? by_direction<__half, 16, 8, 16>(c, p, backward) : pair ? by_direction<__half, 16, 8, 4>(c, p, backward) : by_direction<__half, 8, 4, 2>(c, p, backward);
    case TS2_OUT_BF16:
        return wide ? by_direction<__nv_bfloat16, 16, 8, 16>(c, p, backward) : pair ? by_direction<__nv_bfloat16, 16, 8, 4>(c, p, backward) : by_direction<__nv_bfloat16, 8, 4, 2>(c, p, backward);
    default: return fail(TS2_ERR_INVALID_ARG, "recurrence: unknown type %d", type);
    }
}

int recurrence_forward(const Ctx &c, int type, const void *gate, int64_t gate_ld, const void *x, int64_t x_ld, int T, int D, int n_seq,
                       const int *seq_ptr, const float *h0, void *h, int64_t h_ld, float *h_last)
{
    ScanArgs p = {};
    p.gate = gate, p.gate_ld = (int)gate_ld, p.x = x, p.x_ld = (int)x_ld, p.T = T, p.D = D, p.n_seq = n_seq, p.ptr = seq_ptr, p.h0 = h0;
    p.h = h, p.h_ld = (int)h_ld, p.h_last = h_last;
    return run(c, type, p, false);
}

int recurrence_backward(const Ctx &c, int type, const void *gate, int64_t gate_ld, const void *x, int64_t x_ld, const void *h, int64_t h_ld,
                        int T, int D, int n_seq, const int *seq_ptr, const float *h0, const void *dh, int64_t dh_ld, const float *dh_last,
                        void *dgate, int64_t dgate_ld, void *dx, int64_t dx_ld, float *dh0)
{
    ScanArgs p = {};
    p.gate = gate, p.gate_ld = (int)gate_ld, p.x = x, p.x_ld = (int)x_ld, p.T = T, p.D = D, p.n_seq = n_seq, p.ptr = seq_ptr, p.h0 = h0;
    p.h = const_cast<void *>(h), p.h_ld = (int)h_ld, p.dh = dh, p.dh_ld = (int)dh_ld, p.dh_last = dh_last;
    p.dgate = dgate, p.dgate_ld = (int)dgate_ld, p.dx = dx, p.dx_ld = (int)dx_ld, p.dh0 = dh0;
    return run(c, type, p, true);
}

} // namespace ts2
