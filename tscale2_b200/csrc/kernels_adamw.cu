// One AdamW step of many tensors in one launch.  With g = grad * scale, k the step,
//     m = beta1 m + (1 - beta1) g,   v = beta2 v + (1 - beta2) g^2
//     p = p (1 - r decay) - r m / (1 - beta1^k) / (sqrt(v / (1 - beta2^k)) + eps)
// Every element is read once and written once: memory bandwidth bounds large models, the latency of a launch small ones.  The tensors' table
// travels as the kernel's parameters, so that nothing is copied to the device before it and a captured call keeps its table.  A CTA
// finds its chunk's tensor by bisection and takes eight neighbours a thread, 16 bytes an access where the tensor's arrays are aligned to that.
//
// Moments in 8 bits: e4m3 with a power of two for 32 neighbours.  Rounding to the nearest would hold a slow average where it is: with beta2 0.999 it moves
// by at most a thousandth of itself when gradients get smaller, and two e4m3 values are a sixteenth to an eighth apart.  So a hash decides
// between the two neighbours, with the odds that keep the expectation.  The sums that are rounded so are fp64: their last bits do not decide, and any
// implementation of the formula gives the same bytes.
#include "elem_types.cuh"
#include "kernels.cuh"
#include <algorithm>
#include <cmath>
#include <type_traits>

namespace ts2 {

static constexpr int THREADS = 128, TURN = 8 * THREADS; // TURN: elements that a CTA takes at a time
struct AdamwRecord {
    float *param;
    const void *grad;
    void *m, *v;
    uint8_t *m_scale, *v_scale;
    void *copy;
    int64_t n;
    uint32_t chunk0; // the tensor's first chunk in the launch
    uint32_t key;
    float decay, rate; // r decay, r / (1 - beta1^k)
};
struct AdamwArgs {
    double beta1, beta2;
    float grad_scale, inv_c2, eps; // inv_c2 = 1 / sqrt(1 - beta2^k)
    const float *grad_scale_dev;
    int n, copy_type, turns; // turns: of a CTA, a chunk
};
// a launch's parameters may take 32764 bytes; few tensors travel in a smaller table
template <int CAP>
struct AdamwTable {
    AdamwRecord r[CAP];
};

// eight neighbours from element j on; whole: all of them are there and aligned to 16 bytes (bytes: to 8)
template <class T>
__device__ __forceinline__ void load8(const T *p, int64_t j, int64_t n, bool whole, T (&v)[8])
{
    constexpr int PER = sizeof(T) == 1 ? 8 : 16 / sizeof(T);
    if (whole) {
#pragma unroll
        for (int h = 0; h < 8 / PER; ++h) {
            const Piece<T, PER> q = *(const Piece<T, PER> *)(p + j + h * PER);
#pragma unroll
            for (int i = 0; i < PER; ++i)
                v[h * PER + i] = q.v[i];
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            v[i] = j + i < n ? p[j + i] : T(0.f);
    }
}
template <class T>
__device__ __forceinline__ void store8(T *p, int64_t j, int64_t n, bool whole, const T (&v)[8])
{
    constexpr int PER = sizeof(T) == 1 ? 8 : 16 / sizeof(T);
    if (whole) {
#pragma unroll
        for (int h = 0; h < 8 / PER; ++h) {
            Piece<T, PER> q;
#pragma unroll
            for (int i = 0; i < PER; ++i)
                q.v[i] = v[h * PER + i];
            *(Piece<T, PER> *)(p + j + h * PER) = q;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (j + i < n)
                p[j + i] = v[i];
    }
}
// the same of bytes, four to a word
__device__ __forceinline__ void load8_bytes(const uint8_t *p, int64_t j, int64_t n, bool whole, uint32_t (&w)[2])
{
    if (whole) {
        const uint2 q = *(const uint2 *)(p + j);
        w[0] = q.x, w[1] = q.y;
    } else {
        w[0] = w[1] = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            w[i >> 2] |= j + i < n ? (uint32_t)p[j + i] << (8 * (i & 3)) : 0u;
    }
}
__device__ __forceinline__ void store8_bytes(uint8_t *p, int64_t j, int64_t n, bool whole, const uint32_t (&w)[2])
{
    if (whole) {
        *(uint2 *)(p + j) = make_uint2(w[0], w[1]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (j + i < n)
                p[j + i] = (uint8_t)(w[i >> 2] >> (8 * (i & 3)));
    }
}

// the finaliser of MurmurHash3
__device__ __forceinline__ uint32_t mix32(uint32_t x)
{
    x = (x ^ (x >> 16)) * 0x85EBCA6Bu;
    x = (x ^ (x >> 13)) * 0xC2B2AE35u;
    return x ^ (x >> 16);
}

// four e4m3 bytes as fp32, exactly
__device__ __forceinline__ void e4m3_values(uint32_t codes, float *v)
{
    const __half2_raw a = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(codes & 0xffffu), __NV_E4M3),
                      b = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(codes >> 16), __NV_E4M3);
    const float2 x = __half22float2(*(const __half2 *)&a), y = __half22float2(*(const __half2 *)&b);
    v[0] = x.x, v[1] = x.y, v[2] = y.x, v[3] = y.y;
}
// 2^(scale - 127), NaN for 255
__device__ __forceinline__ double scale_value(int scale)
{
    return __hiloint2double(scale == 255 ? 0x7ff80000 : (scale + 1023 - 127) << 20, 0);
}
constexpr uint32_t BEYOND = (1023u + 128) << 20; // the upper word of 2^128: no fp32 number
// Eight values as e4m3 bytes, in the blocks of 32 that four lanes hold.  y is a magnitude in the smallest steps of e4m3, 2^-9 of the block's power of two, and
// u16 / 2^16 of a step of its own is added before the rest is cut off: from 8 on a step is what the exponent's upper bits and three of the mantissa's count, so the
// byte is those bits; below, a step is one, as it is from 8 to 16, and 8 is added to y and taken off the byte.  The upper word of a double has 20 bits of the
// mantissa, of which 17 are cut off, and u has 16: what the lower word holds does not matter.
template <bool FLOOR_AT_ONE>
__device__ __forceinline__ void encode8(const double (&x)[8], const uint32_t (&h)[8], bool upper_half, uint32_t (&codes)[2], int &scale)
{
    uint32_t top = 0, hi[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        hi[k] = (uint32_t)__double2hiint(x[k]);
        top = max(top, hi[k] & 0x7fffffffu);
    }
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const int e = max((int)(top >> 20) - 1023 - 7, -127);
    const bool bad = top >= BEYOND;
    scale = bad ? 255 : e + 127;
    const double steps = __hiloint2double((1023 + 9 - e) << 20, 0);
    uint32_t c[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const double y = fabs(x[k]) * steps;
        const bool small = (uint32_t)__double2hiint(y) < (1023u + 3) << 20;
        const uint32_t w = small ? (uint32_t)__double2hiint(y + 8.) - (8u << 17) : (uint32_t)__double2hiint(y),
                       u = upper_half ? (h[k] >> 15) & 0x1fffeu : (h[k] << 1) & 0x1fffeu;
        c[k] = (w + u - ((1023u + 2) << 20)) >> 17;
        if (FLOOR_AT_ONE)
            c[k] = max(c[k], min(hi[k], 1u));
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        codes[i] = __byte_perm(__byte_perm(c[4 * i], c[4 * i + 1], 0x0040), __byte_perm(c[4 * i + 2], c[4 * i + 3], 0x0040), 0x5410);
        if (!FLOOR_AT_ONE)
            codes[i] |= __byte_perm(__byte_perm(hi[4 * i], hi[4 * i + 1], 0x0073), __byte_perm(hi[4 * i + 2], hi[4 * i + 3], 0x0073), 0x5410) & 0x80808080u;
        codes[i] = bad ? 0u : codes[i];
    }
}

// A v below 2^-126 counts as zero beside eps (its root is below 2^-63).  The decay is taken off with the update, since 1 - r decay would be rounded to steps of 2^-24: r decay
// of 1e-7 would be 1.2e-7 for every element and step.
__device__ __forceinline__ float step_of(const AdamwArgs &a, const AdamwRecord &r, float p, float m, float v)
{
    float root, inverse;
    asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(root) : "f"(v));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inverse) : "f"(fmaf(root, a.inv_c2, a.eps)));
    return p - fmaf(r.decay, p, r.rate * m * inverse);
}

// what a thread reads in a turn, as it lies in memory
template <class G, int BITS>
struct AdamwTurn {
    float p[8];
    G g[8];
    typename std::conditional<BITS == 32, float, uint32_t>::type m[BITS == 32 ? 8 : 2], v[BITS == 32 ? 8 : 2];
    int ms, vs;
    __device__ __forceinline__ void load(const AdamwRecord &r, int64_t j, bool aligned)
    {
        const bool whole = aligned && j + 8 <= r.n;
        if constexpr (BITS == 32) {
            load8((const float *)r.m, j, r.n, whole, m);
            load8((const float *)r.v, j, r.n, whole, v);
        } else {
            load8_bytes((const uint8_t *)r.m, j, r.n, whole, m);
            load8_bytes((const uint8_t *)r.v, j, r.n, whole, v);
            ms = j < r.n ? r.m_scale[j >> 5] : 0, vs = j < r.n ? r.v_scale[j >> 5] : 0;
        }
        load8((const G *)r.grad, j, r.n, whole, g);
        load8(r.param, j, r.n, whole, p);
    }
};

// Moments in 8 bits take 80 instructions an element against 16 bytes of memory, so warps have to cover both: 64 registers, 32 warps an SM.  166 M parameters: 521 us
// (blocks of 256 threads 551; 24 warps with the next turn's loads ahead of this one's arithmetic 554, 16 warps 651; 36 warps, which spill, 552).
template <class G, int BITS, int CAP>
__global__ void __launch_bounds__(THREADS, BITS == 32 ? 5 : 8) adamw_kernel(const __grid_constant__ AdamwTable<CAP> table, const AdamwArgs a)
{
    int lo = 0, hi = a.n; // the last record that begins at or before this chunk
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (table.r[mid].chunk0 <= blockIdx.x)
            lo = mid;
        else
            hi = mid;
    }
    const AdamwRecord r = table.r[lo];
    grid_dep_wait();
    const float gs = a.grad_scale_dev ? a.grad_scale * *a.grad_scale_dev : a.grad_scale;
    const int64_t n = r.n, begin = (int64_t)(blockIdx.x - r.chunk0) * a.turns * TURN, end = min(n, begin + (int64_t)a.turns * TURN);
    const uintptr_t states = ((uintptr_t)r.m | (uintptr_t)r.v) * (BITS == 32 ? 1 : 2);
    const bool aligned = ((uintptr_t)r.param | states | (uintptr_t)r.copy | (uintptr_t)r.grad) % 16 == 0;
    int64_t j = begin + (int)threadIdx.x * 8;
#pragma unroll 1
    for (int64_t turn = begin; turn < end; turn += TURN, j += TURN) {
        const bool whole = aligned && j + 8 <= n;
        AdamwTurn<G, BITS> now;
        now.load(r, j, aligned);
        float p[8], m[8], v[8];
        if constexpr (BITS == 32) {
            const float b1 = (float)a.beta1, c1 = (float)(1. - a.beta1), b2 = (float)a.beta2, c2 = (float)(1. - a.beta2);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const float x = widen(now.g[k]) * gs;
                m[k] = fmaf(b1, now.m[k], c1 * x);
                v[k] = fmaf(b2, now.v[k], c2 * x * x);
            }
            store8((float *)r.m, j, n, whole, m);
            store8((float *)r.v, j, n, whole, v);
        } else {
            const double mb = a.beta1 * scale_value(now.ms), vb = a.beta2 * scale_value(now.vs), c1 = 1. - a.beta1, c2 = 1. - a.beta2;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                e4m3_values(now.m[k], m + 4 * k);
                e4m3_values(now.v[k], v + 4 * k);
            }
            double mm[8], vv[8];
            uint32_t h[8], codes[2];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const double x = (double)(widen(now.g[k]) * gs);
                mm[k] = fma(mb, (double)m[k], c1 * x);
                vv[k] = fma(vb, (double)v[k], c2 * (x * x));
                m[k] = (float)mm[k], v[k] = (float)vv[k];
                h[k] = mix32((uint32_t)(j + k) * 0x9E3779B1u + r.key);
            }
            int me, ve;
            encode8<false>(mm, h, true, codes, me);
            store8_bytes((uint8_t *)r.m, j, n, whole, codes);
            encode8<true>(vv, h, false, codes, ve);
            store8_bytes((uint8_t *)r.v, j, n, whole, codes);
            if (j < n && (threadIdx.x & 3) == 0)
                r.m_scale[j >> 5] = (uint8_t)me, r.v_scale[j >> 5] = (uint8_t)ve;
        }
#pragma unroll
        for (int k = 0; k < 8; ++k)
            p[k] = step_of(a, r, now.p[k], m[k], v[k]);
        store8(r.param, j, n, whole, p);
        if (r.copy && a.copy_type == TS2_OUT_F16) {
            __half c[8];
#pragma unroll
            for (int k = 0; k < 8; ++k)
                c[k] = narrow<__half>(p[k]);
            store8((__half *)r.copy, j, n, whole, c);
        } else if (r.copy) {
            __nv_bfloat16 c[8];
#pragma unroll
            for (int k = 0; k < 8; ++k)
                c[k] = narrow<__nv_bfloat16>(p[k]);
            store8((__nv_bfloat16 *)r.copy, j, n, whole, c);
        }
    }
}

// ---- host ------------------------------------------------------------------------------------------------------------
// SplitMix64 (Steele, Lea, Flood): the output that follows this state
static uint64_t mix64(uint64_t x)
{
    x += 0x9E3779B97F4A7C15ull;
    x = (x ^ (x >> 30)) * 0xBF58476D1CE4E5B9ull;
    x = (x ^ (x >> 27)) * 0x94D049BB133111EBull;
    return x ^ (x >> 31);
}

template <class G, int BITS, int CAP>
static int launch(const Ctx &c, const AdamwTable<400> &table, uint32_t chunks, const AdamwArgs &a)
{
    static_assert(sizeof(AdamwTable<CAP>) <= sizeof(table) && sizeof(AdamwTable<400>) + sizeof(AdamwArgs) <= 32764, "kernel parameters");
    TS2_LAUNCH((adamw_kernel<G, BITS, CAP>), chunks, THREADS, 0, c.stream, *(const AdamwTable<CAP> *)&table, a);
    return TS2_OK;
}
template <class G, int BITS>
static int launch(const Ctx &c, const AdamwTable<400> &table, uint32_t chunks, const AdamwArgs &a)
{
    return a.n <= 32 ? launch<G, BITS, 32>(c, table, chunks, a) : a.n <= 128 ? launch<G, BITS, 128>(c, table, chunks, a) : launch<G, BITS, 400>(c, table, chunks, a);
}
template <class G>
static int launch(const Ctx &c, int bits, const AdamwTable<400> &table, uint32_t chunks, const AdamwArgs &a)
{
    return bits == 32 ? launch<G, 32>(c, table, chunks, a) : launch<G, 8>(c, table, chunks, a);
}

int adamw(const Ctx &c, int grad_type, int state_bits, int copy_type, const ts2_adamw_tensor *tensors, int n, float rate, float beta1, float beta2,
          float eps, int64_t step, float grad_scale, const float *grad_scale_dev, uint64_t seed)
{
    const double c1 = -std::expm1((double)step * std::log((double)beta1)), c2 = -std::expm1((double)step * std::log((double)beta2)); // beta 0: 1
    AdamwArgs a = {};
    a.beta1 = beta1, a.beta2 = beta2, a.grad_scale = grad_scale, a.inv_c2 = (float)(1. / std::sqrt(c2)), a.eps = eps, a.grad_scale_dev = grad_scale_dev;
    a.copy_type = copy_type;
    // chunks long enough that what a CTA does once does not count, and enough of them to fill the device
    int64_t total = 0;
    for (int i = 0; i < n; ++i)
        total += tensors[i].n;
    a.turns = (int)std::max<int64_t>(1, std::min<int64_t>(8, total / ((int64_t)16 * sm_count(c.device) * TURN)));
    AdamwTable<400> table;
    uint64_t chunks = 0;
    const auto flush = [&] {
        if (!a.n)
            return (int)TS2_OK;
        const int rc = grad_type == TS2_OUT_F32   ? launch<float>(c, state_bits, table, (uint32_t)chunks, a)
                       : grad_type == TS2_OUT_F16 ? launch<__half>(c, state_bits, table, (uint32_t)chunks, a)
                                                  : launch<__nv_bfloat16>(c, state_bits, table, (uint32_t)chunks, a);
        a.n = 0, chunks = 0;
        return rc;
    };
    for (int i = 0; i < n; ++i) {
        const ts2_adamw_tensor &t = tensors[i];
        const uint64_t mine = (uint64_t)ceil_div(t.n, (int64_t)a.turns * TURN); // 2^29 at most
        if (!mine)
            continue;
        if (a.n == 400 || chunks + mine > 0x7fffffffu)
            if (const int rc = flush())
                return rc;
        AdamwRecord &r = table.r[a.n++];
        r.param = t.param, r.grad = t.grad, r.m = t.m, r.v = t.v, r.m_scale = t.m_scale, r.v_scale = t.v_scale, r.copy = t.copy, r.n = t.n;
        r.chunk0 = (uint32_t)chunks;
        r.key = (uint32_t)mix64(mix64(seed + (uint64_t)step) ^ (uint64_t)i);
        r.decay = (float)((double)rate * t.rate * t.decay);
        r.rate = (float)((double)rate * t.rate / c1);
        chunks += mine;
    }
    return flush();
}

} // namespace ts2
