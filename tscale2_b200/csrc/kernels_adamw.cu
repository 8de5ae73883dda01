// One AdamW step of many tensors in one launch.  With g = grad * scale, k the step,
//     m = beta1 m + (1 - beta1) g,   v = beta2 v + (1 - beta2) g^2
//     p = p (1 - r decay) - r m / (1 - beta1^k) / (sqrt(v / (1 - beta2^k)) + eps)
// Every element is read once and written once: memory bandwidth bounds large models, the latency of a launch small ones.  The tensors' table
// travels as the kernel's parameters, so that nothing is copied to the device before it and a captured call keeps its table.  A CTA
// finds its chunk's tensor by bisection and takes four neighbours a thread and access where the tensor's arrays are aligned to that.
//
// Moments in 8 bits: e4m3 with a power of two for 32 neighbours.  Rounding to the nearest would hold a slow average where it is: with beta2 0.999 it moves
// by at most a thousandth of itself when gradients get smaller, and two e4m3 values are a sixteenth to an eighth apart.  So a hash decides
// between the two neighbours, with the odds that keep the expectation.  The sums that are rounded so are fp64: their last bits do not decide, and any
// implementation of the formula gives the same bytes.
#include "elem_types.cuh"
#include "kernels.cuh"
#include <algorithm>
#include <cmath>

namespace ts2 {

static constexpr int THREADS = 256, CHUNK = 4096; // elements of a CTA
struct AdamwRecord {
    float *param;
    const void *grad;
    void *m, *v;
    uint8_t *m_scale, *v_scale;
    void *copy;
    int64_t n;
    uint32_t chunk0; // the tensor's first chunk in the launch
    uint32_t key;
    float keep, rate; // 1 - r decay, r / (1 - beta1^k)
};
struct AdamwArgs {
    double beta1, beta2;
    float grad_scale, inv_c2, eps; // inv_c2 = 1 / sqrt(1 - beta2^k)
    const float *grad_scale_dev;
    int n, copy_type;
};
// a launch's parameters may take 32764 bytes; few tensors travel in a smaller table
template <int CAP>
struct AdamwTable {
    AdamwRecord r[CAP];
};

// four neighbours from element j on; whole: all of them are there and aligned to four
template <class T>
__device__ __forceinline__ void load4(const T *p, int64_t j, int64_t n, bool whole, T (&v)[4])
{
    if (whole) {
        const Piece<T, 4> q = *(const Piece<T, 4> *)(p + j);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            v[i] = q.v[i];
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            v[i] = j + i < n ? p[j + i] : T(0.f);
    }
}
template <class T>
__device__ __forceinline__ void store4(T *p, int64_t j, int64_t n, bool whole, const T (&v)[4])
{
    if (whole) {
        Piece<T, 4> q;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            q.v[i] = v[i];
        *(Piece<T, 4> *)(p + j) = q;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (j + i < n)
                p[j + i] = v[i];
    }
}
__device__ __forceinline__ uint32_t load4_bytes(const uint8_t *p, int64_t j, int64_t n, bool whole)
{
    if (whole)
        return *(const uint32_t *)(p + j);
    uint32_t r = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        r |= j + i < n ? (uint32_t)p[j + i] << (8 * i) : 0u;
    return r;
}
__device__ __forceinline__ void store4_bytes(uint8_t *p, int64_t j, int64_t n, bool whole, uint32_t v)
{
    if (whole) {
        *(uint32_t *)(p + j) = v;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (j + i < n)
                p[j + i] = (uint8_t)(v >> (8 * i));
    }
}

// the finaliser of MurmurHash3
__device__ __forceinline__ uint32_t mix32(uint32_t x)
{
    x = (x ^ (x >> 16)) * 0x85EBCA6Bu;
    x = (x ^ (x >> 13)) * 0xC2B2AE35u;
    return x ^ (x >> 16);
}

// The value of an e4m3 byte times 2^(scale - 127), exactly.  The exponent and the mantissa's three bits go to the upper word of a double as they are; a
// byte below 8 has no implicit one, which is added and taken off.  A scale of 255 stands for NaNs (an e4m3 NaN is never written).
__device__ __forceinline__ double decode(uint32_t code, int scale)
{
    const uint32_t mag = code & 127u;
    const int base = 1023 - 7 + scale - 127; // the exponent of bytes whose exponent field is 0
    const double v = __hiloint2double(((mag | (mag < 8u ? 8u : 0u)) << 17) + (base << 20), 0) - (mag < 8u ? __hiloint2double((base + 1) << 20, 0) : 0.);
    return scale == 255 ? __longlong_as_double(0x7ff8000000000000ll) : (code & 128u ? -v : v);
}
// A byte for the magnitude of x over 2^e (hi: upper word of |x|), in the smallest steps of e4m3, 2^-9: u16 / 2^16 of a step is added before the rest is cut
// off.  Twenty bits of the mantissa are in that word, three stay, and u has sixteen: what is below does not matter.
__device__ __forceinline__ uint32_t encode(uint32_t hi, int e, uint32_t u16)
{
    if (hi == 0)
        return 0;
    const int a = (int)hi + ((9 - e) << 20), exponent = (a >> 20) - 1023; // of |x| / 2^e * 2^9, below 17
    if (exponent >= 3)
        return (uint32_t)((a + (int)(u16 << 1)) >> 17) - ((1023 + 2) << 3);
    const uint32_t mantissa = ((uint32_t)a & 0xfffffu) | 0x100000u;
    const int shift = 4 - exponent; // to multiples of 2^-16
    return ((shift < 32 ? mantissa >> shift : 0u) + u16) >> 16;
}
// the exponent of the power of two of the 32 elements that 8 lanes hold, from the largest upper word among them
__device__ __forceinline__ uint32_t block_top(uint32_t hi)
{
#pragma unroll
    for (int o = 4; o > 0; o >>= 1)
        hi = max(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    return hi;
}
__device__ __forceinline__ int block_exponent(uint32_t top) { return max((int)(top >> 20) - 1023 - 7, -127); }

__device__ __forceinline__ float step_of(const AdamwArgs &a, const AdamwRecord &r, float p, float m, float v)
{
    float root;
    asm("sqrt.approx.f32 %0, %1;" : "=f"(root) : "f"(v));
    return fmaf(p, r.keep, -r.rate * __fdividef(m, fmaf(root, a.inv_c2, a.eps)));
}

template <class G, int BITS, int CAP>
__global__ void __launch_bounds__(THREADS) adamw_kernel(const __grid_constant__ AdamwTable<CAP> table, const AdamwArgs a)
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
    const int64_t n = r.n, begin = (int64_t)(blockIdx.x - r.chunk0) * CHUNK;
    const uintptr_t states = BITS == 32 ? ((uintptr_t)r.m | (uintptr_t)r.v) : ((uintptr_t)r.m | (uintptr_t)r.v) * 4;
    const bool aligned = ((uintptr_t)r.param | states | (uintptr_t)r.copy * 2 | (uintptr_t)r.grad * (16 / (4 * sizeof(G)))) % 16 == 0;
#pragma unroll 2
    for (int i = 0; i < CHUNK / (4 * THREADS); ++i) {
        const int64_t j = begin + (i * THREADS + (int)threadIdx.x) * 4;
        if (begin + i * THREADS * 4 >= n)
            break; // of the whole CTA
        const bool whole = aligned && j + 4 <= n;
        float p[4], m[4], v[4];
        G g[4];
        load4(r.param, j, n, whole, p);
        load4((const G *)r.grad, j, n, whole, g);
        if constexpr (BITS == 32) {
            load4((const float *)r.m, j, n, whole, m);
            load4((const float *)r.v, j, n, whole, v);
            const float b1 = (float)a.beta1, c1 = (float)(1. - a.beta1), b2 = (float)a.beta2, c2 = (float)(1. - a.beta2);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float x = widen(g[k]) * gs;
                m[k] = fmaf(b1, m[k], c1 * x);
                v[k] = fmaf(b2, v[k], c2 * x * x);
            }
            store4((float *)r.m, j, n, whole, m);
            store4((float *)r.v, j, n, whole, v);
        } else {
            const bool there = j < n;
            const uint32_t mc = load4_bytes((const uint8_t *)r.m, j, n, whole), vc = load4_bytes((const uint8_t *)r.v, j, n, whole);
            const int ms = there ? r.m_scale[j >> 5] : 0, vs = there ? r.v_scale[j >> 5] : 0;
            uint32_t mh[4], vh[4], sign = 0, mtop = 0, vtop = 0;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const double x = (double)(widen(g[k]) * gs);
                const double mm = fma(a.beta1, decode((mc >> (8 * k)) & 255u, ms), (1. - a.beta1) * x);
                const double vv = fma(a.beta2, decode((vc >> (8 * k)) & 255u, vs), (1. - a.beta2) * (x * x));
                mh[k] = (uint32_t)__double2hiint(mm) & 0x7fffffffu, vh[k] = (uint32_t)__double2hiint(vv) & 0x7fffffffu;
                sign |= ((uint32_t)__double2hiint(mm) >> 31) << (8 * k + 7);
                m[k] = (float)mm, v[k] = (float)vv;
                mtop = max(mtop, mh[k]), vtop = max(vtop, vh[k]);
            }
            mtop = block_top(mtop), vtop = block_top(vtop);
            const int me = block_exponent(mtop), ve = block_exponent(vtop);
            uint32_t mo = 0, vo = 0;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t h = mix32((uint32_t)(j + k) * 0x9E3779B1u + r.key);
                mo |= encode(mh[k], me, h >> 16) << (8 * k);
                const uint32_t code = encode(vh[k], ve, h & 0xffffu);
                vo |= (vh[k] != 0 && code == 0 ? 1u : code) << (8 * k);
            }
            store4_bytes((uint8_t *)r.m, j, n, whole, mtop >= 0x7ff00000u ? 0u : mo | sign);
            store4_bytes((uint8_t *)r.v, j, n, whole, vtop >= 0x7ff00000u ? 0u : vo);
            if (there && (threadIdx.x & 7) == 0) {
                r.m_scale[j >> 5] = (uint8_t)(mtop >= 0x7ff00000u ? 255 : me + 127);
                r.v_scale[j >> 5] = (uint8_t)(vtop >= 0x7ff00000u ? 255 : ve + 127);
            }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k)
            p[k] = step_of(a, r, p[k], m[k], v[k]);
        store4(r.param, j, n, whole, p);
        if (r.copy) {
            if (a.copy_type == TS2_OUT_F16) {
                const __half c[4] = {narrow<__half>(p[0]), narrow<__half>(p[1]), narrow<__half>(p[2]), narrow<__half>(p[3])};
                store4((__half *)r.copy, j, n, whole, c);
            } else {
                const __nv_bfloat16 c[4] = {narrow<__nv_bfloat16>(p[0]), narrow<__nv_bfloat16>(p[1]), narrow<__nv_bfloat16>(p[2]), narrow<__nv_bfloat16>(p[3])};
                store4((__nv_bfloat16 *)r.copy, j, n, whole, c);
            }
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
        const uint64_t mine = (uint64_t)ceil_div(t.n, CHUNK); // 2^28 at most
        if (!mine)
            continue;
        if (a.n == 400 || chunks + mine > 0x7fffffffu)
            if (const int rc = flush())
                return rc;
        AdamwRecord &r = table.r[a.n++];
        r.param = t.param, r.grad = t.grad, r.m = t.m, r.v = t.v, r.m_scale = t.m_scale, r.v_scale = t.v_scale, r.copy = t.copy, r.n = t.n;
        r.chunk0 = (uint32_t)chunks;
        r.key = (uint32_t)mix64(mix64(seed + (uint64_t)step) ^ (uint64_t)i);
        r.keep = (float)(1. - (double)rate * t.rate * t.decay);
        r.rate = (float)((double)rate * t.rate / c1);
        chunks += mine;
    }
    return flush();
}

} // namespace ts2
