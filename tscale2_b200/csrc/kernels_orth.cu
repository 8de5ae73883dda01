// Orthogonalised updates by Newton-Schulz products.  Every matrix G of a batch becomes U p(p(..p(S / |G|)..)) V^T, where G = U S V^T
// and p(s) = a s + b s^3 + c s^5 acts on each singular value: with |G| the Frobenius norm
//     X = G / |G|;   `steps` times:  A = X X^T,  B = b A + c A A,  X = a X + B X
// in the orientation with fewer rows than columns.  A zero matrix gives zeros.
//
// The products are fp16 with fp32 sums on the tensor cores.  X itself is kept in 32 bits, as two halves: small singular values
// are carried by the term a X and grow by a factor a in every step, so one rounding of X to 16 bits grows with them (a spectrum
// that falls off as 1/k^2, 512 x 1024, coefficients 3.4445, -4.7750, 2.0315, 5 steps: relative error 2.0e-2 with X in fp16,
// 1.8e-4 with X in two halves; flat spectra 2.0e-3 and 1.3e-3).  All fp16 values are scaled by powers of two that keep them
// below 65504 for every X the coefficients can reach (orth_check).
#include "kernels.cuh"
#include "gemm.cuh"
#include <algorithm>
#include <cmath>

namespace ts2 {

// X, A = X X^T and B as they are stored: value * 2^14, 2^12, 2^11; |X| <= 3.9, |B| <= 31
static constexpr float SX = 16384.f, SA = 4096.f, SB = 2048.f;
static constexpr float MAX_X = 3.9f, MAX_B = 31.f;
static constexpr float LO = 2048.f; // the low half is stored times 2^11: its values are below 2^-11 of the high half's

template <class T>
__device__ __forceinline__ float widen(T v) { return (float)v; }

__device__ __forceinline__ void split(float x, __half &hi, __half &lo)
{
    hi = __low2half(sat_half2(x, x));
    const float r = (x - __half2float(hi)) * LO;
    lo = __low2half(sat_half2(r, r));
}
__device__ __forceinline__ float joined(__half hi, __half lo) { return fmaf(__half2float(lo), 1.f / LO, __half2float(hi)); }

// ---- G -> X ----------------------------------------------------------------------------------------------------------
// partial sums of squares in fp64: no input over- or underflows, and nothing is lost over 2^32 terms
template <class T>
__global__ void __launch_bounds__(256) orth_sum2_kernel(const T *__restrict__ g, long long ld, long long stride, int rows, int cols, double *part)
{
    grid_dep_wait();
    __shared__ double warps[8];
    g += blockIdx.y * stride;
    double sum = 0.;
    for (int r = blockIdx.x; r < rows; r += gridDim.x)
        for (int c = threadIdx.x; c < cols; c += 256) {
            const double v = widen(g[r * ld + c]);
            sum += v * v;
        }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if ((threadIdx.x & 31) == 0)
        warps[threadIdx.x >> 5] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 8; ++w)
            sum += warps[w];
        part[blockIdx.y * gridDim.x + blockIdx.x] = sum;
    }
}

// 32 x 32 blocks of X [n][m] (padded to np x mp with zeros) from G, transposed where G has more rows than columns
template <class T>
__global__ void __launch_bounds__(256) orth_load_kernel(const T *__restrict__ g, long long ld, long long stride, int rows, int cols, bool tall,
                                                        const double *part, int n_part, int np, int mp, __half *hi, __half *lo)
{
    grid_dep_wait();
    __shared__ float tile[32][33];
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5, b = blockIdx.z;
    double sum = 0.;
    for (int i = 0; i < n_part; ++i)
        sum += part[b * n_part + i];
    const double scale = sum == 0. ? 0. : SX / sqrt(sum);
    const int i0 = blockIdx.y * 32, j0 = blockIdx.x * 32; // rows and columns of X
    g += b * stride;
    for (int k = ty; k < 32; k += 8) {
        const int r = (tall ? j0 : i0) + k, c = (tall ? i0 : j0) + tx;
        tile[k][tx] = r < rows && c < cols ? (float)(widen(g[r * ld + c]) * scale) : 0.f;
    }
    __syncthreads();
    for (int k = ty; k < 32; k += 8) {
        const size_t at = ((size_t)b * np + i0 + k) * mp + j0 + tx;
        split(tall ? tile[tx][k] : tile[k][tx], hi[at], lo[at]);
    }
}

__global__ void __launch_bounds__(256) orth_store_kernel(const __half *__restrict__ hi, const __half *__restrict__ lo, int np, int mp, bool tall,
                                                         float scale, __nv_bfloat16 *out, long long ld, long long stride, int rows, int cols)
{
    grid_dep_wait();
    __shared__ float tile[32][33];
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5, b = blockIdx.z;
    const int i0 = blockIdx.y * 32, j0 = blockIdx.x * 32;
    for (int k = ty; k < 32; k += 8) {
        const size_t at = ((size_t)b * np + i0 + k) * mp + j0 + tx;
        tile[k][tx] = joined(hi[at], lo[at]) * scale;
    }
    __syncthreads();
    out += b * stride;
    for (int k = ty; k < 32; k += 8) {
        const int r = (tall ? j0 : i0) + k, c = (tall ? i0 : j0) + tx;
        if (r < rows && c < cols)
            out[r * ld + c] = __float2bfloat16_rn(tall ? tile[tx][k] : tile[k][tx]);
    }
}

// B = b A + c A A
__global__ void __launch_bounds__(256) orth_poly_kernel(const __half *__restrict__ a, const float *__restrict__ aa, size_t n, float b, float c,
                                                        __half *out)
{
    grid_dep_wait();
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (size_t)gridDim.x * 256) {
        const float v = SB * (b / SA * __half2float(a[i]) + c / (SA * SA) * aa[i]);
        out[i] = __low2half(sat_half2(v, v));
    }
}
// X = a X + B X
__global__ void __launch_bounds__(256) orth_update_kernel(__half *hi, __half *lo, const float *__restrict__ bx, size_t n, float a)
{
    grid_dep_wait();
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (size_t)gridDim.x * 256)
        split(fmaf(a, joined(hi[i], lo[i]), bx[i] * (1.f / SB)), hi[i], lo[i]);
}

// ---- host ------------------------------------------------------------------------------------------------------------
// largest |a s + b s^3 + c s^5| (odd) or |b q + c q^2| over [0, top]: at the end or where the derivative is zero
static double poly_max(double a, double b, double c, double top)
{
    const auto p = [&](double s) { return std::fabs(s * (a + s * s * (b + s * s * c))); };
    double most = p(top);
    const double disc = 9 * b * b - 20 * a * c;
    if (disc >= 0) {
        const double root[3] = {c ? (-3 * b + std::sqrt(disc)) / (10 * c) : -1, c ? (-3 * b - std::sqrt(disc)) / (10 * c) : -1,
                                b ? -a / (3 * b) : -1};
        for (int i = c ? 0 : 2; i < (c ? 2 : 3); ++i)
            if (root[i] > 0 && root[i] < top * top)
                most = std::max(most, p(std::sqrt(root[i])));
    }
    return most;
}
static bool orth_check(const float coef[3], int steps)
{
    double x = 1.;
    for (int k = 0; k < steps; ++k) {
        x *= 1.02; // the roundings of a step move a singular value by less
        const double q = x * x, b = coef[1], c = coef[2];
        double most = std::fabs(b * q + c * q * q);
        if (c && -b / (2 * c) > 0 && -b / (2 * c) < q)
            most = std::max(most, b * b / (4 * std::fabs(c)));
        if (!(x <= MAX_X) || !(most <= MAX_B))
            return false;
        x = poly_max(coef[0], b, c, x);
    }
    return x * 1.02 <= MAX_X;
}

struct Scratch {
    void *p = nullptr;
    cudaStream_t stream;
    int rc;
    Scratch(const Ctx &c, size_t bytes) : stream(c.stream) { rc = scratch_alloc(c.device, bytes, c.stream, &p); }
    ~Scratch()
    {
        if (p)
            scratch_free(stream, p);
    }
    Scratch(const Scratch &) = delete;
    Scratch &operator=(const Scratch &) = delete;
};

template <class T>
static int orthogonalize_typed(const Ctx &c, const T *g, int64_t ld, int64_t stride, int batch, int rows, int cols, const float coef[3], int steps,
                               float out_scale, __nv_bfloat16 *out, int64_t ld_out, int64_t out_stride)
{
    const bool tall = rows > cols;
    const int n = std::min(rows, cols), m = std::max(rows, cols), np = (int)ceil_div(n, 128) * 128, mp = (int)ceil_div(m, 128) * 128;
    const int n_part = std::min(rows, 64);
    const size_t x = (size_t)np * mp, a = (size_t)np * np;
    size_t ws = gemm_workspace_bytes(c.device, KIND_F16, false, np, np, mp);
    ws = std::max(ws, gemm_workspace_bytes(c.device, KIND_F16, false, np, np, np));
    ws = (std::max(ws, gemm_workspace_bytes(c.device, KIND_F16, true, np, mp, np)) + 255) / 256 * 256;
    Scratch s(c, ws + batch * x * 4 + a * 4 + x * 4 + (size_t)batch * n_part * 8);
    if (s.rc != TS2_OK)
        return s.rc;
    __half *hi = (__half *)((uint8_t *)s.p + ws), *lo = hi + batch * x, *A = lo + batch * x, *B = A + a;
    float *prod = (float *)(B + a);
    double *part = (double *)(prod + x);

    TS2_LAUNCH((orth_sum2_kernel<T>), dim3(n_part, batch), 256, 0, c.stream, g, ld, stride, rows, cols, part);
    TS2_LAUNCH((orth_load_kernel<T>), dim3(mp / 32, np / 32, batch), 256, 0, c.stream, g, ld, stride, rows, cols, tall, part, n_part, np, mp, hi, lo);
    GemmArgs p;
    p.device = c.device, p.stream = c.stream, p.kind = KIND_F16, p.workspace = s.p, p.workspace_bytes = ws;
    const int grid = sm_count(c.device) * 8;
    for (int i = 0; i < batch; ++i) {
        __half *xh = hi + i * x, *xl = lo + i * x;
        for (int k = 0; k < steps; ++k) {
            p.mn_major = false;
            p.M = p.N = np, p.K = mp, p.A = p.B = xh, p.lda = p.ldb = mp, p.C = A, p.ldc = np;
            p.epi.out_kind = TS2_OUT_F16, p.epi.alpha = SA / (SX * SX);
            if (int rc = gemm(p))
                return rc;
            p.K = np, p.A = p.B = A, p.lda = p.ldb = np, p.C = prod;
            p.epi.out_kind = TS2_OUT_F32, p.epi.alpha = 1.f;
            if (int rc = gemm(p))
                return rc;
            TS2_LAUNCH(orth_poly_kernel, (unsigned)std::min<size_t>(grid, a / 256), 256, 0, c.stream, A, prod, a, coef[1], coef[2], B);
            p.mn_major = true; // B is its own transpose
            p.N = mp, p.A = B, p.B = xh, p.ldb = p.ldc = mp;
            if (int rc = gemm(p))
                return rc;
            TS2_LAUNCH(orth_update_kernel, (unsigned)std::min<size_t>(grid, x / 256), 256, 0, c.stream, xh, xl, prod, x, coef[0]);
        }
    }
    TS2_LAUNCH(orth_store_kernel, dim3(mp / 32, np / 32, batch), 256, 0, c.stream, hi, lo, np, mp, tall, out_scale / SX, out, ld_out, out_stride, rows,
               cols);
    return TS2_OK;
}

int orthogonalize(const Ctx &c, int type, const void *g, int64_t ld, int64_t stride, int batch, int rows, int cols, const float coef[3], int steps,
                  float out_scale, void *out, int64_t ld_out, int64_t out_stride)
{
    if (!orth_check(coef, steps))
        return fail(TS2_ERR_UNSUPPORTED, "orthogonalize: the coefficients take singular values beyond %g", (double)MAX_X);
    __nv_bfloat16 *o = (__nv_bfloat16 *)out;
    switch (type) {
    case TS2_OUT_F32: return orthogonalize_typed(c, (const float *)g, ld, stride, batch, rows, cols, coef, steps, out_scale, o, ld_out, out_stride);
    case TS2_OUT_F16: return orthogonalize_typed(c, (const __half *)g, ld, stride, batch, rows, cols, coef, steps, out_scale, o, ld_out, out_stride);
    case TS2_OUT_BF16:
        return orthogonalize_typed(c, (const __nv_bfloat16 *)g, ld, stride, batch, rows, cols, coef, steps, out_scale, o, ld_out, out_stride);
    default: return fail(TS2_ERR_INVALID_ARG, "orthogonalize: unknown type %d", type);
    }
}

} // namespace ts2
