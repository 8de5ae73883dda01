// What the kernels of the orthogonalised update share (kernels_orth.cu, kernels_orth_chip.cu).
#pragma once
#include "kernels.cuh"

namespace ts2 {

// X, A = X X^T and B = b A + c A A as fp16 holds them: value * 2^14, 2^12, 2^11; |X| <= 3.9, |B| <= 31
constexpr float ORTH_SX = 16384.f, ORTH_SA = 4096.f, ORTH_SB = 2048.f;
constexpr float ORTH_MAX_X = 3.9f, ORTH_MAX_B = 31.f;

// the form for matrices that a cluster holds: how many CTAs it takes (0: none), and the call
int orth_chip_ranks(int rows, int cols);
int orth_chip(const Ctx &c, int type, const void *g, int64_t ld, int64_t stride, int batch, int rows, int cols, const float coef[3], int steps,
              float out_scale, void *out, int64_t ld_out, int64_t out_stride);

#ifdef __CUDACC__
// x = hi + lo to 2^-22 of it: two fp16 halves as which the products take their operands.  The low half is below 2^-11 of the high one; at
// the scales above its smallest step, 2^-24, is 2^-35 of one.  A NaN stays one (hi), an infinity never comes here.
__device__ __forceinline__ void orth_split(float x, float y, __half2 &hi, __half2 &lo)
{
    hi = sat_half2(x, y);
    const float2 f = __half22float2(hi);
    lo = sat_half2(x - f.x, y - f.y);
}
__device__ __forceinline__ void orth_split8(const float (&v)[8], uint4 &hi, uint4 &lo)
{
    uint32_t h[4], l[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        __half2 a, b;
        orth_split(v[2 * k], v[2 * k + 1], a, b);
        h[k] = *(const uint32_t *)&a, l[k] = *(const uint32_t *)&b;
    }
    hi = make_uint4(h[0], h[1], h[2], h[3]), lo = make_uint4(l[0], l[1], l[2], l[3]);
}
__device__ __forceinline__ void orth_join8(uint4 hi, uint4 lo, float (&v)[8])
{
    const uint32_t h[4] = {hi.x, hi.y, hi.z, hi.w}, l[4] = {lo.x, lo.y, lo.z, lo.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const float2 a = __half22float2(*(const __half2 *)&h[k]), b = __half22float2(*(const __half2 *)&l[k]);
        v[2 * k] = a.x + b.x, v[2 * k + 1] = a.y + b.y;
    }
}

// 8 elements of a row from column c on as floats, zeros from column `cols` on; vec: 16-byte accesses are aligned
template <class T>
__device__ __forceinline__ void orth_load8(const T *row, int c, int cols, bool vec, float (&v)[8])
{
    if (vec && c + 8 <= cols) {
        constexpr int PER = 16 / sizeof(T);
#pragma unroll
        for (int i = 0; i < 8 / PER; ++i) {
            const uint4 raw = *(const uint4 *)(row + c + i * PER);
            const T *e = (const T *)&raw;
#pragma unroll
            for (int j = 0; j < PER; ++j)
                v[i * PER + j] = (float)e[j];
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            v[i] = c + i < cols ? (float)row[c + i] : 0.f;
    }
}
#endif

} // namespace ts2
