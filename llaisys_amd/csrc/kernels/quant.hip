// Rows of floats to 8-bit integers with a scale each.
//
// q = x / s to the nearest whole number, ties to even, s = top / 127 rounded
// to 32 bits. The quotient in 32 bits can land on a tie that the exact one
// misses, or leave one that it is; the remainder x - q s decides: it is exact
// (its bits reach from those of s to half of s), so q is the exact quotient's
// rounding whatever the division did.
#include "launch.hpp"

#include "../device/hip_check.hpp"

#include <hip/hip_runtime.h>

namespace llaisys::kernels {

namespace {

template <ElemType T> struct Elem;
template <> struct Elem<ElemType::BF16> { using type = __bf16; };
template <> struct Elem<ElemType::F16> { using type = _Float16; };
template <> struct Elem<ElemType::F32> { using type = float; };

// x / s to the nearest whole number (|x| <= 127.5 s, s > 0); inv about 1 / s.
__device__ __forceinline__ int quantized(float x, float s, float inv) {
    float q = rintf(x * inv);
    const float rest = fmaf(-q, s, x), twice = 2.f * fabsf(rest);
    const bool odd = int(q) & 1;
    if (twice > s || (twice == s && odd)) q += copysignf(1.f, rest);
    return int(fminf(fmaxf(q, -127.f), 127.f));
}

__device__ __forceinline__ float waveMax(float x) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) x = fmaxf(x, __shfl_xor(x, off));
    return x;
}

// One wave per row: its largest magnitude, then its codes.
template <ElemType T>
__global__ void __launch_bounds__(256) quantizeRowsKernel(int8_t *__restrict__ q, float *__restrict__ scale,
                                                          const void *__restrict__ x, int M, int K) {
    using E = typename Elem<T>::type;
    const int lane = threadIdx.x & 63;
    const int m = int(blockIdx.x) * 4 + int(threadIdx.x >> 6);
    if (m >= M) return;
    const E *row = static_cast<const E *>(x) + size_t(m) * K;
    int8_t *to = q + size_t(m) * K;
    float top = 0.f;
    bool finite = true;
    for (int k = lane; k < K; k += 64) {
        const float v = fabsf(float(row[k]));
        finite = finite && v < INFINITY;
        top = fmaxf(top, v);
    }
    top = waveMax(top);
    finite = __ballot(!finite) == 0;
    const float s = finite ? top / 127.f : __uint_as_float(0x7fc00000u);
    if (lane == 0) scale[m] = s;
    // Rows of very small values: the same quotients from larger numbers, whose inverse is finite.
    const float grow = top < 0x1p-60f ? 0x1p80f : 1.f, sg = s * grow, inv = 1.f / sg;
    const bool some = finite && s > 0.f;
    for (int k = lane; k < K; k += 64) to[k] = some ? int8_t(quantized(float(row[k]) * grow, sg, inv)) : int8_t(0);
}

} // namespace

void quantizeRows(int8_t *q, float *scale, const void *x, ElemType t, int M, int K, void *stream) {
    if (M == 0) return;
    const dim3 grid(unsigned((M + 3) / 4)), block(256);
    auto s = static_cast<hipStream_t>(stream);
    switch (t) {
    case ElemType::F32: hipLaunchKernelGGL(quantizeRowsKernel<ElemType::F32>, grid, block, 0, s, q, scale, x, M, K); break;
    case ElemType::F16: hipLaunchKernelGGL(quantizeRowsKernel<ElemType::F16>, grid, block, 0, s, q, scale, x, M, K); break;
    case ElemType::BF16: hipLaunchKernelGGL(quantizeRowsKernel<ElemType::BF16>, grid, block, 0, s, q, scale, x, M, K); break;
    }
    HIP_CHECK(hipGetLastError());
}

} // namespace llaisys::kernels
