// Rows of floats to 8-bit integers with a scale each.
//
// q = x / s to the nearest whole number, ties to even, s = top / 127 rounded
// to 32 bits. The quotient in 32 bits can land on a tie that the exact one
// misses, or leave one that it is; the remainder x - q s decides: it is exact
// (its bits reach from those of s to half of s), so q is the exact quotient's
// rounding whatever the division did.
//
// A row is read once and its codes written once: a thread keeps its pieces of
// the row (16 B each) in registers from the search for the largest magnitude
// to the codes; what goes past kPieces of them is read again, from the caches.
// Bound by HBM where there are many rows (8192 x 1536 bf16, 38 MB, 14.4 us; a
// copy of them 8) and by one row's latency where there are few (1 x 8960 2.7 us).
#include "launch.hpp"
#include "mfma_common.hpp"

#include "../device/hip_check.hpp"

#include <hip/hip_runtime.h>

#include <algorithm>

namespace llaisys::kernels {

namespace {

using mfma::u32x4;

template <ElemType T> struct Elem;
template <> struct Elem<ElemType::BF16> { using type = __bf16; };
template <> struct Elem<ElemType::F16> { using type = _Float16; };
template <> struct Elem<ElemType::F32> { using type = float; };

constexpr int kPieces = 5; // of a thread, in registers

// x / s to the nearest whole number (|x| <= 127.5 s, s > 0); inv about 1 / s.
__device__ __forceinline__ int quantized(float x, float s, float inv) {
    float q = rintf(x * inv);
    const float rest = fmaf(-q, s, x), twice = 2.f * fabsf(rest);
    const bool odd = int(q) & 1;
    if (twice > s || (twice == s && odd)) q += copysignf(1.f, rest);
    return int(fminf(fmaxf(q, -127.f), 127.f));
}

// The same where x inv is not next to a tie, which it says: the product plus
// 1.5 * 2^23 has the nearest whole number in its low bits. inv is off by 2^-24
// of itself, so |x| inv <= 127 by 2^-17 at most.
constexpr float kShift = 12582912.f, kSure = 0.5f - 0x1p-16f;
__device__ __forceinline__ uint32_t quantizedFast(float x, float inv, float &far) {
    const float y = fmaf(x, inv, kShift);
    far = fmaxf(far, fabsf(fmaf(x, inv, kShift - y)));
    return __float_as_uint(y);
}

// Largest over the 64 lanes of numbers >= 0 (as bits, which order as they do).
__device__ __forceinline__ uint32_t waveMax(uint32_t bits) { return uint32_t(mfma::waveMaxInt(int(bits))); }

// A row by WAVES waves (WAVES == 1: four rows a workgroup). VEC: rows of whole
// 16 B pieces, aligned; else piece by piece of one element.
template <ElemType T, int WAVES, bool VEC>
__global__ void __launch_bounds__(WAVES == 1 ? 256 : 64 * WAVES)
    quantizeRowsKernel(int8_t *__restrict__ q, float *__restrict__ scale, const void *__restrict__ x, int M, int K) {
    using E = typename Elem<T>::type;
    constexpr int EL = VEC ? 16 / int(sizeof(E)) : 1; // elements of a piece
    constexpr int THREADS = 64 * WAVES;
    __shared__ float tops[WAVES];
    const int tid = WAVES == 1 ? int(threadIdx.x & 63) : int(threadIdx.x);
    const int m = WAVES == 1 ? int(blockIdx.x) * 4 + int(threadIdx.x >> 6) : int(blockIdx.x);
    if (m >= M) return;
    const E *row = static_cast<const E *>(x) + size_t(m) * K;
    int8_t *to = q + size_t(m) * K;
    const int pieces = K / EL;
    struct Piece {
        E e[EL];
    };
    auto load = [&](int p) {
        Piece r;
        if constexpr (VEC)
            r = __builtin_bit_cast(Piece, reinterpret_cast<const u32x4 *>(row)[p]);
        else
            r.e[0] = row[p];
        return r;
    };
    // The largest magnitude as bits: they order as the numbers do, and those of
    // infinities and NaNs come last.
    uint32_t top = 0;
    auto search = [&](const Piece &r) {
#pragma unroll
        for (int e = 0; e < EL; ++e) top = max(top, __float_as_uint(float(r.e[e])) & 0x7fffffffu);
    };
    Piece held[kPieces] = {};
    if (pieces > 0) { // (past the row its last piece again)
#pragma unroll
        for (int i = 0; i < kPieces; ++i) held[i] = load(min(tid + i * THREADS, pieces - 1));
#pragma unroll
        for (int i = 0; i < kPieces; ++i) search(held[i]);
    }
    for (int p = tid + kPieces * THREADS; p < pieces; p += THREADS) search(load(p));
    top = waveMax(top);
    if constexpr (WAVES > 1) {
        if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = __uint_as_float(top);
        __syncthreads();
#pragma unroll
        for (int w = 0; w < WAVES; ++w) top = max(top, __float_as_uint(tops[w]));
    }
    const bool finite = top < 0x7f800000u;
    const float most = __uint_as_float(top);
    const float s = finite ? most / 127.f : __uint_as_float(0x7fc00000u);
    if (tid == 0) scale[m] = s;
    // Rows of very small values: the same quotients from larger numbers, whose inverse is finite.
    const float grow = most < 0x1p-60f ? 0x1p80f : 1.f, sg = s * grow, inv = 1.f / sg;
    const bool some = finite && s > 0.f;
    // (A scale of few bits, next to underflow, gives quotients past 127.)
    const bool plain = some && s >= 0x1p-110f;
    auto store = [&](int p, const Piece &r) {
        uint32_t w[EL > 4 ? 2 : 1] = {};
        float far = plain ? 0.f : 1.f;
        if (plain) {
            uint32_t c[EL];
#pragma unroll
            for (int e = 0; e < EL; ++e) c[e] = quantizedFast(float(r.e[e]) * grow, inv, far);
#pragma unroll
            for (int e = 0; e < EL; e += 4) {
                if constexpr (EL >= 4)
                    w[e / 4] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(c[e + 3], c[e + 2], 0x0c0c0400u),
                                                     __builtin_amdgcn_perm(c[e + 1], c[e], 0x0c0c0400u), 0x05040100u);
                else
                    w[0] = c[e];
            }
        }
        if (far > kSure) {
#pragma unroll
            for (int e = 0; e < (EL > 4 ? 2 : 1); ++e) w[e] = 0;
#pragma unroll
            for (int e = 0; e < EL; ++e) {
                const int c = some ? quantized(float(r.e[e]) * grow, sg, inv) : 0;
                w[e / 4] |= (uint32_t(c) & 0xffu) << (8 * (e & 3));
            }
        }
        if constexpr (EL == 8)
            reinterpret_cast<uint2 *>(to)[p] = make_uint2(w[0], w[1]);
        else if constexpr (EL == 4)
            reinterpret_cast<uint32_t *>(to)[p] = w[0];
        else
            to[p] = int8_t(w[0]);
    };
#pragma unroll
    for (int i = 0; i < kPieces; ++i)
        if (tid + i * THREADS < pieces) store(tid + i * THREADS, held[i]);
    for (int p = tid + kPieces * THREADS; p < pieces; p += THREADS) store(p, load(p));
}

template <ElemType T, bool VEC>
void launchQuantize(int8_t *q, float *scale, const void *x, int M, int K, hipStream_t s) {
    const int pieces = VEC ? K / (16 / int(sizeof(typename Elem<T>::type))) : K;
    // As many waves as hold the row (1500 x 8960: a wave per row, reading most
    // of it twice, 14.6 us).
    if (pieces <= 64 * kPieces)
        hipLaunchKernelGGL((quantizeRowsKernel<T, 1, VEC>), dim3(unsigned((M + 3) / 4)), dim3(256), 0, s, q, scale, x, M, K);
    else if (pieces <= 256 * kPieces)
        hipLaunchKernelGGL((quantizeRowsKernel<T, 4, VEC>), dim3(unsigned(M)), dim3(256), 0, s, q, scale, x, M, K);
    else
        hipLaunchKernelGGL((quantizeRowsKernel<T, 16, VEC>), dim3(unsigned(M)), dim3(1024), 0, s, q, scale, x, M, K);
    HIP_CHECK(hipGetLastError());
}

template <ElemType T> void quantizeAs(int8_t *q, float *scale, const void *x, int M, int K, hipStream_t s) {
    constexpr int es = int(sizeof(typename Elem<T>::type));
    const bool vec = size_t(K) * es % 16 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0 &&
                     reinterpret_cast<uintptr_t>(q) % (16 / es) == 0;
    if (vec)
        launchQuantize<T, true>(q, scale, x, M, K, s);
    else
        launchQuantize<T, false>(q, scale, x, M, K, s);
}

} // namespace

void quantizeRows(int8_t *q, float *scale, const void *x, ElemType t, int M, int K, void *stream) {
    if (M == 0) return;
    auto s = static_cast<hipStream_t>(stream);
    switch (t) {
    case ElemType::F32: quantizeAs<ElemType::F32>(q, scale, x, M, K, s); break;
    case ElemType::F16: quantizeAs<ElemType::F16>(q, scale, x, M, K, s); break;
    case ElemType::BF16: quantizeAs<ElemType::BF16>(q, scale, x, M, K, s); break;
    }
}

} // namespace llaisys::kernels
