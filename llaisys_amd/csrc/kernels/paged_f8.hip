// Append, gather and block copy of the 8-bit paged KV (f8_page.hpp has the
// format).
#include "f8_page.hpp"
#include "mfma_common.hpp"

#include "../device/hip_check.hpp"

#include <type_traits>

namespace llaisys::kernels {

namespace {

using namespace mfma;

typedef float f32x2 __attribute__((ext_vector_type(2)));

// ---------------------------------------------------------------- append

// Four values to e4m3 codes, the first in the low byte. Rounds to the nearest
// code, ties to even; |v| <= 448 or NaN.
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d) {
    const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return uint32_t(__builtin_amdgcn_cvt_pk_fp8_f32(c, d, lo, true));
}

// Four codes of a block whose scale was multiplied by 1 / f (f a power of two).
__device__ __forceinline__ uint32_t recode4(uint32_t w, float f) {
    const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(int(w), false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(int(w), true);
    return encode4(lo[0] * f, lo[1] * f, hi[0] * f, hi[1] * f);
}

// bf16 bits times f (a power of two); not finite: NaN.
__device__ __forceinline__ float scaled(uint32_t bits, float f) {
    const float x = __uint_as_float(bits << 16);
    return (bits & 0x7f80u) == 0x7f80u ? __uint_as_float(0x7fc00000u) : x * f;
}

constexpr int kRowPitch = kHeadDim + 8; // LDS row of 128 bf16, 16 B on

// A workgroup looks at ROWS rows of one kv head and writes the runs of
// consecutive slots of a block that begin among them, one after the other. Two
// waves hold the K page, two the V page, 16 B of it per thread. The largest
// magnitude of the run's rows and the block's scale give the new scale; if it
// grew, every code of the page is re-encoded. Bound by latency: slots, then
// rows and page together, then the stores. One row per workgroup where every
// row begins a run (64 rows 3.5 us); eight where most only continue one and
// 2048 workgroups hold them all at once (8170 rows, 2 kv heads: 12.2 us with
// one, whose idle workgroups take eight rounds).
template <int ROWS>
__global__ void __launch_bounds__(256)
    appendF8Kernel(uint8_t *__restrict__ k_pool, uint8_t *__restrict__ v_pool, float *__restrict__ k_scale,
                   float *__restrict__ v_scale, const uint16_t *__restrict__ k_new, const uint16_t *__restrict__ v_new,
                   const int64_t *__restrict__ slots, int T, int nkvh, int num_blocks, int *err) {
    static_assert(kF8LookBack + ROWS - 1 + kPageTokens <= 64, "a lane per slot");
    __shared__ __align__(16) uint16_t rows[2][kPageTokens][kRowPitch];
    __shared__ int tops[4];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r0 = int(blockIdx.x) * ROWS, h = blockIdx.y;
    const bool is_v = wave >= 2;
    const int i = tid & 127;
    // Lane l: the slot of row r0 + l - kF8LookBack.
    int64_t slot = -1;
    const int seen = r0 + lane - kF8LookBack;
    if (seen >= 0 && seen < T) slot = slots[seen];
    const int64_t prev = __shfl_up(slot, 1);
    const bool begins = lane >= kF8LookBack && lane < kF8LookBack + ROWS && slot >= 0 &&
                        !(prev >= 0 && prev + 1 == slot && (slot & 15) != 0);
    bool again = false;
    for (unsigned long long todo = __ballot(begins); todo; todo &= todo - 1) {
        const int l = __ffsll(todo) - 1, r = r0 + l - kF8LookBack;
        const int64_t mine = __shfl(slot, l);
        const int64_t block = mine >> 4;
        const int off = int(mine & 15);
        if (block >= num_blocks) {
            if (tid == 0 && h == 0) atomicOr(err, kErrBadBlock);
            continue;
        }
        if (__ballot(lane < l && lane >= l - kF8LookBack && slot >= 0 && (slot >> 4) == block)) {
            if (tid == 0 && h == 0) atomicOr(err, kErrTooLong); // a second run of the block
            continue;
        }
        const unsigned long long run = __ballot(lane >= l && lane < l + kPageTokens - off && slot == mine + (lane - l));
        const int n = __ffsll(~(run >> l)) - 1; // rows of the run

        uint8_t *page = (is_v ? v_pool : k_pool) + (size_t(block) * nkvh + h) * kF8PageBytes;
        float *scale = (is_v ? v_scale : k_scale) + size_t(block) * nkvh + h;
        const u32x4 old_codes = reinterpret_cast<const u32x4 *>(page)[i];
        const float old_scale = *scale;
        // Rows to LDS, by slot: thread (slot t, eighth p) moves 16 dims.
        const int t = i >> 3, p = i & 7;
        int top = 0;
        u32x4 x[2] = {};
        if (t >= off && t < off + n) {
            const uint16_t *src = (is_v ? v_new : k_new) + (size_t(r + t - off) * nkvh + h) * kHeadDim + p * 16;
#pragma unroll
            for (int j = 0; j < 2; ++j) x[j] = reinterpret_cast<const u32x4 *>(src)[j];
        }
        if (again) __syncthreads(); // the run before has been read
        again = true;
        if (t >= off && t < off + n) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                *reinterpret_cast<u32x4 *>(&rows[is_v][t][p * 16 + 8 * j]) = x[j];
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const int lo = int(x[j][w] & 0x7fffu), hi = int((x[j][w] >> 16) & 0x7fffu);
                    top = max(top, lo < 0x7f80 ? lo : 0);
                    top = max(top, hi < 0x7f80 ? hi : 0);
                }
            }
        }
        top = waveMaxInt(top);
        if (lane == 0) tops[wave] = top;
        __syncthreads();
        top = max(tops[wave & 2], tops[wave | 1]);
        const int was = off == 0 ? kF8LeastExp : f8ExpOfScale(old_scale);
        const int now = max(was, f8ExpOf(top));
        const float f = f8Exp2(-now);
        const bool recode = now != was && off != 0;
        const float fr = f8Exp2(max(was - now, -126));
        u32x4 codes = old_codes;
        if (recode) {
#pragma unroll
            for (int w = 0; w < 4; ++w) codes[w] = recode4(codes[w], fr);
        }
        bool store = recode;
        if (!is_v) {
            // 16 B of one token: dims 64 half + 8 g + (0..7) and 32 further.
            const int tok = i & 15, half = i >> 6, g = (i >> 4) & 3;
            if (tok >= off && tok < off + n) {
                store = true;
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const u32x4 y = *reinterpret_cast<const u32x4 *>(&rows[0][tok][64 * half + 32 * j + 8 * g]);
#pragma unroll
                    for (int w = 0; w < 2; ++w)
                        codes[2 * j + w] = encode4(scaled(y[2 * w] & 0xffff, f), scaled(y[2 * w] >> 16, f),
                                                   scaled(y[2 * w + 1] & 0xffff, f), scaled(y[2 * w + 1] >> 16, f));
                }
            }
        } else {
            // Four tokens 4 g + (0..3) of dims 64 half + 16 w + n16.
            const int half = i >> 6, g = (i >> 4) & 3, n16 = i & 15;
            uint32_t keep = 0xffffffffu; // bytes of tokens that are not new
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (4 * g + e >= off && 4 * g + e < off + n) keep &= ~(0xffu << (8 * e));
            if (keep != 0xffffffffu) {
                store = true;
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    float y[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        y[e] = (keep >> (8 * e)) & 1 ? 0.f : scaled(rows[1][4 * g + e][64 * half + 16 * w + n16], f);
                    codes[w] = (codes[w] & keep) | (encode4(y[0], y[1], y[2], y[3]) & ~keep);
                }
            }
        }
        if (store) reinterpret_cast<u32x4 *>(page)[i] = codes;
        if (i == 0) *scale = f8Exp2(now);
    }
}

// ---------------------------------------------------------------- gather

// One 256-thread workgroup per (page, sequence, kv head): the pages go through
// LDS as bf16 rows and out row by row. Bound by HBM: 32 sequences of up to 2048
// tokens, 2 kv heads, 50 MB in 10 us.
__global__ void __launch_bounds__(256)
    gatherF8Kernel(uint16_t *__restrict__ k_out, uint16_t *__restrict__ v_out, const uint8_t *__restrict__ k_pool,
                   const uint8_t *__restrict__ v_pool, const float *__restrict__ k_scale,
                   const float *__restrict__ v_scale, const int32_t *__restrict__ table,
                   const int32_t *__restrict__ cu, int T, int nkvh, int max_pages, int num_blocks, int *err) {
    __shared__ __align__(16) uint16_t rows[2][kPageTokens][kRowPitch];
    const int page = blockIdx.x, b = blockIdx.y, h = blockIdx.z, tid = threadIdx.x;
    const int blk = table[size_t(b) * max_pages + page];
    const int row0 = cu[b];
    const int len = cu[b + 1] - row0;
    if (page * 16 >= len) return;
    if (row0 < 0 || cu[b + 1] > T) { // rows outside k_out/v_out: refuse the sequence
        if (tid == 0) atomicOr(err, kErrTooLong);
        return;
    }
    if (page == max_pages - 1 && len > max_pages * 16 && tid == 0) atomicOr(err, kErrTooLong);
    if (blk < 0 || blk >= num_blocks) {
        if (tid == 0) atomicOr(err, kErrBadBlock);
        return;
    }
    const bool is_v = tid >= 128;
    const int i = tid & 127;
    const size_t unit = size_t(blk) * nkvh + h;
    const u32x4 x = reinterpret_cast<const u32x4 *>((is_v ? v_pool : k_pool) + unit * kF8PageBytes)[i];
    const float scale = (is_v ? v_scale : k_scale)[unit];
    const int half = i >> 6, g = (i >> 4) & 3, n16 = i & 15;
    uint32_t y[8];
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        y[2 * w] = widen2<false>(x[w], scale);
        y[2 * w + 1] = widen2<true>(x[w], scale);
    }
    if (!is_v) {
#pragma unroll
        for (int j = 0; j < 2; ++j)
            *reinterpret_cast<u32x4 *>(&rows[0][n16][64 * half + 32 * j + 8 * g]) =
                u32x4{y[4 * j], y[4 * j + 1], y[4 * j + 2], y[4 * j + 3]};
    } else {
#pragma unroll
        for (int w = 0; w < 4; ++w)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                rows[1][4 * g + e][64 * half + 16 * w + n16] = uint16_t(y[2 * w + (e >> 1)] >> (16 * (e & 1)));
    }
    __syncthreads();
    const int t = tid >> 4, c = tid & 15;
    if (page * 16 + t >= len) return;
    const size_t dst = (size_t(row0 + page * 16 + t) * nkvh + h) * kHeadDim + c * 8;
    *reinterpret_cast<u32x4 *>(k_out + dst) = *reinterpret_cast<const u32x4 *>(&rows[0][t][c * 8]);
    *reinterpret_cast<u32x4 *>(v_out + dst) = *reinterpret_cast<const u32x4 *>(&rows[1][t][c * 8]);
}

// ------------------------------------------------------------- copy blocks

// One 256-thread workgroup per (pair, pool): a copy, bound by its launch at the
// few pairs of a step.
__global__ void __launch_bounds__(256)
    copyBlocksF8Kernel(uint8_t *k_pool, uint8_t *v_pool, float *k_scale, float *v_scale,
                       const int32_t *__restrict__ pairs, int nkvh, int num_blocks, int *err) {
    const int src = pairs[2 * blockIdx.x], dst = pairs[2 * blockIdx.x + 1];
    if (src < 0 || src >= num_blocks || dst < 0 || dst >= num_blocks) {
        if (threadIdx.x == 0) atomicOr(err, kErrBadBlock);
        return;
    }
    uint4 *pool = reinterpret_cast<uint4 *>(blockIdx.y == 0 ? k_pool : v_pool);
    float *scale = blockIdx.y == 0 ? k_scale : v_scale;
    const size_t per_block = size_t(nkvh) * kF8PageBytes / 16;
    for (size_t i = threadIdx.x; i < per_block; i += 256) pool[dst * per_block + i] = pool[src * per_block + i];
    for (int h = threadIdx.x; h < nkvh; h += 256) scale[size_t(dst) * nkvh + h] = scale[size_t(src) * nkvh + h];
}

} // namespace

void pagedAppendF8(uint8_t *k_pool, uint8_t *v_pool, float *k_scale, float *v_scale, const uint16_t *k_new,
                   const uint16_t *v_new, const int64_t *slots, int T, int nkvh, int num_blocks, int *err,
                   void *stream) {
    if (T == 0) return;
    auto launch = [&](auto rows) {
        constexpr int ROWS = decltype(rows)::value;
        hipLaunchKernelGGL(appendF8Kernel<ROWS>, dim3(unsigned((T + ROWS - 1) / ROWS), unsigned(nkvh)), dim3(256), 0,
                           static_cast<hipStream_t>(stream), k_pool, v_pool, k_scale, v_scale, k_new, v_new, slots, T,
                           nkvh, num_blocks, err);
    };
    if ((long long)T * nkvh <= 1024)
        launch(std::integral_constant<int, 1>());
    else
        launch(std::integral_constant<int, 8>());
    HIP_CHECK(hipGetLastError());
}

void pagedGatherF8(uint16_t *k_out, uint16_t *v_out, const uint8_t *k_pool, const uint8_t *v_pool,
                   const float *k_scale, const float *v_scale, const int32_t *block_table, const int32_t *cu_seqlens,
                   int T, int B, int nkvh, int max_pages, int num_blocks, int *err, void *stream) {
    if (B == 0 || max_pages == 0) return;
    hipLaunchKernelGGL(gatherF8Kernel, dim3(unsigned(max_pages), unsigned(B), unsigned(nkvh)), dim3(256), 0,
                       static_cast<hipStream_t>(stream), k_out, v_out, k_pool, v_pool, k_scale, v_scale, block_table,
                       cu_seqlens, T, nkvh, max_pages, num_blocks, err);
    HIP_CHECK(hipGetLastError());
}

void pagedCopyBlocksF8(uint8_t *k_pool, uint8_t *v_pool, float *k_scale, float *v_scale, const int32_t *pairs, int P,
                       int nkvh, int num_blocks, int *err, void *stream) {
    if (P == 0) return;
    hipLaunchKernelGGL(copyBlocksF8Kernel, dim3(unsigned(P), 2), dim3(256), 0, static_cast<hipStream_t>(stream),
                       k_pool, v_pool, k_scale, v_scale, pairs, nkvh, num_blocks, err);
    HIP_CHECK(hipGetLastError());
}

} // namespace llaisys::kernels
