// Varlen attention over the 8-bit paged KV in one launch: a workgroup per
// (block of 16 TILES query columns, kv head), whose waves share the block's
// pages rather than its columns.
//
// Column n of a sequence is the (query, query head) pair n, pairs ordered
// query-major, so a single query is one tile that is partly empty: chunks and
// decodes take the same path. The UW waves take the block's page pairs in turn,
// straight from memory into registers, widen them to bf16 operands, keep a
// running (O, m, l) each, o = sum 2^(s-m) v and l = sum 2^(s-m), and merge them
// through LDS at the end. There are no item tables, no stage that waves wait
// for each other at, no partial records and no second launch; the persistent
// kernel spends some 20 us on those. The price is that every block reads its
// pages from L2 again and widens them for TILES tiles only (8 TILES in the
// persistent kernel), so wide tables go there (unitShape).
//
// What bounds it is the vector unit: widening, exponentials (128 of a tile's
// some 400 cycles per page pair) and rounding beside 256 cycles of matrix
// instructions, on two waves a SIMD. 12 query and 2 kv heads, us, here and the
// persistent kernel: a chunk of 777 queries 12.8, 27.5; 4 chunks of 512 after
// 4096 tokens beside 60 single queries 66.0, 77.9.
//
// Consecutive workgroups take the kv heads in turn, as consecutive workgroups go
// to the XCDs in turn: where the heads divide the 8 XCDs, an XCD's L2 holds the
// pages of one head. Runs of two workgroups of a head and two of the next took 4
// x 512 after 4096 from 68 to 84 us; longer runs of one head on an XCD gained
// nothing (66-70).
#include "mfma_common.hpp"

#include "../device/hip_check.hpp"

#include <type_traits>

namespace llaisys::kernels {

namespace {

using namespace mfma;

struct UnitArgs {
    const uint16_t *q;
    void *out;
    const uint16_t *k_pool, *v_pool; // bytes
    const float *k_scale, *v_scale;
    const int32_t *table, *ctx, *cu_q;
    int *err;
    int B, T, nh, nkvh, G, max_pages, num_blocks, units;
    float scale_log2;
};

// Where a block of columns lies: its sequence, that sequence's first query row,
// queries and length, and the block's index within it.
struct Place {
    int b, q0, Lq, ctx, block;
};
// A sequence whose rows or length do not fit counts as one query, whose blocks
// raise the error.
__device__ bool fits(int q0, int q1, int ctx, const UnitArgs &a) {
    return q0 >= 0 && q1 <= a.T && ctx <= a.max_pages * 16 && q1 - q0 <= ctx;
}
// The place of block `index` over the whole batch, ceil(queries * G / columns)
// blocks a sequence; false past the last one. Every lane of a wave.
__device__ bool placeOf(const UnitArgs &a, int index, int columns, Place &p) {
    const int lane = threadIdx.x & 63;
    int remaining = index;
    for (int base = 0; base < a.B; base += 64) {
        const int bb = min(base + lane, a.B - 1);
        const int q0 = a.cu_q[bb], q1 = a.cu_q[bb + 1], c = a.ctx[bb];
        const int lq = base + lane < a.B && q1 > q0 ? (fits(q0, q1, c, a) ? q1 - q0 : 1) : 0;
        const int blocks = (lq * a.G + columns - 1) / columns;
        const int incl = waveInclusiveSum(blocks);
        const int total = __builtin_amdgcn_readlane(incl, 63);
        if (remaining < total) {
            const int first = __ffsll(__ballot(incl > remaining)) - 1;
            p.b = base + first;
            p.q0 = __builtin_amdgcn_readlane(q0, first);
            p.Lq = __builtin_amdgcn_readlane(q1, first) - p.q0;
            p.ctx = __builtin_amdgcn_readlane(c, first);
            p.block = remaining - (__builtin_amdgcn_readlane(incl, first) - __builtin_amdgcn_readlane(blocks, first));
            return true;
        }
        remaining -= total;
    }
    return false;
}

// softmaxUpdate with weights of one bf16 part, whose sum the matrix cores take as
// rounded (a row of ones beside V): the rounding moves the quotient's two sides
// alike, and the vector unit is the one that has no time (8000 queries alone 231 ->
// 226 us).
__device__ __forceinline__ void weightsOnce(Acc &acc, f32x4 &sum, const float (&sv)[8], PairP<1> &P, float scale_log2) {
    constexpr float kLazyLog2 = 8.f;
    float most = sv[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) most = fmaxf(most, sv[i]);
    if (__builtin_amdgcn_ballot_w64(most * scale_log2 > acc.m + kLazyLog2) != 0) {
        const float m = fmaxf(acc.m, maxOverGroups(most) * scale_log2);
        const float alpha = exp2Fast(acc.m - (m == -INFINITY ? 0.f : m));
        sum *= alpha;
#pragma unroll
        for (int i = 0; i < 8; ++i) acc.o[i] *= alpha;
        acc.m = m;
    }
    const float m_use = acc.m == -INFINITY ? 0.f : acc.m;
#pragma unroll
    for (int i = 0; i < 8; ++i) P.part[0][i] = (__bf16)exp2Fast(__builtin_fmaf(sv[i], scale_log2, -m_use));
    const uint32_t one = 0x3f803f80u;
    sum = mfma::mfma(asBf16(u32x4{one, one, one, one}), P.part[0], sum);
}

// The 16 TILES columns from col0 on, of kv head h.
template <bool OUT_F32, int TILES, int UW, int PARTS>
__device__ __forceinline__ void attendBlock(const UnitArgs &a, const Place &p, int h, int col0) {
    constexpr int NSTAGE = 2, COLS = 16 * TILES, WINDOW = 64;
    __shared__ f32x4 part_o[UW / 2][8][64];
    __shared__ float part_ml[UW / 2][2][64];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lane = threadIdx.x & 63, n = lane & 15, grp = lane >> 4;
    const int G = a.G;
    const int before = p.ctx - p.Lq;
    const int min_pos = before + col0 / G; // the first column's, the least
    const int np = (before + min(p.Lq - 1, (col0 + COLS - 1) / G) + 16) >> 4, npr = (np + 1) >> 1;
    const int nw = npr > wave ? (npr - wave + UW - 1) / UW : 0; // this wave's pairs: wave, wave + UW, ...

    const int32_t *trow = a.table + size_t(p.b) * a.max_pages;
    int base = 0, cnt = 0, bidA = 0, bidB = 0;
    LaneScales scales;
    bool bad_block = false;
    // Lane i describes the wave's pair base + i.
    auto loadWindow = [&]() {
        const int pa = 2 * (wave + UW * (base + lane));
        bidA = trow[min(pa, np - 1)];
        bidB = trow[min(pa + 1, np - 1)];
    };
    loadWindow();
    int qi[TILES], g[TILES], pos[TILES];
    bool ok[TILES];
    u32x4 qop[TILES][4];
#pragma unroll
    for (int k = 0; k < TILES; ++k) {
        const int c = col0 + 16 * k + n;
        qi[k] = c / G;
        g[k] = c - qi[k] * G;
        ok[k] = qi[k] < p.Lq;
        pos[k] = ok[k] ? before + qi[k] : -1;
        const uint16_t *qrow =
            a.q + (size_t(p.q0 + (ok[k] ? qi[k] : 0)) * a.nh + h * G + (ok[k] ? g[k] : 0)) * kHeadDim + grp * 8;
#pragma unroll
        for (int s = 0; s < 4; ++s) qop[k][s] = *reinterpret_cast<const u32x4 *>(qrow + 32 * s);
    }
    const u32x4 *kp = reinterpret_cast<const u32x4 *>(a.k_pool) + lane;
    const u32x4 *vp = reinterpret_cast<const u32x4 *>(a.v_pool) + lane;
    KvF8::Pair ring[NSTAGE];
    // Past the window's end its last pair again, so loads are never conditional.
    auto issue = [&](int st, int k) {
        const int kk = max(min(k, cnt - 1), 0);
        int bA = __builtin_amdgcn_readlane(bidA, kk), bB = __builtin_amdgcn_readlane(bidB, kk);
        const bool bad = unsigned(bA) >= unsigned(a.num_blocks) || unsigned(bB) >= unsigned(a.num_blocks);
        bad_block |= bad && cnt > 0;
        bA = bad ? 0 : bA;
        bB = bad ? 0 : bB;
        KvF8::load(ring[st], kp, vp, (size_t(bA) * a.nkvh + h) * KvF8::kPageVecs,
                   (size_t(bB) * a.nkvh + h) * KvF8::kPageVecs);
    };
    Acc acc[TILES];
    f32x4 sums[TILES]; // of weights of one part
#pragma unroll
    for (int k = 0; k < TILES; ++k) {
        acc[k].reset();
        sums[k] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    for (; base < nw; base += WINDOW) {
        cnt = min(WINDOW, nw - base);
        if (base != 0) loadWindow();
        scales.load(a.k_scale, a.v_scale, bidA, bidB, a.num_blocks, a.nkvh, h);
#pragma unroll
        for (int st = 0; st < NSTAGE; ++st) issue(st, st);
        if (base == 0) {
#pragma unroll
            for (int k = 0; k < TILES; ++k)
#pragma unroll
                for (int s = 0; s < 4; ++s) qop[k][s] = ok[k] ? qop[k][s] : u32x4{0, 0, 0, 0};
        }
        for (int k0 = 0; k0 < cnt; k0 += NSTAGE) {
#pragma unroll
            for (int st = 0; st < NSTAGE; ++st) {
                const int i = k0 + st;
                if (i < cnt) {
                    const int j = wave + UW * (base + i); // the block's pair
                    const PairScales ps = scales.of(i);
                    const bool hasB = 2 * j + 1 < np;
                    KvF8::Pair &r = ring[st];
                    float sv[TILES][8];
                    {
                        u32x4 ka[4], kb[4];
#pragma unroll
                        for (int half = 0; half < 2; ++half) {
                            widenHalf(ka[2 * half], ka[2 * half + 1], r.ka[half], ps.ka);
                            widenHalf(kb[2 * half], kb[2 * half + 1], r.kb[half], ps.kb);
                        }
                        pairScoresN<TILES>(sv, ka, kb, qop, 32 * j, pos, hasB, grp, hasB && 32 * j + 31 <= min_pos);
                    }
                    PairP<PARTS> P[TILES];
#pragma unroll
                    for (int k = 0; k < TILES; ++k) {
                        if constexpr (PARTS == 1) {
                            weightsOnce(acc[k], sums[k], sv[k], P[k], a.scale_log2);
                        } else {
                            const float(&s1)[1][8] = *reinterpret_cast<const float(*)[1][8]>(&sv[k]);
                            PairP<PARTS>(&p1)[1] = *reinterpret_cast<PairP<PARTS>(*)[1]>(&P[k]);
                            softmaxUpdate<PARTS, 1>(acc[k], s1, p1, a.scale_log2);
                        }
                    }
                    u32x4 va[4], vb[4];
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        widenHalf(va[2 * half], va[2 * half + 1], r.va[half], ps.va);
                        widenHalf(vb[2 * half], vb[2 * half + 1], r.vb[half], ps.vb);
                    }
                    maskStaleV(va, vb, 32 * j, p.ctx, hasB, grp);
#pragma unroll
                    for (int k = 0; k < TILES; ++k) accumulatePV<PARTS>(acc[k], va, vb, P[k]);
                }
                issue(st, i + NSTAGE);
            }
        }
    }
    if (bad_block && lane == 0) atomicOr(a.err, kErrBadBlock);
    // The upper half of the waves hand their state to the lower half, tile by
    // tile, until wave 0 has it all.
#pragma unroll
    for (int k = 0; k < TILES; ++k) {
        float L = sums[k][0], M = acc[k].m;
        if constexpr (PARTS > 1) {
            L = acc[k].l + __shfl_xor(acc[k].l, 16);
            L += __shfl_xor(L, 32);
        }
#pragma unroll
        for (int half = UW / 2; half > 0; half /= 2) {
            if (k > 0 || half < UW / 2) __syncthreads(); // the states before have been read
            if (wave >= half && wave < 2 * half) {
#pragma unroll
                for (int i = 0; i < 8; ++i) part_o[wave - half][i][lane] = acc[k].o[i];
                part_ml[wave - half][0][lane] = M;
                part_ml[wave - half][1][lane] = L;
            }
            __syncthreads();
            const float mv = wave < half ? part_ml[wave][0][lane] : -INFINITY;
            if (mv != -INFINITY) {
                const float Mn = fmaxf(M, mv);
                const float sa = exp2Fast(M - Mn);
                const float sb = exp2Fast(mv - Mn);
                L = L * sa + part_ml[wave][1][lane] * sb;
#pragma unroll
                for (int i = 0; i < 8; ++i) acc[k].o[i] = acc[k].o[i] * sa + part_o[wave][i][lane] * sb;
                M = Mn;
            }
        }
        if (wave == 0 && ok[k]) {
            const float inv = 1.f / L;
            const size_t row = (size_t(p.q0 + qi[k]) * a.nh + h * G + g[k]) * kHeadDim;
#pragma unroll
            for (int i = 0; i < 8; ++i) storeOut<OUT_F32>(a.out, row, i, grp, acc[k].o[i] * inv);
        }
    }
}

template <bool OUT_F32, int TILES, int UW>
__global__ void __launch_bounds__(64 * UW) __attribute__((amdgpu_waves_per_eu(2, 2))) varlenUnitKernel(UnitArgs a) {
    // Parts of bf16 that a weight is summed in: 32-bit outputs hold 2^-24 of it,
    // 16-bit ones of a tile 2^-16. Large batches with 16-bit outputs (TILES == 2)
    // take one, 2^-9, which the output's own rounding is as large as: 3 chunks of
    // 700 after 1500 tokens 42.1 -> 37.9 us.
    constexpr int PARTS = OUT_F32 ? 3 : TILES == 2 ? 1 : 2;
    // The last blocks first: they see the most keys of their sequence.
    const int u = a.units - 1 - int(blockIdx.x);
    const int h = u % a.nkvh;
    Place p;
    if (!placeOf(a, u / a.nkvh, 16 * TILES, p)) return;
    if (!fits(p.q0, p.q0 + p.Lq, p.ctx, a)) {
        if (threadIdx.x == 0) atomicOr(a.err, kErrTooLong);
        return;
    }
    const int col0 = p.block * 16 * TILES;
    // Where the second tile is empty, as a single query's is: 512 queries beside 200
    // single ones 107 -> 103 us.
    if (TILES == 2 && col0 + 16 >= p.Lq * a.G) return attendBlock<OUT_F32, 1, UW, PARTS>(a, p, h, col0);
    attendBlock<OUT_F32, TILES, UW, PARTS>(a, p, h, col0);
}

} // namespace

// By the number of workgroups that blocks of one tile make, at 12 query and 2 kv
// heads (us: persistent kernel, then 1 tile and 4 waves, 1 and 8, 2 and 4, the
// last still with two parts of a weight):
//   up to 256: 64 after 1900 tokens 25.8, 15.1, 13.5, 21.9; 64 after 8000 39.2,
//     45.6, 39.4, 67.1; 256 after 8000 45.3, 47.2, 39.3, 69.6; 333 alone 22.6,
//     7.1, 7.2, 9.7: 8 waves, which halve the walk over a long context, in
//     tables of more than 64 pages
//   up to 900: 777 alone 27.5, 12.8, 18.0, 14.3; 2 x 256 and 60 single queries
//     25.7, 20.0, 23.9, 28.2; 1200 alone (902) 34.8, 19.7, 28.1, 19.4
//   more: 4 x 1000 44.7, 50.7, 80.7, 41.9; 6 x 340 after 1700 50.4, 44.1, 54.6,
//     38.6; 700 after 1000 twice and 150 single ones 72.6, 67.5, 78.7, 68.9
// A block's walk is as long as its context, which only the table's width bounds
// here, and the persistent kernel splits long ones. Up to 8192 tokens that
// decides little (us, persistent and this: 2 x 2000 after 4000 130, 100; 8000
// alone 273, 233; 4 x 1000 after 8000 173, 154; 8 x 512 after 8000 and 60 single
// ones up to 8000 182, 211; 4 x 256 after 6000 and 60 67, 76); beyond, a few
// queries after 16000 tokens walk alone for 80 us.
// Three and four tiles a block need one wave on a SIMD: 6 x 340 after 1700 55.6
// and 61.0. Blocks of one tile for the last round, to fill it: 4 x 512 after 4096
// 67.7 -> 82.
UnitShape unitShape(int B, int T, int nkvh, int group, int max_pages) {
    if (max_pages > 512) return {0, 0};
    const long long blocks = (((long long)T * group + 15) / 16 + B) * nkvh;
    if (blocks > 900) return {2, 4};
    return {1, blocks <= 256 && max_pages > 64 ? 8 : 4};
}

void pagedVarlenUnits(void *out, bool out_f32, const uint16_t *q, const uint16_t *k_pool, const uint16_t *v_pool,
                      const float *k_scale, const float *v_scale, const int32_t *block_table, const int32_t *ctx_len,
                      const int32_t *cu_q, int B, int T, int nh, int nkvh, int max_pages, int num_blocks, float scale,
                      UnitShape shape, int *err, void *stream) {
    if (B == 0 || T == 0) return;
    UnitArgs a{q, out, k_pool, v_pool, k_scale, v_scale, block_table, ctx_len, cu_q, err, B, T, nh, nkvh, nh / nkvh,
               max_pages, num_blocks, 0, scale * 1.4426950408889634f};
    auto s = static_cast<hipStream_t>(stream);
    auto launch = [&](auto f32, auto t, auto w) {
        constexpr int TILES = decltype(t)::value, UW = decltype(w)::value;
        // At most: every sequence's last block may be a partial one.
        const long long blocks = ((long long)T * a.G + 16 * TILES - 1) / (16 * TILES) + B;
        a.units = int(blocks * nkvh);
        hipLaunchKernelGGL((varlenUnitKernel<decltype(f32)::value, TILES, UW>), dim3(unsigned(a.units)), dim3(64 * UW),
                           0, s, a);
    };
    auto pick = [&](auto f32) {
        using std::integral_constant;
        if (shape.tiles == 2)
            launch(f32, integral_constant<int, 2>(), integral_constant<int, 4>());
        else if (shape.waves == 8)
            launch(f32, integral_constant<int, 1>(), integral_constant<int, 8>());
        else
            launch(f32, integral_constant<int, 1>(), integral_constant<int, 4>());
    };
    if (out_f32)
        pick(std::true_type());
    else
        pick(std::false_type());
    HIP_CHECK(hipGetLastError());
}

} // namespace llaisys::kernels
