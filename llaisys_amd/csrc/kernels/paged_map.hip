// A step's block-table entries, row offsets, lengths, positions and slots from
// the requests' lengths, on the GPU.
//
// Sequence b holds c tokens and gets n: its rows are [S_b, S_b + n) with S the
// prefix sums of n, and it takes pages [ceil(c / 16), ceil((c + n) / 16)) from
// the free list, at the prefix sum of what the sequences before it take. A
// sequence takes part if its lengths are valid, its rows lie within T, the
// page that its first row continues is mapped, and the list reaches for it
// (the sums run over all that the first three let through, so that once one
// does not fit, no later one takes blocks either).
//
// Two prefix sums over a few hundred numbers and a few bytes per row: the time
// is launches and memory round trips. One workgroup does all of it
// (mapKernel); the rows of larger steps go to a second launch (rowsKernel).
#include "launch.hpp"

#include "../device/hip_check.hpp"
#include "mfma_common.hpp"

namespace llaisys::kernels {

namespace {

using mfma::kErrBadBlock;
using mfma::kErrTooLong;

constexpr int kMapThreads = 1024;

struct MapArgs {
    int32_t *table, *cu, *after;
    int64_t *pos, *slots;
    const int32_t *ctx, *fresh; // lengths before, new tokens
    const int32_t *free_blocks, *free_used;
    int32_t *free_after;
    int B, T, max_pages, F;
    int *err;
};

// Sums over the workgroup of the x (0 <= x <= cap < 2^30) of the threads up to
// this one, and (`before_me`) of those before it, kept at cap once they reach
// it (min(sum, cap) of sums that grow is a sum like any other: the order of the
// additions does not show); `total`: that of all.
__device__ __forceinline__ int blockSums(int x, int cap, int *tmp, int &before_me, int &total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    x = min(cap, x + __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false));
    x = min(cap, x + __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false));
    x = min(cap, x + __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false));
    x = min(cap, x + __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false));
    x = min(cap, x + __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false));
    x = min(cap, x + __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false));
    __syncthreads(); // tmp's last readers are done
    if (lane == 63) tmp[wave] = x;
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kMapThreads / 64; ++w) {
        const int v = tmp[w];
        before = w < wave ? min(cap, before + v) : before;
        all = min(cap, all + v);
    }
    total = all;
    const int left = __shfl_up(x, 1);
    before_me = lane ? min(cap, left + before) : before;
    return min(cap, x + before);
}

// `rows`: this launch writes all rows (else each sequence's first one, and
// rowsKernel the rest).
__global__ void __launch_bounds__(kMapThreads) mapKernel(MapArgs a, int rows) {
    __shared__ int tmp[kMapThreads / 64];
    const int tid = threadIdx.x, lane = tid & 63;
    const int rows_cap = a.T + 1, free_cap = a.F + 1;
    const int used = a.free_blocks ? *a.free_used : 0;
    const int avail = a.free_blocks && used >= 0 ? max(0, a.F - used) : 0;
    int row_carry = 0, free_carry = 0, flags = 0;
    int last_free = 0; // blocks taken by the sequences that fit
    if (tid == 0) a.cu[0] = 0;
    for (int b0 = 0; b0 < a.B; b0 += kMapThreads) {
        const int b = b0 + tid;
        const bool live = b < a.B;
        const int c = live ? a.ctx[b] : 0, n = live ? a.fresh[b] : 0;
        int total, begin, need_begin;
        const int end = min(rows_cap, blockSums(min(max(n, 0), rows_cap), rows_cap, tmp, begin, total) + row_carry);
        begin = min(a.T, begin + row_carry); // (past T no row is written)
        row_carry = min(rows_cap, row_carry + total);
        bool ok = live && c >= 0 && n >= 0 && (long long)c + n <= (long long)a.max_pages * 16 && end <= a.T;
        if (live && !ok) flags |= kErrTooLong;
        const int first = (c >> 4) + ((c & 15) != 0), last = ok ? int(((long long)c + n + 15) >> 4) : 0;
        // The block that the first row goes to where the sequence has one.
        int32_t *row = a.table + size_t(live ? b : 0) * a.max_pages;
        int block = -1;
        const bool mapped = (c & 15) != 0 || !a.free_blocks;
        if (ok && n > 0 && mapped) {
            block = row[c >> 4];
            if (block < 0) {
                flags |= kErrBadBlock;
                ok = false;
            }
        }
        int need = ok && a.free_blocks ? last - first : 0;
        const int need_end =
            min(free_cap, blockSums(min(need, free_cap), free_cap, tmp, need_begin, total) + free_carry);
        need_begin += free_carry;
        free_carry = min(free_cap, free_carry + total);
        if (need > 0 && need_end > avail) {
            flags |= kErrNoBlocks;
            ok = false;
            need = 0;
        }
        if (need > 0) last_free = need_end;
        if (need > 0) {
            const int id = a.free_blocks[used + need_begin];
            row[first] = id;
            if (!mapped) block = id;
            if (!mapped && id < 0) flags |= kErrBadBlock;
        }
        const int count = ok ? n : 0; // rows that get a slot
        if (live) {
            a.cu[b + 1] = min(end, a.T);
            a.after[b] = c + count;
        }
        // The first row; then, wave by wave, the pages and rows of the sequences with more.
        const bool placed = count > 0 && block >= 0;
        if (live && n > 0 && begin < a.T) {
            a.pos[begin] = placed ? c : 0;
            a.slots[begin] = placed ? (int64_t(block) << 4) + (c & 15) : -1;
        }
        for (unsigned long long more = __ballot(need > 1); more; more &= more - 1) {
            const int l = __ffsll(more) - 1;
            const int nb = __builtin_amdgcn_readlane(need, l), at = __builtin_amdgcn_readlane(need_begin, l);
            int32_t *to = a.table + size_t(__builtin_amdgcn_readlane(b, l)) * a.max_pages +
                          __builtin_amdgcn_readlane(first, l);
            for (int i = 1 + lane; i < nb; i += 64) to[i] = a.free_blocks[used + at + i];
        }
        if (rows) {
            for (unsigned long long more = __ballot(live && n > 1); more; more &= more - 1) {
                const int l = __ffsll(more) - 1;
                const int rb = __builtin_amdgcn_readlane(begin, l), re = min(__builtin_amdgcn_readlane(end, l), a.T);
                const int c0 = __builtin_amdgcn_readlane(c, l), f = __builtin_amdgcn_readlane(first, l);
                const int at = __builtin_amdgcn_readlane(need_begin, l);
                const bool put = __builtin_amdgcn_readlane(placed, l);
                const int32_t *from = a.table + size_t(__builtin_amdgcn_readlane(b, l)) * a.max_pages;
                for (int r = rb + 1 + lane; r < re; r += 64) {
                    const int p = c0 + (r - rb), page = p >> 4;
                    int id = -1;
                    if (put) id = a.free_blocks && page >= f ? a.free_blocks[used + at + page - f] : from[page];
                    if (put && id < 0) flags |= kErrBadBlock;
                    a.pos[r] = id >= 0 ? p : 0;
                    a.slots[r] = id >= 0 ? (int64_t(id) << 4) + (p & 15) : -1;
                }
            }
        }
    }
    // Rows behind the last sequence: no slot.
    if (rows)
        for (int r = row_carry + tid; r < a.T; r += kMapThreads) {
            a.pos[r] = 0;
            a.slots[r] = -1;
        }
    if (a.free_blocks) {
        // What the sequences that fit took: the largest of the threads' ends.
        last_free = mfma::waveMaxInt(last_free);
        __syncthreads();
        if (lane == 0) tmp[tid >> 6] = last_free;
        __syncthreads();
        if (tid == 0) {
            int most = 0;
            for (int w = 0; w < kMapThreads / 64; ++w) most = max(most, tmp[w]);
            *a.free_after = used + most;
        }
    }
    if (flags) atomicOr(a.err, flags);
}

// The rows that mapKernel left: each sequence's after its first, and those
// behind the last sequence. A row's sequence is the last one with cu <= row; a
// sequence whose first row has no slot has none at all.
__global__ void __launch_bounds__(256) rowsKernel(MapArgs a) {
    const int r = int(blockIdx.x) * 256 + int(threadIdx.x);
    if (r >= a.T) return;
    const int all = a.cu[a.B];
    if (r >= all) {
        a.pos[r] = 0;
        a.slots[r] = -1;
        return;
    }
    int lo = 0, hi = a.B - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (a.cu[mid] <= r)
            lo = mid;
        else
            hi = mid - 1;
    }
    const int begin = a.cu[lo];
    if (r == begin) return;
    int id = -1, p = 0;
    if (a.slots[begin] >= 0) {
        p = int(a.pos[begin]) + (r - begin);
        id = a.table[size_t(lo) * a.max_pages + (p >> 4)];
        if (id < 0) atomicOr(a.err, kErrBadBlock);
    }
    a.pos[r] = id >= 0 ? p : 0;
    a.slots[r] = id >= 0 ? (int64_t(id) << 4) + (p & 15) : -1;
}

} // namespace

void pagedMap(int32_t *block_table, int32_t *cu_new, int32_t *ctx_after, int64_t *pos_ids, int64_t *slots,
              const int32_t *ctx_len, const int32_t *new_len, const int32_t *free_blocks, const int32_t *free_used,
              int32_t *free_after, int B, int T, int max_pages, int F, int *err, void *stream) {
    const MapArgs a{block_table, cu_new, ctx_after, pos_ids, slots, ctx_len, new_len, free_blocks, free_used, free_after,
                    B, T, max_pages, F, err};
    auto s = static_cast<hipStream_t>(stream);
    const bool one = T <= 4096;
    hipLaunchKernelGGL(mapKernel, dim3(1), dim3(kMapThreads), 0, s, a, one ? 1 : 0);
    if (!one) hipLaunchKernelGGL(rowsKernel, dim3(unsigned((T + 255) / 256)), dim3(256), 0, s, a);
    HIP_CHECK(hipGetLastError());
}

} // namespace llaisys::kernels
