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
// is launches and memory round trips. One workgroup does all of it (mapKernel).
// The rows of larger steps go to further workgroups of the same launch, each of
// which works out the sums once more; where the lengths or the list's place are
// updated in place, which the first workgroup would do under the others' eyes,
// they go to a second launch (rowsKernel).
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

// Who writes the rows: kAll: this workgroup; kFirst: each sequence's first one,
// and rowsKernel the rest; kSpread: workgroup 0 none, the others a row a thread,
// and the table's entry with the page's first row (at most kMapThreads
// sequences).
enum RowsBy { kAll, kFirst, kSpread };
template <RowsBy ROWS> __global__ void __launch_bounds__(kMapThreads) mapKernel(MapArgs a) {
    __shared__ int tmp[kMapThreads / 64];
    // A sequence's first row; if its rows have slots, its length before, the
    // first page it takes and that one's place in the list (-1: takes none).
    __shared__ int begins[ROWS == kSpread ? kMapThreads : 1];
    __shared__ int4 seqs[ROWS == kSpread ? kMapThreads : 1];
    const int tid = threadIdx.x, lane = tid & 63;
    const bool lead = ROWS != kSpread || blockIdx.x == 0;
    const int rows_cap = a.T + 1, free_cap = a.F + 1;
    const int used = a.free_blocks ? *a.free_used : 0;
    const int avail = a.free_blocks && used >= 0 ? max(0, a.F - used) : 0;
    int row_carry = 0, free_carry = 0, flags = 0;
    int last_free = 0; // blocks taken by the sequences that fit
    if (lead && tid == 0) a.cu[0] = 0;
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
            if (ROWS != kSpread) row[first] = id;
            if (!mapped) block = id;
            if (!mapped && id < 0) flags |= kErrBadBlock;
        }
        const int count = ok ? n : 0; // rows that get a slot
        const bool placed = count > 0 && block >= 0;
        if (ROWS == kSpread && !lead) {
            begins[tid] = begin;
            seqs[tid] = make_int4(placed, c, first, need > 0 ? used + need_begin : -1);
            continue;
        }
        if (live) {
            a.cu[b + 1] = min(end, a.T);
            a.after[b] = c + count;
        }
        // The first row; then, wave by wave, the pages and rows of the sequences with more.
        if (ROWS != kSpread && live && n > 0 && begin < a.T) {
            a.pos[begin] = placed ? c : 0;
            a.slots[begin] = placed ? (int64_t(block) << 4) + (c & 15) : -1;
        }
        for (unsigned long long more = ROWS == kSpread ? 0 : __ballot(need > 1); more; more &= more - 1) {
            const int l = __ffsll(more) - 1;
            const int nb = __builtin_amdgcn_readlane(need, l), at = __builtin_amdgcn_readlane(need_begin, l);
            int32_t *to = a.table + size_t(__builtin_amdgcn_readlane(b, l)) * a.max_pages +
                          __builtin_amdgcn_readlane(first, l);
            for (int i = 1 + lane; i < nb; i += 64) to[i] = a.free_blocks[used + at + i];
        }
        if (ROWS == kAll) {
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
    if (ROWS == kSpread && !lead) {
        __syncthreads();
        const int r = (int(blockIdx.x) - 1) * kMapThreads + tid;
        if (r >= a.T) return;
        // The row's sequence is the last one that begins at it or before (dead
        // threads hold a sequence of no rows, past the last).
        int lo = 0;
#pragma unroll
        for (int step = kMapThreads / 2; step > 0; step /= 2) lo += begins[lo + step] <= r ? step : 0;
        const int4 q = seqs[lo];
        int id = -1, p = 0;
        if (r < row_carry && (q.x || q.w >= 0)) {
            p = q.y + (r - begins[lo]);
            const int page = p >> 4;
            int32_t *entry = a.table + size_t(lo) * a.max_pages + page;
            const bool takes = q.w >= 0 && page >= q.z;
            id = takes ? a.free_blocks[q.w + page - q.z] : *entry;
            if (takes && (p & 15) == 0) *entry = id;
            if (id < 0) atomicOr(a.err, kErrBadBlock);
            if (!q.x) id = -1;
        }
        a.pos[r] = id >= 0 ? p : 0;
        a.slots[r] = id >= 0 ? (int64_t(id) << 4) + (p & 15) : -1;
        return;
    }
    // Rows behind the last sequence: no slot.
    if (ROWS == kAll)
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
    // A row or 512 of them 4.5 us either way; 64 sequences with 1563 rows in all
    // 7.6 us by one workgroup and 4.9 spread, 4063 rows 14.0 and 4.9. In place,
    // two launches take 9.9 us.
    const bool apart = ctx_after != ctx_len && (!free_blocks || free_after != free_used);
    const bool spread = apart && B <= kMapThreads;
    if (T <= (spread ? 512 : 4096))
        hipLaunchKernelGGL(mapKernel<kAll>, dim3(1), dim3(kMapThreads), 0, s, a);
    else if (spread)
        hipLaunchKernelGGL(mapKernel<kSpread>, dim3(unsigned(1 + (T + kMapThreads - 1) / kMapThreads)),
                           dim3(kMapThreads), 0, s, a);
    else {
        hipLaunchKernelGGL(mapKernel<kFirst>, dim3(1), dim3(kMapThreads), 0, s, a);
        hipLaunchKernelGGL(rowsKernel, dim3(unsigned((T + 255) / 256)), dim3(256), 0, s, a);
    }
    HIP_CHECK(hipGetLastError());
}

} // namespace llaisys::kernels
