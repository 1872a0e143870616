/*
 * Operator C-ABI.
 *
 * llaisysSelfAttention and the eight other reference ops keep the reference's
 * declarations (include/llaisys/ops.h:7-15) so python/llaisys/libllaisys/ops.py
 * binds unchanged. Every op dispatches on its tensors' device, as the
 * reference's src/ops/add/op.cpp:16-33 does: LLAISYS_DEVICE_AMD tensors run the
 * HIP kernels, LLAISYS_DEVICE_CPU tensors the host implementations (fp32 math,
 * host threads); one call may not mix devices. F32, F16, BF16; indices I64;
 * contiguous unless stated. Contracts are the reference README's
 * (README.md:157-292).
 *
 * The llaisysPagedKV* / llaisysPagedAttention* entry points are new. The
 * reference has no paged KV code; they follow its op conventions
 * (include/llaisys/ops.h:6-16: tensor handles and scalars in, void out, output
 * written in place, errors reported as the reference reports them).
 *
 * Paged KV pool (one per layer, one for K and one for V):
 *   shape [num_blocks, nkvh, 16, 128], dtype BF16, contiguous, on the AMD
 *   device or the host (the same page format on both).
 *   A (block, kv-head) page holds 16 tokens x 128 dims = 4 KiB. Inside a page
 *   the bytes are in the MI355X page format, not row-major [16][128]:
 *     K page: element (token t, dim d) at bf16 index
 *             (d / 8) * 128 + t * 8 + (d % 8)              ([16 dim-chunks][16 t][8])
 *     V page: element (t, d) at bf16 index
 *             (d / 32) * 512 + (t / 4) * 128 + (d % 16) * 8 + ((d / 16) % 2) * 4 + t % 4
 *   so that every 1 KiB of a page is exactly one 64-lane x 16-byte load that
 *   feeds a gfx950 MFMA operand. Only llaisysPagedKVAppend writes this format
 *   and llaisysPagedKVGather reads it back to row-major; callers never need it.
 * Block table: [B, max_pages] I32; entry (b, p) is the physical block holding
 *   tokens [16p, 16p+16) of sequence b. ctx_len: [B] I32 = tokens in the cache.
 */
#ifndef LLAISYS_OPS_H
#define LLAISYS_OPS_H

#include "tensor.h"

__C {
    /* ops.h:7: c = a + b, one shape and dtype. */
    __export void llaisysAdd(llaisysTensor_t c, llaisysTensor_t a, llaisysTensor_t b);
    /* ops.h:8: max over the last dim of vals; max_idx I64 and max_val (may be
     * NULL) hold one element per row (1 for a 1-D vals, README.md:161-167). */
    __export void llaisysArgmax(llaisysTensor_t max_idx, llaisysTensor_t max_val, llaisysTensor_t vals);
    /* ops.h:9: out[i] = weight[index[i]], index I64 (README.md:171-177). */
    __export void llaisysEmbedding(llaisysTensor_t out, llaisysTensor_t index, llaisysTensor_t weight);
    /* ops.h:10: out = in . weight^T + bias, weight [out, in], bias may be NULL
     * (README.md:181-198); a hand-written MFMA GEMM, fp32 accumulation,
     * one rounding; no GEMM library is linked. */
    __export void llaisysLinear(llaisysTensor_t out, llaisysTensor_t in, llaisysTensor_t weight, llaisysTensor_t bias);
    /* New; no counterpart in the reference (whose linear is ops.h:10). The
     * weight of llaisysLinear, rewritten once into the layout the decode GEMM
     * streams (tiles of 16 rows x 32 columns in MFMA operand order): packed
     * and weight are [N, K] BF16 on the AMD device, N % 16 == 0, K % 32 == 0. */
    __export void llaisysLinearPackWeight(llaisysTensor_t packed, llaisysTensor_t weight);
    /* New; no counterpart in the reference. out = in . W^T + bias (bias may be
     * NULL) as llaisysLinear computes it (fp32 accumulation, one rounding),
     * with W given packed by llaisysLinearPackWeight; for decode-sized batches:
     * in [M, K], out [M, N] BF16 on the AMD device, 1 <= M <= 128, and
     * either K == 1536, N % 16 == 0, or 1536 < K <= 16384, K % 32 == 0,
     * N % 128 == 0 (split over K into fp32 partials in the runtime's device
     * workspace, summed in a fixed order); other shapes: llaisysLinear. */
    __export void llaisysLinearPacked(llaisysTensor_t out, llaisysTensor_t in, llaisysTensor_t packed,
                                      llaisysTensor_t bias);
    /* ops.h:11: copy between equal shapes with any strides (README.md:286-292). */
    __export void llaisysRearrange(llaisysTensor_t out, llaisysTensor_t in);
    /* ops.h:12: y = w * x / sqrt(mean(x^2) + eps) per row (README.md:202-217). */
    __export void llaisysRmsNorm(llaisysTensor_t out, llaisysTensor_t in, llaisysTensor_t weight, float eps);
    /* ops.h:13: rotary embedding of [seqlen, nhead, d] by pos_ids I64 (README.md:221-242). */
    __export void llaisysROPE(llaisysTensor_t out, llaisysTensor_t in, llaisysTensor_t pos_ids, float theta);
    /* ops.h:15: out = up * gate / (1 + exp(-gate)) (README.md:268-278). */
    __export void llaisysSwiGLU(llaisysTensor_t out, llaisysTensor_t gate, llaisysTensor_t up);

    /* Replaces include/llaisys/ops.h:14 (stub src/ops/self_attention/op.cpp:4-6;
     * semantics README.md:244-266, test/ops/self_attention.py:11-28).
     * attn_val [L, nh, dv], q [L, nh, d], k [S, nkvh, d], v [S, nkvh, dv], all
     * contiguous, one dtype (F32, F16 or BF16), nh % nkvh == 0, S >= L,
     * d, dv <= 256. Query i attends keys j <= i + S - L; query head h reads
     * kv head h / (nh / nkvh). Accumulates in fp32, rounds once to the dtype. */
    __export void llaisysSelfAttention(llaisysTensor_t attn_val, llaisysTensor_t q, llaisysTensor_t k,
                                       llaisysTensor_t v, float scale);

    /* New. Scatter new K/V tokens into their pages.
     * k_new, v_new: [T, nkvh, 128] BF16. cu_new: [B+1] I32 prefix offsets, or
     * NULL meaning T == B and one token per sequence. Row r of sequence b
     * (cu_new[b] <= r < cu_new[b+1]) is written at position
     * ctx_len[b] + (r - cu_new[b]), i.e. ctx_len is the length BEFORE the append
     * and is not modified. Pages for every written position must already be
     * mapped in block_table. Bit-exact copy. */
    __export void llaisysPagedKVAppend(llaisysTensor_t k_pool, llaisysTensor_t v_pool, llaisysTensor_t k_new,
                                       llaisysTensor_t v_new, llaisysTensor_t block_table, llaisysTensor_t ctx_len,
                                       llaisysTensor_t cu_new);

    /* New. Copy the first cu_seqlens[b+1]-cu_seqlens[b] tokens of each
     * sequence out of the pool into rows [cu_seqlens[b], cu_seqlens[b+1]) of
     * k_out, v_out: [T, nkvh, 128] BF16 row-major. Bit-exact. */
    __export void llaisysPagedKVGather(llaisysTensor_t k_out, llaisysTensor_t v_out, llaisysTensor_t k_pool,
                                       llaisysTensor_t v_pool, llaisysTensor_t block_table,
                                       llaisysTensor_t cu_seqlens);

    /* New; no counterpart in the reference (its KV cache is a README prompt,
     * README.md:316, :412). llaisysPagedKVAppend of one token per sequence
     * (k_new, v_new: [B, nkvh, 128] BF16, written at position ctx_len[b])
     * followed by llaisysPagedKVGather of the contexts including it, in one
     * launch: cu_seqlens [B+1] must give every sequence ctx_len[b] + 1 output
     * rows (a sequence that does not raises device error flag 2 and is
     * skipped). Same bytes in the pool and in k_out, v_out as the two calls. */
    __export void llaisysPagedKVAppendGather(llaisysTensor_t k_out, llaisysTensor_t v_out, llaisysTensor_t k_pool,
                                             llaisysTensor_t v_pool, llaisysTensor_t k_new, llaisysTensor_t v_new,
                                             llaisysTensor_t block_table, llaisysTensor_t ctx_len,
                                             llaisysTensor_t cu_seqlens);

    /* New. Copy whole (block, all kv heads) pages inside the pools:
     * pairs [P, 2] I32 of (src, dst) block ids, as produced by
     * llaisysKVSeqReserve for copy-on-write of a shared last block. */
    __export void llaisysPagedKVCopyBlocks(llaisysTensor_t k_pool, llaisysTensor_t v_pool, llaisysTensor_t pairs);

    /* New. Batched decode attention (flash-decoding with split-KV and a
     * log-sum-exp combine): q [B, nh, 128] BF16, out [B, nh, 128] BF16 or F32.
     * Sequence b's single query attends all ctx_len[b] (>= 1) cached tokens,
     * which include the token appended for this step.
     * nh % nkvh == 0 and nh / nkvh <= 16. fp32 accumulation. */
    __export void llaisysPagedAttention(llaisysTensor_t out, llaisysTensor_t q, llaisysTensor_t k_pool,
                                        llaisysTensor_t v_pool, llaisysTensor_t block_table, llaisysTensor_t ctx_len,
                                        float scale);

    /* No counterpart in the reference. llaisysPagedAttention (same arguments,
     * same results to fp32 rounding, AMD tensors only) for callers that cannot
     * allocate device memory: HIP graph capture, fixed-memory serving loops.
     * The split records live in a fixed 16 MiB array that each GPU holds for
     * the life of the process; a batch whose records need more (2 x W x G x
     * 130 floats, W = max(1.75 x CUs, pairs / 64)) is refused with an error.
     * Calls that overlap on one GPU (two streams, two host threads) share the
     * array and race. The device's set-up (its first library call) allocates
     * the error word; this entry point itself allocates nothing. */
    __export void llaisysPagedAttentionNoAlloc(llaisysTensor_t out, llaisysTensor_t q, llaisysTensor_t k_pool,
                                               llaisysTensor_t v_pool, llaisysTensor_t block_table,
                                               llaisysTensor_t ctx_len, float scale);

    /* New. Mixed chunked-prefill + decode attention over paged KV.
     * q, out [T, nh, 128]; sequence b owns query rows [cu_q[b], cu_q[b+1]) and
     * Lq = cu_q[b+1]-cu_q[b] (>= 1, <= ctx_len[b]) of its ctx_len[b] cached
     * tokens are those queries' own tokens (already appended). Query i sits at
     * position ctx_len[b] - Lq + i and attends keys at positions <= that
     * (bottom-right causal alignment, test/ops/self_attention.py:18). */
    __export void llaisysPagedAttentionVarlen(llaisysTensor_t out, llaisysTensor_t q, llaisysTensor_t k_pool,
                                              llaisysTensor_t v_pool, llaisysTensor_t block_table,
                                              llaisysTensor_t cu_q, llaisysTensor_t ctx_len, float scale);

    /* New; no counterpart in the reference. A step's tables from the requests'
     * lengths, so that a serving loop's steps need no host work on them.
     * Sequence b holds ctx_len[b] tokens and gets new_len[b]: [B] I32 each.
     *   cu_new [B+1] I32: prefix sums of new_len (negative: 0), at most T.
     *   block_table [B, max_pages] I32, updated in place: the pages that the new
     *     tokens begin get blocks from free_blocks [F] I32, from free_used[0]
     *     on, in the order of the sequences and pages; free_after[0] is
     *     free_used[0] plus the blocks taken ([1] I32 each). All three NULL:
     *     every page is mapped already.
     *   ctx_after [B] I32: ctx_len + new_len.
     *   pos_ids, slots [T] I64: row cu_new[b] + i is token ctx_len[b] + i of
     *     sequence b: its position, and block * 16 + offset, the place that
     *     llaisysPagedKVAppendF8 writes. Rows behind the last sequence: position
     *     0 and slot -1.
     * A sequence is left as it is (ctx_after = ctx_len, no blocks, its rows as
     * those behind the last sequence) if its lengths are negative or pass the
     * table or its rows pass T (error bit 2), if the page its first row
     * continues is not mapped (bit 1), or if free_blocks does not reach for it:
     * then no later sequence takes blocks either (bit 8). A row whose page is
     * not mapped gets position 0 and slot -1 (bit 1). ctx_after may be ctx_len
     * itself and free_after free_used; T, F, B, max_pages under 2^30. */
    __export void llaisysPagedKVMap(llaisysTensor_t block_table, llaisysTensor_t cu_new, llaisysTensor_t ctx_after,
                                    llaisysTensor_t pos_ids, llaisysTensor_t slots, llaisysTensor_t ctx_len,
                                    llaisysTensor_t new_len, llaisysTensor_t free_blocks, llaisysTensor_t free_used,
                                    llaisysTensor_t free_after);

    /* New; no counterpart in the reference: the paged KV in 8 bits. Pools
     * [num_blocks, nkvh, 16, 128] F8 hold e4m3 codes in a page format of their
     * own (csrc/kernels/f8_page.hpp), k_scale and v_scale [num_blocks, nkvh] F32
     * the scale 2^E of each block and kv head: E the least whole number, -100 at
     * least, whose 448 * 2^E reaches the block's largest value. A value is read
     * back within 2^-4 of its size, or within 2^-10 * 2^E where that is more.
     * Block tables are as for the bf16 pool. Pools, rows, queries and outputs
     * of these calls begin on 16 B boundaries.
     *
     * Append: row r of k_new, v_new [T, nkvh, 128] BF16 to slots[r] (I64, block
     * * 16 + offset, as llaisysPagedKVMap builds them; negative: the row is not
     * written). A block's rows are one run: consecutive rows at consecutive
     * slots. Rows that break it or begin a second one within 32 rows are not
     * written (error bit 2); a block written from places of the batch further
     * apart is the caller's mistake, and its contents are then undefined. A run
     * that begins at a block's offset 0 starts the block's scale anew; otherwise
     * the scale grows if the new rows need it, and the block's codes are
     * re-encoded, which rounds only those that become subnormal. A value that is
     * not finite is kept as NaN and leaves the scale alone. A slot past the
     * pool: error bit 1. */
    __export void llaisysPagedKVAppendF8(llaisysTensor_t k_pool, llaisysTensor_t v_pool, llaisysTensor_t k_scale,
                                         llaisysTensor_t v_scale, llaisysTensor_t k_new, llaisysTensor_t v_new,
                                         llaisysTensor_t slots);
    /* llaisysPagedKVGather out of the 8-bit pool: k_out, v_out [T, nkvh, 128]
     * BF16, which holds every value of the cache exactly. */
    __export void llaisysPagedKVGatherF8(llaisysTensor_t k_out, llaisysTensor_t v_out, llaisysTensor_t k_pool,
                                         llaisysTensor_t v_pool, llaisysTensor_t k_scale, llaisysTensor_t v_scale,
                                         llaisysTensor_t block_table, llaisysTensor_t cu_seqlens);
    /* llaisysPagedKVCopyBlocks of the 8-bit pool, scales included. */
    __export void llaisysPagedKVCopyBlocksF8(llaisysTensor_t k_pool, llaisysTensor_t v_pool, llaisysTensor_t k_scale,
                                             llaisysTensor_t v_scale, llaisysTensor_t pairs);
    /* llaisysPagedAttention and llaisysPagedAttentionVarlen over the 8-bit pool:
     * the same arguments otherwise, with a positive scale; the softmax and the
     * sums in 32 bits. Rows of a sequence that raises an error bit hold no
     * result; rows that belong to no sequence are left as they were. Wide tables
     * and batches take the runtime's workspace, which grows by allocation: under
     * stream capture a call of the same sizes has to have run before. */
    __export void llaisysPagedAttentionF8(llaisysTensor_t out, llaisysTensor_t q, llaisysTensor_t k_pool,
                                          llaisysTensor_t v_pool, llaisysTensor_t k_scale, llaisysTensor_t v_scale,
                                          llaisysTensor_t block_table, llaisysTensor_t ctx_len, float scale);
    __export void llaisysPagedAttentionVarlenF8(llaisysTensor_t out, llaisysTensor_t q, llaisysTensor_t k_pool,
                                                llaisysTensor_t v_pool, llaisysTensor_t k_scale,
                                                llaisysTensor_t v_scale, llaisysTensor_t block_table,
                                                llaisysTensor_t cu_q, llaisysTensor_t ctx_len, float scale);

    /* New; no counterpart in the reference. Rows of x [M, K] (F32, F16 or BF16)
     * as 8-bit integers: scale[m] = max |x[m, :]| / 127 (F32 [M]) and q[m, k] =
     * x[m, k] / scale[m] to the nearest whole number, ties to even (I8 [M, K]).
     * A row of zeros has the scale 0; a row with a value that is not finite the
     * scale NaN and codes 0. For activations (a scale per token) and, over a
     * weight's rows, for its output channels. */
    __export void llaisysQuantizeRows(llaisysTensor_t q, llaisysTensor_t scale, llaisysTensor_t x);
    /* New; no counterpart in the reference (whose linear is ops.h:10).
     * llaisysLinear in 8-bit integers: out[m, n] = (sum_k in[m, k] weight[n, k])
     * * (in_scale[m] * weight_scale[n]) (+ bias[n], may be NULL), in [M, K] and
     * weight [N, K] I8, scales F32, out and bias F32, F16 or BF16. The products
     * are summed exactly in 32-bit integers (K <= 131071), the rest is 32-bit
     * floats and one rounding. Takes the runtime's workspace as llaisysLinear
     * does. */
    __export void llaisysLinearI8(llaisysTensor_t out, llaisysTensor_t in, llaisysTensor_t in_scale,
                                  llaisysTensor_t weight, llaisysTensor_t weight_scale, llaisysTensor_t bias);
}

#endif /* LLAISYS_OPS_H */
