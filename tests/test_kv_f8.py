"""The 8-bit paged KV's append, gather and block copy against the format's
definition in 64 bits: codes, scales and read-back values, equal."""
import numpy as np
import pytest
import torch

import llaisys_amd as L
from cases_8bit import (BAD_BLOCK, CODES, DEVICES, LEAST, TOO_LONG, Cache, attend64, bf16, encode64, exp_of, f64,
                        give, table_of, take)


def rows_of(seed, T, nkvh, spread=2.0):
    """K and V rows with sizes spread over powers of two."""
    r = np.random.RandomState(seed)
    size = 2.0 ** (spread * r.randn(T, 1, 1))
    return [bf16(r.randn(T, nkvh, 128) * size) for _ in range(2)]


def append(device, pools, k, v, slots):
    L.Ops.paged_kv_append_f8(*pools, give(k, device), give(v, device), give(np.asarray(slots, np.int64), device))


def slots_of(table, ctx, new):
    return np.array([int(table[b, p // 16]) * 16 + p % 16 for b, (c, n) in enumerate(zip(ctx, new))
                     for p in range(c, c + n)], np.int64)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("nkvh", [1, 2, 5])
@pytest.mark.parametrize("ctx, new", [
    ([0], [1]), ([0], [16]), ([7], [9]), ([15, 16, 17], [1, 1, 1]), ([3, 0, 14, 32], [30, 17, 2, 50]),
    ([200], [333]),
])
def test_appended_runs(device, nkvh, ctx, new):
    table, blocks = table_of(1, [c + n for c, n in zip(ctx, new)])
    cache = Cache(blocks, nkvh, 2)
    pools = cache.device(device)
    k, v = rows_of(3, sum(new), nkvh)
    slots = slots_of(table, ctx, new)
    append(device, pools, k, v, slots)
    assert L.device_error_flags() == 0
    cache.append(f64(k), f64(v), slots)
    cache.check(*pools)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("nkvh", [1, 2])
@pytest.mark.parametrize("seed", range(4))
def test_large_batches_of_ragged_runs(device, nkvh, seed):
    """Single tokens, short runs and chunks in one batch, rows without a slot between them."""
    r = np.random.RandomState(seed)
    ctx = r.randint(0, 100, 300)
    new = np.where(r.rand(300) < 0.7, 1, r.randint(1, 40, 300))
    table, blocks = table_of(seed, ctx + new)
    cache = Cache(blocks, nkvh, seed)
    pools = cache.device(device)
    slots = slots_of(table, ctx, new)
    gap = np.repeat(r.rand(300) < 0.05, new)  # sequences whose rows are not written
    slots[gap] = -1
    k, v = rows_of(seed, len(slots), nkvh)
    append(device, pools, k, v, slots)
    assert L.device_error_flags() == 0
    cache.append(f64(k), f64(v), slots)
    cache.check(*pools)


@pytest.mark.parametrize("device", DEVICES)
def test_a_scale_that_grows_token_by_token(device):
    """Sixteen appends to a block, each larger than the last by a factor that
    varies: the codes are those of the growing scale, and no value that stays
    normal is rounded twice."""
    cache = Cache(2, 2, 5)
    pools = cache.device(device)
    r = np.random.RandomState(6)
    first = None
    for t in range(16):
        k, v = (bf16(r.randn(1, 2, 128) * 1.6 ** t * 1e-3) for _ in range(2))
        append(device, pools, k, v, [16 + t])
        cache.append(f64(k), f64(v), [16 + t])
        cache.check(*pools)
        if t == 0:
            first = cache.values(0)[1, :, 0]
    last = cache.values(0)[1, :, 0]
    normal = np.abs(first) >= 2.0 ** (cache.exps[0][1] - 6.0)[:, None]  # (a smaller one may round up to that)
    assert normal.any() and (last[normal] == first[normal]).all()


@pytest.mark.parametrize("device", DEVICES)
def test_a_block_begun_anew_forgets_its_scale(device):
    cache = Cache(1, 1, 7)
    pools = cache.device(device)
    for size, slots in ((1e4, [0, 1]), (1.0, [2]), (1e-3, [0])):
        k, v = (bf16(np.random.RandomState(8).randn(len(slots), 1, 128) * size) for _ in range(2))
        append(device, pools, k, v, slots)
        cache.append(f64(k), f64(v), slots)
        cache.check(*pools)
    assert cache.exps[0][0, 0] < -8


@pytest.mark.parametrize("device", DEVICES)
def test_every_bf16_at_many_scales(device):
    """All finite bf16 numbers of a block's range below its largest value, at
    scales from the least to the greatest: rounding, subnormal codes, the
    scale's own step at 448 * 2^E."""
    bits = torch.arange(0, 1 << 16, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    bits = bits[torch.isfinite(bits.float())]
    order = bits[torch.argsort(bits.float().abs(), stable=True)]
    n = order.numel() // 2048 * 2048
    x = order[-n:].view(-1, 16, 128)  # blocks of neighbouring magnitudes
    mixed = order[torch.randperm(order.numel(), generator=torch.Generator().manual_seed(1))][:n].view(-1, 16, 128)
    rows = torch.cat([x, mixed]).reshape(-1, 1, 128)
    blocks = rows.shape[0] // 16
    cache = Cache(blocks, 1, 9)
    pools = cache.device(device)
    append(device, pools, rows, rows, np.arange(blocks * 16))
    assert L.device_error_flags() == 0
    cache.append(f64(rows), f64(rows), np.arange(blocks * 16))
    cache.check(*pools)
    assert cache.exps[0].min() == LEAST and cache.exps[0].max() == 120


@pytest.mark.parametrize("device", DEVICES)
def test_values_that_are_not_finite_and_zeros(device):
    cache = Cache(3, 1, 10)
    pools = cache.device(device)
    x = np.random.RandomState(11).randn(40, 1, 128)
    x[0, 0, 3], x[1, 0, 5], x[17, 0, 0] = np.inf, np.nan, -np.inf
    x[16], x[32:40] = np.nan, 0.0
    k, v = bf16(x), bf16(x[::-1].copy())
    append(device, pools, k, v, np.arange(40))
    cache.append(f64(k), f64(v), np.arange(40))
    cache.check(*pools)
    assert (cache.exps[0][2] == LEAST).all() and np.isnan(cache.values(0)[0, 0, 0, 3])
    # a larger token later: the NaN stays one, the zeros stay zeros
    k = bf16(np.full((1, 1, 128), 1e5))
    append(device, pools, k, k, [40])
    cache.append(f64(k), f64(k), [40])
    cache.check(*pools)
    ko, vo = (give(torch.zeros(41, 1, 128, dtype=torch.bfloat16), device) for _ in range(2))
    L.Ops.paged_kv_gather_f8(ko, vo, *pools, give(np.array([[0, 1, 2]], np.int32), device),
                             give(np.array([0, 41], np.int32), device))
    got = take(ko).double().numpy()
    np.testing.assert_array_equal(got, cache.values(0).reshape(48, 1, 128)[:41])


@pytest.mark.parametrize("device", DEVICES)
def test_rows_without_a_slot_and_bad_slots(device):
    cache = Cache(4, 2, 12)
    pools = cache.device(device)
    k, v = rows_of(13, 10, 2)
    slots = np.array([5, 6, -1, 7, -1, -3, 33, 34, -1, -1])
    append(device, pools, k, v, slots)
    assert L.device_error_flags() == TOO_LONG  # slot 7: a second run of its block
    slots[3] = -1
    cache.append(f64(k), f64(v), slots)
    cache.check(*pools)
    append(device, pools, k, v, slots)  # the same rows again: the same cache
    assert L.device_error_flags() == 0
    cache.check(*pools)
    # slots past the pool; one block's slots out of order, and twice the same
    for bad, flag, kept in (([64, 1, 1 << 40], BAD_BLOCK, [-1, 1, -1]), ([3, 9, 10, 40], TOO_LONG, [3, -1, -1, 40]),
                            ([3, 3, 40, 2], TOO_LONG, [3, -1, 40, -1]),
                            ([10, 9, 64, 3], TOO_LONG | BAD_BLOCK, [10, -1, -1, -1])):
        append(device, pools, k[:len(bad)], v[:len(bad)], bad)
        assert L.device_error_flags() == flag
        cache.append(f64(k), f64(v), np.array(kept))
        cache.check(*pools)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("lens", [[1], [16], [17, 0, 5], [100, 33, 64, 1]])
def test_gather(device, lens):
    table, blocks = table_of(14, lens, extra_pages=2)
    cache = Cache(blocks, 2, 15)
    pools = cache.device(device)
    total = sum(lens)
    cu = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    ko, vo = (give(torch.full((total + 2, 2, 128), 7.0, dtype=torch.bfloat16), device) for _ in range(2))
    L.Ops.paged_kv_gather_f8(ko, vo, *pools, give(table, device), give(cu, device))
    assert L.device_error_flags() == 0
    for which, out in enumerate((ko, vo)):
        got = take(out).double().numpy()
        want = np.concatenate([cache.values(which)[table[b, :-(-n // 16)]].transpose(0, 2, 1, 3).reshape(-1, 2, 128)[:n]
                               for b, n in enumerate(lens)])
        np.testing.assert_array_equal(got[:total], want)
        assert (got[total:] == 7.0).all()


@pytest.mark.parametrize("device", DEVICES)
def test_gather_errors(device):
    table = np.array([[0, 9, 1], [2, -1, -1]], np.int32)
    cache = Cache(3, 1, 16)
    pools = cache.device(device)
    out = lambda: give(torch.full((60, 1, 128), 7.0, dtype=torch.bfloat16), device)  # noqa: E731
    for cu, flag in (([0, 40, 50], BAD_BLOCK), ([0, 5, 61], TOO_LONG), ([-1, 5, 6], TOO_LONG), ([0, 0, 49], TOO_LONG | BAD_BLOCK)):
        ko, vo = out(), out()
        L.Ops.paged_kv_gather_f8(ko, vo, *pools, give(table, device), give(np.array(cu, np.int32), device))
        assert L.device_error_flags() == flag


@pytest.mark.parametrize("device", DEVICES)
def test_copied_blocks_grow_apart(device):
    """A block copied for a forked sequence: both continue it with scales of their own."""
    cache = Cache(5, 2, 17)
    pools = cache.device(device)
    k, v = rows_of(18, 5, 2)
    append(device, pools, k, v, np.arange(16, 21))
    cache.append(f64(k), f64(v), np.arange(16, 21))
    L.Ops.paged_kv_copy_blocks_f8(*pools, give(np.array([[1, 3], [9, 0]], np.int32), device))
    assert L.device_error_flags() == BAD_BLOCK
    for which in range(2):
        cache.codes[which][3], cache.exps[which][3] = cache.codes[which][1], cache.exps[which][1]
    cache.check(*pools)
    k, v = (bf16(f64(x[:2]) * np.array([1e4, 1e-4])[:, None, None]) for x in (k, v))
    append(device, pools, k, v, [53, 21])
    cache.append(f64(k), f64(v), np.array([53, 21]))
    cache.check(*pools)
    assert (cache.exps[0][3] > cache.exps[0][1]).all()


@pytest.mark.gpu
def test_a_pool_of_more_than_4_gib():
    """Append, block copy, gather and attention at both ends of it."""
    blocks, nkvh, nh, lens = 1_100_000, 2, 12, [37, 50]
    pools = [L.Tensor((blocks, nkvh, 16, 128), dtype=L.DataType.F8, device=L.DeviceType.AMD) for _ in range(2)]
    pools += [L.Tensor((blocks, nkvh), dtype=L.DataType.F32, device=L.DeviceType.AMD) for _ in range(2)]
    table = np.array([[blocks - 1, 3, blocks - 7, 0], [1_048_577, blocks - 30, 1_048_570, 12]], np.int32)
    at = {int(b): i for i, b in enumerate(table.ravel())}
    near = Cache(8, nkvh, 41)  # the same blocks, numbered from 0
    k, v = rows_of(42, sum(lens), nkvh)
    slots = slots_of(table, [0, 0], lens)
    append("amd", pools, k, v, slots)
    near.append(f64(k), f64(v), [at[int(x) // 16] * 16 + int(x) % 16 for x in slots])
    q = bf16(np.random.RandomState(43).randn(2, nh, 128))
    src = table.ravel()
    pairs = np.stack([src, np.where(src > 2000, src - 300, src + 300)], 1)  # to blocks of no sequence
    L.Ops.paged_kv_copy_blocks_f8(*pools, give(pairs.astype(np.int32), "amd"))
    copied = np.array([[dict(pairs.tolist())[int(b)] for b in row] for row in table], np.int32)
    for tab in (table, copied):
        ko, vo = (give(torch.zeros(sum(lens), nkvh, 128, dtype=torch.bfloat16), "amd") for _ in range(2))
        L.Ops.paged_kv_gather_f8(ko, vo, *pools, give(tab, "amd"), give(np.array([0, 37, 87], np.int32), "amd"))
        outs = [give(torch.zeros(q.shape, dtype=torch.float32), "amd") for _ in range(2)]
        ctx = give(np.array(lens, np.int32), "amd")
        L.Ops.paged_attention_f8(outs[0], give(q, "amd"), *pools, give(tab, "amd"), ctx, 128 ** -0.5)
        L.Ops.paged_attention_varlen_f8(outs[1], give(q, "amd"), *pools, give(tab, "amd"),
                                        give(np.array([0, 1, 2], np.int32), "amd"), ctx, 128 ** -0.5)
        assert L.device_error_flags() == 0
        for b, n in enumerate(lens):
            K, V = (near.values(w).reshape(2, 4, nkvh, 16, 128)[b].transpose(0, 2, 1, 3).reshape(64, nkvh, 128)[:n]
                    for w in range(2))
            r = slice(37 * b, 37 * b + n)
            np.testing.assert_array_equal(take(ko)[r].double().numpy(), K)
            np.testing.assert_array_equal(take(vo)[r].double().numpy(), V)
            want, most = attend64(f64(q[b:b + 1]), K, V, 128 ** -0.5)
            bound = np.abs(V).max() * (2 * 130 * 2.0 ** -24 * most + 2.0 ** -16 + 64 * 2.0 ** -24)
            for o in outs:
                assert np.abs(take(o)[b].double().numpy() - want[0]).max() <= bound + 2.0 ** -24 * np.abs(want).max()


def test_the_plain_form_itself():
    assert exp_of(448.0) == 0 and exp_of(448.1) == 1 and exp_of(0.0) == LEAST and exp_of(224.0) == -1
    np.testing.assert_array_equal(encode64(CODES[:127]), np.arange(127))
    assert CODES[encode64(np.array([2.0 ** -10]))[0]] == 0 and CODES[encode64(np.array([3 * 2.0 ** -10]))[0]] == 2.0 ** -8
    ours = torch.from_numpy(np.linspace(-448, 448, 100003)).float()
    np.testing.assert_array_equal(ours.to(torch.float8_e4m3fn).view(torch.uint8).numpy(), encode64(ours.double().numpy()))


def test_refusals():
    dev = "cpu"
    pools = Cache(3, 2, 0).device(dev)
    kn = give(torch.zeros(4, 2, 128, dtype=torch.bfloat16), dev)
    sl = give(np.zeros(4, np.int64), dev)
    b16 = give(torch.zeros(3, 2, 16, 128, dtype=torch.bfloat16), dev)
    scale = give(torch.ones(3, 1), dev)
    table, cu = give(np.zeros((1, 1), np.int32), dev), give(np.zeros(2, np.int32), dev)
    pairs = give(np.zeros((1, 2), np.int32), dev)
    for bad in ((b16, b16, *pools[2:]), (pools[0], pools[1], scale, pools[3]), (pools[0], pools[1], pools[2], pools[0])):
        with pytest.raises(L.LlaisysError, match="must be f8|scale"):
            L.Ops.paged_kv_append_f8(*bad, kn, kn, sl)
        with pytest.raises(L.LlaisysError, match="must be f8|scale"):
            L.Ops.paged_kv_gather_f8(kn, kn, *bad, table, cu)
        with pytest.raises(L.LlaisysError, match="must be f8|scale"):
            L.Ops.paged_kv_copy_blocks_f8(*bad, pairs)
    with pytest.raises(L.LlaisysError, match="slots"):
        L.Ops.paged_kv_append_f8(*pools, kn, kn, give(np.zeros(3, np.int64), dev))
    with pytest.raises(L.LlaisysError, match="slots must be i64"):
        L.Ops.paged_kv_append_f8(*pools, kn, kn, give(np.zeros(4, np.int32), dev))
    with pytest.raises(L.LlaisysError, match="k_new"):
        L.Ops.paged_kv_append_f8(*pools, give(torch.zeros(4, 1, 128, dtype=torch.bfloat16), dev), kn, sl)
    with pytest.raises(L.LlaisysError, match="bf16"):
        L.Ops.paged_kv_append_f8(*pools, give(torch.zeros(4, 2, 128), dev), give(torch.zeros(4, 2, 128), dev), sl)
    with pytest.raises(L.LlaisysError, match="contiguous"):
        flat = give(torch.zeros(4, 128, 2, dtype=torch.bfloat16), dev).permute(0, 2, 1)
        L.Ops.paged_kv_append_f8(*pools, flat, flat, sl)
    flat = give(torch.zeros(4 * 256 + 4, dtype=torch.bfloat16), dev).slice(0, 4, 4 * 256 + 4).view(4, 2, 128)
    for rows in ((flat, kn), (kn, flat)):
        with pytest.raises(L.LlaisysError, match="16 B boundary"):
            L.Ops.paged_kv_append_f8(*pools, *rows, sl)
        with pytest.raises(L.LlaisysError, match="16 B boundary"):
            L.Ops.paged_kv_gather_f8(*rows, *pools, table, cu)
    with pytest.raises(L.LlaisysError, match="16 B boundary"):
        bytes_ = give(torch.zeros(3 * 2 * 2048 + 8, dtype=torch.uint8), dev).slice(0, 8, 3 * 2 * 2048 + 8)
        L.Ops.paged_kv_append_f8(pools[0], bytes_.view(3, 2, 16, 128), *pools[2:], kn, kn, sl)
    with pytest.raises(L.LlaisysError, match="pairs"):
        L.Ops.paged_kv_copy_blocks_f8(*pools, cu)
