"""llaisysPagedAttentionF8 and ...VarlenF8 against attention in 64 bits over the
values that the 8-bit cache holds.

Tolerance, for one output o = sum p_j v_j / sum p_j: the scores are 32-bit sums
of 128 products (error at most 130 * 2^-24 * sum |q k| * scale, each weight's
relative error as much, twice in the quotient), each weight's exponential and
parts 2^-20 more in 32-bit outputs and in decode, the sums n * 2^-24, all of it
relative to the largest |v|; where 16-bit outputs hold the weights and the
partial sums in bf16 (chunks), two roundings of 2^-8 to each; and the output's
own rounding, half a step: 2^-8 or 2^-24 of its size."""
import numpy as np
import pytest
import torch

import llaisys_amd as L
from cases_8bit import BAD_BLOCK, DEVICES, TOO_LONG, Cache, attend64, bf16, f64, give, table_of, take

SCALE = 128 ** -0.5


def case(seed, lens, nh, nkvh, qn, extra_pages=0, stale_nan=False):
    table, blocks = table_of(seed, lens, extra_pages=extra_pages)
    cache = Cache(blocks, nkvh, seed + 1)
    r = np.random.RandomState(seed + 2)
    for which in range(2):
        c = cache.codes[which]
        c[(c & 127) == 127] = 5  # no NaN among the values
        cache.exps[which][:] = r.randint(-11, -7, cache.exps[which].shape)
    clean = cache
    if stale_nan:
        for which in range(2):
            held = np.zeros(cache.codes[which].shape[:1] + (16,), bool)
            for b, n in enumerate(lens):
                for p in range(n):
                    held[table[b, p // 16], p % 16] = True
            cache.codes[which][~np.broadcast_to(held[:, None, :], cache.codes[which].shape[:3])] = 127
    q = bf16(r.randn(sum(qn), nh, 128))
    return clean, table, q


def want_of(cache, table, lens, qn, q):
    K, V = cache.values(0), cache.values(1)
    out, most, r = [], 0.0, 0
    for b, (n, c) in enumerate(zip(qn, lens)):
        if n == 0:
            continue
        at = table[b, :-(-c // 16)]
        rows = lambda x: x[at].transpose(0, 2, 1, 3).reshape(-1, x.shape[1], 128)[:c]  # noqa: E731
        o, m = attend64(f64(q[r:r + n]), rows(K), rows(V), SCALE)
        out.append(o)
        most = max(most, m)
        r += n
    return np.concatenate(out), most


def check(got, want, most, cache, dtype, longest, chunks):
    vmax = np.nanmax(np.abs(cache.values(1)))
    bound = vmax * (2 * 130 * 2.0 ** -24 * most + 2.0 ** -20 + longest * 2.0 ** -24)
    if dtype == torch.bfloat16 and chunks:
        bound += vmax * 2 * 2.0 ** -8
    elif chunks:
        bound += vmax * 2.0 ** -16  # the chunks' weights in two bf16 parts
    step = torch.finfo(dtype).eps / 2
    err = np.abs(got.double().numpy() - want)
    assert (err <= bound + step * np.abs(want)).all(), (err.max(), bound)


def decode(device, cache, table, q, ctx, dtype, fill=7.0):
    out = give(torch.full(q.shape, fill, dtype=dtype), device)
    L.Ops.paged_attention_f8(out, give(q, device), *cache.device(device), give(table, device),
                             give(np.asarray(ctx, np.int32), device), SCALE)
    return take(out)


def varlen(device, cache, table, q, cu, ctx, dtype, fill=7.0):
    out = give(torch.full(q.shape, fill, dtype=dtype), device)
    L.Ops.paged_attention_varlen_f8(out, give(q, device), *cache.device(device), give(table, device),
                                    give(np.asarray(cu, np.int32), device), give(np.asarray(ctx, np.int32), device), SCALE)
    return take(out)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nh, nkvh", [(12, 2), (16, 1), (4, 4), (7, 1)])
@pytest.mark.parametrize("lens", [[1], [16], [17], [32, 33, 1, 15], [300, 5, 64, 129, 31]])
def test_decode(device, dtype, nh, nkvh, lens):
    cache, table, q = case(1, lens, nh, nkvh, [1] * len(lens), stale_nan=True)
    got = decode(device, cache, table, q, lens, dtype)
    assert L.device_error_flags() == 0
    want, most = want_of(cache, table, lens, [1] * len(lens), q)
    check(got, want, most, cache, dtype, max(lens), False)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lens, extra", [
    ([2000], 0), ([700], 60), ([9000, 3], 0), (list(range(600, 1024, 7)), 0), (list(range(1, 8192, 177)), 10),
    ([1] * 200, 3), (list(range(1, 300)), 100), ([1 + i % 37 for i in range(4100)], 0),  # more than a launch takes
    # on both sides of the lines between the kernels: tables of 48 and 49, 80 and 81, 96 and 97, 128 and 129 pages
    ([768, 5], 0), ([769, 5], 0), ([1280] + [1] * 9, 0), ([1281] + [1] * 9, 0), ([1536] + [70] * 31, 0),
    ([1537] + [70] * 31, 0), ([2048] + [33] * 63, 0), ([2049] + [33] * 63, 0),
])
def test_decode_long_and_many(dtype, lens, extra):
    cache, table, q = case(4, lens, 12, 2, [1] * len(lens), extra_pages=extra, stale_nan=True)
    got = decode("amd", cache, table, q, lens, dtype)
    assert L.device_error_flags() == 0
    want, most = want_of(cache, table, lens, [1] * len(lens), q)
    check(got, want, most, cache, dtype, max(lens), False)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nh, nkvh", [(12, 2), (8, 2), (3, 3), (16, 1)])
@pytest.mark.parametrize("qn, prior", [([2], [0]), ([16], [1]), ([33, 1], [0, 40]), ([5, 1, 50, 1], [100, 0, 3, 16]),
                                       ([1, 1], [4, 20])])
def test_chunks(device, dtype, nh, nkvh, qn, prior):
    lens = [a + b for a, b in zip(qn, prior)]
    cache, table, q = case(7, lens, nh, nkvh, qn, stale_nan=True)
    cu = np.concatenate([[0], np.cumsum(qn)])
    got = varlen(device, cache, table, q, cu, lens, dtype)
    assert L.device_error_flags() == 0
    want, most = want_of(cache, table, lens, qn, q)
    check(got, want, most, cache, dtype, max(lens), True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("qn, prior, extra", [
    ([700], [0], 0), ([333], [1500], 0), ([300, 200, 1, 77], [2000, 0, 900, 1100], 90), ([64] + [1] * 70, [500] + list(range(1, 1400, 20)), 0),
    ([2] * 40, list(range(40)), 0),
])
def test_chunks_long_and_many(dtype, qn, prior, extra):
    lens = [a + b for a, b in zip(qn, prior)]
    cache, table, q = case(9, lens, 12, 2, qn, extra_pages=extra, stale_nan=True)
    cu = np.concatenate([[0], np.cumsum(qn)])
    got = varlen("amd", cache, table, q, cu, lens, dtype)
    assert L.device_error_flags() == 0
    want, most = want_of(cache, table, lens, qn, q)
    check(got, want, most, cache, dtype, max(lens), True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("qn, prior, pages", [
    # on both sides of the lines between the kernels: 256 and 258 blocks of queries, 900 and 902
    ([338], [0], 0), ([341], [0], 0), ([338], [0], 65), ([341], [0], 65), ([33], [991], 64), ([33], [992], 65), ([1197], [0], 0), ([1200], [0], 0), ([1100] + [1] * 90, [40] + [300] * 90, 0),
    # tables of 256 and 257 pages with 528 blocks, of 300 with 512 and 516, of 512 and 513 with few
    ([700], [3396], 256), ([700], [3397], 257), ([680], [33], 300), ([683], [33], 300), ([64], [8128], 512),
    ([64], [8129], 513), ([2, 1, 1, 70], [0, 0, 8191, 4000], 512),
    # sequences without queries among the others
    ([0, 20, 0, 0, 1, 0], [9, 40, 0, 70, 8, 1], 0),
])
def test_chunks_at_the_lines(dtype, qn, prior, pages):
    lens = [a + b for a, b in zip(qn, prior)]
    cache, table, q = case(19, lens, 12, 2, qn, extra_pages=max(0, pages - -(-max(lens) // 16)), stale_nan=True)
    assert pages in (0, table.shape[1])
    cu = np.concatenate([[0], np.cumsum(qn)])
    got = varlen("amd", cache, table, q, cu, lens, dtype)
    assert L.device_error_flags() == 0
    want, most = want_of(cache, table, lens, qn, q)
    check(got, want, most, cache, dtype, max(lens), True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nh, nkvh", [(12, 2), (3, 1)])
@pytest.mark.parametrize("qn", [
    [1] * 300,  # single queries only
    [40, 1, 3] + [1] * 600, [2] * 1100 + [70], [1] * 3000 + [50], [300, 300] + [0] * 50 + [1] * 4000,
])
def test_many_sequences_over_wide_tables(dtype, nh, nkvh, qn):
    """Past 512 pages, in batches that the work queue's tables hold, sort and do not."""
    lens = [n + 7 * b % 40 for b, n in enumerate(qn)]
    lens = [max(1, n) for n in lens]
    lens[len(lens) // 2] += 900
    cache, table, q = case(29, lens, nh, nkvh, qn, extra_pages=520, stale_nan=True)
    got = varlen("amd", cache, table, q, np.concatenate([[0], np.cumsum(qn)]), lens, dtype)
    assert L.device_error_flags() == 0
    want, most = want_of(cache, table, lens, qn, q)
    check(got, want, most, cache, dtype, max(lens), True)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("bad", [[60, 19, 33], [60, 1000, 33], [60, 0, 33]])  # too short, past the table, none
@pytest.mark.parametrize("pages", [0, 600])
def test_a_bad_sequence_leaves_the_others(device, bad, pages):
    qn, lens = [40, 20, 33], [60, 20, 33]
    cache, table, q = case(23, lens, 12, 2, qn, extra_pages=pages if device == "amd" else 0)
    cu = np.concatenate([[0], np.cumsum(qn)])
    ctx = bad if table.shape[1] * 16 < 1000 or 1000 not in bad else [60, 100000, 33]
    got = varlen(device, cache, table, q, cu, ctx, torch.bfloat16)
    assert L.device_error_flags() == TOO_LONG
    want, most = want_of(cache, table, lens, qn, q)
    good = np.r_[0:40, 60:93]
    check(got[good], want[good], most, cache, torch.bfloat16, 60, True)


@pytest.mark.parametrize("device", DEVICES)
def test_scales_far_apart(device):
    """Blocks whose scales differ by powers of two up to 2^40, as a value cache may hold."""
    lens = [60, 33]
    cache, table, q = case(11, lens, 12, 2, [1, 1])
    cache.exps[1][:] = np.random.RandomState(1).randint(-50, -10, cache.exps[1].shape)
    for dtype in (torch.bfloat16, torch.float32):
        got = decode(device, cache, table, q, lens, dtype)
        want, most = want_of(cache, table, lens, [1, 1], q)
        check(got, want, most, cache, dtype, 60, False)


@pytest.mark.parametrize("device", DEVICES)
def test_rows_behind_the_last_sequence_are_left(device):
    qn, lens = [3, 1, 20], [10, 40, 33]
    cache, table, q = case(13, lens, 12, 2, qn + [6])
    cu = np.concatenate([[0], np.cumsum(qn)])
    got = varlen(device, cache, table, q, cu, lens, torch.bfloat16)
    assert (got[24:] == 7.0).all() and L.device_error_flags() == 0
    want, most = want_of(cache, table, lens, qn, q[:24])
    check(got[:24], want, most, cache, torch.bfloat16, 40, True)


@pytest.mark.parametrize("device", DEVICES)
def test_bad_lengths_and_blocks(device):
    lens = [30, 20, 25]
    cache, table, q = case(15, lens, 12, 2, [1] * 3)
    for ctx in ([30, 0, 25], [30, 33, 25]):  # no keys; past the table of 32
        got = decode(device, cache, table, q, ctx, torch.float32)
        assert L.device_error_flags() == TOO_LONG
        want, most = want_of(cache, table, lens, [1] * 3, q)
        check(got[[0, 2]], want[[0, 2]], most, cache, torch.float32, 30, False)
    table = table.copy()
    table[1, 0] = 1 << 20
    decode(device, cache, table, q, lens, torch.float32)
    assert L.device_error_flags() == BAD_BLOCK
    varlen(device, cache, table, q, [0, 1, 2, 3], lens, torch.float32)
    assert L.device_error_flags() == BAD_BLOCK
    varlen(device, cache, table, q, [0, 1, 3, 3], [30, 1, 25], torch.float32)  # two queries of a length of one
    assert L.device_error_flags() & TOO_LONG


def test_refusals():
    dev = "cpu"
    pools = Cache(3, 2, 0).device(dev)
    q = give(torch.zeros(2, 12, 128, dtype=torch.bfloat16), dev)
    out = give(torch.zeros(2, 12, 128, dtype=torch.bfloat16), dev)
    table, ctx, cu = (give(np.ones(s, np.int32), dev) for s in ((2, 2), 2, 3))
    b16 = give(torch.zeros(3, 2, 16, 128, dtype=torch.bfloat16), dev)
    with pytest.raises(L.LlaisysError, match="f8"):
        L.Ops.paged_attention_f8(out, q, b16, b16, *pools[2:], table, ctx, 0.1)
    with pytest.raises(L.LlaisysError, match="scale"):
        L.Ops.paged_attention_f8(out, q, *pools[:2], ctx, ctx, table, ctx, 0.1)
    with pytest.raises(L.LlaisysError, match="q must be"):
        L.Ops.paged_attention_f8(out, give(torch.zeros(2, 12, 64, dtype=torch.bfloat16), dev), *pools, table, ctx, 0.1)
    with pytest.raises(L.LlaisysError, match="nh"):
        odd = give(torch.zeros(2, 13, 128, dtype=torch.bfloat16), dev)
        L.Ops.paged_attention_f8(odd, odd, *pools, table, ctx, 0.1)
    with pytest.raises(L.LlaisysError, match="one query per sequence"):
        three = give(torch.zeros(3, 12, 128, dtype=torch.bfloat16), dev)
        L.Ops.paged_attention_f8(three, three, *pools, table, ctx, 0.1)
    with pytest.raises(L.LlaisysError, match="cu_q"):
        L.Ops.paged_attention_varlen_f8(out, q, *pools, table, ctx, ctx, 0.1)
    with pytest.raises(L.LlaisysError, match="out"):
        L.Ops.paged_attention_varlen_f8(cu, q, *pools, table, cu, ctx, 0.1)
    for scale in (0.0, -0.1, float("nan"), float("inf")):
        with pytest.raises(L.LlaisysError, match="scale must be positive"):
            L.Ops.paged_attention_f8(out, q, *pools, table, ctx, scale)
        with pytest.raises(L.LlaisysError, match="scale must be positive"):
            L.Ops.paged_attention_varlen_f8(out, q, *pools, table, cu, ctx, scale)
    odd = give(torch.zeros(2 * 12 * 128 + 4, dtype=torch.bfloat16), dev).slice(0, 4, 2 * 12 * 128 + 4).view(2, 12, 128)
    for args in ((out, odd), (odd, q)):
        with pytest.raises(L.LlaisysError, match="16 B boundary"):
            L.Ops.paged_attention_f8(*args, *pools, table, ctx, 0.1)
    with pytest.raises(L.LlaisysError, match="f8"):  # an 8-bit pool to the bf16 entry point
        L.Ops.paged_attention(out, q, pools[0], pools[1], table, ctx, 0.1)
