"""llaisysPagedKVMap (a step's table entries, row offsets, lengths, positions
and slots) against its definition worked out row by row: whole numbers, equal."""
import numpy as np
import pytest

import llaisys_amd as L
from cases_8bit import BAD_BLOCK, DEVICES, NO_BLOCKS, TOO_LONG, give, map_plain, take


def i32(a, device):
    return give(np.asarray(a, np.int32), device)


def run(device, table, ctx, new, T, free=None, used=0, in_place=False):
    """The op's results and error bits."""
    B = len(ctx)
    t = i32(table, device)
    c = i32(ctx, device)
    cu, after = i32(np.full(B + 1, -7), device), c if in_place else i32(np.full(B, -7), device)
    pos, slots = (give(np.full(T, -7, np.int64), device) for _ in range(2))
    lists = ()
    if free is not None:
        u = i32([used], device)
        lists = (i32(free, device), u, u if in_place else i32([-7], device))
    L.Ops.paged_kv_map(t, cu, after, pos, slots, c, i32(new, device), *lists)
    flags = L.device_error_flags()
    got = [take(x).numpy() for x in (t, cu, after, pos, slots)]
    return (*got, int(take(lists[2])[0]) if lists else used, flags)


def check(device, table, ctx, new, T, free=None, used=0, in_place=False):
    got = run(device, table, ctx, new, T, free, used, in_place)
    want = map_plain(np.asarray(table, np.int32), ctx, new, T, free, used)
    for name, g, w in zip(("table", "cu_new", "ctx_after", "pos_ids", "slots", "free_after", "flags"), got, want):
        np.testing.assert_array_equal(g, w, err_msg=name)
    return want


def mapped(seed, ctx, width, spare):
    """A table with the pages of ctx mapped, and the other blocks in random order."""
    pages = [-(-int(c) // 16) for c in ctx]
    order = np.random.RandomState(seed).permutation(sum(pages) + spare).astype(np.int32)
    table = np.full((len(ctx), width), -1, np.int32)
    at = 0
    for b, p in enumerate(pages):
        table[b, :p] = order[at:at + p]
        at += p
    return table, order[at:]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("ctx, new, pad", [
    ([0], [1], 0),
    ([15, 16, 17, 31, 0], [1, 1, 1, 1, 1], 0),
    ([0, 3, 16, 40], [16, 13, 1, 0], 3),
    ([5, 0, 33, 7], [0, 0, 0, 0], 2),
    ([100, 1, 47], [700, 33, 1], 5),
])
def test_lengths_with_a_free_list(device, ctx, new, pad):
    table, free = mapped(1, ctx, 60, 80)
    check(device, table, ctx, new, sum(new) + pad, free, 3)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("B, longest, chunks", [(64, 8192, 0), (1023, 300, 4), (1025, 300, 30), (3000, 64, 0)])
def test_large_batches(device, B, longest, chunks):
    r = np.random.RandomState(B)
    ctx, new = r.randint(0, longest, B), np.ones(B, np.int64)
    new[r.permutation(B)[:chunks]] = r.randint(2, 400, chunks)
    new[r.permutation(B)[:B // 7]] = 0
    table, free = mapped(B, ctx, (longest + 400) // 16 + 1, B + 26 * chunks)
    check(device, table, ctx, new, int(new.sum()) + 11, free)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("extra", [-4096, -1, 0, 1, 5000])
def test_rows_on_both_sides_of_one_launch(device, extra):
    # 4096 rows go out in one launch, more of them in a second one.
    total = 4096 + extra
    ctx, new = ([9, 0], [0, 0]) if total == 0 else ([9, 200, 0], [total // 3, 1, total - total // 3 - 1])
    table, free = mapped(2, ctx, 700, 1500)
    check(device, table, ctx, new, total, free)
    check(device, table, ctx, new, total + 300, free)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("T", [512, 513, 1024, 1025, 4096, 4097, 9000])
@pytest.mark.parametrize("B", [1, 5, 1024, 1025])
@pytest.mark.parametrize("how", ["list", "in place", "no list", "no reach"])
def test_rows_spread_over_workgroups(device, T, B, how):
    """Ragged batches that fill T rows but for a few; with a list that ends early; mapped by the host."""
    r = np.random.RandomState(T + B)
    new = r.multinomial(T - 3 if T > B else T // 2, np.full(B, 1 / B) if B > 5 else r.dirichlet(np.ones(B)))
    ctx = r.randint(0, 200, B)
    width = int((ctx + new).max()) // 16 + 2
    table, free = mapped(T, ctx + new if how == "no list" else ctx, width, int((new // 16 + 2).sum()))
    if how == "no list":
        check(device, table, ctx, new, T)
    else:
        check(device, table, ctx, new, T, free[:len(free) // 4] if how == "no reach" else free, in_place=how == "in place")


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("T", [500, 600])
def test_blocks_that_are_negative(device, T):
    """In the list, in the table; at a sequence's first page or a later one."""
    ctx, new = [0, 20, 16, 5, 31], [100, 90, 64, 0, 200]
    for at in (0, 3, 9, 12, 17):
        table, free = mapped(9, ctx, 20, 40)
        free[at] = -5
        check(device, table, ctx, new, T, free)
    table, free = mapped(9, ctx, 20, 40)
    table[1, 1] = -1
    check(device, table, ctx, new, T, free)
    full, _ = mapped(9, [c + n for c, n in zip(ctx, new)], 20, 3)
    full[0, 4] = full[4, 2] = full[1, 1] = -3
    check(device, full, ctx, new, T)


@pytest.mark.parametrize("device", DEVICES)
def test_tables_that_the_host_mapped(device):
    ctx, new = [0, 15, 16, 30], [5, 2, 16, 40]
    table, _ = mapped(3, [c + n for c, n in zip(ctx, new)], 6, 2)
    check(device, table, ctx, new, sum(new))
    table[1, 1] = -1  # the second row's page of sequence 1: that row alone has no slot
    want = check(device, table, ctx, new, sum(new))
    assert want[-1] == BAD_BLOCK and want[4][5] >= 0 and want[4][6] == -1
    table[2, 1] = -1  # the first row's page: the whole sequence
    want = check(device, table, ctx, new, sum(new))
    assert (want[4][7:23] == -1).all() and want[2][2] == 16
    check(device, table, ctx, new, sum(new) + 5000)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("pad", [0, 5000])
def test_refused_sequences_leave_the_others(device, pad):
    ctx = [20, -1, 40, 150, 8, 16]
    new = [13, 1, -2, 20, 9, 0]
    table, free = mapped(4, [max(c, 0) for c in ctx], 10, 40)
    want = check(device, table, ctx, new, 43 + pad, free, 2)  # sequence 3 passes its table of 160
    assert want[-1] == TOO_LONG and list(want[2]) == [33, -1, 40, 150, 17, 16]
    table[0, 1] = -1  # sequence 0's partly filled page is not mapped
    want = check(device, table, ctx, new, 43 + pad, free, 2)
    assert want[-1] == TOO_LONG | BAD_BLOCK and want[2][0] == 20


@pytest.mark.parametrize("device", DEVICES)
def test_rows_past_the_batch(device):
    ctx, new = [0, 10, 5, 0], [6, 7, 2, 1]
    table, free = mapped(5, ctx, 4, 9)
    for T in (16, 15, 14, 13, 6, 5, 0):
        want = check(device, table, ctx, new, T, free)
        assert want[-1] == (0 if T == 16 else TOO_LONG)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("used", [0, 2, 4, 5, 6, 7, -1])
def test_a_free_list_that_ends(device, used):
    ctx, new = [16, 3, 32, 7, 0, 48], [17, 2, 1, 1, 20, 1]  # blocks: 2, 0, 1, 0, 2, 1
    table, free = mapped(6, ctx, 5, 6)
    want = check(device, table, ctx, new, sum(new), free, used)
    assert want[-1] == (0 if used == 0 else NO_BLOCKS)
    assert want[2][1] == 5 and want[2][3] == 8  # those that need none go on


@pytest.mark.parametrize("device", DEVICES)
def test_no_sequences_and_a_bad_free_block(device):
    check(device, np.zeros((0, 4), np.int32), [], [], 3, np.zeros(0, np.int32))
    check(device, np.zeros((0, 4), np.int32), [], [], 0)
    want = check(device, np.full((2, 3), -1, np.int32), [0, 0], [20, 3], 23, np.array([5, -4, 6], np.int32))
    assert want[-1] == BAD_BLOCK and (want[4][16:20] == -1).all() and want[4][20] == 96


@pytest.mark.parametrize("device", DEVICES)
def test_in_place_steps_follow_each_other(device):
    """ctx_after in ctx_len and free_after in free_used: a decode loop's calls, every state as the definition's."""
    ctx = np.array([0, 14, 31, 16], np.int32)
    table, free = mapped(7, ctx, 8, 30)
    t, c, n = i32(table, device), i32(ctx, device), i32([1, 1, 1, 1], device)
    cu, u, f = i32(np.zeros(5), device), i32([0], device), i32(free, device)
    pos, slots = (give(np.zeros(4, np.int64), device) for _ in range(2))
    used = 0
    for _ in range(40):
        L.Ops.paged_kv_map(t, cu, c, pos, slots, c, n, f, u, u)
        table, _, ctx, p, s, used, _ = map_plain(table, ctx, [1] * 4, 4, free, used)
        assert L.device_error_flags() == 0
        for got, want in ((t, table), (c, ctx), (pos, p), (slots, s), (u, [used])):
            np.testing.assert_array_equal(take(got).numpy(), want)


def test_refusals():
    dev = "cpu"
    z = lambda n: i32(np.zeros(n), dev)  # noqa: E731
    rows = lambda n: give(np.zeros(n, np.int64), dev)  # noqa: E731
    good = [i32(np.zeros((2, 3)), dev), z(3), z(2), rows(4), rows(4), z(2), z(2)]
    L.Ops.paged_kv_map(*good)
    L.device_error_flags()
    for at, bad in ((0, z(2)), (0, i32(np.zeros((3, 3)), dev)), (1, z(2)), (2, z(3)), (3, rows(5)), (4, z(4)),
                    (5, z(3)), (6, give(np.zeros(2, np.int64), dev)), (0, give(np.zeros((2, 3), np.int64), dev))):
        args = list(good)
        args[at] = bad
        with pytest.raises(L.LlaisysError, match="paged_kv_map"):
            L.Ops.paged_kv_map(*args)
    with pytest.raises(L.LlaisysError, match="go together"):
        L.Ops.paged_kv_map(*good, z(4))
    with pytest.raises(L.LlaisysError, match="free_used"):
        L.Ops.paged_kv_map(*good, z(4), z(2), z(1))
    with pytest.raises(L.LlaisysError):
        L.Ops.paged_kv_map(None, *good[1:])
