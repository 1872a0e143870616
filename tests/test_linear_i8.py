"""llaisysQuantizeRows and llaisysLinearI8 against their formulas in 64 bits.

The codes and scales are equal to the definition's (the scale is the quotient
rounded to 32 bits, the code the exact quotient's rounding). A product's error
is that of float(sum) * (a * b) + bias in 32 bits: three roundings of 2^-24
relative to the product, one more relative to the result, and the output's own
half step."""
import numpy as np
import pytest
import torch

import llaisys_amd as L
from cases_8bit import DEVICES, give, take

TYPES = [torch.bfloat16, torch.float16, torch.float32]


def quantize64(x: torch.Tensor):
    x = x.double().numpy()
    s = (np.abs(x).max(1, initial=0.0) / 127).astype(np.float32)
    s[~np.isfinite(x).all(1)] = np.nan
    with np.errstate(invalid="ignore", divide="ignore"):
        q = np.where(s[:, None] > 0, np.clip(np.rint(x / s.astype(np.float64)[:, None]), -127, 127), 0)
    return q.astype(np.int8), s


def quantize(device, x):
    q, s = give(torch.zeros(x.shape, dtype=torch.int8), device), give(torch.zeros(x.shape[0]), device)
    L.Ops.quantize_rows(q, s, give(x, device))
    return take(q).numpy(), take(s).numpy()


def check_rows(device, x):
    (q, s), (wq, ws) = quantize(device, x), quantize64(x)
    np.testing.assert_array_equal(s, ws)
    np.testing.assert_array_equal(q, wq)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M, K", [(1, 1), (1, 1536), (3, 7), (5, 64), (130, 129), (17, 8960), (2, 40000), (1, 8), (4, 2056)])
def test_rows(device, dtype, M, K):
    g = torch.Generator().manual_seed(M * 1000 + K)
    x = torch.randn(M, K, generator=g) * torch.exp2(4 * torch.randn(M, 1, generator=g))
    check_rows(device, x.to(dtype))


@pytest.mark.parametrize("device", DEVICES)
def test_rows_on_ties_and_next_to_them(device):
    # 127 s exactly, so that multiples of s / 2 are ties; and their neighbours in 32 bits.
    for s in (1.0, 0.75, 2.0 ** -20, 3.0 / 1024):
        ties = torch.arange(-254, 255, dtype=torch.float32) * (s / 2)
        x = torch.stack([ties, torch.nextafter(ties, torch.tensor(np.inf)), torch.nextafter(ties, torch.tensor(-np.inf))])
        x = x.clamp(-127 * s, 127 * s)
        x[:, 0] = 127 * s
        check_rows(device, x)
    # scales with all 24 bits, values at every half of them
    r = np.random.RandomState(5)
    top = torch.from_numpy(r.uniform(1, 2, (400, 1)).astype(np.float32))
    s = (top / 127).double()
    x = (s * (torch.arange(1, 254) / 2)[None, :].double()).float()
    check_rows(device, torch.cat([top, x], 1))


@pytest.mark.parametrize("device", DEVICES)
def test_rows_of_zeros_small_large_and_not_finite(device):
    x = torch.randn(9, 70, generator=torch.Generator().manual_seed(2))
    x[0] = 0
    x[1] *= 1e-38
    x[2] *= 1e-44
    x[3] = 3e38 * torch.sign(x[3])
    x[4, 5] = float("inf")
    x[5, 69] = float("nan")
    x[6] = 1e-45
    x[7] *= 1e-20
    x[8, 0] = -0.0
    check_rows(device, x)
    check_rows(device, x.to(torch.bfloat16))
    check_rows(device, (x.clamp(-6e4, 6e4)).to(torch.float16))


def product(device, q, s, w, ws, bias, dtype):
    y = give(torch.full((q.shape[0], w.shape[0]), 7.0, dtype=dtype), device)
    L.Ops.linear_i8(y, give(q, device), give(s, device), give(w, device), give(ws, device),
                    None if bias is None else give(bias, device))
    return take(y)


def check_product(device, M, N, K, dtype, with_bias, most=127, seed=0):
    g = torch.Generator().manual_seed(seed + 31 * M + N + K)
    q = torch.randint(-most, most + 1, (M, K), dtype=torch.int8, generator=g)
    w = torch.randint(-most, most + 1, (N, K), dtype=torch.int8, generator=g)
    s, ws = torch.rand(M, generator=g) * 0.05 / K ** 0.5, torch.rand(N, generator=g) * 0.05
    bias = torch.randn(N, generator=g).to(dtype) if with_bias else None
    got = product(device, q, s, w, ws, bias, dtype).double()
    dot = q.double() @ w.double().t() * s.double()[:, None] * ws.double()[None, :]
    want = dot if bias is None else dot + bias.double()
    bound = 3 * 2.0 ** -24 * dot.abs() + 2.0 ** -24 * want.abs() + torch.finfo(dtype).eps / 2 * want.abs() * 1.01
    bound += torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps  # a subnormal result's half step
    assert ((got - want).abs() <= bound).all(), ((got - want).abs() - bound).max()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M, N, K", [(1, 1, 1), (1, 100, 64), (3, 5, 7), (2, 130, 129), (17, 33, 48), (70, 65, 272), (33, 256, 1000)])
def test_products(device, dtype, M, N, K):
    check_product(device, M, N, K, dtype, M % 2 == 1)


@pytest.mark.gpu
@pytest.mark.parametrize("M, N, K, dtype, bias", [
    (1, 1536, 8960, torch.bfloat16, False), (4, 2048, 1536, torch.bfloat16, True), (7, 8960, 1536, torch.float16, True),
    (16, 1536, 1536, torch.float32, True), (30, 1536, 1040, torch.bfloat16, False), (64, 1536, 1536, torch.bfloat16, True),
    (129, 520, 8960, torch.bfloat16, True), (300, 1537, 528, torch.float16, False), (777, 2048, 1536, torch.bfloat16, True),
    (1024, 1000, 4096, torch.float32, False), (2050, 4100, 656, torch.bfloat16, True), (8192, 1536, 1536, torch.bfloat16, False),
    (257, 300, 130, torch.bfloat16, True), (1030, 514, 16, torch.float32, True), (5, 1536, 16384, torch.bfloat16, False),
    (2000, 4100, 129, torch.bfloat16, True), (9, 3000, 1001, torch.float16, False), (600, 700, 4099, torch.float32, True),
])
def test_larger_products(M, N, K, dtype, bias):
    check_product("amd", M, N, K, dtype, bias)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("off", [1, 4, 16])
@pytest.mark.parametrize("M, N, K", [(3, 40, 32), (130, 100, 96)])
def test_operands_that_begin_anywhere(device, off, M, N, K):
    """Views into larger buffers: contiguous, but not on a 16 B boundary."""
    g = torch.Generator().manual_seed(off + M)
    q, w = (torch.randint(-127, 128, (n, K), dtype=torch.int8, generator=g) for n in (M, N))
    x = torch.randn(M, K, generator=g).to(torch.bfloat16)
    one = lambda n: give(torch.ones(n), device)  # noqa: E731

    def view(t, dtype):
        flat = torch.zeros(off + t.numel(), dtype=dtype)
        flat[off:] = t.reshape(-1)
        return give(flat, device).slice(0, off, off + t.numel()).view(*t.shape)

    want = q.double() @ w.double().t()
    for a, b in ((view(q, torch.int8), give(w, device)), (give(q, device), view(w, torch.int8))):
        y = view(torch.zeros(M, N), torch.float32)
        L.Ops.linear_i8(y, a, one(M), b, one(N))
        flat = y.view(M * N)
        out = give(torch.zeros(M * N), device)
        L.Ops.rearrange(out, flat)
        assert (take(out).double().view(M, N) == want).all()
    codes, scale = view(torch.zeros(M, K), torch.int8), give(torch.zeros(M), device)
    L.Ops.quantize_rows(codes, scale, view(x, torch.bfloat16))
    out = give(torch.zeros(M, N), device)
    L.Ops.linear_i8(out, codes, scale, give(w, device), one(N))
    wq, ws = quantize64(x)
    np.testing.assert_array_equal(take(scale).numpy(), ws)
    dot = torch.from_numpy(wq).double() @ w.double().t() * torch.from_numpy(ws).double()[:, None]
    assert ((take(out).double() - dot).abs() <= 4 * 2.0 ** -24 * dot.abs()).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("K", [131071, 131056])
def test_the_longest_sums_are_exact(device, K):
    """All products of one sign and size, -128 among the codes: the sum is just under 2^31."""
    q, w = torch.full((2, K), -128, dtype=torch.int8), torch.full((3, K), -128, dtype=torch.int8)
    w[1] = 127
    w[2, ::2] = 127
    one = torch.ones(3)
    got = product(device, q, one[:2], w, one, None, torch.float32).double()
    want = q.double() @ w.double().t()
    assert ((got - want).abs() <= 2.0 ** -24 * want.abs()).all()


@pytest.mark.parametrize("device", DEVICES)
def test_scales_that_are_not_finite_show(device):
    x = torch.randn(3, 32)
    x[1, 4] = float("inf")
    q, s = quantize(device, x)
    w = torch.ones(4, 32, dtype=torch.int8)
    y = product(device, torch.from_numpy(q), torch.from_numpy(s), w, torch.ones(4), None, torch.float32)
    assert torch.isnan(y[1]).all() and torch.isfinite(y[[0, 2]]).all()


@pytest.mark.parametrize("device", DEVICES)
def test_empty_sizes(device):
    for M, N, K in ((0, 4, 16), (3, 0, 16), (3, 4, 0)):
        y = product(device, torch.zeros(M, K, dtype=torch.int8), torch.ones(M), torch.zeros(N, K, dtype=torch.int8),
                    torch.ones(N), torch.arange(N).float(), torch.float32)
        assert y.shape == (M, N) and (y == torch.arange(N).float()).all()
    q, s = quantize(device, torch.zeros(3, 0))
    assert (s == 0).all()
    quantize(device, torch.zeros(0, 5))


def test_refusals():
    dev = "cpu"
    i8 = lambda *s: give(torch.zeros(*s, dtype=torch.int8), dev)  # noqa: E731
    f = lambda *s: give(torch.zeros(*s), dev)  # noqa: E731
    x = f(4, 8)
    for bad in ((i8(4, 7), f(4), x), (i8(4, 8), f(3), x), (f(4, 8), f(4), x), (i8(4, 8), i8(4), x),
                (i8(4, 8), f(4), i8(4, 8)), (i8(8), f(4), f(8)), (i8(4, 8), f(4), f(8, 4).permute(1, 0))):
        with pytest.raises(L.LlaisysError, match="quantize_rows"):
            L.Ops.quantize_rows(*bad)
    good = [f(4, 5), i8(4, 8), f(4), i8(5, 8), f(5), f(5)]
    L.Ops.linear_i8(*good)
    for at, bad in ((0, f(5, 4)), (1, i8(4, 9)), (1, f(4, 8)), (2, f(5)), (3, f(5, 8)), (4, f(4)), (5, f(4)),
                    (5, give(torch.zeros(5, dtype=torch.bfloat16), dev)), (0, i8(4, 5)), (2, i8(4)),
                    (3, i8(8, 5).permute(1, 0))):
        args = list(good)
        args[at] = bad
        with pytest.raises(L.LlaisysError, match="linear_i8"):
            L.Ops.linear_i8(*args)
    with pytest.raises(L.LlaisysError, match="at most 131071"):
        L.Ops.linear_i8(f(1, 1), i8(1, 131072), f(1), i8(1, 131072), f(1))
