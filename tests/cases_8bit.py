"""Plain 64-bit forms of the 8-bit serving operators and their bridging: the
e4m3 page format, appends, attention, a step's tables, 8-bit integer products."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import llaisys_amd as L
from llaisys_amd import DataType, DeviceType, MemcpyKind

DEVICES = ["cpu", pytest.param("amd", marks=pytest.mark.gpu)]
LEAST = -100
TOO_LONG, BAD_BLOCK, NO_BLOCKS = 2, 1, 8

_LL = {torch.float32: DataType.F32, torch.float16: DataType.F16, torch.bfloat16: DataType.BF16,
       torch.int32: DataType.I32, torch.int64: DataType.I64, torch.int8: DataType.I8, torch.uint8: DataType.F8}
_TORCH = {v: k for k, v in _LL.items()}


def give(t, device: str) -> L.Tensor:
    """A fresh library tensor with a copy of t (torch; uint8 becomes F8)."""
    if isinstance(t, np.ndarray):
        t = torch.from_numpy(np.ascontiguousarray(t))
    t = t.contiguous().cpu()
    lt = L.Tensor(tuple(t.shape), dtype=_LL[t.dtype], device=DeviceType.CPU if device == "cpu" else DeviceType.AMD)
    if t.numel():
        lt.load(t.data_ptr())
    return lt


def take(lt: L.Tensor) -> torch.Tensor:
    """Its contents as a torch tensor on the host."""
    out = torch.empty(lt.shape(), dtype=_TORCH[lt.dtype()])
    if out.numel():
        cpu = lt.device_type() == DeviceType.CPU
        L.RuntimeAPI(lt.device_type()).memcpy_sync(out.data_ptr(), lt.data_ptr(), out.numel() * out.element_size(),
                                                   MemcpyKind.H2H if cpu else MemcpyKind.D2H)
    return out


# ------------------------------------------------------------------- format

_T, _D = np.meshgrid(np.arange(16), np.arange(128), indexing="ij")
K_AT = (_D // 64) * 1024 + (_D // 8 % 4) * 256 + _T * 16 + (_D // 32 % 2) * 8 + _D % 8
V_AT = (_D // 64) * 1024 + (_T // 4) * 256 + (_D % 16) * 16 + (_D // 16 % 4) * 4 + _T % 4


def _all_codes():
    c = np.arange(256)
    e, m = (c >> 3) & 15, c & 7
    v = np.where(e > 0, (8 + m) * 2.0 ** (e - 10.0), m * 2.0 ** -9)
    v[(c & 127) == 127] = np.nan
    return np.where(c & 128, -v, v)


CODES = _all_codes()  # the value of each code
_SORTED = np.sort(CODES[:127])  # the magnitudes, code by code


def encode64(y: np.ndarray) -> np.ndarray:
    """Codes nearest to y (|y| <= 448), ties to the even code; not finite: NaN."""
    a = np.minimum(np.abs(y), 448.0)
    fine = np.isfinite(y)
    a = np.where(fine, a, 0.0)
    hi = np.searchsorted(_SORTED, a)  # the first magnitude >= a
    lo = np.maximum(hi - 1, 0)
    up, down = _SORTED[hi] - a, a - _SORTED[lo]
    code = np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    code = np.where(_SORTED[hi] == a, hi, code)
    return np.where(fine, code | np.where(np.signbit(y), 128, 0), 127).astype(np.uint8)


def exp_of(top: np.ndarray) -> np.ndarray:
    """The exponent of a block's scale from its largest finite magnitude."""
    top = np.asarray(top, np.float64)
    m, e = np.frexp(top / 448)
    return np.where(top > 0, np.maximum(np.where(m == 0.5, e - 1, e), LEAST), LEAST)


class Cache:
    """A logical 8-bit cache: codes by [block, head, token, dim] and exponents."""

    def __init__(self, blocks: int, nkvh: int, seed: int):
        r = np.random.RandomState(seed)
        self.codes = [r.randint(0, 256, (blocks, nkvh, 16, 128)).astype(np.uint8) for _ in range(2)]
        self.exps = [r.randint(-12, 6, (blocks, nkvh)) for _ in range(2)]

    def device(self, device: str):
        """(k_pool, v_pool, k_scale, v_scale) on a device."""
        pools = []
        for codes, at in zip(self.codes, (K_AT, V_AT)):
            flat = np.empty(codes.shape[:2] + (2048,), np.uint8)
            flat[:, :, at] = codes
            pools.append(give(flat.reshape(codes.shape), device))
        return (*pools, *(give((2.0 ** e).astype(np.float32), device) for e in self.exps))

    def values(self, which: int) -> np.ndarray:
        return CODES[self.codes[which]] * 2.0 ** self.exps[which][..., None, None]

    def check(self, kp, vp, ks, vs):
        """The device's cache holds these codes (any NaN code for a NaN) and scales."""
        for which, (pool, scale, at) in enumerate(((kp, ks, K_AT), (vp, vs, V_AT))):
            np.testing.assert_array_equal(take(scale).numpy(), (2.0 ** self.exps[which]).astype(np.float32))
            got = take(pool).numpy().reshape(self.codes[which].shape[:2] + (2048,))[:, :, at]
            want = self.codes[which]
            same = (got == want) | (((got & 127) == 127) & ((want & 127) == 127))
            assert same.all(), f"{'KV'[which]}: {np.argwhere(~same)[:4]}"

    def append(self, k_new, v_new, slots):
        """Rows [T, nkvh, 128] (64-bit values of bf16 numbers) to slots; runs of a block are consecutive."""
        r = 0
        while r < len(slots):
            if slots[r] < 0:
                r += 1
                continue
            block, off, n = slots[r] // 16, slots[r] % 16, 1
            while off + n < 16 and r + n < len(slots) and slots[r + n] == slots[r] + n:
                n += 1
            for which, rows in enumerate((k_new, v_new)):
                x = rows[r:r + n].transpose(1, 0, 2)  # [nkvh, n, 128]
                need = exp_of(np.where(np.isfinite(x), np.abs(x), 0).max((1, 2)))
                was = np.full_like(need, LEAST) if off == 0 else self.exps[which][block]
                now = np.maximum(was, need)
                for h in range(len(now)):
                    if off and now[h] != was[h]:
                        old = self.codes[which][block, h]
                        again = encode64(CODES[old] * 2.0 ** (was[h] - now[h]))
                        self.codes[which][block, h] = np.where((old & 127) == 127, old, again)
                    self.codes[which][block, h, off:off + n] = encode64(x[h] * 2.0 ** -float(now[h]))
                self.exps[which][block] = now
            r += n


def bf16(x) -> torch.Tensor:
    return torch.as_tensor(np.asarray(x), dtype=torch.float64).to(torch.bfloat16)


def f64(t: torch.Tensor) -> np.ndarray:
    return t.to(torch.float64).numpy()


def table_of(seed: int, lens, spare: int = 3, extra_pages: int = 0):
    """A block table of randomly placed blocks for these lengths, and the number of blocks."""
    pages = [-(-int(n) // 16) for n in lens]
    blocks = sum(pages) + spare
    order = np.random.RandomState(seed).permutation(blocks)
    table = np.full((len(lens), max(pages + [1]) + extra_pages), -1, np.int32)
    at = 0
    for b, p in enumerate(pages):
        table[b, :p] = order[at:at + p]
        at += p
    return table, blocks


def attend64(q, K, V, scale):
    """q [L, nh, d], K, V [S, nkvh, d]: causal, the last rows aligned. Returns (out, most |score| sum, most |v|)."""
    n, nh, _ = q.shape
    S, nkvh = K.shape[:2]
    out = np.empty_like(q)
    most = 0.0
    for h in range(nh):
        k, v = K[:, h // (nh // nkvh)], V[:, h // (nh // nkvh)]
        s = (q[:, h] @ k.T) * scale
        most = max(most, float((np.abs(q[:, h]) @ np.abs(k).T).max()) * scale)
        s[np.arange(S)[None, :] > np.arange(n)[:, None] + S - n] = -np.inf
        p = np.exp(s - s.max(-1, keepdims=True))
        out[:, h] = p @ v / p.sum(-1, keepdims=True)
    return out, most


# ------------------------------------------------------------- step's tables

def map_plain(table, ctx, new, T, free=None, used=0):
    """(table, cu, after, pos, slots, free_after, error bits) by the definition, one row at a time."""
    table = table.copy()
    B, width = table.shape
    cu, after = [0], []
    pos, slots = np.zeros(T, np.int64), np.full(T, -1, np.int64)
    avail = max(0, len(free) - used) if free is not None and used >= 0 else 0
    asked, wanted, taken, flags = 0, 0, 0, 0
    for b in range(B):
        c, n = int(ctx[b]), int(new[b])
        begin = min(asked, T)
        asked += max(n, 0)
        ok = c >= 0 and n >= 0 and c + n <= width * 16 and asked <= T
        flags |= 0 if ok else TOO_LONG
        if ok and n > 0 and (c % 16 or free is None) and table[b, c // 16] < 0:
            ok, flags = False, flags | BAD_BLOCK
        if ok and free is not None:
            pages = list(range(-(-c // 16), -(-(c + n) // 16)))
            wanted += len(pages)
            if pages and wanted > avail:
                ok, flags = False, flags | NO_BLOCKS
            elif pages:
                for i, p in enumerate(pages):
                    table[b, p] = free[used + taken + i]
                taken = wanted
        put = ok and n > 0
        for r in range(begin, min(asked, T)):
            p = c + r - begin
            if put and table[b, p // 16] < 0:
                flags |= BAD_BLOCK
                put = put and r > begin
            elif put:
                pos[r], slots[r] = p, int(table[b, p // 16]) * 16 + p % 16
        cu.append(min(asked, T))
        after.append(c + (n if ok else 0))
    return (table, np.array(cu, np.int32), np.array(after, np.int32), pos, slots, used + taken, flags)
