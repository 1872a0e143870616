"""The 8-bit serving operators as cases that can be timed and checked.

Kinds of case (key "kind"), each one pass of a serving step's part:

  map     Ops.paged_kv_map: a step's block table entries, row offsets, lengths,
          positions and slots from the requests' lengths
  append  Ops.paged_kv_append_f8: new K/V rows into the 8-bit cache by their
          slots (with "gather": then every context out as rows by
          Ops.paged_kv_gather_f8)
  decode  Ops.paged_attention_f8: one query per sequence over the 8-bit cache
  mixed   Ops.paged_attention_varlen_f8: prompt chunks and decodes in one batch
  linear  Ops.quantize_rows, then Ops.linear_i8 with a weight kept in 8 bits

Each kind has a plain form beside it, of elementary torch operations. The 8-bit
cache holds e4m3 codes and, for each block of 16 tokens and kv head, one scale
2^E, E the least whole number (of -100 and more) whose scale reaches the
block's largest value. A (block, kv head) page holds code (token t, dim d) at
byte
  K: (d / 64) * 1024 + (d / 8 % 4) * 256 + t * 16 + (d / 32 % 2) * 8 + d % 8
  V: (d / 64) * 1024 + (t / 4) * 256 + (d % 16) * 16 + (d / 16 % 4) * 4 + t % 4

Sizes are the shape the benchmark and the tests use (hidden 1536, 12 query and
2 KV heads of 128, FFN 8960) and odd neighbours of it. Lengths within a batch
are spread evenly over their range and shuffled by the seed, so a case's work
does not depend on it.
"""
import math

import numpy as np
import torch

own = False  # the framework's kernels (True) or the plain forms

HEAD = 128  # head dim of the paged KV
PAGE = 16   # tokens of a page
LEAST = -100  # the least exponent of a block's scale
SCALE = 1.0 / math.sqrt(HEAD)

_FLOAT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}


# ---------------------------------------------------------------- the cases

def listed():
    return [
        # The host-free decode step of a server: one new token for each of 64 requests.
        {"name": "map_decode", "kind": "map", "batch": 64, "ctx_hi": 8192, "chunks": 0, "chunk": 1, "pad": 0},
        # A large step: 24 prompt chunks beside 400 decodes, rows padded to a fixed size.
        {"name": "map_step", "kind": "map", "batch": 424, "ctx_hi": 16384, "chunks": 24, "chunk": 2048, "pad": 333},
        # One layer's append of a decode step.
        {"name": "append_decode", "kind": "append", "batch": 64, "ctx_hi": 8192, "new": 1, "nkvh": 2,
         "gather": False},
        # One layer's append of a long prefill step: ragged chunks, 8k tokens.
        {"name": "append_prompt", "kind": "append", "batch": 5, "ctx_hi": 4100, "new": 1640, "nkvh": 2,
         "gather": False},
        # The append and gather benchmark's shape, from the 8-bit cache.
        {"name": "append_gather", "kind": "append", "batch": 32, "ctx_hi": 2048, "new": 1, "nkvh": 2,
         "gather": True},
        # A single chat's next token: one sequence, a short context; latency.
        {"name": "decode_one", "kind": "decode", "batch": 1, "ctx_lo": 700, "ctx_hi": 700, "nh": 12, "nkvh": 2,
         "out": "bf16"},
        # The benchmark's decode batch: 64 sequences of very different lengths.
        {"name": "decode_batch", "kind": "decode", "batch": 64, "ctx_lo": 512, "ctx_hi": 8192, "nh": 12, "nkvh": 2,
         "out": "bf16"},
        # A fresh prompt alone.
        {"name": "prompt_alone", "kind": "mixed", "chunks": 1, "chunk": 777, "prior": 0, "decodes": 0, "ctx_lo": 1,
         "ctx_hi": 1, "nh": 12, "nkvh": 2},
        # The benchmark's mixed step of a server: 4 prompt chunks and 60 decodes.
        {"name": "mixed_step", "kind": "mixed", "chunks": 4, "chunk": 512, "prior": 4096, "decodes": 60,
         "ctx_lo": 256, "ctx_hi": 4096, "nh": 12, "nkvh": 2},
        # One token through the output of a feed-forward layer.
        {"name": "linear_token", "kind": "linear", "m": 1, "n": 1536, "k": 8960, "x": "bf16", "y": "bf16",
         "bias": False},
        # A ragged prompt through a biased projection.
        {"name": "linear_ragged", "kind": "linear", "m": 777, "n": 2048, "k": 1536, "x": "bf16", "y": "bf16",
         "bias": True},
        # The largest projection of a long prefill step.
        {"name": "linear_prompt", "kind": "linear", "m": 8192, "n": 17920, "k": 1536, "x": "bf16", "y": "bf16",
         "bias": False},
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    kind = rng.choice(["map", "append", "append", "decode", "decode", "mixed", "mixed", "linear", "linear"])
    if kind == "map":
        batch, hi = _log(rng, 1, 424), _log(rng, 32, 16384)
        chunks = rng.choice([0, rng.randint(0, min(batch, 24))])
        return {"kind": kind, "batch": batch, "ctx_hi": hi, "chunks": chunks,
                "chunk": _log(rng, 2, 2048) if chunks else 1, "pad": rng.choice([0, rng.randint(1, 333)])}
    if kind == "append":
        gather = rng.random() < 0.4
        batch, hi = _log(rng, 1, 64), _log(rng, 1, 8192)
        if gather:
            return {"kind": kind, "batch": batch, "ctx_hi": min(hi, max(1, 65_000 // batch)), "new": 1,
                    "nkvh": rng.choice([2, 2, 1, 4]), "gather": True}
        return {"kind": kind, "batch": batch, "ctx_hi": hi, "new": rng.choice([1, min(_log(rng, 2, 4000), 8000 // batch)]),
                "nkvh": rng.choice([2, 2, 2, 1]), "gather": False}
    if kind == "decode":
        batch, hi = _log(rng, 1, 128), _log(rng, 32, 16384)
        hi = min(hi, max(32, 560_000 // batch))
        nh, nkvh = rng.choice([(12, 2), (12, 2), (12, 2), (8, 2), (16, 1), (4, 4)])
        if nkvh > 2:
            hi = min(hi, max(32, 280_000 // batch))
        return {"kind": kind, "batch": batch, "ctx_lo": rng.randint(1, hi), "ctx_hi": hi, "nh": nh, "nkvh": nkvh,
                "out": rng.choice(["bf16", "bf16", "bf16", "f32"])}
    if kind == "mixed":
        chunk, chunks = _log(rng, 17, 2000), rng.randint(1, 6)
        chunk = min(chunk, 2048 // chunks)
        hi = _log(rng, 64, 4096)
        nh, nkvh = rng.choice([(12, 2), (12, 2), (8, 2)])
        return {"kind": kind, "chunks": chunks, "chunk": chunk, "prior": rng.choice([0, _log(rng, 16, 4096)]),
                "decodes": rng.choice([0, _log(rng, 1, 60)]), "ctx_lo": rng.randint(1, hi), "ctx_hi": hi, "nh": nh,
                "nkvh": nkvh}
    n, k = rng.choice([(2048, 1536), (1536, 1536), (17920, 1536), (1536, 8960),
                       (_log(rng, 100, 9000), rng.choice([1, 16, 16]) * _log(rng, 40, 256))])
    x = rng.choice(["bf16", "bf16", "bf16", "f16", "f32"])
    return {"kind": kind, "m": rng.choice([_log(rng, 1, 64), _log(rng, 1, 8000)]), "n": n, "k": k, "x": x,
            "y": rng.choice([x, x, "f32" if n < 9000 else x]), "bias": rng.random() < 0.5}


# ------------------------------------------------- torch and the library

class _Memory:
    def __init__(self, ptr, shape, typestr, owner):
        self.owner = owner
        self.__cuda_array_interface__ = {"data": (ptr, False), "shape": tuple(shape), "typestr": typestr,
                                         "strides": None, "version": 3}


def _library():
    """{torch dtype: (library dtype, typestr of its memory)}, and the AMD runtime."""
    from llaisys_amd import DataType as D, DeviceType, RuntimeAPI
    return {torch.float32: (D.F32, "<f4"), torch.float16: (D.F16, "<f2"), torch.bfloat16: (D.BF16, "<i2"),
            torch.int32: (D.I32, "<i4"), torch.int64: (D.I64, "<i8"), torch.int8: (D.I8, "|i1"),
            torch.float8_e4m3fn: (D.F8, "|u1")}, RuntimeAPI(DeviceType.AMD)


def _give(s, **tensors):
    """Puts the tensors into the state: as they are, or as library tensors with
    torch views of the same memory beside them."""
    for name, t in tensors.items():
        if own:
            from llaisys_amd import DeviceType, MemcpyKind, Tensor
            types, api = _library()
            t = t.contiguous()
            lt = Tensor(tuple(t.shape), dtype=types[t.dtype][0], device=DeviceType.AMD)
            if t.numel():
                torch.cuda.current_stream().synchronize()
                api.memcpy_sync(lt.data_ptr(), t.data_ptr(), t.numel() * t.element_size(), MemcpyKind.D2D)
            s["lib"][name] = lt
            if t.numel():
                t = torch.as_tensor(_Memory(lt.data_ptr(), lt.shape(), types[t.dtype][1], lt),
                                    device="cuda:0").view(t.dtype)
        s[name] = t


def _gen(seed, salt=0):
    return torch.Generator(device="cuda:0").manual_seed((int(seed) * 1_000_003 + salt) & ((1 << 62) - 1))


def _normal(g, shape, std=1.0, dtype=torch.float32):
    return torch.empty(tuple(shape), dtype=torch.float32, device="cuda:0").normal_(0.0, std, generator=g).to(dtype)


def _spread(lo, hi, n, seed=None):
    """n lengths evenly over [lo, hi], in the seed's order (None: rising)."""
    v = [int(round(lo + (hi - lo) * ((i + 0.5) / n if n > 1 else 1.0))) for i in range(n)]
    if seed is not None:
        v = [v[i] for i in np.random.RandomState(int(seed) % (1 << 31)).permutation(n)]
    return v


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda:0")


# ------------------------------------------------------------ paged inputs

def _pages(x):
    return (x + PAGE - 1) // PAGE


def _table(seed, lens, spare, blocks=0):
    """A block table that maps these lengths to random blocks of a pool with
    `spare` more than they take (or with `blocks`), its free blocks in a random
    order, and the number of blocks."""
    pages = [max(1, _pages(n)) for n in lens]
    blocks = blocks or sum(pages) + spare
    order = np.random.RandomState((int(seed) + 17) % (1 << 31)).permutation(blocks)
    table = np.full((len(lens), max(pages)), -1, np.int32)
    at = 0
    for b, p in enumerate(pages):
        table[b, :p] = order[at:at + p]
        at += p
    return table, order[at:].astype(np.int32), blocks


def _cache(g, blocks, nkvh, is_v):
    """Codes of a cache as it is after some serving (all slots written) in page
    order, and the blocks' scales. Keys have channels of larger values."""
    x = _normal(g, (blocks, nkvh, PAGE, HEAD))
    if not is_v:
        bias = _normal(g, (nkvh, 1, HEAD))
        bias[..., ::32] *= 8
        x += bias
    top = x.abs().amax((2, 3), keepdim=True)
    m, e = torch.frexp(top / 448)
    e = (e - (m == 0.5).to(e.dtype)).clamp_(min=LEAST)
    codes = torch.ldexp(x, -e)
    if is_v:  # [t / 4][t % 4][d / 64][d / 16 % 4][d % 16] -> [d / 64][t / 4][d % 16][d / 16 % 4][t % 4]
        codes = codes.view(blocks, nkvh, 4, 4, 2, 4, 16).permute(0, 1, 4, 2, 6, 5, 3)
    else:  # [t][d / 64][d / 32 % 2][d / 8 % 4][d % 8] -> [d / 64][d / 8 % 4][t][d / 32 % 2][d % 8]
        codes = codes.view(blocks, nkvh, PAGE, 2, 2, 4, 8).permute(0, 1, 3, 5, 2, 4, 6)
    codes = codes.reshape(blocks, nkvh, PAGE, HEAD).to(torch.float8_e4m3fn)
    return codes, torch.ldexp(torch.ones_like(m), e).view(blocks, nkvh)


def _rows_of(codes, scale, table, is_v):
    """Every sequence's keys or values, [B, pages * 16, nkvh, 128] in 32 bits; table entries of -1 count as 0."""
    at = table.long().clamp(min=0)
    x = codes.view(torch.uint8)[at].view(torch.float8_e4m3fn).float()  # [B, P, nkvh, 16, 128], in page order
    B, P, nkvh = x.shape[:3]
    x = x * scale[at][..., None, None]
    if is_v:
        x = x.view(B, P, nkvh, 2, 4, 16, 4, 4).permute(0, 1, 4, 7, 2, 3, 6, 5)
    else:
        x = x.view(B, P, nkvh, 2, 4, PAGE, 2, 8).permute(0, 1, 5, 2, 3, 6, 4, 7)
    return x.reshape(B, P * PAGE, nkvh, HEAD)


def _places(is_v):
    """Byte of (token, dim) within a page, [16, 128]."""
    t = torch.arange(PAGE, device="cuda:0")[:, None]
    d = torch.arange(HEAD, device="cuda:0")[None, :]
    if is_v:
        return (d // 64) * 1024 + (t // 4) * 256 + (d % 16) * 16 + (d // 16 % 4) * 4 + t % 4
    return (d // 64) * 1024 + (d // 8 % 4) * 256 + t * 16 + (d // 32 % 2) * 8 + d % 8


def _map_shape(case, seed):
    """(lengths before, new tokens) of a step's requests, in the seed's order."""
    ctx = _spread(0, case["ctx_hi"], case["batch"])
    new = [1 + (case["chunk"] - 1) * (i + 1) // case["chunks"] for i in range(case["chunks"])]
    new += [1] * (case["batch"] - case["chunks"])
    if seed is not None:
        r = np.random.RandomState(int(seed) % (1 << 31))
        ctx = [ctx[i] for i in r.permutation(len(ctx))]
        new = [new[i] for i in r.permutation(len(new))]
    return ctx, new


def _append_shape(case, seed):
    """(lengths before, new tokens): ragged chunks, each a little shorter than the one before."""
    ctx = _spread(0, case["ctx_hi"], case["batch"], seed)
    return ctx, [max(1, case["new"] - 3 * i) for i in range(case["batch"])]


def _append_table(case, seed):
    """Lengths, new tokens, block table and pool size (the same in every order of the lengths)."""
    ctx, new = _append_shape(case, seed)
    blocks = sum(_pages(c) + _pages(n) + 1 for c, n in zip(ctx, new)) + 3
    table, _, blocks = _table(seed, [c + n for c, n in zip(ctx, new)], 0, blocks)
    return ctx, new, table, blocks


def _append_rows(case, seed, total):
    """New keys and values, some tokens larger than the rest, so that scales grow."""
    g = _gen(seed, 3)
    size = torch.exp2(_normal(g, (total, 1, 1)))
    shape = (total, case["nkvh"], HEAD)
    return ((_normal(g, shape) * size).to(torch.bfloat16), (_normal(g, shape) * size).to(torch.bfloat16))


def _append_slots(table, ctx, new):
    """Slot (block * 16 + offset) of every new row."""
    out = []
    for b, (c, n) in enumerate(zip(ctx, new)):
        pos = np.arange(c, c + n)
        out.append(table[b, pos // PAGE].astype(np.int64) * PAGE + pos % PAGE)
    return np.concatenate(out)


def _mixed_shape(case, seed):
    """(queries per sequence, contexts) of a mixed batch: chunks first (None) or in the seed's order."""
    last = max(1, case["chunks"] - 1)
    priors = [case["prior"] * i // last if case["chunks"] > 1 else case["prior"] for i in range(case["chunks"])]
    q = [max(2, case["chunk"] - 3 * i) for i in range(case["chunks"])]
    ctx = [p + n for p, n in zip(priors, q)]
    q += [1] * case["decodes"]
    ctx += _spread(case["ctx_lo"], case["ctx_hi"], case["decodes"]) if case["decodes"] else []
    if seed is not None:
        o = np.random.RandomState(int(seed) % (1 << 31)).permutation(len(q))
        q, ctx = [q[i] for i in o], [ctx[i] for i in o]
    return q, ctx


def _attention_inputs(case, seed):
    """Lengths, table, cache and queries of a decode or mixed case."""
    if case["kind"] == "mixed":
        qn, lens = _mixed_shape(case, seed)
    else:
        lens = _spread(case["ctx_lo"], case["ctx_hi"], case["batch"], seed)
        qn = [1] * len(lens)
    table, _, blocks = _table(seed, lens, 3)
    g = _gen(seed, 1)
    k = _cache(g, blocks, case["nkvh"], False)
    v = _cache(g, blocks, case["nkvh"], True)
    q = _normal(g, (sum(qn), case["nh"], HEAD), 1.0, torch.bfloat16)
    return qn, lens, torch.from_numpy(table).cuda(), k, v, q


def _linear_inputs(case, seed):
    """Rows of x, the weight's codes and scales, the bias."""
    g = _gen(seed, 2)
    x = _normal(g, (case["m"], case["k"]))
    x[:, :: 97] *= 6  # a few large channels, as hidden states have
    x = x.to(_FLOAT[case["x"]])
    w = _normal(g, (case["n"], case["k"]), 0.02)
    ws = w.abs().amax(1) / 127
    wq = torch.round(w / ws[:, None]).clamp_(-127, 127).to(torch.int8)
    bias = _normal(g, (case["n"],), 0.1, _FLOAT[case["y"]]) if case["bias"] else None
    return x, wq, ws, bias


# ------------------------------------------------------------------ prepare

def prepare(case, seed):
    kind = case["kind"]
    s = {"case": case, "lib": {}}
    zeros = lambda shape, dtype: torch.zeros(shape, dtype=dtype, device="cuda:0")  # noqa: E731
    if kind == "map":
        ctx, new = _map_shape(case, seed)
        table, free, _ = _table(seed, ctx, sum(_pages(c + n) - _pages(c) for c, n in zip(ctx, new)) + 40)
        wide = np.full((len(ctx), _pages(case["ctx_hi"] + case["chunk"]) + 2), -1, np.int32)
        for b, c in enumerate(ctx):
            wide[b, :_pages(c)] = table[b, :_pages(c)]
        rows = sum(new) + case["pad"]
        _give(s, table=torch.from_numpy(wide).cuda(), ctx=_i32(ctx), new=_i32(new), free=torch.from_numpy(free).cuda(),
              used=_i32([7]), cu=zeros(len(ctx) + 1, torch.int32), after=zeros(len(ctx), torch.int32),
              pos=zeros(rows, torch.int64), slots=zeros(rows, torch.int64), used_after=zeros(1, torch.int32))
    elif kind == "append":
        ctx, new, table, blocks = _append_table(case, seed)
        total = [c + n for c, n in zip(ctx, new)]
        g = _gen(seed, 1)
        kp, ks = _cache(g, blocks, case["nkvh"], False)
        vp, vs = _cache(g, blocks, case["nkvh"], True)
        kn, vn = _append_rows(case, seed, sum(new))
        _give(s, kp=kp, ks=ks, vp=vp, vs=vs, kn=kn, vn=vn,
              slots=torch.from_numpy(_append_slots(table, ctx, new)).cuda())
        if case["gather"]:
            rows = (sum(total), case["nkvh"], HEAD)
            _give(s, table=torch.from_numpy(table).cuda(), cu=_i32(np.concatenate([[0], np.cumsum(total)])),
                  ko=zeros(rows, torch.bfloat16), vo=zeros(rows, torch.bfloat16))
    elif kind in ("decode", "mixed"):
        qn, lens, table, k, v, q = _attention_inputs(case, seed)
        _give(s, kp=k[0], ks=k[1], vp=v[0], vs=v[1], table=table, ctx=_i32(lens), q=q)
        if kind == "mixed":
            cu = np.concatenate([[0], np.cumsum(qn)])
            _give(s, cu=_i32(cu), out=zeros(q.shape, torch.bfloat16))
            # which sequences are chunks and which single queries, as the host that forms the batch knows
            s["groups"] = [torch.tensor(ids, device="cuda:0") for ids in
                           ([i for i, n in enumerate(qn) if n > 1], [i for i, n in enumerate(qn) if n == 1]) if ids]
            s["longest"] = [max(n for n in qn if n > 1), 1] if max(qn) > 1 else [1]
        else:
            _give(s, out=zeros(q.shape, _FLOAT[case["out"]]))
    else:
        x, wq, ws, bias = _linear_inputs(case, seed)
        _give(s, x=x, wq=wq, ws=ws, xq=zeros(x.shape, torch.int8), xs=zeros(x.shape[0], torch.float32),
              y=zeros((case["m"], case["n"]), _FLOAT[case["y"]]))
        if bias is not None:
            _give(s, bias=bias)
    return s


# ---------------------------------------------------------- the plain forms

def _plain_map(s):
    table, T = s["table"], s["slots"].shape[0]
    B, width = table.shape
    ctx, new, used = s["ctx"].long(), s["new"].long().clamp(min=0), s["used"].long()
    ends = torch.cumsum(new, 0)
    cu = torch.cat([torch.zeros_like(used), ends]).clamp(max=T)
    ok = (s["new"] >= 0) & (ctx >= 0) & (ctx + new <= width * PAGE) & (ends <= T)
    first, last = _pages(ctx), _pages(ctx + new)
    need = torch.where(ok, last - first, 0)
    before = torch.cumsum(need, 0) - need
    ok &= (need == 0) | (before + need <= s["free"].shape[0] - used)
    need = torch.where(ok, need, 0)
    page = torch.arange(width, device=table.device)[None, :]
    fresh = ok[:, None] & (page >= first[:, None]) & (page < last[:, None])
    at = (used + before - first)[:, None] + page
    table = torch.where(fresh, s["free"][at.clamp(0, s["free"].shape[0] - 1)], table)
    r = torch.arange(T, device=table.device)
    b = torch.searchsorted(ends, r, right=True)
    some = b < B
    b = b.clamp(max=B - 1)
    pos = ctx[b] + r - cu[b]
    some &= ok[b]
    block = table[b, (pos // PAGE).clamp(0, width - 1)].long()
    return {"table": table, "cu": cu.int(), "ctx": torch.where(ok, ctx + new, ctx).int(),
            "pos": torch.where(some, pos, 0), "slots": torch.where(some & (block >= 0), block * PAGE + pos % PAGE, -1),
            "used": (used + need.sum()).int()}


def _plain_append_one(codes, scale, rows, slots, is_v):
    flat = codes.view(torch.uint8).view(codes.shape[0], codes.shape[1], PAGE * HEAD)
    block, off = slots // PAGE, slots % PAGE
    top = rows.float().abs().amax(2) / 448
    m, e = torch.frexp(top)
    e = torch.where(top > 0, e - (m == 0.5).to(e.dtype), LEAST).clamp(min=LEAST)
    old = torch.frexp(scale)[1] - 1
    fresh = torch.zeros(codes.shape[0], dtype=torch.bool, device=codes.device)
    fresh[block[off == 0]] = True
    new = torch.where(fresh[:, None], LEAST, old)
    new = new.scatter_reduce(0, block[:, None].expand(-1, codes.shape[1]), e, "amax")
    # the blocks' earlier tokens at their new scale (slots that are written next come with them), then the new rows
    touched = torch.unique(block)
    was = flat[touched].view(torch.float8_e4m3fn).float()
    was = torch.ldexp(was, (old - new)[touched][..., None])
    kept = ~fresh[touched][:, None, None] & ((new != old)[touched][..., None])
    flat[touched] = torch.where(kept, was.to(torch.float8_e4m3fn).view(torch.uint8), flat[touched])
    fill = torch.ldexp(rows.float(), -new[block][..., None]).to(torch.float8_e4m3fn).view(torch.uint8)
    heads = torch.arange(codes.shape[1], device=codes.device)
    flat[block[:, None, None], heads[None, :, None], _places(is_v)[off][:, None, :]] = fill
    scale.copy_(torch.ldexp(torch.ones_like(scale), new))


def _plain_gather(s, codes, scale, is_v):
    x = _rows_of(codes, scale, s["table"], is_v)
    lens = s["cu"][1:] - s["cu"][:-1]
    return x[torch.arange(x.shape[1], device=x.device)[None, :] < lens[:, None]].to(torch.bfloat16)


def _plain_attend(q, k, v, ctx, lq):
    """q [B, L, nh, 128] (sequence b's lq[b] rows first), k, v [B, S, nkvh, 128] -> as q, in 32 bits."""
    B, L, nh, _ = q.shape
    S, nkvh = k.shape[1:3]
    q = q.float().view(B, L, nkvh, nh // nkvh, HEAD).permute(0, 2, 3, 1, 4).reshape(B, nkvh, -1, HEAD)
    a = torch.matmul(q, k.permute(0, 2, 3, 1).contiguous()) * SCALE
    a = a.view(B, nkvh, nh // nkvh, L, S)
    seen = ctx[:, None] - lq[:, None] + torch.arange(L, device=q.device)[None, :]
    a = a.masked_fill(torch.arange(S, device=q.device) > seen[:, None, None, :, None], -math.inf)
    p = torch.exp(a - a.amax(-1, keepdim=True))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(B, nkvh, -1, S), v.permute(0, 2, 1, 3).contiguous())
    o = o.view(B, nkvh, nh // nkvh, L, HEAD) / total
    return o.permute(0, 3, 1, 2, 4).reshape(B, L, nh, HEAD)


def _plain_attention(s, ids, longest, out):
    """The queries of the sequences `ids` (None: all, one each) into out."""
    table, ctx = s["table"], s["ctx"].long()
    if ids is None:
        rows = torch.arange(ctx.shape[0], device=ctx.device)[:, None]
        lq = torch.ones_like(ctx)
    else:
        table, ctx = table[ids], ctx[ids]
        lq = (s["cu"][1:] - s["cu"][:-1]).long()[ids]
        rows = s["cu"].long()[ids][:, None] + torch.arange(longest, device=ctx.device)[None, :]
    have = torch.arange(longest, device=ctx.device)[None, :] < lq[:, None]
    # rows past a sequence's last query attend as its last one does and are dropped
    q = s["q"][torch.minimum(rows, rows[:, :1] + lq[:, None] - 1)]
    k = _rows_of(s["kp"], s["ks"], table, False)
    v = _rows_of(s["vp"], s["vs"], table, True)
    o = _plain_attend(q, k, v, ctx, lq)
    out[rows[have]] = o[have].to(out.dtype)


def _plain_linear(s):
    x, bias = s["x"].float(), s.get("bias")
    xs = (x.abs().amax(1).double() / 127).float()  # (a quotient by a number would be a product by its rounded inverse)
    q = torch.round(x.double() / torch.where(xs > 0, xs, 1).double()[:, None]).clamp(-127, 127).float()
    y = torch.matmul(q, s["wq"].float().t()) * (xs[:, None] * s["ws"][None, :])
    return {"y": (y if bias is None else y + bias.float()).to(s["y"].dtype), "scale": xs}


# ---------------------------------------------------------------------- run

def run(s):
    case = s["case"]
    kind = case["kind"]
    if own:
        from llaisys_amd import Ops
        t = s["lib"]
        if kind == "map":
            Ops.paged_kv_map(t["table"], t["cu"], t["after"], t["pos"], t["slots"], t["ctx"], t["new"], t["free"],
                             t["used"], t["used_after"])
            return {"table": s["table"], "cu": s["cu"], "ctx": s["after"], "pos": s["pos"], "slots": s["slots"],
                    "used": s["used_after"]}
        if kind == "append":
            Ops.paged_kv_append_f8(t["kp"], t["vp"], t["ks"], t["vs"], t["kn"], t["vn"], t["slots"])
            if case["gather"]:
                Ops.paged_kv_gather_f8(t["ko"], t["vo"], t["kp"], t["vp"], t["ks"], t["vs"], t["table"], t["cu"])
        elif kind == "decode":
            Ops.paged_attention_f8(t["out"], t["q"], t["kp"], t["vp"], t["ks"], t["vs"], t["table"], t["ctx"], SCALE)
            return s["out"]
        elif kind == "mixed":
            Ops.paged_attention_varlen_f8(t["out"], t["q"], t["kp"], t["vp"], t["ks"], t["vs"], t["table"], t["cu"],
                                          t["ctx"], SCALE)
            return s["out"]
        else:
            Ops.quantize_rows(t["xq"], t["xs"], t["x"])
            Ops.linear_i8(t["y"], t["xq"], t["xs"], t["wq"], t["ws"], t.get("bias"))
            return {"y": s["y"], "scale": s["xs"]}
    elif kind == "map":
        return _plain_map(s)
    elif kind == "append":
        _plain_append_one(s["kp"], s["ks"], s["kn"], s["slots"], False)
        _plain_append_one(s["vp"], s["vs"], s["vn"], s["slots"], True)
        if case["gather"]:
            s["ko"] = _plain_gather(s, s["kp"], s["ks"], False)
            s["vo"] = _plain_gather(s, s["vp"], s["vs"], True)
    elif kind == "decode":
        _plain_attention(s, None, 1, s["out"])
        return s["out"]
    elif kind == "mixed":
        for ids, longest in zip(s["groups"], s["longest"]):
            _plain_attention(s, ids, longest, s["out"])
        return s["out"]
    else:
        return _plain_linear(s)
    # an append's outputs: the cache, as 8-bit floats with their scales, and the rows read back
    out = {"k": s["kp"], "v": s["vp"], "k_scale": s["ks"], "v_scale": s["vs"]}
    if case["gather"]:
        out.update(k_rows=s["ko"], v_rows=s["vo"])
    return out


# --------------------------------------------------------------------- work

def work(case):
    kind = case["kind"]
    if kind == "map":
        ctx, new = _map_shape(case, None)
        fresh = sum(_pages(c + n) - _pages(c) for c, n in zip(ctx, new))
        return {"bytes": len(ctx) * 16 + fresh * 8 + (sum(new) + case["pad"]) * 16, "flops": 0}
    if kind == "append":
        ctx, new = _append_shape(case, None)
        T, row = sum(new), case["nkvh"] * HEAD
        total = {"bytes": T * (row * 2 * 3 + 8), "flops": 0}
        if case["gather"]:
            total["bytes"] += (sum(ctx) + T) * row * 2 * 3
        return total
    if kind in ("decode", "mixed"):
        if kind == "mixed":
            q, ctx = _mixed_shape(case, None)
        else:
            ctx = _spread(case["ctx_lo"], case["ctx_hi"], case["batch"])
            q = [1] * len(ctx)
        pairs = sum(n * c - n * (n - 1) // 2 for n, c in zip(q, ctx))
        pages = sum(_pages(c) for c in ctx)
        return {"bytes": sum(ctx) * case["nkvh"] * HEAD * 2 + pages * (4 + case["nkvh"] * 8)
                + sum(q) * case["nh"] * HEAD * (2 + _BYTES[case.get("out", "bf16")]),
                "flops": 4.0 * pairs * case["nh"] * HEAD}
    m, n, k = case["m"], case["n"], case["k"]
    return {"bytes": m * k * _BYTES[case["x"]] + n * k + m * n * _BYTES[case["y"]] + 4 * (m + n), "flops": 2.0 * m * n * k}


# -------------------------------------------------------------------- exact

def _values64(codes, scale, is_v):
    """The cache's values in 64 bits, [blocks, nkvh, 16, 128] by token and dim."""
    flat = codes.double().view(codes.shape[0], codes.shape[1], -1)
    return flat[..., _places(is_v)] * scale.double()[..., None, None]


def _e4m3_64(y):
    """y rounded to the nearest e4m3 value (ties to even), in 64 bits; |y| <= 448."""
    step = torch.exp2((torch.frexp(y)[1] - 1).clamp(min=-6).double() - 3)
    return torch.round(y / step) * step


def _append64(codes, scale, rows, ctx, new, table, is_v):
    values = _values64(codes, scale, is_v)
    scale = scale.double().clone()
    at = 0
    for b, (c, n) in enumerate(zip(ctx, new)):
        for p in range(c // PAGE, (c + n - 1) // PAGE + 1):
            lo, hi = max(c, p * PAGE), min(c + n, (p + 1) * PAGE)
            block, add = int(table[b, p]), rows[at + lo - c:at + hi - c].double().transpose(0, 1)
            wide = add.abs().amax((1, 2)) / 448
            need = torch.exp2(torch.ceil(torch.log2(wide)))  # wide is a power of two or 2^-8 from one at least
            need = torch.where(need / 2 >= wide, need / 2, torch.where(need < wide, need * 2, need))
            need = need.clamp(min=2.0 ** LEAST)
            if lo > p * PAGE:
                need = torch.maximum(need, scale[block])
                old = values[block]
                values[block] = torch.where((need > scale[block])[:, None, None],
                                            _e4m3_64(old / need[:, None, None]) * need[:, None, None], old)
            scale_was, scale[block] = scale[block].clone(), need
            if lo == p * PAGE:  # slots past the new rows keep their codes, whatever those now stand for
                values[block] *= (need / scale_was)[:, None, None]
            values[block, :, lo - p * PAGE:hi - p * PAGE] = _e4m3_64(add / need[:, None, None]) * need[:, None, None]
        at += n
    return values, scale


def _codes64(values, scale, is_v):
    """The codes' values in page order."""
    flat = torch.empty(values.shape[0], values.shape[1], PAGE * HEAD, dtype=torch.float64, device=values.device)
    flat[..., _places(is_v)] = values / scale[..., None, None]
    return flat.view(values.shape)


def exact(case, seed):
    kind = case["kind"]
    d64 = torch.float64
    if kind == "map":
        return None  # whole numbers
    if kind == "append":
        ctx, new, table, blocks = _append_table(case, seed)
        g = _gen(seed, 1)
        k, v = _cache(g, blocks, case["nkvh"], False), _cache(g, blocks, case["nkvh"], True)
        kn, vn = _append_rows(case, seed, sum(new))
        kv, ks = _append64(*k, kn, ctx, new, table, False)
        vv, vs = _append64(*v, vn, ctx, new, table, True)
        out = {"k": _codes64(kv, ks, False), "v": _codes64(vv, vs, True), "k_scale": ks, "v_scale": vs}
        if case["gather"]:
            for name, x in (("k_rows", kv), ("v_rows", vv)):
                out[name] = torch.cat([x[torch.from_numpy(table[b, :_pages(c + n)]).cuda().long()].transpose(1, 2)
                                       .reshape(-1, case["nkvh"], HEAD)[:c + n] for b, (c, n) in enumerate(zip(ctx, new))])
        return out
    if kind in ("decode", "mixed"):
        qn, lens, table, k, v, q = _attention_inputs(case, seed)
        kv, vv = _values64(*k, False), _values64(*v, True)
        out, r = torch.empty(q.shape, dtype=d64, device=q.device), 0
        for b, (n, c) in enumerate(zip(qn, lens)):
            at = table[b, :_pages(c)].long()
            keys = kv[at].transpose(1, 2).reshape(-1, case["nkvh"], HEAD)[:c]
            vals = vv[at].transpose(1, 2).reshape(-1, case["nkvh"], HEAD)[:c]
            see = torch.arange(c, device=q.device)[None, :] <= torch.arange(c - n, c, device=q.device)[:, None]
            for h in range(case["nkvh"]):
                heads = slice(h * (case["nh"] // case["nkvh"]), (h + 1) * (case["nh"] // case["nkvh"]))
                a = torch.matmul(q[r:r + n, heads].to(d64).transpose(0, 1), keys[:, h].t().contiguous()) * SCALE
                a = torch.softmax(a.masked_fill(~see, -math.inf), dim=-1)
                out[r:r + n, heads] = torch.matmul(a, vals[:, h].contiguous()).transpose(0, 1)
            r += n
        return out
    x, wq, ws, bias = _linear_inputs(case, seed)
    x = x.to(d64)
    xs = (x.abs().amax(1) / 127).float().to(d64)  # the scale is a 32-bit number; the codes are multiples of it
    y = torch.round(x / torch.where(xs > 0, xs, 1.0)[:, None]).clamp(-127, 127)
    y = torch.matmul(y, wq.to(d64).t()) * xs[:, None] * ws.to(d64)[None, :]
    return {"y": y if bias is None else y + bias.to(d64), "scale": xs}
