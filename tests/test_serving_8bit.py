"""The 8-bit serving operators as a layer of a served model calls them: prompts
and single tokens through quantised projections, a step's tables built on the
device, the 8-bit cache, attention over it, and the output projection. Each
stage is compared with its 64-bit form on what the stage before it gave, and the
cache with a cache that the host kept; then the same on another stream and
captured into a graph."""
import contextlib
import threading
from types import SimpleNamespace

import numpy as np
import pytest
import torch

import llaisys_amd as L
from cases_8bit import DEVICES, Cache, bf16, f64, give, map_plain, take
from test_attention_f8 import SCALE, check, want_of
from test_linear_i8 import quantize64

NH, NKVH, D, HIDDEN = 6, 2, 128, 200
WIDTH, BLOCKS = 12, 40


class Layer:
    def __init__(self, device, seed):
        r = np.random.RandomState(seed)
        self.device = device
        self.w = {}
        for name, n, k in (("q", NH * D, HIDDEN), ("k", NKVH * D, HIDDEN), ("v", NKVH * D, HIDDEN), ("o", HIDDEN, NH * D)):
            w = give(bf16(r.randn(n, k) * k ** -0.5), device)
            codes, scale = self.i8(n, k), self.f32(n)
            L.Ops.quantize_rows(codes, scale, w)
            bias = None if name == "o" else give(bf16(r.randn(n) * 0.1), device)
            self.w[name] = (codes, scale, bias)

    def i8(self, *shape):
        return give(torch.zeros(shape, dtype=torch.int8), self.device)

    def f32(self, *shape):
        return give(torch.zeros(shape), self.device)

    def b16(self, *shape):
        return give(torch.zeros(shape, dtype=torch.bfloat16), self.device)

    def i32(self, a):
        return give(np.asarray(a, np.int32), self.device)

    def state(self, B, width=WIDTH):
        """An empty cache and the tables of B sequences."""
        host = Cache(BLOCKS, NKVH, 1)
        free = np.random.RandomState(B).permutation(BLOCKS).astype(np.int32)
        return dict(host=host, pools=host.device(self.device), free_host=free, free=self.i32(free), used=self.i32([0]),
                    table=self.i32(np.full((B, width), -1)), ctx=self.i32(np.zeros(B)))

    def step(self, B, T):
        """Buffers of a step of T rows."""
        return dict(T=T, x=self.b16(T, HIDDEN), new=self.i32(np.zeros(B)), cu=self.i32(np.zeros(B + 1)),
                    pos=give(np.zeros(T, np.int64), self.device), slots=give(np.zeros(T, np.int64), self.device),
                    xq=self.i8(T, HIDDEN), xs=self.f32(T), oq=self.i8(T, NH * D), os=self.f32(T), y=self.b16(T, HIDDEN),
                    **{n: self.b16(T, h, D) for n, h in (("q", NH), ("k", NKVH), ("v", NKVH), ("qr", NH), ("kr", NKVH), ("a", NH))})

    def run(self, state, s):
        T = s["T"]
        L.Ops.paged_kv_map(state["table"], s["cu"], state["ctx"], s["pos"], s["slots"], state["ctx"], s["new"],
                           state["free"], state["used"], state["used"])
        L.Ops.quantize_rows(s["xq"], s["xs"], s["x"])
        for n, h in (("q", NH), ("k", NKVH), ("v", NKVH)):
            L.Ops.linear_i8(s[n].view(T, h * D), s["xq"], s["xs"], *self.w[n])
        L.Ops.rope(s["qr"], s["q"], s["pos"], 10000.0)
        L.Ops.rope(s["kr"], s["k"], s["pos"], 10000.0)
        L.Ops.paged_kv_append_f8(*state["pools"], s["kr"], s["v"], s["slots"])
        if T == state["ctx"].shape()[0]:
            L.Ops.paged_attention_f8(s["a"], s["qr"], *state["pools"], state["table"], state["ctx"], SCALE)
        else:
            L.Ops.paged_attention_varlen_f8(s["a"], s["qr"], *state["pools"], state["table"], s["cu"], state["ctx"], SCALE)
        L.Ops.quantize_rows(s["oq"], s["os"], s["a"].view(T, NH * D))
        L.Ops.linear_i8(s["y"], s["oq"], s["os"], *self.w["o"])

    def check_linear(self, got, codes, scale, name):
        w, ws, bias = self.w[name]
        dot = (take(codes).double() @ take(w).double().t()) * take(scale).double()[:, None] * take(ws).double()
        want = dot if bias is None else dot + take(bias).double()
        bound = 3 * 2.0 ** -24 * dot.abs() + (2.0 ** -24 + 1.01 * 2.0 ** -8) * want.abs() + 2.0 ** -140
        assert ((take(got).double().reshape(want.shape) - want).abs() <= bound).all(), name

    def check_step(self, state, s, before, new):
        """`before`: the table, lengths and used blocks that the step began with (host)."""
        table, ctx, used = before
        want = map_plain(table, ctx, new, s["T"], state["free_host"], used)
        got = [take(state["table"]), take(s["cu"]), take(state["ctx"]), take(s["pos"]), take(s["slots"])]
        for g, w in zip(got, want):
            np.testing.assert_array_equal(g.numpy(), w)
        table, cu, ctx, pos, slots, used, flags = want
        assert int(take(state["used"])[0]) == used and flags == 0 and L.device_error_flags() == 0
        for x, codes, scale in ((take(s["x"]), "xq", "xs"), (take(s["a"]).reshape(s["T"], -1), "oq", "os")):
            wq, wscale = quantize64(x)
            np.testing.assert_array_equal(take(s[codes]).numpy(), wq)
            np.testing.assert_array_equal(take(s[scale]).numpy(), wscale)
        for n in "qkv":
            self.check_linear(s[n], s["xq"], s["xs"], n)
        self.check_linear(s["y"], s["oq"], s["os"], "o")
        state["host"].append(f64(take(s["kr"])), f64(take(s["v"])), slots)
        state["host"].check(*state["pools"])
        rows = int(cu[-1])
        o, most = want_of(state["host"], table, ctx, new, take(s["qr"])[:rows])
        host, held = state["host"], np.unique(table[table >= 0])
        seen = SimpleNamespace(values=lambda which: host.values(which)[held])  # (what no table holds is larger)
        check(take(s["a"])[:rows], o, most, seen, torch.bfloat16, int(ctx.max()), s["T"] != len(new))
        return table, ctx, used


def fill(t, values):
    src = give(values, "cpu")
    cpu = t.device_type() == L.DeviceType.CPU
    L.RuntimeAPI(t.device_type()).memcpy_sync(t.data_ptr(), src.data_ptr(), values.nbytes,
                                              L.MemcpyKind.H2H if cpu else L.MemcpyKind.H2D)


def begin(B, width=WIDTH):
    return np.full((B, width), -1, np.int32), np.zeros(B, np.int32), 0


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("steps", [
    [[5, 33, 16], [1, 1, 1], [1, 1, 1], [20, 1, 0], [1, 1, 1]],
    [[1], [1], [30], [1], [1]],
    [[0, 100, 1, 17], [64, 1, 1, 1]] + [[1] * 4] * 3,
])
def test_steps_of_a_layer(device, steps):
    B = len(steps[0])
    layer = Layer(device, 3)
    state, before = layer.state(B), begin(B)
    for i, new in enumerate(steps):
        s = layer.step(B, max(sum(new), 1))
        fill(s["x"], bf16(np.random.RandomState(i).randn(s["T"], HIDDEN)))
        fill(s["new"], torch.tensor(new, dtype=torch.int32))
        layer.run(state, s)
        before = layer.check_step(state, s, before, new)


@contextlib.contextmanager
def on_stream(stream):
    L.set_context_stream(stream.cuda_stream)
    try:
        yield
    finally:
        L.set_context_stream(0)


@pytest.mark.gpu
def test_steps_on_another_stream():
    """The first step fills the stream with work, so that a kernel on any other one would run before it."""
    layer = Layer("amd", 5)
    state, before = layer.state(3), begin(3)
    stream = torch.cuda.Stream()
    busy = torch.zeros(64 << 20, device="cuda")
    for i, new in enumerate(([40, 1, 7], [1, 1, 1], [1, 30, 2])):
        s = layer.step(3, sum(new))
        fill(s["x"], bf16(np.random.RandomState(i).randn(s["T"], HIDDEN)))
        fill(s["new"], torch.tensor(new, dtype=torch.int32))
        torch.cuda.synchronize()
        with on_stream(stream):
            with torch.cuda.stream(stream):
                for _ in range(20):
                    busy.add_(1)
            layer.run(state, s)
            stream.synchronize()
            before = layer.check_step(state, s, before, new)


@pytest.mark.gpu
@pytest.mark.parametrize("rows, width", [(5, WIDTH), (9, WIDTH), (9, 600)])
def test_captured_steps_replayed(rows, width):
    """A step of five sequences in `rows` rows, captured once and replayed with
    other inputs, lengths and row counts each time, as the sequences grow past
    several pages, with eager steps of another size in between. Two layers'
    graphs share the thread's workspace in turn."""
    B = 5
    stream = torch.cuda.Stream()
    runs = []
    for i in range(2):
        layer = Layer("amd", 7 + i)
        state = layer.state(B, width)
        runs.append([layer, state, layer.step(B, rows), begin(B, width), torch.cuda.CUDAGraph(), layer.step(B, 40)])

    def step(run, which, seed, new, go):
        layer, state, _, before, _, _ = run
        s = run[which]
        fill(s["x"], bf16(np.random.RandomState(seed).randn(s["T"], HIDDEN)))
        fill(s["new"], torch.tensor(new, dtype=torch.int32))
        go(state, s)
        torch.cuda.synchronize()
        run[3] = layer.check_step(state, s, before, new)

    for i, run in enumerate(runs):
        step(run, 5, i, [20, 1, 3, 7, 9], run[0].run)
        step(run, 2, i + 10, [1] * B, run[0].run)  # eager: the workspaces have their sizes now
    for layer, state, s, _, graph, _ in runs:
        with on_stream(stream), torch.cuda.graph(graph, stream=stream):
            layer.run(state, s)
    r = np.random.RandomState(rows)
    for i in range(16):
        for run in runs:
            if i % 5 == 4:
                step(run, 5, 100 + i, [3, 0, 1, 9, 1], run[0].run)
            else:
                new = [1] * B
                if rows > B:
                    new[r.randint(B)] += r.randint(rows - B + 1)
                    new[r.randint(B)] = 0
                step(run, 2, 100 + i, new, lambda state, s: run[4].replay())


@pytest.mark.gpu
def test_steps_on_two_threads_at_once():
    """Each thread has a runtime, a stream and a workspace of its own."""
    def serve(seed, failures):
        try:
            layer = Layer("amd", seed)
            for turn in range(4):
                state, before = layer.state(4, 600 if turn % 2 else WIDTH), begin(4, 600 if turn % 2 else WIDTH)
                for i, new in enumerate(([40, 1, 7, 20], [1, 1, 1, 1], [1, 30, 2, 1], [1, 1, 1, 1])):
                    s = layer.step(4, sum(new))
                    fill(s["x"], bf16(np.random.RandomState(seed + i).randn(s["T"], HIDDEN)))
                    fill(s["new"], torch.tensor(new, dtype=torch.int32))
                    layer.run(state, s)
                    before = layer.check_step(state, s, before, new)
        except BaseException as e:  # noqa: BLE001 (reported by the test's own thread)
            failures.append(e)

    failures = []
    threads = [threading.Thread(target=serve, args=(seed, failures)) for seed in (51, 52)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures, failures
