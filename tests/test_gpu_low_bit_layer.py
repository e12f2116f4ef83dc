"""A decoder layer on 4-bit weights and the 8-bit paged cache, as a server would run it: ragged prompts, then steps of
the whole batch, eagerly and from a recorded graph.  Every call's result is checked against 64 bits on the inputs that
the device had (the calls before it), so each is held to the bound of its own roundings."""
from __future__ import annotations

import numpy as np
import pytest

import low_bit_reference as ref
from test_gpu_q4 import product

pytestmark = pytest.mark.gpu
THETA, EPS = 1e6, 1e-5


class Layer:
    def __init__(self, mmr, hidden, hq, hkv, d, ffn, group, rows, rng):
        self.mmr, self.hidden, self.hq, self.hkv, self.d, self.group = mmr, hidden, hq, hkv, d, group
        self.shapes = {"qkv": ((hq + 2 * hkv) * d, hidden), "o": (hidden, hq * d), "gate_up": (2 * ffn, hidden),
                       "down": (hidden, ffn)}
        self.w, self.device, self.exact = {}, {}, {}
        for name, (r, c) in self.shapes.items():
            codes, scales = mmr.q4_quantize((rng.standard_normal((r, c)) / np.sqrt(c)).astype(np.float32), group)
            self.exact[name] = ref.q4_weights(codes, scales, c, group)
            self.device[name] = mmr.DeviceArray.from_numpy(codes), mmr.DeviceArray.from_numpy(scales)
        self.norms = {n: (1 + 0.1 * rng.standard_normal(size)).astype(np.float32)
                      for n, size in (("input", hidden), ("post", hidden), ("q", d), ("k", d))}
        self.dnorms = {n: mmr.DeviceArray.from_numpy(v) for n, v in self.norms.items()}
        self.rope = mmr.RopeTable(4096, d, THETA)
        sizes = {"qkv": self.shapes["qkv"][0], "query": hq * d, "attended": hq * d, "mid": hidden, "act": ffn,
                 "out": hidden, "hidden": hidden}
        self.b = {n: mmr.DeviceArray((rows, s), np.float32) for n, s in sizes.items()}
        most = max(mmr.matvec_q4_workspace_size(c, rows) for _, c in self.shapes.values())
        self.b["workspace"] = mmr.DeviceArray(max(most, 1), np.uint8)
        self.error = mmr.DeviceArray.from_numpy(np.zeros(1, np.int32))

    def matvec(self, name, x, y, rows, stream, **more):
        self.mmr.matvec_q4(*self.device[name], self.group, *self.shapes[name], self.b[x], rows, self.b[y], eps=EPS,
                           workspace=self.b["workspace"], stream=stream, **more)

    def run(self, pages, offsets, context, rows, max_rows, max_tokens, attention_workspace, stream=None):
        m, b = self.mmr, self.b
        self.matvec("qkv", "hidden", "qkv", rows, stream, norm_w=self.dnorms["input"], prologue=m.PRO_RMSNORM)
        m.kv8_append(b["qkv"], self.dnorms["q"], self.dnorms["k"], EPS, self.rope, pages, offsets, context, rows,
                     max_rows, self.hq, b["query"], self.error, stream=stream)
        m.kv8_attention(b["query"], pages, offsets, context, rows, max_rows, max_tokens, self.hq, b["attended"],
                        attention_workspace, self.error, stream=stream)
        self.matvec("o", "attended", "mid", rows, stream, residual=b["hidden"], epilogue=m.EPI_RESIDUAL)
        self.matvec("gate_up", "mid", "act", rows, stream, norm_w=self.dnorms["post"], prologue=m.PRO_RMSNORM,
                    epilogue=m.EPI_SWIGLU)
        self.matvec("down", "act", "out", rows, stream, residual=b["mid"], epilogue=m.EPI_RESIDUAL)

    def check(self, cache, pages, offsets, context, rows):
        m = self.mmr
        got = {n: self.b[n].numpy()[:rows] for n in ("hidden", "qkv", "query", "attended", "mid", "act", "out")}
        for name, x, y, norm, epilogue, residual in (
                ("qkv", "hidden", "qkv", "input", m.EPI_STORE, None), ("o", "attended", "mid", None, m.EPI_RESIDUAL, "hidden"),
                ("gate_up", "mid", "act", "post", m.EPI_SWIGLU, None), ("down", "act", "out", None, m.EPI_RESIDUAL, "mid")):
            want, off = product(self.exact[name], got[x], self.norms.get(norm), int(norm is not None), EPS, epilogue,
                                got.get(residual), m)
            assert (np.abs(got[y] - want) <= off).all(), name
        want = ref.append(cache, got["qkv"], offsets, context, self.hq, THETA, self.norms["q"], self.norms["k"], EPS,
                          got["query"])
        cache.assert_equals(pages)
        assert (np.abs(got["query"] - want) <= 2.0 ** -24 * np.abs(want) + 1e-12).all()
        want, bound = ref.attention(cache, got["query"], offsets, context, self.hq, got["attended"])
        assert (np.abs(got["attended"] - want) <= bound).all()
        assert int(self.error.numpy()[0]) == 0


@pytest.mark.parametrize("shape,group", [((256, 4, 2, 64, 512), 32), ((768, 8, 2, 96, 2048), 64), ((512, 8, 2, 64, 1408), 128)])
def test_prompts_and_steps(gpu, shape, group):
    mmr, rng = gpu, np.random.default_rng(shape[0])
    hidden, hq, hkv, d, ffn = shape
    prompts, per = [70, 1, 33], 3
    seqs, total = len(prompts), sum(prompts)
    layer = Layer(mmr, hidden, hq, hkv, d, ffn, group, total, rng)
    cache = ref.Cache(rng, seqs * per + 1, seqs, per, hkv, d)
    pages = cache.upload(mmr)
    most = per * ref.PAGE

    def workspace(rows, max_rows):
        size = mmr.kv8_attention_workspace_size(hq, hkv, d, seqs, rows, max_rows, most)
        return mmr.DeviceArray(max(size, 1), np.uint8)

    def ints(values):
        return mmr.DeviceArray.from_numpy(np.asarray(values, np.int32))

    offsets = np.concatenate([[0], np.cumsum(prompts)])
    layer.b["hidden"].upload(rng.standard_normal((total, hidden)).astype(np.float32))
    ws = workspace(total, max(prompts))
    layer.run(pages, ints(offsets), ints([0] * seqs), total, max(prompts), most, ws)
    mmr.synchronize()
    layer.check(cache, pages, offsets, [0] * seqs, total)

    # Steps: the first eagerly, the others from one graph that follows the device arrays.
    stream, step_ws = mmr.Stream(), workspace(seqs, 1)
    d_offsets, d_context = ints(np.arange(seqs + 1)), ints([0] * seqs)

    def step():
        layer.run(pages, d_offsets, d_context, seqs, 1, most, step_ws, stream)

    with mmr.Graph(stream) as graph:
        step()
    for i in range(6):
        context = [n + i for n in prompts]
        x = np.zeros((total, hidden), np.float32)
        x[:seqs] = rng.standard_normal((seqs, hidden))
        layer.b["hidden"].upload(x)
        d_context.upload(np.asarray(context, np.int32))
        if i == 0:
            step()
        else:
            graph.launch()
        mmr.synchronize()
        layer.check(cache, pages, np.arange(seqs + 1), context, seqs)


def test_graphs_on_one_workspace(gpu):
    """Three recorded calls that share a workspace, replayed in changing order on their stream with eager calls between:
    nothing is kept in it from one call to the next."""
    mmr, rng = gpu, np.random.default_rng(61)
    hq, hkv, d, per = 8, 2, 96, 40
    cache = ref.Cache(rng, 3 * per, 3, per, hkv, d)
    cache.fill(rng, [2500, 700, 130])
    pages, stream = cache.upload(mmr), mmr.Stream()

    def upload(a):
        return mmr.DeviceArray.from_numpy(a)

    def attention(rows, context):
        n, most = sum(rows), max(rows)
        offsets = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
        q, out = upload(rng.standard_normal((n, hq * d)).astype(np.float32)), mmr.DeviceArray((n, hq * d), np.float32)
        arrays = upload(offsets), upload(np.asarray(context, np.int32)), upload(np.zeros(1, np.int32))
        size = mmr.kv8_attention_workspace_size(hq, hkv, d, 3, n, most, per * ref.PAGE)
        return size, out, lambda ws, s: mmr.kv8_attention(q, pages, *arrays[:2], n, most, per * ref.PAGE, hq, out, ws,
                                                          arrays[2], stream=s)

    def matvec(rows, cols, batch):
        codes, scales = mmr.q4_quantize(rng.standard_normal((rows, cols)).astype(np.float32), 32)
        w, x = (upload(codes), upload(scales)), upload(rng.standard_normal((batch, cols)).astype(np.float32))
        y = mmr.DeviceArray((batch, rows), np.float32)
        return mmr.matvec_q4_workspace_size(cols, batch), y, lambda ws, s: mmr.matvec_q4(
            *w, 32, rows, cols, x, batch, y, workspace=ws, stream=s)

    calls = [attention([1, 1, 1], [2499, 699, 129]), attention([30, 40, 20], [2470, 660, 110]), matvec(300, 768, 40)]
    workspace = mmr.DeviceArray(max(c[0] for c in calls), np.uint8)
    assert min(c[0] for c in calls) > 0
    mmr.synchronize()
    want, graphs = [], []
    for size, out, call in calls:
        call(workspace, stream)
        mmr.synchronize()
        want.append(out.numpy())
        with mmr.Graph(stream) as graph:
            call(workspace, stream)
        graphs.append(graph)
    for order in ([0, 1, 2], [2, 1, 0], [1, 1, 0, 2], [0, 2, 0, 1], [2, 0, 1]):
        for _, out, _ in calls:
            out.zero()
        workspace.upload(np.full(workspace.shape, 0xFF, np.uint8))
        mmr.synchronize()
        for i in order:
            graphs[i].launch(stream)
        calls[order[0]][2](workspace, stream)
        mmr.synchronize()
        for (_, out, _), a in zip(calls, want):
            np.testing.assert_array_equal(out.numpy(), a)
