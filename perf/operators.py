"""Operators of decoding on 4-bit weights and an 8-bit paged cache.

What a decode step reads, in the bits that it is kept in: projections whose
weights are 4-bit codes under a scale per group of columns, and attention over a
paged cache of 8-bit codes under a power-of-two scale per block of 16 tokens and
head, with the call that appends a step's (or a prompt's) rows to that cache,
normalised and rotated on the way.

Where `own` is false the operators are computed in elementary torch operations,
where it is true by the framework's calls.
"""
from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

DEVICE = "cuda"
EPS = 1e-5
THETA = 1e6
POSITIONS = 32768  # of the rotation table
PAGE, BLOCK = 64, 16  # tokens of a page, and of a block under one exponent
LOW, HIGH = -126, 122  # exponents
VOCAB = 6400

#: hidden, query heads, KV heads, head dimension, FFN width
SHAPES = {
    "minimind2": (768, 8, 2, 96, 2048),
    "minimind2-small": (512, 8, 2, 64, 1408),
}


def listed():
    return [
        # One layer's new token of one chat: the smallest call, all latency.
        dict(name="append_step", kind="append", seqs=1, rows=1, context=777, q_heads=8, kv_heads=2, head_dim=96),
        # One step of a batch of sequences at their own positions.
        dict(name="append_batch", kind="append", seqs=32, rows=1, context=4095, q_heads=8, kv_heads=2, head_dim=96),
        # Ragged prompts of a batch, after what earlier calls cached.
        dict(name="append_prompts", kind="append", seqs=5, rows=1000, context=1111, q_heads=8, kv_heads=2,
             head_dim=128),
        # One query in the middle of a chat: the smallest attention call.
        dict(name="attention_step", kind="attention", seqs=1, rows=1, context=777, q_heads=8, kv_heads=2,
             head_dim=96),
        # One query at the end of the longest context.
        dict(name="attention_long", kind="attention", seqs=1, rows=1, context=32767, q_heads=8, kv_heads=2,
             head_dim=96),
        # A step of a batch deep into its contexts: the cache is what is read.
        dict(name="attention_batch", kind="attention", seqs=32, rows=1, context=8191, q_heads=8, kv_heads=2,
             head_dim=96),
        # Several rows a sequence (drafted tokens to check), of the small model's heads.
        dict(name="attention_rows", kind="attention", seqs=16, rows=5, context=2500, q_heads=8, kv_heads=2,
             head_dim=64),
        # A long prompt's later part, after the rows that an earlier call cached.
        dict(name="attention_prompt", kind="attention", seqs=1, rows=3000, context=1111, q_heads=8, kv_heads=2,
             head_dim=96),
        # The fused norm and QKV projection of one token.
        dict(name="matvec_qkv", kind="matvec", rows=1152, cols=768, group=32, batch=1, form="norm"),
        # Gate and up rows with SwiGLU for a batch of sequences.
        dict(name="matvec_gate_up_batch", kind="matvec", rows=4096, cols=768, group=64, batch=32, form="swiglu"),
        # Down projection and residual of the small model, three rows, ragged columns.
        dict(name="matvec_down_rows", kind="matvec", rows=512, cols=1408, group=32, batch=3, form="residual"),
        # A matrix too large for the caches near the compute units, one token.
        dict(name="matvec_large", kind="matvec", rows=32768, cols=4096, group=128, batch=1, form="plain"),
    ]


def _between(rng, low, high):
    """A whole number in [low, high], even over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["append", "attention", "attention", "matvec", "matvec"])
    if kind == "matvec":
        model = rng.choice(sorted(SHAPES))
        hidden, hq, hkv, d, ffn = SHAPES[model]
        rows, cols, form = rng.choice([((hq + 2 * hkv) * d, hidden, "norm"), (hidden, hq * d, "residual"),
                                       (2 * ffn, hidden, "swiglu"), (hidden, ffn, "residual"),
                                       (_between(rng, 100, 20000), 32 * _between(rng, 4, 128), "plain")])
        return dict(kind=kind, rows=rows, cols=cols, group=rng.choice([32, 64, 128]),
                    batch=rng.choice([1, 1, 2, 3, 4, _between(rng, 5, 48)]), form=form)
    q_heads, kv_heads = rng.choice([(8, 2), (8, 2), (4, 4), (8, 1), (12, 4)])
    d = rng.choice([64, 96, 128])
    what = rng.choice(["step", "rows", "prompt"])
    if what == "step":
        seqs = _between(rng, 1, 48)
        context = _between(rng, 5, min(32767, 262144 // seqs))
        rows = 1
    elif what == "rows":
        seqs, rows = _between(rng, 1, 24), rng.randrange(2, 9)
        context = _between(rng, 5, min(32000, 65536 // seqs))
    else:
        seqs = rng.choice([1, 1, 2, 5])
        rows = _between(rng, 12, 2400 // seqs)
        context = rng.choice([0, rng.randrange(1200)])
    return dict(kind=kind, seqs=seqs, rows=rows, context=context, q_heads=q_heads, kv_heads=kv_heads, head_dim=d)


# ---------------------------------------------------------------- inputs ----


class Buffer:
    """Device memory of a torch tensor in the shape that mmr's calls take."""

    def __init__(self, tensor):
        self.tensor = tensor
        self.ptr = tensor.data_ptr()
        self.nbytes = tensor.numel() * tensor.element_size()


def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(int(seed))


def _normal(g, shape, std=1.0):
    return torch.randn(shape, generator=g, device=DEVICE, dtype=torch.float32) * std


def _mmr():
    folder = str(Path("minimind-orangepi_amd").resolve())
    if folder not in sys.path:
        sys.path.insert(0, folder)
    import mmr

    return mmr


def _lengths(case):
    """Rows and contexts of each sequence: the first as the case says, the others ragged down to a quarter; of four
    or more sequences with several rows each, one brings none."""
    rows, context = [case["rows"]], [case["context"]]
    state = 12345
    for s in range(1, case["seqs"]):
        state = (state * 1103515245 + 12345) % 2**31
        part = 0.25 + 0.75 * (state / 2**31)
        rows.append(0 if s == 3 and case["rows"] > 1 else max(1, round(case["rows"] * part)))
        context.append(round(case["context"] * (0.25 + 0.75 * ((state // 7) % 1000) / 1000)))
    return rows, context


def _ints(values):
    return torch.tensor(values, device=DEVICE, dtype=torch.int32)


def _exponent(top):
    """The least e with top <= 127 * 2^e, in [LOW, HIGH]."""
    m, x = torch.frexp(top)
    return torch.where(top > 0, x - 7 + (m > 127 / 128).int(), LOW).clamp(LOW, HIGH)


def _scaled(x, e):
    """x * 2^e, exact where it is a normal number."""
    return torch.ldexp(x, e)


def _cache(g, case, rows, context):
    """Pages in any order, full of cached tokens of several sizes, and a table of each sequence's pages."""
    h, d = case["kv_heads"], case["head_dim"]
    per = max(-(-(n + c) // PAGE) for n, c in zip(rows, context))
    pages = per * len(rows) + 3
    table = torch.randperm(pages, generator=g, device=DEVICE)[: per * len(rows)].reshape(len(rows), per).int()
    parts = {}
    for name, std in (("key", 1.0), ("value", 0.6)):
        x = _normal(g, (pages, h, PAGE, d), std) * torch.exp(_normal(g, (pages, h, PAGE, 1), 0.3))
        e = _exponent(x.reshape(pages, h, PAGE // BLOCK, -1).abs().amax(-1))
        x = _scaled(x, -e.repeat_interleave(BLOCK, -1)[..., None]).round().to(torch.int8)
        parts[name + "s"] = (x if name == "key" else x.transpose(-1, -2)).contiguous()
        parts[name + "_exps"] = e.to(torch.int8)
    return {"table": table, **parts}


# --------------------------------------------------------------- prepare ----


def prepare(case, seed):
    state = {"case": case, **_PREPARE[case["kind"]](case, _generator(seed))}
    if own:  # the handles that a program keeps
        state["mmr"] = _mmr()
        state["buffer"] = {n: Buffer(t) for n, t in state.items() if isinstance(t, torch.Tensor)}
        _KEEP[case["kind"]](state, state["mmr"], state["buffer"])
    return state


def _prepare_append(case, g):
    rows, context = _lengths(case)
    hq, h, d = case["q_heads"], case["kv_heads"], case["head_dim"]
    n = sum(rows)
    return dict(_cache(g, case, rows, context), qkv=_normal(g, (n, (hq + 2 * h) * d), 0.6),
                q_norm=1 + _normal(g, (d,), 0.1), k_norm=1 + _normal(g, (d,), 0.1),
                query=torch.zeros((n, hq * d), device=DEVICE), error=_ints([0]),
                offsets=_ints([sum(rows[:i]) for i in range(len(rows) + 1)]), context=_ints(context),
                max_rows=max(rows), max_tokens=max(a + b for a, b in zip(rows, context)))


def _prepare_attention(case, g):
    rows, context = _lengths(case)
    hq, d, n = case["q_heads"], case["head_dim"], sum(rows)
    return dict(_cache(g, case, rows, context), query=_normal(g, (n, hq * d)),
                out=torch.zeros((n, hq * d), device=DEVICE), error=_ints([0]),
                offsets=_ints([sum(rows[:i]) for i in range(len(rows) + 1)]), context=_ints(context),
                max_rows=max(rows), max_tokens=max(a + b for a, b in zip(rows, context)))


def _prepare_matvec(case, g):
    rows, cols, group, batch, form = (case[k] for k in ("rows", "cols", "group", "batch", "form"))
    wide = -(-cols // 128) * 128
    q = (_normal(g, (rows, wide)) * 2.6).round().clamp(-8, 7).to(torch.int32)
    q[:, cols:] = 0
    # Codes in two's complement: of each 128 columns, 16 four-byte words, word 4 p + j of columns 32 j + 8 p on.
    q = (q & 15).reshape(rows, wide // 128, 4, 4, 4, 2).transpose(2, 3)
    codes = (q[..., 0] | (q[..., 1] << 4)).to(torch.uint8).reshape(rows, wide // 2).contiguous()
    scales = (0.008 * torch.exp(_normal(g, (rows, -(-cols // group)), 0.3))).half()
    many = rows // 2 if form == "swiglu" else rows
    state = dict(codes=codes, scales=scales, x=_normal(g, (batch, cols)) * torch.exp(_normal(g, (cols,), 0.7)),
                 y=torch.zeros((batch, many), device=DEVICE))
    if form in ("norm", "swiglu"):
        state["norm"] = 1 + _normal(g, (cols,), 0.1)
    if form == "residual":
        state["residual"] = _normal(g, (batch, rows))
    return state


_PREPARE = {"append": _prepare_append, "attention": _prepare_attention, "matvec": _prepare_matvec}


def _keep_pages(state, mmr, b):
    c = state["case"]
    state["pages"] = mmr.Kv8Pages(b["keys"], b["values"], b["key_exps"], b["value_exps"], b["table"],
                                  state["keys"].shape[0], *state["table"].shape, c["kv_heads"], c["head_dim"])


def _keep_append(state, mmr, b):
    _keep_pages(state, mmr, b)
    state["rope"] = mmr.RopeTable(POSITIONS, state["case"]["head_dim"], THETA)


def _keep_attention(state, mmr, b):
    _keep_pages(state, mmr, b)
    c = state["case"]
    size = mmr.kv8_attention_workspace_size(c["q_heads"], c["kv_heads"], c["head_dim"], c["seqs"],
                                            state["query"].shape[0], state["max_rows"], state["max_tokens"])
    b["workspace"] = Buffer(torch.empty(max(1, size), device=DEVICE, dtype=torch.uint8))


def _keep_matvec(state, mmr, b):
    c = state["case"]
    size = mmr.matvec_q4_workspace_size(c["cols"], c["batch"])
    b["workspace"] = Buffer(torch.empty(max(1, size), device=DEVICE, dtype=torch.uint8))


_KEEP = {"append": _keep_append, "attention": _keep_attention, "matvec": _keep_matvec}


# ------------------------------------------------------------------- run ----


def run(state):
    return _RUN[state["case"]["kind"]](state)


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _run_append(s):
    if own:
        b = s["buffer"]
        s["mmr"].kv8_append(b["qkv"], b["q_norm"], b["k_norm"], EPS, s["rope"], s["pages"], b["offsets"],
                            b["context"], s["qkv"].shape[0], s["max_rows"], s["case"]["q_heads"], b["query"],
                            b["error"], stream=_stream())
    else:
        _plain_append(s)
    # A cached value is a code times a power of two, both fixed by the definition to the last bit, so the whole cache
    # is compared as the whole numbers that it holds.
    return {"query": s["query"], "error": s["error"], "keys": s["keys"], "values": s["values"],
            "key_exps": s["key_exps"], "value_exps": s["value_exps"]}


def _run_attention(s):
    if own:
        b = s["buffer"]
        s["mmr"].kv8_attention(b["query"], s["pages"], b["offsets"], b["context"], s["query"].shape[0], s["max_rows"],
                               s["max_tokens"], s["case"]["q_heads"], b["out"], b["workspace"], b["error"],
                               stream=_stream())
    else:
        _plain_attention(s)
    return {"out": s["out"], "error": s["error"]}


def _run_matvec(s):
    if own:
        c, b, m = s["case"], s["buffer"], s["mmr"]
        m.matvec_q4(b["codes"], b["scales"], c["group"], c["rows"], c["cols"], b["x"], c["batch"], b["y"],
                    norm_w=b.get("norm"), eps=EPS, prologue=m.PRO_RMSNORM if "norm" in b else m.PRO_PLAIN,
                    epilogue={"residual": m.EPI_RESIDUAL, "swiglu": m.EPI_SWIGLU}.get(c["form"], m.EPI_STORE),
                    residual=b.get("residual"), workspace=b["workspace"], stream=_stream())
        return {"y": s["y"]}
    return {"y": _plain_matvec(s)}


_RUN = {"append": _run_append, "attention": _run_attention, "matvec": _run_matvec}


# ----------------------------------------------------------- plain forms ----


def _row_places(s, n):
    """Sequence, position and index within its sequence of each of n rows."""
    r = torch.arange(n, device=DEVICE)
    seq = torch.searchsorted(s["offsets"][1:].long().contiguous(), r, right=True)
    index = r - s["offsets"][seq].long()
    return seq, s["context"][seq].long() + index, index


def _plain_append(s):
    c = s["case"]
    hq, h, d = c["q_heads"], c["kv_heads"], c["head_dim"]
    n, seqs, per = s["qkv"].shape[0], *s["table"].shape
    seq, at, _ = _row_places(s, n)
    # In 64 bits: the angles of far positions, and codes of values next to a rounding border.
    x = s["qkv"].double().reshape(n, hq + 2 * h, d)
    qk, v = x[:, : hq + h], x[:, hq + h:]
    w = torch.cat([s["q_norm"].expand(hq, d), s["k_norm"].expand(h, d)]).double()
    qk = qk * torch.rsqrt((qk * qk).mean(-1, keepdim=True) + EPS) * w
    angle = at.double()[:, None, None] * THETA ** (-torch.arange(0, d, 2, device=DEVICE, dtype=torch.float64) / d)
    cos, sin, a, b = angle.cos(), angle.sin(), qk[..., : d // 2], qk[..., d // 2:]
    qk = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    s["query"].copy_(qk[:, :hq].reshape(n, hq * d))
    page = s["table"].long()[seq, at // PAGE]
    block, slot = at % PAGE // BLOCK, at % PAGE
    head = torch.arange(h, device=DEVICE)
    # Where the new rows of a sequence begin, if that is within a block of cached ones.
    touched = (s["offsets"][1:] > s["offsets"][:-1]) & (s["context"] % BLOCK > 0)
    first = torch.where(touched, s["context"], 0).long()
    first_page = s["table"].long().gather(1, (first // PAGE)[:, None])[:, 0]
    cell = (first // BLOCK % (PAGE // BLOCK))[:, None]
    token = first[:, None] // BLOCK * BLOCK % PAGE + torch.arange(BLOCK, device=DEVICE)  # of that block
    old = touched[:, None] & (torch.arange(BLOCK, device=DEVICE) < first[:, None] % BLOCK)
    for codes, exps, new in ((s["keys"], s["key_exps"], qk[:, hq:]), (s["values"], s["value_exps"], v)):
        rows = codes if codes is s["keys"] else codes.transpose(-1, -2)
        number = seq * (per * PAGE // BLOCK) + at // BLOCK  # of the row's block
        top = torch.zeros((seqs * per * PAGE // BLOCK, h), device=DEVICE, dtype=torch.float64)
        top = top.scatter_reduce(0, number[:, None].expand(n, h), new.abs().amax(-1), "amax")
        e = _exponent(top)
        held = exps[first_page[:, None], head, cell].int()  # [seqs, h]
        at_first = torch.arange(seqs, device=DEVICE) * (per * PAGE // BLOCK) + first // BLOCK
        e[at_first] = torch.where(touched[:, None], torch.maximum(e[at_first], held), e[at_first])
        was = rows[first_page[:, None, None], head[:, None], token[:, None, :]]  # [seqs, h, BLOCK, d]
        moved = _scaled(was.double(), (held - e[at_first])[..., None, None]).round().to(torch.int8)
        rows[first_page[:, None, None], head[:, None], token[:, None, :]] = torch.where(old[:, None, :, None], moved,
                                                                                       was)
        row_e = e[number]
        rows[page[:, None], head, slot[:, None]] = _scaled(new, -row_e[..., None]).round().to(torch.int8)
        exps[page[:, None], head, block[:, None]] = row_e.to(torch.int8)


def _plain_attention(s):
    c = s["case"]
    hq, h, d = c["q_heads"], c["kv_heads"], c["head_dim"]
    n, most, (seqs, per) = s["query"].shape[0], s["max_rows"], s["table"].shape
    seq, _, index = _row_places(s, n)
    table = s["table"].long()
    k = _scaled(s["keys"][table].float(), s["key_exps"][table].int().repeat_interleave(BLOCK, -1)[..., None])
    v = _scaled(s["values"][table].float(), s["value_exps"][table].int().repeat_interleave(BLOCK, -1)[..., None, :])
    k = k.permute(0, 2, 4, 1, 3).reshape(seqs, h, d, per * PAGE)
    v = v.permute(0, 2, 1, 4, 3).reshape(seqs, h, per * PAGE, d)
    row = (s["offsets"][:-1, None].long() + torch.arange(most, device=DEVICE)).clamp(max=n - 1)
    q = s["query"][row].reshape(seqs, most, h, hq // h, d).permute(0, 2, 3, 1, 4).reshape(seqs, h, -1, d)
    score = torch.matmul(q, k) * d ** -0.5
    limit = s["context"][:, None].long() + torch.arange(most, device=DEVICE)  # a row's last key
    seen = torch.arange(per * PAGE, device=DEVICE) <= limit[..., None]
    score = score.reshape(seqs, h, hq // h, most, -1).masked_fill(~seen[:, None, None], -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True))
    o = torch.matmul(p.reshape(seqs, h, -1, per * PAGE), v).reshape(seqs, h, hq // h, most, d)
    o = o / p.sum(-1, keepdim=True)
    s["out"].copy_(o.permute(0, 3, 1, 2, 4)[seq, index].reshape(n, hq * d))


def _plain_matvec(s):
    c = s["case"]
    rows, cols, group, form = c["rows"], c["cols"], c["group"], c["form"]
    both = torch.stack([s["codes"] & 15, s["codes"] >> 4], -1).to(torch.int8)
    q = both.reshape(rows, -1, 4, 4, 8).transpose(2, 3).reshape(rows, -1)[:, :cols]
    w = ((q ^ 8) - 8).float() * s["scales"].float().repeat_interleave(group, 1)[:, :cols]
    x = s["x"]
    if "norm" in s:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * s["norm"]
    y = torch.matmul(x, w.t())
    if form == "residual":
        y = y + s["residual"]
    if form == "swiglu":
        gate, up = y[:, 0::2], y[:, 1::2]
        y = gate / (1 + torch.exp(-gate)) * up
    return y


# ------------------------------------------------------------------ work ----


def work(case):
    if case["kind"] == "matvec":
        rows, cols, batch = case["rows"], case["cols"], case["batch"]
        gives = rows // 2 if case["form"] == "swiglu" else rows
        more = batch * rows if case["form"] == "residual" else cols if case["form"] != "plain" else 0
        weights = rows * cols // 2 + 2 * rows * -(-cols // case["group"])
        return {"bytes": weights + 4 * batch * (cols + gives) + 4 * more, "flops": 2 * batch * rows * cols}
    rows, context = _lengths(case)
    hq, h, d, n = case["q_heads"], case["kv_heads"], case["head_dim"], sum(rows)
    if case["kind"] == "append":
        # qkv in, the query out, codes and exponents of the new rows out.
        return {"bytes": n * (4 * (2 * hq + 2 * h) * d + 2 * h * d) + 2 * h * -(-n // BLOCK),
                "flops": 10 * n * (hq + 2 * h) * d}
    pairs = sum(a * b + a * (a + 1) // 2 for a, b in zip(rows, context))
    tokens = sum(a + b for a, b in zip(rows, context) if a)
    return {"bytes": 2 * tokens * h * d + 2 * h * -(-tokens // BLOCK) + 8 * n * hq * d, "flops": 4 * pairs * hq * d}


# ----------------------------------------------------------------- exact ----


def exact(case, seed):
    """run()'s floating outputs in 64 bits, from the operators' definitions."""
    global own
    kept, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = kept
    return _EXACT[case["kind"]](case, s)


def _exact_append(case, s):
    hq, d = case["q_heads"], case["head_dim"]
    rows, context = _lengths(case)
    out, first = [], 0
    turn = torch.tensor([THETA ** (-2.0 * i / d) for i in range(d // 2)], device=DEVICE, dtype=torch.float64)
    for n, c in zip(rows, context):
        x = s["qkv"][first:first + n, : hq * d].double().reshape(n, hq, d)
        x = x / ((x ** 2).sum(-1, keepdim=True) / d + EPS).sqrt() * s["q_norm"].double()
        z = torch.complex(x[..., : d // 2], x[..., d // 2:])
        angle = torch.arange(c, c + n, device=DEVICE, dtype=torch.float64)[:, None] * turn
        z = z * torch.polar(torch.ones_like(angle), angle)[:, None]
        out.append(torch.cat([z.real, z.imag], -1).reshape(n, hq * d))
        first += n
    return {"query": torch.cat(out), "error": None, "keys": None, "values": None, "key_exps": None,
            "value_exps": None}


def _exact_attention(case, s):
    hq, h, d = case["q_heads"], case["kv_heads"], case["head_dim"]
    rows, context = _lengths(case)
    out, first = [], 0
    for i, (n, c) in enumerate(zip(rows, context)):
        if not n:
            continue
        pages = s["table"][i].tolist()[: -(-(n + c) // PAGE)]
        key_scale, value_scale = (2.0 ** s[name][pages].double().repeat_interleave(BLOCK, -1)[..., None]
                                  for name in ("key_exps", "value_exps"))
        o = torch.empty((n, hq, d), device=DEVICE, dtype=torch.float64)
        for head in range(hq):
            g = head // (hq // h)
            k = s["keys"][pages, g].double() * key_scale[:, g]
            v = s["values"][pages, g].double().transpose(1, 2) * value_scale[:, g]
            k, v = k.reshape(-1, d)[: n + c].contiguous(), v.reshape(-1, d)[: n + c].contiguous()
            q = s["query"][first:first + n].reshape(n, hq, d)[:, head].double()
            score = (q @ k.t().contiguous()) / math.sqrt(d)
            behind = torch.ones((n, n + c), device=DEVICE, dtype=torch.bool).triu(c + 1)
            o[:, head] = torch.softmax(score.masked_fill(behind, -math.inf), -1) @ v
        out.append(o.reshape(n, hq * d))
        first += n
    return {"out": torch.cat(out), "error": None}


def _exact_matvec(case, s):
    rows, cols, group = case["rows"], case["cols"], case["group"]
    column = torch.arange(cols, device=DEVICE)
    word = column // 128 * 16 + column % 32 // 8 * 4 + column % 128 // 32
    byte = s["codes"][:, word * 4 + column % 8 // 2].long()
    nibble = torch.where(column % 2 == 1, byte // 16, byte % 16)
    w = torch.where(nibble > 7, nibble - 16, nibble).double() * s["scales"].double()[:, column // group]
    x = s["x"].double()
    if "norm" in s:
        x = x / (x.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * s["norm"].double()
    y = x @ w.t().contiguous()
    if case["form"] == "residual":
        y = y + s["residual"].double()
    if case["form"] == "swiglu":
        y = torch.nn.functional.silu(y[:, 0::2]) * y[:, 1::2]
    return {"y": y}


_EXACT = {"append": _exact_append, "attention": _exact_attention, "matvec": _exact_matvec}
