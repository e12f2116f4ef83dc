"""Operators of beam search and long chats on the 8-bit paged cache.

What a server does between and around decode steps when it keeps several
hypotheses of a sequence, or lets sequences run past what their attention looks
back on: the selection of the best continuations over beams and vocabulary, the
forking of sequences in the page tables (sharing, copying, growing and freeing
pages), the compaction of a pool of pages, and attention over the last keys and
a few first ones.

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
PAGE, BLOCK = 64, 16  # tokens of a page, and of a block under one exponent
BLOCKS = PAGE // BLOCK
BAD_ROWS, NOT_FINITE, NO_PAGES = 1, 2, 4  # bits of an error word
EOS = 2


def listed():
    return [
        # One search of four beams over the model's vocabulary: the smallest selection, all latency.
        dict(name="select_step", kind="select", searches=1, beams=4, vocab=6400, power=0.0),
        # A batch of searches, ranked by their length too.
        dict(name="select_batch", kind="select", searches=32, beams=4, vocab=6400, power=0.6),
        # A wide vocabulary of odd size, more beams: the logits are what is read.
        dict(name="select_wide", kind="select", searches=16, beams=8, vocab=100003, power=1.0),
        # One search's beams after a selection: shared pages, two copied ones in each of 16 layers.
        dict(name="fork_step", kind="fork", what="beams", seqs=4, group=4, context=777, layers=16, kv_heads=2,
             head_dim=96, sinks=0, window=0),
        # A batch of searches in the middle of long answers.
        dict(name="fork_beams", kind="fork", what="beams", seqs=256, group=8, context=2030, layers=16, kv_heads=2,
             head_dim=96, sinks=0, window=0),
        # A server's step: sequences that grow by a row or by a prompt, ended ones that free their pages, drafts that
        # are taken back, and pages that fell behind the window.
        dict(name="fork_serve", kind="fork", what="serve", seqs=200, group=1, context=6000, layers=8, kv_heads=2,
             head_dim=64, sinks=64, window=2048),
        # A small pool between two requests.
        dict(name="compact_small", kind="compact", pages=300, seqs=6, context=1500, layers=16, kv_heads=2,
             head_dim=96),
        # A large pool, half of it in use, before its tail is given back.
        dict(name="compact_large", kind="compact", pages=5000, seqs=60, context=4000, layers=8, kv_heads=2,
             head_dim=64),
        # One query far into a chat that looks back on 1,000 keys.
        dict(name="window_step", kind="window", seqs=1, rows=1, context=32000, q_heads=8, kv_heads=2, head_dim=96,
             sinks=4, window=1000),
        # A step of a batch deep into its contexts.
        dict(name="window_batch", kind="window", seqs=64, rows=1, context=8191, q_heads=8, kv_heads=2, head_dim=96,
             sinks=4, window=2048),
        # Several rows a sequence (drafted tokens to check), of the small model's heads.
        dict(name="window_rows", kind="window", seqs=16, rows=5, context=2500, q_heads=8, kv_heads=2, head_dim=64,
             sinks=70, window=500),
        # A long prompt's later part, after the rows that an earlier call cached.
        dict(name="window_prompt", kind="window", seqs=1, rows=5000, context=1111, q_heads=8, kv_heads=2,
             head_dim=96, sinks=16, window=1500),
    ]


def _between(rng, low, high):
    """A whole number in [low, high], even over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["select", "fork", "fork", "compact", "window", "window"])
    if kind == "select":
        beams = rng.choice([1, 2, 3, 4, 5, 8, 16])
        vocab = rng.choice([6400, _between(rng, 200, 100000)])
        return dict(kind=kind, searches=_between(rng, 1, max(1, min(64, 12800000 // (beams * vocab)))), beams=beams,
                    vocab=vocab, power=rng.choice([0.0, 0.6, 1.0]))
    heads, d, layers = rng.choice([(2, 96, 16), (2, 64, 8), (4, 32, 5), (1, 128, 12)])
    if kind == "fork":
        if rng.random() < 0.5:
            group = rng.choice([2, 3, 4, 8])
            return dict(kind=kind, what="beams", seqs=group * _between(rng, 1, 256 // group), group=group,
                        context=_between(rng, 3, 2000), layers=layers, kv_heads=heads, head_dim=d, sinks=0, window=0)
        return dict(kind=kind, what="serve", seqs=_between(rng, 2, 128), group=1, context=_between(rng, 300, 4000),
                    layers=layers, kv_heads=heads, head_dim=d, sinks=rng.choice([0, 4, 100]),
                    window=rng.choice([0, 100, _between(rng, 64, 2000)]))
    if kind == "compact":
        pages = _between(rng, 10, 2500)
        seqs = _between(rng, 1, max(1, pages // 10))
        return dict(kind=kind, pages=pages, seqs=seqs, context=_between(rng, 30, max(31, 40 * pages // seqs)),
                    layers=layers, kv_heads=heads, head_dim=d)
    q_heads, kv_heads = rng.choice([(8, 2), (8, 2), (4, 4), (8, 1), (12, 4)])
    d = rng.choice([64, 96, 128])
    what = rng.choice(["step", "rows", "prompt"])
    if what == "step":
        seqs, rows = _between(rng, 1, 64), 1
        context = _between(rng, 5, min(32000, 400000 // seqs))
    elif what == "rows":
        seqs, rows = _between(rng, 1, 24), rng.randrange(2, 9)
        context = _between(rng, 5, min(20000, 65536 // seqs))
    else:
        seqs = rng.choice([1, 1, 2, 5])
        rows = _between(rng, 12, 2400 // seqs)
        context = rng.choice([0, rng.randrange(1200)])
    return dict(kind=kind, seqs=seqs, rows=rows, context=context, q_heads=q_heads, kv_heads=kv_heads, head_dim=d,
                sinks=rng.choice([0, 1, 4, 64, rng.randrange(200)]),
                window=_between(rng, 1, 1000 if what == "prompt" else 2500))


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


def _codes(g, shape):
    return torch.randint(-127, 128, shape, generator=g, device=DEVICE, dtype=torch.int8)


def _ints(values):
    return torch.tensor(values, device=DEVICE, dtype=torch.int32)


def _mmr():
    folder = str(Path("minimind-orangepi_amd").resolve())
    if folder not in sys.path:
        sys.path.insert(0, folder)
    import mmr

    return mmr


class _Numbers:
    """Whole numbers that depend on nothing but what they are for."""

    def __init__(self, start=12345):
        self.state = start

    def __call__(self, n):
        self.state = (self.state * 1103515245 + 12345) % 2**31
        return (self.state >> 8) % n


def _lengths(case):
    """Rows and contexts of each sequence: the first as the case says, the others ragged down to a quarter; of four
    or more sequences with several rows each, one brings none."""
    rows, context, number = [case["rows"]], [case["context"]], _Numbers()
    for s in range(1, case["seqs"]):
        rows.append(0 if s == 3 and case["rows"] > 1 else max(1, case["rows"] * (250 + number(751)) // 1000))
        context.append(case["context"] * (250 + number(751)) // 1000)
    return rows, context


def _dropped(p, keep, sinks, window):
    """Whether page p is behind the window of every row from position `keep` on."""
    return window > 0 and p * PAGE >= sinks and p * PAGE + PAGE - 1 < keep - window + 1


def _forks(case):
    """Of each sequence: the tokens it has, and the parent, kept tokens and room that it is to have."""
    seqs, number = case["seqs"], _Numbers()
    has, parent, keep, room = [], [], [], []
    if case["what"] == "beams":
        for first in range(0, seqs, case["group"]):
            context = case["context"] if first == 0 else case["context"] * (250 + number(751)) // 1000
            for _ in range(case["group"]):  # of beams some go on twice or more often
                has.append(context)
                parent.append(first + number(case["group"]))
                keep.append(context)
                room.append(1)
        return has, parent, keep, room
    for s in range(seqs):
        context = case["context"] if s == 0 else case["context"] * (250 + number(751)) // 1000
        what = number(16)
        has.append(context)
        parent.append(-1 if what < 3 else s)  # ended; of those, some are followed by a new prompt
        keep.append(0 if what < 3 else context - number(5) if what < 6 else context)
        room.append(0 if what == 0 else 1 + number(case["context"] // 2) if what < 3 else 1 + number(6)
                    if what < 6 else 1)
    return has, parent, keep, room


# --------------------------------------------------------------- prepare ----


def prepare(case, seed):
    state = {"case": case, **_PREPARE[case["kind"]](case, _generator(seed))}
    if own:  # the handles that a program keeps
        state["mmr"] = _mmr()
        state["buffer"] = {n: Buffer(t) for n, t in state.items() if isinstance(t, torch.Tensor)}
        _KEEP[case["kind"]](state, state["mmr"], state["buffer"])
    return state


def _prepare_select(case, g):
    rows, vocab = case["searches"] * case["beams"], case["vocab"]
    # A few tokens far above the rest, as a trained model's logits have.
    logits = _normal(g, (rows, vocab), 1.5) + 6.0 * torch.exp(_normal(g, (rows, vocab), 0.5) - 2.0)
    steps = torch.randint(1, 40, (rows,), generator=g, device=DEVICE, dtype=torch.int32)
    ended = (torch.rand((rows,), generator=g, device=DEVICE) < 0.1).int()
    return dict(logits=logits, scores=-2.0 * steps.float() * torch.exp(_normal(g, (rows,), 0.2)), lengths=steps,
                ended=ended, scores_out=torch.zeros(rows, device=DEVICE), lengths_out=torch.zeros_like(steps),
                ended_out=torch.zeros_like(steps), parent=torch.zeros_like(steps), token=torch.zeros_like(steps),
                error=_ints([0]))


def _pool(g, case, pages):
    """Pages of every layer, of any content, and one more of each that the plain form writes where nothing is due."""
    h, d, n = case["kv_heads"], case["head_dim"], case["layers"]
    return dict(keys=_codes(g, (n, pages + 1, h, PAGE, d)), values=_codes(g, (n, pages + 1, h, d, PAGE)),
                key_exps=_codes(g, (n, pages + 1, h, BLOCKS)), value_exps=_codes(g, (n, pages + 1, h, BLOCKS)))


def _prepare_fork(case, g):
    has, parent, keep, room = _forks(case)
    per = max(-(-max(a, k + r) // PAGE) for a, k, r in zip(has, keep, room)) + 1
    held = [[p for p in range(-(-n // PAGE)) if not _dropped(p, n - 1, case["sinks"], case["window"])] for n in has]
    pages = sum(map(len, held)) + sum(-(-r // PAGE) + 1 for r in room)
    order = torch.randperm(pages, generator=g, device=DEVICE).tolist()
    table = [[-1] * per for _ in has]
    users = [0] * pages
    for s, mine in enumerate(held):
        first = s // case["group"] * case["group"]
        for p in mine:
            # Beams of one search have the same first half of their pages.
            same = s > first and p < len(held[first]) // 2
            table[s][p] = table[first][p] if same else order.pop()
            users[table[s][p]] += 1
    return dict(_pool(g, case, pages), table=_ints(table), users=_ints(users), parent=_ints(parent),
                keep=_ints(keep), room=_ints(room), error=_ints([0]))


def _prepare_compact(case, g):
    pages, seqs, number = case["pages"], case["seqs"], _Numbers()
    context = [case["context"] * (250 + number(751)) // 1000 for _ in range(seqs)]
    per = max(-(-n // PAGE) for n in context) + 2
    order = torch.randperm(pages, generator=g, device=DEVICE).tolist()
    table, users = [[-1] * per for _ in range(seqs)], [0] * pages
    for s, n in enumerate(context):
        for p in range(-(-n // PAGE)):
            if s % 3 == 1 and p < 2 and table[s - 1][p] >= 0:  # a prompt that two sequences share
                table[s][p] = table[s - 1][p]
            elif order:
                table[s][p] = order.pop()
            if table[s][p] >= 0:
                users[table[s][p]] += 1
    return dict(_pool(g, case, pages), table=_ints(table), users=_ints(users), table_out=_ints(table),
                users_out=_ints(users), moved=_ints([0] * pages), live=_ints([0]))


def _exponent(top):
    """The least e with top <= 127 * 2^e, in the cache's range."""
    m, x = torch.frexp(top)
    return torch.where(top > 0, x - 7 + (m > 127 / 128).int(), -126).clamp(-126, 122)


def _prepare_window(case, g):
    """Pages in any order, full of cached tokens of several sizes; those behind every row's window are gone."""
    rows, context = _lengths(case)
    hq, h, d, n = case["q_heads"], case["kv_heads"], case["head_dim"], sum(rows)
    per = max(-(-(a + b) // PAGE) for a, b in zip(rows, context))
    place = torch.arange(per, device=DEVICE)
    first = _ints(context)[:, None] - case["window"] + 1  # of the keys of a sequence's first row
    gone = (place * PAGE >= case["sinks"]) & (place * PAGE + PAGE - 1 < first)
    gone |= place * PAGE >= _ints([a + b for a, b in zip(rows, context)])[:, None]
    number = (~gone).reshape(-1).int().cumsum(0).reshape(gone.shape) - 1
    pages = sum(1 for s in range(len(rows)) for p in range(-(-(rows[s] + context[s]) // PAGE))
                if not _dropped(p, context[s], case["sinks"], case["window"])) + 3
    order = torch.randperm(pages, generator=g, device=DEVICE)
    state = dict(table=torch.where(gone, -1, order[number.clamp(0)]).int())
    for name, std in (("key", 1.0), ("value", 0.6)):
        x = _normal(g, (pages, h, PAGE, d), std) * torch.exp(_normal(g, (pages, h, PAGE, 1), 0.3))
        e = _exponent(x.reshape(pages, h, BLOCKS, -1).abs().amax(-1))
        x = torch.ldexp(x, -e.repeat_interleave(BLOCK, -1)[..., None]).round().to(torch.int8)
        state[name + "s"] = (x if name == "key" else x.transpose(-1, -2)).contiguous()
        state[name + "_exps"] = e.to(torch.int8)
    return dict(state, query=_normal(g, (n, hq * d)), out=torch.zeros((n, hq * d), device=DEVICE), error=_ints([0]),
                offsets=_ints([sum(rows[:i]) for i in range(len(rows) + 1)]), context=_ints(context),
                max_rows=max(rows), max_tokens=max(a + b for a, b in zip(rows, context)))


_PREPARE = {"select": _prepare_select, "fork": _prepare_fork, "compact": _prepare_compact, "window": _prepare_window}


def _workspace(buffers, size):
    buffers["workspace"] = Buffer(torch.empty(max(1, size), device=DEVICE, dtype=torch.uint8))


def _keep_select(state, mmr, b):
    c = state["case"]
    _workspace(b, mmr.beam_select_workspace_size(c["searches"], c["beams"], c["vocab"]))
    state["from"] = mmr.Beams(b["scores"], b["lengths"], b["ended"])
    state["to"] = mmr.Beams(b["scores_out"], b["lengths_out"], b["ended_out"])


def _keep_layers(state, mmr, b):
    c, parts = state["case"], [state[n] for n in ("keys", "values", "key_exps", "value_exps")]
    pages = [mmr.Kv8Pages(*(Buffer(t[layer]) for t in parts), b["table"], state["users"].numel(),
                          *state["table"].shape, c["kv_heads"], c["head_dim"]) for layer in range(c["layers"])]
    state["layers"] = mmr.Kv8Layers(pages)


def _keep_fork(state, mmr, b):
    _keep_layers(state, mmr, b)
    _workspace(b, mmr.kv8_fork_workspace_size(*state["table"].shape, state["users"].numel()))


def _keep_compact(state, mmr, b):
    _keep_layers(state, mmr, b)
    _workspace(b, mmr.kv8_compact_workspace_size(state["users"].numel()))


def _keep_window(state, mmr, b):
    c = state["case"]
    state["pages"] = mmr.Kv8Pages(b["keys"], b["values"], b["key_exps"], b["value_exps"], b["table"],
                                  state["keys"].shape[0], *state["table"].shape, c["kv_heads"], c["head_dim"])
    _workspace(b, mmr.kv8_window_attention_workspace_size(
        c["q_heads"], c["kv_heads"], c["head_dim"], c["seqs"], state["query"].shape[0], state["max_rows"],
        state["max_tokens"], c["sinks"], c["window"]))


_KEEP = {"select": _keep_select, "fork": _keep_fork, "compact": _keep_compact, "window": _keep_window}


# ------------------------------------------------------------------- run ----


def run(state):
    return _RUN[state["case"]["kind"]](state)


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _run_select(s):
    if own:
        c, b = s["case"], s["buffer"]
        s["mmr"].beam_select(b["logits"], c["searches"], c["beams"], c["vocab"], EOS, c["power"], s["from"], s["to"],
                             b["parent"], b["token"], b["workspace"], b["error"], stream=_stream())
    else:
        _plain_select(s)
    return {"scores": s["scores_out"], "lengths": s["lengths_out"], "ended": s["ended_out"], "parent": s["parent"],
            "token": s["token"], "error": s["error"]}


def _pages_of(s):
    """The pool without the plain form's spare page: codes and exponents as the whole numbers that they are."""
    return {n: s[n][:, :-1] for n in ("keys", "values", "key_exps", "value_exps")}


def _run_fork(s):
    if own:
        c, b = s["case"], s["buffer"]
        s["mmr"].kv8_fork(s["layers"], b["users"], b["parent"], b["keep"], b["room"], b["workspace"], b["error"],
                          sinks=c["sinks"], window=c["window"], stream=_stream())
    else:
        _plain_fork(s)
    return {"table": s["table"], "users": s["users"], "error": s["error"], **_pages_of(s)}


def _run_compact(s):
    if own:
        b = s["buffer"]
        s["mmr"].kv8_compact(s["layers"], b["users"], b["table_out"], b["users_out"], b["moved"], b["live"],
                             b["workspace"], stream=_stream())
    else:
        _plain_compact(s)
    return {"table": s["table_out"], "users": s["users_out"], "moved": s["moved"], "live": s["live"], **_pages_of(s)}


def _run_window(s):
    if own:
        c, b = s["case"], s["buffer"]
        s["mmr"].kv8_window_attention(b["query"], s["pages"], b["offsets"], b["context"], s["query"].shape[0],
                                      s["max_rows"], s["max_tokens"], c["sinks"], c["window"], c["q_heads"], b["out"],
                                      b["workspace"], b["error"], stream=_stream())
    else:
        _plain_window(s)
    return {"out": s["out"], "error": s["error"]}


_RUN = {"select": _run_select, "fork": _run_fork, "compact": _run_compact, "window": _run_window}


# ----------------------------------------------------------- plain forms ----


def _plain_select(s):
    c = s["case"]
    searches, beams, vocab, power = c["searches"], c["beams"], c["vocab"], c["power"]
    # In 64 bits: what is chosen are values next to each other.
    x = s["logits"].double()
    top = x.amax(-1, keepdim=True)
    lse = top + (x - top).exp().sum(-1, keepdim=True).log()
    fine = (lse.abs() < math.inf)
    s["error"] |= torch.where((x == math.inf).any() | x.isnan().any(), NOT_FINITE, 0).int()
    done = s["ended"] != 0
    token = torch.arange(vocab, device=DEVICE)
    before = s["scores"].double()[:, None]
    score = torch.where(fine, before + (x - lse), -math.inf)
    score = torch.where(done[:, None], torch.where(token == EOS, before, -math.inf), score)
    score = torch.where(score.float() > -math.inf, score, -math.inf)
    length = s["lengths"] + (~done).int()
    rank = score * length.double().clamp(min=1)[:, None] ** -power
    rank, at = torch.sort(rank.reshape(searches, beams * vocab), dim=-1, descending=True, stable=True)
    short = beams - at.shape[1]
    if short > 0:  # fewer continuations than beams
        rank = torch.nn.functional.pad(rank, (0, short), value=-math.inf)
        at = torch.nn.functional.pad(at, (0, short))
    rank, at = rank[:, :beams].reshape(-1), at[:, :beams].reshape(-1)
    left = rank > -math.inf
    row = at // vocab + torch.arange(searches, device=DEVICE).repeat_interleave(beams) * beams
    chosen = score[row, at % vocab]
    s["scores_out"].copy_(torch.where(left, chosen, -math.inf))
    s["parent"].copy_(torch.where(left, row, -1))
    s["token"].copy_(torch.where(left, at % vocab, EOS))
    s["lengths_out"].copy_(torch.where(left, length[row], 0))
    s["ended_out"].copy_(torch.where(left, at % vocab == EOS, True))


def _plain_fork(s):
    c = s["case"]
    (seqs, per), pages = s["table"].shape, s["users"].numel()
    table, parent = s["table"].long(), s["parent"].long()
    keep, room = s["keep"].long()[:, None], s["room"].long()[:, None]
    place = torch.arange(per, device=DEVICE)
    full, part = keep // PAGE, keep % PAGE

    def count(entries, valid):
        return torch.zeros(pages + 1, device=DEVICE, dtype=torch.int32).index_add(
            0, torch.where(valid, entries, pages).reshape(-1),
            torch.ones(entries.numel(), device=DEVICE, dtype=torch.int32))[:pages]

    # Pages that a sequence takes over, and the users that all have then.
    taken = torch.where((parent >= 0)[:, None] & (place * PAGE < keep), table[parent.clamp(0)], -1)
    if c["window"]:
        behind = (place * PAGE >= c["sinks"]) & (place * PAGE + PAGE - 1 < keep - c["window"] + 1)
        taken = torch.where(behind, -1, taken)
    users = s["users"] - count(table, table >= 0) + count(taken, taken >= 0)
    # Partly filled pages that will be written: the first of those who write keeps the page if nobody reads it.
    partly = taken.gather(1, full.clamp(max=per - 1))
    writes = (part > 0) & (room > 0) & (partly >= 0)
    writers = count(partly, writes)
    row = torch.arange(seqs, device=DEVICE)[:, None]
    first = torch.full((pages + 1,), seqs, device=DEVICE).scatter_reduce(
        0, torch.where(writes, partly, pages)[:, 0], row[:, 0], "amin")[:pages]
    page = partly.clamp(0)
    copies = writes & ~((users[page] == writers[page]) & (first[page] == row))
    users = users - count(partly, copies)
    # New pages: the lowest free ones, in the order of sequences and their pages.
    new = (place >= full) & (place * PAGE < keep + room)
    new &= ~((place == full) & (part > 0) & (partly >= 0) & ~copies)
    rank = new.reshape(-1).long().cumsum(0).reshape(seqs, per) - 1
    free = users == 0
    number = torch.full((pages + seqs * per + 1,), -1, device=DEVICE)
    number[torch.where(free, free.long().cumsum(0) - 1, pages + seqs * per)] = torch.arange(pages, device=DEVICE)
    got = torch.where(new, number[:-1][rank.clamp(0)], -1)
    s["error"] |= torch.where((new & (got < 0)).any(), NO_PAGES, 0).int()
    s["users"].copy_(users + count(got, got >= 0))
    s["table"].copy_(torch.where(new, got, taken))
    to = got.gather(1, full.clamp(max=per - 1))
    to, page = torch.where(copies & (to >= 0), to, pages)[:, 0], page[:, 0]  # the spare page where nothing is due
    mine = torch.arange(PAGE, device=DEVICE) // BLOCK * BLOCK < part  # of the blocks with kept tokens
    for layer in range(c["layers"]):
        k, v = s["keys"][layer], s["values"][layer]
        k[to] = torch.where(mine[:, None, :, None], k[page], k[to])
        v[to] = torch.where(mine[:, None, None, :], v[page], v[to])
        for e in (s["key_exps"][layer], s["value_exps"][layer]):
            e[to] = torch.where(mine[:, None, ::BLOCK], e[page], e[to])


def _plain_compact(s):
    pages = s["users"].numel()
    used = s["users"] > 0
    live = used.sum()
    number = torch.arange(pages, device=DEVICE)
    source, hole = torch.nonzero(used & (number >= live))[:, 0], torch.nonzero(~used & (number < live))[:, 0]
    moved = torch.where(used, number, -1)
    moved[source] = hole
    for layer in range(s["case"]["layers"]):
        for name in ("keys", "values", "key_exps", "value_exps"):
            s[name][layer][hole] = s[name][layer][source]
    s["moved"].copy_(moved)
    s["live"].copy_(live)
    s["users_out"].copy_(s["users"])
    s["users_out"][hole] = s["users"][source]
    s["users_out"][source] = 0
    s["table_out"].copy_(torch.where(s["table"] >= 0, moved[s["table"].long().clamp(0)], -1))


def _plain_window(s):
    c = s["case"]
    hq, h, d, sinks, window = c["q_heads"], c["kv_heads"], c["head_dim"], c["sinks"], c["window"]
    n, most, seqs = s["query"].shape[0], s["max_rows"], c["seqs"]
    r = torch.arange(n, device=DEVICE)
    seq = torch.searchsorted(s["offsets"][1:].long().contiguous(), r, right=True)
    index = r - s["offsets"][seq].long()
    # Keys that some row of a sequence attends: its first ones, and those from its first row's window on.
    context = s["context"].long()[:, None]
    first = (context - window + 1).clamp(min=0)
    recent = first + torch.arange(min(window + most - 1, s["max_tokens"]), device=DEVICE)
    early = torch.arange(min(sinks, s["max_tokens"]), device=DEVICE).expand(seqs, -1)
    at = torch.cat([early, recent], 1)
    there = torch.cat([early < first, recent < context + (s["offsets"][1:] - s["offsets"][:-1])[:, None]], 1)
    page = s["table"].long().gather(1, (at // PAGE).clamp(max=s["table"].shape[1] - 1)).clamp(0)
    block, slot = at % PAGE // BLOCK, at % PAGE
    k = torch.ldexp(s["keys"][page, :, slot].float(), s["key_exps"][page, :, block].int()[..., None])
    v = torch.ldexp(s["values"][page, :, :, slot].float(), s["value_exps"][page, :, block].int()[..., None])
    k, v = k.permute(0, 2, 3, 1).contiguous(), v.permute(0, 2, 1, 3).contiguous()
    row = (s["offsets"][:-1, None].long() + torch.arange(most, device=DEVICE)).clamp(max=n - 1)
    q = s["query"][row].reshape(seqs, most, h, hq // h, d).permute(0, 2, 3, 1, 4).reshape(seqs, h, -1, d)
    score = torch.matmul(q, k) * d ** -0.5
    place = (context + torch.arange(most, device=DEVICE))[..., None]  # of a row
    seen = there[:, None] & (at[:, None] <= place) & ((at[:, None] < sinks) | (place - at[:, None] < window))
    score = score.reshape(seqs, h, hq // h, most, -1).masked_fill(~seen[:, None, None], -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True).clamp(min=-1e30))
    o = torch.matmul(p.reshape(seqs, h, -1, at.shape[1]), v).reshape(seqs, h, hq // h, most, d)
    o = o / p.sum(-1, keepdim=True).clamp(min=1e-30)
    s["out"].copy_(o.permute(0, 3, 1, 2, 4)[seq, index].reshape(n, hq * d))


# ------------------------------------------------------------------ work ----


def work(case):
    kind = case["kind"]
    if kind == "select":
        rows = case["searches"] * case["beams"]
        return {"bytes": 4 * rows * case["vocab"] + 32 * rows, "flops": 4 * rows * case["vocab"]}
    if kind == "window":
        rows, context = _lengths(case)
        sinks, window = case["sinks"], case["window"]
        hq, h, d, n = case["q_heads"], case["kv_heads"], case["head_dim"], sum(rows)
        pairs = tokens = 0
        for a, b in zip(rows, context):
            places = range(b, b + a)
            pairs += sum(min(window, p + 1) + min(sinks, max(0, p + 1 - window)) for p in places)
            if a:
                first = max(0, b - window + 1)
                tokens += min(sinks, first) + a + b - first
        return {"bytes": 2 * tokens * h * d + 2 * h * -(-tokens // BLOCK) + 8 * n * hq * d, "flops": 4 * pairs * hq * d}
    h, d = case["kv_heads"], case["head_dim"]
    block = h * (2 * BLOCK * d + 2)  # bytes of a block of tokens: codes and exponents
    if kind == "fork":
        has, parent, keep, room = _forks(case)
        writers = {}
        blocks = table = 0
        for s in range(len(has)):
            table += 4 * (-(-has[s] // PAGE) + -(-(keep[s] + room[s]) // PAGE))  # entries in and out
            if parent[s] >= 0 and keep[s] % PAGE and room[s]:
                first = writers.setdefault((parent[s], keep[s] // PAGE), s)
                blocks += 0 if first == s else -(-(keep[s] % PAGE) // BLOCK)
        return {"bytes": 2 * blocks * block * case["layers"] + table + 12 * len(has), "flops": 0}
    number, pages, left, entries, used = _Numbers(), case["pages"], case["pages"], 0, 0
    context = [case["context"] * (250 + number(751)) // 1000 for _ in range(case["seqs"])]
    for s, n in enumerate(context):
        mine = -(-n // PAGE)
        shared = min(mine, 2, -(-context[s - 1] // PAGE)) if s % 3 == 1 else 0
        entries += mine
        used += min(left, mine - shared)
        left -= min(left, mine - shared)
    moves = round(used * (pages - used) / pages)  # in the mean, of pages in any order
    return {"bytes": 2 * moves * BLOCKS * block * case["layers"] + 8 * entries + 12 * pages, "flops": 0}


# ----------------------------------------------------------------- exact ----


def exact(case, seed):
    """run()'s computed outputs in 64 bits, from the operators' definitions; pages are copied, not computed."""
    global own
    if case["kind"] not in _EXACT:
        return None
    kept, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = kept
    return _EXACT[case["kind"]](case, s)


def _exact_select(case, s):
    searches, beams, power = case["searches"], case["beams"], case["power"]
    out = torch.full((searches * beams,), -math.inf, device=DEVICE, dtype=torch.float64)
    for i in range(searches):
        scores, ranks = [], []
        for b in range(i * beams, (i + 1) * beams):
            if s["ended"][b]:
                scores.append(s["scores"][b].double()[None])
                length = int(s["lengths"][b])
            else:
                scores.append(s["scores"][b].double() + torch.log_softmax(s["logits"][b].double(), 0))
                length = int(s["lengths"][b]) + 1
            ranks.append(scores[-1] / float(max(length, 1)) ** power)
        best = torch.cat(ranks).topk(min(beams, sum(map(len, ranks)))).indices
        out[i * beams: i * beams + len(best)] = torch.cat(scores)[best]
    return {"scores": out, "lengths": None, "ended": None, "parent": None, "token": None, "error": None}


def _exact_window(case, s):
    hq, h, d, sinks, window = (case[k] for k in ("q_heads", "kv_heads", "head_dim", "sinks", "window"))
    rows, context = _lengths(case)
    out, first = [], 0
    for i, (n, c) in enumerate(zip(rows, context)):
        if not n:
            continue
        pages = s["table"][i].clamp(min=0).tolist()[: -(-(n + c) // PAGE)]
        key_scale, value_scale = (2.0 ** s[name][pages].double().repeat_interleave(BLOCK, -1)[..., None]
                                  for name in ("key_exps", "value_exps"))
        back = torch.arange(c, c + n, device=DEVICE)[:, None] - torch.arange(n + c, device=DEVICE)
        unseen = (back < 0) | ((back >= window) & (torch.arange(n + c, device=DEVICE) >= sinks))
        o = torch.empty((n, hq, d), device=DEVICE, dtype=torch.float64)
        for head in range(hq):
            g = head // (hq // h)
            k = s["keys"][pages, g].double() * key_scale[:, g]
            v = s["values"][pages, g].double().transpose(1, 2) * value_scale[:, g]
            k, v = k.reshape(-1, d)[: n + c].contiguous(), v.reshape(-1, d)[: n + c].contiguous()
            q = s["query"][first:first + n].reshape(n, hq, d)[:, head].double()
            score = (q @ k.t().contiguous()) / math.sqrt(d)
            o[:, head] = torch.softmax(score.masked_fill(unseen, -math.inf), -1) @ v
        out.append(o.reshape(n, hq * d))
        first += n
    return {"out": torch.cat(out), "error": None}


_EXACT = {"select": _exact_select, "window": _exact_window}
