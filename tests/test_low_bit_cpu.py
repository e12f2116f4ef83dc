"""Host side of the 8-bit cache and the 4-bit products: packing of weights, sizes, refusals (no GPU needed: every
refusal comes before any launch)."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

import low_bit_reference as ref


class At:
    """A buffer at an address that is never read."""

    def __init__(self, ptr=4096, nbytes=1 << 20):
        self.ptr, self.nbytes = ptr, nbytes


@pytest.mark.parametrize("rows,cols,group", [(3, 32, 32), (5, 160, 64), (2, 768, 128), (7, 1408, 32), (1, 96, 128)])
def test_quantize_and_back(mmr, rows, cols, group):
    rng = np.random.default_rng(rows + cols)
    w = (rng.standard_normal((rows, cols)) * 0.02).astype(np.float32)
    w[0, :32] = 0
    codes, scales = mmr.q4_quantize(w, group)
    assert codes.shape == (rows, -(-cols // 128) * 64) and scales.shape == (rows, -(-cols // group))
    back = mmr.q4_dequantize(codes, scales, cols, group)
    np.testing.assert_array_equal(back, ref.q4_weights(codes, scales, cols, group).astype(np.float32))
    for g in range(scales.shape[1]):
        part = slice(g * group, min((g + 1) * group, cols))
        top = np.abs(w[:, part]).max(-1)
        np.testing.assert_array_equal(scales[:, g], (top / np.float32(7)).astype(np.float16))
        # Half a step of the scale, and what the largest weight loses where its scale was rounded down.
        assert (np.abs(back[:, part] - w[:, part]) <= (0.5 + 8 * 2.0 ** -11) * scales[:, g:g + 1].astype(np.float32) + 1e-12).all()
    # Whole numbers under a scale come back as they are.
    q = rng.integers(-7, 8, (rows, cols)).astype(np.float32)
    q[:, ::32] = 7
    codes, scales = mmr.q4_quantize(q, group)
    np.testing.assert_array_equal(mmr.q4_dequantize(codes, scales, cols, group), q)
    # Columns past the last are code 0.
    if cols % 128:
        c = np.arange(cols, -(-cols // 128) * 128)
        byte = c // 128 * 64 + (c % 32 // 8 * 4 + c % 128 // 32) * 4 + c % 8 // 2
        assert (codes[:, byte] == 0).all()


def test_quantize_refuses(mmr):
    w = np.ones((2, 64), np.float32)
    for bad in (np.ones((2, 40), np.float32), np.full((2, 64), np.inf, np.float32), np.full((2, 64), np.nan, np.float32)):
        with pytest.raises(mmr.InvalidArgument):
            mmr.q4_quantize(bad, 32)
    for group in (0, 16, 96, -32):
        with pytest.raises(mmr.InvalidArgument):
            mmr.q4_quantize(w, group)
    assert mmr.lib().mmr_q4_code_bytes(0, 64) == 0 and mmr.lib().mmr_q4_code_bytes(3, 160) == 3 * 128
    with pytest.raises(mmr.InvalidArgument):
        mmr.check(mmr.lib().mmr_q4_quantize(None, 2, 64, 32, None, None))


def test_matvec_refuses(mmr):
    b = At()
    good = dict(codes=b, scales=b, group=32, rows=64, cols=256, x=b, batch=1, y=b)

    def refused(message, **change):
        a = {**good, **change}
        with pytest.raises(mmr.InvalidArgument, match=message):
            mmr.matvec_q4(a.pop("codes"), a.pop("scales"), a.pop("group"), a.pop("rows"), a.pop("cols"), a.pop("x"),
                          a.pop("batch"), a.pop("y"), **a)

    refused("null", codes=At(None))
    refused("null", y=At(None))
    refused("cols", cols=40)
    refused("range", rows=0)
    refused("range", cols=1 << 21)
    refused("group", group=48)
    refused("batch", batch=0)
    refused("batch", batch=1 << 17)
    refused("aligned", codes=At(4100))
    refused("prologue", prologue=3)
    refused("epilogue", epilogue=3)
    refused("norm_w", prologue=mmr.PRO_RMSNORM)
    refused("residual", epilogue=mmr.EPI_RESIDUAL)
    refused("even", epilogue=mmr.EPI_SWIGLU, rows=63)
    need = mmr.matvec_q4_workspace_size(256, 40)
    assert need > 0 and mmr.matvec_q4_workspace_size(256, 1) == 0 and mmr.matvec_q4_workspace_size(0, 1) == 0
    refused("null workspace", batch=40)
    refused("too small", batch=40, workspace=At(4096, need - 1))
    refused("aligned", batch=40, workspace=At(4104, need))


def pages(mmr, **change):
    sizes = dict(pages=10, seqs=2, pages_per_seq=4, kv_heads=2, head_dim=96)
    buffers = dict(keys=At(), values=At(), key_exps=At(), value_exps=At(), table=At())
    for name, value in change.items():
        (sizes if name in sizes else buffers)[name] = value
    return mmr.Kv8Pages(*buffers.values(), *sizes.values())


BAD_PAGES = [("null", dict(keys=At(None))), ("null", dict(table=At(None))), ("aligned", dict(values=At(4104))),
             ("aligned", dict(key_exps=At(4098))), ("pages", dict(pages=0)), ("pages", dict(pages=1 << 31)),
             ("seqs", dict(seqs=0)), ("seqs", dict(seqs=65536)), ("pages_per_seq", dict(pages_per_seq=0)),
             ("pages_per_seq", dict(pages_per_seq=1 << 25)), ("kv_heads", dict(kv_heads=0)),
             ("kv_heads", dict(kv_heads=65)), ("q_heads", dict(kv_heads=3)), ("head_dim", dict(head_dim=48)),
             ("head_dim", dict(head_dim=256))]


@pytest.mark.parametrize("message,change", BAD_PAGES)
def test_cache_calls_refuse_bad_caches(mmr, message, change):
    b, cache = At(), pages(mmr, **change)
    with pytest.raises(mmr.InvalidArgument, match=message):
        mmr.kv8_attention(b, cache, b, b, 4, 1, 200, 8, b, b, b)
    rope = At()
    rope.handle = None
    with pytest.raises(mmr.InvalidArgument):
        mmr.kv8_append(b, b, b, 1e-5, rope, cache, b, b, 4, 1, 8, b, b)


def test_attention_refuses(mmr):
    b = At()
    good = dict(query=b, cache=pages(mmr), offsets=b, context=b, rows=4, max_rows=1, max_tokens=200, q_heads=8, out=b,
                workspace=b, error=b)

    def refused(message, **change):
        with pytest.raises(mmr.InvalidArgument, match=message):
            mmr.kv8_attention(*{**good, **change}.values())

    for name in ("query", "offsets", "context", "out", "error"):
        refused("null", **{name: At(None)})
    refused("aligned", query=At(4100))
    refused("aligned", out=At(4104))
    refused("aligned", workspace=At(4104))
    refused("max_rows", rows=-1)
    refused("max_rows", max_rows=5)
    refused("max_rows", max_rows=-1)
    refused("rows", rows=1 << 25)
    refused("like lengths", cache=pages(mmr, seqs=4096), rows=1 << 17, max_rows=1 << 15)
    refused("q_heads", q_heads=3)
    refused("q_heads", q_heads=0)
    refused("max_tokens", max_tokens=0)
    refused("max_tokens", max_tokens=257)
    need = mmr.kv8_attention_workspace_size(8, 2, 96, 1, 1, 1, 1 << 18)
    assert need > 0
    big = pages(mmr, seqs=1, pages_per_seq=4096)
    refused("null workspace", cache=big, rows=1, max_tokens=1 << 18, workspace=None)
    refused("too small", cache=big, rows=1, max_tokens=1 << 18, workspace=At(4096, need - 1))
    with pytest.raises(mmr.InvalidArgument, match="null cache"):
        mmr.check(mmr.lib().mmr_kv8_attention(4096, None, 4096, 4096, 1, 1, 64, 8, 4096, None, 0, 4096, None))
    assert mmr.kv8_attention_workspace_size(7, 2, 96, 1, 1, 1, 100) == 0
    assert mmr.kv8_attention_workspace_size(8, 2, 96, 1, 0, 0, 100) == 0


def test_append_without_a_table_or_rows(mmr):
    b = At()
    rope = At()
    rope.handle = None
    with pytest.raises(mmr.InvalidArgument, match="null argument"):
        mmr.kv8_append(b, b, b, 1e-5, rope, pages(mmr), b, b, 4, 1, 8, b, b)
    with pytest.raises(mmr.InvalidArgument, match="q_heads"):
        mmr.kv8_append(b, b, b, 1e-5, rope, pages(mmr), b, b, 4, 1, 7, b, b)
    assert C.sizeof(mmr._Kv8PagesStruct) == 80


def test_sizes_of_what_no_call_takes(mmr):
    """0 bytes, not the wrapped product."""
    def attention(max_tokens):
        return mmr.kv8_attention_workspace_size(8, 2, 96, 1, 1, 1, max_tokens)

    most = 64 << 24  # pages_per_seq is at most 2^24
    assert attention(most) == attention(most - 63) == 64 * 8 * (96 + 2) * 4
    for tokens in (most + 1, 1 << 40, 1 << 62, (1 << 63) - 1, 0, -1):
        assert attention(tokens) == 0, tokens
    code_bytes = mmr.lib().mmr_q4_code_bytes
    assert code_bytes(1 << 24, 1 << 20) == 1 << 43
    for rows, cols in (((1 << 24) + 1, 32), (1, (1 << 20) + 32), (1 << 62, 128), (3, (1 << 63) - 1), (-1, 32)):
        assert code_bytes(rows, cols) == 0, (rows, cols)
