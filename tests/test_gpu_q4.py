"""Products with 4-bit weights on the GPU against the formula in 64 bits."""
from __future__ import annotations

import numpy as np
import pytest

import low_bit_reference as ref

pytestmark = pytest.mark.gpu
HALF_STEP = 2.0 ** -24


def random_weights(rng, rows, cols, group):
    runs = -(-cols // 128)
    codes = rng.integers(0, 256, (rows, runs, 4, 4, 4)).astype(np.uint8)  # part, 32 columns, byte
    for r in range(4):
        if (runs - 1) * 128 + 32 * r >= cols:
            codes[:, -1, :, r] = 0
    codes = codes.reshape(rows, runs * 64)
    scales = (0.01 * np.exp(0.4 * rng.standard_normal((rows, -(-cols // group))))).astype(np.float16)
    return codes, scales, ref.q4_weights(codes, scales, cols, group)


def product(w, x, norm, prologue, eps, epilogue, residual, mmr):
    """y in 64 bits and what fp32 may be off by.

    A result is a sum of one product a group, each exact up to the rounding of x to 2^-31 of its run's largest value
    (a half step at most of that value, on at most 128 weights of 8 scales) and three fp32 roundings, added one after
    another within a wave and then over eight waves: (groups + 8) half steps of the sum of |w x|.  The normalised x is
    off by a serial sum of cols / 256 squares, ten more roundings of its joins, the root, the quotient and two
    products."""
    batch, cols = x.shape
    x = x.astype(np.float64)
    steps = w.shape[1] // 32 + 8.0
    if prologue:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + float(np.float32(eps))) * norm.astype(np.float64)
        steps += cols // 256 + 16
    y = x @ w.T
    runs = [slice(i, i + 128) for i in range(0, cols, 128)]
    fixed = sum(np.abs(x[:, r]).max(-1)[:, None] * 2.0 ** -30 * np.abs(w[:, r]).sum(-1) for r in runs)
    off = steps * HALF_STEP * (np.abs(x) @ np.abs(w).T) + fixed
    if epilogue == mmr.EPI_RESIDUAL:
        y = y + residual
        off = off + HALF_STEP * np.abs(y)
    if epilogue == mmr.EPI_SWIGLU:
        g, u, og, ou = y[:, 0::2], y[:, 1::2], off[:, 0::2], off[:, 1::2]
        silu = g / (1 + np.exp(-g))
        # |silu'| < 1.1; the exponential, the sum, the reciprocal and two products: e^-g is off by its own 2 half
        # steps and by its argument's, |g| of them.
        off = np.abs(u) * (1.1 * og + (8 + 2 * np.abs(g)) * HALF_STEP * np.abs(silu)) + np.abs(silu) * ou + 1.1 * og * ou
        y = silu * u
    return y, off


class Call:
    def __init__(self, mmr, rng, rows, cols, group, batch, prologue=0, epilogue=0):
        self.mmr, self.rows, self.cols, self.group, self.batch = mmr, rows, cols, group, batch
        self.prologue, self.epilogue = prologue, epilogue
        self.codes, self.scales, self.w = random_weights(rng, rows, cols, group)
        self.x = (rng.standard_normal((batch, cols)) * np.exp(rng.standard_normal(cols))).astype(np.float32)
        self.norm = (1 + 0.1 * rng.standard_normal(cols)).astype(np.float32)
        self.residual = rng.standard_normal((batch, rows)).astype(np.float32)
        self.out_rows = rows // 2 if epilogue == mmr.EPI_SWIGLU else rows
        self.dw = mmr.DeviceArray.from_numpy(self.codes), mmr.DeviceArray.from_numpy(self.scales)
        self.dnorm, self.dres = (mmr.DeviceArray.from_numpy(a) for a in (self.norm, self.residual))
        size = mmr.matvec_q4_workspace_size(cols, batch)
        self.workspace = mmr.DeviceArray(size, np.uint8) if size else None

    def run(self, x=None, dx=None, y=None, stream=None):
        mmr = self.mmr
        dx = dx or mmr.DeviceArray.from_numpy(self.x if x is None else x)
        y = y or mmr.DeviceArray((self.batch, self.out_rows), np.float32)
        mmr.matvec_q4(*self.dw, self.group, self.rows, self.cols, dx, self.batch, y,
                      norm_w=self.dnorm if self.prologue else None, eps=1e-5, prologue=self.prologue,
                      epilogue=self.epilogue, residual=self.dres if self.epilogue == mmr.EPI_RESIDUAL else None,
                      workspace=self.workspace, stream=stream)
        return y

    def expected(self, x=None):
        return product(self.w, self.x if x is None else x, self.norm, self.prologue, 1e-5, self.epilogue,
                       self.residual, self.mmr)

    def check(self):
        got, (want, off) = self.run().numpy(), self.expected()
        assert (np.abs(got - want) <= off).all(), float((np.abs(got - want) / off).max())


SHAPES = [(1152, 768), (512, 1408), (16, 32), (1, 96), (17, 160), (4096, 768), (34, 4096), (50, 8224)]


@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("batch", [1, 2, 4, 5, 33])
def test_product(gpu, rows, cols, group, batch):
    print(f"[case] q4 {rows}x{cols} group {group} batch {batch}", flush=True)
    Call(gpu, np.random.default_rng(rows + cols + group + batch), rows, cols, group, batch).check()


@pytest.mark.parametrize("rows,cols", [(8192, 768), (8210, 1408), (8200, 4096), (9001, 96), (40000, 256), (8250, 896),
                                       (16400, 2048), (33000, 128), (8192, 8192)])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("batch", [1, 2, 4])
def test_product_of_many_rows(gpu, rows, cols, group, batch):
    """Blocks that take several tiles of rows in turn; ragged rows, runs, chunks and turns."""
    print(f"[case] q4 {rows}x{cols} group {group} batch {batch}", flush=True)
    Call(gpu, np.random.default_rng(rows + cols + group + batch), rows, cols, group, batch).check()


@pytest.mark.parametrize("batch,cols", [(1, 8192), (1, 8224), (2, 4096), (2, 4128), (3, 2688), (3, 2720), (3, 2752),
                                        (4, 2048), (4, 2080)])
@pytest.mark.parametrize("rows", [40, 8200])
def test_most_columns_of_one_launch(gpu, batch, cols, rows):
    """Where the runs of all rows of x just fit one launch, and just don't: a ragged run counts as a whole one."""
    print(f"[case] q4 {rows}x{cols} batch {batch}", flush=True)
    Call(gpu, np.random.default_rng(cols + batch), rows, cols, 32, batch, 1).check()


@pytest.mark.parametrize("rows,cols,batch", [(8210, 2048, 20), (4112, 4096, 33), (1030, 4096, 130), (16390, 768, 17),
                                             (520, 8192, 260), (40, 512, 4100)])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_product_of_many_rows_and_many_of_x(gpu, rows, cols, batch, group):
    """Two tiles a wave and 16 rows of x, the codes in chunks of four runs; ragged rows, tiles, chunks and rows of x."""
    print(f"[case] q4 {rows}x{cols} group {group} batch {batch}", flush=True)
    Call(gpu, np.random.default_rng(rows + cols + group + batch), rows, cols, group, batch).check()


@pytest.mark.parametrize("prologue,epilogue", [(1, 2), (2, 1), (0, 2)])
def test_fused_forms_of_many_rows_and_many_of_x(gpu, prologue, epilogue):
    Call(gpu, np.random.default_rng(prologue + epilogue), 8222, 2048, 32, 19, prologue, epilogue).check()


def test_most_rows_of_x(gpu):
    Call(gpu, np.random.default_rng(19), 18, 160, 32, 65536).check()


@pytest.mark.parametrize("prologue,epilogue", [(1, 2), (2, 1), (0, 2)])
@pytest.mark.parametrize("batch", [1, 3])
def test_fused_forms_of_many_rows(gpu, prologue, epilogue, batch):
    Call(gpu, np.random.default_rng(prologue + batch), 8222, 768, 32, batch, prologue, epilogue).check()


@pytest.mark.parametrize("prologue", [0, 1, 2])
@pytest.mark.parametrize("epilogue", [0, 1, 2])
@pytest.mark.parametrize("batch", [1, 3, 18])
@pytest.mark.parametrize("rows,cols,group", [(258, 768, 32), (40, 1408, 64), (512, 96, 128)])
def test_fused_forms(gpu, prologue, epilogue, batch, rows, cols, group):
    rng = np.random.default_rng(prologue * 9 + epilogue * 3 + batch + cols)
    Call(gpu, rng, rows, cols, group, batch, prologue, epilogue).check()


def test_residual_in_place(gpu):
    for batch in (1, 7):
        c = Call(gpu, np.random.default_rng(3), 100, 256, 32, batch, 0, gpu.EPI_RESIDUAL)
        want, off = c.expected()
        y = gpu.DeviceArray.from_numpy(c.residual)
        c.dres = y
        assert (np.abs(c.run(y=y).numpy() - want) <= off).all()


@pytest.mark.parametrize("batch", [1, 4, 6])
def test_x_of_any_size(gpu, batch):
    """Zeros, runs that are 2^60 apart, subnormals and the largest values."""
    rng = np.random.default_rng(11)
    c = Call(gpu, rng, 48, 640, 64, batch)
    c.x[:, :128] *= 2.0 ** 60
    c.x[:, 128:256] = 0
    c.x[:, 256:384] *= 2.0 ** -100
    c.check()
    c.x[:] = 0
    assert (c.run().numpy() == 0).all()
    c.x[:] = rng.standard_normal(c.x.shape) * 2.0 ** 120
    c.check()


class Behind:
    """An array behind a few elements of its type: aligned to that type only."""

    def __init__(self, mmr, a, skip):
        self.whole = mmr.DeviceArray.from_numpy(np.concatenate([np.zeros(skip, a.dtype), a.reshape(-1)]))
        self.skip, self.shape, self.nbytes = skip, a.shape, a.nbytes
        self.ptr = self.whole.ptr + skip * a.dtype.itemsize

    def numpy(self):
        return self.whole.numpy()[self.skip:].reshape(self.shape)


@pytest.mark.parametrize("rows,batch", [(70, 1), (70, 9), (8230, 2), (8230, 40)])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_operands_aligned_to_their_type_only(gpu, rows, batch, group):
    c = Call(gpu, np.random.default_rng(rows + batch), rows, 768, group, batch, 1, gpu.EPI_RESIDUAL)
    c.dw = c.dw[0], Behind(gpu, c.scales, 1)
    c.dnorm, c.dres = Behind(gpu, c.norm, 1), Behind(gpu, c.residual, 3)
    y = Behind(gpu, np.zeros((batch, rows), np.float32), 1)
    got, (want, off) = c.run(dx=Behind(gpu, c.x, 3), y=y).numpy(), c.expected()
    assert (np.abs(got - want) <= off).all()
    assert y.whole.numpy()[0] == 0


@pytest.mark.parametrize("batch", [1, 3, 20])
def test_norm_of_zeros(gpu, batch):
    c = Call(gpu, np.random.default_rng(21), 64, 256, 32, batch, 1)
    c.x[-1] = 0
    got, (want, off) = c.run().numpy(), c.expected()
    assert (np.abs(got - want) <= off).all() and (got[-1] == 0).all()


@pytest.mark.parametrize("prologue", [0, 1])
@pytest.mark.parametrize("batch,rows", [(1, 70), (3, 70), (9, 70), (2, 8230), (140, 8230)])
def test_x_that_is_not_finite(gpu, batch, rows, prologue):
    """Infinities and NaN go where the formula takes them, and to no other row of x."""
    rng = np.random.default_rng(13)
    c = Call(gpu, rng, rows, 384, 32, batch, prologue)
    clean = c.run().numpy()
    x = c.x.copy()
    x[batch - 1, 300] = np.inf
    got = c.run(x=x).numpy()
    np.testing.assert_array_equal(got[: batch - 1], clean[: batch - 1])
    if prologue:
        assert np.isnan(got[-1]).all()  # inf times the 0 that its norm gives
    else:
        w = c.w[:, 300]
        want = np.where(w > 0, np.inf, np.where(w < 0, -np.inf, np.nan))
        np.testing.assert_array_equal(got[-1], want.astype(np.float32))
    x[batch - 1, 5] = np.nan
    got = c.run(x=x).numpy()
    np.testing.assert_array_equal(got[: batch - 1], clean[: batch - 1])
    assert np.isnan(got[-1]).all()


@pytest.mark.parametrize("batch", [1, 20])
def test_recorded_and_other_stream(gpu, batch):
    mmr, rng = gpu, np.random.default_rng(15)
    calls = [Call(mmr, np.random.default_rng(16), 1000, 768, 32, batch, 1) for _ in range(2)]
    streams = [mmr.Stream(), mmr.Stream()]
    dx = [mmr.DeviceArray((batch, 768), np.float32) for _ in calls]
    y = [mmr.DeviceArray((batch, 1000), np.float32) for _ in calls]
    graphs = []
    for i in range(2):
        with mmr.Graph(streams[i]) as g:
            calls[i].run(dx=dx[i], y=y[i], stream=streams[i])
        graphs.append(g)
    for step in range(5):
        x = rng.standard_normal((batch, 768)).astype(np.float32)
        want = calls[0].run(x=x).numpy()
        for i in range(2):
            dx[i].upload(x)
        for i in range(2):
            graphs[i].launch()
        mmr.synchronize()
        for i in range(2):
            np.testing.assert_array_equal(y[i].numpy(), want)


def test_quantized_weights_round_trip(gpu):
    """Weights through the packer: the product is that of the weights the codes stand for."""
    rng = np.random.default_rng(17)
    w = (rng.standard_normal((200, 416)) * 0.02).astype(np.float32)
    for group in (32, 64, 128):
        c = Call(gpu, rng, 200, 416, group, 2)
        c.codes, c.scales = gpu.q4_quantize(w, group)
        c.w = gpu.q4_dequantize(c.codes, c.scales, 416, group).astype(np.float64)
        c.dw = gpu.DeviceArray.from_numpy(c.codes), gpu.DeviceArray.from_numpy(c.scales)
        c.check()


@pytest.mark.parametrize("rows,batch", [(48, 1), (48, 4), (48, 6), (8230, 2), (8230, 40)])
@pytest.mark.parametrize("power", [-90, -112, -121, -135])
def test_x_that_is_tiny_throughout(gpu, rows, batch, power):
    """As many bits of x as of any other, down to its subnormals. Besides the relative bound, a rounding to a subnormal
    number is off by half of 2^-149."""
    c = Call(gpu, np.random.default_rng(23), rows, 640, 64, batch)
    c.x = np.ldexp(c.x, power).astype(np.float32)
    got, (want, off) = c.run().numpy(), c.expected()
    off = off + (640 // 32 + 8) * 2.0 ** -150
    assert (np.abs(got - want) <= off).all(), float((np.abs(got - want) / off).max())
