"""cudaRmsNormQuantize against the formula in float64."""
import ctypes

import numpy as np
import pytest

from cudabackend_b200 import api
from oracle import oracle as o
from tests import block_scaled as bs

pytestmark = pytest.mark.gpu

DTYPES = ["float16", "bfloat16", "float32"]
EPSILON = 1e-5
# one block, a short last block, odd lengths, each number of warps per row, rows that do not fit in registers
SHAPES = [(1, 1), (1, 128), (3, 7), (2, 1001), (1, 4096), (5, 264), (600, 264), (600, 1024), (7, 2048), (400, 3000), (333, 8192), (2, 16392), (350, 16384),
          (3, 40000), (310, 33000)]


def norm_bound(columns):
    """Relative error of a float32 y: a thread adds up n squares, 5 shuffles and up to 32 partial sums follow (half of that in the
    square root's result); the sum, the division, + epsilon, square root, reciprocal and two products round once each."""
    squares = 8 * max(4, -(-bs.blocks(columns) // 64))
    return ((squares + 5 + 32) / 2 + 8) * bs.U32


def inputs(shape, seed):
    r = np.random.default_rng(seed)
    x = r.normal(0, 1, shape) * np.exp2(r.integers(-4, 5, (shape[0], 1)))
    x[:, r.integers(0, shape[1], max(1, shape[1] // 100))] *= 15
    return x, r.normal(0, 1, shape), 1 + 0.2 * r.normal(0, 1, shape[1])


def check(x64, z64, gamma64, h, y, s, dtype, epsilon=EPSILON):
    shape = x64.shape
    h64, y64 = o.rms_norm(x64, z64, gamma64, epsilon)
    relative = norm_bound(shape[1])
    scales = o.block_scales(y64)
    # float32(x + z) is off by 2^-24 of h (counted in norm_bound through h's relative error)
    assert np.all(np.abs(s.download() - scales) <= scales * (relative + 3 * bs.U32))
    spread = o.spread_scales(s.download(), *shape)
    assert np.all(np.abs(y.download() * spread - y64) <= bs.code_error_bound(y64, spread, relative + 2 * bs.U32))
    assert y.guards_intact() and s.guards_intact()
    if h is not None:
        assert np.all(np.abs(h.download() - h64) <= np.abs(h64) * (bs.HALF_STEP[dtype] + bs.U32) + bs.LEAST[dtype])
        assert h.guards_intact()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_norm(ctx, dtype, residual, shape):
    x0, z0, g0 = inputs(shape, 81)
    x = bs.Placed(ctx, shape, dtype, values=x0)
    z = bs.Placed(ctx, shape, dtype, values=z0) if residual else None
    h = bs.Placed(ctx, shape, dtype) if residual else None
    gamma = bs.Placed(ctx, (shape[1],), "float32", values=g0)
    y, s = bs.Placed(ctx, shape, "float8_e4m3"), bs.Placed(ctx, (shape[0], bs.blocks(shape[1])), "float32")
    bs.rms_norm_quantize(ctx, x, z, h, gamma, EPSILON, y, s)
    check(x.values, z.values if residual else None, gamma.values, h, y, s, dtype)
    assert np.array_equal(x.download(), x.values)


@pytest.mark.parametrize("which", ["x", "z", "neither", "copy"])
@pytest.mark.parametrize("shape", [(4, 520), (2, 40000), (5, 333)])
def test_where_the_sum_goes(ctx, which, shape):
    """h over x, over z, nowhere, and h = x rounded when there is no residual"""
    x0, z0, g0 = inputs(shape, 82)
    x, z = bs.Placed(ctx, shape, "bfloat16", values=x0), bs.Placed(ctx, shape, "bfloat16", values=z0)
    gamma = bs.Placed(ctx, (shape[1],), "float32", values=g0)
    y, s = bs.Placed(ctx, shape, "float8_e4m3"), bs.Placed(ctx, (shape[0], bs.blocks(shape[1])), "float32")
    h = {"x": x, "z": z, "neither": None, "copy": bs.Placed(ctx, shape, "bfloat16")}[which]
    bs.rms_norm_quantize(ctx, x, None if which == "copy" else z, h, gamma, EPSILON, y, s)
    check(x.values, None if which == "copy" else z.values, gamma.values, h, y, s, "bfloat16")


@pytest.mark.parametrize("x_offset,z_offset,h_offset,g_offset,y_offset", [(2, 0, 0, 0, 0), (0, 8, 0, 0, 0), (0, 0, 4, 0, 0), (0, 0, 0, 4, 0), (0, 0, 0, 0, 1)])
def test_unaligned_views(ctx, x_offset, z_offset, h_offset, g_offset, y_offset):
    shape = (9, 1032)
    x0, z0, g0 = inputs(shape, 83)
    x, z = bs.Placed(ctx, shape, "float16", x_offset, values=x0), bs.Placed(ctx, shape, "float16", z_offset, values=z0)
    h, gamma = bs.Placed(ctx, shape, "float16", h_offset), bs.Placed(ctx, (shape[1],), "float32", g_offset, values=g0)
    y, s = bs.Placed(ctx, shape, "float8_e4m3", y_offset), bs.Placed(ctx, (9, 9), "float32", 4)
    bs.rms_norm_quantize(ctx, x, z, h, gamma, EPSILON, y, s)
    check(x.values, z.values, gamma.values, h, y, s, "float16")


def test_zero_rows_nan_and_infinity_stay_in_their_rows(ctx):
    shape = (6, 384)
    x0, _, g0 = inputs(shape, 84)
    x0[1], x0[2, 130], x0[3, 5] = 0.0, np.nan, np.inf
    x = bs.Placed(ctx, shape, "bfloat16", values=x0)
    gamma = bs.Placed(ctx, (384,), "float32", values=g0)
    y, s = bs.Placed(ctx, shape, "float8_e4m3"), bs.Placed(ctx, (6, 3), "float32")
    bs.rms_norm_quantize(ctx, x, None, None, gamma, EPSILON, y, s)
    q, scales = y.download(), s.download()
    assert np.all(q[1] == 0) and np.all(scales[1] == np.float32(2.0 ** -100) / np.float32(448))
    assert np.all(np.isnan(q[2])) and np.all(np.isnan(scales[2]))  # the mean is NaN
    assert np.all(np.isnan(q[3, :128])) and np.isnan(scales[3, 0])  # infinity * 0 in its own block, x * 0 in the others
    assert np.all(q[3, 128:] == 0)
    keep = [0, 4, 5]
    _, y64 = o.rms_norm(x.values[keep], None, gamma.values, EPSILON)
    spread = o.spread_scales(scales[keep], 3, 384)
    assert np.all(np.abs(q[keep] * spread - y64) <= bs.code_error_bound(y64, spread, norm_bound(384) + 2 * bs.U32))


def test_ranks_and_empty_tensors(ctx):
    shape = (2, 3, 4, 136)
    x0, _, g0 = inputs((24, 136), 85)
    x = bs.Placed(ctx, shape, "float32", values=x0)
    gamma = bs.Placed(ctx, (136,), "float32", values=g0)
    y, s = bs.Placed(ctx, shape, "float8_e4m3"), bs.Placed(ctx, (2, 3, 4, 2), "float32")
    bs.rms_norm_quantize(ctx, x, None, None, gamma, EPSILON, y, s)
    _, y64 = o.rms_norm(x.values.reshape(24, 136), None, gamma.values, EPSILON)
    spread = o.spread_scales(s.download().reshape(24, 2), 24, 136)
    assert np.all(np.abs(y.download().reshape(24, 136) * spread - y64) <= bs.code_error_bound(y64, spread, norm_bound(136) + 2 * bs.U32))
    for empty in ((0, 136), (5, 0)):
        e, ey = bs.Placed(ctx, empty, "float32"), bs.Placed(ctx, empty, "float8_e4m3")
        es, eg = bs.Placed(ctx, (empty[0], bs.blocks(empty[1])), "float32"), bs.Placed(ctx, (empty[1],), "float32")
        bs.rms_norm_quantize(ctx, e, None, None, eg, EPSILON, ey, es)
        assert ey.guards_intact() and es.guards_intact()


def test_refusals(ctx):
    P = bs.Placed
    base = {"x": P(ctx, (4, 256), "bfloat16"), "z": P(ctx, (4, 256), "bfloat16"), "h": P(ctx, (4, 256), "bfloat16"), "gamma": P(ctx, (256,), "float32"),
            "epsilon": 1e-6, "y": P(ctx, (4, 256), "float8_e4m3"), "scale": P(ctx, (4, 2), "float32")}

    def status(**change):
        return bs.rms_norm_quantize(ctx, status=True, **{**base, **change})

    bad, dtype = api.STATUS["BAD_PARAM"], api.STATUS["UNSUPPORTED_DATATYPE"]
    assert status() == api.STATUS["SUCCESS"]
    assert status(x=P(ctx, (4, 256), "float64")) == dtype and status(gamma=P(ctx, (256,), "bfloat16")) == dtype
    assert status(y=P(ctx, (4, 256), "bfloat16")) == dtype and status(scale=P(ctx, (4, 2), "float64")) == dtype
    assert status(gamma=P(ctx, (255,), "float32")) == bad and status(gamma=P(ctx, (1, 256), "float32")) == bad
    assert status(scale=P(ctx, (1, 2), "float32")) == bad and status(scale=P(ctx, (4, 3), "float32")) == bad
    assert status(y=P(ctx, (2, 512), "float8_e4m3")) == bad
    for epsilon in (0.0, -1e-6, float("nan"), float("inf"), 1e-60):
        assert status(epsilon=epsilon) == bad, epsilon
    short = P(ctx, (3, 256), "bfloat16")
    assert status(z=short) == bad and status(h=short) == bad  # memory for three rows only
    shifted = P(ctx, (4, 256), "bfloat16")
    shifted.mem = base["x"].block.view(4 * 256 * 2, bs.Placed.GUARD + 16)
    assert status(h=shifted) == bad
    over_h = P(ctx, (4, 256), "float8_e4m3")
    over_h.mem = base["h"].block.view(4 * 256, bs.Placed.GUARD)
    assert status(y=over_h) == bad
    long = P(ctx, (1, (1 << 20) + 8), "bfloat16")
    assert status(x=long, z=None, h=None, gamma=P(ctx, long.shape[1:], "float32"), y=P(ctx, long.shape, "float8_e4m3"),
                  scale=P(ctx, (1, 8193), "float32")) == api.STATUS["NOT_SUPPORTED"]
    assert base["h"].guards_intact() and base["y"].guards_intact() and base["scale"].guards_intact()


def test_offsets_past_32_bits(ctx):
    rows, c = 1100003, 2056
    desc = api.TensorDescriptor((rows, c), "bfloat16")
    y_desc, s_desc, g_desc = api.TensorDescriptor((rows, c), "float8_e4m3"), api.TensorDescriptor((rows, bs.blocks(c)), "float32"), api.TensorDescriptor((c,), "float32")
    x, h, y, s, g = (api.Memory(d.nbytes) for d in (desc, desc, y_desc, s_desc, g_desc))
    x.zero(ctx)
    x0, _, g0 = inputs((32, c), 86)
    stored, x64 = api.to_storage(x0, "bfloat16")
    gamma, g64 = api.to_storage(g0, "float32")
    g.from_host(ctx, gamma)
    for first in (0, rows - 32):
        x.from_host(ctx, stored, first * c * 2)
    api.call("cudaRmsNormQuantize", ctx.handle, desc.handle, x.handle, x.handle, h.handle, g_desc.handle, g.handle, ctypes.c_double(EPSILON), y_desc.handle,
             y.handle, s_desc.handle, s.handle)
    h64, y64 = o.rms_norm(x64, x64, g64, EPSILON)
    for first in (0, rows - 32):
        got_h = h.to_host(ctx, np.empty((32, c), dtype=np.uint16), first * c * 2)
        got_y = y.to_host(ctx, np.empty((32, c), dtype=np.uint8), first * c)
        got_s = s.to_host(ctx, np.empty((32, bs.blocks(c)), dtype=np.float32), first * bs.blocks(c) * 4)
        ctx.synchronize()
        spread = o.spread_scales(got_s, 32, c)
        assert np.array_equal(api.bfloat16_bits_to_float(got_h), h64)  # x + x is a bfloat16 number
        assert np.all(np.abs(api.float8_bits_to_float(got_y) * spread - y64) <= bs.code_error_bound(y64, spread, norm_bound(c) + 2 * bs.U32))


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("columns", [1, 136, 264, 520, 8192, 33000])
def test_sums_of_squares_up_to_float32s_end_and_past_it(ctx, dtype, columns):
    """rows of +-2^e whose sum of squares is the last one below 2^128, and rows whose sum passes it: these give zeros, and their h"""
    e = int(np.floor((127.99 - np.log2(columns)) / 2))
    r = np.random.default_rng(87)
    shape = (6, columns)
    x0 = np.where(r.random(shape) < 0.5, -1.0, 1.0) * np.exp2([[e], [e + 1], [0.0], [e], [e + 1], [60.0 + 60.0]])
    x, h = bs.Placed(ctx, shape, dtype, values=x0), bs.Placed(ctx, shape, dtype)
    gamma = bs.Placed(ctx, (columns,), "float32", values=1 + 0.2 * r.normal(0, 1, columns))
    y, s = bs.Placed(ctx, shape, "float8_e4m3"), bs.Placed(ctx, (6, bs.blocks(columns)), "float32")
    bs.rms_norm_quantize(ctx, x, None, h, gamma, EPSILON, y, s)
    assert np.array_equal(h.download(), x0) and y.guards_intact() and s.guards_intact()
    q, scales = y.download(), s.download()
    past, keep = [1, 4, 5], [0, 2, 3]
    assert np.all(q[past] == 0.0) and np.all(scales[past] == np.float32(2.0 ** -100) / np.float32(448))
    _, y64 = o.rms_norm(x0[keep], None, gamma.values, EPSILON)
    spread = o.spread_scales(scales[keep], 3, columns)
    assert np.all(np.abs(q[keep] * spread - y64) <= bs.code_error_bound(y64, spread, norm_bound(columns) + 2 * bs.U32))


# Rows enough to fill the machine with a half-warp (or two) per row of two to four blocks, so that different rows share a warp's
# shuffles and the joint maxima; the last thread block has rows past the end.  333 and 131 columns take the path of single elements.
MANY_ROWS = [(4801, 264), (4737, 136), (5003, 512), (4999, 333), (6001, 131), (9475, 264), (2371, 1024), (3001, 640), (2500, 900),
             (3001, 264), (4700, 448), (2999, 250)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("shape", MANY_ROWS)
def test_many_short_rows(ctx, dtype, residual, shape):
    x0, z0, g0 = inputs(shape, 88)
    x = bs.Placed(ctx, shape, dtype, values=x0)
    z = bs.Placed(ctx, shape, dtype, values=z0) if residual else None
    h = bs.Placed(ctx, shape, dtype) if residual else None
    gamma = bs.Placed(ctx, (shape[1],), "float32", values=g0)
    y, s = bs.Placed(ctx, shape, "float8_e4m3"), bs.Placed(ctx, (shape[0], bs.blocks(shape[1])), "float32")
    bs.rms_norm_quantize(ctx, x, z, h, gamma, EPSILON, y, s)
    check(x.values, z.values if residual else None, gamma.values, h, y, s, dtype)
    assert np.array_equal(x.download(), x.values)


@pytest.mark.parametrize("offsets", [(2, 0, 0, 0, 0), (0, 4, 0, 0, 0), (0, 0, 8, 0, 0), (0, 0, 0, 4, 0), (0, 0, 0, 0, 3)])
def test_many_short_rows_in_unaligned_views(ctx, offsets):
    shape = (4801, 264)
    x0, z0, g0 = inputs(shape, 89)
    x, z = bs.Placed(ctx, shape, "bfloat16", offsets[0], values=x0), bs.Placed(ctx, shape, "bfloat16", offsets[1], values=z0)
    h, gamma = bs.Placed(ctx, shape, "bfloat16", offsets[2]), bs.Placed(ctx, (shape[1],), "float32", offsets[3], values=g0)
    y, s = bs.Placed(ctx, shape, "float8_e4m3", offsets[4]), bs.Placed(ctx, (shape[0], 3), "float32", 4)
    bs.rms_norm_quantize(ctx, x, z, h, gamma, EPSILON, y, s)
    check(x.values, z.values, gamma.values, h, y, s, "bfloat16")


def test_nan_and_infinity_among_many_short_rows(ctx):
    """a row's NaN does not reach its neighbours in the same warp, whichever half of it they are in"""
    shape = (4801, 264)
    x0, _, g0 = inputs(shape, 90)
    bad = np.array([0, 1, 6, 33, 4799, 4800])
    x0[bad, [0, 263, 130, 255, 8, 256]] = [np.nan, np.nan, np.inf, -np.inf, np.nan, np.inf]
    x = bs.Placed(ctx, shape, "float16", values=x0)
    gamma = bs.Placed(ctx, (264,), "float32", values=g0)
    y, s = bs.Placed(ctx, shape, "float8_e4m3"), bs.Placed(ctx, (4801, 3), "float32")
    bs.rms_norm_quantize(ctx, x, None, None, gamma, EPSILON, y, s)
    q, scales = y.download(), s.download()
    assert np.all(np.any(np.isnan(q[bad]), axis=1))
    keep = np.setdiff1d(np.arange(4801), bad)
    _, y64 = o.rms_norm(x.values[keep], None, gamma.values, EPSILON)
    spread = o.spread_scales(scales[keep], len(keep), 264)
    assert np.all(np.abs(q[keep] * spread - y64) <= bs.code_error_bound(y64, spread, norm_bound(264) + 2 * bs.U32))
    assert y.guards_intact() and s.guards_intact()
