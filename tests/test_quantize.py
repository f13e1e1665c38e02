"""cudaQuantizeBlocks against its formula: codes bit for bit in float32, code * scale against the input in float64."""
import numpy as np
import pytest

from cudabackend_b200 import api
from oracle import oracle as o
from tests import block_scaled as bs

pytestmark = pytest.mark.gpu

SHAPES = [(1, 1), (1, 128), (1, 4096), (3, 127), (5, 129), (2, 1001), (17, 8), (128, 128), (127, 384), (129, 264), (300, 1000), (257, 2048), (1000, 72)]
DTYPES = ["float16", "bfloat16", "float32"]


def scale_shape(rows, c, square):
    return (bs.blocks(rows) if square else rows, bs.blocks(c))


def expected(x64, height):
    """(codes, scales) of the formula evaluated in float32"""
    rows, c = x64.shape
    x = x64.astype(np.float32)
    amax = (o.block_scales(x64, height) * 448.0).astype(np.float32)  # max(amax, 2^-100): a float32 number, divided and multiplied in float64
    scales = amax / np.float32(448)
    spread = np.repeat(np.repeat(np.float32(448) / amax, height, axis=0)[:rows], 128, axis=1)[:, :c]
    return api.float_to_float8_bits(x * spread), scales


def inputs(shape, seed):
    r = np.random.default_rng(seed)
    x = r.normal(0, 1, shape) * np.exp2(r.integers(-6, 7, (shape[0], 1)))
    x[r.random(shape) < 0.1] = 0.0
    return x


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("square", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_codes_and_scales(ctx, dtype, square, shape):
    x = bs.Placed(ctx, shape, dtype, values=inputs(shape, 71))
    y = bs.Placed(ctx, shape, "float8_e4m3")
    s = bs.Placed(ctx, scale_shape(*shape, square), "float32")
    bs.quantize(ctx, x, y, s)
    height = 128 if square else 1
    codes, scales = expected(x.values, height)
    assert np.array_equal(s.raw(), scales)
    assert np.array_equal(y.raw(), codes)
    spread = o.spread_scales(s.download(), *shape, height)
    assert np.all(np.abs(y.download() * spread - x.values) <= bs.code_error_bound(x.values, spread, 2 * bs.U32))
    assert y.guards_intact() and s.guards_intact() and x.guards_intact()


@pytest.mark.parametrize("square", [False, True])
@pytest.mark.parametrize("x_offset,y_offset", [(2, 0), (4, 0), (8, 0), (0, 1), (0, 4), (6, 3)])
def test_unaligned_views(ctx, square, x_offset, y_offset):
    shape = (131, 264)
    x = bs.Placed(ctx, shape, "bfloat16", x_offset, values=inputs(shape, 72))
    y = bs.Placed(ctx, shape, "float8_e4m3", y_offset)
    s = bs.Placed(ctx, scale_shape(*shape, square), "float32", 4)
    bs.quantize(ctx, x, y, s)
    codes, scales = expected(x.values, 128 if square else 1)
    assert np.array_equal(s.raw(), scales) and np.array_equal(y.raw(), codes)
    assert y.guards_intact() and s.guards_intact()


@pytest.mark.parametrize("square", [False, True])
def test_zeros_tiny_values_nan_and_infinity(ctx, square):
    shape = (256, 512)
    x0 = inputs(shape, 73)
    x0[:128, :128] = 0.0
    x0[:128, 128:256] = 2.0 ** -120
    x0[5, 300], x0[200, 400] = np.nan, -np.inf
    x = bs.Placed(ctx, shape, "float32", values=x0)
    y = bs.Placed(ctx, shape, "float8_e4m3")
    s = bs.Placed(ctx, scale_shape(*shape, square), "float32")
    bs.quantize(ctx, x, y, s)
    height = 128 if square else 1
    q, spread = y.download(), o.spread_scales(s.download(), *shape, height)
    least = np.float32(2.0 ** -100) / np.float32(448)
    assert np.all(q[:128, :128] == 0) and np.all(spread[:128, :256] == least)
    assert np.all(q[:128, 128:256] == o.e4m3_round(448.0 * 2.0 ** -20))
    nan_rows, inf_rows = (slice(0, 128), slice(128, 256)) if square else (slice(5, 6), slice(200, 201))
    assert np.all(np.isnan(q[nan_rows, 256:384])) and np.all(np.isnan(spread[nan_rows, 256:384]))
    block = q[inf_rows, 384:512].copy()
    assert np.all(np.isposinf(spread[inf_rows, 384:512]))
    assert np.isnan(q[200, 400])
    block[200 - inf_rows.start, 400 - 384] = 0
    assert np.all(block == 0)
    bad = np.zeros(shape, dtype=bool)
    bad[nan_rows, 256:384] = True
    bad[inf_rows, 384:512] = True
    bad[:128, :256] = True
    error = np.abs(q * np.where(bad, 0, spread) - np.where(bad, 0, x.values))
    assert np.all(error[~bad] <= bs.code_error_bound(x.values, spread, 2 * bs.U32)[~bad])


def test_ranks_and_empty_tensors(ctx):
    shape = (2, 3, 5, 200)
    x = bs.Placed(ctx, shape, "float16", values=inputs((30, 200), 74))
    y = bs.Placed(ctx, shape, "float8_e4m3")
    s = bs.Placed(ctx, (2, 3, 5, 2), "float32")
    bs.quantize(ctx, x, y, s)
    codes, scales = expected(x.values.reshape(30, 200), 1)
    assert np.array_equal(y.raw().reshape(30, 200), codes) and np.array_equal(s.raw().reshape(30, 2), scales)
    line = bs.Placed(ctx, (200,), "float16", values=x.values[0, 0, 0])
    line_y, line_s = bs.Placed(ctx, (200,), "float8_e4m3"), bs.Placed(ctx, (2,), "float32")
    bs.quantize(ctx, line, line_y, line_s)
    assert np.array_equal(line_y.raw(), codes[0]) and np.array_equal(line_s.raw(), scales[0])
    for empty in ((0, 200), (4, 0)):
        e = bs.Placed(ctx, empty, "float16")
        ey, es = bs.Placed(ctx, empty, "float8_e4m3"), bs.Placed(ctx, scale_shape(*empty, False), "float32")
        bs.quantize(ctx, e, ey, es)
        assert ey.guards_intact() and es.guards_intact()


def test_refusals(ctx):
    P = bs.Placed
    x, y, s = P(ctx, (200, 256), "bfloat16"), P(ctx, (200, 256), "float8_e4m3"), P(ctx, (200, 2), "float32")

    def status(x=x, y=y, s=s):
        return bs.quantize(ctx, x, y, s, status=True)

    assert status() == api.STATUS["SUCCESS"]
    assert status(x=P(ctx, (200, 256), "int8")) == api.STATUS["UNSUPPORTED_DATATYPE"]
    assert status(x=P(ctx, (200, 256), "float64")) == api.STATUS["UNSUPPORTED_DATATYPE"]
    assert status(y=P(ctx, (200, 256), "int8")) == api.STATUS["UNSUPPORTED_DATATYPE"]
    assert status(s=P(ctx, (200, 2), "float16")) == api.STATUS["UNSUPPORTED_DATATYPE"]
    assert status(y=P(ctx, (256, 200), "float8_e4m3")) == api.STATUS["BAD_PARAM"]
    assert status(y=P(ctx, (51200,), "float8_e4m3")) == api.STATUS["BAD_PARAM"]
    for shape in ((200, 3), (199, 2), (3, 2), (1, 2), (400,), (2, 200)):
        assert status(s=P(ctx, shape, "float32")) == api.STATUS["BAD_PARAM"], shape
    small = P(ctx, (200, 256), "float8_e4m3")
    small.mem = small.block.view(200 * 256 - 1, 0)
    assert status(y=small) == api.STATUS["BAD_PARAM"]
    odd = P(ctx, (200, 256), "bfloat16")
    odd.mem = odd.block.view(200 * 256 * 2, 1)  # off the element's boundary
    assert status(x=odd) == api.STATUS["BAD_PARAM"]
    over = P(ctx, (200, 256), "float8_e4m3")
    over.mem = x.block.view(200 * 256, 200)  # inside x
    assert status(y=over) == api.STATUS["BAD_PARAM"]
    negative = P(ctx, (200, 256), "bfloat16")
    dims = (api._INT * 2)(-200, 256)
    api.call("cudaSetTensorDescriptor", negative.desc.handle, api.DTYPES["bfloat16"], 2, dims)
    assert status(x=negative) == api.STATUS["BAD_PARAM"]
    wide = P(ctx, (1, 8), "bfloat16")
    api.call("cudaSetTensorDescriptor", wide.desc.handle, api.DTYPES["bfloat16"], 8, (api._INT * 8)(*([2 ** 31 - 1] * 8)))
    assert status(x=wide) == api.STATUS["BAD_PARAM"]
    assert x.guards_intact() and y.guards_intact() and s.guards_intact()


def test_offsets_past_32_bits(ctx):
    """more than 2^32 bytes of input and 2^31 codes: the first and the last rows are where 32-bit offsets would miss them"""
    rows, c = 1100003, 2056
    x_desc, y_desc, s_desc = api.TensorDescriptor((rows, c), "bfloat16"), api.TensorDescriptor((rows, c), "float8_e4m3"), api.TensorDescriptor((rows, bs.blocks(c)), "float32")
    square_desc = api.TensorDescriptor((bs.blocks(rows), bs.blocks(c)), "float32")
    x, y, s = api.Memory(x_desc.nbytes), api.Memory(y_desc.nbytes), api.Memory(s_desc.nbytes)
    x.zero(ctx)
    edge = inputs((64, c), 75)
    stored, values = api.to_storage(edge, "bfloat16")
    for first in (0, rows - 64):
        x.from_host(ctx, stored, first * c * 2)
    for desc, height, keep in ((s_desc, 1, 64), (square_desc, 128, 1)):
        api.call("cudaQuantizeBlocks", ctx.handle, x_desc.handle, x.handle, y_desc.handle, y.handle, desc.handle, s.handle)
        codes, scales = expected(values, height)
        for first in (0, rows - 64):
            got = y.to_host(ctx, np.empty((64, c), dtype=np.uint8), first * c)
            at = (first // height) * bs.blocks(c) * 4
            got_s = s.to_host(ctx, np.empty((keep, bs.blocks(c)), dtype=np.float32), at)
            ctx.synchronize()
            if height == 1 or first == 0:
                assert np.array_equal(got_s, scales) and np.array_equal(got, codes)
            else:  # the last square starts at a multiple of 128: the 64 rows may reach into the one before it
                split = rows // 128 * 128 - first
                tail, tail_scales = expected(values[max(split, 0):], 128)
                last = s.to_host(ctx, np.empty((1, bs.blocks(c)), dtype=np.float32), (rows // 128) * bs.blocks(c) * 4)
                ctx.synchronize()
                assert np.array_equal(last, tail_scales) and np.array_equal(got[max(split, 0):], tail)
