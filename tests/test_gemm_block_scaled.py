"""cudaGemmBlockScaled against the formula in float64."""
import numpy as np
import pytest

from cudabackend_b200 import api
from oracle import oracle as o
from tests import block_scaled as bs

pytestmark = pytest.mark.gpu

# (M, N, K): one token and small batches, tile edges on both sides, short last blocks of K, several tiles and blocks of every kernel
SHAPES = [(1, 1, 16), (1, 128, 128), (1, 257, 384), (2, 64, 16), (7, 130, 144), (1, 4096, 2048), (16, 128, 1008), (17, 129, 256), (33, 200, 2048),
          (64, 512, 640), (65, 384, 128), (128, 128, 4096), (129, 127, 112), (130, 513, 272), (255, 256, 512), (300, 520, 1040), (1000, 264, 2304),
          (257, 512, 128), (513, 1024, 384), (2100, 1300, 1280), (4100, 256, 576), (3000, 2056, 272)]
# row pitches that are no multiple of 16 bytes
ODD_SHAPES = [(1, 1, 1), (1, 300, 77), (5, 70, 33), (64, 64, 7), (130, 140, 129), (200, 300, 517), (33, 257, 260), (300, 129, 1002), (513, 520, 264), (1, 1024, 4095)]


class Problem:
    def __init__(self, ctx, m, n, k, dtype, seed=91, a_offset=0, b_offset=0, c_offset=0, c_values=None):
        r = np.random.default_rng(seed)
        self.ctx, self.k, self.dtype = ctx, k, dtype
        self.a = bs.Placed(ctx, (m, k), "float8_e4m3", a_offset, bs.random_codes(r, m, k))
        self.b = bs.Placed(ctx, (n, k), "float8_e4m3", b_offset, bs.random_codes(r, n, k))
        # scales over several powers of two, so that one applied to the wrong block shows
        self.sa = bs.Placed(ctx, (m, bs.blocks(k)), "float32", 4, np.exp2(r.uniform(-9, -3, (m, bs.blocks(k)))))
        self.sb = bs.Placed(ctx, (bs.blocks(n), bs.blocks(k)), "float32", 8, np.exp2(r.uniform(-9, -3, (bs.blocks(n), bs.blocks(k)))))
        self.c = bs.Placed(ctx, (m, n), dtype, c_offset, r.normal(0, 1, (m, n)) if c_values is None else c_values)

    def run(self, alpha=None, beta=None):
        bs.gemm(self.ctx, self.a, self.sa, self.b, self.sb, self.c, alpha, beta)

    def expected(self, alpha=1.0, beta=0.0):
        f = lambda v: float(np.float32(v))
        return o.gemm_block_scaled(self.a.values, self.sa.values, self.b.values, self.sb.values, f(alpha), f(beta), self.c.values)

    def check(self, alpha=1.0, beta=0.0):
        ref, size = self.expected(alpha, beta)
        got = self.c.download()
        assert np.all(np.abs(got - ref) <= bs.gemm_error_bound(ref, size, self.k, self.dtype))
        assert self.c.guards_intact()
        return got


@pytest.mark.parametrize("dtype", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("shape", SHAPES)
def test_products(ctx, dtype, shape):
    p = Problem(ctx, *shape, dtype)
    p.run()
    p.check()


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("shape", ODD_SHAPES)
def test_odd_row_pitches(ctx, dtype, shape):
    p = Problem(ctx, *shape, dtype)
    p.run()
    p.check()


# enough tiles of 256 x 256 for the CTA-pair kernel: ragged rows and columns, C pitches that no bulk copy takes, one block of K
PAIR_SHAPES = [(2049, 1025, 272), (1500, 1501, 144), (8200, 130, 256), (257, 8004, 400), (5000, 520, 16), (2300, 2302, 1024)]


@pytest.mark.parametrize("dtype", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("shape", PAIR_SHAPES)
@pytest.mark.parametrize("alpha,beta", [(1.0, 0.0), (-0.6, 0.7)])
def test_many_rows_on_both_sides(ctx, dtype, shape, alpha, beta):
    p = Problem(ctx, *shape, dtype, c_offset=4 if shape[1] == 8004 else 0)
    p.run(alpha, beta)
    p.check(alpha, beta)


@pytest.mark.parametrize("k", [128, 256, 384, 1408])
def test_exact_on_large_tiles(ctx, k):
    """integers and powers of two through the CTA-pair kernel: even and odd numbers of blocks per tile"""
    m, n = 3333, 1100
    p = Problem(ctx, m, n, k, "float32")
    r = np.random.default_rng(94)
    p.a.upload(r.integers(-8, 9, (m, k)))
    p.b.upload(r.integers(-8, 9, (n, k)))
    p.sa.upload(np.exp2(r.integers(-2, 2, (m, bs.blocks(k)))))
    p.sb.upload(np.exp2(r.integers(-2, 2, (bs.blocks(n), bs.blocks(k)))))
    for _ in range(2):
        p.run()
        assert np.array_equal(p.c.download(), p.expected()[0])


@pytest.mark.parametrize("a_offset,b_offset,c_offset", [(1, 0, 0), (0, 2, 0), (4, 4, 0), (8, 0, 2), (0, 8, 4), (0, 0, 2), (0, 0, 8), (16, 32, 16)])
@pytest.mark.parametrize("shape", [(3, 264, 256), (140, 300, 272), (600, 512, 256)])
def test_unaligned_views(ctx, a_offset, b_offset, c_offset, shape):
    p = Problem(ctx, *shape, "bfloat16", a_offset=a_offset, b_offset=b_offset, c_offset=c_offset)
    p.run()
    p.check()


@pytest.mark.parametrize("shape", [(1, 300, 256), (40, 128, 384), (100, 300, 1000), (130, 257, 528), (1111, 1032, 640), (1000, 300, 77)])
def test_small_integers_are_exact(ctx, shape):
    """codes that are integers up to 8 and scales that are powers of two: every partial sum is a float32 number, whatever the order"""
    m, n, k = shape
    p = Problem(ctx, m, n, k, "float32")
    r = np.random.default_rng(92)
    p.a.upload(r.integers(-8, 9, (m, k)))
    p.b.upload(r.integers(-8, 9, (n, k)))
    p.sa.upload(np.exp2(r.integers(-2, 2, (m, bs.blocks(k)))))
    p.sb.upload(np.exp2(r.integers(-2, 2, (bs.blocks(n), bs.blocks(k)))))
    p.run()
    assert np.array_equal(p.c.download(), p.expected()[0])


@pytest.mark.parametrize("dtype", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("shape", [(5, 136, 272), (200, 300, 512), (700, 520, 256), (33, 130, 77)])
def test_alpha_and_beta(ctx, dtype, shape):
    p = Problem(ctx, *shape, dtype)
    p.run(0.37, -1.25)
    p.check(0.37, -1.25)


@pytest.mark.parametrize("shape", [(3, 256, 256), (130, 128, 128), (600, 300, 256)])
def test_c_is_not_read_without_beta(ctx, shape):
    m, n, _ = shape
    p = Problem(ctx, *shape, "float32", c_values=np.full((m, n), np.nan))
    p.run(2.0, 0.0)
    ref, size = o.gemm_block_scaled(p.a.values, p.sa.values, p.b.values, p.sb.values, 2.0)
    assert np.all(np.abs(p.c.download() - ref) <= bs.gemm_error_bound(ref, size, p.k, "float32"))


@pytest.mark.parametrize("shape", [(20, 300, 384), (150, 300, 384), (600, 512, 384)])
def test_nan_and_infinity_stay_in_their_rows(ctx, shape):
    m, n, k = shape
    p = Problem(ctx, m, n, k, "float32")
    a = p.a.values.copy()
    a[3, 200] = np.nan
    p.a.upload(a)
    sa = p.sa.values.copy()
    sa[7, 2], sa[11, 0] = np.nan, np.inf
    p.sa.upload(sa)
    p.run()
    got = p.c.download()
    assert np.all(np.isnan(got[[3, 7]])) and not np.any(np.isfinite(got[11]))
    keep = np.setdiff1d(np.arange(m), [3, 7, 11])
    ref, size = o.gemm_block_scaled(p.a.values[keep], p.sa.values[keep], p.b.values, p.sb.values)
    assert np.all(np.abs(got[keep] - ref) <= bs.gemm_error_bound(ref, size, k, "float32"))


@pytest.mark.parametrize("shape", [(16, 4096, 4096), (100, 520, 2048), (2000, 1032, 1024), (65, 200, 999)])
def test_same_bits_every_time(ctx, shape):
    p = Problem(ctx, *shape, "float32")
    p.run()
    first = p.c.raw().copy()
    for _ in range(3):
        p.run()
        assert np.array_equal(first.view(np.uint32), p.c.raw().view(np.uint32))


def test_rows_do_not_depend_on_the_batch_they_are_in_within_a_kernel(ctx):
    """rows 0..7 of a batch of 8 and of 13: the same kernel and split, so the same bits"""
    p = Problem(ctx, 13, 1024, 2048, "float32")
    p.run()
    whole = p.c.download()
    q = Problem(ctx, 8, 1024, 2048, "float32")
    q.a.upload(p.a.values[:8])
    q.sa.upload(p.sa.values[:8])
    q.b.upload(p.b.values)
    q.sb.upload(p.sb.values)
    q.run()
    assert np.array_equal(q.c.download(), whole[:8])


@pytest.mark.parametrize("shape", [(0, 5, 128), (5, 0, 128)])
def test_no_rows_or_columns(ctx, shape):
    m, n, k = shape
    a, b, c = bs.Placed(ctx, (m, k), "float8_e4m3"), bs.Placed(ctx, (n, k), "float8_e4m3"), bs.Placed(ctx, (m, n), "float32")
    sa, sb = bs.Placed(ctx, (m, 1), "float32"), bs.Placed(ctx, (bs.blocks(n), 1), "float32")
    bs.gemm(ctx, a, sa, b, sb, c)
    assert c.guards_intact()


@pytest.mark.parametrize("dtype", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("shape", [(1, 1), (3, 5), (300, 257)])
def test_an_empty_sum(ctx, dtype, shape):
    """K = 0: C = beta * C"""
    m, n = shape
    a, b, c = bs.Placed(ctx, (m, 0), "float8_e4m3"), bs.Placed(ctx, (n, 0), "float8_e4m3"), bs.Placed(ctx, (m, n), dtype, values=np.full((m, n), 3.0))
    sa, sb = bs.Placed(ctx, (m, 0), "float32"), bs.Placed(ctx, (bs.blocks(n), 0), "float32")
    bs.gemm(ctx, a, sa, b, sb, c, beta=0.5)
    assert np.all(c.download() == 1.5) and c.guards_intact()
    bs.gemm(ctx, a, sa, b, sb, c)
    assert np.all(c.download() == 0.0) and c.guards_intact()


def test_refusals(ctx):
    P = bs.Placed
    base = {"a": P(ctx, (40, 300), "float8_e4m3"), "a_scale": P(ctx, (40, 3), "float32"), "b": P(ctx, (200, 300), "float8_e4m3"),
            "b_scale": P(ctx, (2, 3), "float32"), "c": P(ctx, (40, 200), "bfloat16")}
    for name in ("a", "b", "a_scale", "b_scale"):
        base[name].upload(np.zeros(base[name].shape))

    def status(**change):
        return bs.gemm(ctx, status=True, **{**base, **change})

    bad, dtype = api.STATUS["BAD_PARAM"], api.STATUS["UNSUPPORTED_DATATYPE"]
    assert status() == api.STATUS["SUCCESS"]
    for ops in ((0, 0), (1, 1), (1, 0)):
        assert status(ops=ops) == api.STATUS["NOT_SUPPORTED"]
    assert status(a=P(ctx, (40, 300), "int8")) == dtype and status(b=P(ctx, (200, 300), "bfloat16")) == dtype
    assert status(c=P(ctx, (40, 200), "float64")) == dtype and status(c=P(ctx, (40, 200), "int32")) == dtype
    assert status(a_scale=P(ctx, (40, 3), "float16")) == dtype and status(b_scale=P(ctx, (2, 3), "float64")) == dtype
    assert status(a=P(ctx, (40, 299), "float8_e4m3")) == bad and status(b=P(ctx, (200, 301), "float8_e4m3")) == bad
    assert status(c=P(ctx, (200, 40), "bfloat16")) == bad and status(c=P(ctx, (1, 40, 200), "bfloat16")) == bad
    for shape in ((40, 2), (1, 3), (120,), (3, 40)):
        assert status(a_scale=P(ctx, shape, "float32")) == bad, shape
    for shape in ((200, 3), (2, 2), (1, 3), (3, 2)):
        assert status(b_scale=P(ctx, shape, "float32")) == bad, shape
    short = P(ctx, (200, 300), "float8_e4m3")
    short.mem = short.block.view(200 * 300 - 1, 0)
    assert status(b=short) == bad
    over = P(ctx, (40, 200), "bfloat16")
    over.mem = base["b"].block.view(40 * 200 * 2, 100)
    assert status(c=over) == bad
    off = P(ctx, (40, 200), "bfloat16")
    off.mem = off.block.view(40 * 200 * 2, 1)
    assert status(c=off) == bad
    huge = P(ctx, (1, 1), "float8_e4m3")
    api.call("cudaSetTensorDescriptor", huge.desc.handle, api.DTYPES["float8_e4m3"], 2, (api._INT * 2)(2 ** 31 - 1, 2 ** 31 - 1))
    assert status(a=huge) == bad
    assert base["c"].guards_intact()


@pytest.mark.parametrize("n,k", [(2056, 2048), (4, 2050)])
def test_offsets_past_32_bits(ctx, n, k):
    """A of more than 2^31 bytes and, in the first case, C of more than 2^31 elements (2^32 bytes)"""
    m = 1100003
    a_desc, c_desc = api.TensorDescriptor((m, k), "float8_e4m3"), api.TensorDescriptor((m, n), "bfloat16")
    sa_desc = api.TensorDescriptor((m, bs.blocks(k)), "float32")
    a, c, sa = api.Memory(a_desc.nbytes), api.Memory(c_desc.nbytes), api.Memory(sa_desc.nbytes)
    a.zero(ctx), sa.zero(ctx)
    r = np.random.default_rng(93)
    keep = 64
    codes, a64 = api.to_storage(bs.random_codes(r, keep, k), "float8_e4m3")
    scales, sa64 = api.to_storage(np.exp2(r.uniform(-9, -3, (keep, bs.blocks(k)))), "float32")
    for first in (0, m - keep):
        a.from_host(ctx, codes, first * k)
        sa.from_host(ctx, scales, first * bs.blocks(k) * 4)
    b = bs.Placed(ctx, (n, k), "float8_e4m3", values=bs.random_codes(r, n, k))
    sb = bs.Placed(ctx, (bs.blocks(n), bs.blocks(k)), "float32", values=np.exp2(r.uniform(-9, -3, (bs.blocks(n), bs.blocks(k)))))
    api.call("cudaGemmBlockScaled", ctx.handle, api.GEMM_N, api.GEMM_T, None, a_desc.handle, a.handle, sa_desc.handle, sa.handle, b.desc.handle, b.mem.handle,
             sb.desc.handle, sb.mem.handle, None, c_desc.handle, c.handle)
    ref, size = o.gemm_block_scaled(a64, sa64, b.values, sb.values)
    for first in (0, m - keep):
        got = c.to_host(ctx, np.empty((keep, n), dtype=np.uint16), first * n * 2)
        ctx.synchronize()
        assert np.all(np.abs(api.bfloat16_bits_to_float(got) - ref) <= bs.gemm_error_bound(ref, size, k, "bfloat16"))


def test_the_other_calls_refuse_the_type(ctx):
    """entry points that compute with elements know nothing of e4m3; cudaIm2Row, which only moves them, is tested with the chain"""
    dtype = api.STATUS["UNSUPPORTED_DATATYPE"]
    a, b, c = (bs.Placed(ctx, (32, 32), "float8_e4m3") for _ in range(3))
    args = (a.desc.handle, a.mem.handle, b.desc.handle, b.mem.handle, None, c.desc.handle, c.mem.handle)
    assert api.call_status("cudaGemm", ctx.handle, 0, 1, None, *args) == dtype
    a3, b3, c3 = (bs.Placed(ctx, (1, 32, 32), "float8_e4m3") for _ in range(3))
    args = (a3.desc.handle, a3.mem.handle, b3.desc.handle, b3.mem.handle, None, c3.desc.handle, c3.mem.handle)
    assert api.call_status("cudaGemmBatched", ctx.handle, 0, 1, None, *args) == dtype
    f = bs.Placed(ctx, (32, 32), "float32")
    args = (a.desc.handle, a.mem.handle, b.desc.handle, b.mem.handle, None, f.desc.handle, f.mem.handle)
    assert api.call_status("cudaGemm", ctx.handle, 0, 1, None, *args) == dtype
    assert api.call_status("cudaActivationForward", ctx.handle, 3, None, a.desc.handle, a.mem.handle, None, b.desc.handle, b.mem.handle) == dtype
    bias = bs.Placed(ctx, (32,), "float32")
    assert api.call_status("cudaAddBias", ctx.handle, None, None, a.desc.handle, a.mem.handle, bias.desc.handle, bias.mem.handle, b.desc.handle, b.mem.handle,
                           None, None, None, api.INVALID, 0) == dtype
    conv = api.ConvolutionDescriptor(api.CONVOLUTION_MODE, (-1, -1))
    x, w, y = bs.Placed(ctx, (1, 8, 8, 16), "float8_e4m3"), bs.Placed(ctx, (16, 3, 3, 16), "float8_e4m3"), bs.Placed(ctx, (1, 8, 8, 16), "float8_e4m3")
    for entry in ("cudaConvolutionImplicitGemmForward", "cudaConvolutionWinogradFusedForward"):
        status = api.call_status(entry, ctx.handle, conv.handle, None, x.desc.handle, x.mem.handle, w.desc.handle, w.mem.handle, api.INVALID, api.INVALID, None,
                                 api.INVALID, api.INVALID, None, y.desc.handle, y.mem.handle, 0)
        assert status in (dtype, api.STATUS["NOT_SUPPORTED"]), entry
    for t in (a, b, c, c3, f, y):
        assert np.all(t.raw().view(np.uint8) == 0x5A) and t.guards_intact()


# More tiles than CTA pairs, so that a pair stores one tile behind another, with next to no contraction in between, and last columns
# that leave a warp with one or three sub-tiles of C (64 16-bit or 32 float32 columns): both staging buffers are the next tile's.
@pytest.mark.parametrize("dtype", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("alpha,beta", [(1.0, 0.0), (-0.6, 0.7)])
@pytest.mark.parametrize("shape", [(20000, 520, 16), (20000, 328, 128), (12000, 1032, 128)])
def test_ragged_columns_over_many_tiles(ctx, dtype, alpha, beta, shape):
    p = Problem(ctx, *shape, dtype)
    p.run(alpha, beta)
    p.check(alpha, beta)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_ragged_columns_over_many_tiles_have_the_same_bits_every_time(ctx, dtype):
    p = Problem(ctx, 20000, 520, 16, dtype)
    p.run()
    first = p.c.raw().copy()
    for _ in range(20):
        p.run()
        assert np.array_equal(first.view(np.uint8), p.c.raw().view(np.uint8))


@pytest.mark.parametrize("shape", [(1, 520, 8192), (32, 1032, 8192), (64, 520, 8192), (128, 264, 8192), (50, 392, 8190), (2100, 1032, 8192)])
def test_every_block_meets_its_own_scale(ctx, shape):
    """64 blocks of K whose scales are all different from their neighbours', over and over: integers below 2^22, so any mix-up shows"""
    m, n, k = shape
    p = Problem(ctx, m, n, k, "float32")
    r = np.random.default_rng(95)
    p.a.upload(r.integers(-2, 3, (m, k)))
    p.b.upload(r.integers(-2, 3, (n, k)))
    g = np.arange(bs.blocks(k))
    p.sa.upload(np.exp2((g[None, :] + np.arange(m)[:, None]) % 4))
    p.sb.upload(np.exp2((g[None, :] * 3 + np.arange(bs.blocks(n))[:, None]) % 3))
    ref = p.expected()[0]
    for _ in range(10):
        p.c.upload(np.full((m, n), 0.5))
        p.run()
        assert np.array_equal(p.c.download(), ref)


# one of every kernel and number of tokens: few rows, unaligned rows, CTA pairs
EVERY_KERNEL = [(9, 392, 512), (30, 392, 512), (64, 392, 512), (128, 392, 512), (50, 392, 510), (2100, 1032, 512)]


@pytest.mark.parametrize("shape", EVERY_KERNEL)
def test_scales_up_to_the_ends_of_their_products(ctx, shape):
    """Products of scales from 2^-126 to 2^127.  Codes are multiples of 2^-9 up to 7 * 2^-9, so every partial sum is an integer below
    2^15 times 2^-18, and a sum of them is exact unless it lies below the normal numbers, where each of its roundings (blocks, shares of
    K, alpha) costs 2^-150.  Zero rows stay zero however large their scale is."""
    m, n, k = shape
    p = Problem(ctx, m, n, k, "float32")
    r = np.random.default_rng(96)
    a = r.integers(-7, 8, (m, k)) * 2.0 ** -9
    a[4::5] = 0.0
    p.a.upload(a)
    p.b.upload(r.integers(-7, 8, (n, k)) * 2.0 ** -9)
    rows, columns = np.array([0.0, -66.0, 63.0, 20.0]), np.array([64.0, -60.0, 0.0, -1.0])
    p.sa.upload(np.exp2(np.repeat(rows[r.integers(0, 4, m)][:, None], bs.blocks(k), 1)))
    p.sb.upload(np.exp2(np.repeat(columns[np.arange(bs.blocks(n)) % 4][:, None], bs.blocks(k), 1)))
    p.run()
    ref, _ = p.expected()
    got = p.c.download()
    assert np.all(np.abs(got - ref) <= (bs.blocks(k) + 8 + 1) * 2.0 ** -150 * (np.abs(ref) < 2.0 ** -126))


@pytest.mark.parametrize("shape", EVERY_KERNEL)
def test_scales_past_the_ends_of_their_products(ctx, shape):
    """a product below the normal numbers is off by 2^-150, times partial sums of up to 128 * 448^2; one past them is infinite"""
    m, n, k = shape
    p = Problem(ctx, m, n, k, "float32")
    sa, sb = np.exp2(np.full(p.sa.shape, -70.0)) * 1.1, np.exp2(np.full(p.sb.shape, -66.0)) * 1.3
    p.sa.upload(sa)
    p.sb.upload(sb)
    p.run()
    ref, size = p.expected()
    limit = bs.blocks(k) * 2.0 ** -150 * 128 * 448 ** 2
    assert np.all(np.abs(p.c.download() - ref) <= limit + bs.gemm_error_bound(ref, size, k, "float32"))
    a = np.ones((m, k))
    a[1] = 0.0
    p.a.upload(a)
    p.b.upload(np.ones((n, k)))
    p.sa.upload(np.full(p.sa.shape, 2.0 ** 64))
    p.sb.upload(np.full(p.sb.shape, 2.0 ** 64))
    p.run()
    got = p.c.download()
    assert np.all(np.isnan(got[1])) and np.all(np.isposinf(np.delete(got, 1, 0)))


@pytest.mark.parametrize("shape", EVERY_KERNEL)
def test_zero_scales_and_infinite_ones(ctx, shape):
    """zero times anything finite is zero, zero times infinity NaN, whatever stands beside it"""
    m, n, k = shape
    p = Problem(ctx, m, n, k, "float32")
    p.a.upload(np.ones((m, k)))
    p.b.upload(np.ones((n, k)))
    sa, sb = np.full(p.sa.shape, 2.0 ** -9), np.full(p.sb.shape, 2.0 ** -9)
    sa[1], sa[2], sa[3], sb[1] = 0.0, np.inf, 2.0 ** -130, 2.0 ** 100
    sa[5] = 2.0 ** -110  # with 2^-9: a normal product
    p.sa.upload(sa)
    p.sb.upload(sb)
    p.run()
    got = p.c.download()
    ref = k * np.repeat(sa[:, :1], n, 1) * np.repeat(sb[:, 0], 128)[None, :n]
    assert np.array_equal(got, ref)
    sb[0] = 0.0
    p.sb.upload(sb)
    p.run()
    got = p.c.download()
    assert np.all(np.isnan(got[2, :128])) and np.all(np.isposinf(got[2, 128:]))
    keep = np.arange(m) != 2
    assert np.all(got[keep, :128] == 0.0) and np.array_equal(got[keep, 128:], ref[keep, 128:])


@pytest.mark.parametrize("m", [1, 70])
@pytest.mark.parametrize("tiles", [1, 14, 15, 16, 18, 19, 22, 23, 26, 27, 33, 34, 45, 46, 74, 75, 149])
def test_tile_counts_around_what_clusters_of_each_size_hold(ctx, m, tiles):
    """the number of shares of K follows from how many clusters of each size the device runs at once; integers, so any share shows"""
    n, k = tiles * 128 - 8, 1152
    p = Problem(ctx, m, n, k, "float32")
    r = np.random.default_rng(97)
    p.a.upload(r.integers(-8, 9, (m, k)))
    p.b.upload(r.integers(-8, 9, (n, k)))
    p.sa.upload(np.exp2(r.integers(-2, 2, (m, bs.blocks(k)))))
    p.sb.upload(np.exp2(r.integers(-2, 2, (bs.blocks(n), bs.blocks(k)))))
    p.run()
    assert np.array_equal(p.c.download(), p.expected()[0]) and p.c.guards_intact()
