"""The block-scaled 8-bit operators as they are used together, and under graphs, several contexts and other kernels in between."""
import ctypes

import numpy as np
import pytest

from cudabackend_b200 import api
from oracle import oracle as o
from tests import block_scaled as bs

pytestmark = pytest.mark.gpu

EPSILON = 1e-5


def bf16(v):
    return api.bfloat16_bits_to_float(api.float_to_bfloat16_bits(v)).astype(np.float64)


def dequantized(ctx, codes, scales, height=1):
    rows, c = codes.shape
    return codes.download() * o.spread_scales(scales.download(), rows, c, height)


class Block:
    """A pre-norm residual block with two products: h = x + z;  out = h + relu(norm(h) W1^T + b) W2^T."""

    def __init__(self, ctx, rows, c, hidden, seed=101):
        self.ctx, r = ctx, np.random.default_rng(seed)
        P = bs.Placed
        self.x, self.z = P(ctx, (rows, c), "bfloat16", values=r.normal(0, 1, (rows, c))), P(ctx, (rows, c), "bfloat16", values=r.normal(0, 1, (rows, c)))
        self.gamma, self.bias = P(ctx, (c,), "float32", values=1 + 0.1 * r.normal(0, 1, c)), P(ctx, (hidden,), "float32", values=0.1 * r.normal(0, 1, hidden))
        self.out = P(ctx, (rows, c), "bfloat16")
        self.weights = []
        for n, k in ((hidden, c), (c, hidden)):
            w = P(ctx, (n, k), "bfloat16", values=r.normal(0, k ** -0.5, (n, k)))
            q, s = P(ctx, (n, k), "float8_e4m3"), P(ctx, (bs.blocks(n), bs.blocks(k)), "float32")
            bs.quantize(ctx, w, q, s)
            self.weights.append((w, q, s))
        self.q1, self.s1 = P(ctx, (rows, c), "float8_e4m3"), P(ctx, (rows, bs.blocks(c)), "float32")
        self.mid, self.act = P(ctx, (rows, hidden), "bfloat16"), P(ctx, (rows, hidden), "bfloat16")
        self.q2, self.s2 = P(ctx, (rows, hidden), "float8_e4m3"), P(ctx, (rows, bs.blocks(hidden)), "float32")

    def run(self, ctx=None):
        ctx = ctx or self.ctx
        (_, w1, t1), (_, w2, t2) = self.weights
        bs.rms_norm_quantize(ctx, self.x, self.z, self.out, self.gamma, EPSILON, self.q1, self.s1)
        bs.gemm(ctx, self.q1, self.s1, w1, t1, self.mid)
        api.call("cudaAddBias", ctx.handle, None, None, self.mid.desc.handle, self.mid.mem.handle, self.bias.desc.handle, self.bias.mem.handle,
                 self.act.desc.handle, self.act.mem.handle, None, None, None, api.INVALID, api.ACTIVATIONS["relu"])
        bs.quantize(ctx, self.act, self.q2, self.s2)
        bs.gemm(ctx, self.q2, self.s2, w2, t2, self.out, beta=1.0)

    def check_stages(self):
        """each stage against its formula on the inputs that it had on the device"""
        h64, y64 = o.rms_norm(self.x.values, self.z.values, self.gamma.values, EPSILON)
        y = dequantized(self.ctx, self.q1, self.s1)
        spread = o.spread_scales(self.s1.download(), *self.q1.shape)
        assert np.all(np.abs(y - y64) <= bs.code_error_bound(y64, spread, 40 * bs.U32))
        (_, w1, t1), (_, w2, t2) = self.weights
        ref, size = o.gemm_block_scaled(self.q1.download(), self.s1.download(), w1.download(), t1.download())
        mid = self.mid.download()
        assert np.all(np.abs(mid - ref) <= bs.gemm_error_bound(ref, size, self.q1.shape[1], "bfloat16"))
        act = self.act.download()
        assert np.all(np.abs(act - np.maximum(mid + self.bias.values, 0)) <= (np.abs(mid) + np.abs(self.bias.values)) * (2.0 ** -8 + 2 * bs.U32) + 2.0 ** -134)
        spread = o.spread_scales(self.s2.download(), *self.q2.shape)
        assert np.all(np.abs(dequantized(self.ctx, self.q2, self.s2) - act) <= bs.code_error_bound(act, spread, 2 * bs.U32))
        ref, size = o.gemm_block_scaled(self.q2.download(), self.s2.download(), w2.download(), t2.download(), 1.0, 1.0, bf16(h64.astype(np.float32)))
        # the residual was rounded twice: to float32 by the sum, to bfloat16 by the store
        assert np.all(np.abs(self.out.download() - ref) <= bs.gemm_error_bound(ref, size, self.q2.shape[1], "bfloat16") + np.abs(h64) * 2.0 ** -8)
        return h64, y64

    def check_whole(self):
        """The whole block against float64 without quantisation.  A code stands for its value within 2^-4 of it, or 2^-18 of the
        block's largest (2^-10 of the scale, which is that / 448); a bfloat16 rounding is 2^-8, counted twice per product (its
        result and the step behind it).  Errors of both factors add up, magnified by each other's size."""
        def off(v, axis):
            return np.abs(v) * 2.0 ** -4 + np.abs(v).max(axis=axis, keepdims=True) * 2.0 ** -18

        h64, y64 = o.rms_norm(self.x.values, self.z.values, self.gamma.values, EPSILON)
        (w1, _, _), (w2, _, _) = self.weights
        mid = np.maximum(y64 @ w1.values.T + self.bias.values, 0)
        ref = h64 + mid @ w2.values.T
        y_off, w1_off, w2_off = off(y64, 1), off(w1.values, None), off(w2.values, None)
        size = (np.abs(y64) + y_off) @ (np.abs(w1.values) + w1_off).T + np.abs(self.bias.values)
        mid_off = y_off @ np.abs(w1.values).T + (np.abs(y64) + y_off) @ w1_off.T + size * 2 * 2.0 ** -8 * (1 + 2.0 ** -8)
        act_off = mid_off + off(mid + mid_off, 1)
        bound = act_off @ np.abs(w2.values).T + (mid + act_off) @ w2_off.T + 2 * 2.0 ** -8 * (np.abs(h64) + (mid + act_off) @ (np.abs(w2.values) + w2_off).T)
        assert np.all(np.abs(self.out.download() - ref) <= bound * (1 + 2.0 ** -10))


@pytest.mark.parametrize("rows,c,hidden", [(1, 512, 1024), (13, 384, 640), (150, 264, 520), (2500, 512, 1024)])
def test_a_residual_block(ctx, rows, c, hidden):
    block = Block(ctx, rows, c, hidden)
    block.run()
    block.check_stages()
    block.check_whole()


def test_a_convolution_in_float8(ctx):
    """quantise pixels, lower codes and scales alike with cudaIm2Row, multiply: a 3x3 convolution; the padding's scale is 0"""
    n, h, w, c, k = 3, 9, 11, 256, 136
    r = np.random.default_rng(102)
    x = bs.Placed(ctx, (n, h, w, c), "float16", values=r.normal(0, 1, (n, h, w, c)))
    wt = bs.Placed(ctx, (k, 3 * 3 * c), "float16", values=r.normal(0, (9 * c) ** -0.5, (k, 9 * c)))
    q, s = bs.Placed(ctx, (n, h, w, c), "float8_e4m3"), bs.Placed(ctx, (n, h, w, c // 128), "float32")
    wq, ws = bs.Placed(ctx, (k, 9 * c), "float8_e4m3"), bs.Placed(ctx, (bs.blocks(k), 9 * c // 128), "float32")
    bs.quantize(ctx, x, q, s)
    bs.quantize(ctx, wt, wq, ws)
    conv = api.ConvolutionDescriptor(api.CONVOLUTION_MODE, (-1, -1))
    rows = n * h * w
    rq, rs = bs.Placed(ctx, (rows, 9 * c), "float8_e4m3"), bs.Placed(ctx, (rows, 9 * c // 128), "float32")
    for src, dst, channels, dtype in ((q, rq, c, "float8_e4m3"), (s, rs, c // 128, "float32")):
        filters = api.TensorDescriptor((k, 3, 3, channels), dtype)
        api.call("cudaIm2Row", ctx.handle, conv.handle, filters.handle, src.desc.handle, src.mem.handle, dst.desc.handle, dst.mem.handle)
    y = bs.Placed(ctx, (rows, k), "float16")
    bs.gemm(ctx, rq, rs, wq, ws, y)
    pixels = q.download() * np.repeat(s.download(), 128, axis=3)
    filters = (wq.download() * o.spread_scales(ws.download(), k, 9 * c, 128)).reshape(k, 3, 3, c)
    ref = o.conv2d_forward(pixels, filters, padding=(-1, -1)).reshape(rows, k)
    size = o.conv2d_forward(np.abs(pixels), np.abs(filters), padding=(-1, -1)).reshape(rows, k)
    assert np.all(np.abs(y.download() - ref) <= bs.gemm_error_bound(ref, size, 9 * c, "float16"))


@pytest.mark.parametrize("rows", [1, 90, 1700])
def test_captured_and_replayed_on_new_inputs(ctx, rows):
    block = Block(ctx, rows, 512, 1280)
    graph = ctx.capture(block.run)
    for seed in (5, 6):
        r = np.random.default_rng(seed)
        block.x.upload(r.normal(0, 2, block.x.shape))
        block.z.upload(r.normal(0, 1, block.z.shape))
        graph.launch()
        ctx.synchronize()
        block.check_stages()
    graph.destroy()


def test_two_graphs_and_two_contexts_at_once(ctx):
    """the operators keep nothing between calls and share no scratch: graphs of two contexts replayed side by side"""
    other = api.Context(0)
    blocks = [Block(ctx, 40, 512, 1024, 7), Block(other, 40, 512, 1024, 8), Block(ctx, 1100, 512, 2048, 9), Block(other, 1100, 512, 2048, 10)]
    graphs = [b.ctx.capture(b.run) for b in blocks]
    for _ in range(20):
        for g in graphs:
            g.launch()
    for c in (ctx, other):
        c.synchronize()
    for b in blocks:
        b.check_stages()
    for g in graphs:
        g.destroy()
    assert other.last_device_status() == 0
    other.destroy()


def test_default_context_and_another_stream_by_events(ctx):
    """the default context's stream, and work of a second context ordered behind it"""
    default = api.Context.default(0)
    block = Block(default, 200, 384, 640)
    block.run()
    default.synchronize()
    block.check_stages()
    side = api.Context(0)
    block = Block(ctx, 200, 384, 640)
    side.wait_for(ctx)
    block.run(side)
    ctx.wait_for(side)
    ctx.synchronize()
    block.check_stages()
    side.synchronize()
    side.destroy()


def test_a_held_back_call_runs_first(ctx):
    """a context that fuses Winograd calls holds one back: the new operators launch it before their own work, as every call does"""
    ctx.set_winograd_fusion(True)
    r = np.random.default_rng(103)
    a, b = (bs.Placed(ctx, (36, 128, 64), "float16", values=r.normal(0, 1, (36, 128, 64))) for _ in range(2))
    c = bs.Placed(ctx, (36, 128, 128), "float16")
    api.call("cudaGemmBatched", ctx.handle, api.GEMM_N, api.GEMM_T, None, a.desc.handle, a.mem.handle, b.desc.handle, b.mem.handle, None, c.desc.handle, c.mem.handle)
    flat = api.TensorDescriptor((36 * 128, 128), "float16")
    y, s = bs.Placed(ctx, (36 * 128, 128), "float8_e4m3"), bs.Placed(ctx, (36 * 128, 1), "float32")
    api.call("cudaQuantizeBlocks", ctx.handle, flat.handle, c.mem.handle, y.desc.handle, y.mem.handle, s.desc.handle, s.mem.handle)
    got = y.download() * o.spread_scales(s.download(), 36 * 128, 128)
    c64 = c.download().reshape(36 * 128, 128)
    assert np.all(np.abs(got - c64) <= bs.code_error_bound(c64, o.spread_scales(s.download(), 36 * 128, 128), 2 * bs.U32))
    assert np.all(np.abs(c64 - o.gemm_batched(a.values, b.values, False, True).reshape(36 * 128, 128)) <= 0.05)
    ctx.set_winograd_fusion(0)


def test_calls_from_several_host_threads(library, device_count):
    """one context per thread, first calls at the same moment"""
    import threading
    failures = []

    def work(seed):
        try:
            context = api.Context(0)
            block = Block(context, 33 + seed, 384, 512, seed)
            for _ in range(5):
                block.run(context)
            context.synchronize()
            block.check_stages()
            assert context.last_device_status() == 0
            context.destroy()
        except Exception as e:  # noqa: BLE001
            failures.append(repr(e))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures
