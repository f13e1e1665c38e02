"""Shared pieces of the tests of the block-scaled 8-bit operators: tensors on the device, calls, error bounds."""
import ctypes

import numpy as np

from cudabackend_b200 import api
from oracle import oracle as o

U32 = 2.0 ** -24  # half a step of float32, relative
HALF_STEP = {"float16": 2.0 ** -11, "bfloat16": 2.0 ** -8, "float32": 2.0 ** -24}
LEAST = {"float16": 2.0 ** -25, "bfloat16": 2.0 ** -134, "float32": 2.0 ** -150}  # half a step of the subnormal numbers


def blocks(extent):
    return -(-extent // 128)


class Placed:
    """A tensor that starts `offset` bytes into its memory block, with guard bytes in front of it and behind it."""

    GUARD = 64

    def __init__(self, ctx, shape, dtype, offset=0, values=None):
        self.ctx, self.dtype, self.shape, self.offset = ctx, dtype, tuple(shape), offset
        self.desc = api.TensorDescriptor(shape, dtype)
        self.block = api.Memory(self.GUARD + offset + self.desc.nbytes + self.GUARD)
        self.block.from_host(ctx, np.full(self.block.size, 0x5A, dtype=np.uint8))
        self.mem = self.block.view(self.desc.nbytes, self.GUARD + offset)
        if values is not None:
            self.upload(values)

    def upload(self, values):
        stored, self.values = api.to_storage(np.asarray(values).reshape(self.shape), self.dtype)
        if stored.size:
            self.mem.from_host(self.ctx, stored)
        return self.values

    def raw(self):
        buf = api.host_buffer(self.shape, self.dtype)
        if buf.size:
            self.mem.to_host(self.ctx, buf)
        self.ctx.synchronize()
        return buf

    def download(self):
        return api.from_storage(self.raw(), self.dtype)

    def guards_intact(self):
        whole = self.block.to_host(self.ctx, np.empty(self.block.size, dtype=np.uint8))
        self.ctx.synchronize()
        start = self.GUARD + self.offset
        return bool(np.all(whole[:start] == 0x5A) and np.all(whole[start + self.desc.nbytes:] == 0x5A))


def quantize(ctx, x, y, scale, status=False):
    call = api.call_status if status else api.call
    return call("cudaQuantizeBlocks", ctx.handle, x.desc.handle, x.mem.handle, y.desc.handle, y.mem.handle, scale.desc.handle, scale.mem.handle)


def rms_norm_quantize(ctx, x, z, h, gamma, epsilon, y, scale, status=False):
    call = api.call_status if status else api.call
    return call("cudaRmsNormQuantize", ctx.handle, x.desc.handle, x.mem.handle, z.mem.handle if z is not None else api.INVALID,
                h.mem.handle if h is not None else api.INVALID, gamma.desc.handle, gamma.mem.handle, float(epsilon), y.desc.handle, y.mem.handle,
                scale.desc.handle, scale.mem.handle)


def gemm(ctx, a, a_scale, b, b_scale, c, alpha=None, beta=None, ops=(api.GEMM_N, api.GEMM_T), status=False):
    pa, ka = api.scalar_pointer(alpha, "float32")
    pb, kb = api.scalar_pointer(beta, "float32")
    call = api.call_status if status else api.call
    result = call("cudaGemmBlockScaled", ctx.handle, ops[0], ops[1], pa, a.desc.handle, a.mem.handle, a_scale.desc.handle, a_scale.mem.handle, b.desc.handle,
                  b.mem.handle, b_scale.desc.handle, b_scale.mem.handle, pb, c.desc.handle, c.mem.handle)
    del ka, kb
    return result


def code_error_bound(y, scale, relative=0.0):
    """How far code * scale may be from y: half an e4m3 step (2^-4 of the value, 2^-10 of the scale below the normal numbers),
    where the value that was rounded is itself off by `relative`."""
    return np.maximum(2.0 ** -4 * np.abs(y), 2.0 ** -10 * scale) * (1 + 2.0 ** -20 + 2 * relative) + np.abs(y) * (relative + 4 * U32)


def gemm_error_bound(ref, size, k, dtype):
    """A sum of n terms added in any order in float32, each addition off by at most a unit in the last place (2^-23) of the
    largest partial sum: a block's terms (at most 128, in the tensor core), the blocks, two scale factors, alpha and beta; then
    half a step of the result's type."""
    terms = min(k, 128) + blocks(k) + 4
    return size * terms * 2.0 ** -23 + np.abs(ref) * HALF_STEP[dtype] * (1 + 2.0 ** -10) + LEAST[dtype]


def random_codes(rng, rows, c):
    """e4m3 values as a quantiser leaves them, subnormal ones and the largest among them"""
    v = rng.normal(0, 120, (rows, c))
    v[rng.random((rows, c)) < 0.05] *= 2.0 ** -12
    return o.e4m3_round(np.clip(v, -448, 448))
