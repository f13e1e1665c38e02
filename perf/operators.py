"""The 8-bit floating-point operators: what is measured, in plain form and through the library.

Three operators that belong together, the quantised-inference path in e4m3:

  quantize   cudaQuantizeBlocks    x -> e4m3 codes and float32 scales, one per 1 x 128 group (activations) or 128 x 128 block (weights)
  norm       cudaRmsNormQuantize   h = x + z, RMS norm of h, the result quantised in 1 x 128 groups
  gemm       cudaGemmBlockScaled   C = A B^T of two such operands, A in 1 x 128 groups (tokens or pixels), B in 128 x 128 blocks (weights)
"""
import torch

own = False

GROUP = 128
LARGEST = 448.0        # largest e4m3 value
SMALLEST = 2.0 ** -100  # a group whose largest magnitude is below this is scaled as if it were this
DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}
SIZES = {"float16": 2, "bfloat16": 2, "float32": 4}


def listed():
    return [
        # one token against one weight matrix: a decoding step, where the launch and the weights' bytes are everything
        {"name": "gemm one token", "op": "gemm", "m": 1, "n": 4096, "k": 4096, "out": "bfloat16"},
        # a small decoding batch of odd size
        {"name": "gemm 13 tokens", "op": "gemm", "m": 13, "n": 8192, "k": 4096, "out": "float16"},
        # a batch that fills neither kind of tile, K not a whole number of groups, float32 result
        {"name": "gemm ragged", "op": "gemm", "m": 333, "n": 2056, "k": 1616, "out": "float32"},
        # a 3x3 layer of 256 channels over 256 images of 14x14, lowered to a product (the layer of the int8 benchmark)
        {"name": "gemm lowered layer", "op": "gemm", "m": 50176, "n": 256, "k": 2304, "out": "bfloat16"},
        # a long prompt through a wide layer
        {"name": "gemm prompt", "op": "gemm", "m": 4096, "n": 8192, "k": 4096, "out": "bfloat16"},
        # the largest product
        {"name": "gemm large", "op": "gemm", "m": 8192, "n": 8192, "k": 8192, "out": "bfloat16"},
        # activations of a prompt between two products
        {"name": "quantize activations", "op": "quantize", "rows": 4096, "c": 8192, "dtype": "bfloat16", "square": False},
        # float32 rows of odd length, the last group short
        {"name": "quantize odd rows", "op": "quantize", "rows": 777, "c": 1001, "dtype": "float32", "square": False},
        # weights, once when a model is loaded
        {"name": "quantize weights", "op": "quantize", "rows": 8192, "c": 8192, "dtype": "bfloat16", "square": True},
        # one token
        {"name": "norm one token", "op": "norm", "rows": 1, "c": 4096, "dtype": "bfloat16", "residual": True},
        # pixels of a convolutional layer, no residual
        {"name": "norm pixels", "op": "norm", "rows": 50176, "c": 264, "dtype": "float16", "residual": False},
        # a long prompt
        {"name": "norm prompt", "op": "norm", "rows": 8192, "c": 8192, "dtype": "bfloat16", "residual": True},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["gemm", "gemm", "quantize", "norm"])
    if op == "gemm":
        m, n = _log(rng, 1, 8192), _log(rng, 96, 8192)
        if rng.random() < 0.5:
            n = max(128, n // 64 * 64)
        unit = rng.choice([128, 128, 64, 16, 16, 1])  # 1: a row pitch of any length
        k = max(unit, _log(rng, 96, 8192) // unit * unit)
        return {"op": "gemm", "m": m, "n": n, "k": k, "out": rng.choice(["bfloat16", "bfloat16", "float16", "float32"])}
    rows, c = _log(rng, 1, 8192), _log(rng, 48, 8192)
    if rng.random() < 0.6:
        c = max(8, c // 8 * 8)
    dtype = rng.choice(["bfloat16", "float16", "float32"])
    if op == "quantize":
        return {"op": "quantize", "rows": rows, "c": c, "dtype": dtype, "square": rng.random() < 0.4}
    return {"op": "norm", "rows": rows, "c": c, "dtype": dtype, "residual": rng.random() < 0.6}


def work(case):
    if case["op"] == "gemm":
        m, n, k = case["m"], case["n"], case["k"]
        groups = -(-k // GROUP)
        return {"bytes": m * k + n * k + 4 * groups * (m + -(-n // GROUP)) + SIZES[case["out"]] * m * n, "flops": 2 * m * n * k}
    rows, c, size = case["rows"], case["c"], SIZES[case["dtype"]]
    groups = -(-c // GROUP)
    if case["op"] == "quantize":
        scales = (-(-rows // GROUP) if case["square"] else rows) * groups
        return {"bytes": rows * c * (size + 1) + 4 * scales, "flops": 2 * rows * c}
    return {"bytes": rows * c * (size * (3 if case["residual"] else 1) + 1) + 4 * rows * groups + 4 * c, "flops": 6 * rows * c}


# ---- inputs -----------------------------------------------------------------------------------------------------------

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(shape, g, dtype=torch.float32):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _codes(rows, c, g):
    """e4m3 codes as a quantiser leaves them: normal values that fill the range of their group."""
    return (_normal((rows, c), g) * 120).clamp_(-LARGEST, LARGEST).to(torch.float8_e4m3fn)


def prepare(case, seed):
    g = _generator(seed)
    if case["op"] == "gemm":
        m, n, k = case["m"], case["n"], case["k"]
        groups = -(-k // GROUP)
        held = {
            "a": _codes(m, k, g),
            "a_scale": torch.rand((m, groups), generator=g, device="cuda") * 0.02 + 0.002,
            "b": _codes(n, k, g),
            "b_scale": (torch.rand((-(-n // GROUP), groups), generator=g, device="cuda") * 0.5 + 0.5) * (0.008 / k ** 0.5),
            "c": torch.zeros((m, n), dtype=DTYPES[case["out"]], device="cuda"),
        }
    else:
        rows, c, dtype = case["rows"], case["c"], DTYPES[case["dtype"]]
        groups = -(-c // GROUP)
        x = _normal((rows, c), g)
        x[:, torch.randint(0, c, (max(1, c // 256),), generator=g, device="cuda")] *= 20  # a few channels with large values
        held = {"x": x.to(dtype), "q": torch.zeros((rows, c), dtype=torch.float8_e4m3fn, device="cuda")}
        square = case["op"] == "quantize" and case["square"]
        held["scale"] = torch.zeros((-(-rows // GROUP) if square else rows, groups), device="cuda")
        if case["op"] == "norm":
            held["gamma"] = 1 + 0.1 * _normal((c,), g)
            if case["residual"]:
                held["z"] = _normal((rows, c), g, dtype)
                held["h"] = torch.zeros((rows, c), dtype=dtype, device="cuda")
    return {"case": dict(case), **_in_hand(held)}


def _in_hand(held):
    """The same tensors where a program of the library keeps them: in its memory blocks, with their descriptors."""
    if not own:
        return {"t": held}
    from cudabackend_b200 import api
    names = {torch.float8_e4m3fn: "float8_e4m3", torch.float16: "float16", torch.bfloat16: "bfloat16", torch.float32: "float32"}
    blocks = {k: api.DeviceTensor(tuple(v.shape), names[v.dtype]) for k, v in held.items()}
    views = {}
    for k, v in held.items():
        views[k] = _view(blocks[k].mem.pointer(), v)
        views[k].copy_(v)
    torch.cuda.synchronize()
    return {"t": views, "d": blocks, "ctx": api.Context.default(0), "api": api}


def _view(pointer, like):
    class Holder:
        pass
    holder = Holder()
    holder.__cuda_array_interface__ = {"shape": (like.numel() * like.element_size(),), "typestr": "|u1", "data": (pointer, False), "version": 3}
    return torch.as_tensor(holder, device="cuda").view(like.dtype).view(like.shape)


# ---- one pass ---------------------------------------------------------------------------------------------------------

EPSILON = 1e-6


def run(state):
    case, t = state["case"], state["t"]
    if own:
        api, d, ctx = state["api"], state["d"], state["ctx"].handle
        if case["op"] == "gemm":
            a, sa, b, sb, c = d["a"], d["a_scale"], d["b"], d["b_scale"], d["c"]
            api.call("cudaGemmBlockScaled", ctx, api.GEMM_N, api.GEMM_T, None, a.desc.handle, a.mem.handle, sa.desc.handle, sa.mem.handle,
                     b.desc.handle, b.mem.handle, sb.desc.handle, sb.mem.handle, None, c.desc.handle, c.mem.handle)
            return t["c"]
        x, q, s = d["x"], d["q"], d["scale"]
        if case["op"] == "quantize":
            api.call("cudaQuantizeBlocks", ctx, x.desc.handle, x.mem.handle, q.desc.handle, q.mem.handle, s.desc.handle, s.mem.handle)
            return {"q": t["q"], "scale": t["scale"]}
        g = d["gamma"]
        z = d["z"].mem.handle if "z" in d else api.INVALID
        h = d["h"].mem.handle if "h" in d else api.INVALID
        api.call("cudaRmsNormQuantize", ctx, x.desc.handle, x.mem.handle, z, h, g.desc.handle, g.mem.handle, EPSILON, q.desc.handle, q.mem.handle,
                 s.desc.handle, s.mem.handle)
        return {"q": t["q"], "scale": t["scale"], **({"h": t["h"]} if "h" in t else {})}
    if case["op"] == "gemm":
        return (_dequantized(t["a"], t["a_scale"], 1) @ _dequantized(t["b"], t["b_scale"], GROUP).T).to(t["c"].dtype)
    x = t["x"].float()
    if case["op"] == "quantize":
        q, scale = _quantized(x, GROUP if case["square"] else 1)
        return {"q": q, "scale": scale}
    if "z" in t:
        x = x + t["z"].float()
    y = x * (x.square().mean(-1, keepdim=True) + EPSILON).rsqrt() * t["gamma"]
    q, scale = _quantized(y, 1)
    return {"q": q, "scale": scale, **({"h": x.to(t["h"].dtype)} if "h" in t else {})}


def _spread(scale, shape, rows):
    """One scale per element of a matrix of `shape`, from one per `rows` x 128 block."""
    if rows > 1:
        scale = scale.repeat_interleave(rows, 0)[:shape[0]]
    return scale.repeat_interleave(GROUP, 1)[:, :shape[1]]


def _dequantized(q, scale, rows):
    return q.float() * _spread(scale, q.shape, rows)


def _quantized(x, rows):
    r, c = x.shape
    padded = torch.nn.functional.pad(x.abs(), (0, -c % GROUP, 0, -r % rows))
    amax = padded.view(-(-r // rows), rows, -(-c // GROUP), GROUP).amax((1, 3)).clamp_min(SMALLEST)
    q = (x * _spread(LARGEST / amax, x.shape, rows)).to(torch.float8_e4m3fn)
    return q, amax / LARGEST


# ---- the definition in 64 bits ------------------------------------------------------------------------------------------

def exact(case, seed):
    t = prepare(case, seed)["t"]
    if case["op"] == "gemm":
        out = torch.zeros((case["m"], case["n"]), dtype=torch.float64, device="cuda")
        for g in range(-(-case["k"] // GROUP)):
            at = slice(g * GROUP, (g + 1) * GROUP)
            weights = t["b_scale"][:, g].double()[torch.arange(case["n"], device="cuda") // GROUP]
            out.addmm_(t["a"][:, at].double() * t["a_scale"][:, g:g + 1].double(), (t["b"][:, at].double() * weights[:, None]).T)
        return out
    y = t["x"].double()
    found = {}
    if case["op"] == "norm":
        if "z" in t:
            y = y + t["z"].double()
            found["h"] = y
        y = y / torch.sqrt((y * y).sum(-1, keepdim=True) / case["c"] + EPSILON) * t["gamma"].double()
    square = case["op"] == "quantize" and case["square"]
    height = GROUP if square else 1
    q, scale = torch.empty_like(y), torch.empty(t["scale"].shape, dtype=torch.float64, device="cuda")
    for g in range(scale.shape[1]):
        block = y[:, g * GROUP:(g + 1) * GROUP]
        top = block.abs().amax(1)
        if square:
            row = torch.arange(case["rows"], device="cuda") // height
            top = torch.zeros(scale.shape[0], dtype=torch.float64, device="cuda").scatter_reduce_(0, row, top, "amax")
        scale[:, g] = top.clamp_min(SMALLEST) / LARGEST
        each = scale[:, g][row] if square else scale[:, g]
        v = block / each[:, None]
        step = torch.exp2(torch.frexp(v)[1].clamp_min(-5).double() - 4)  # 3 mantissa bits, exponents from -6
        q[:, g * GROUP:(g + 1) * GROUP] = torch.round(v / step) * step
    return {"q": q, "scale": scale, **found}
