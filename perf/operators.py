"""The block-scaled FP8 operators: what is timed, on which inputs, and their plain forms.

A packed matrix holds E4M3 codes with one power-of-two scale for each block of 128:
an activation's block is 128 columns of one row, a weight's 128 rows by 128 columns
(the last ones may be cut off). The scale of a block is 2^e with the least e for which
max|x| <= 448 * 2^e, and e >= -64; a code is x / 2^e rounded to nearest even.

  linear  y[rows, n] = bf16(x . w^T + bias), x packed or BF16 (then packed by the call), w packed
  norm    the residual row r = bf16(residual + branch) or bf16(residual + branch * gate), and
          r's root-mean-square norm, (with AdaLN's scale and shift) packed
  swiglu  silu(gate) * up of rows that hold gate, then up, packed
  mlp     linear to gate and up -> silu(gate) * up, packed -> linear; 32 bits in between

Packed results come back as the BF16 values that their codes and scales stand for, which
hold them exactly.

Sizes are those of the two block geometries that the library ships
(h3cli_amd.runtime.DitSynth), "synthetic" (hidden 5120, MLP 13824, 27 x 30 x 40 video rows
and 1024 audio rows) and "h3" (hidden 5376, attention 7168, MLP 14336, frames of 27 x 27
rows), and generic odd ones.
"""
import ctypes as C
import math

import torch

own = False

HIDDEN, INNER, MLP = 5376, 7168, 14336
SHAPES = [(HIDDEN, 3 * INNER), (INNER, HIDDEN), (HIDDEN, 2 * MLP), (MLP, HIDDEN),
          (5120, 3 * 5120), (5120, 5120), (5120, 13824), (13824, 5120)]
EPS = 1e-5


def listed():
    return [
        # The timestep embedding's first projection: the smallest call, where latency counts.
        {"name": "linear_time", "kind": "linear", "rows": 1, "k": 256, "n": HIDDEN, "input": "bf16", "bias": False},
        # The modulation of a few conditioning rows: the weight is read once for them.
        {"name": "linear_modulation", "kind": "linear", "rows": 9, "k": HIDDEN, "n": 6 * HIDDEN, "input": "packed",
         "bias": True},
        # Nothing is a multiple of a block.
        {"name": "linear_ragged", "kind": "linear", "rows": 301, "k": 1000, "n": 777, "input": "bf16", "bias": True},
        # One 27 x 27 latent frame through the QKV projection, its input packed by the norm.
        {"name": "linear_frame", "kind": "linear", "rows": 729, "k": HIDDEN, "n": 3 * INNER, "input": "packed",
         "bias": False},
        # The output projection of a clip, its input packed by the call.
        {"name": "linear_clip", "kind": "linear", "rows": 8193, "k": INNER, "n": HIDDEN, "input": "bf16", "bias": False},
        # The widest projection at the long sequence.
        {"name": "linear_video", "kind": "linear", "rows": 18225, "k": HIDDEN, "n": 2 * MLP, "input": "packed",
         "bias": False},
        # A few conditioning rows with their residual.
        {"name": "norm_rows", "kind": "norm", "rows": 5, "width": HIDDEN, "adaln": False},
        # The block's second norm over the benchmark's joint sequence: gated residual, modulation.
        {"name": "norm_video", "kind": "norm", "rows": 33424, "width": 5120, "adaln": True},
        # The activation between an MLP's projections, one latent frame and a clip.
        {"name": "swiglu_frame", "kind": "swiglu", "rows": 729, "width": MLP},
        {"name": "swiglu_clip", "kind": "swiglu", "rows": 8193, "width": MLP},
        # The MLP as one call: few rows, bound by its weights, and a clip.
        {"name": "mlp_rows", "kind": "mlp", "rows": 16, "k": HIDDEN, "hidden": MLP, "n": HIDDEN, "input": "bf16"},
        {"name": "mlp_clip", "kind": "mlp", "rows": 8193, "k": HIDDEN, "hidden": MLP, "n": HIDDEN, "input": "packed"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the ranges above; costs are bounded by the listed ones."""
    kind = rng.choice(["linear", "linear", "linear", "ragged", "norm", "swiglu", "mlp"])
    source = rng.choice(["bf16", "packed"])
    if kind == "linear":
        k, n = rng.choice(SHAPES)
        return {"kind": kind, "rows": _log(rng, 1, 18225), "k": k, "n": n, "input": source, "bias": rng.random() < 0.3}
    if kind == "ragged":
        return {"kind": "linear", "rows": _log(rng, 1, 4000), "k": _log(rng, 40, 8000), "n": _log(rng, 40, 8000),
                "input": source, "bias": rng.random() < 0.5}
    if kind == "norm":
        width = rng.choice([5120, HIDDEN, 8 * rng.randint(1, 1024)])
        return {"kind": kind, "rows": _log(rng, 1, min(33424, 33424 * 5120 // width)), "width": width,
                "adaln": rng.random() < 0.5}
    if kind == "swiglu":
        return {"kind": kind, "rows": _log(rng, 1, 8193), "width": rng.choice([13824, MLP, _log(rng, 40, 14000)])}
    k, hidden = rng.choice([(HIDDEN, MLP), (5120, 13824), (8 * rng.randint(16, 640), 128 * rng.randint(1, 110))])
    return {"kind": kind, "rows": _log(rng, 1, 12000), "k": k, "hidden": hidden, "n": k, "input": source}


# ------------------------------------------------------------------ inputs
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 7919 + 29)
    return g


def _normal(g, shape, scale=1.0, shift=0.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale + shift).to(torch.bfloat16)


def _activation(g, rows, k):
    """Rows whose channels differ in scale, one of a hundred by much, as norms give them."""
    scale = torch.exp(0.5 * torch.randn((k,), generator=g, device="cuda"))
    scale = torch.where(torch.rand((k,), generator=g, device="cuda") < 0.01, 16 * scale, scale)
    return (torch.randn((rows, k), generator=g, device="cuda") * scale).to(torch.bfloat16)


def _weight(g, n, k):
    return _normal(g, (n, k), 1 / math.sqrt(k))


def _inputs(case, seed):
    g, kind, rows = _generator(seed), case["kind"], case["rows"]
    if kind == "linear":
        t = {"x": _activation(g, rows, case["k"]), "w": _weight(g, case["n"], case["k"])}
        if case["bias"]:
            t["bias"] = _normal(g, (case["n"],), 0.1)
        return t
    if kind == "mlp":
        return {"x": _activation(g, rows, case["k"]), "w1": _weight(g, 2 * case["hidden"], case["k"]),
                "w2": _weight(g, case["n"], case["hidden"])}
    if kind == "swiglu":
        return {"fused": _normal(g, (rows, 2 * case["width"]), 1.5)}
    width = case["width"]
    t = {"residual": _activation(g, rows, width), "branch": _normal(g, (rows, width)),
         "norm": _normal(g, (width,), 0.1, 1.0)}
    if case["adaln"]:
        # Slots of the modulation: shift and scale of the first norm, gate, shift, scale, gate;
        # video rows first, then audio rows with modulation of their own.
        t["mod"] = _normal(g, (2, 6, width), 0.1)
        t["map"] = (torch.arange(rows, device="cuda") >= rows - rows // 32).to(torch.int32)
    return t


# ------------------------------------------------------------------ the library's tensors
class _Buffer:
    """A device tensor of the library, seen by torch without a copy. torch keeps this object
    alive with the views, and the memory goes back with it."""

    def __init__(self, gpu, shape, dtype=torch.bfloat16):
        from h3cli_amd import _lib
        kind, code = {torch.bfloat16: (_lib.BF16, "<i2"), torch.int32: (_lib.U32, "<i4")}[dtype]
        self.gpu, self.tensor, self.dtype = gpu, gpu.empty(math.prod(shape), kind), dtype
        self.handle = self.tensor.handle
        self.__cuda_array_interface__ = {
            "shape": tuple(shape), "typestr": code, "version": 2, "strides": None,
            "data": (gpu.lib.h3_hip_tensor_device_pointer(self.handle), False)}

    def view(self):
        t = torch.as_tensor(self, device="cuda")
        return t.view(torch.bfloat16) if self.dtype == torch.bfloat16 else t

    def __del__(self):
        if self.gpu.handle:
            self.gpu.free(self.tensor)


class _Packed:
    """A packed matrix of the library."""

    def __init__(self, gpu, handle):
        gpu.check(handle, "packed matrix")
        self.gpu, self.handle = gpu, handle

    def __del__(self):
        if self.gpu.handle:
            self.gpu.lib.h3_gpu_tensor_free(self.handle)


_contexts = []


def _context():
    """One context for the life of the process, its command open, as within a denoise step."""
    if not _contexts:
        from h3cli_amd.runtime import Gpu
        _contexts.append(Gpu())
        _contexts[0].begin()
    return _contexts[0]


def _put(gpu, value):
    b = _Buffer(gpu, tuple(value.shape), value.dtype)
    b.view().copy_(value)
    torch.cuda.synchronize()
    return b


def _put_packed(gpu, value, weight):
    source, (rows, columns) = _put(gpu, value), value.shape
    if weight:
        return _Packed(gpu, gpu.lib.h3_hip_fp8_block_weight_from_bf16(gpu.handle, source.handle, rows, columns))
    packed = _Packed(gpu, gpu.lib.h3_hip_fp8_block_new(gpu.handle, rows, columns, 1))
    gpu.check(gpu.lib.h3_hip_fp8_block_pack(gpu.handle, packed.handle, source.handle, rows, columns), "pack")
    gpu.check(gpu.lib.h3_gpu_synchronize(gpu.handle), "pack")
    return packed


def _calls(case, t):
    """The library's calls of one pass, and the tensors that they write."""
    gpu = _context()
    lib, g, kind, rows = gpu.lib, gpu.handle, case["kind"], case["rows"]
    held = {name: _put_packed(gpu, v, name != "x") if name in ("w", "w1", "w2") or (name == "x" and case["input"] == "packed")
            else _put(gpu, v) for name, v in t.items()}
    h = {name: b.handle for name, b in held.items()}
    packed_input = case.get("input") == "packed"
    if kind == "linear":
        out = _Buffer(gpu, (rows, case["n"]))
        f = lib.h3_hip_linear_fp8_block if packed_input else lib.h3_gpu_linear_bf16
        calls, outs = [(f, (g, out.handle, h["x"], h["w"], h.get("bias"), rows, case["k"], case["n"]))], [out]
    elif kind == "mlp":
        out = _Buffer(gpu, (rows, case["n"]))
        f = lib.h3_hip_mlp_fp8_block if packed_input else lib.h3_gpu_mlp_bf16
        calls = [(f, (g, out.handle, h["x"], h["w1"], h["w2"], rows, case["k"], case["hidden"], case["n"]))]
        outs = [out]
    else:
        width = case["width"]
        packed = _Packed(gpu, lib.h3_hip_fp8_block_new(g, rows, width, 1))
        held["packed"], values = packed, _Buffer(gpu, (rows, width))
        outs = [values]
        if kind == "swiglu":
            calls = [(lib.h3_hip_swiglu_fp8_block, (g, packed.handle, h["fused"], rows, width))]
        else:
            total = _Buffer(gpu, (rows, width))
            outs = [total, values]
            if case["adaln"]:
                calls = [(lib.h3_hip_gate_adaln_fp8_block,
                          (g, total.handle, packed.handle, h["residual"], h["branch"], h["norm"], h["mod"], h["mod"],
                           h["map"], rows, width, 6, 2, 3, 4, C.c_float(EPS)))]
            else:
                calls = [(lib.h3_hip_add_rms_norm_fp8_block,
                          (g, total.handle, packed.handle, h["residual"], h["branch"], h["norm"], rows, width,
                           C.c_float(EPS)))]
        calls.append((lib.h3_hip_fp8_block_unpack, (g, values.handle, packed.handle, rows, width)))
    return {"gpu": gpu, "calls": calls, "keep": held, "out": [b.view() for b in outs]}


# ------------------------------------------------------------------ the plain forms
def _blocks(x, tile):
    """x in 32 bits as [row blocks, tile, column blocks, 128], zeros behind its ends."""
    rows, k = x.shape
    x = torch.nn.functional.pad(x.float(), (0, -k % 128, 0, -rows % tile))
    return x.reshape(x.shape[0] // tile, tile, -1, 128)


def _pack(x, tile):
    """Codes [row blocks, tile, column blocks, 128] and exponents [row blocks, 1, column blocks, 1]."""
    b = _blocks(x, tile)
    # max = m * 2^p with m in [0.5, 1), and 448 * 2^e = 0.875 * 2^(9 + e).
    m, p = torch.frexp(b.abs().amax(dim=(1, 3), keepdim=True))
    e = torch.where(m > 0, p - 9 + (m > 0.875).to(torch.int32), -64).clamp(min=-64)
    return torch.ldexp(b, -e).to(torch.float8_e4m3fn), e


def _unpack(codes, e, rows, k):
    v = torch.ldexp(codes.float(), e)
    return v.reshape(v.shape[0] * v.shape[1], -1)[:rows, :k]


def _operand(t, name, rows, k):
    """An operand as 32-bit values: packed before, or packed here."""
    codes, e = t[name] if isinstance(t[name], tuple) else _pack(t[name], 1)
    return _unpack(codes, e, rows, k)


def prepare(case, seed):
    t = _inputs(case, seed)
    if own:
        return _calls(case, t)
    for name in ("w", "w1", "w2"):
        if name in t:
            t[name] = _pack(t[name], 128)
    if case.get("input") == "packed":
        t["x"] = _pack(t["x"], 1)
    return {"case": case, "in": t}


def run(state):
    if own:
        gpu = state["gpu"]
        [gpu.check(function(*args), function.__name__) for function, args in state["calls"]]
        return state["out"]
    case, t = state["case"], state["in"]
    rows, kind = case["rows"], case["kind"]
    if kind == "linear":
        y = _operand(t, "x", rows, case["k"]) @ _operand(t, "w", case["n"], case["k"]).T
        if case["bias"]:
            y = y + t["bias"].float()
        return [y.to(torch.bfloat16)]
    if kind == "mlp":
        hidden = case["hidden"]
        y = _operand(t, "x", rows, case["k"]) @ _operand(t, "w1", 2 * hidden, case["k"]).T
        a = y[:, :hidden] / (1 + torch.exp(-y[:, :hidden])) * y[:, hidden:]
        a = _unpack(*_pack(a, 1), rows, hidden)
        return [(a @ _operand(t, "w2", case["n"], hidden).T).to(torch.bfloat16)]
    width = case["width"]
    if kind == "swiglu":
        gate, up = t["fused"].float().split(width, dim=1)
        return [_unpack(*_pack(gate / (1 + torch.exp(-gate)) * up, 1), rows, width).to(torch.bfloat16)]
    r, branch = t["residual"].float(), t["branch"].float()
    if case["adaln"]:
        at = t["map"].long()
        gate, shift, scale = (t["mod"][:, s].float()[at] for s in (2, 3, 4))
        branch = branch * gate
    total = (r + branch).to(torch.bfloat16)
    r = total.float()
    y = r * torch.rsqrt((r * r).mean(dim=1, keepdim=True) + EPS) * t["norm"].float()
    if case["adaln"]:
        y = y * (1 + scale) + shift
    return [total, _unpack(*_pack(y, 1), rows, width).to(torch.bfloat16)]


# ------------------------------------------------------------------ work
def work(case):
    """Each input read once and each result written once; a packed matrix has a byte a value,
    and a byte for each block."""
    kind, m = case["kind"], case["rows"]
    blocks = lambda k: -(-k // 128)  # noqa: E731
    packed = lambda rows, k: rows * (k + blocks(k))  # noqa: E731
    weight = lambda n, k: n * k + blocks(n) * blocks(k)  # noqa: E731
    if kind in ("linear", "mlp"):
        k, n = case["k"], case["n"]
        x = packed(m, k) if case["input"] == "packed" else m * k * 2
        if kind == "linear":
            return {"bytes": x + weight(n, k) + m * n * 2 + (2 * n if case["bias"] else 0), "flops": 2.0 * m * n * k}
        h = case["hidden"]
        return {"bytes": x + weight(2 * h, k) + weight(n, h) + m * n * 2, "flops": 2.0 * m * (2 * h * k + n * h)}
    w = case["width"]
    if kind == "swiglu":
        return {"bytes": m * w * 4 + packed(m, w), "flops": 12.0 * m * w}
    extra = 2 * 3 * w * 2 + m * 4 if case["adaln"] else 0
    return {"bytes": m * w * 6 + packed(m, w) + w * 2 + extra, "flops": (14.0 if case["adaln"] else 10.0) * m * w}


# ------------------------------------------------------------------ 64-bit answers
def _e4m3(v):
    """v in 64 bits to the nearest value of E4M3, ties to even: steps of 2^-9 below 2^-6, of an
    eighth of the power of two above."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(v / step) * step


def _quantized(x, tile):
    """The 64-bit values that the packed x stands for."""
    rows, k = x.shape
    full = torch.zeros((-(-rows // tile) * tile, -(-k // 128) * 128), device=x.device, dtype=torch.float64)
    full[:rows, :k] = x.double()
    b = full.view(-1, tile, full.shape[1] // 128, 128)
    top = b.abs().amax(dim=(1, 3), keepdim=True)
    e = torch.ceil(torch.log2((top / 448).clamp(min=2.0 ** -64)))
    # log2's last bit next to a power of two.
    e = torch.where(top > 448 * torch.exp2(e), e + 1, torch.where((top <= 448 * torch.exp2(e - 1)) & (e > -64), e - 1, e))
    scale = torch.exp2(e)
    return (_e4m3(b / scale) * scale).view(full.shape)[:rows, :k]


def exact(case, seed):
    t, kind = _inputs(case, seed), case["kind"]
    if kind == "linear":
        y = _quantized(t["x"], 1) @ _quantized(t["w"], 128).T
        return [y + t["bias"].double() if case["bias"] else y]
    if kind == "mlp":
        y = _quantized(t["x"], 1) @ _quantized(t["w1"], 128).T
        gate, up = y[:, :case["hidden"]], y[:, case["hidden"]:]
        return [_quantized(gate * torch.sigmoid(gate) * up, 1) @ _quantized(t["w2"], 128).T]
    if kind == "swiglu":
        gate, up = (v.double() for v in t["fused"].chunk(2, dim=1))
        return [_quantized(gate * torch.sigmoid(gate) * up, 1)]
    residual, branch = t["residual"].double(), t["branch"].double()
    mod = t["mod"].double()[t["map"].long()] if case["adaln"] else None
    total = residual + (branch * mod[:, 2] if case["adaln"] else branch)
    r = total.to(torch.bfloat16).double()
    y = r / torch.sqrt((r ** 2).mean(dim=1, keepdim=True) + EPS) * t["norm"].double()
    if case["adaln"]:
        y = y + y * mod[:, 4] + mod[:, 3]
    return [total, _quantized(y, 1)]
