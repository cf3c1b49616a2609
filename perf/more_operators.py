"""The operators of a step that serves several requests at once: what is timed, on which
inputs, and their plain forms.

The rows of the requests (two of a guidance pair, or users' clips of different sizes and
lengths) lie behind one another in one tensor and share the model's weights.

  attention  softmax(scale * Q K^T) V within each of the sequences that the rows hold, for
             queries and keys of different lengths and for fewer key heads than query heads;
             a query of a sequence without keys gets zeros
  rope       the root-mean-square norm of each query and key head and its rotation by a
             position of several axes (time, row, column), from the fused QKV rows
  adapters   base + scale_a * (x . A_a^T) . B_a^T, a low-rank adapter a of its own for each row
             or none; with the shared projection base = x . W^T + bias in the same call, or
             beside a base that is there

Sizes are those of the two block geometries that the library ships
(h3cli_amd.runtime.DitSynth), "synthetic" (hidden 5120, 40 heads, 27 x 30 x 40 video rows and
1024 audio rows) and "h3" (hidden 5376, 56 heads, 48 rotated pairs, frames of 27 x 27 rows),
and generic odd ones.
"""
import ctypes as C
import math

import numpy as np
import torch

own = False

DIM = 128
HIDDEN, INNER = 5376, 7168
SHAPES = [(HIDDEN, 3 * INNER), (INNER, HIDDEN), (5120, 3 * 5120), (5120, 5120)]
SCALE = 0.08837890625   # 1 / sqrt(128) in BF16
EPS = 1e-5
PAIRS_MOST, ATTENTION_MOST = 33424 * 120 * 128, 40 * 7.5e7


def listed():
    return [
        # A query row or a few of each of three short sequences: the smallest call.
        {"name": "attention_short", "kind": "attention", "q": "1,7,64", "k": "1,7,64", "heads": 8, "kv_heads": 8},
        # One 27 x 27 latent frame with and without its condition rows, a guidance pair.
        {"name": "attention_pair", "kind": "attention", "q": "729,806", "k": "729,806", "heads": 56, "kv_heads": 56},
        # Single rows over long contexts that are kept, one of them empty: bound by the keys' reads.
        {"name": "attention_rows", "kind": "attention", "q": "1,1,3,1,1", "k": "18225,4001,729,0,9000", "heads": 40,
         "kv_heads": 8},
        # Clips of four users, no length a multiple of anything.
        {"name": "attention_clips", "kind": "attention", "q": "8193,301,2917,1", "k": "8193,301,2917,1", "heads": 40,
         "kv_heads": 40},
        # A few condition rows: the smallest call.
        {"name": "rope_rows", "kind": "rope", "grids": "1x1x5", "heads": 56, "kv_heads": 56, "dim": 128, "pairs": 48,
         "grouped": True, "norm": True, "interleaved": False, "start": 0.0, "pace": 1.0},
        # A clip of the "h3" geometry, its last frames far into a long video.
        {"name": "rope_clip", "kind": "rope", "grids": "25x27x27", "heads": 56, "kv_heads": 56, "dim": 128, "pairs": 48,
         "grouped": True, "norm": True, "interleaved": False, "start": 90000.0, "pace": 1.0},
        # The joint sequence of the "synthetic" geometry, video then audio (one row a tick).
        {"name": "rope_joint", "kind": "rope", "grids": "27x30x40,1024x1x1", "heads": 40, "kv_heads": 40, "dim": 128,
         "pairs": 64, "grouped": False, "norm": True, "interleaved": False, "start": 0.0, "pace": 0.96},
        # Nothing is a multiple of eight, key heads are shared.
        {"name": "rope_ragged", "kind": "rope", "grids": "3x17x19,1x5x1", "heads": 6, "kv_heads": 2, "dim": 90,
         "pairs": 37, "grouped": False, "norm": True, "interleaved": True, "start": 1000.0, "pace": 0.37},
        # Conditioning rows of nine users, each with an adapter: bound by the adapters' reads.
        {"name": "adapters_rows", "kind": "adapters", "rows": 9, "k": HIDDEN, "n": 6 * HIDDEN, "ranks": "16," * 8 + "64",
         "order": "runs", "none": 0.0, "weight": False, "bias": False},
        # Mixed rows, odd ranks, nothing is a multiple of eight.
        {"name": "adapters_ragged", "kind": "adapters", "rows": 301, "k": 1001, "n": 777, "ranks": "1,40,7,19", "order": "mixed",
         "none": 0.25, "weight": True, "bias": True},
        # Four clips of one latent frame beside the QKV rows that the shared projection left.
        {"name": "adapters_frames", "kind": "adapters", "rows": 2916, "k": HIDDEN, "n": 3 * INNER, "ranks": "32,16,64,32",
         "order": "runs", "none": 0.0, "weight": False, "bias": False},
        # A long clip and the next ones through the output projection, one of them without adapter.
        {"name": "adapters_clips", "kind": "adapters", "rows": 8193, "k": INNER, "n": HIDDEN, "ranks": "32,128,64",
         "order": "runs", "none": 0.25, "weight": True, "bias": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the ranges above; costs are bounded by the listed ones."""
    kind = rng.choice(["attention", "rope", "adapters"])
    if kind == "attention":
        kv_heads = rng.choice([1, 2, 3, 8, 40, 56])
        heads = kv_heads * (1 if kv_heads >= 40 else rng.choice([1, 2, 5, 7]))
        form = rng.choice(["self", "self", "cross", "rows"])
        most = ATTENTION_MOST / heads
        q, k = [], []
        for _ in range(rng.randint(1, 8)):
            left = most - sum(a * b for a, b in zip(q, k))
            a = rng.randint(1, 4) if form == "rows" else _log(rng, 1, max(1, min(9000, math.isqrt(int(left)))))
            b = a if form == "self" else 0 if rng.random() < 0.1 else _log(rng, 1, max(1, min(18225, left / a)))
            if left < a * max(b, 1):
                break
            q.append(a)
            k.append(b)
        return {"kind": kind, "q": ",".join(map(str, q or [1])), "k": ",".join(map(str, k or [1])), "heads": heads,
                "kv_heads": kv_heads}
    if kind == "rope":
        dim = rng.choice([128, 128, 64, 2 * rng.randint(3, 128)])
        kv_heads = rng.choice([1, 2, 3, 8, 40, 56])
        heads = kv_heads * (1 if kv_heads >= 40 else rng.choice([1, 2, 5, 7]))
        pairs = rng.choice([dim // 2, max(3, dim * 3 // 8), rng.randint(3, dim // 2)])
        rows = _log(rng, 1, min(33424, PAIRS_MOST // ((heads + 2 * kv_heads) * dim)))
        grids = []
        while rows > 0 and len(grids) < 4:
            h, w = rng.randint(1, min(30, rows)), rng.randint(1, 40)
            w = min(w, max(1, rows // h))
            f = max(1, _log(rng, 1, max(1, rows // (h * w))))
            grids.append("%dx%dx%d" % (f, h, w))
            rows -= f * h * w
        return {"kind": kind, "grids": ",".join(grids), "heads": heads, "kv_heads": kv_heads, "dim": dim, "pairs": pairs,
                "grouped": rng.random() < 0.5, "norm": rng.random() < 0.7, "interleaved": rng.random() < 0.5,
                "start": float(rng.choice([0, 0, 1000, rng.randint(0, 90000)])), "pace": rng.choice([1.0, 0.96, rng.uniform(0.1, 2)])}
    ranks = [rng.choice([4, 8, 16, 16, 32, 32, 64, 128, rng.randint(1, 128)]) for _ in range(rng.choice([1, 2, 3, 4, 9]))]
    k, n = rng.choice(SHAPES + [(_log(rng, 40, 8000), _log(rng, 40, 8000))])
    weight = rng.random() < 0.4
    rows = _log(rng, 1, min(8193, 8193 * INNER * HIDDEN // (k * n)) if weight else 8193)
    return {"kind": kind, "rows": rows, "k": k, "n": n, "ranks": ",".join(map(str, ranks)), "order": rng.choice(["runs", "mixed"]),
            "none": rng.choice([0.0, 0.0, 0.25]), "weight": weight, "bias": weight and rng.random() < 0.5}


# ------------------------------------------------------------------ inputs
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 6151 + 17)
    return g


def _normal(g, shape, scale=1.0, shift=0.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale + shift).to(torch.bfloat16)


def _activation(g, rows, k):
    """Rows whose channels differ in scale, one of a hundred by much, as norms give them."""
    scale = torch.exp(0.5 * torch.randn((k,), generator=g, device="cuda"))
    scale = torch.where(torch.rand((k,), generator=g, device="cuda") < 0.01, 16 * scale, scale)
    return (torch.randn((rows, k), generator=g, device="cuda") * scale).to(torch.bfloat16)


def _lengths(text):
    return [int(v) for v in text.split(",")]


def _grids(case):
    return [[int(v) for v in grid.split("x")] for grid in case["grids"].split(",")]


def _frequencies(pairs):
    """The rotation's pairs: a third of them for each axis, theta^(-i / pairs of the axis)."""
    count = [pairs - 2 * (pairs // 3), pairs // 3, pairs // 3]
    values = [10000.0 ** (-i / n) for n in count for i in range(n)]
    return np.asarray(values, np.float64), np.repeat(np.arange(3, dtype=np.uint32), count)


def _row_map(case, seed):
    """The adapter of each row; the number of adapters stands for none."""
    rng, rows, count = np.random.RandomState(seed % (1 << 31)), case["rows"], len(_lengths(case["ranks"]))
    kept = rows - int(rows * case["none"])
    at = np.full(rows, count, np.uint32)
    cuts = np.sort(rng.randint(0, kept + 1, count - 1)) if count < kept else np.arange(1, count)
    at[:kept] = np.searchsorted(cuts, np.arange(kept), side="right")
    return rng.permutation(at) if case["order"] == "mixed" else at


def _inputs(case, seed):
    g, kind = _generator(seed), case["kind"]
    if kind == "attention":
        q, k = sum(_lengths(case["q"])), sum(_lengths(case["k"]))
        return {"q": _normal(g, (q, case["heads"], DIM), 1.5), "k": _normal(g, (k, case["kv_heads"], DIM), 1.5),
                "v": _normal(g, (k, case["kv_heads"], DIM))}
    if kind == "rope":
        parts = []
        for f, h, w in _grids(case):
            f, h, w = torch.meshgrid(*(torch.arange(n, device="cuda", dtype=torch.float64) for n in (f, h, w)), indexing="ij")
            parts.append(torch.stack([case["start"] + case["pace"] * f, h, w], dim=-1).reshape(-1, 3))
        positions = torch.cat(parts).float()
        heads = case["heads"] + 2 * case["kv_heads"]
        t = {"qkv": _activation(g, positions.shape[0], heads * case["dim"]), "positions": positions}
        if case["norm"]:
            t["q_norm"], t["k_norm"] = _normal(g, (case["dim"],), 0.1, 1.0), _normal(g, (case["dim"],), 0.1, 1.0)
        return t
    rows, k, n, ranks = case["rows"], case["k"], case["n"], _lengths(case["ranks"])
    t = {"x": _activation(g, rows, k), "map": _row_map(case, seed),
         "down": [_normal(g, (r, k), 1 / math.sqrt(k)) for r in ranks],
         "up": [_normal(g, (n, r), 0.5 / math.sqrt(r)) for r in ranks], "scales": [2.0 / (1 + a % 3) for a in range(len(ranks))]}
    if case["weight"]:
        t["w"] = _normal(g, (n, k), 1 / math.sqrt(k))
        if case["bias"]:
            t["bias"] = _normal(g, (n,), 0.1)
    else:
        t["base"] = _normal(g, (rows, n))
    return t


# ------------------------------------------------------------------ the library's tensors
class _Buffer:
    """A device tensor of the library, seen by torch without a copy. torch keeps this object
    alive with the views, and the memory goes back with it."""

    def __init__(self, gpu, shape, dtype=torch.bfloat16):
        from h3cli_amd import _lib
        kind, code = {torch.bfloat16: (_lib.BF16, "<i2"), torch.float32: (_lib.F32, "<f4")}[dtype]
        self.gpu, self.dtype = gpu, dtype
        self.tensor = gpu.empty(max(math.prod(shape), 1), kind)
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


class _Plan:
    """A plan or a set of weights of the library, with what frees it."""

    def __init__(self, gpu, handle, free):
        gpu.check(handle, "plan")
        self.gpu, self.handle, self.free = gpu, handle, free

    def __del__(self):
        if self.gpu.handle:
            self.free(self.handle)


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


def _u32(values):
    return (C.c_uint32 * len(values))(*(int(v) for v in values))


def _calls(case, t):
    """The library's calls of one pass, and the tensors that they write."""
    gpu = _context()
    lib, g, kind = gpu.lib, gpu.handle, case["kind"]
    held = {name: _put(gpu, v) for name, v in t.items() if isinstance(v, torch.Tensor)}
    h = {name: b.handle for name, b in held.items()}
    if kind == "attention":
        ends = [np.cumsum([0] + _lengths(case[name])) for name in ("q", "k")]
        plan = _Plan(gpu, lib.h3_hip_sequences_new(g, _u32(ends[0]), _u32(ends[1]), len(ends[0]) - 1, case["heads"],
                                                   case["kv_heads"]), lib.h3_hip_sequences_free)
        outs = [_Buffer(gpu, tuple(t["q"].shape))]
        call = (lib.h3_hip_sdpa_sequences_bf16, (g, outs[0].handle, h["q"], h["k"], h["v"], plan.handle, C.c_float(SCALE)))
        keep = [held, plan]
    elif kind == "rope":
        values, axis = _frequencies(case["pairs"])
        plan = _Plan(gpu, lib.h3_hip_rope_axes_new(g, (C.c_double * len(values))(*values), _u32(axis), case["pairs"], 3,
                                                   int(case["interleaved"])), lib.h3_hip_rope_axes_free)
        rows, heads, kv_heads, dim = t["qkv"].shape[0], case["heads"], case["kv_heads"], case["dim"]
        outs = [_Buffer(gpu, (rows, n, dim)) for n in (heads, kv_heads, kv_heads)]
        call = (lib.h3_hip_qkv_rope_axes_bf16,
                (g, outs[0].handle, outs[1].handle, outs[2].handle, h["qkv"], h.get("q_norm"), h.get("k_norm"), plan.handle,
                 h["positions"], rows, heads, kv_heads, dim, int(case["grouped"]), C.c_float(EPS)))
        keep = [held, plan]
    else:
        rows, k, n, ranks = case["rows"], case["k"], case["n"], _lengths(case["ranks"])
        adapters = _Plan(gpu, lib.h3_hip_adapters_new(g, _u32(ranks), len(ranks), k, n), lib.h3_hip_adapters_free)
        for a in range(len(ranks)):
            down, up = _put(gpu, t["down"][a]), _put(gpu, t["up"][a])
            gpu.check(lib.h3_hip_adapters_set(g, adapters.handle, a, down.handle, up.handle, C.c_float(t["scales"][a])), "adapter")
            gpu.check(lib.h3_gpu_synchronize(g), "adapter")
        plan = _Plan(gpu, lib.h3_hip_adapter_rows_new(g, _u32(t["map"]), rows, len(ranks), max(ranks)),
                     lib.h3_hip_adapter_rows_free)
        outs = [_Buffer(gpu, (rows, n))]
        if case["weight"]:
            call = (lib.h3_hip_linear_adapters_bf16, (g, outs[0].handle, h["x"], h["w"], h.get("bias"), adapters.handle,
                                                      plan.handle, rows, k, n))
        else:
            call = (lib.h3_hip_adapters_add_bf16, (g, outs[0].handle, h["base"], h["x"], adapters.handle, plan.handle,
                                                   rows, k, n))
        keep = [held, adapters, plan]
    return {"gpu": gpu, "call": call, "keep": keep, "out": [b.view() for b in outs]}


# ------------------------------------------------------------------ the plain forms
def prepare(case, seed):
    t = _inputs(case, seed)
    if own:
        return _calls(case, t)
    if case["kind"] == "rope":
        values, axis = _frequencies(case["pairs"])
        t["frequencies"], t["axis"] = torch.from_numpy(values).cuda(), torch.from_numpy(axis.astype(np.int64)).cuda()
    if case["kind"] == "adapters":
        # All adapters' ranks behind one another; row r takes the ones of its adapter.
        ranks = _lengths(case["ranks"])
        owner = torch.repeat_interleave(torch.arange(len(ranks)), torch.tensor(ranks)).cuda()
        t["takes"] = torch.from_numpy(t.pop("map").astype(np.int64)).cuda()[:, None] == owner
        t["scale"] = torch.tensor(t.pop("scales"), device="cuda")[owner]
        t["down"], t["up"] = torch.cat(t["down"]), torch.cat(t["up"], dim=1)
    return {"case": case, "in": t}


def _attention(q, k, v, share):
    """softmax(SCALE * q k^T) v: q [rows, heads, DIM], a key head for `share` query heads."""
    if not k.shape[0]:
        return torch.zeros_like(q)
    q = q.float().unflatten(1, (-1, share)).permute(1, 2, 0, 3).flatten(1, 2)
    s = SCALE * (q @ k.float().permute(1, 2, 0).contiguous())
    p = torch.exp(s - s.amax(dim=2, keepdim=True))
    y = (p @ v.float().transpose(0, 1).contiguous()) / p.sum(dim=2, keepdim=True)
    return y.unflatten(1, (share, -1)).permute(2, 0, 1, 3).flatten(1, 2).to(torch.bfloat16)


def run(state):
    if own:
        function, args = state["call"]
        state["gpu"].check(function(*args), function.__name__)
        return state["out"]
    case, t = state["case"], state["in"]
    if case["kind"] == "attention":
        share = case["heads"] // case["kv_heads"]
        q, (k, v) = t["q"].split(_lengths(case["q"])), (t[n].split(_lengths(case["k"])) for n in ("k", "v"))
        return [torch.cat([_attention(*part, share) for part in zip(q, k, v)])]
    if case["kind"] == "rope":
        rows, heads, kv_heads, dim, pairs = t["qkv"].shape[0], case["heads"], case["kv_heads"], case["dim"], case["pairs"]
        if case["grouped"]:
            q, k, v = t["qkv"].view(rows, kv_heads, -1, dim).split([heads // kv_heads, 1, 1], dim=2)
            q, k, v = q.flatten(1, 2), k.flatten(1, 2), v.flatten(1, 2)
        else:
            q, k, v = t["qkv"].view(rows, -1, dim).split([heads, kv_heads, kv_heads], dim=1)
        angle = t["positions"].double()[:, t["axis"]] * t["frequencies"]
        c, s = (f(angle).float()[:, None] for f in (torch.cos, torch.sin))

        def turned(x, weight):
            x = x.float()
            if weight is not None:
                x = x * torch.rsqrt((x * x).mean(dim=2, keepdim=True) + EPS) * weight.float()
            a, b, rest = x.split([pairs, pairs, dim - 2 * pairs], dim=2)
            if case["interleaved"]:
                a, b = x[:, :, 0:2 * pairs:2], x[:, :, 1:2 * pairs:2]
                return torch.cat([torch.stack([a * c - b * s, b * c + a * s], dim=3).flatten(2), rest], dim=2).to(torch.bfloat16)
            return torch.cat([a * c - b * s, b * c + a * s, rest], dim=2).to(torch.bfloat16)

        return [turned(q, t.get("q_norm")), turned(k, t.get("k_norm")), v.clone()]
    low = (t["x"].float() @ t["down"].float().T) * t["scale"] * t["takes"]
    y = low @ t["up"].float().T
    if case["weight"]:
        y = y + t["x"].float() @ t["w"].float().T
        return [(y + t["bias"].float() if case["bias"] else y).to(torch.bfloat16)]
    return [(t["base"].float() + y).to(torch.bfloat16)]


# ------------------------------------------------------------------ work
def work(case):
    """Each input read once and each result written once; weights of 2 bytes."""
    kind = case["kind"]
    if kind == "attention":
        q, k = _lengths(case["q"]), _lengths(case["k"])
        return {"bytes": 4 * DIM * (case["heads"] * sum(q) + case["kv_heads"] * sum(k)),
                "flops": 4.0 * DIM * case["heads"] * sum(a * b for a, b in zip(q, k))}
    if kind == "rope":
        rows = sum(math.prod(grid) for grid in _grids(case))
        values = rows * (case["heads"] + 2 * case["kv_heads"]) * case["dim"]
        turned = rows * (case["heads"] + case["kv_heads"]) * case["dim"]
        return {"bytes": 4 * values + 12 * rows, "flops": turned * (8.0 if case["norm"] else 3.0)}
    rows, k, n, ranks = case["rows"], case["k"], case["n"], _lengths(case["ranks"])
    at = _row_map(case, 1)
    used = np.bincount(at, minlength=len(ranks) + 1)
    low = sum(int(used[a]) * r for a, r in enumerate(ranks))
    adapted = rows - int(used[len(ranks)])
    weights = sum(r * (k + n) for a, r in enumerate(ranks) if used[a])
    if case["weight"]:
        return {"bytes": 2 * (rows * (k + n) + n * k + weights + (n if case["bias"] else 0)),
                "flops": 2.0 * (rows * k * n + low * (k + n))}
    return {"bytes": 2 * (adapted * k + 2 * rows * n + weights) + 4 * rows, "flops": 2.0 * low * (k + n)}


# ------------------------------------------------------------------ 64-bit answers
def exact(case, seed):
    t = _inputs(case, seed)
    if case["kind"] == "attention":
        heads, share = case["heads"], case["heads"] // case["kv_heads"]
        out = torch.zeros(t["q"].shape, device="cuda", dtype=torch.float64)
        ends = [np.cumsum([0] + _lengths(case[name])) for name in ("q", "k")]
        for i in range(len(ends[0]) - 1):
            q0, q1, k0, k1 = int(ends[0][i]), int(ends[0][i + 1]), int(ends[1][i]), int(ends[1][i + 1])
            for head in range(heads if k1 > k0 else 0):
                k, v = (t[n][k0:k1, head // share].double() for n in ("k", "v"))
                out[q0:q1, head] = torch.softmax(SCALE * torch.mm(t["q"][q0:q1, head].double(), k.T), dim=1).mm(v)
        return [out]
    if case["kind"] == "rope":
        rows, heads, kv_heads, dim, pairs = t["qkv"].shape[0], case["heads"], case["kv_heads"], case["dim"], case["pairs"]
        share, x = heads // kv_heads, t["qkv"].double().view(t["qkv"].shape[0], -1, dim)
        at = torch.arange(heads + 2 * kv_heads, device="cuda")
        if case["grouped"]:
            at = at.view(kv_heads, share + 2)
            at = [at[:, :share].flatten(), at[:, share], at[:, share + 1]]
        else:
            at = [at[:heads], at[heads:heads + kv_heads], at[heads + kv_heads:]]
        values, axis = _frequencies(pairs)
        angle = t["positions"].double()[:, torch.from_numpy(axis.astype(np.int64)).cuda()] * torch.from_numpy(values).cuda()
        turn = torch.polar(torch.ones_like(angle), angle)[:, None]
        first = torch.arange(pairs, device="cuda") * (2 if case["interleaved"] else 1)
        second = first + (1 if case["interleaved"] else pairs)
        outs = []
        for part, name in zip(at, ("q_norm", "k_norm", None)):
            y = x[:, part]
            if name is not None:
                if case["norm"]:
                    y = y / torch.sqrt(y.square().mean(dim=2, keepdim=True) + EPS) * t[name].double()
                z = torch.complex(y[:, :, first], y[:, :, second]) * turn
                y[:, :, first], y[:, :, second] = z.real, z.imag
            outs.append(y)
        return outs
    x = t["x"].double()
    y = torch.mm(x, t["w"].double().T) if case["weight"] else t["base"].double()
    if case["bias"]:
        y += t["bias"].double()
    for a, scale in enumerate(t["scales"]):
        at = torch.from_numpy(np.flatnonzero(t["map"] == a)).cuda()
        y[at] += scale * x[at].mm(t["down"][a].double().T).mm(t["up"][a].double().T)
    return [y]
