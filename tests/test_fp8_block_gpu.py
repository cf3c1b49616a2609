"""Block-scaled FP8 (include/h3_hip_ext.h, h3_hip_fp8_block_*): packing bit for bit, the
projections, norms, SwiGLU and the MLP against their definitions in 64 bits, as a chain, in a
graph, and what they refuse.

Bounds. A packed value is off by half a step: 2^-4 of it, or 2^-10 of its scale below E4M3's
normal range. A BF16 result rounds by 2^-8. The matrix core adds the products of an instruction
with about 14 bits behind the largest (measured: at most 1.5e-4 of the sum of their magnitudes,
for codes of all exponents): 2^-12 of the sum of the magnitudes covers it, and the FP32 sums
across instructions (K / 64 of them, 2^-24 each) are small beside that."""
import ctypes as C
import math

import numpy as np
import pytest

from h3cli_amd import _lib, synth
from h3cli_amd.runtime import Gpu, H3Error
from tests.helpers import bf16
from tests.test_capture_gpu import Graph

pytestmark = pytest.mark.gpu

MFMA = 2.0 ** -12
HALF_BF16 = 2.0 ** -8


def e4m3(v):
    """v to the nearest E4M3 value, ties to even."""
    a = np.abs(v)
    step = np.exp2(np.maximum(np.floor(np.log2(np.maximum(a, 2.0 ** -20))), -6) - 3)
    return np.rint(v / step) * step


def decode(codes):
    c = codes.astype(np.int64)
    e, m = (c >> 3) & 15, c & 7
    v = np.where(e > 0, np.ldexp(1 + m / 8, e - 7), m * 2.0 ** -9)
    return np.where(c & 128, -v, v)


def exponents(amax):
    """Least e >= -64 with amax <= 448 * 2^e."""
    m, p = np.frexp(amax)
    return np.where(amax > 0, np.maximum(p - 9 + (m > 0.875), -64), -64).astype(np.int64)


def blocks(x, tile):
    """x [rows, k] as [row blocks, tile, column blocks, 128]."""
    rows, k = x.shape
    full = np.zeros((-(-rows // tile) * tile, -(-k // 128) * 128))
    full[:rows, :k] = x
    return full.reshape(-1, tile, full.shape[1] // 128, 128)


def quantized(x, tile):
    """(values that the packed x stands for, exponents [row blocks, column blocks])."""
    b = blocks(x, tile)
    e = exponents(np.abs(b).max(axis=(1, 3)))
    s = np.ldexp(1.0, e)[:, None, :, None]
    return (e4m3(b / s) * s).reshape(-1, b.shape[2] * 128)[:x.shape[0], :x.shape[1]], e


class Packed:
    def __init__(self, g, handle, rows, columns, tile):
        if not handle:
            raise H3Error(g.error())
        self.g, self.rows, self.columns, self.tile = g, rows, columns, tile
        stride, scales, groups, size = (C.c_size_t() for _ in range(4))
        assert g.lib.h3_hip_fp8_block_layout(rows, columns, tile, stride, scales, groups, size)
        self.stride, self.scales, self.groups, self.bytes = (v.value for v in (stride, scales, groups, size))
        self.tensor = g._track(handle, rows * columns, _lib.I8)
        self.handle = handle

    def raw(self):
        out = np.empty(self.bytes, np.uint8)
        self.g.check(self.g.lib.h3_hip_tensor_copy_to_host(self.handle, out.ctypes.data, out.size), "read")
        return out

    def read(self):
        """codes [rows, stride], scale bytes [scale rows, blocks]."""
        raw = self.raw()
        n = -(-self.rows // self.tile)
        codes = raw[:self.rows * self.stride].reshape(self.rows, self.stride)
        scales = raw[self.scales:].reshape(-1, self.groups, 32, 4).transpose(0, 2, 1, 3).reshape(-1, self.groups * 4)
        scales = scales[:n, :-(-self.columns // 128)]
        return codes, scales

    def values(self):
        codes, scales = self.read()
        s = np.ldexp(1.0, scales.astype(np.int64) - 127)
        s = np.repeat(np.repeat(s, self.tile, axis=0)[:self.rows], 128, axis=1)
        return (decode(codes) * s)[:, :self.columns]


def new(g, rows, columns, tile=1):
    return Packed(g, g.lib.h3_hip_fp8_block_new(g.handle, rows, columns, tile), rows, columns, tile)


def weight(g, bits, rows, columns):
    t = g.from_bf16(bits)
    return Packed(g, g.lib.h3_hip_fp8_block_weight_from_bf16(g.handle, t.handle, rows, columns), rows, columns, 128)


def activation(g, bits, rows, columns):
    t, p = g.from_bf16(bits), new(g, rows, columns)
    g.begin()
    g.check(g.lib.h3_hip_fp8_block_pack(g.handle, p.handle, t.handle, rows, columns), "pack")
    g.submit()
    return p


def values(rows, columns, seed, spread=3.0):
    """BF16 bits whose scale differs from column to column and from row to row."""
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((rows, columns)) * np.exp2(rng.uniform(-spread, spread, columns)) * \
        np.exp2(rng.uniform(-spread, spread, (rows, 1)))
    return synth.f32_to_bf16(x.astype(np.float32))


def within(got, want, bound, what=""):
    off = np.abs(np.asarray(got, np.float64) - want) - bound
    assert np.all(off <= 0), (what, np.unravel_index(np.argmax(off), off.shape), float(off.max()))


# ------------------------------------------------------------------ packing
@pytest.mark.parametrize("rows,columns", [(1, 1), (1, 128), (3, 127), (5, 129), (2, 8), (130, 1000), (7, 5376), (257, 264)])
def test_pack_bit_exact(rows, columns):
    """Codes, scales and padding of both tiles; a zero block, a block with the largest BF16
    value, values at a scale's border (448, the next BF16 value) and far below it."""
    print(f"[fp8 block] pack {rows}x{columns}", flush=True)
    bits = values(rows, columns, rows + columns)
    x = bf16(bits).reshape(rows, columns).copy()
    x[0, 0] = 448.0 if columns < 200 else 450.0
    if columns > 256:
        x[0, 128:256] = 0.0
        x[rows - 1, columns - 1] = bf16(np.array([0x7f7f], np.uint16))[0]
        x[rows // 2, 0:128] = np.ldexp(x[rows // 2, 0:128], -90)
    bits = synth.f32_to_bf16(x.astype(np.float32).reshape(-1))
    x = bf16(bits).reshape(rows, columns).astype(np.float64)
    with Gpu() as g:
        for tile in (1, 128):
            p = activation(g, bits, rows, columns) if tile == 1 else weight(g, bits, rows, columns)
            want, e = quantized(x, tile)
            codes, scales = p.read()
            assert np.array_equal(scales.astype(np.int64) - 127, e)
            assert np.array_equal(p.values(), want)
            assert not codes[:, columns:].any()
            out = g.empty(rows * columns)
            g.begin()
            g.check(g.lib.h3_hip_fp8_block_unpack(g.handle, out.handle, p.handle, rows, columns), "unpack")
            g.submit()
            # BF16's largest value is 1.9921875 * 2^127, which E4M3 rounds to 2^8 times a scale of
            # 2^120: 2^128, which the packed matrix holds and BF16 does not (infinity).
            with np.errstate(over="ignore"):
                assert np.array_equal(bf16(out.read()).reshape(rows, columns), want.astype(np.float32))


def test_from_packed_and_copy_back():
    rng = np.random.default_rng(3)
    with Gpu() as g:
        for rows, columns, tile in ((1, 1, 1), (5, 300, 1), (300, 200, 128)):
            codes = rng.integers(0, 255, (rows, columns)).astype(np.uint8)
            codes[(codes | 0x80) == 0xff] = 0
            scales = rng.integers(0, 255, (-(-rows // tile), -(-columns // 128))).astype(np.uint8)
            args = (g.handle, codes.ctypes.data, scales.ctypes.data, rows, columns, tile)
            p = Packed(g, g.lib.h3_hip_fp8_block_from_packed(*args), rows, columns, tile)
            got, got_scales = p.read()
            assert np.array_equal(got[:, :columns], codes) and not got[:, columns:].any()
            assert np.array_equal(got_scales, scales)
            codes[rows - 1, columns - 1] = 0xff
            assert not g.lib.h3_hip_fp8_block_from_packed(*args) and "code is not a number" in g.error()
            codes[rows - 1, columns - 1] = 0
            scales[-1, -1] = 0xff
            assert not g.lib.h3_hip_fp8_block_from_packed(*args) and "scale is not a number" in g.error()


# ------------------------------------------------------------------ projections
SHAPES = [(1, 1, 1), (1, 256, 5376), (2, 128, 128), (16, 1000, 77), (17, 129, 130), (33, 640, 257), (64, 4096, 512),
          (65, 5376, 96), (100, 127, 1000), (128, 2048, 640), (129, 1100, 300), (301, 1000, 777), (700, 512, 384),
          (260, 9000, 256), (1025, 256, 520)]


def linear(g, out, x, w, bias, rows, k, n):
    g.begin()
    f = g.lib.h3_hip_linear_fp8_block if isinstance(x, Packed) else g.lib.h3_gpu_linear_bf16
    g.check(f(g.handle, out.handle, x.handle, w.handle, bias.handle if bias else None, rows, k, n), "linear")
    kernel = g.last_kernel()
    g.submit()
    return out.read(rows * n).reshape(rows, n), kernel


@pytest.mark.parametrize("m,k,n", SHAPES)
def test_linear(m, k, n):
    print(f"[fp8 block] linear {m}x{k}x{n}", flush=True)
    with Gpu() as g:
        xb, wb = values(m, k, m + k), values(n, k, n + k + 1, 2.0)
        x, w = activation(g, xb, m, k), weight(g, wb, n, k)
        bits = values(1, n, n)
        bias = g.from_bf16(bits)
        out = g.empty(m * n)
        xv, wv = x.values(), w.values()
        want, size = xv @ wv.T, np.abs(xv) @ np.abs(wv).T
        got, kernel = linear(g, out, x, w, None, m, k, n)
        print(f"[fp8 block] {kernel}", flush=True)
        within(bf16(got), want, HALF_BF16 * np.abs(want) + 2 * MFMA * size, kernel)
        # A BF16 input is packed as h3_hip_fp8_block_pack does, and the bias is added before rounding.
        again, _ = linear(g, out, g.from_bf16(xb), w, None, m, k, n)
        assert np.array_equal(again, got)
        biased, _ = linear(g, out, x, w, bias, m, k, n)
        want = want + bf16(bits).reshape(1, n)
        within(bf16(biased), want, HALF_BF16 * np.abs(want) + 2 * MFMA * size + 2.0 ** -23 * np.abs(want), "bias")


@pytest.mark.parametrize("m,k,n", [s for s in SHAPES if s[1] >= 128] + [(3000, 1500, 1000)])
def test_linear_exact(m, k, n):
    """Codes +-1, +-2 and scales of four powers of two: sums of up to 2^13 * 9000 units of the
    least product, below 2^24 of them per scale, are exact in any order, and each block's scale
    shows. Every output has to be the BF16 rounding of its sum."""
    print(f"[fp8 block] exact {m}x{k}x{n}", flush=True)
    rng = np.random.default_rng(m + n)
    values_of = np.array([0x38, 0xb8, 0x40, 0xc0], np.uint8)      # 1, -1, 2, -2
    kb = -(-k // 128)
    with Gpu() as g:
        xc, wc = (values_of[rng.integers(0, 4, s)] for s in ((m, k), (n, k)))
        xs, ws = (rng.integers(126, 130, s).astype(np.uint8) for s in ((m, kb), (-(-n // 128), kb)))
        x = Packed(g, g.lib.h3_hip_fp8_block_from_packed(g.handle, xc.ctypes.data, xs.ctypes.data, m, k, 1), m, k, 1)
        w = Packed(g, g.lib.h3_hip_fp8_block_from_packed(g.handle, wc.ctypes.data, ws.ctypes.data, n, k, 128), n, k, 128)
        got, kernel = linear(g, g.empty(m * n), x, w, None, m, k, n)
        print(f"[fp8 block] {kernel}", flush=True)
        want = x.values() @ w.values().T
        assert np.array_equal(got, synth.f32_to_bf16(want.astype(np.float32))), kernel


def test_linear_rows_of_a_larger_tensor():
    """Fewer rows than the packed tensor holds: those behind are not read, nor written by the packers."""
    m, held, k, n = 70, 200, 520, 260
    with Gpu() as g:
        xb = values(held, k, 5)
        w = weight(g, values(n, k, 6, 2.0), n, k)
        small, large = activation(g, xb[:m * k], m, k), activation(g, xb, held, k)
        out = g.empty(held * n)
        first, _ = linear(g, out, small, w, None, m, k, n)
        second, _ = linear(g, out, large, w, None, m, k, n)
        assert np.array_equal(first, second)
        before, scales_before = large.read()
        t = g.from_bf16(values(m, k, 7))
        g.begin()
        g.check(g.lib.h3_hip_fp8_block_pack(g.handle, large.handle, t.handle, m, k), "pack")
        g.submit()
        after, scales_after = large.read()
        assert np.array_equal(before[m:], after[m:]) and np.array_equal(scales_before[m:], scales_after[m:])
        assert not np.array_equal(before[:m], after[:m])


# ------------------------------------------------------------------ norms and SwiGLU
def packed_bound(p, y, error):
    """Half a step around y (its FP32 value is `error` off), and the scales' rule."""
    _, scales = p.read()
    s = np.ldexp(1.0, scales.astype(np.int64) - 127)
    amax = np.abs(blocks(y, 1)).max(axis=(1, 3))
    slack = 1 + 2.0 ** -20
    assert np.all(amax <= 448 * s * slack) and np.all((amax * slack > 224 * s) | (scales == 63))
    wide = np.repeat(s, 128, axis=1)[:, :y.shape[1]]
    return np.maximum(2.0 ** -4 * np.abs(y), 2.0 ** -10 * wide) + error


@pytest.mark.parametrize("rows,width", [(1, 8), (2, 128), (3, 136), (5, 5376), (64, 1000), (1100, 520), (2050, 4096), (3, 8192)])
@pytest.mark.parametrize("kind", ["rms", "add", "adaln", "gate"])
def test_norms(rows, width, kind):
    print(f"[fp8 block] {kind} {rows}x{width}", flush=True)
    rng = np.random.default_rng(rows + width)
    eps, slots = 1e-5, 6
    res, branch, norm = values(rows, width, 1, 1.0), values(rows, width, 2, 1.0), values(1, width, 3, 0.5)
    mod = synth.f32_to_bf16((0.3 * rng.standard_normal((3, slots, width))).astype(np.float32))
    row_map = rng.integers(0, 3, rows).astype(np.uint32)
    r, b, w = (bf16(v).reshape(-1, width).astype(np.float64) for v in (res, branch, norm))
    mv = bf16(mod).reshape(3, slots, width).astype(np.float64)[row_map]
    with Gpu() as g:
        tr, tb, tw, tm, tmap = (g.from_bf16(res), g.from_bf16(branch), g.from_bf16(norm), g.from_bf16(mod), g.from_u32(row_map))
        total, packed = g.empty(rows * width), new(g, rows, width)
        lib, h = g.lib, g.handle
        g.begin()
        if kind == "rms":
            ok = lib.h3_hip_add_rms_norm_fp8_block(h, None, packed.handle, tr.handle, None, tw.handle, rows, width, eps)
        elif kind == "add":
            ok = lib.h3_hip_add_rms_norm_fp8_block(h, total.handle, packed.handle, tr.handle, tb.handle, tw.handle, rows,
                                                   width, eps)
        elif kind == "adaln":
            ok = lib.h3_hip_adaln_fp8_block(h, packed.handle, tr.handle, tw.handle, tm.handle, tmap.handle, rows, width,
                                            slots, 3, 4, eps)
        else:
            ok = lib.h3_hip_gate_adaln_fp8_block(h, total.handle, packed.handle, tr.handle, tb.handle, tw.handle, tm.handle,
                                                 tm.handle, tmap.handle, rows, width, slots, 2, 3, 4, eps)
        g.check(ok, kind)
        g.submit()
        x = r
        if kind in ("add", "gate"):
            want = r + (b * mv[:, 2] if kind == "gate" else b)
            x = bf16(total.read()).reshape(rows, width).astype(np.float64)
            # One FP32 addition (or FMA), then BF16.
            within(x, want, (HALF_BF16 + 2.0 ** -23) * np.abs(want))
        y = x / np.sqrt((x * x).mean(axis=1, keepdims=True) + eps) * w
        # The mean's FP32 sum (in 64 and more partial sums of up to 128 terms) and a handful of roundings.
        error = 2.0 ** -19 * np.abs(y)
        if kind in ("adaln", "gate"):
            error = error * np.abs(1 + mv[:, 4]) + 2.0 ** -22 * (np.abs(y) + np.abs(mv[:, 3]))
            y = y * (1 + mv[:, 4]) + mv[:, 3]
        within(packed.values(), y, packed_bound(packed, y, error), kind)
        codes, _ = packed.read()
        assert not codes[:, width:].any()


@pytest.mark.parametrize("rows,width", [(1, 1), (1, 128), (3, 200), (5, 13), (130, 1000), (33, 14336)])
def test_swiglu(rows, width):
    print(f"[fp8 block] swiglu {rows}x{width}", flush=True)
    bits = values(rows, 2 * width, width, 2.0)
    x = bf16(bits).reshape(rows, 2 * width).copy()
    if width > 100:
        x[0, :10] = [0.0, -0.0, 87.0, -87.0, -88.5, -120.0, 300.0, -3e38, 3e38, 1e-39]
        x[0, width:width + 10] = [1.0, 5.0, 1.0, 1e4, 1e4, 1e4, 2.0, 1.0, 0.5, 1.0]
    bits = synth.f32_to_bf16(x.astype(np.float32).reshape(-1))
    x = bf16(bits).reshape(rows, 2 * width).astype(np.float64)
    with Gpu() as g:
        t, packed = g.from_bf16(bits), new(g, rows, width)
        g.begin()
        g.check(g.lib.h3_hip_swiglu_fp8_block(g.handle, packed.handle, t.handle, rows, width), "swiglu")
        g.submit()
        gate, up = x[:, :width], x[:, width:]
        y = gate * np.exp(-np.logaddexp(0, -gate)) * up
        within(packed.values(), y, packed_bound(packed, y, 2.0 ** -21 * np.abs(y)))
        assert not packed.read()[0][:, width:].any()


# ------------------------------------------------------------------ the MLP
def mlp_reference(x, w1, w2, hidden):
    """The MLP of packed values in 64 bits, and how far a right result may be from it: the
    first product's error moves values across a midpoint of E4M3, each by a step."""
    y, size = x @ w1.T, MFMA * 2 * (np.abs(x) @ np.abs(w1).T)
    gate, up = y[:, :hidden], y[:, hidden:]
    sig = np.exp(-np.logaddexp(0, -gate))
    a = gate * sig * up
    error = 1.1 * np.abs(up) * size[:, :hidden] + np.abs(gate * sig) * size[:, hidden:] + \
        1.1 * size[:, :hidden] * size[:, hidden:] + 2.0 ** -21 * np.abs(a)
    q, e = quantized(a, 1)
    scale = np.repeat(np.ldexp(1.0, e), 128, axis=1)[:, :hidden]
    # Either end of the interval, at the scale of the block or at its neighbour's.
    off = np.zeros_like(a)
    for s in (scale / 2, scale, scale * 2):
        top = 448 * s
        for v in (a - error, a + error):
            off = np.maximum(off, np.where(np.abs(a) <= top * 1.01, np.abs(e4m3(np.clip(v, -top, top) / s) * s - q), 0))
    near = (blocks(np.abs(a) + error, 1).max(axis=(1, 3)) > 448 * np.ldexp(1.0, e)) | \
        (blocks(np.abs(a) - error, 1).max(axis=(1, 3)) <= 224 * np.ldexp(1.0, e))
    near = np.repeat(near, 128, axis=1)[:, :hidden]
    same = np.maximum(np.abs(e4m3((a - error) / scale) * scale - q), np.abs(e4m3((a + error) / scale) * scale - q))
    off = np.where(near, off, same)
    want = q @ w2.T
    return want, HALF_BF16 * np.abs(want) + 2 * MFMA * (np.abs(q) @ np.abs(w2).T) + off @ np.abs(w2).T


@pytest.mark.parametrize("m,k,hidden,n", [(1, 128, 128, 128), (3, 256, 384, 130), (16, 1000, 256, 77), (40, 5376, 512, 260),
                                          (130, 300, 1024, 256), (300, 640, 640, 520), (1025, 256, 256, 256)])
def test_mlp(m, k, hidden, n):
    print(f"[fp8 block] mlp {m}x{k}x{hidden}x{n}", flush=True)
    with Gpu() as g:
        xb = values(m, k, m, 1.0)
        x = activation(g, xb, m, k)
        w1 = weight(g, synth.normal_bf16(1, 2 * hidden * k, scale=1 / math.sqrt(k)), 2 * hidden, k)
        w2 = weight(g, synth.normal_bf16(2, n * hidden, scale=1 / math.sqrt(hidden)), n, hidden)
        out, tx = g.empty(m * n), g.from_bf16(xb)
        g.begin()
        g.check(g.lib.h3_hip_mlp_fp8_block(g.handle, out.handle, x.handle, w1.handle, w2.handle, m, k, hidden, n), "mlp")
        g.submit()
        got = out.read()
        want, bound = mlp_reference(x.values(), w1.values(), w2.values(), hidden)
        within(bf16(got).reshape(m, n), want, bound)
        # The bound is one on single values; as a whole the result is much nearer.
        assert np.linalg.norm(bf16(got).reshape(m, n) - want) <= 1e-2 * np.linalg.norm(want)
        g.begin()
        g.check(g.lib.h3_gpu_mlp_bf16(g.handle, out.handle, tx.handle, w1.handle, w2.handle, m, k, hidden, n), "mlp")
        g.submit()
        assert np.array_equal(out.read(), got)


# ------------------------------------------------------------------ together, in a graph, refusals
def test_block_chain():
    """Norm -> projection -> norm with the residual -> MLP, each stage against the definition
    on what the stage before gave."""
    rows, width, hidden, eps = 200, 640, 512, 1e-5
    with Gpu() as g:
        lib, h = g.lib, g.handle
        res = values(rows, width, 1, 1.0)
        norm = synth.f32_to_bf16((1 + 0.1 * np.random.default_rng(2).standard_normal(width)).astype(np.float32))
        w0 = weight(g, synth.normal_bf16(3, width * width, scale=1 / math.sqrt(width)), width, width)
        w1 = weight(g, synth.normal_bf16(4, 2 * hidden * width, scale=1 / math.sqrt(width)), 2 * hidden, width)
        w2 = weight(g, synth.normal_bf16(5, hidden * width, scale=1 / math.sqrt(hidden)), width, hidden)
        tr, tn = g.from_bf16(res), g.from_bf16(norm)
        first, second = new(g, rows, width), new(g, rows, width)
        branch, total, out = (g.empty(rows * width) for _ in range(3))
        g.begin()
        g.check(lib.h3_hip_add_rms_norm_fp8_block(h, None, first.handle, tr.handle, None, tn.handle, rows, width, eps), "norm")
        g.check(lib.h3_hip_linear_fp8_block(h, branch.handle, first.handle, w0.handle, None, rows, width, width), "linear")
        g.check(lib.h3_hip_add_rms_norm_fp8_block(h, total.handle, second.handle, tr.handle, branch.handle, tn.handle, rows,
                                                  width, eps), "add norm")
        g.check(lib.h3_hip_mlp_fp8_block(h, out.handle, second.handle, w1.handle, w2.handle, rows, width, hidden, width), "mlp")
        g.submit()

        def norm_of(x):
            return x / np.sqrt((x * x).mean(axis=1, keepdims=True) + eps) * bf16(norm).astype(np.float64)

        shape = (rows, width)
        y = norm_of(bf16(res).reshape(shape).astype(np.float64))
        within(first.values(), y, packed_bound(first, y, 2.0 ** -19 * np.abs(y)), "norm")
        xv, wv = first.values(), w0.values()
        want = xv @ wv.T
        b = bf16(branch.read()).reshape(shape).astype(np.float64)
        within(b, want, HALF_BF16 * np.abs(want) + 2 * MFMA * (np.abs(xv) @ np.abs(wv).T), "linear")
        s = bf16(total.read()).reshape(shape).astype(np.float64)
        want = bf16(res).reshape(shape) + b
        within(s, want, (HALF_BF16 + 2.0 ** -23) * np.abs(want), "sum")
        y = norm_of(s)
        within(second.values(), y, packed_bound(second, y, 2.0 ** -19 * np.abs(y)), "add norm")
        want, bound = mlp_reference(second.values(), w1.values(), w2.values(), hidden)
        within(bf16(out.read()).reshape(shape), want, bound, "mlp")


def test_captured_chain():
    """Packing, norms, SwiGLU and a projection of packed rows in a graph, replayed between eager
    work that uses the context's workspaces; calls that need one of those are refused."""
    rows, width, n = 300, 1024, 512
    with Gpu() as g:
        lib, h = g.lib, g.handle
        res, norm = g.from_bf16(values(rows, width, 1, 1.0)), g.from_bf16(values(1, width, 2, 0.3))
        w = weight(g, synth.normal_bf16(3, n * width, scale=1 / math.sqrt(width)), n, width)
        w1 = weight(g, synth.normal_bf16(4, 2 * 256 * width, scale=0.03), 512, width)
        w2 = weight(g, synth.normal_bf16(5, n * 256, scale=0.06), n, 256)
        first, act = new(g, rows, width), new(g, rows, n // 2)
        product, out = g.empty(rows * n), g.empty(rows * n // 2)

        def chain():
            g.check(lib.h3_hip_add_rms_norm_fp8_block(h, None, first.handle, res.handle, None, norm.handle, rows, width, 1e-5), "norm")
            g.check(lib.h3_hip_linear_fp8_block(h, product.handle, first.handle, w.handle, None, rows, width, n), "linear")
            g.check(lib.h3_hip_swiglu_fp8_block(h, act.handle, product.handle, rows, n // 2), "swiglu")
            g.check(lib.h3_hip_fp8_block_unpack(h, out.handle, act.handle, rows, n // 2), "unpack")

        graph = Graph(g)
        g.begin()
        with graph:
            chain()
            kernel = g.last_kernel()
            assert not lib.h3_gpu_linear_bf16(h, product.handle, res.handle, w.handle, None, rows, width, n)
            assert "captured" in g.error()
            assert not lib.h3_hip_mlp_fp8_block(h, product.handle, first.handle, w1.handle, w2.handle, rows, width, 256, n)
            assert "captured" in g.error()
            assert not lib.h3_hip_fp8_block_new(h, 1, 1, 1) and "captured" in g.error()
        assert "shares=" not in kernel
        big, bigger = g.empty(2000 * width), g.empty(2000 * n)
        got = []
        for i in range(3):
            g.check(lib.h3_hip_fill_normal_bf16(h, big.handle, i, C.c_float(1.0), big.elements), "fill")
            g.check(lib.h3_gpu_linear_bf16(h, bigger.handle, big.handle, w.handle, None, 2000, width, n), "eager")
            g.check(lib.h3_gpu_mlp_bf16(h, bigger.handle, big.handle, w1.handle, w2.handle, 2000, width, 256, n), "eager")
            g.check(lib.h3_hip_fill_normal_bf16(h, product.handle, 9, C.c_float(1.0), product.elements), "fill")
            graph.launch()
            g.submit()
            got.append((product.read(), out.read(), act.raw()))
            g.begin()
        g.submit()
        # Eager, without splits over K either: the same values in the same order, or a rounding apart.
        g.begin()
        chain()
        g.submit()
        for p, o, a in got:
            assert np.array_equal(p, got[0][0]) and np.array_equal(o, got[0][1]) and np.array_equal(a, got[0][2])
        xv, wv = first.values(), w.values()
        within(bf16(got[0][0]).reshape(rows, n), xv @ wv.T,
               HALF_BF16 * np.abs(xv @ wv.T) + 2 * MFMA * (np.abs(xv) @ np.abs(wv).T))
        graph.close()


def test_nonfinite_values_fail_the_submit():
    rows, width = 4, 256
    with Gpu() as g:
        lib, h = g.lib, g.handle
        for bad in (0x7f80, 0xff80, 0x7fc0):
            bits = values(rows, width, 1)
            flat = bits.reshape(-1).copy()
            flat[300] = bad
            t, packed, half = g.from_bf16(flat), new(g, rows, width), new(g, rows, width // 2)
            one = g.from_bf16(np.full(width, 0x3f80, np.uint16))
            for call in (lambda: lib.h3_hip_fp8_block_pack(h, packed.handle, t.handle, rows, width),
                         lambda: lib.h3_hip_swiglu_fp8_block(h, half.handle, t.handle, rows, width // 2),
                         lambda: lib.h3_hip_add_rms_norm_fp8_block(h, None, packed.handle, t.handle, None, one.handle, rows, width, 1e-5)):
                g.begin()
                assert call()
                with pytest.raises(H3Error, match="nonfinite"):
                    g.submit()
                g.cancel()
            assert not lib.h3_hip_fp8_block_weight_from_bf16(h, t.handle, rows, width) and "nonfinite" in g.error()
            # The refusal leaves no fault behind.
            g.begin()
            g.submit()


def test_refusals():
    with Gpu() as g:
        lib, h = g.lib, g.handle
        x, w, w2 = new(g, 10, 256), new(g, 300, 256, 128), new(g, 64, 128, 128)
        act, plain, out = new(g, 10, 150), g.empty(10 * 256), g.empty(10 * 300)
        short, other = g.empty(5), new(g, 10, 255)

        def refused(text, call, *args):
            assert not call(h, *args)
            assert text in g.error(), (text, g.error())

        refused("no active", lib.h3_hip_fp8_block_pack, x.handle, plain.handle, 10, 256)
        g.begin()
        for rows, columns, tile in ((0, 1, 1), (1, 0, 1), (1, 1, 2), (1, 1, 64), (1, (1 << 24) - 127, 1)):
            refused("FP8 block matrix", lib.h3_hip_fp8_block_new, rows, columns, tile)
        refused("missing", lib.h3_hip_fp8_block_from_packed, None, None, 1, 1, 1)
        refused("elements", lib.h3_hip_fp8_block_weight_from_bf16, short.handle, 10, 256)
        refused("need 11x256", lib.h3_hip_fp8_block_pack, x.handle, plain.handle, 11, 256)
        refused("need 10x255", lib.h3_hip_fp8_block_pack, x.handle, plain.handle, 10, 255)
        refused("need an FP8 block activation", lib.h3_hip_fp8_block_pack, w.handle, plain.handle, 10, 256)
        refused("need an FP8 block activation", lib.h3_hip_fp8_block_pack, plain.handle, plain.handle, 10, 256)
        refused("elements", lib.h3_hip_fp8_block_pack, x.handle, short.handle, 10, 256)
        refused("not a plain tensor", lib.h3_hip_fp8_block_pack, x.handle, x.handle, 10, 256)
        refused("need an FP8 block matrix", lib.h3_hip_fp8_block_unpack, plain.handle, plain.handle, 10, 256)
        refused("need 299x256", lib.h3_hip_fp8_block_unpack, out.handle, w.handle, 299, 256)
        args = (out.handle, x.handle, w.handle, None)
        refused("invalid shape", lib.h3_hip_linear_fp8_block, *args, 0, 256, 300)
        refused("elements", lib.h3_hip_linear_fp8_block, out.handle, x.handle, w.handle, None, 11, 256, 300)
        wide = g.empty(11 * 300)
        refused("need 11x256", lib.h3_hip_linear_fp8_block, wide.handle, x.handle, w.handle, None, 11, 256, 300)
        refused("need 299x256", lib.h3_hip_linear_fp8_block, *args, 10, 256, 299)
        refused("need 10x256", lib.h3_hip_linear_fp8_block, out.handle, other.handle, w.handle, None, 10, 256, 300)
        refused("need an FP8 block activation", lib.h3_hip_linear_fp8_block, out.handle, plain.handle, w.handle, None, 10, 256, 300)
        refused("need an FP8 block weight", lib.h3_hip_linear_fp8_block, out.handle, x.handle, x.handle, None, 10, 256, 300)
        refused("missing", lib.h3_hip_linear_fp8_block, out.handle, x.handle, None, None, 10, 256, 300)
        refused("elements", lib.h3_hip_linear_fp8_block, short.handle, x.handle, w.handle, None, 10, 256, 300)
        refused("elements", lib.h3_hip_linear_fp8_block, out.handle, x.handle, w.handle, short.handle, 10, 256, 300)
        refused("h3_hip_linear_fp8_block", lib.h3_gpu_linear_bf16, out.handle, x.handle, w.handle, None, 10, 256, 300)
        refused("not a plain tensor", lib.h3_gpu_linear_bf16, out.handle, x.handle, plain.handle, None, 10, 256, 1)
        refused("no activation", lib.h3_hip_linear_gelu_bf16, out.handle, plain.handle, w.handle, None, 10, 256, 300)
        refused("aliases", lib.h3_gpu_linear_bf16, plain.handle, plain.handle, w.handle, None, 8, 256, 300)
        refused("multiple of 128", lib.h3_hip_mlp_fp8_block, out.handle, x.handle, w.handle, w2.handle, 10, 256, 150, 64)
        refused("need 256x256", lib.h3_hip_mlp_fp8_block, out.handle, x.handle, w.handle, w2.handle, 10, 256, 128, 64)
        refused("h3_hip_mlp_fp8_block", lib.h3_gpu_mlp_bf16, out.handle, x.handle, w.handle, w2.handle, 10, 256, 128, 64)
        refused("need 10x256", lib.h3_hip_swiglu_fp8_block, act.handle, plain.handle, 10, 256)
        refused("elements", lib.h3_hip_swiglu_fp8_block, x.handle, plain.handle, 10, 256)
        refused("multiple of 8", lib.h3_hip_add_rms_norm_fp8_block, None, act.handle, plain.handle, None, plain.handle, 10, 150, 1e-5)
        refused("come together", lib.h3_hip_add_rms_norm_fp8_block, plain.handle, x.handle, plain.handle, None, plain.handle, 10, 256, 1e-5)
        refused("slots", lib.h3_hip_adaln_fp8_block, x.handle, plain.handle, plain.handle, plain.handle, None, 10, 256, 2, 0, 2, 1e-5)
        refused("row map", lib.h3_hip_adaln_fp8_block, x.handle, plain.handle, plain.handle, plain.handle, None, 10, 256, 2, 0, 1, 1e-5)
        refused("not a plain tensor", lib.h3_gpu_add_bf16, plain.handle, x.handle, plain.handle, 10)
        g.submit()
        with Gpu() as second:
            second.begin()
            assert not second.lib.h3_hip_fp8_block_pack(second.handle, x.handle, plain.handle, 10, 256)
            assert "another context" in second.error()
            second.submit()
