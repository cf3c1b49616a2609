"""Block-scaled FP8 at the ends of what the types hold: weights and rows of any size in the norms,
gates whose sigmoid leaves FP32's range, faults and refusals that meet. Bounds as in
test_fp8_block_gpu.py."""
import ctypes as C
import math

import numpy as np
import pytest

from h3cli_amd import synth
from h3cli_amd._lib import U32
from h3cli_amd.runtime import DitSynth, Gpu, H3Error
from tests.helpers import bf16
from tests.test_fp8_block_gpu import (HALF_BF16, MFMA, Packed, activation, blocks, e4m3, exponents, linear, new, quantized,
                                        values, weight, within)

pytestmark = pytest.mark.gpu


def codes_within(p, y, error):
    """Each code is that of y, or of a value that is `error` times it away, and so is each scale."""
    _, scales = p.read()
    e = scales.astype(np.int64) - 127
    top = np.abs(blocks(y, 1)).max(axis=(1, 3))
    assert np.all(exponents(top * (1 - error)) <= e) and np.all(e <= exponents(top * (1 + error)))
    s = np.repeat(np.ldexp(1.0, e), 128, axis=1)[:, :y.shape[1]]
    got, size = p.values() / s, np.abs(y) / s
    assert np.all((got == 0) | (np.sign(got) == np.sign(y)))
    low, high = e4m3(np.minimum(size * (1 - error), 448)), e4m3(np.minimum(size * (1 + error), 448))
    off = np.maximum(low - np.abs(got), np.abs(got) - high)
    assert np.all(off <= 0), (int((off > 0).sum()), np.unravel_index(np.argmax(off), off.shape), float(off.max()))


@pytest.mark.parametrize("eps", [1e-5, 0.0])
def test_norm_weights_of_any_size(eps):
    """Row values times weights beyond FP32's range on either side, where the normalized result is not."""
    width = 264
    with Gpu() as g:
        rng = np.random.default_rng(1)
        size = np.array([[3e37], [1e30], [1.0]] + ([[1e-30], [1e-38]] if eps == 0 else [[1e-3], [1e-9]]))
        bits = synth.f32_to_bf16((rng.standard_normal((5, width)) * size).astype(np.float32))
        scale = np.where(np.arange(width) < 128, 40.0, np.where(np.arange(width) < 256, 1e-12, 1e37))
        norm = synth.f32_to_bf16((scale * rng.uniform(1, 2, width)).astype(np.float32))
        t, w, packed = g.from_bf16(bits), g.from_bf16(norm), new(g, 5, width)
        g.begin()
        g.check(g.lib.h3_hip_add_rms_norm_fp8_block(g.handle, None, packed.handle, t.handle, None, w.handle, 5, width, eps),
                "norm")
        g.submit()
        x = bf16(bits).reshape(5, width).astype(np.float64)
        y = x / np.sqrt((x * x).mean(axis=1, keepdims=True) + float(np.float32(eps))) * bf16(norm)
        codes_within(packed, y, 2.0 ** -23)


@pytest.mark.parametrize("rows,width", [(5, 5376), (700, 2048), (2050, 4096)])
@pytest.mark.parametrize("kind", ["rms", "add", "adaln", "gate"])
def test_norms_in_64_bits(rows, width, kind):
    """The codes are those of the values but for one FP32 rounding (2^-24; 2^-23 here). Of a million
    values some are near enough to a midpoint that a sum in FP32 would show."""
    print(f"[fp8 block] {kind} {rows}x{width}", flush=True)
    rng = np.random.default_rng(rows + width)
    eps, slots = 1e-5, 6
    res, branch, norm = values(rows, width, 1, 1.0), values(rows, width, 2, 1.0), values(1, width, 3, 0.5)
    mod = synth.f32_to_bf16((0.3 * rng.standard_normal((3, slots, width))).astype(np.float32))
    row_map = rng.integers(0, 3, rows).astype(np.uint32)
    with Gpu() as g:
        tr, tb, tw, tm, tmap = (g.from_bf16(res), g.from_bf16(branch), g.from_bf16(norm), g.from_bf16(mod), g.from_u32(row_map))
        total, packed, lib, h = g.empty(rows * width), new(g, rows, width), g.lib, g.handle
        g.begin()
        if kind in ("rms", "add"):
            s, b = (total.handle, tb.handle) if kind == "add" else (None, None)
            ok = lib.h3_hip_add_rms_norm_fp8_block(h, s, packed.handle, tr.handle, b, tw.handle, rows, width, eps)
        elif kind == "adaln":
            ok = lib.h3_hip_adaln_fp8_block(h, packed.handle, tr.handle, tw.handle, tm.handle, tmap.handle, rows, width,
                                            slots, 3, 4, eps)
        else:
            ok = lib.h3_hip_gate_adaln_fp8_block(h, total.handle, packed.handle, tr.handle, tb.handle, tw.handle, tm.handle,
                                                 tm.handle, tmap.handle, rows, width, slots, 2, 3, 4, eps)
        g.check(ok, kind)
        g.submit()
        x = bf16(total.read() if kind in ("add", "gate") else res.reshape(-1)).reshape(rows, width).astype(np.float64)
        y = x / np.sqrt((x * x).mean(axis=1, keepdims=True) + float(np.float32(eps))) * bf16(norm).reshape(1, width)
        if kind in ("adaln", "gate"):
            mv = bf16(mod).reshape(3, slots, width).astype(np.float64)[row_map]
            y = y * (1 + mv[:, 4]) + mv[:, 3]
        codes_within(packed, y, 2.0 ** -23)


def test_weight_behind_a_pending_fault():
    """A fault that waits for the next submit hides no weight that is not finite, and stays; nor does
    it refuse a finite one."""
    rows, width = 4, 256
    with Gpu() as g:
        lib, h = g.lib, g.handle
        good = values(rows, width, 1)
        flat = good.reshape(-1).copy()
        flat[300] = 0x7fc0
        t, finite, packed = g.from_bf16(flat), g.from_bf16(good), new(g, rows, width)
        g.begin()
        g.check(lib.h3_hip_fp8_block_pack(h, packed.handle, t.handle, rows, width), "pack")
        assert not lib.h3_hip_fp8_block_weight_from_bf16(h, t.handle, rows, width) and "nonfinite" in g.error()
        w = Packed(g, lib.h3_hip_fp8_block_weight_from_bf16(h, finite.handle, rows, width), rows, width, 128)
        assert np.array_equal(w.values(), quantized(bf16(good).reshape(rows, width).astype(np.float64), 128)[0])
        with pytest.raises(H3Error, match="nonfinite"):
            g.submit()
        g.cancel()
        g.begin()
        g.submit()


def test_short_memory_leaves_no_error_behind():
    """A projection whose packed input is larger than the device's memory: refused, and the next call
    and its submit are fine."""
    rows = 3 << 30
    with Gpu() as g:
        lib, h = g.lib, g.handle
        w = weight(g, values(1, 1, 1), 1, 1)
        x, out = g.empty(rows), g.empty(rows)
        g.begin()
        assert not lib.h3_gpu_linear_bf16(h, out.handle, x.handle, w.handle, None, rows, 1, 1) and "memory" in g.error()
        g.check(lib.h3_hip_fill_normal_bf16(h, x.handle, 1, C.c_float(1.0), 300), "fill")
        g.check(lib.h3_gpu_linear_bf16(h, out.handle, x.handle, w.handle, None, 300, 1, 1), "linear")
        g.submit()
        xv, _ = quantized(bf16(x.read(300)).reshape(300, 1).astype(np.float64), 1)
        want = xv * w.values()
        within(bf16(out.read(300)).reshape(300, 1), want, (HALF_BF16 + 2 * MFMA) * np.abs(want))


def silu(gate):
    return gate * np.exp(-np.logaddexp(0, -gate))


def test_swiglu_of_gates_below_the_end_of_exp():
    """Gates whose sigmoid is below FP32's normal range, beside ups with which the product is not
    nothing: a block for each, since the largest value of a block hides the others."""
    gates = [-60.0, -60.5, -80.0, -86.5, -87.0, -87.5, -88.0, -88.5, -89.0, -95.0, -100.0, -104.0, -120.0, -140.0, -152.0,
             -153.0, -153.5, -154.0, -160.0, -1e4, -3e38]
    width = 128
    up = np.concatenate([np.exp2(np.linspace(0, 127.9, len(gates) - 6)), np.full(6, 3e38)])
    x = np.zeros((len(gates), 2 * width))
    x[:, :width] = np.array(gates)[:, None]
    x[:, width:] = up[:, None] * np.linspace(1 / 64, 1, width) * np.where(np.arange(width) % 3, 1, -1)
    for scale in (1.0, 2.0 ** -20, 3e38):
        bits = synth.f32_to_bf16(np.clip(x * np.where(np.arange(2 * width) < width, 1, scale), -3.3e38, 3.3e38).astype(np.float32))
        v = bf16(bits).reshape(x.shape).astype(np.float64)
        with Gpu() as g:
            t, packed = g.from_bf16(bits), new(g, len(gates), width)
            g.begin()
            g.check(g.lib.h3_hip_swiglu_fp8_block(g.handle, packed.handle, t.handle, len(gates), width), "swiglu")
            g.submit()
            y = silu(v[:, :width]) * v[:, width:]
            codes_within(packed, y, 2.0 ** -21)


@pytest.mark.parametrize("m,kernel", [(5, None), (1500, "fp8_block_mid rows=64"), (4097, "fp8_block_pipe rows=128"),
                                      (8193, "fp8_block_pipe rows=256")])
def test_mlp_of_gates_below_the_end_of_exp(m, kernel):
    """The same in the MLP, its activation packed by fc1's epilogue (5 rows: from FP32 sums): one
    input value, a block of the activation for each gate, an fc2 that copies a value of each. fc1's
    kernel is that of the plain projection of its shape."""
    gates, ups = [-60.0, -88.0, -96.0, -104.0, -120.0], [40, 100, 100, 120, 126]
    k, hidden, n = 256 if kernel else 640, 128 * len(gates), 8
    print(f"[fp8 block] mlp gates {m} rows", flush=True)
    x, w1, w2 = np.zeros((m, k)), np.zeros((2 * hidden, k)), np.zeros((n, hidden))
    x[:, 0] = 1
    w1[:hidden, 0], w1[hidden:, 0] = np.repeat(gates, 128), np.repeat(np.exp2(ups), 128)
    w2[np.arange(len(gates)), 128 * np.arange(len(gates)) + 7] = 1
    with Gpu() as g:
        tx, t1, t2 = (synth.f32_to_bf16(v.astype(np.float32).reshape(-1)) for v in (x, w1, w2))
        px, p1, p2 = activation(g, tx, m, k), weight(g, t1, 2 * hidden, k), weight(g, t2, n, hidden)
        assert np.array_equal(p1.values(), w1)
        if kernel:
            assert linear(g, g.empty(m * 2 * hidden), px, p1, None, m, k, 2 * hidden)[1] == kernel
        out = g.empty(m * n)
        g.begin()
        g.check(g.lib.h3_hip_mlp_fp8_block(g.handle, out.handle, px.handle, p1.handle, p2.handle, m, k, hidden, n), "mlp")
        g.submit()
        want = np.zeros(n)
        want[:len(gates)] = silu(np.array(gates)) * np.exp2(ups)
        # A value is off by half a step of E4M3; its gate's product with 1 / ln 2 by 2^-24 of it.
        within(bf16(out.read()).reshape(m, n), np.broadcast_to(want, (m, n)), (2.0 ** -4 + 2.0 ** -15) * np.abs(want))


def copied(g, t, at, width):
    """Rows of a tensor that is too large to read."""
    part = g.empty(len(at) * width)
    g.begin()
    for i, row in enumerate(at):
        g.check(g.lib.h3_gpu_copy_bf16(g.handle, part.handle, i * width, t.handle, int(row) * width, width), "copy")
    g.submit()
    return bf16(part.read()).reshape(len(at), width).astype(np.float64)


@pytest.mark.parametrize("rows,k,n", [(1 << 22, 128, 8192), (1 << 20, 128, 33000)])
def test_more_threads_than_a_launch_takes(rows, k, n):
    """Projections of one K block, for which the few-row kernels are modelled fastest, but whose
    workgroups would be 2^24 of 256 threads: 64 GiB of results, by another kernel."""
    print(f"[fp8 block] {rows}x{k}x{n}", flush=True)
    with Gpu() as g:
        t, out, packed = g.empty(rows * k), g.empty(rows * n), new(g, rows, k)
        w = weight(g, values(n, k, 2, 1.0), n, k)
        g.begin()
        g.check(g.lib.h3_hip_fill_normal_bf16(g.handle, t.handle, 1, C.c_float(1.0), rows * k), "fill")
        g.check(g.lib.h3_hip_fp8_block_pack(g.handle, packed.handle, t.handle, rows, k), "pack")
        g.check(g.lib.h3_hip_linear_fp8_block(g.handle, out.handle, packed.handle, w.handle, None, rows, k, n), "linear")
        kernel = g.last_kernel()
        g.submit()
        print(f"[fp8 block] {kernel}", flush=True)
        at = np.unique(np.r_[0, 1, np.linspace(0, rows - 1, 30).astype(int), rows - 2, rows - 1])
        xv, wv = quantized(copied(g, t, at, k), 1)[0], w.values()
        want = xv @ wv.T
        within(copied(g, out, at, n), want, HALF_BF16 * np.abs(want) + 2 * MFMA * (np.abs(xv) @ np.abs(wv).T), kernel)


def test_norms_of_too_many_rows():
    """Rows whose waves are more threads than a launch takes are refused, and the command goes on."""
    rows, width = 1 << 26, 8
    with Gpu() as g:
        lib, h = g.lib, g.handle
        t, norm, mod = g.empty(rows * width), g.from_bf16(values(1, width, 1)), g.from_bf16(values(6, width, 2))
        total, row_map, packed = g.empty(rows * width), g.empty(rows, U32), new(g, rows, width)
        g.begin()
        for call in (lambda r: lib.h3_hip_add_rms_norm_fp8_block(h, None, packed.handle, t.handle, None, norm.handle, r, width, 1e-5),
                     lambda r: lib.h3_hip_adaln_fp8_block(h, packed.handle, t.handle, norm.handle, mod.handle, row_map.handle, r,
                                                          width, 6, 0, 1, 1e-5),
                     lambda r: lib.h3_hip_gate_adaln_fp8_block(h, total.handle, packed.handle, t.handle, t.handle, norm.handle,
                                                               mod.handle, mod.handle, row_map.handle, r, width, 6, 2, 3, 4, 1e-5)):
            for r in (rows, rows - 3):      # 2^24 workgroups of 256
                assert not call(r) and "too many" in g.error()
        n = rows - 4
        g.check(lib.h3_hip_fill_normal_bf16(h, t.handle, 1, C.c_float(1.0), n * width), "fill")
        g.check(lib.h3_hip_add_rms_norm_fp8_block(h, None, packed.handle, t.handle, None, norm.handle, n, width, 1e-5), "norm")
        g.check(lib.h3_hip_fp8_block_unpack(h, total.handle, packed.handle, rows, width), "unpack")
        g.submit()
        at = np.r_[0:8, n // 2:n // 2 + 8, n - 8:n]
        x = copied(g, t, at, width)
        y = x / np.sqrt((x * x).mean(axis=1, keepdims=True) + float(np.float32(1e-5))) * bf16(norm.read())
        top = np.abs(y).max(axis=1, keepdims=True)
        within(copied(g, total, at, width), y, np.maximum(2.0 ** -4 * np.abs(y), 2.0 ** -10 * top / 224) * (1 + 2.0 ** -20))
        assert not copied(g, total, np.array([n]), width).any()


@pytest.mark.parametrize("quant", [1, 3])
def test_dit_of_too_many_hidden_values(quant):
    """The GELU MLP of quantized projections takes fewer than 2^32 hidden values; more were cut off."""
    with pytest.raises(H3Error, match="too many for the GELU MLP"):
        DitSynth(geometry="h3", blocks=1, hidden=256, heads=1, mlp=1 << 16, frames=256, height=16, width=16, audio_rows=0,
                 latent=256, streamed_first=1, swiglu=0, projection_quant=quant)
