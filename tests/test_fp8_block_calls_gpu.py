"""Calls of the block-scaled FP8 operators that the definitions' own tests do not make: every
projection kernel by name, rows by the million, results in place, rows of larger tensors,
streamed weights and two graphs of one context. Bounds as in test_fp8_block_gpu.py."""
import ctypes as C
import math

import numpy as np
import pytest

from h3cli_amd import synth
from h3cli_amd.runtime import Gpu, H3Error
from tests.helpers import bf16
from tests.test_capture_gpu import Graph
from tests.test_fp8_block_gpu import (HALF_BF16, MFMA, Packed, activation, linear, mlp_reference, new, packed_bound,
                                        quantized, values, weight, within)

pytestmark = pytest.mark.gpu


def normal(g, count, seed, scale):
    t = g.empty(count)
    g.begin()
    g.check(g.lib.h3_hip_fill_normal_bf16(g.handle, t.handle, seed, C.c_float(scale), count), "fill")
    g.submit()
    return t


def weight_of(g, t, n, k):
    return Packed(g, g.lib.h3_hip_fp8_block_weight_from_bf16(g.handle, t.handle, n, k), n, k, 128)


def rows_within(g, t, w, out, rows, k, n, kernel):
    """Some rows of a projection of the BF16 tensor t against the packed values' products."""
    at = np.unique(np.linspace(0, rows - 1, 24).astype(int))
    xv, _ = quantized(bf16(t.read().reshape(rows, k)[at]).astype(np.float64), 1)
    wv = w.values()
    want = xv @ wv.T
    within(bf16(out[at]), want, HALF_BF16 * np.abs(want) + 2 * MFMA * (np.abs(xv) @ np.abs(wv).T), kernel)


def test_every_kernel():
    """The same rows from a BF16 input and a packed one, bit for bit, and against the definition,
    by every kernel: few rows in blocks of 16, 32 and 48, tiles of 64, 128 and 256 rows, whole
    and in shares of K."""
    seen = set()
    for rows, k, n in [(1, 256, 5376), (9, 5376, 5376), (17, 1000, 777), (17, 7168, 5376), (48, 1000, 777), (70, 128, 4096),
                       (8193, 2048, 4096), (1000, 14336, 8000), (300, 1000, 5000), (300, 7168, 5376), (300, 5376, 21504), (300, 13824, 5120),
                       (2300, 13824, 5120), (640, 5376, 28672), (1500, 5376, 21504)]:
        print(f"[fp8 block] {rows}x{k}x{n}", flush=True)
        with Gpu() as g:
            t = normal(g, rows * k, rows, 1.0)
            w = weight_of(g, normal(g, n * k, n + 1, 1 / math.sqrt(k)), n, k)
            packed = new(g, rows, k)
            g.begin()
            g.check(g.lib.h3_hip_fp8_block_pack(g.handle, packed.handle, t.handle, rows, k), "pack")
            g.submit()
            out = g.empty(rows * n)
            got, kernel = linear(g, out, t, w, None, rows, k, n)
            rows_within(g, t, w, got, rows, k, n, kernel)
            again, other = linear(g, out, packed, w, None, rows, k, n)
            assert np.array_equal(got, again)
            print(f"[fp8 block] {kernel}, {other}", flush=True)
            for name in (kernel, other):
                seen.add(name.split(" shares=")[0] + (" split" if "shares=" in name else ""))
    want = {f"fp8_block_stream rows={r}" for r in (16, 32, 48)} | {"fp8_block_stream packing rows=16"} | \
        {f"fp8_block_{kind}{split}" for kind in ("mid rows=64", "pipe rows=128", "pipe rows=256") for split in ("", " split")}
    assert want <= seen, want - seen


def test_rows_by_the_million():
    """More rows than one launch takes: run in parts."""
    rows, k, n = (1 << 22) + 300, 8, 8
    with Gpu() as g:
        t, w = normal(g, rows * k, 1, 1.0), weight(g, values(n, k, 2), n, k)
        bits = values(1, n, 3)
        got, kernel = linear(g, g.empty(rows * n), t, w, g.from_bf16(bits), rows, k, n)
        print(f"[fp8 block] {kernel}", flush=True)
        x = t.read().reshape(rows, k)
        for at in (slice(0, 2000), slice((1 << 22) - 1000, rows)):
            xv, _ = quantized(bf16(x[at]).astype(np.float64), 1)
            wv = w.values()
            want = xv @ wv.T + bf16(bits).reshape(1, n)
            bound = HALF_BF16 * np.abs(want) + 2 * MFMA * (np.abs(xv) @ np.abs(wv).T) + 2.0 ** -23 * np.abs(want)
            within(bf16(got[at]), want, bound)


@pytest.mark.parametrize("rows", [5, 16, 300, 1025])
def test_mlp_in_place(rows):
    k, hidden = 256, 384
    with Gpu() as g:
        w1 = weight(g, synth.normal_bf16(1, 2 * hidden * k, scale=1 / math.sqrt(k)), 2 * hidden, k)
        w2 = weight(g, synth.normal_bf16(2, k * hidden, scale=1 / math.sqrt(hidden)), k, hidden)
        t, out = g.from_bf16(values(rows, k, 3, 1.0)), g.empty(rows * k)
        for into in (out, t):
            g.begin()
            g.check(g.lib.h3_gpu_mlp_bf16(g.handle, into.handle, t.handle, w1.handle, w2.handle, rows, k, hidden, k), "mlp")
            g.submit()
        assert np.array_equal(out.read(), t.read())


def test_mlp_in_parts():
    """More rows than the activation's workspace of 1 GiB holds, the output in the input's place."""
    rows, k, hidden = 80000, 128, 14336
    with Gpu() as g:
        w1 = weight(g, synth.normal_bf16(1, 2 * hidden * k, scale=1 / math.sqrt(k)), 2 * hidden, k)
        w2 = weight(g, synth.normal_bf16(2, k * hidden, scale=1 / math.sqrt(hidden)), k, hidden)
        t = normal(g, rows * k, 3, 1.0)
        x = t.read().reshape(rows, k)
        g.begin()
        g.check(g.lib.h3_gpu_mlp_bf16(g.handle, t.handle, t.handle, w1.handle, w2.handle, rows, k, hidden, k), "mlp")
        g.submit()
        got = t.read().reshape(rows, k)
        at = np.r_[0:6, 30000:30006, 59898:59910, 70000:70006, rows - 6:rows]
        want, bound = mlp_reference(quantized(bf16(x[at]).astype(np.float64), 1)[0], w1.values(), w2.values(), hidden)
        within(bf16(got[at]), want, bound)
        assert np.linalg.norm(bf16(got[at]) - want) <= 1e-2 * np.linalg.norm(want)


def test_norm_sums_in_place():
    """The sum in the residual's or the branch's memory, and the gated residual in the residual's."""
    rows, width, eps = 70, 640, 1e-5
    res, branch = values(rows, width, 1, 1.0), values(rows, width, 2, 1.0)
    with Gpu() as g:
        lib, h = g.lib, g.handle
        norm = g.from_bf16(values(1, width, 3, 0.3))
        mod, row_map = g.from_bf16(values(6, width, 4, 0.3)), g.from_u32(np.zeros(rows, np.uint32))
        want = None
        for place in (None, 0, 1):
            t = [g.from_bf16(res), g.from_bf16(branch), g.empty(rows * width)]
            total, packed = t[2 if place is None else place], new(g, rows, width)
            g.begin()
            g.check(lib.h3_hip_add_rms_norm_fp8_block(h, total.handle, packed.handle, t[0].handle, t[1].handle, norm.handle,
                                                      rows, width, eps), "add norm")
            g.submit()
            got = total.read(), packed.raw()
            want = want or got
            assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])
        want = None
        for place in (None, 0):
            t = [g.from_bf16(res), g.from_bf16(branch), g.empty(rows * width)]
            total, packed = t[2 if place is None else place], new(g, rows, width)
            g.begin()
            g.check(lib.h3_hip_gate_adaln_fp8_block(h, total.handle, packed.handle, t[0].handle, t[1].handle, norm.handle,
                                                    mod.handle, mod.handle, row_map.handle, rows, width, 6, 2, 3, 4, eps), "gate")
            g.submit()
            got = total.read(), packed.raw()
            want = want or got
            assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])


def test_rows_behind_stay():
    """Norms and SwiGLU over fewer rows than their output holds."""
    rows, held, width = 33, 100, 264
    with Gpu() as g:
        lib, h = g.lib, g.handle
        t, norm = g.from_bf16(values(held, 2 * width, 1, 1.0)), g.from_bf16(values(1, width, 2, 0.3))
        for call in (lambda p: lib.h3_hip_add_rms_norm_fp8_block(h, None, p.handle, t.handle, None, norm.handle, rows, width, 1e-5),
                     lambda p: lib.h3_hip_swiglu_fp8_block(h, p.handle, t.handle, rows, width)):
            p = activation(g, values(held, width, 3), held, width)
            codes, scales = (v.copy() for v in p.read())
            g.begin()
            g.check(call(p), "call")
            g.submit()
            after, scales_after = p.read()
            assert np.array_equal(codes[rows:], after[rows:]) and np.array_equal(scales[rows:], scales_after[rows:])
            assert not np.array_equal(codes[:rows], after[:rows])


def test_streamed_weight():
    """A packed weight's memory from the host, on the copy stream, between two projections."""
    rows, k, n = 100, 300, 260
    with Gpu() as g:
        x = activation(g, values(rows, k, 1), rows, k)
        first, second = weight(g, values(n, k, 2), n, k), weight(g, values(n, k, 3), n, k)
        want, _ = linear(g, g.empty(rows * n), x, second, None, rows, k, n)
        out, raw = g.empty(rows * n), second.raw()
        g.begin()
        g.check(g.lib.h3_hip_linear_fp8_block(g.handle, out.handle, x.handle, first.handle, None, rows, k, n), "linear")
        g.check(g.lib.h3_hip_tensor_stream_host(first.handle, raw.ctypes.data, raw.size), "stream")
        g.check(g.lib.h3_hip_linear_fp8_block(g.handle, out.handle, x.handle, first.handle, None, rows, k, n), "linear")
        g.submit()
        assert np.array_equal(out.read().reshape(rows, n), want)
        assert not g.lib.h3_hip_tensor_stream_host(first.handle, raw.ctypes.data, raw.size - 1)


def test_two_graphs():
    """Two graphs of projections that eager calls would split over K, replayed in turn."""
    shapes = [(300, 7168, 520), (70, 5376, 1000)]
    with Gpu() as g:
        work, graphs = [], []
        for i, (rows, k, n) in enumerate(shapes):
            work.append((new(g, rows, k), weight(g, values(n, k, i, 1.0), n, k), g.empty(rows * n), normal(g, rows * k, i, 1.0)))
        for (rows, k, n), (x, w, out, t) in zip(shapes, work):
            graph = Graph(g)
            g.begin()
            with graph:
                g.check(g.lib.h3_hip_fp8_block_pack(g.handle, x.handle, t.handle, rows, k), "pack")
                g.check(g.lib.h3_hip_linear_fp8_block(g.handle, out.handle, x.handle, w.handle, None, rows, k, n), "linear")
                assert "shares=" not in g.last_kernel()
            g.submit()
            graphs.append(graph)
        first = None
        for i in range(3):
            g.begin()
            for graph, (rows, k, n), (x, w, out, t) in zip(graphs, shapes, work):
                g.check(g.lib.h3_hip_fill_normal_bf16(g.handle, out.handle, 7 + i, C.c_float(1.0), rows * n), "fill")
                graph.launch()
            g.submit()
            got = [out.read() for _, _, out, _ in work]
            first = first or got
            assert all(np.array_equal(a, b) for a, b in zip(first, got))
            # Eager work between the replays, with the split's and the packing's workspaces.
            (rows, k, n), (x, w, out, t) = shapes[0], work[0]
            linear(g, g.empty(rows * n), t, w, None, rows, k, n)
        for (rows, k, n), (x, w, out, t), got in zip(shapes, work, first):
            rows_within(g, t, w, got.reshape(rows, n), rows, k, n, "graph")
        for graph in graphs:
            graph.close()


@pytest.mark.parametrize("rows", [16, 300, 1500])
def test_mlp_overflow_fails_the_submit(rows):
    """Sums beyond FP32's range: the activation is not finite."""
    k, hidden = 256, 14336
    with Gpu() as g:
        def ones(n, columns, tile, scale):
            codes = np.full((n, columns), 0x38, np.uint8)
            scales = np.full((-(-n // tile), -(-columns // 128)), scale, np.uint8)
            return Packed(g, g.lib.h3_hip_fp8_block_from_packed(g.handle, codes.ctypes.data, scales.ctypes.data, n, columns, tile),
                          n, columns, tile)
        w1, w2, out = ones(2 * hidden, k, 128, 254), ones(k, hidden, 128, 100), g.empty(rows * k)
        x = ones(rows, k, 1, 254)
        g.begin()
        g.check(g.lib.h3_hip_mlp_fp8_block(g.handle, out.handle, x.handle, w1.handle, w2.handle, rows, k, hidden, k), "mlp")
        with pytest.raises(H3Error, match="nonfinite"):
            g.submit()
        g.cancel()


def test_norm_of_large_and_small_rows():
    """Rows whose squares leave FP32's range on either side."""
    width, eps = 256, 1e-5
    with Gpu() as g:
        lib, h = g.lib, g.handle
        x = np.random.default_rng(1).standard_normal((4, width)) * np.array([[1e25], [1e-25], [1.0], [3e37]])
        bits = synth.f32_to_bf16(x.astype(np.float32))
        norm = synth.f32_to_bf16(np.ones(width, np.float32))
        t, w, packed = g.from_bf16(bits), g.from_bf16(norm), new(g, 4, width)
        g.begin()
        g.check(lib.h3_hip_add_rms_norm_fp8_block(h, None, packed.handle, t.handle, None, w.handle, 4, width, eps), "norm")
        g.submit()
        x = bf16(bits).reshape(4, width).astype(np.float64)
        y = x / np.sqrt((x * x).mean(axis=1, keepdims=True) + float(np.float32(eps)))
        within(packed.values(), y, packed_bound(packed, y, 2.0 ** -23 * np.abs(y)), "norm")


@pytest.mark.parametrize("rows", [5, 257])
def test_longest_rows(rows):
    """The most columns a matrix may have: offsets near and above 32 bits. All codes are zero but
    for a few columns, whose small integers give exact sums."""
    k, n = (1 << 24) - 128, 130
    code = {0: 0, 1: 0x38, 2: 0x40, 3: 0x44, 4: 0x48}
    columns = [0, 127, 128, (1 << 23) + 5, (1 << 24) - 300, k - 1]
    rng = np.random.default_rng(rows)
    with Gpu() as g:
        print(f"[fp8 block] {rows}x{k}x{n}", flush=True)

        def sparse(count, tile):
            p, v = new(g, count, k, tile), rng.integers(0, 5, (count, len(columns)))
            raw = np.zeros(p.bytes, np.uint8)
            raw[:count * p.stride].reshape(count, p.stride)[:, columns] = np.vectorize(code.get)(v)
            raw[p.scales:] = 127
            assert g.lib.h3_hip_tensor_stream_host(p.handle, raw.ctypes.data, raw.size), g.error()
            return p, v

        (x, xv), (w, wv) = sparse(rows, 1), sparse(n, 128)
        got, kernel = linear(g, g.empty(rows * n), x, w, None, rows, k, n)
        print(f"[fp8 block] {kernel}", flush=True)
        assert np.array_equal(bf16(got), (xv @ wv.T).astype(np.float32)), kernel
