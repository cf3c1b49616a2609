"""The block-scaled FP8 projections' kernels with each of their epilogues, by name, whole and in
shares of K, and the rule that a graph keeps no partial sums. Bounds as in test_fp8_block_gpu.py."""
import ctypes as C
import math
from concurrent.futures import ThreadPoolExecutor

import numpy as np
import pytest

from h3cli_amd import synth
from h3cli_amd.runtime import Gpu
from tests.helpers import bf16
from tests.test_capture_gpu import Graph
from tests.test_fp8_block_calls_gpu import normal, rows_within, weight_of
from tests.test_fp8_block_gpu import Packed, linear, mlp_reference, new, values, within

pytestmark = pytest.mark.gpu


def is_kernel(kernel, name, shared):
    return kernel.split(" shares=")[0] == name and ("shares=" in kernel) == shared


MID, PIPE128, PIPE256 = "fp8_block_mid rows=64", "fp8_block_pipe rows=128", "fp8_block_pipe rows=256"
EXACT = [(300, 256, 5000, MID, False), (300, 256, 5001, MID, False), (130, 7168, 1000, MID, True), (130, 7168, 1001, MID, True),
         (1025, 256, 4096, PIPE128, False), (4097, 256, 1001, PIPE128, False), (640, 5376, 2056, PIPE128, True),
         (1500, 5376, 1001, PIPE128, True), (1025, 256, 8000, PIPE256, False), (8193, 256, 1001, PIPE256, False),
         (8193, 13824, 264, PIPE256, True), (8193, 13824, 265, PIPE256, True)]


@pytest.mark.parametrize("m,k,n,name,shared", EXACT)
def test_tiles_exact(m, k, n, name, shared):
    """Every output of a tile kernel without and with a bias, columns a multiple of 8 and not. Codes
    +-1, +-2 and scales 1/2 to 4: products are multiples of 1/4, and their sums (of up to 13824 with
    random signs, a few thousand) and the bias, multiples of 1/4 up to 16, are exact in FP32 in any
    order, so that each result has to be the BF16 rounding of its sum."""
    print(f"[fp8 block] exact {m}x{k}x{n}", flush=True)
    rng = np.random.default_rng(m + n)
    values_of = np.array([0x38, 0xb8, 0x40, 0xc0], np.uint8)      # 1, -1, 2, -2
    kb = -(-k // 128)
    with Gpu() as g:
        xc, wc = (values_of[rng.integers(0, 4, s)] for s in ((m, k), (n, k)))
        xs, ws = (rng.integers(126, 130, s).astype(np.uint8) for s in ((m, kb), (-(-n // 128), kb)))
        x = Packed(g, g.lib.h3_hip_fp8_block_from_packed(g.handle, xc.ctypes.data, xs.ctypes.data, m, k, 1), m, k, 1)
        w = Packed(g, g.lib.h3_hip_fp8_block_from_packed(g.handle, wc.ctypes.data, ws.ctypes.data, n, k, 128), n, k, 128)
        bias = (rng.integers(-64, 65, n) / 4).astype(np.float32)
        t, out = g.from_bf16(synth.f32_to_bf16(bias)), g.empty(m * n)
        want = (x.values().astype(np.float32) @ w.values().astype(np.float32).T).astype(np.float64)
        for b in (None, t):
            got, kernel = linear(g, out, x, w, b, m, k, n)
            assert is_kernel(kernel, name, shared), kernel
            full = want if b is None else want + bias
            assert np.abs(full).max() < 2 ** 20
            assert np.array_equal(got, synth.f32_to_bf16(full.astype(np.float32))), kernel


@pytest.mark.parametrize("m,k,n,rows", [(200, 256, 1000, 32), (72, 512, 4096, 48)])
@pytest.mark.parametrize("columns", ["whole", "cut"])
def test_few_rows_pack(m, k, n, rows, columns):
    """The few-row kernels of 32 and 48 rows that pack their BF16 input: the packed input's result."""
    k = k if columns == "whole" else k - 5
    with Gpu() as g:
        t, packed = normal(g, m * k, m, 1.0), new(g, m, k)
        w = weight_of(g, normal(g, n * k, n + 1, 1 / math.sqrt(k)), n, k)
        bias = g.from_bf16(values(1, n, 3, 1.0))
        g.begin()
        g.check(g.lib.h3_hip_fp8_block_pack(g.handle, packed.handle, t.handle, m, k), "pack")
        g.submit()
        out = g.empty(m * n)
        for b in (None, bias):
            got, kernel = linear(g, out, t, w, b, m, k, n)
            assert kernel == f"fp8_block_stream packing rows={rows}", kernel
            again, _ = linear(g, out, packed, w, b, m, k, n)
            assert np.array_equal(got, again)
            if b is None:
                rows_within(g, t, w, got, m, k, n, kernel)


@pytest.mark.parametrize("m,k,hidden,name,shared", [
    (300, 256, 2560, MID, False), (64, 13824, 128, MID, True), (513, 7168, 128, MID, True), (1025, 256, 2048, PIPE128, False),
    (1500, 5376, 512, PIPE128, True), (4097, 13824, 128, PIPE128, True), (1025, 256, 4096, PIPE256, False),
    (8193, 256, 640, PIPE256, False), (8193, 13824, 256, PIPE256, True)])
def test_swiglu_epilogues(m, k, hidden, name, shared):
    """The MLP where SwiGLU and packing are the epilogue of each tile kernel, whole and in shares of K.
    fc1's kernel is that of the plain projection of its shape: where that is a tile kernel, the MLP
    takes the same with SwiGLU."""
    n = 72
    print(f"[fp8 block] mlp {m}x{k}x{hidden}", flush=True)
    with Gpu() as g:
        t, x = normal(g, m * k, m, 1.0), new(g, m, k)
        w1 = weight_of(g, normal(g, 2 * hidden * k, 1, 1 / math.sqrt(k)), 2 * hidden, k)
        w2 = weight_of(g, normal(g, n * hidden, 2, 1 / math.sqrt(hidden)), n, hidden)
        product, out = g.empty(m * 2 * hidden), g.empty(m * n)
        g.begin()
        g.check(g.lib.h3_hip_fp8_block_pack(g.handle, x.handle, t.handle, m, k), "pack")
        g.check(g.lib.h3_hip_linear_fp8_block(g.handle, product.handle, x.handle, w1.handle, None, m, k, 2 * hidden), "fc1")
        assert is_kernel(g.last_kernel(), name, shared), g.last_kernel()
        g.check(g.lib.h3_hip_mlp_fp8_block(g.handle, out.handle, x.handle, w1.handle, w2.handle, m, k, hidden, n), "mlp")
        g.submit()
        got = bf16(out.read()).reshape(m, n)
        assert np.all(np.isfinite(got))
        # Rows of every tile and of every place in one.
        at = np.unique(np.r_[0:m:max(1, m // 61), np.linspace(0, m - 1, 64).astype(int), max(0, m - 33):m])
        want, bound = mlp_reference(x.values()[at], w1.values(), w2.values(), hidden)
        within(got[at], want, bound)
        assert np.linalg.norm(got[at] - want) <= 1e-2 * np.linalg.norm(want)


def test_graphs_keep_no_partial_sums():
    """Projections that eager calls share over K are whole in a graph, whose replays give the same
    between eager calls that use the partial sums' workspace and grow it."""
    shapes = [(300, 7168, 5376, MID), (300, 13824, 5120, PIPE128)]
    with Gpu() as g:
        lib, h = g.lib, g.handle
        work, graphs = [], []
        for i, (m, k, n, _) in enumerate(shapes):
            t, x = normal(g, m * k, i, 1.0), new(g, m, k)
            w = weight_of(g, normal(g, n * k, 7 + i, 1 / math.sqrt(k)), n, k)
            work.append((t, x, w, g.empty(m * n)))
            g.begin()
            g.check(lib.h3_hip_fp8_block_pack(h, x.handle, t.handle, m, k), "pack")
            g.submit()
        (m, k, n, name), (t, x, w, out) = shapes[0], work[0]
        eager, kernel = linear(g, out, x, w, None, m, k, n)      # a workspace that later calls grow
        assert is_kernel(kernel, name, True), kernel
        for (m, k, n, name), (t, x, w, out) in zip(shapes, work):
            graph = Graph(g)
            g.begin()
            with graph:
                g.check(lib.h3_hip_linear_fp8_block(h, out.handle, x.handle, w.handle, None, m, k, n), "linear")
                assert "shares=" not in g.last_kernel()
            g.submit()
            graphs.append(graph)
        first = None
        for i in range(3):
            g.begin()
            for graph, (m, k, n, _), (t, x, w, out) in zip(graphs, shapes, work):
                g.check(lib.h3_hip_fill_normal_bf16(h, out.handle, 7 + i, C.c_float(1.0), m * n), "fill")
                graph.launch()
            g.submit()
            got = [out.read() for _, _, _, out in work]
            first = first or got
            assert all(np.array_equal(a, b) for a, b in zip(first, got))
            for (m, k, n, name), (t, x, w, out) in list(zip(shapes, work))[i % 2:]:
                other = g.empty(m * n)
                again, kernel = linear(g, other, x, w, None, m, k, n)
                assert is_kernel(kernel, name, True), kernel
                rows_within(g, t, w, again, m, k, n, kernel)
        for (m, k, n, _), (t, x, w, out), got in zip(shapes, work, first):
            rows_within(g, t, w, got.reshape(m, n), m, k, n, "graph")
        for graph in graphs:
            graph.close()


def test_two_contexts_at_once():
    """Two contexts, a thread each: shares of K, packing and the MLP's workspace are each its own."""
    m, k, hidden = 300, 5376, 2560

    def model(seed):
        g = Gpu()
        t = normal(g, m * k, seed, 1.0)
        w1 = weight_of(g, normal(g, 2 * hidden * k, seed + 1, 1 / math.sqrt(k)), 2 * hidden, k)
        w2 = weight_of(g, normal(g, k * hidden, seed + 2, 1 / math.sqrt(hidden)), k, hidden)
        return g, t, w1, w2, g.empty(m * k), g.empty(m * 2 * hidden)

    def run(model, times):
        g, t, w1, w2, out, product = model
        got = []
        for _ in range(times):
            g.begin()
            g.check(g.lib.h3_gpu_linear_bf16(g.handle, product.handle, t.handle, w1.handle, None, m, k, 2 * hidden), "linear")
            g.check(g.lib.h3_gpu_mlp_bf16(g.handle, out.handle, t.handle, w1.handle, w2.handle, m, k, hidden, k), "mlp")
            g.submit()
            got.append((product.read(), out.read()))
        return got

    models = [model(seed) for seed in (1, 11)]
    try:
        want = [run(x, 1)[0] for x in models]
        with ThreadPoolExecutor(2) as pool:
            for (product, out), got in zip(want, pool.map(lambda x: run(x, 10), models)):
                assert all(np.array_equal(product, p) and np.array_equal(out, o) for p, o in got)
    finally:
        for x in models:
            x[0].close()
