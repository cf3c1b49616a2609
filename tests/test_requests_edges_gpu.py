"""Operators of a step that serves several requests at once, at the ends of their ranges: far
positions, sequences that one kernel cannot take beside those it can, workgroups that take several
tasks or steps in turn, every type of weight, tensors that are still being filled.

Bounds as in test_requests_gpu.py: HALF is BF16's largest rounding error relative to the value, F32
that of FP32; a sum of n products in FP32 is off by at most n * F32 times the sum of their magnitudes."""
import ctypes as C
import math

import numpy as np
import pytest

from h3cli_amd.runtime import Gpu
from tests.helpers import bf16
from tests.test_requests_gpu import (EPS, F32, HALF, SCALE, Adapters, Streamed, adapter_rows, attention_reference, check_attention, fill,
                                     normal, rope_axes, row_map, sequences, within)

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ attention of sequences
@pytest.mark.parametrize("q_rows,k_rows,heads,launches,kernel", [
    ((9000, 8193), (256, 8193), 40, 2, "attn_sequences rows=128"),       # the most queries have few keys, or none
    ((9000, 8193), (0, 8193), 40, 2, "attn_sequences rows=128"),
    ((5000, 5001), (5000, 200), 8, 2, "attn_sequences rows=128"),
    ((5000, 1500, 1, 1), (5000, 250, 9000, 9000), 40, 3, "attn_sequences rows=32 shares=2"),
])
def test_plans_of_several_kernels(q_rows, k_rows, heads, launches, kernel):
    """Each sequence by the kernel that suits it, all in one call: tiles of 256 rows for the long ones whatever
    else there is. Sampled rows of three heads against 64 bits."""
    print(f"[sequences] {q_rows} {k_rows} {heads}", flush=True)
    q_ends, k_ends = (np.cumsum([0] + list(n)) for n in (q_rows, k_rows))
    with Gpu() as g:
        t = [g.empty(int(n) * heads * 128) for n in (q_ends[-1], k_ends[-1], k_ends[-1], q_ends[-1])]
        total, count = C.c_double(), C.c_uint64()
        with sequences(g, q_ends, k_ends, heads, heads) as plan:
            g.check(g.lib.h3_hip_kernel_timing(g.handle, 1))
            g.begin()
            for i in range(4):
                fill(g, t[i], i + 1)
            g.check(g.lib.h3_hip_sdpa_sequences_bf16(g.handle, t[3].handle, *(x.handle for x in t[:3]), plan, C.c_float(SCALE)), "attention")
            assert g.last_kernel() == kernel, g.last_kernel()
            g.submit()
            g.check(g.lib.h3_hip_kernel_timing_read(g.handle, C.byref(total), C.byref(count)))
            g.check(g.lib.h3_hip_kernel_timing(g.handle, 0))
        assert count.value == launches
        q, k, v, got = (x.read().reshape(-1, heads, 128) for x in t)
    for i, (lq, lk) in enumerate(zip(q_rows, k_rows)):
        at = q_ends[i] + np.unique(np.append(np.arange(0, lq, 37), lq - 1))
        for h in (0, heads // 2 + 1, heads - 1):
            if not lk:
                assert not np.any(got[at, h] & 0x7fff)
                continue
            keys = slice(k_ends[i], k_ends[i + 1])
            fq, fk, fv = (bf16(x).astype(np.float64) for x in (q[at, h], k[keys, h], v[keys, h]))
            within(bf16(got[at, h]), *attention_reference(fq, fk, fv, SCALE), (i, h))


@pytest.mark.parametrize("q_offsets,k_offsets,heads,kv_heads", [
    ([0, 900, 1600], [0, 200, 900], 4, 4),
    ([0, 700, 1300, 1301, 1400], [3, 203, 903, 1700, 1700], 4, 2),       # a single row by tiles; queries without keys
    ([2, 802, 803, 1500], [0, 0, 256, 700], 2, 2),
])
def test_sequences_by_tiles_beside_those_of_few_keys(q_offsets, k_offsets, heads, kv_heads, monkeypatch):
    print(f"[sequences] {q_offsets} {k_offsets} {heads}/{kv_heads}", flush=True)
    monkeypatch.setenv("H3_HIP_ATTENTION_VARIANT", "22")
    with Gpu() as g:
        assert check_attention(g, q_offsets, k_offsets, heads, kv_heads, seed=13) == "attn_sequences rows=128"


# ------------------------------------------------------------------ rotation by axes
def turned(g, qkv, positions, frequencies, dim, interleaved, axis=None, axes=1):
    """Query rows of one head, without norms."""
    rows = len(positions)
    t, p, outs = g.from_bf16(qkv), g.from_f32(positions), [g.empty(rows * dim) for _ in range(3)]
    with rope_axes(g, frequencies, [0] * len(frequencies) if axis is None else axis, axes, interleaved) as plan:
        g.begin()
        g.check(g.lib.h3_hip_qkv_rope_axes_bf16(g.handle, *(o.handle for o in outs), t.handle, None, None, plan, p.handle, rows, 1, 1,
                                                dim, 0, C.c_float(EPS)), "rope")
        g.submit()
    return outs[0].read().reshape(rows, dim)


@pytest.mark.parametrize("interleaved", [0, 1])
@pytest.mark.parametrize("far", [2.0 ** 27, 3e9, 4.2e10, 1e11, 1e12, -1e12])
def test_rope_by_axes_of_any_number_of_turns(far, interleaved):
    """A phase is off by at most 2^-23 turns up to 2^24 turns and by 2^-47 of the angle beyond."""
    rows, dim, pairs = 64, 128, 64
    with Gpu() as g:
        rng = np.random.RandomState(3)
        qkv = normal(rows * 3 * dim, 5).reshape(rows, 3, dim)
        positions = (far * (1 + rng.rand(rows))).astype(np.float32)
        frequencies = np.concatenate([[1.0, 0.999], 10000.0 ** -rng.rand(pairs - 2)])
        got = bf16(turned(g, qkv, positions, list(frequencies), dim, interleaved))
    x = bf16(qkv[:, 0]).astype(np.float64)
    angle = positions.astype(np.float64)[:, None] * frequencies
    first = np.arange(pairs) * (2 if interleaved else 1)
    second = first + (1 if interleaved else pairs)
    a, b, c, s = x[:, first], x[:, second], np.cos(angle), np.sin(angle)
    y = x.copy()
    y[:, first], y[:, second] = a * c - b * s, b * c + a * s
    # The hardware's sine and cosine to 2^-18, the phase as above; this reference's own angle to 2^-52 of it; two FP32
    # products and their sum; one rounding to BF16.
    phase = 2 * math.pi * np.maximum(2.0 ** -23, 2.0 ** -47 * np.abs(angle) / (2 * math.pi)) + 2.0 ** -52 * np.abs(angle)
    size = np.empty_like(x)
    size[:, first] = size[:, second] = (np.abs(a) + np.abs(b)) * (2.0 ** -18 + phase + 4 * F32)
    within(got, y, HALF * np.abs(y) + size * (1 + HALF), (far, interleaved))


def test_rope_by_axes_beyond_any_phase_still_turns():
    """Where a turn is lost in the position's own rounding, pairs keep their lengths."""
    rows, dim = 8, 64
    with Gpu() as g:
        qkv = normal(rows * 3 * dim, 5).reshape(rows, 3, dim)
        positions = (1e20 * 10.0 ** (2 * np.arange(rows))).astype(np.float32)
        got = bf16(turned(g, qkv, positions, list(10000.0 ** -(np.arange(32) / 32)), dim, 0)).astype(np.float64)
    x = bf16(qkv[:, 0]).astype(np.float64)
    want = np.hypot(x[:, :32], x[:, 32:])
    # sin^2 + cos^2 is off by 4 * 2^-18 at most, each result by HALF of its size.
    within(np.hypot(got[:, :32], got[:, 32:]), want, want * (HALF + 2.0 ** -15))


# ------------------------------------------------------------------ adapters
@pytest.mark.parametrize("k", [4096, 4097])
def test_projections_with_adapters_wait_for_streamed_rows_and_bias(k):
    """x of 32 MB and then the bias are on their way when the call is made, and are filled anew behind it."""
    rows, n = 4000, 72
    with Gpu() as g:
        xs, biases = [normal(rows * k, 5 + i) for i in range(2)], [normal(n, 8 + i) for i in range(2)]
        sx, sb = Streamed(g, xs), Streamed(g, biases)
        w, ad = g.from_bf16(normal(n * k, 3, scale=1 / math.sqrt(k))), Adapters(g, [8, 24], k, n)
        plain, outs = [[g.from_bf16(x), g.from_bf16(b)] for x, b in zip(xs, biases)], [g.empty(rows * n) for _ in range(4)]
        with adapter_rows(g, row_map(rows, 2, 3), 2, 24) as plan:
            g.begin()
            for i in range(4):
                if i < 2:
                    sx.fill(i)
                    sb.fill(i)
                x, b = (sx.tensor, sb.tensor) if i < 2 else plain[i - 2]
                g.check(g.lib.h3_hip_linear_adapters_bf16(g.handle, outs[i].handle, x.handle, w.handle, b.handle, ad.handle, plan,
                                                          rows, k, n), "linear")
            g.submit()
        for i in range(2):
            assert np.array_equal(outs[i].read(), outs[i + 2].read()), i
        assert not np.array_equal(outs[0].read(), outs[1].read())
        for s in (sx, sb):
            s.close()
        ad.close()
