"""Operators of a step that serves several requests at once, at the ends of their ranges: far
positions, sequences that one kernel cannot take beside those it can, workgroups that take several
tasks or steps in turn, every type of weight, tensors that are still being filled.

Bounds as in test_requests_gpu.py: HALF is BF16's largest rounding error relative to the value, F32
that of FP32; a sum of n products in FP32 is off by at most n * F32 times the sum of their magnitudes."""
import ctypes as C
import math

import numpy as np
import pytest

from h3cli_amd import synth
from h3cli_amd.runtime import Gpu
from tests.helpers import bf16
from tests.test_quant_gpu import configure, load, write_weight
from tests.test_requests_gpu import (EPS, F32, HALF, SCALE, Adapters, Step, Streamed, adapter_rows, attention_reference, check_adapters,
                                     check_attention, check_rope, fill, normal, rope_axes, rope_reference, row_map, sequences, within)

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


@pytest.mark.parametrize("interleaved", [0, 1])
@pytest.mark.parametrize("grouped", [0, 1])
@pytest.mark.parametrize("rows,heads,kv_heads,dim,pairs", [
    (2049, 3, 1, 128, 48), (4099, 3, 1, 128, 64), (4099, 2, 1, 64, 24), (4099, 2, 2, 90, 37), (2051, 1, 1, 256, 96), (4097, 1, 1, 24, 7),
    (262151, 1, 1, 2, 1), (262146, 1, 1, 7, 3),
])
def test_rope_by_axes_of_rows_that_share_a_workgroup(rows, heads, kv_heads, dim, pairs, grouped, interleaved):
    """Two or four rows of few heads at a time, the last ones fewer; a workgroup's second such rows, from 262144 rows on."""
    print(f"[rope] {rows} {heads}/{kv_heads} {dim} {pairs} {grouped} {interleaved}", flush=True)
    with Gpu() as g:
        check_rope(g, rows, heads, kv_heads, dim, pairs, grouped=grouped, interleaved=interleaved, seed=dim)
        check_rope(g, rows, heads, kv_heads, dim, pairs, axes=2, grouped=grouped, interleaved=interleaved, norm=False, seed=pairs)


@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("dim,pairs,interleaved", [(136, 64, 0), (130, 45, 0), (130, 45, 1)])
def test_rope_by_axes_of_more_rows_than_workgroups(dim, pairs, interleaved, norm):
    """Workgroups that take a second row after their first. Sampled rows of both, the last ones among them."""
    rows, heads, kv_heads, axes = 66001, 15, 1, 3
    print(f"[rope] {rows} {dim} {pairs} {interleaved} {norm}", flush=True)
    rng = np.random.RandomState(dim)
    frequencies, axis = 10000.0 ** -rng.rand(pairs), rng.randint(0, axes, pairs)
    positions = (rng.randint(-40, 40, (rows, axes)) * 0.37).astype(np.float32)
    weights = [normal(dim, 3 + i) for i in range(2)] if norm else [None, None]
    with Gpu() as g:
        qkv, p, outs = g.empty(rows * 17 * dim), g.from_f32(positions), [g.empty(rows * n * dim) for n in (heads, kv_heads, kv_heads)]
        w = [g.from_bf16(x).handle if norm else None for x in weights]
        with rope_axes(g, list(frequencies), axis, axes, interleaved) as plan:
            g.begin()
            fill(g, qkv, 1, 2.0)
            g.check(g.lib.h3_hip_qkv_rope_axes_bf16(g.handle, *(o.handle for o in outs), qkv.handle, *w, plan, p.handle, rows, heads,
                                                    kv_heads, dim, 0, C.c_float(EPS)), "rope")
            g.submit()
        at = np.unique(np.concatenate([np.arange(64), rng.randint(0, rows, 500), np.arange(32900, 33100), np.arange(rows - 64, rows)]))
        want = rope_reference(bf16(qkv.read().reshape(rows, 17, dim)[at]).astype(np.float64),
                              [None if x is None else bf16(x).astype(np.float64) for x in weights], frequencies, axis, positions[at],
                              heads, kv_heads, 0, interleaved)
        for o, n, (y, bound) in zip(outs, (heads, kv_heads, kv_heads), want):
            within(bf16(o.read().reshape(rows, n, dim)[at]), y, bound, (dim, n))


# ------------------------------------------------------------------ adapters
@pytest.mark.parametrize("rows,k,n,ranks", [(1500, 64, 6000, [16, 40, 128]), (3500, 72, 5999, [16, 40, 128]), (2900, 200, 5001, [70, 3])])
def test_adapters_of_many_columns_a_workgroup(rows, k, n, ranks):
    """Workgroups that go through 8 to 16 steps of 64 columns, the last one through fewer, in place too."""
    print(f"[adapters] {rows}x{k}x{n} {ranks}", flush=True)
    with Gpu() as g:
        first = check_adapters(g, rows, k, n, ranks, seed=rows)
        assert np.array_equal(check_adapters(g, rows, k, n, ranks, seed=rows, in_place=True), first)


def test_adapters_of_the_most_columns_a_workgroup():
    """32 steps of 64 columns: sampled rows have the bits that they get in a call of their own."""
    rows, k, n, ranks = 17000, 64, 11999, [16, 40]
    with Gpu() as g:
        x, base, out = g.from_bf16(normal(rows * k, 1)), g.empty(rows * n), g.empty(rows * n)
        at, ad = row_map(rows, 2, 5), Adapters(g, ranks, k, n)
        some = np.unique(np.random.RandomState(2).randint(0, rows, 150))
        with adapter_rows(g, at, 2, 40) as plan:
            g.begin()
            fill(g, base, 7)
            g.check(g.lib.h3_hip_adapters_add_bf16(g.handle, out.handle, base.handle, x.handle, ad.handle, plan, rows, k, n), "adapters")
            g.submit()
        few = [g.from_bf16(np.ascontiguousarray(t.read().reshape(rows, -1)[some])) for t in (base, x)]
        got, own = out.read().reshape(rows, n)[some], g.empty(len(some) * n)
        with adapter_rows(g, at[some], 2, 40) as plan:
            g.begin()
            g.check(g.lib.h3_hip_adapters_add_bf16(g.handle, own.handle, few[0].handle, few[1].handle, ad.handle, plan, len(some), k, n))
            g.submit()
        assert np.array_equal(got, own.read().reshape(-1, n))
        ad.close()


def test_adapters_hand_their_first_product_on_in_two_roundings():
    """base takes the rounded product away, so that what is left shows how the product was held: two BF16 values
    leave 2^-17 of it, the second rounding of what the first, 2^-8, left."""
    rows, k, n = 96, 64, 8
    with Gpu() as g:
        ad = Adapters(g, [1], k, n, scales=[1.0])
        ad.set(0, b=np.full((n, 1), 0x3f80, np.uint16))
        x = np.zeros((rows, k), np.uint16)
        x[:, [3, 20, 61]] = normal(rows * 3, 4).reshape(rows, 3)
        fx, fa = bf16(x).astype(np.float64), bf16(ad.a[0]).astype(np.float64)
        t, size = fx @ fa.T, np.abs(fx) @ np.abs(fa).T
        base = np.repeat(synth.f32_to_bf16(-t.astype(np.float32)), n, axis=1)
        tx, tb, out = g.from_bf16(x), g.from_bf16(base), g.empty(rows * n)
        with adapter_rows(g, [0] * rows, 1, 1) as plan:
            g.begin()
            g.check(g.lib.h3_hip_adapters_add_bf16(g.handle, out.handle, tb.handle, tx.handle, ad.handle, plan, rows, k, n), "adapters")
            g.submit()
        want = t + bf16(base).astype(np.float64)
        # Three exact products' sum, the scaling, the two values' sum and base's: FP32; one rounding to BF16.
        bound = 2.0 ** -17 * np.abs(t) + 6 * F32 * size
        within(bf16(out.read()).reshape(rows, n), want, bound + HALF * (np.abs(want) + bound))
        ad.close()


@pytest.mark.parametrize("mode", [1, 2], ids=["fp8", "nvfp4"])
@pytest.mark.parametrize("rows", [1, 70, 300])
def test_adapters_beside_packed_weights(mode, rows, tmp_path):
    """Beside per-tensor FP8 and NVFP4 weights: the same bits as the two calls."""
    k, n, ranks = 512, 1024, [16, 48]
    write_weight(tmp_path / "w.bin", normal(n * k, 2, scale=0.05))
    with Gpu() as g:
        g.check(configure(g, tmp_path / "cache", mode=mode), "configure")
        w, x, at = load(g, tmp_path / "w.bin", n, k, mode=mode), normal(rows * k, 1), row_map(rows, 2, 3)
        tx, out, base, both = g.from_bf16(x), g.empty(rows * n), g.empty(rows * n), g.empty(rows * n)
        ad = Adapters(g, ranks, k, n)
        with adapter_rows(g, at, 2, 48) as plan:
            g.begin()
            g.check(g.lib.h3_hip_linear_adapters_bf16(g.handle, out.handle, tx.handle, w.handle, None, ad.handle, plan, rows, k, n), "linear")
            g.check(g.lib.h3_gpu_linear_bf16(g.handle, base.handle, tx.handle, w.handle, None, rows, k, n))
            g.check(g.lib.h3_hip_adapters_add_bf16(g.handle, both.handle, base.handle, tx.handle, ad.handle, plan, rows, k, n))
            g.submit()
        got = out.read()
        assert np.array_equal(got, both.read())
        fb = bf16(base.read()).astype(np.float64).reshape(rows, n)
        within(bf16(got).reshape(rows, n), *ad.reference(bf16(x).astype(np.float64).reshape(rows, k), at, fb, np.zeros_like(fb)))
        ad.close()


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


# ------------------------------------------------------------------ together
@pytest.mark.parametrize("lengths", [(1,), (70, 1, 0, 133), (300, 260, 33)])
def test_each_stage_of_a_step(lengths):
    """Every value of every stage, against 64 bits of what the stage before it left."""
    print(f"[step] {lengths}", flush=True)

    def projected(x, w, n, adapters):
        fx, fw = bf16(x).astype(np.float64).reshape(step.rows, -1), bf16(w.read()).astype(np.float64).reshape(n, -1)
        base, sums = fx @ fw.T, (fw.shape[1] + 64) * F32 * (np.abs(fx) @ np.abs(fw).T)
        return adapters.reference(fx, step.at, base, sums + HALF * (np.abs(base) + sums))

    with Gpu() as g:
        step = Step(g, lengths)
        x = normal(step.rows * step.hidden, 5)
        tx = g.from_bf16(x)
        g.begin()
        step.run(tx)
        g.submit()
        t = {name: v.read() for name, v in step.t.items()}
        f = {name: bf16(v).astype(np.float64).reshape(step.rows, -1, 128) for name, v in t.items()}
        within(f["qkv"].reshape(step.rows, -1), *projected(x, step.w[0], step.qkv_width, step.adapters[0]), "projection")
        turned_parts = rope_reference(f["qkv"], [bf16(w.read()).astype(np.float64) for w in step.norms], 10000.0 ** -(np.arange(64) / 64),
                                      np.array([0, 1] * 32), step.positions.read().reshape(-1, 2), step.heads, step.kv_heads, 0, 0)
        for name, (want, bound) in zip("qkv", turned_parts):
            within(f[name], want, bound, name)
        ends = np.cumsum([0] + list(lengths))
        for a, b in zip(ends, ends[1:]):
            for h in range(step.heads if b > a else 0):
                kv = h // (step.heads // step.kv_heads)
                within(f["o"][a:b, h], *attention_reference(f["q"][a:b, h], f["k"][a:b, kv], f["v"][a:b, kv], SCALE), (a, h))
        within(f["y"].reshape(step.rows, -1), *projected(t["o"], step.w[1], step.hidden, step.adapters[1]), "output")
        step.close()
