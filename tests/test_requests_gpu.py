"""Operators of a step that serves several requests at once: attention of packed sequences,
rotation by positions of several axes with the norms of Q and K, low-rank adapters beside a
projection. Each against its formula in 64 bits.

Bounds. HALF is BF16's largest rounding error relative to the value, F32 that of FP32; a sum
of n products in FP32 is off by at most n * F32 times the sum of the products' magnitudes."""
import ctypes as C
import math

import numpy as np
import pytest

from h3cli_amd import synth
from h3cli_amd._lib import F32 as F32_TENSOR
from h3cli_amd.runtime import Gpu, H3Error
from tests.helpers import bf16
from tests.test_capture_gpu import Graph

pytestmark = pytest.mark.gpu

HALF, F32 = 2.0 ** -8, 2.0 ** -24
SCALE = 0.08837890625   # 1 / sqrt(128) in BF16
EPS = 1e-5


def u32(values):
    return (C.c_uint32 * len(values))(*(int(v) for v in values))


def normal(count, seed, scale=1.0):
    return synth.normal_bf16(seed, max(int(count), 1), scale=scale)[:int(count)]


def within(got, want, bound, what=""):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    off = np.abs(got - want) - bound
    assert np.all(np.isfinite(got)) and np.all(off <= 0), (what, float(np.max(off)), int(np.argmax(off)))


class Plan:
    def __init__(self, g, handle, free):
        g.check(handle, "plan")
        self.g, self.handle, self.free_handle = g, handle, free

    def __enter__(self):
        return self.handle

    def __exit__(self, *exc):
        self.free_handle(self.handle)


# ------------------------------------------------------------------ attention of sequences
def sequences(g, q_offsets, k_offsets, heads, kv_heads):
    h = g.lib.h3_hip_sequences_new(g.handle, u32(q_offsets), None if k_offsets is None else u32(k_offsets),
                                   len(q_offsets) - 1, heads, kv_heads)
    return Plan(g, h, g.lib.h3_hip_sequences_free)


def attention_reference(q, k, v, scale):
    """softmax(scale q k^T) v of one head in 64 bits, and the bound of the operator's error."""
    s = scale * (q @ k.T)
    size = scale * (np.abs(q) @ np.abs(k).T)
    p = np.exp(s - s.max(axis=1, keepdims=True))
    p /= p.sum(axis=1, keepdims=True)
    out, weight = p @ v, p @ np.abs(v)
    # A score is off by 128 products' sum, its scaling and the exponential's argument and result; a
    # probability relatively by as much, in the numerator and in the sum; P is rounded to BF16.
    score = (130 * F32 * size + 8 * F32 * (1 + np.abs(s))).max(axis=1, keepdims=True) + 8 * F32
    return out, HALF * np.abs(out) + (HALF + 2 * score + 2 * (len(k) + 64) * F32) * weight * (1 + HALF)


def check_attention(g, q_offsets, k_offsets, heads, kv_heads, seed=1, spread=1.0, scale=SCALE, rows=None, rising=0.0, heads_seen=None):
    """One call against the reference; rows of no sequence hold NaN in the inputs and must stay in the
    output. rising: how much a sequence's last keys are larger than its first."""
    at = k_offsets if k_offsets is not None else q_offsets
    rows = rows or (q_offsets[-1] + 3, at[-1] + 5)
    share = heads // kv_heads
    q, k, v = (normal(rows[i > 0] * n * 128, seed + i, scale=spread if i < 2 else 1.0).reshape(rows[i > 0], n, 128).copy()
               for i, n in ((0, heads), (1, kv_heads), (2, kv_heads)))
    if rising:
        for a, b in zip(at, at[1:]):
            k[a:b] = synth.f32_to_bf16(bf16(k[a:b]) * np.linspace(1, 1 + rising, b - a, dtype=np.float32)[:, None, None])
    for t, ends in ((q, q_offsets), (k, at), (v, at)):
        t[:ends[0]] = 0x7fc0
        t[ends[-1]:] = 0x7f80
    mark = normal(q.size, seed + 9).reshape(q.shape)
    tq, tk, tv, out = (g.from_bf16(t) for t in (q, k, v, mark))
    with sequences(g, q_offsets, k_offsets, heads, kv_heads) as plan:
        g.begin()
        g.check(g.lib.h3_hip_sdpa_sequences_bf16(g.handle, out.handle, tq.handle, tk.handle, tv.handle, plan, C.c_float(scale)),
                "attention")
        kernel = g.last_kernel()
        g.submit()
        got = out.read().reshape(q.shape)
        g.begin()
        g.check(g.lib.h3_hip_sdpa_sequences_bf16(g.handle, out.handle, tq.handle, tk.handle, tv.handle, plan, C.c_float(scale)),
                "attention")
        g.submit()
        assert np.array_equal(out.read().reshape(q.shape), got)
    assert np.array_equal(got[:q_offsets[0]], mark[:q_offsets[0]]) and np.array_equal(got[q_offsets[-1]:], mark[q_offsets[-1]:])
    fq, fk, fv = (bf16(t).astype(np.float64) for t in (q, k, v))
    for i in range(len(q_offsets) - 1):
        qs, ks = slice(q_offsets[i], q_offsets[i + 1]), slice(at[i], at[i + 1])
        if at[i] == at[i + 1]:
            assert not np.any(got[qs] & 0x7fff)
            continue
        for h in range(heads) if heads_seen is None else heads_seen:
            want, bound = attention_reference(fq[qs, h], fk[ks, h // share], fv[ks, h // share], scale)
            within(bf16(got[qs, h]), want, bound, (kernel, i, h))
    for t in (tq, tk, tv, out):
        g.free(t)
    return kernel


@pytest.mark.parametrize("q_offsets,k_offsets,heads,kv_heads", [
    ([0, 1], None, 1, 1),
    ([0, 1, 8, 72], None, 8, 8),
    ([2, 65, 65, 194, 195], None, 3, 3),                    # rows before the first, an empty sequence
    ([0, 31, 64, 97], [0, 63, 127, 192], 2, 1),             # tiles of 64 keys, less one and one more
    ([0, 1, 2, 5, 6], [0, 700, 701, 701, 1300], 10, 2),     # single rows, one of a sequence without keys
    ([0, 5, 5, 9], [7, 7, 20, 333], 6, 3),                  # queries without keys, keys without queries
    ([0, 33], [0, 129], 7, 1),                              # all query heads share a key head
    ([0, 300, 1100, 1130], None, 4, 4),
    ([0, 200], [0, 900], 40, 8),
])
@pytest.mark.parametrize("variant", [0, 20, 21, 22])
def test_attention_of_sequences(q_offsets, k_offsets, heads, kv_heads, variant, monkeypatch):
    """By the kernel that the plan chooses, and by those of 32, 128 and (from 257 keys on) 256 rows."""
    print(f"[sequences] {q_offsets} {k_offsets} {heads}/{kv_heads} {variant}", flush=True)
    monkeypatch.setenv("H3_HIP_ATTENTION_VARIANT", str(variant))
    with Gpu() as g:
        check_attention(g, q_offsets, k_offsets, heads, kv_heads, seed=len(q_offsets) * 17 + heads)


@pytest.mark.parametrize("variant", [20, 21, 22])
@pytest.mark.parametrize("spread,scale", [(6.0, SCALE), (0.01, SCALE), (1.0, 3.0), (1.0, 2.0 ** -20)])
def test_attention_of_sequences_peaks_and_flat_rows(spread, scale, variant, monkeypatch):
    monkeypatch.setenv("H3_HIP_ATTENTION_VARIANT", str(variant))
    with Gpu() as g:
        check_attention(g, [0, 70, 135], [0, 300, 650], 2, 2, seed=5, spread=spread, scale=scale)


@pytest.mark.parametrize("q_offsets,k_offsets,heads,kv_heads,rising", [
    ([0, 700, 1500], None, 4, 4, 0.0),
    ([1, 258, 258, 1000, 1513], None, 3, 3, 30.0),                  # later keys' scores far above the first's
    ([0, 600, 1000], [3, 260, 900], 10, 2, 0.0),                    # shared key heads: rows of five heads in a tile
    ([0, 513, 770, 1500], [0, 640, 897, 2000], 2, 2, 5.0),
    ([0, 1100, 1130, 1131, 1200], [0, 900, 1000, 2400, 2400], 4, 4, 0.0),   # and short ones beside them
])
def test_attention_of_sequences_by_tiles(q_offsets, k_offsets, heads, kv_heads, rising, monkeypatch):
    """The kernel of 256-row tiles, with the recomputation where a row's scores rise."""
    print(f"[sequences] {q_offsets} {k_offsets} {heads}/{kv_heads}", flush=True)
    monkeypatch.setenv("H3_HIP_ATTENTION_VARIANT", "22")
    with Gpu() as g:
        kernel = check_attention(g, q_offsets, k_offsets, heads, kv_heads, seed=7, rising=rising)
        assert kernel in ("attn_bf16_pipe", "attn_sequences rows=128"), kernel


def test_attention_of_one_sequence_is_the_dense_attention():
    seq, heads = 4133, 12
    with Gpu() as g:
        ts = [g.from_bf16(normal(seq * heads * 128, i)) for i in range(3)]
        a, b = g.empty(seq * heads * 128), g.empty(seq * heads * 128)
        with sequences(g, [0, seq], None, heads, heads) as plan:
            g.begin()
            g.check(g.lib.h3_hip_sdpa_sequences_bf16(g.handle, a.handle, *(t.handle for t in ts), plan, C.c_float(SCALE)))
            assert g.last_kernel() == "attn_bf16_pipe"
            g.check(g.lib.h3_gpu_sdpa_bf16(g.handle, b.handle, *(t.handle for t in ts), seq, heads, 128, C.c_float(SCALE)))
            assert g.last_kernel() == "attn_bf16_pipe"
            g.submit()
        assert np.array_equal(a.read(), b.read())


@pytest.mark.parametrize("q_offsets,k_offsets,heads,kv_heads,rising", [
    ([0, 729, 1535], None, 3, 3, 0.0),
    ([2, 131, 131, 260, 700], None, 4, 4, 20.0),                    # 128 rows and one more
    ([0, 100, 250, 251], [0, 64, 64, 700], 10, 2, 0.0),             # queries without keys; rows of five heads in a block
    ([0, 128, 400], [0, 65, 330], 9, 3, 6.0),
])
def test_attention_of_sequences_by_128_rows(q_offsets, k_offsets, heads, kv_heads, rising, monkeypatch):
    print(f"[sequences] {q_offsets} {k_offsets} {heads}/{kv_heads}", flush=True)
    monkeypatch.setenv("H3_HIP_ATTENTION_VARIANT", "21")
    with Gpu() as g:
        kernel = check_attention(g, q_offsets, k_offsets, heads, kv_heads, seed=11, rising=rising)
        assert kernel == "attn_sequences rows=128", kernel


@pytest.mark.parametrize("lengths,heads,kernel", [((1000,), 8, "rows=32"), ((729, 806), 56, "rows=128"), ((8193,), 12, "attn_bf16_pipe")])
def test_plans_choose_by_rows_and_heads(lengths, heads, kernel):
    with Gpu() as g:
        rows = sum(lengths)
        t, out = g.empty(rows * heads * 128), g.empty(rows * heads * 128)
        with sequences(g, np.cumsum([0] + list(lengths)), None, heads, heads) as plan:
            g.begin()
            g.check(g.lib.h3_hip_fill_normal_bf16(g.handle, t.handle, 1, C.c_float(1.0), t.elements))
            g.check(g.lib.h3_hip_sdpa_sequences_bf16(g.handle, out.handle, t.handle, t.handle, t.handle, plan, C.c_float(SCALE)))
            assert kernel in g.last_kernel(), g.last_kernel()
            g.submit()


@pytest.mark.parametrize("q_offsets,k_offsets,heads,kv_heads", [
    ([0, 1], [0, 18225], 5, 1),
    ([0, 1, 2, 5, 6], [0, 6000, 6001, 6001, 9000], 10, 2),
    ([0, 40, 41], [0, 5000, 9001], 3, 1),                    # two blocks of rows, the second cut off
    ([0, 4], [2, 8195], 1, 1),
    ([0, 2, 3], [0, 3000, 5200], 40, 40),                    # few parts each
])
def test_attention_of_few_rows_over_many_keys(q_offsets, k_offsets, heads, kv_heads):
    print(f"[sequences] {q_offsets} {k_offsets} {heads}/{kv_heads}", flush=True)
    with Gpu() as g:
        for rising in (0.0, 4.0):
            kernel = check_attention(g, q_offsets, k_offsets, heads, kv_heads, seed=3, rising=rising)
            assert kernel == "attn_sequences rows=32 shares=2", kernel     # parts, joined


@pytest.mark.parametrize("variant,q_rows,keys", [(20, 3, 700), (21, 130, 700), (22, 300, 700)])
def test_attention_of_keys_behind_4_gib(variant, q_rows, keys, monkeypatch):
    monkeypatch.setenv("H3_HIP_ATTENTION_VARIANT", str(variant))
    first = (1 << 32) // 256 + 5                            # a row of K is 256 bytes
    with Gpu() as g:
        q = g.from_bf16(normal(q_rows * 128, 1))
        k, v, out = g.empty((first + keys) * 128), g.empty((first + keys) * 128), g.empty(q_rows * 128)
        for t, seed in ((k, 2), (v, 3)):
            g.begin()
            g.check(g.lib.h3_hip_fill_normal_bf16(g.handle, t.handle, seed, C.c_float(1), (first + keys) * 128), "fill")
            g.submit()
        with sequences(g, [0, q_rows], [first, first + keys], 1, 1) as plan:
            g.begin()
            g.check(g.lib.h3_hip_sdpa_sequences_bf16(g.handle, out.handle, q.handle, k.handle, v.handle, plan, C.c_float(SCALE)),
                    "attention")
            g.submit()
        fq, fk, fv = (bf16(t.read()[-rows * 128:]).reshape(rows, 128).astype(np.float64)
                      for t, rows in ((q, q_rows), (k, keys), (v, keys)))
        within(bf16(out.read()).reshape(q_rows, 128), *attention_reference(fq, fk, fv, SCALE))


@pytest.mark.parametrize("variant", [20, 21, 22])
def test_attention_of_sequences_reports_values_that_are_not_finite(variant, monkeypatch):
    """In a query, key or value of any sequence; the others' results stay whole."""
    monkeypatch.setenv("H3_HIP_ATTENTION_VARIANT", str(variant))
    rows, cut = 400, 60
    for which in range(3):
        with Gpu() as g:
            ts = [normal(rows * 256, 3 + i).reshape(rows, 2, 128).copy() for i in range(3)]
            clean = [g.from_bf16(t) for t in ts]
            ts[which][77 + 4 * variant, 1, 5] = 0x7f80 if which else 0x7fc0
            dirty = [g.from_bf16(t) for t in ts]
            out, other = g.empty(rows * 256), g.empty(rows * 256)
            with sequences(g, [0, cut, rows], None, 2, 2) as plan:
                args = (plan, C.c_float(SCALE))
                g.begin()
                g.check(g.lib.h3_hip_sdpa_sequences_bf16(g.handle, out.handle, *(t.handle for t in clean), *args))
                g.submit()
                g.begin()
                g.check(g.lib.h3_hip_sdpa_sequences_bf16(g.handle, other.handle, *(t.handle for t in dirty), *args))
                with pytest.raises(H3Error, match="nonfinite attention"):
                    g.submit()
                g.cancel()
                a, b = out.read().reshape(rows, 2, 128), other.read().reshape(rows, 2, 128)
                assert np.array_equal(a[:cut], b[:cut]) and np.array_equal(a[cut:, 0], b[cut:, 0])


# ------------------------------------------------------------------ rotation by axes
def rope_axes(g, frequencies, axis, axes, interleaved):
    h = g.lib.h3_hip_rope_axes_new(g.handle, (C.c_double * len(frequencies))(*frequencies), u32(axis), len(frequencies), axes,
                                   interleaved)
    return Plan(g, h, g.lib.h3_hip_rope_axes_free)


def rope_reference(qkv, weights, frequencies, axis, positions, heads, kv_heads, grouped, interleaved):
    """Query, key and value in 64 bits, each with the bound of the operator's error."""
    rows, dim, pairs, share = qkv.shape[0], qkv.shape[2], len(frequencies), heads // kv_heads
    if grouped:
        x = qkv.reshape(rows, kv_heads, share + 2, dim)
        parts = [x[:, :, :share].reshape(rows, heads, dim), x[:, :, share], x[:, :, share + 1]]
    else:
        parts = [qkv[:, :heads], qkv[:, heads:heads + kv_heads], qkv[:, heads + kv_heads:]]
    angle = positions.astype(np.float64)[:, axis] * np.asarray(frequencies)
    c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
    first = np.arange(pairs) * (2 if interleaved else 1)
    second = first + (1 if interleaved else pairs)
    out = []
    for x, w in zip(parts, weights):
        y = x / np.sqrt((x * x).mean(axis=2, keepdims=True) + EPS) * w if w is not None else x.copy()
        a, b = y[..., first].copy(), y[..., second].copy()
        size = np.abs(y)
        y[..., first], y[..., second] = a * c - b * s, b * c + a * s
        size[..., first] = size[..., second] = np.abs(a) + np.abs(b)
        # The norm: a sum of dim squares, its root's reciprocal, three products; the rotation: the
        # hardware's sine and cosine to 2^-18 at phases off by 2^-23 turns; one rounding to BF16.
        out.append((y, HALF * np.abs(y) + size * (1 + HALF) * (2.0 ** -18 + 2 * math.pi * 2.0 ** -23 + (dim + 12) * F32)))
    out.append((parts[2], np.zeros_like(parts[2])))
    return out


def check_rope(g, rows, heads, kv_heads, dim, pairs, axes=3, grouped=0, interleaved=0, norm=True, far=0.0, seed=1):
    rng = np.random.RandomState(seed)
    qkv = normal(rows * (heads + 2 * kv_heads) * dim, seed, scale=2.0).reshape(rows, -1, dim)
    weights = [synth.f32_to_bf16((1 + 0.2 * rng.randn(dim)).astype(np.float32)) for _ in range(2)] if norm else [None, None]
    frequencies, axis = 10000.0 ** -rng.rand(pairs), rng.randint(0, axes, pairs)
    positions = (rng.randint(-40, 40, (rows, axes)) * 0.37 + far).astype(np.float32)
    mark = [normal((rows + 2) * n * dim, seed + 3) for n in (heads, kv_heads, kv_heads)]
    outs = [g.from_bf16(m) for m in mark]
    held = [g.from_bf16(qkv), g.from_f32(positions)] + [g.from_bf16(w) for w in weights if w is not None]
    with rope_axes(g, frequencies, axis, axes, interleaved) as plan:
        g.begin()
        g.check(g.lib.h3_hip_qkv_rope_axes_bf16(
            g.handle, *(o.handle for o in outs), held[0].handle, held[2].handle if norm else None,
            held[3].handle if norm else None, plan, held[1].handle, rows, heads, kv_heads, dim, grouped, C.c_float(EPS)), "rope")
        g.submit()
    want = rope_reference(bf16(qkv).astype(np.float64), [None if w is None else bf16(w).astype(np.float64) for w in weights],
                          frequencies, axis, positions, heads, kv_heads, grouped, interleaved)
    for o, m, (y, bound), n in zip(outs, mark, want, (heads, kv_heads, kv_heads)):
        got = o.read().reshape(-1, n, dim)
        assert np.array_equal(got[rows:].reshape(-1), m[rows * n * dim:])
        within(bf16(got[:rows]), y, bound, (rows, heads, kv_heads, dim, pairs, grouped, interleaved))
    for t in outs + held:
        g.free(t)


@pytest.mark.parametrize("interleaved", [0, 1])
@pytest.mark.parametrize("grouped", [0, 1])
@pytest.mark.parametrize("rows,heads,kv_heads,dim,pairs", [
    (1, 1, 1, 128, 64), (1, 56, 56, 128, 48), (5, 6, 2, 90, 37), (33, 4, 1, 64, 32), (7, 5, 5, 128, 3), (3, 3, 3, 7, 3),
    (19, 2, 2, 256, 128), (6, 8, 2, 256, 96), (5, 2, 1, 80, 24), (9, 3, 3, 24, 8), (300, 7, 7, 128, 48), (2, 4, 2, 255, 127),
    (4, 1, 1, 2, 1), (11, 17, 17, 8, 4), (23, 6, 3, 16, 8), (3, 2, 2, 32, 12),
])
def test_rope_by_axes(rows, heads, kv_heads, dim, pairs, grouped, interleaved):
    with Gpu() as g:
        check_rope(g, rows, heads, kv_heads, dim, pairs, grouped=grouped, interleaved=interleaved, seed=rows + dim)
        check_rope(g, rows, heads, kv_heads, dim, pairs, axes=1, grouped=grouped, interleaved=interleaved, norm=False, seed=rows)


@pytest.mark.parametrize("far", [1e5, -1e5, 1.6e7, 3e9])
def test_rope_by_axes_keeps_the_phase_of_far_positions(far):
    with Gpu() as g:
        check_rope(g, 12, 2, 2, 128, 48, axes=16, far=far)
        check_rope(g, 12, 2, 2, 90, 45, interleaved=1, far=far)


def test_rope_by_axes_passes_other_channels_as_they_are():
    """Without norms, channels behind the pairs and all of V: infinities and NaN's bits among them."""
    for dim, pairs in ((128, 32), (90, 21)):
        with Gpu() as g:
            qkv = normal(6 * 3 * dim, 4).reshape(6, 3, dim).copy()
            qkv[2, :, 2 * pairs + 1], qkv[3, 2, 0], qkv[4, 2, 1] = 0x7f80, 0x7fc1, 0xff80
            t, p = g.from_bf16(qkv), g.from_f32(np.ones((6, 1), np.float32))
            outs = [g.empty(6 * dim) for _ in range(3)]
            with rope_axes(g, [0.5] * pairs, [0] * pairs, 1, 0) as plan:
                g.begin()
                g.check(g.lib.h3_hip_qkv_rope_axes_bf16(g.handle, *(o.handle for o in outs), t.handle, None, None, plan, p.handle,
                                                        6, 1, 1, dim, 0, C.c_float(EPS)), "rope")
                g.submit()
            q, k, v = (o.read().reshape(6, dim) for o in outs)
            assert np.array_equal(v, qkv[:, 2])
            assert np.array_equal(q[:, 2 * pairs:], qkv[:, 0, 2 * pairs:]) and np.array_equal(k[:, 2 * pairs:], qkv[:, 1, 2 * pairs:])


# ------------------------------------------------------------------ adapters
class Adapters:
    def __init__(self, g, ranks, k, n, seed=1, scales=None):
        self.g, self.ranks, self.k, self.n = g, ranks, k, n
        self.handle = g.check(g.lib.h3_hip_adapters_new(g.handle, u32(ranks), len(ranks), k, n), "adapters")
        self.a = [normal(r * k, seed + 2 * i, scale=1 / math.sqrt(k)).reshape(r, k) for i, r in enumerate(ranks)]
        self.b = [normal(n * r, seed + 2 * i + 1, scale=1 / math.sqrt(r)).reshape(n, r) for i, r in enumerate(ranks)]
        self.scales = scales or [0.5 + 0.75 * (i % 3) for i in range(len(ranks))]
        for i in range(len(ranks)):
            self.set(i)

    def set(self, i, a=None, b=None, scale=None):
        g = self.g
        self.a[i], self.b[i] = self.a[i] if a is None else a, self.b[i] if b is None else b
        self.scales[i] = self.scales[i] if scale is None else scale
        ta, tb = g.from_bf16(self.a[i]), g.from_bf16(self.b[i])
        g.begin()
        g.check(g.lib.h3_hip_adapters_set(g.handle, self.handle, i, ta.handle, tb.handle, C.c_float(self.scales[i])), "set")
        g.submit()
        g.free(ta)
        g.free(tb)

    def close(self):
        self.g.lib.h3_hip_adapters_free(self.handle)

    def reference(self, x, at, base, base_error):
        """base + the parts of the rows' adapters in 64 bits, and the bound of the operator's error."""
        y, bound = base.copy(), base_error.copy()
        for i, r in enumerate(self.ranks):
            rows = np.flatnonzero(at == i)
            a, b, scale = bf16(self.a[i]).astype(np.float64), bf16(self.b[i]).astype(np.float64), float(np.float32(self.scales[i]))
            t, size = x[rows] @ a.T, np.abs(x[rows]) @ np.abs(a).T
            y[rows] += scale * t @ b.T
            # t: K products (in shares) and their scaling; two BF16 roundings in turn; 2 r products.
            t_error = (self.k + 16) * F32 * size + HALF ** 2 * np.abs(t)
            bound[rows] += abs(scale) * (t_error @ np.abs(b).T + (2 * r + 40) * F32 * (np.abs(t) + t_error) @ np.abs(b).T)
        return y, bound + HALF * (np.abs(y) + bound) + F32 * np.abs(y)


def adapter_rows(g, at, count, max_rank):
    h = g.lib.h3_hip_adapter_rows_new(g.handle, u32(at), len(at), count, max_rank)
    return Plan(g, h, g.lib.h3_hip_adapter_rows_free)


def row_map(rows, count, seed, none=True, mixed=True):
    rng = np.random.RandomState(seed)
    at = np.sort(rng.randint(0, count + (1 if none else 0), rows))
    return rng.permutation(at) if mixed else at


def check_adapters(g, rows, k, n, ranks, at=None, seed=1, in_place=False, max_rank=None):
    at = row_map(rows, len(ranks), seed) if at is None else np.asarray(at)
    x, base = normal(rows * k, seed + 50).reshape(rows, k), normal(rows * n, seed + 51).reshape(rows, n)
    w = Adapters(g, ranks, k, n, seed=seed)
    mark = normal((rows + 2) * n, seed + 52)
    if in_place:
        mark[:rows * n] = base.reshape(-1)
    tx, tb, out = g.from_bf16(x), g.from_bf16(base), g.from_bf16(mark)
    with adapter_rows(g, at, len(ranks), max_rank or max(ranks)) as plan:
        g.begin()
        g.check(g.lib.h3_hip_adapters_add_bf16(g.handle, out.handle, out.handle if in_place else tb.handle, tx.handle, w.handle,
                                               plan, rows, k, n), "adapters")
        g.submit()
    got = out.read()
    assert np.array_equal(got[rows * n:], mark[rows * n:])
    got = got[:rows * n].reshape(rows, n)
    none = at >= len(ranks)
    assert np.array_equal(got[none], base[none])
    fb = bf16(base).astype(np.float64)
    want, bound = w.reference(bf16(x).astype(np.float64), at, fb, np.zeros_like(fb))
    within(bf16(got[~none]), want[~none], bound[~none], (rows, k, n, ranks))
    w.close()
    for t in (tx, tb, out):
        g.free(t)
    return got


@pytest.mark.parametrize("rows,k,n,ranks", [
    (1, 64, 128, [16]), (1, 1, 1, [1]), (9, 256, 640, [16] * 8 + [64]), (31, 1001, 777, [1, 40, 7, 19]), (33, 72, 136, [33]),
    (64, 128, 1000, [32, 31]), (300, 136, 264, [128, 4, 65]), (130, 520, 1032, [256, 200, 96]), (1000, 64, 64, [8, 8, 8]),
    (5, 5376, 96, [16, 3]), (70, 2056, 516, [64]), (257, 500, 130, [17, 128]),
])
def test_adapters(rows, k, n, ranks):
    print(f"[adapters] {rows}x{k}x{n} {ranks}", flush=True)
    with Gpu() as g:
        first = check_adapters(g, rows, k, n, ranks, seed=rows + n)
        assert np.array_equal(check_adapters(g, rows, k, n, ranks, seed=rows + n, in_place=True, max_rank=256), first)


def test_adapters_of_rows_in_runs_and_of_no_row():
    with Gpu() as g:
        check_adapters(g, 100, 64, 192, [16, 32, 8], at=np.repeat([0, 2, 3], [40, 33, 27]))
        check_adapters(g, 100, 64, 192, [16, 32], at=[2] * 100)                    # none: base as it is
        check_adapters(g, 3, 64, 192, [16, 32], at=[0xffffffff, 1, 7])             # any index past the last is none


def test_adapters_are_replaced_and_start_as_zero():
    rows, k, n = 40, 96, 200
    with Gpu() as g:
        x, base = normal(rows * k, 1).reshape(rows, k), normal(rows * n, 2).reshape(rows, n)
        tx, tb, out = g.from_bf16(x), g.from_bf16(base), g.empty(rows * n)
        w = Adapters(g, [8, 24], k, n)
        fresh = g.check(g.lib.h3_hip_adapters_new(g.handle, u32([8, 24]), 2, k, n))
        at = row_map(rows, 2, 3)
        with adapter_rows(g, at, 2, 24) as plan:
            def call(handle):
                g.begin()
                g.check(g.lib.h3_hip_adapters_add_bf16(g.handle, out.handle, tb.handle, tx.handle, handle, plan, rows, k, n))
                g.submit()
                return out.read().reshape(rows, n)

            assert np.array_equal(call(fresh), base)
            first = call(w.handle)
            w.set(1, a=normal(24 * k, 70, scale=0.1).reshape(24, k), scale=-1.25)
            second = call(w.handle)
            assert np.array_equal(first[at != 1], second[at != 1]) and not np.array_equal(first[at == 1], second[at == 1])
            fb = bf16(base).astype(np.float64)
            want, bound = w.reference(bf16(x).astype(np.float64), at, fb, np.zeros_like(fb))
            within(bf16(second), want, bound)
        g.lib.h3_hip_adapters_free(fresh)
        w.close()


@pytest.mark.parametrize("k,n", [(128, 200), (65, 199)])
def test_adapters_keep_infinities_to_their_rows_and_signs(k, n):
    """Rank 1 with weights of one sign: an infinity of x gives infinities of the formula's signs in its
    own row, with no NaN from the ranks that fill the packed weights up; other rows are as without it."""
    rows = 40
    with Gpu() as g:
        w = Adapters(g, [1, 3], k, n)
        w.set(0, a=normal(k, 1) & 0x7fff, b=normal(n, 2), scale=1.0)
        at = np.arange(rows) % 3
        x = normal(rows * k, 3).reshape(rows, k).copy()
        tw = g.from_bf16(np.zeros(n * k, np.uint16))
        base, out = g.from_bf16(np.zeros(rows * n, np.uint16)), g.empty(rows * n)

        def call(values):
            tx = g.from_bf16(values)
            with adapter_rows(g, at, 2, 3) as plan:
                g.begin()
                if k % 64:
                    g.check(g.lib.h3_hip_linear_adapters_bf16(g.handle, out.handle, tx.handle, tw.handle, None, w.handle, plan, rows, k, n))
                else:
                    g.check(g.lib.h3_hip_adapters_add_bf16(g.handle, out.handle, base.handle, tx.handle, w.handle, plan, rows, k, n))
                g.submit()
            return out.read().reshape(rows, n)

        clean = call(x)
        x[6, 5], x[9, k - 1] = 0x7f80, 0xff80                # rows of adapter 0
        got = call(x)
        others = np.setdiff1d(np.arange(rows), (6, 9))
        assert np.array_equal(got[others], clean[others])
        if k % 64 == 0:                                      # the projection's weights of zero make NaN of an infinity
            positive = w.b[0].reshape(-1) < 0x8000
            assert np.array_equal(got[6], np.where(positive, 0x7f80, 0xff80))
            assert np.array_equal(got[9], np.where(positive, 0xff80, 0x7f80))
        w.close()


@pytest.mark.parametrize("kind", ["bf16", "q8", "fp8_block"])
@pytest.mark.parametrize("rows", [1, 70, 300])
def test_linear_with_adapters_is_the_projection_and_the_adapters(kind, rows):
    """Beside a projection of any type: the same bits as the two calls."""
    k, n, ranks = 512, 1024, [16, 48]
    with Gpu() as g:
        x = normal(rows * k, 1)
        tx, bias, out, base, sum_ = g.from_bf16(x), g.from_bf16(normal(n, 5)), g.empty(rows * n), g.empty(rows * n), g.empty(rows * n)
        bits = normal(n * k, 2, scale=1 / math.sqrt(k))
        if kind == "bf16":
            w = g.from_bf16(bits).handle
        elif kind == "q8":
            codes = np.random.RandomState(1).randint(-127, 128, (n, k)).astype(np.int8)
            scales = np.full((n, 1), 4e-4, np.float32)
            w = g.check(g.lib.h3_hip_q8_from_packed(g.handle, codes.ctypes.data, scales.ctypes.data, n, k, k))
        else:
            w = g.check(g.lib.h3_hip_fp8_block_weight_from_bf16(g.handle, g.from_bf16(bits).handle, n, k))
        at = row_map(rows, 2, 3)
        ad = Adapters(g, ranks, k, n)
        with adapter_rows(g, at, 2, 48) as plan:
            g.begin()
            g.check(g.lib.h3_hip_linear_adapters_bf16(g.handle, out.handle, tx.handle, w, bias.handle, ad.handle, plan, rows, k, n))
            g.check(g.lib.h3_gpu_linear_bf16(g.handle, base.handle, tx.handle, w, bias.handle, rows, k, n))
            g.check(g.lib.h3_hip_adapters_add_bf16(g.handle, sum_.handle, base.handle, tx.handle, ad.handle, plan, rows, k, n))
            g.submit()
        got = out.read()
        assert np.array_equal(got, sum_.read())
        fb = bf16(base.read()).astype(np.float64).reshape(rows, n)
        want, bound = ad.reference(bf16(x).astype(np.float64).reshape(rows, k), at, fb, np.zeros_like(fb))
        within(bf16(got).reshape(rows, n), want, bound)
        ad.close()
        if kind != "bf16":
            g.lib.h3_gpu_tensor_free(w)


@pytest.mark.parametrize("rows,k,n,ranks,bias", [
    (1, 1, 1, [1], True), (5, 65, 130, [16], False), (301, 1001, 777, [1, 40, 7, 19], True), (130, 72, 1000, [33, 64], False),
    (33, 5000, 64, [256], True), (1700, 4200, 1500, [70, 9], False), (1000, 200, 2049, [16, 8, 100], True),
    (2100, 520, 4100, [32, 32], False), (64, 1000, 7, [5], True),
])
def test_linear_with_adapters_of_any_width(rows, k, n, ranks, bias):
    """A BF16 weight whose K is no multiple of 64: one sum and one rounding for projection, bias and adapters."""
    print(f"[adapters] linear {rows}x{k}x{n} {ranks}", flush=True)
    with Gpu() as g:
        x, w, b = normal(rows * k, 1).reshape(rows, k), normal(n * k, 2, scale=1 / math.sqrt(k)).reshape(n, k), normal(n, 3)
        mark = normal((rows + 1) * n, 4)
        tx, tw, tb, out = (g.from_bf16(t) for t in (x, w, b, mark))
        at = row_map(rows, len(ranks), 5)
        ad = Adapters(g, ranks, k, n, seed=7)
        with adapter_rows(g, at, len(ranks), max(ranks)) as plan:
            g.begin()
            g.check(g.lib.h3_hip_linear_adapters_bf16(g.handle, out.handle, tx.handle, tw.handle, tb.handle if bias else None, ad.handle,
                                                      plan, rows, k, n), "linear")
            assert "adapter_gemm" in g.last_kernel()
            g.submit()
        got = out.read()
        assert np.array_equal(got[rows * n:], mark[rows * n:])
        fx, fw = bf16(x).astype(np.float64), bf16(w).astype(np.float64)
        base = fx @ fw.T + (bf16(b).astype(np.float64) if bias else 0)
        error = (k + 64) * F32 * (np.abs(fx) @ np.abs(fw).T + np.abs(bf16(b)) * bias)
        want, bound = ad.reference(fx, at, base, error)
        within(bf16(got[:rows * n]).reshape(rows, n), want, bound)
        ad.close()


# ------------------------------------------------------------------ together
def fill(g, t, seed, scale=1.0):
    g.check(g.lib.h3_hip_fill_normal_bf16(g.handle, t.handle, seed, C.c_float(scale), t.elements), "fill")


class Step:
    """Attention's half of a block for the rows of several requests: projection with adapters, norms and
    rotation, attention of the sequences, projection with adapters."""

    def __init__(self, g, lengths, hidden=384, heads=6, kv_heads=2, ranks=(16, 40), seed=1):
        self.g, self.rows, self.hidden, self.heads, self.kv_heads = g, sum(lengths), hidden, heads, kv_heads
        self.inner, self.qkv_width = heads * 128, (heads + 2 * kv_heads) * 128
        rng = np.random.RandomState(seed)
        ends = np.cumsum([0] + list(lengths))
        self.w = [g.from_bf16(normal(self.qkv_width * hidden, 11, scale=1 / math.sqrt(hidden))),
                  g.from_bf16(normal(hidden * self.inner, 12, scale=1 / math.sqrt(self.inner)))]
        self.norms = [g.from_bf16(synth.f32_to_bf16((1 + 0.1 * np.random.RandomState(i).randn(128)).astype(np.float32))) for i in (3, 4)]
        positions = np.concatenate([np.stack([np.arange(n) // 8 + 1000 * i, np.arange(n) % 8], axis=1) for i, n in enumerate(lengths)])
        self.positions = g.from_f32(positions.astype(np.float32))
        frequencies = 10000.0 ** -(np.arange(64) / 64)
        self.adapters = [Adapters(g, list(ranks), hidden, self.qkv_width, seed=21), Adapters(g, list(ranks), self.inner, hidden, seed=31)]
        at = np.repeat(np.arange(len(lengths)) % (len(ranks) + 1), lengths)
        self.at = at
        self.plans = [rope_axes(g, list(frequencies), [0, 1] * 32, 2, 0), sequences(g, ends, None, heads, kv_heads),
                      adapter_rows(g, at, len(ranks), max(ranks))]
        self.t = {name: g.empty(self.rows * width) for name, width in (
            ("qkv", self.qkv_width), ("q", self.inner), ("k", kv_heads * 128), ("v", kv_heads * 128), ("o", self.inner), ("y", hidden))}

    def run(self, x):
        g, lib, t, h = self.g, self.g.lib, {n: v.handle for n, v in self.t.items()}, self.g.handle
        rope, seqs, rows = (p.handle for p in self.plans)
        g.check(lib.h3_hip_linear_adapters_bf16(h, t["qkv"], x.handle, self.w[0].handle, None, self.adapters[0].handle, rows, self.rows,
                                                self.hidden, self.qkv_width), "qkv")
        g.check(lib.h3_hip_qkv_rope_axes_bf16(h, t["q"], t["k"], t["v"], t["qkv"], self.norms[0].handle, self.norms[1].handle, rope,
                                              self.positions.handle, self.rows, self.heads, self.kv_heads, 128, 0, C.c_float(EPS)), "rope")
        g.check(lib.h3_hip_sdpa_sequences_bf16(h, t["o"], t["q"], t["k"], t["v"], seqs, C.c_float(SCALE)), "attention")
        g.check(lib.h3_hip_linear_adapters_bf16(h, t["y"], t["o"], self.w[1].handle, None, self.adapters[1].handle, rows, self.rows,
                                                self.inner, self.hidden), "out")

    def close(self):
        for p in self.plans:
            p.__exit__()
        for a in self.adapters:
            a.close()


def step_reference(step, x, lengths):
    """The step in 64 bits, each stage's result rounded to BF16 as the operators hand it on."""
    def rounded(v):
        return bf16(synth.f32_to_bf16(np.asarray(v, np.float32))).astype(np.float64)

    def projected(v, w, n, adapters):
        base = rounded(v @ bf16(w.read()).astype(np.float64).reshape(n, -1).T)
        return rounded(adapters.reference(v, step.at, base, np.zeros_like(base))[0])

    qkv = projected(x, step.w[0], step.qkv_width, step.adapters[0]).reshape(step.rows, -1, 128)
    weights = [bf16(w.read()).astype(np.float64) for w in step.norms]
    (q, _), (k, _), (v, _) = rope_reference(qkv, weights, 10000.0 ** -(np.arange(64) / 64), np.array([0, 1] * 32),
                                            step.positions.read().reshape(-1, 2), step.heads, step.kv_heads, 0, 0)
    q, k, out, ends = rounded(q), rounded(k), np.zeros(q.shape), np.cumsum([0] + list(lengths))
    for a, b in zip(ends, ends[1:]):
        for h in range(step.heads if b > a else 0):
            kv = h // (step.heads // step.kv_heads)
            out[a:b, h] = attention_reference(q[a:b, h], k[a:b, kv], v[a:b, kv], SCALE)[0]
    return projected(rounded(out).reshape(step.rows, -1), step.w[1], step.hidden, step.adapters[1])


@pytest.mark.parametrize("lengths", [(1,), (70, 1, 0, 133), (300, 260, 33)])
def test_a_step_of_several_requests(lengths):
    """The operators one after another, against 64 bits: each stage keeps to BF16's rounding, so the
    result is off by a few of them; and every request's rows as in a step of its own."""
    print(f"[step] {lengths}", flush=True)
    with Gpu() as g:
        step = Step(g, lengths)
        x = normal(step.rows * step.hidden, 5)
        tx = g.from_bf16(x)
        g.begin()
        step.run(tx)
        g.submit()
        got = bf16(step.t["y"].read()).astype(np.float64).reshape(step.rows, -1)
        want = step_reference(step, bf16(x).astype(np.float64).reshape(step.rows, -1), lengths)
        # Six stages round (two of them twice), P once more: at most nine half steps if all went one way,
        # relative to the result's size.
        assert np.linalg.norm(got - want) <= 9 * HALF * np.linalg.norm(want)
        step.close()


def test_steps_captured_into_two_graphs():
    """Two graphs of one context with plans of their own, replayed in turn between eager work that uses
    the context's workspaces: every replay gives the same bits. (Captured projections are not split
    over K, so the eager step's bits may differ, by what rounding allows.)"""
    lengths = [(150, 90, 31), (400, 520)]
    with Gpu() as g:
        steps = [Step(g, n, seed=i) for i, n in enumerate(lengths)]
        xs = [g.from_bf16(normal(s.rows * s.hidden, 40 + i)) for i, s in enumerate(steps)]
        other = [g.empty(900 * 4096), g.empty(4096 * 4096), g.empty(900 * 4096)]
        want = []
        for s, x in zip(steps, xs):
            g.begin()
            s.run(x)
            g.submit()
            want.append(s.t["y"].read())
        graphs = []
        g.begin()
        for s, x in zip(steps, xs):
            graphs.append(Graph(g))
            with graphs[-1]:
                s.run(x)
        first = [None, None]
        for turn in range(3):
            for i in (0, 1, 0):
                fill(g, steps[i].t["y"], turn + 9)
                fill(g, other[0], turn)
                g.check(g.lib.h3_gpu_linear_bf16(g.handle, other[2].handle, other[0].handle, other[1].handle, None, 900, 4096, 4096))
                graphs[i].launch()
                g.submit()
                got = steps[i].t["y"].read()
                first[i] = got if first[i] is None else first[i]
                assert np.array_equal(got, first[i]), (turn, i)
                a, b = bf16(got).astype(np.float64), bf16(want[i]).astype(np.float64)
                assert np.linalg.norm(a - b) <= 18 * HALF * np.linalg.norm(b), (turn, i)
                g.begin()
        g.submit()
        for graph in graphs:
            graph.close()
        for s in steps:
            s.close()


def test_every_kernel_captured_with_its_plan():
    """Each kernel in one graph, adapters set within it: replays give the same bits, the eager call's but for
    a projection, whose sum an eager call may share out."""
    with Gpu() as g:
        plans, calls = [], []

        def attention(q_offsets, k_offsets, heads, kv_heads):
            rows = [(q_offsets[-1], heads), (k_offsets[-1], kv_heads), (k_offsets[-1], kv_heads)]
            t, out = [g.from_bf16(normal(n * h * 128, i)) for i, (n, h) in enumerate(rows)], g.empty(rows[0][0] * heads * 128)
            plans.append(sequences(g, q_offsets, k_offsets, heads, kv_heads))
            plan = plans[-1].handle
            calls.append((lambda: g.lib.h3_hip_sdpa_sequences_bf16(g.handle, out.handle, *(x.handle for x in t), plan, C.c_float(SCALE)),
                          out, True))

        def projection(rows, k, n, rank=70):
            x, w, out = g.from_bf16(normal(rows * k, 1)), g.from_bf16(normal(n * k, 2)), g.empty(rows * n)
            a, b = g.from_bf16(normal(rank * k, 3, scale=0.05)), g.from_bf16(normal(n * rank, 4))
            plans.append(Plan(g, g.lib.h3_hip_adapters_new(g.handle, u32([16, rank]), 2, k, n), g.lib.h3_hip_adapters_free))
            plans.append(adapter_rows(g, [i % 3 for i in range(rows)], 2, rank))
            weights, plan = plans[-2].handle, plans[-1].handle
            calls.append((lambda: g.lib.h3_hip_adapters_set(g.handle, weights, 1, a.handle, b.handle, C.c_float(0.5)) and
                          g.lib.h3_hip_linear_adapters_bf16(g.handle, out.handle, x.handle, w.handle, None, weights, plan, rows, k, n),
                          out, k % 64 != 0))

        attention([0, 1], [0, 18225], 5, 1)
        attention([0, 300, 700], [0, 300, 700], 8, 8)
        attention([0, 5000], [0, 5000], 8, 8)
        projection(301, 1001, 777)
        projection(300, 1024, 777)
        projection(600, 999, 3000)
        qkv, turned, positions = g.from_bf16(normal(40 * 3 * 128, 5)), [g.empty(40 * 128) for _ in range(3)], g.from_f32(np.arange(40.0))
        plans.append(rope_axes(g, [1.0, 0.1], [0, 0], 1, 0))
        calls.append((lambda: g.lib.h3_hip_qkv_rope_axes_bf16(g.handle, *(t.handle for t in turned), qkv.handle, None, None, plans[-1].handle,
                                                              positions.handle, 40, 1, 1, 128, 0, C.c_float(EPS)), turned[0], True))
        g.begin()
        graph = Graph(g)
        with graph:
            for call, _, _ in calls:
                g.check(call(), "captured")
        first = None
        for _ in range(3):
            graph.launch()
            g.submit()
            got = [out.read() for _, out, _ in calls]
            first = first or got
            assert all(np.array_equal(a, b) for a, b in zip(got, first))
            g.begin()
            for call, _, _ in calls:
                g.check(call(), "eager")
            g.submit()
            for i, ((_, out, same), captured) in enumerate(zip(calls, first)):
                eager = out.read()
                assert np.any(eager) and (not same or np.array_equal(eager, captured)), i
            g.begin()
        g.submit()
        graph.close()
        for p in plans:
            p.free_handle(p.handle)


class Streamed:
    """A BF16 tensor that is filled from pinned memory, again and again."""

    def __init__(self, g, versions):
        self.g, self.size = g, versions[0].size * 2
        self.tensor = g.empty(versions[0].size)
        self.sources = [g.check(g.lib.h3_hip_host_alloc(g.handle, self.size), "pinned memory") for _ in versions]
        for p, v in zip(self.sources, versions):
            C.memmove(p, np.ascontiguousarray(v).ctypes.data, self.size)

    def fill(self, i):
        self.g.check(self.g.lib.h3_hip_tensor_stream_host(self.tensor.handle, self.sources[i], self.size), "stream")

    def close(self):
        for p in self.sources:
            self.g.lib.h3_hip_host_free(self.g.handle, p, self.size)


def test_streamed_inputs_are_waited_for():
    """Adapters, keys and rows that are on their way when a call is made, and are filled anew behind it."""
    with Gpu() as g:
        # Two adapters from one tensor of 32 MB.
        rows, k, n, rank = 3, 1 << 16, 72, 256
        downs, up = [normal(rank * k, 5 + i, scale=0.01) for i in range(2)], g.from_bf16(normal(n * rank, 7))
        x, base = g.from_bf16(normal(rows * k, 8)), g.from_bf16(normal(rows * n, 9))
        streamed, plain = Streamed(g, downs), [g.from_bf16(d) for d in downs]
        outs = [g.empty(rows * n) for _ in range(2)]
        weights = [g.check(g.lib.h3_hip_adapters_new(g.handle, u32([rank, rank]), 2, k, n)) for _ in range(2)]
        with adapter_rows(g, [0, 1, 0], 2, rank) as plan:
            g.begin()
            for w, out, late in zip(weights, outs, (True, False)):
                for i in range(2):
                    if late:
                        streamed.fill(i)
                    a = streamed.tensor if late else plain[i]
                    g.check(g.lib.h3_hip_adapters_set(g.handle, w, i, a.handle, up.handle, C.c_float(1)), "set")
                g.check(g.lib.h3_hip_adapters_add_bf16(g.handle, out.handle, base.handle, x.handle, w, plan, rows, k, n), "adapters")
            g.submit()
        assert np.array_equal(outs[0].read(), outs[1].read()) and not np.array_equal(outs[0].read(), base.read())
        streamed.close()
        for w in weights:
            g.lib.h3_hip_adapters_free(w)
        # Keys of two contexts in one tensor of 41 MB, and the rows of a step.
        keys, heads = 20000, 8
        versions = [normal(keys * heads * 128, 20 + i) for i in range(2)]
        streamed, plain, v = Streamed(g, versions), [g.from_bf16(d) for d in versions], g.from_bf16(normal(keys * heads * 128, 23))
        q = g.from_bf16(normal(heads * 128, 24))
        outs = [g.empty(heads * 128) for _ in range(4)]
        turned = [[g.empty(keys // 3 * n * 128) for n in (6, 1, 1)] for _ in range(4)]
        positions = g.from_f32(np.arange(keys // 3, dtype=np.float32))
        with sequences(g, [0, 1], [0, keys], heads, heads) as plan, rope_axes(g, [1.0, 0.1], [0, 0], 1, 0) as rope:
            g.begin()
            for i in range(4):
                if i < 2:
                    streamed.fill(i)
                t = streamed.tensor if i < 2 else plain[i - 2]
                g.check(g.lib.h3_hip_sdpa_sequences_bf16(g.handle, outs[i].handle, q.handle, t.handle, v.handle, plan, C.c_float(SCALE)))
                if i < 2:
                    streamed.fill(i)
                g.check(g.lib.h3_hip_qkv_rope_axes_bf16(g.handle, *(o.handle for o in turned[i]), t.handle, None, None, rope,
                                                        positions.handle, keys // 3, 6, 1, 128, 0, C.c_float(EPS)))
            g.submit()
        for i in range(2):
            assert np.array_equal(outs[i].read(), outs[i + 2].read())
            assert all(np.array_equal(a.read(), b.read()) for a, b in zip(turned[i], turned[i + 2]))
        streamed.close()


def test_steps_of_two_contexts_at_once():
    """Two contexts, whose streams run side by side: the same bits as each alone."""
    with Gpu() as a, Gpu() as b:
        pairs = []
        for i, g in enumerate((a, b)):
            s = Step(g, (200 + 100 * i, 77), seed=i)
            x = g.from_bf16(normal(s.rows * s.hidden, 60 + i))
            g.begin()
            s.run(x)
            g.submit()
            pairs.append((g, s, x, s.t["y"].read()))
        for _ in range(3):
            for g, s, x, _ in pairs:
                g.begin()
                fill(g, s.t["y"], 3)
            for _ in range(4):
                for g, s, x, _ in pairs:
                    s.run(x)
            for g, s, x, want in pairs:
                g.submit()
                assert np.array_equal(s.t["y"].read(), want)
        for _, s, _, _ in pairs:
            s.close()


# ------------------------------------------------------------------ refusals
def refused(g, ok, text):
    assert not ok
    assert text in g.error(), g.error()


def test_refusals():
    with Gpu() as g, Gpu() as other:
        lib = g.lib
        # Plans.
        for ends, heads, kv in (([0, 4], 3, 2), ([0, 4], 0, 1), ([0, 4], 4, 0), ([4, 3], 1, 1), ([0, 4], 65536, 1)):
            refused(g, lib.h3_hip_sequences_new(g.handle, u32(ends), None, 1, heads, kv), "sequences")
        refused(g, lib.h3_hip_sequences_new(g.handle, u32([0, 4]), u32([5, 4]), 1, 1, 1), "fall")
        refused(g, lib.h3_hip_sequences_new(g.handle, u32([0]), None, 0, 1, 1), "sequences")
        refused(g, lib.h3_hip_sequences_new(g.handle, u32([0, 2 ** 32 - 1]), None, 1, 1, 1), "longer")
        f = (C.c_double * 2)(1.0, 0.5)
        for args in ((f, u32([0, 1]), 0, 2, 0), (f, u32([0, 1]), 129, 2, 0), (f, u32([0, 1]), 2, 0, 0), (f, u32([0, 1]), 2, 17, 0),
                     (f, u32([0, 1]), 2, 2, 2), (None, u32([0, 1]), 2, 2, 0), (f, None, 2, 2, 0), (f, u32([0, 2]), 2, 2, 0),
                     ((C.c_double * 2)(1.0, math.inf), u32([0, 1]), 2, 2, 0), ((C.c_double * 2)(math.nan, 1.0), u32([0, 1]), 2, 2, 0)):
            refused(g, lib.h3_hip_rope_axes_new(g.handle, *args), "RoPE axes")
        for ranks, k, n in (([], 8, 8), ([0], 8, 8), ([257], 8, 8), ([4], 0, 8), ([4], 8, 0), ([4], 2 ** 24 + 1, 8)):
            refused(g, lib.h3_hip_adapters_new(g.handle, u32(ranks), len(ranks), k, n), "adapters")
        for at, count, rank in (([], 1, 8), ([0], 0, 8), ([0], 1, 0), ([0], 1, 257)):
            refused(g, lib.h3_hip_adapter_rows_new(g.handle, u32(at), len(at), count, rank), "adapter rows")

        q, small, f32, foreign = g.empty(8 * 256), g.empty(100), g.empty(8 * 256, F32_TENSOR), other.empty(8 * 256)
        k, v, out, qkv = g.empty(8 * 256), g.empty(8 * 256), g.empty(8 * 256), g.empty(8 * 3 * 256)
        plan = lib.h3_hip_sequences_new(g.handle, u32([0, 3, 8]), None, 2, 2, 2)
        theirs = lib.h3_hip_sequences_new(other.handle, u32([0, 3, 8]), None, 2, 2, 2)

        def attend(o=out, a=q, b=k, c=v, p=plan, scale=1.0):
            return lib.h3_hip_sdpa_sequences_bf16(g.handle, *(t.handle if t else None for t in (o, a, b, c)), p, C.c_float(scale))

        refused(g, attend(), "no active")
        g.begin()
        for bad, text in ((dict(p=None), "plan"), (dict(p=theirs), "context"), (dict(scale=0.0), "scale"), (dict(scale=math.nan), "scale"),
                          (dict(o=q), "disjoint"), (dict(o=k), "disjoint"), (dict(o=None), "disjoint"), (dict(a=small), "need"),
                          (dict(b=small), "need"), (dict(c=f32), "dtype"), (dict(o=foreign), "another context"), (dict(a=None), "missing")):
            refused(g, attend(**bad), text)

        rope = lib.h3_hip_rope_axes_new(g.handle, f, u32([0, 1]), 2, 2, 0)
        pos, w = g.empty(16, F32_TENSOR), g.empty(128)

        def turn(o=(q, k, v), x=qkv, qw=w, kw=w, r=rope, p=pos, rows=8, heads=2, kv=2, dim=128, grouped=0, eps=EPS):
            return lib.h3_hip_qkv_rope_axes_bf16(g.handle, *(t.handle for t in o), x.handle, qw and qw.handle, kw and kw.handle, r,
                                                 p.handle, rows, heads, kv, dim, grouped, C.c_float(eps))

        for bad, text in ((dict(r=None), "axes"), (dict(rows=0), "rows"), (dict(heads=3), "heads"), (dict(kv=0), "heads"),
                          (dict(dim=257), "dim"), (dict(dim=3), "pairs"), (dict(qw=None), "norm"), (dict(grouped=2), "grouped"),
                          (dict(eps=-1.0), "eps"), (dict(eps=math.nan), "eps"), (dict(o=(q, q, v)), "disjoint"),
                          (dict(o=(qkv, k, v)), "disjoint"), (dict(p=f32, x=small), "need"), (dict(p=w), "dtype"), (dict(rows=9), "need"),
                          (dict(qw=small, kw=small), "need")):
            refused(g, turn(**bad), text)

        ad = lib.h3_hip_adapters_new(g.handle, u32([4, 40]), 2, 16, 32)
        rows = lib.h3_hip_adapter_rows_new(g.handle, u32([0, 1, 2]), 3, 2, 40)
        low = lib.h3_hip_adapter_rows_new(g.handle, u32([0, 1, 2]), 3, 2, 8)
        x, base = g.empty(48), g.empty(96)
        for index, a, b, scale, text in ((2, q, q, 1.0, "index"), (0, q, q, math.inf, "finite"), (1, small, q, 1.0, "need"),
                                         (0, q, f32, 1.0, "dtype")):
            refused(g, lib.h3_hip_adapters_set(g.handle, ad, index, a.handle, b.handle, C.c_float(scale)), text)

        def adapt(o=out, b=base, i=x, a=ad, p=rows, m=3, k=16, n=32):
            return lib.h3_hip_adapters_add_bf16(g.handle, o.handle, b.handle, i.handle, a, p, m, k, n)

        for bad, text in ((dict(a=None), "missing"), (dict(p=None), "missing"), (dict(m=4), "need"), (dict(k=8), "need"),
                          (dict(n=33), "need"), (dict(p=low), "rank"), (dict(o=x), "need"), (dict(i=small, o=small), "aliases"),
                          (dict(b=f32), "dtype"), (dict(i=foreign), "another context")):
            refused(g, adapt(**bad), text)
        refused(g, lib.h3_hip_linear_adapters_bf16(g.handle, out.handle, x.handle, None, None, ad, rows, 3, 16, 32), "weight")
        g.submit()
        lib.h3_hip_sequences_free(plan)
        lib.h3_hip_sequences_free(theirs)
        lib.h3_hip_rope_axes_free(rope)
        lib.h3_hip_adapters_free(ad)
        lib.h3_hip_adapter_rows_free(rows)
        lib.h3_hip_adapter_rows_free(low)
