"""The DiT step with projections in FP8 blocks (projection_quant 3): every stage of a block
against its definition in 64 bits on what the stage before gave, streamed weights, and a
checkpoint. Bounds as in test_fp8_block_gpu.py; cos > 0.99 beside W8A16 projections as for
tensorwide FP8 (an E4M3 value is 2.7% off in the root mean square, a product of two 3.7%,
which moves the cosine of a projection's result by 0.0007)."""
import numpy as np
import pytest

from h3cli_amd.runtime import DitSynth, H3Error
from tests.helpers import bf16
from tests.test_fp8_block_gpu import HALF_BF16, MFMA, blocks, mlp_reference, quantized, within
from tests.test_h3_load_gpu import SMALL, checkpoint

pytestmark = pytest.mark.gpu
NAMES = ("attn.qkv_proj.weight", "attn.out_proj.weight", "mlp.fc1.weight", "mlp.fc2.weight")


def config(swiglu, **more):
    return dict(dict(blocks=2, hidden=512, heads=3, mlp=768, frames=3, height=7, width=13, latent=256, seed=5,
                     streamed_first=2, swiglu=swiglu, projection_quant=3), **more)


def shapes(c):
    inner = c["heads"] * 128
    return {"attn.qkv_proj.weight": (3 * inner, c["hidden"]), "attn.out_proj.weight": (c["hidden"], inner),
            "mlp.fc1.weight": ((2 if c["swiglu"] else 1) * c["mlp"], c["hidden"]), "mlp.fc2.weight": (c["hidden"], c["mlp"])}


def weight_values(m, block, name, n, k):
    """The BF16 values that a resident weight's blocks stand for."""
    g = m.gpu
    h = m.lib.h3_hip_dit_synth_tensor(m.handle, f"blocks.{block}.{name}".encode())
    out = g.empty(n * k)
    g.begin()
    g.check(g.lib.h3_hip_fp8_block_unpack(g.handle, out.handle, h, n, k), "unpack")
    g.submit()
    return bf16(out.read()).reshape(n, k).astype(np.float64)


@pytest.mark.parametrize("swiglu", [1, 0])
def test_stages(swiglu):
    c = config(swiglu, trace_block=1)
    H, F = c["hidden"], c["mlp"]
    with DitSynth(geometry="h3", **c) as m:
        m.step(step=0, dt=-0.1)
        R = m.rows
        w = [weight_values(m, 0, name, *shapes(c)[name]) for name in NAMES]

        def stage(name, width):
            return bf16(m.read("trace." + name)).reshape(R, width).astype(np.float64)

        mod = bf16(m.read("blocks.0.modulation")).reshape(2, 6, H).astype(np.float64)[0]
        assert not m.read("row_map").any()
        eps = float(np.float32(m.config.eps))

        def norm(x, name, shift, scale):
            y = x / np.sqrt((x * x).mean(axis=1, keepdims=True) + eps) * bf16(m.read("blocks.0." + name)).astype(np.float64)
            error = 2.0 ** -19 * np.abs(y) * np.abs(1 + mod[scale]) + 2.0 ** -22 * (np.abs(y) + np.abs(mod[shift]))
            y = y * (1 + mod[scale]) + mod[shift]
            # A block's scale is less than its largest magnitude / 224.
            top = np.repeat(blocks(np.abs(y), 1).max(axis=(1, 3)), 128, axis=1)[:, :H]
            return y, np.maximum(2.0 ** -4 * np.abs(y), 2.0 ** -10 * top / 224) * (1 + 2.0 ** -20) + error

        def product(x, w):
            want = x @ w.T
            return want, HALF_BF16 * np.abs(want) + 2 * MFMA * (np.abs(x) @ np.abs(w).T)

        def gate(x, branch, slot):
            want = x + branch * mod[slot]
            return want, (HALF_BF16 + 2.0 ** -23) * np.abs(want)

        x0, xn1, o, x1, xn2, f = (stage(name, H) for name in ("x0", "xn1", "o", "x1", "xn2", "f"))
        within(xn1, *norm(x0, "norm1.weight", 0, 1), "xn1")
        within(stage("qkv", w[0].shape[0]), *product(xn1, w[0]), "qkv")
        within(o, *product(quantized(stage("attn", w[1].shape[1]), 1)[0], w[1]), "o")
        within(x1, *gate(x0, o, 2), "x1")
        within(xn2, *norm(x1, "norm2.weight", 3, 4), "xn2")
        within(stage("h", w[2].shape[0]), *product(xn2, w[2]), "h")
        if swiglu:
            within(f, *mlp_reference(xn2, w[2], w[3], F), "f")
        else:
            within(f, *product(quantized(stage("act", F), 1)[0], w[3]), "f")
        within(stage("x2", H), *gate(x1, f, 5), "x2")


def test_streamed_as_resident():
    """Blocks from pinned memory through the two slots give what resident ones give, step by step."""
    runs = []
    for streamed in (3, 0, 1):
        with DitSynth(geometry="h3", **config(1, blocks=3, streamed_first=streamed)) as m:
            for step in range(2):
                m.step(step=step, dt=-0.1)
            runs.append((m.read("latent"), m.read("hidden")))
    assert np.all(np.isfinite(runs[0][0]))
    for latent, hidden in runs[1:]:
        assert np.array_equal(latent, runs[0][0]) and np.array_equal(hidden, runs[0][1])


def test_load(tmp_path):
    path = tmp_path / "h3.safetensors"
    ref = checkpoint(path)
    c = dict(SMALL, swiglu=1)
    with DitSynth(geometry="h3", projection_quant=3, **SMALL) as m:
        m.load(path)
        for b in range(c["blocks"]):
            for name, (n, k) in shapes(c).items():
                want, _ = quantized(bf16(ref[f"blocks.{b}.{name}"]).reshape(n, k).astype(np.float64), 128)
                assert np.array_equal(weight_values(m, b, name, n, k), want), name
        m.step(step=0, dt=-0.1)
        blocked = bf16(m.read("hidden")).astype(np.float64)
    with DitSynth(geometry="h3", **SMALL) as m:
        m.load(path)
        m.step(step=0, dt=-0.1)
        q8 = bf16(m.read("hidden")).astype(np.float64)
    cos = blocked @ q8 / np.sqrt((blocked @ blocked) * (q8 @ q8))
    assert cos > 0.99, cos


def test_refusals():
    with pytest.raises(H3Error, match="projection_quant"):
        DitSynth(geometry="h3", **config(1, projection_quant=4))
