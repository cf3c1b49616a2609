"""The layout of block-scaled FP8 matrices, and calls without a context, on the CPU."""
import ctypes as C

import pytest

from h3cli_amd import _lib

def layout(*args):
    v = [C.c_size_t() for _ in range(4)]
    return tuple(x.value for x in v) if _lib.load().h3_hip_fp8_block_layout(*args, *v) else None


@pytest.mark.parametrize("rows,columns,tile", [(1, 1, 1), (1, 128, 1), (7, 129, 1), (128, 5376, 128), (129, 1000, 128),
                                               (100000, 14336, 1), (1 << 20, 8192, 1), (3, (1 << 24) - 128, 128)])
def test_layout(rows, columns, tile):
    stride, scales, groups, size = layout(rows, columns, tile)
    blocks = -(-columns // 128)
    assert stride == 128 * blocks
    assert scales % 256 == 0 and rows * stride <= scales < rows * stride + 256
    assert groups == -(-blocks // 4)
    assert size == scales + -(--(-rows // tile) // 32) * groups * 128


def test_layout_refuses():
    for args in ((0, 1, 1), (1, 0, 1), (1, 1, 0), (1, 1, 64), (1, (1 << 24) - 127, 1)):
        assert layout(*args) is None, args
    assert _lib.load().h3_hip_fp8_block_layout(1, 1, 1, None, None, None, None) == 1


def test_without_a_context():
    lib = _lib.load()
    assert not lib.h3_hip_fp8_block_new(None, 1, 1, 1)
    assert not lib.h3_hip_fp8_block_from_packed(None, None, None, 1, 1, 1)
    assert not lib.h3_hip_fp8_block_weight_from_bf16(None, None, 1, 1)
    assert not lib.h3_hip_fp8_block_pack(None, None, None, 1, 1)
    assert not lib.h3_hip_fp8_block_unpack(None, None, None, 1, 1)
    assert not lib.h3_hip_linear_fp8_block(None, None, None, None, None, 1, 1, 1)
    assert not lib.h3_hip_mlp_fp8_block(None, None, None, None, None, 1, 1, 1, 1)
    assert not lib.h3_hip_swiglu_fp8_block(None, None, None, 1, 1)
    assert not lib.h3_hip_adaln_fp8_block(None, None, None, None, None, None, 1, 1, 1, 0, 0, 0.0)
    assert not lib.h3_hip_gate_adaln_fp8_block(None, None, None, None, None, None, None, None, None, 1, 1, 1, 0, 0, 0, 0.0)
    assert not lib.h3_hip_add_rms_norm_fp8_block(None, None, None, None, None, None, 1, 1, 0.0)
