"""Plans of a step that serves several requests at once: what needs no GPU."""
import ctypes as C

import pytest

from h3cli_amd import _lib


def u32(values):
    return (C.c_uint32 * len(values))(*values)


def layout(q, k, heads, kv_heads, count=None):
    size = C.c_size_t()
    ok = _lib.load().h3_hip_sequences_layout(q and u32(q), k and u32(k), len(q) - 1 if count is None else count, heads, kv_heads,
                                             C.byref(size))
    return size.value if ok else None


@pytest.mark.parametrize("q,k,heads,kv_heads,count", [
    ([0, 4], None, 3, 2, None), ([0, 4], None, 0, 1, None), ([0, 4], None, 4, 0, None), ([4, 3], None, 1, 1, None),
    ([0, 4], [5, 4], 1, 1, None), ([0, 4, 3], None, 1, 1, None), ([0, 4], None, 65536, 1, None), ([0], None, 1, 1, 0),
    (None, [0, 1], 1, 1, 1), ([0, 2 ** 31], None, 1, 1, None), ([0, 2 ** 30], None, 2, 1, None), ([0, 1], [0, 2 ** 31], 1, 1, None),
    ([0, 2 ** 31 - 1], [0, 1], 1, 1, None), ([0, 2 ** 25], [0, 0], 60000, 60000, None), ([0, 2 ** 31 - 1], [0, 2 ** 31 - 1], 1, 1, None),
])
def test_refused_sequences(q, k, heads, kv_heads, count):
    assert layout(q, k, heads, kv_heads, count) is None


def test_sequences_hold_what_their_kernels_need():
    assert 0 < layout([0, 1], None, 1, 1) < 1000
    assert layout([0, 0, 0], None, 1, 1) > 0                     # no rows at all
    assert layout([5, 5, 9], [7, 20, 20], 4, 2) > 0
    # Transposed values of 4133 keys in whole tiles of 64, and retry bytes.
    assert layout([0, 4133], None, 12, 12) > 65 * 64 * 12 * 256
    # One row over many keys: parts of 32 rows, and no transposed values.
    assert 2 * 130 * 128 < layout([0, 1], [0, 18225], 5, 1) < 128 * 32 * 130 * 4 + 4096
    # A K of 4 GiB and more, in which a tile's offsets would not fit 32 bits, goes without them too.
    assert layout([0, 300], [0, 2 ** 24], 1, 1) < 1 << 25
    assert layout([0, 10 ** 5], [0, 2 ** 24 - 1], 1, 1) < 1 << 25     # its transposed V, in whole tiles, would have 4 GiB
    assert layout([0, 10 ** 5], [0, 2 ** 24 - 64], 1, 1) > 1 << 31


@pytest.mark.parametrize("queries,keys", [(9000, 256), (9000, 100), (9000, 0), (8000, 256)])
@pytest.mark.parametrize("first", [True, False])
def test_a_sequence_of_few_keys_leaves_the_others_their_tiles(queries, keys, first):
    """Transposed values of 8193 rows of self-attention, whether fewer or more queries over few keys stand beside them."""
    lengths = [(queries, keys), (8193, 8193)][::1 if first else -1]
    ends = [[0, lengths[0][i], lengths[0][i] + lengths[1][i]] for i in range(2)]
    assert layout(ends[0], ends[1], 40, 40) > 129 * 64 * 40 * 256


def test_no_context():
    lib = _lib.load()
    assert not lib.h3_hip_sequences_new(None, u32([0, 1]), None, 1, 1, 1)
    assert not lib.h3_hip_sdpa_sequences_bf16(None, None, None, None, None, None, C.c_float(1))
    assert not lib.h3_hip_rope_axes_new(None, None, None, 1, 1, 0)
    assert not lib.h3_hip_qkv_rope_axes_bf16(None, None, None, None, None, None, None, None, None, 1, 1, 1, 1, 0, C.c_float(0))
    assert not lib.h3_hip_adapters_new(None, u32([1]), 1, 1, 1)
    assert not lib.h3_hip_adapters_set(None, None, 0, None, None, C.c_float(1))
    assert not lib.h3_hip_adapter_rows_new(None, u32([0]), 1, 1, 1)
    assert not lib.h3_hip_adapters_add_bf16(None, None, None, None, None, None, 1, 1, 1)
    assert not lib.h3_hip_linear_adapters_bf16(None, None, None, None, None, None, None, 1, 1, 1)
    for free in (lib.h3_hip_sequences_free, lib.h3_hip_rope_axes_free, lib.h3_hip_adapters_free, lib.h3_hip_adapter_rows_free):
        free(None)
