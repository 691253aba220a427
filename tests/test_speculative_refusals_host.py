"""What the speculative-decoding entry points accept and refuse at the edge, before they touch CUDA."""
from __future__ import annotations

import pytest

from llama1b_megakernel_b200 import _lib
from tests import test_speculative_host as base
from tests.test_speculative_host import lib  # noqa: F401  (a fixture)


@pytest.mark.parametrize("off", [4, 8, 12])
def test_scales_on_four_bytes(lib, off):  # noqa: F811
    """A layer's slice of a pool of scale bytes starts where it starts."""
    layer = base._layer(k_scales=base.PTR + off, v_scales=base.PTR + 4)
    assert base._write(lib, layer, rows=0) == _lib.MK_OK
    assert base._read(lib, layer, max_len=0) == _lib.MK_OK
    assert base._attend(lib, layer, rows=0) == _lib.MK_OK
    for bad in (dict(k_scales=base.PTR + off + 2), dict(v_scales=base.PTR + off + 1)):
        assert base._attend(lib, base._layer(**bad)) == _lib.MK_EINVAL
        assert "aligned" in lib.mk_last_error().decode()


def test_arrays_of_nothing_may_be_null(lib):  # noqa: F811
    """Empty tensors have no address; sizes are still looked at."""
    layer = base._layer()
    assert base._write(lib, layer, rows=0, qkv=None, slots=None, q_out=None) == _lib.MK_OK
    assert base._read(lib, layer, max_len=0, k=None, v=None) == _lib.MK_OK
    assert base._attend(lib, layer, rows=0, q=None, mask=None, out=None) == _lib.MK_OK
    assert base._logprobs(lib, rows=0, logits=None, targets=None, lp=None, ent=None, ids=None, tlp=None) == _lib.MK_OK
    assert base._write(lib, layer, rows=0, nq=0) == _lib.MK_EINVAL
    assert base._read(lib, layer, max_len=-1, k=None) == _lib.MK_EINVAL
    assert base._attend(lib, layer, rows=0, max_nodes=257) == _lib.MK_EINVAL
    assert base._logprobs(lib, rows=0, top=33) == _lib.MK_EINVAL


@pytest.mark.parametrize("max_len", [(1 << 30) + 1, (1 << 31) - 128, (1 << 31) - 8])
def test_lengths_beyond_the_kernels_indexes(lib, max_len):  # noqa: F811
    """Positions are ints that a range's or block's end is added to: 2^30 is the limit, and
    what is above it is refused by name."""
    layer = base._layer(page_size=8, max_blocks=(1 << 28) - 1)
    for rows in (0, 6):
        assert base._attend(lib, layer, max_len=max_len, rows=rows) == _lib.MK_EINVAL
        assert "max_len" in lib.mk_last_error().decode()
    assert base._attend(lib, layer, max_len=1 << 30, rows=0) == _lib.MK_OK


@pytest.mark.parametrize("args", [(1, 8, 2, 257, 17000), (1, 8, 2, 1 << 30, 17000), (1, 8, 2, 3, (1 << 31) - 8),
                                  (70000, 8, 2, 3, 17000), (1, 1 << 30, 1, 2, 17000)])
def test_workspace_of_what_is_refused_is_nothing(lib, args):  # noqa: F811
    assert lib.mk_tree_attention_workspace(*args) == 0
