"""Launches of the attention entry points that would pass the device's limits: a status, no launch."""
import pytest
import torch

from conftest import pkg

EINVAL, ELIMIT = -1, -2


def test_selection_of_more_queries_than_a_launch_holds():
    """64 queries of a key head a wave, four waves a workgroup of 256 threads: at most 2^24 - 1 workgroups."""
    L = pkg("_lib")

    def status(b):
        q = L.Heads(1 << 20, 0, 0, 0, 64)
        return L.lib().tpu3_block_select(None, 0, b, 16, 64, 8, q, 64, 1 << 20, None, None, 0, 1, 1 << 20, None, 0)
    assert status(1 << 20) == ELIMIT
    assert status((1 << 20) - 1) == EINVAL                  # (within it: the missing workspace is what is wrong)


def test_sizes_beyond_31_bits():
    """Rows of the last tile of 64 queries, and the places of a block's means, are counted in 31 bits."""
    L = pkg("_lib")
    q = L.Heads(1 << 20, 0, 0, 0, 1)

    def select(m):
        return L.lib().tpu3_block_select(None, 0, 1, m, 64, 8, q, 1, 1 << 20, None, None, 0, 1, 1 << 20, None, 0)
    assert select(2**31 - 1) == ELIMIT and select(2**31 - 63) == ELIMIT
    assert select(2**31 - 64) == EINVAL                     # (the missing workspace)

    def means(heads, d, out=None):
        return L.lib().tpu3_block_means(None, 0, 1, 64, d, L.Heads(1 << 20, 0, 0, 0, heads), None, -1, out)
    assert means(1 << 28, 8) == ELIMIT and means(1 << 24, 128) == ELIMIT
    assert means((1 << 28) - 1, 8) == EINVAL                # (the missing result)


def test_dimensions_beyond_31_bits():
    """A dimension that does not fit the C functions' int is refused, not cut off (before anything else is looked at)."""
    ops = pkg("network.operations")
    one = torch.zeros((1, 1, 1, 8))
    pos, freq = torch.zeros((1, 1)), ops.rotation_frequencies(1, 4)
    for shape in ((2**32 + 1, 1, 1, 8), (1, 2**31, 1, 8), (1, 1, 2**33, 8)):
        x = one.expand(shape)
        blocks = torch.zeros((1, 1, 1, 1), dtype=torch.int32)
        for call in (lambda: ops.norm_rotate(x, None, None, None, pos, freq),
                     lambda: ops.block_means(x), lambda: ops.select_blocks(x, one, 64, 1),
                     lambda: ops.block_attention(x, one, one, blocks), lambda: ops.sparse_attention(x, one, one, 1)):
            with pytest.raises(RuntimeError, match="2\\^31"):
                call()
