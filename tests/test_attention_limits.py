"""Launches of the attention entry points that would pass the device's limits: a status, no launch."""
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
