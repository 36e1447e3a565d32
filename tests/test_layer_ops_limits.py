"""Which lengths need a workspace (the chunked kernels), without a GPU."""
import pytest

import _lib


def limit(n_seqs, heads, dk, dv):
    """The longest sequence that the token recurrence takes."""
    f = _lib.lib().qfn_deltanet_chunk_workspace
    return next(t for t in range(1, 200) if f(t, n_seqs, heads, heads, dk, dv) > 0) - 1


@pytest.mark.parametrize("dk", [64, 128])
@pytest.mark.parametrize("dv", [32, 64, 96, 128, 256, 4096])
@pytest.mark.parametrize("heads", [1, 8, 32])
def test_more_sequences_never_lower_the_limit(heads, dk, dv):
    limits = [limit(n, heads, dk, dv) for n in (1, 2, 7, 64, 1000)]
    assert limits == sorted(limits) and 10 <= limits[0] and limits[-1] <= 24


def test_limits_of_measured_sizes():
    assert limit(1, 32, 128, 128) == 10 and limit(16, 32, 128, 128) == 12 and limit(64, 32, 128, 128) == 12
    assert limit(16, 32, 128, 64) == 16 and limit(16, 32, 64, 128) == 16 and limit(64, 16, 64, 64) == 24


def test_sizes_that_need_none():
    f = _lib.lib().qfn_deltanet_chunk_workspace
    assert f(100000, 1, 8, 8, 256, 128) == 0   # dk = 256: the token recurrence
    assert f(100, 0, 8, 8, 128, 128) == f(-1, 1, 8, 8, 128, 128) == f(100, 1, 0, 8, 128, 128) == f(100, 1, 8, 0, 128, 128) == 0
    assert f(100, 1, 8, 8, 0, 128) == f(100, 1, 8, 8, 128, 0) == 0
