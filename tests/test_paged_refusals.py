"""Calls of the paged entry points that would give wrong results and are refused on the host, before anything is launched: the
addresses here are never read."""
import ctypes

import pytest

from vsa_lm_b200 import _lib

ERR_ARG = 1
A = 1 << 20                                               # addresses 1 MB apart


def _evict(**over):
    a = dict(B=4, HKV=2, HD=64, pages=A, n_pages=64, page=16, table=2 * A, table_stride=8, width=8, weight=3 * A, order=4 * A,
             n=100, keep=50, recent=10, lens=5 * A, lens_out=6 * A, workspace=None, workspace_bytes=0, status=None)
    a.update(over)
    return _lib.load().bolt3_paged_evict(ctypes.byref(_lib.PagedEvictArgs(**a)), None)


@pytest.mark.parametrize("at", [0, 4, 12, -4, -12])
def test_an_eviction_does_not_overwrite_its_own_lengths(at):
    assert _evict(lens_out=5 * A + at) == ERR_ARG
