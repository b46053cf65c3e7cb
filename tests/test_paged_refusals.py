"""Calls of the paged caches that would give wrong results, or have no effect, and are refused on the host, before anything is
launched: the addresses here are never read."""
import ctypes

import pytest

from vsa_lm_b200 import Bolt3Decoder, _lib
from vsa_lm_b200.model import Bolt3LM
from vsa_lm_b200.workloads import MODEL_SHAPES

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


def _attend(**over):
    """2 sequences of 8 tokens, 4 query heads of 64 on one KV head: queries of a wider projection of 384 values a token."""
    a = dict(B=2, T=8, H=4, HKV=1, HD=64, q=A, q_sb=8 * 384, q_st=384, pages=2 * A, n_pages=64, page=16, table=3 * A, table_stride=8,
             width=8, weight=4 * A, n=20, lens=None, y=5 * A, sm_scale=0.125, workspace=6 * A, workspace_bytes=A, status=None)
    a.update(over)
    return _lib.load().bolt3_paged_attend(ctypes.byref(_lib.PagedAttendArgs(**a)), None)


@pytest.mark.parametrize("at", [0, 16, -16, 2 * 8 * 4 * 64 * 2 - 16, -(2 * 8 * 4 * 64 * 2 - 16), (15 * 384 + 256) * 2 - 16])
def test_records_of_many_rows_need_their_queries_whole(at):
    assert _attend(y=A + at) == ERR_ARG


@pytest.mark.parametrize("weight", [None, 4 * A])
@pytest.mark.parametrize("T", [1, 4, 8, 200])
@pytest.mark.parametrize("at,stride", [(0, 384), (256, 384), (16, 256), (-16, 256), (512, 256), (-512, 256), (0, 0), (0, -256)])
def test_outputs_are_not_written_over_queries_of_other_rows(T, weight, at, stride):
    """Over queries that are not laid out like the outputs, or over some of them."""
    sb = max(abs(stride) * T, 384)                        # of one token the token's stride says nothing
    assert _attend(T=T, n=0, width=16, weight=weight, q=A, q_sb=sb if stride != 0 else 0, q_st=stride, y=A + at) == ERR_ARG


@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("page", [48, 32, 0])
def test_a_page_size_goes_with_paged_caches(kind, page):
    model = Bolt3LM(**dict(MODEL_SHAPES["tiny_lm"]))
    for call in (lambda **kw: Bolt3Decoder(model, **kw), lambda **kw: Bolt3Decoder.blank_state(model, 1, "cpu", **kw),
                 lambda **kw: Bolt3Decoder.state_bytes(model, **kw)):
        with pytest.raises(ValueError, match="page size"):
            call(kv_cache=kind, kv_page=page)
    Bolt3Decoder(model, kv_cache=kind, kv_page=64)
