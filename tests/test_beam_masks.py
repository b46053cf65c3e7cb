"""Beam search's selection over logits that are masked with the type's lowest value, with large negative numbers,
or lie at the ends of fp32's range; and selections of different sizes at once.

The reference takes log_softmax as (x - max) - log(sum e^(x - max)) in 64 bits. Tolerance of a score: three fp32
roundings of terms no larger than |s| + |x - max| + |log sum| (2^-22 of that), and 2e-6 for the logarithm of the sum.
"""
import ctypes
import math
import threading

import pytest
import torch

from vsa_lm_b200 import _lib
from vsa_lm_b200 import kernels as K


def plain(logits, scores):
    """(score, parent, token) of the K best continuations by slot, from [B, K, V] logits, in 64 bits."""
    B, Kb, V = logits.shape
    x = logits.double()
    d = x - x.amax(-1, keepdim=True)
    ls = torch.log(torch.exp(d).sum(-1, keepdim=True))
    cand = (scores.double()[..., None] + (d - ls)).view(B, -1)
    size = (scores.double()[..., None].abs() + d.abs() + ls.abs()).view(B, -1)
    size = torch.where(size.isfinite(), size, 0.0)
    best, at = torch.sort(cand, dim=1, descending=True, stable=True)
    out = torch.full((B, Kb), -math.inf, dtype=torch.float64), torch.arange(Kb).repeat(B, 1), torch.zeros(B, Kb).long()
    tol = torch.zeros(B, Kb, dtype=torch.float64)
    for b in range(B):
        free, later = list(range(Kb)), []
        chosen = [i for i in range(Kb) if best[b, i] > -math.inf]
        for i in chosen:
            p = int(at[b, i]) // V
            later.append(i) if p not in free else (free.remove(p), put(out, tol, b, p, best, at, size, i, V))
        for i in later:
            put(out, tol, b, free.pop(0), best, at, size, i, V)
    return out, 2e-6 + 2 ** -22 * tol


def put(out, tol, b, slot, best, at, size, i, V):
    c = int(at[b, i])
    out[0][b, slot], out[1][b, slot], out[2][b, slot], tol[b, slot] = best[b, i], c // V, c % V, size[b, c]


def check(logits, scores):
    got = [t.cpu() for t in K.beam_select(logits.cuda(), scores.cuda())]
    ref, tol = plain(logits, scores)
    live = ref[0] > -math.inf
    assert torch.equal(got[0] > -math.inf, live)
    assert torch.equal(got[1].long()[live], ref[1][live]) and torch.equal(got[2][live], ref[2][live])
    assert bool(((got[0].double() - ref[0]).abs()[live] <= tol[live]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [100, 8192, 34000])
@pytest.mark.parametrize("mask", ["lowest", -1e9, -1e10, -3e38, -1e30, -70000.0])
def test_masked_vocabulary(dtype, V, mask):
    """A few allowed tokens: whole threads, and whole chunks, hold nothing but the mask."""
    g = torch.Generator().manual_seed(5)
    B, Kb = 3, 4
    x = torch.full((B, Kb, V), torch.finfo(dtype).min if mask == "lowest" else mask, dtype=dtype)
    for b in range(B):
        for k in range(Kb):
            at = torch.randperm(V, generator=g)[:6]
            x[b, k, at] = torch.arange(6, dtype=dtype) + 7 * b + k / 8
    check(x, -3 * torch.rand(B, Kb, generator=g))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [100, 20000])
@pytest.mark.parametrize("at", ["lowest", "highest", -1e9, -1e10, 1e9, 1e10, 4e4, -4e4, 2.0 ** 30, -2.0 ** 30])
def test_beam_of_equal_logits_of_any_size(dtype, V, at):
    """Equal logits, whatever they are, are a uniform distribution: such a beam scores its own score less log V."""
    big = torch.finfo(dtype)
    x = torch.full((2, 2, V), {"lowest": big.min, "highest": big.max}.get(at, at), dtype=dtype)
    x[:, 1] = torch.linspace(-4, 4, V).to(dtype)
    x[1, 1] = x[1, 0]
    x[0, 1, V // 2] = 24.0                           # that beam's own first token has nearly all of its probability
    check(x, torch.tensor([[0.0, -1.0], [-2.0, -0.5]]))


@pytest.mark.gpu
def test_neighbours_at_large_magnitudes():
    """Logits a few units in the last place apart, from 2^17 to 2^30: the gaps count."""
    B, Kb, V = 14, 2, 3000
    g = torch.Generator().manual_seed(6)
    x = torch.empty(B, Kb, V)
    for b in range(B):
        base = 2.0 ** (17 + b) * (1 if b % 2 else -1)
        step = 2.0 ** (17 + b - 23)
        x[b] = base - step * torch.randint(1, 40, (Kb, V), generator=g).float()
        x[b, :, 17 + b], x[b, :, 40 + b], x[b, :, 90 + b] = base, base - step, base
    check(x, torch.tensor([[0.0, -0.37]]).repeat(B, 1))


@pytest.mark.gpu
def test_selections_of_different_sizes_from_many_threads():
    """Calls whose second kernel takes 43 or 133 KB of shared memory, from eight host threads that do nothing else."""
    lib = _lib.load()
    failed = []

    def work(i):
        try:
            select_often(i, 524288 if i % 2 else 170000)
        except Exception as e:
            failed.append(repr(e))

    def select_often(i, V):
        with torch.cuda.stream(torch.cuda.Stream()):
            x = torch.randn(16, V, generator=torch.Generator().manual_seed(i)).cuda()
            s = torch.linspace(0, -5, 16, device="cuda").view(1, 16)
            first = K.beam_select(x, s)
            out = tuple(torch.empty_like(t) for t in first)
            nbytes = lib.bolt3_beam_select_workspace(1, 16, V)
            ws = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
            a = _lib.BeamSelectArgs(B=1, K=16, V=V, logits=x.data_ptr(), row_stride=V, logits_fp32=1, scores=s.data_ptr(),
                                    out_scores=out[0].data_ptr(), out_parent=out[1].data_ptr(), out_token=out[2].data_ptr(),
                                    out_finished=out[3].data_ptr(), workspace=ws.data_ptr(), workspace_bytes=nbytes)
            at, stream = ctypes.byref(a), torch.cuda.current_stream().cuda_stream
            rc = [lib.bolt3_beam_select(at, stream) for _ in range(3000)]
            torch.cuda.current_stream().synchronize()
            if any(rc) or not all(torch.equal(p, q) for p, q in zip(first, out)):
                failed.append((V, sum(map(bool, rc))))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(8)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
