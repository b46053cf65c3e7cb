"""Beam search's selection and the reordering of states (bolt3_beam_select, bolt3_beam_reorder) against
plain implementations: 64-bit scores on the CPU, index moves.

Tolerance of a score: cum + (x - lse) in fp32 is three roundings of terms no larger than their sum of
magnitudes (2^-22 of it), the log-sum-exp's own error is below 2e-6 (a sum of exponentials in fp32 in
a tree, each term good to a few 2^-24). Whole outputs are equal; the inputs are checked to have no two
different scores within 1e-4 at the places that decide.
"""
import ctypes
import math

import pytest
import torch

from vsa_lm_b200 import _lib
from vsa_lm_b200 import kernels as K


def ref_select(logits, scores, finished, eos, check_gap=True):
    """logits [B, K, V]; the definition of include/bolt3.h in 64 bits."""
    B, Kb, V = logits.shape
    pad = eos[0] if eos else 0
    out = (torch.full((B, Kb), -math.inf, dtype=torch.float64), torch.arange(Kb, dtype=torch.int32).repeat(B, 1),
           torch.full((B, Kb), pad), torch.ones(B, Kb, dtype=torch.bool))
    size = torch.zeros(B, Kb, dtype=torch.float64)
    for b in range(B):
        cands = []
        for k in range(Kb):
            s = float(scores[b, k])
            if not s > -math.inf:
                continue
            if finished is not None and finished[b, k]:
                cands.append((s, k, 0, pad, abs(s)))
                continue
            x = logits[b, k].double()
            x = torch.where(x.isnan(), -math.inf, x)
            lse = torch.logsumexp(x, 0)
            top, at = torch.sort(x, descending=True, stable=True)
            for i in range(min(Kb, V)):
                if top[i] > -math.inf:
                    mag = abs(s) + abs(float(top[i])) + abs(float(lse))
                    cands.append((s + float(top[i] - lse), k, i, int(at[i]), mag))
        cands = [c for c in cands if c[0] > -math.inf]
        cands.sort(key=lambda c: (-c[0], c[1], c[2]))
        if check_gap:
            v = [c[0] for c in cands[:Kb + 1]]
            assert all(a == b2 or a - b2 > 1e-4 for a, b2 in zip(v, v[1:])), "the test's own scores are too close"
        free, later = list(range(Kb)), []
        place = {}
        for c in cands[:Kb]:
            if c[1] in free:
                free.remove(c[1])
                place[c[1]] = c
            else:
                later.append(c)
        for c in later:
            place[free.pop(0)] = c
        for j, (s, k, i, tok, mag) in place.items():
            out[0][b, j], out[1][b, j], out[2][b, j] = s, k, tok
            out[3][b, j] = bool(finished is not None and finished[b, k]) or tok in eos
            size[b, j] = mag
    return out, size


def check_select(logits, scores, finished, eos, **kw):
    got = [t.cpu() for t in K.beam_select(logits.cuda(), scores.cuda(), None if finished is None else finished.cuda(),
                                          eos_ids=eos)]
    B, Kb = scores.shape
    ref, size = ref_select(logits.reshape(B, Kb, -1).float(), scores, finished, eos, **kw)
    for g, r in zip(got[1:], ref[1:]):
        assert torch.equal(g, r)
    live = ref[0] > -math.inf
    assert torch.equal(got[0] > -math.inf, live)
    assert bool(((got[0].double() - ref[0]).abs()[live] <= (2e-6 + 2 ** -22 * size)[live]).all())
    # a slot's parent is a beam that lives on in its own slot, or itself
    assert torch.equal(got[1].gather(1, got[1].long()), got[1])
    return got


def randn(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


@pytest.mark.gpu
@pytest.mark.parametrize("B,Kb,V,dtype", [
    (1, 1, 1, torch.float32), (1, 1, 7, torch.float32), (2, 3, 2, torch.float32), (3, 4, 50, torch.float32),
    (1, 2, 8191, torch.float32), (2, 5, 8193, torch.float32), (1, 16, 20001, torch.float32),
    (5, 4, 32000, torch.float32), (2, 8, 151936, torch.float32), (1, 3, 524288, torch.float32),
    (4, 4, 33, torch.bfloat16), (1, 16, 16, torch.bfloat16)])
def test_select_matches_64_bits(B, Kb, V, dtype):
    x = 3 * randn(V + Kb, B * Kb, V)
    if dtype == torch.bfloat16:     # distinct bf16 logits with wide gaps
        x = torch.stack([torch.randperm(V, generator=torch.Generator().manual_seed(i)).float() / 4 for i in range(B * Kb)])
    check_select(x.to(dtype), -5 * torch.rand(B, Kb, generator=torch.Generator().manual_seed(1)), None, ())


@pytest.mark.gpu
def test_select_wide_bf16_vocabulary():
    """bf16 logits tie often within a row: ties go to the lowest index."""
    B, Kb, V = 3, 4, 151936
    x = (3 * randn(4, B, Kb, V)).to(torch.bfloat16)
    check_select(x, -2 * torch.rand(B, Kb, generator=torch.Generator().manual_seed(2)), None, (5,))


@pytest.mark.gpu
@pytest.mark.parametrize("V", [100, 9000])
@pytest.mark.parametrize("Kb", [1, 4, 16])
def test_select_ties(V, Kb):
    """All logits equal (the list overflows), a few equal maxima, and the first step's empty beams."""
    s = torch.full((3, Kb), -math.inf)
    s[:, 0] = 0.0
    x = torch.zeros(3, Kb, V)
    x[1, :, V // 2:V // 2 + 3] = 2.0
    x[2, :, ::7] = 1.0
    check_select(x, s, None, (3,))
    check_select(x.to(torch.bfloat16), s, None, ())
    # equal scores across beams: the lower beam first
    check_select(x, torch.zeros(3, Kb), None, (3,))


@pytest.mark.gpu
def test_select_finished_dead_nan_and_masked():
    Kb, V, eos = 4, 40, (6, 9)
    x = 4 * randn(21, 6, Kb, V)
    s = -torch.rand(6, Kb, generator=torch.Generator().manual_seed(22))
    fin = torch.zeros(6, Kb, dtype=torch.bool)
    fin[0] = True                                    # a group that has finished
    fin[1, 1:3] = True
    x[1, 1:3] = float("nan")                         # not read
    s[2] = -math.inf                                 # nothing lives
    s[3, 1], s[3, 2] = float("nan"), -math.inf       # two beams live
    x[4] = -math.inf                                 # one allowed token in one beam
    x[4, 2, 9] = 1.0
    x[5, :, 1::2] = float("nan")                     # NaN logits count as masked
    x[5, 0] = -math.inf
    check_select(x, s, fin, eos)
    check_select(x[..., :40].to(torch.bfloat16).float(), s, fin, eos)
    # an infinite logit leaves its beam without a score
    x[5, 1, 0] = math.inf
    got = K.beam_select(x.cuda(), s.cuda(), fin.cuda(), eos_ids=eos)
    assert 1 not in got[1][5].tolist() or float(got[0][5, 1]) == -math.inf


@pytest.mark.gpu
def test_select_strided_rows_outputs_in_place_and_other_stream():
    B, Kb, V = 2, 3, 1000
    wide = 3 * randn(31, B * Kb, V + 9)
    s, fin = -torch.rand(B, Kb, generator=torch.Generator().manual_seed(3)), torch.tensor([[False, True, False]] * B)
    ref = check_select(wide[:, 3:3 + V].contiguous(), s, fin, (1,))
    g, gs, gf = wide.cuda(), s.cuda(), fin.cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = (gs, torch.empty(B, Kb, dtype=torch.int32, device="cuda"),
               torch.empty(B, Kb, dtype=torch.int64, device="cuda"), gf)
        K.beam_select(g[:, 3:3 + V], gs, gf, eos_ids=(1,), out=out)     # rows 12 bytes off a 16-byte boundary
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a.cpu(), b) for a, b in zip(out, ref))


def test_select_refuses_bad_arguments_without_a_gpu():
    lib = _lib.load()
    assert lib.bolt3_beam_select(None, None) == 1 and lib.bolt3_beam_reorder(None, None) == 1
    fake = 1 << 20

    def sel(**kw):
        a = _lib.BeamSelectArgs(B=2, K=4, V=100, logits=fake, row_stride=100, scores=fake, out_scores=fake,
                                out_parent=fake, out_token=fake, out_finished=fake, workspace=fake,
                                workspace_bytes=1 << 20)
        for k, v in kw.items():
            setattr(a, k, v)
        return lib.bolt3_beam_select(ctypes.byref(a), None)

    assert sel(K=17) == 2 and sel(V=524289, row_stride=1 << 20) == 2 and sel(V=0) == 2 and sel(B=0) == 2
    assert sel(row_stride=99) == 4 and sel(workspace_bytes=8) == 4 and sel(logits=fake + 1) == 3
    assert sel(finished=fake) == 1 and sel(n_eos=9) == 1 and sel(n_eos=1, eos_ids=(ctypes.c_int64 * 8)(100)) == 1
    assert lib.bolt3_beam_select_workspace(1, 17, 100) == 0

    item = _lib.BeamItem(base=fake, outer_stride=256, beam_stride=64, row_stride=64, row_bytes=64, token_bytes=16,
                         n_outer=1, n_row=1, unit=16)

    def mov(t0=0, t1=4, K_=4, **kw):
        it = _lib.BeamItem.from_buffer_copy(item)
        for k, v in kw.items():
            setattr(it, k, v)
        a = _lib.BeamReorderArgs(B=1, K=K_, parent=fake, items=ctypes.pointer(it), n_items=1, t0=t0, t1=t1)
        return lib.bolt3_beam_reorder(ctypes.byref(a), None)

    assert mov(t1=5) == 4 and mov(t0=3, t1=2) == 1 and mov(t0=-1) == 1 and mov(K_=17) == 2 and mov(unit=8) == 1
    assert mov(base=fake + 4) == 3 and mov(token_bytes=8) == 3 and mov(base=0) == 1 and mov(n_row=0) == 1
    assert mov(t0=2, t1=2) == 0                       # nothing to move: no launch


@pytest.mark.gpu
def test_select_refusals():
    x, s = torch.zeros(2, 3, 10, device="cuda"), torch.zeros(2, 3, device="cuda")
    f = torch.zeros(2, 3, dtype=torch.bool, device="cuda")
    for exc, args, kw in ((RuntimeError, (x.cpu(), s), {}), (TypeError, (x.half(), s), {}), (TypeError, (x, s.double()), {}),
                          (ValueError, (x[:, :2], s), {}), (ValueError, (x, s[0]), {}), (ValueError, (x, s, f), {}),
                          (ValueError, (x, s, f), dict(eos_ids=(10,))), (ValueError, (x, s, f), dict(eos_ids=range(9))),
                          (ValueError, (x.transpose(1, 2).contiguous().transpose(1, 2), s), {}),
                          (RuntimeError, (torch.zeros(1, 17, 4, device="cuda"), torch.zeros(1, 17, device="cuda")), {})):
        with pytest.raises(exc):
            K.beam_select(*args, **kw)


def moved(t, beam_dim, token_dim, parent, t0, t1):
    B, Kb = parent.shape
    src = (parent.long() + torch.arange(B)[:, None] * Kb).view(-1)
    out = t.clone()
    a, b = (t, out) if token_dim is None else (t.narrow(token_dim, t0, t1 - t0), out.narrow(token_dim, t0, t1 - t0))
    b.unflatten(beam_dim, (B * Kb, -1)).copy_(a.unflatten(beam_dim, (B * Kb, -1)).index_select(beam_dim, src))
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("B,Kb,seed", [(1, 1, 0), (3, 2, 1), (2, 4, 2), (5, 3, 3), (1, 8, 4), (2, 5, 5), (2, 16, 6)])
def test_reorder_any_map_in_place(B, Kb, seed):
    """Cycles, swaps and many children of one parent; every unit size, rows per beam, outer dimension."""
    g = torch.Generator().manual_seed(seed)
    n = B * Kb

    def rows(dtype, *shape):
        return torch.randint(-100, 100, shape, generator=g).to(dtype)

    items = [(rows(torch.int8, 2, n, 3, 50, 64), 1, 3), (rows(torch.float32, 2, n, 3, 50), 1, 3),
             (rows(torch.bfloat16, n * 2, 5, 8), 0, None), (rows(torch.int32, n), 0, None),
             (rows(torch.uint8, n, 7), 0, None), (rows(torch.bfloat16, n, 3), 0, None),
             (rows(torch.float32, n * 4, 37, 64), 0, None), (rows(torch.int8, n, 11, 3), 0, 1)]
    maps = [torch.randint(0, Kb, (B, Kb), generator=g), torch.arange(Kb).repeat(B, 1),
            torch.arange(Kb).roll(1).repeat(B, 1), torch.full((B, Kb), Kb - 1)]
    for parent in maps:
        for t0, t1 in ((0, 11), (3, 10), (5, 5)):
            dev = [(t.cuda(), a, b) for t, a, b in items]
            K.beam_reorder(dev, parent.int().cuda(), t0=t0, t1=t1)
            for (t, a, b), (d, _, _) in zip(items, dev):
                assert torch.equal(d.cpu(), moved(t, a, b, parent, t0, t1))


@pytest.mark.gpu
def test_reorder_many_items_bad_parents_and_reuse():
    n = 6
    items = [(torch.arange(n * (i + 1)).view(n, i + 1).float().cuda(), 0, None) for i in range(300)]   # three launches
    plan = K.BeamReorder(items, 2, 3)
    status = K.DeviceStatus("cuda")
    parent = torch.tensor([[1, 7, -1], [2, 2, 2]], dtype=torch.int32)
    plan(parent.cuda(), status=status)
    assert int(status.word) == 8                      # 7 and -1 leave their beams as they are
    good = torch.tensor([[1, 1, 2], [2, 2, 2]])
    for i, (t, _, _) in enumerate(items):
        was = torch.arange(n * (i + 1)).view(n, i + 1).float()
        assert torch.equal(t.cpu(), moved(was, 0, None, good, 0, 0))


@pytest.mark.gpu
def test_reorder_large_strides():
    """Beams more than 2^31 bytes apart."""
    t = torch.zeros(2, 2_300_000_000, dtype=torch.int8, device="cuda")
    t[0, -40:], t[1, :16] = 3, 5
    plan = K.BeamReorder([(t, 0, None)], 1, 2)
    plan(torch.tensor([[1, 0]], dtype=torch.int32, device="cuda"))
    assert bool((t[1, -40:] == 3).all()) and bool((t[0, :16] == 5).all()) and int(t[0, 16:].any()) == 0 and int(t[1, :-40].any()) == 0


@pytest.mark.gpu
def test_reorder_refusals():
    t = torch.zeros(4, 8, 16, device="cuda")
    p = torch.zeros(2, 2, dtype=torch.int32, device="cuda")
    for exc, items in ((ValueError, [(t[:, ::2], 0, None)]), (RuntimeError, [(t.cpu(), 0, None)]),
                       (ValueError, [(t[:3], 0, None)]), (ValueError, [(t, 1, 0)]), (ValueError, [(t, 3, None)]),
                       (ValueError, [(t, 0, None), (t[1:].view(3, 128)[:2].repeat(1, 1).view(4, 64), 0, None), (t, 0, None)])):
        with pytest.raises(exc):
            K.beam_reorder(items, p)
    for exc, kw in ((TypeError, dict(parent=p.long())), (ValueError, dict(parent=p[:1])), (ValueError, dict(parent=p, t0=2, t1=9)),
                    (ValueError, dict(parent=p, t0=3, t1=2))):
        with pytest.raises(exc):
            K.BeamReorder([(t, 0, 1)], 2, 2)(**kw)
