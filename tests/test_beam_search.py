"""The 8-bit anchor caches and beam search inside the decoder.

A hypothesis' score is checked by feeding its tokens through a second state, expanded the same way and
never reordered: the same kernels at the same sizes, so a hypothesis that was scored on a state of
another beam (a missed or wrong move) shows at once, while rounding is the same on both sides.
"""
import copy

import pytest
import torch

from vsa_lm_b200 import AnchorKV8, Bolt3Decoder, Bolt3LayerState, kernels as K
from vsa_lm_b200.beam import backtrack, expand_beams
from vsa_lm_b200.model import Bolt3LM, SoftmaxAttn
from vsa_lm_b200.workloads import MODEL_SHAPES, make_model_params
from test_kv8 import check_attend


def _model(shape):
    mcfg = dict(MODEL_SHAPES[shape])
    model = Bolt3LM(**mcfg)
    model.load_state_dict(make_model_params(mcfg, 0), strict=True)
    return mcfg, model.to(device="cuda", dtype=torch.bfloat16).eval()


def test_backtrack_follows_the_parents():
    tokens = [torch.tensor([[5, 6, 7]]), torch.tensor([[1, 2, 3]]), torch.tensor([[8, 9, 4]])]
    parents = [torch.tensor([[0, 1, 2]], dtype=torch.int32), torch.tensor([[0, 0, 2]], dtype=torch.int32),
               torch.tensor([[2, 1, 2]], dtype=torch.int32)]
    assert backtrack(tokens, parents, 0).tolist() == [[[7, 3, 8], [5, 2, 9], [7, 3, 4]]]


def test_int8_cache_bookkeeping_on_cpu():
    c = AnchorKV8(2, 3, 100, 64, "cpu")
    assert c.capacity == 256 and c.n == 0 and tuple(c.read().shape) == (2, 2, 3, 0, 64)
    c.data.random_(-5, 5)
    c.scale.uniform_()
    c.n = 250
    d, s = c.data.clone(), c.scale.clone()
    c.reserve(7)
    assert c.capacity == 512 and torch.equal(c.data[:, :, :, :250], d[:, :, :, :250])
    assert torch.equal(c.scale[:, :, :, :250], s[:, :, :, :250])
    r = c.repeated(3)
    assert r.n == 250 and torch.equal(r.data[:, 4], c.data[:, 1]) and torch.equal(r.scale[:, 2], c.scale[:, 0])
    with pytest.raises(ValueError):
        c.read(0, 251)
    model = Bolt3LM(**dict(MODEL_SHAPES["tiny_lm"]))
    with pytest.raises(ValueError):
        Bolt3Decoder(model, kv_cache="int4")
    bf16, int8 = Bolt3Decoder.state_bytes(model), Bolt3Decoder.state_bytes(model, kv_cache="int8")
    a = [b.attn for b in model.blocks if not hasattr(b, "vsa")]
    assert bf16[0] == int8[0] and int8[1] == sum(2 * x.HKV * (x.HD + 4) for x in a)
    with pytest.raises(ValueError):
        Bolt3Decoder(model).beam_search(torch.zeros(1, 4, dtype=torch.long), 17, 5)


@pytest.mark.gpu
@pytest.mark.parametrize("qk_norm,HD,HKV", [(True, 128, 2), (False, 64, 4)])
def test_anchor_attention_over_int8_cache(qk_norm, HD, HKV):
    """Prompt slices, an odd slice and single tokens through AnchorKV8.attention: what the cache holds is the
    quantised norm and rotation of the projections, and the outputs are the softmax over it."""
    cfg = dict(dim=256, num_heads=8, num_kv_heads=HKV, head_dim=HD, rope_theta=1e4, eps=1e-6, qk_norm=qk_norm)
    torch.manual_seed(1)
    ly = SoftmaxAttn(cfg).to(device="cuda", dtype=torch.bfloat16).eval()
    if qk_norm:
        for m in (ly.q_norm, ly.k_norm):
            m.weight.data.uniform_(0.8, 1.2)
    B, cache = 2, AnchorKV8(2, HKV, 200, HD, "cuda")
    pos = 0
    with torch.no_grad():
        for t in (128, 128, 37, 1, 1, 3, 1):
            h = torch.randn(B, t, 256, device="cuda").bfloat16()
            y = cache.attention(ly, h, pos)
            q = torch.empty(B, t, 8, HD, dtype=torch.bfloat16, device="cuda")
            spare = copy.deepcopy(cache)
            K.kv8_append(q=ly.q_proj(h), k=ly.k_proj(h), v=ly.v_proj(h), data=spare.data, scale=spare.scale, n=pos, pos0=pos,
                         inv_freq=ly.rope.inv_freq.float().contiguous(), q_out=q,
                         q_norm=ly.q_norm.weight.float() if qk_norm else None,
                         k_norm=ly.k_norm.weight.float() if qk_norm else None, eps=1e-6)
            assert torch.equal(spare.data, cache.data)
            check_attend(q.cpu(), cache.data.cpu(), cache.scale.cpu(), pos, None, HD ** -0.5, y.cpu())
            k = ly.k_norm(ly.k_proj(h).view(B, t, HKV, HD)) if qk_norm else ly.k_proj(h).view(B, t, HKV, HD)
            k = ly.rope(k.transpose(1, 2).float(), pos_start=pos)
            got = cache.read(pos, pos + t)[0].float()
            # half a step of 1 / 127, bf16's rounding of the norm before the rotation, of the product read back
            top = k.abs().amax(-1, keepdim=True)
            assert bool(((got - k).abs() <= top * (0.5 / 127 + 3 * 2 ** -8)).all())
            pos += t
    assert cache.n == pos == 299 and cache.capacity == 512       # grew once
    assert tuple(cache.k.shape) == (B, HKV, pos, HD) and torch.equal(cache.v, cache.read()[1])


@pytest.mark.gpu
def test_int8_cache_reports_its_kernels_errors():
    """A device step position past the span of its launches is found by Bolt3Decoder.check_status, once."""
    cfg = dict(dim=256, num_heads=8, num_kv_heads=2, head_dim=64, rope_theta=1e4, eps=1e-6, qk_norm=False)
    ly = SoftmaxAttn(cfg).to(device="cuda", dtype=torch.bfloat16).eval()
    cache = AnchorKV8(1, 2, 200, 64, "cuda")
    pos = K.DevicePosition("cuda")
    pos.ref, pos.span = 0, 4
    h = torch.randn(1, 1, 256, device="cuda").bfloat16()
    with torch.no_grad():
        pos.set(3)
        cache.attention(ly, h, 0, pos)
        Bolt3Decoder.check_status([cache])
        pos.set(4)
        y = cache.attention(ly, h, 0, pos)
        assert bool((y == 0).all())
        with pytest.raises(RuntimeError, match="out of range|outside the range"):
            Bolt3Decoder.check_status([cache])
        Bolt3Decoder.check_status([cache])


@pytest.mark.gpu
@pytest.mark.parametrize("shape", ["small_lm", "tiny_lm"])
def test_int8_step_graph_equals_eager_steps(shape):
    mcfg, model = _model(shape)
    dec = Bolt3Decoder(model, kv_cache="int8")
    g = torch.Generator().manual_seed(3)
    B, T = 2, 300
    ids = torch.randint(0, mcfg["vocab_size"], (B, T), generator=g).cuda()
    steps = torch.randint(0, mcfg["vocab_size"], (B, 100), generator=g).cuda()
    h0, st_e, kv_e = dec.prefill(ids)
    h1, st_g, kv_g = dec.prefill(ids)
    assert torch.equal(h0, h1) and any(isinstance(c, AnchorKV8) for c in kv_e)
    runner = dec.step_graph(st_g, kv_g)
    for i in range(steps.shape[1]):
        tok = steps[:, i:i + 1]
        he, st_e, kv_e = dec.step(tok, T + i, st_e, kv_e)
        hg = runner.step(tok, T + i)
        # the split of the cache goes by the length a launch was built for: sums in another order
        err = (hg.float() - he.float()).abs().amax()
        assert err <= 0.05 * he.float().pow(2).mean().sqrt(), (i, float(err))
    runner.close()
    # the same model over bf16 caches: one int8 step of the anchors' rows apart
    ref = Bolt3Decoder(model)
    h2, _, _ = ref.prefill(ids)
    assert (h2.float() - h0.float()).abs().mean() <= 0.05 * h2.float().abs().mean()


@pytest.mark.gpu
@pytest.mark.parametrize("shape,kv_cache,beams,T,graphs", [
    ("small_lm", "int8", 4, 200, True), ("small_lm", "bf16", 3, 200, False), ("tiny_lm", "int8", 16, 128, True),
    ("tiny_lm", "bf16", 1, 77, True), ("small_lm", "int8", 2, 5, False)])
def test_beam_scores_are_those_of_the_returned_tokens(shape, kv_cache, beams, T, graphs):
    mcfg, model = _model(shape)
    dec = Bolt3Decoder(model, kv_cache=kv_cache, cuda_graphs=graphs)
    g = torch.Generator().manual_seed(T)
    B, new = 2, 70
    ids = torch.randint(0, mcfg["vocab_size"], (B, T), generator=g).cuda()
    toks, scores, lengths = dec.beam_search(ids, beams, new)
    assert toks.shape == (B, beams, new) and bool((lengths == new).all())
    assert bool((scores[:, :-1] >= scores[:, 1:]).all())
    assert len({tuple(t) for t in toks[0].tolist()}) == beams
    # rescored on states that nothing moved
    h, states, kv = dec.prefill(ids, max_kv_len=T + new + 64)
    logits = model.lm_head(h[:, -1, :]).repeat_interleave(beams, dim=0)
    states, kv = expand_beams(model, states, kv, beams)
    runner = dec.step_graph(states, kv) if graphs else None
    total = torch.zeros(B * beams, dtype=torch.float64, device="cuda")
    flat = toks.view(B * beams, new)
    for i in range(new):
        total += torch.log_softmax(logits.double(), -1).gather(1, flat[:, i:i + 1])[:, 0]
        tok = flat[:, i:i + 1].contiguous()
        h = runner.step(tok, T + i) if graphs else dec.step(tok, T + i, states, kv)[0]
        logits = model.lm_head(h[:, -1, :])
    if runner is not None:
        runner.close()
    # 70 fp32 sums of scores of a few hundred: 70 * 2^-24 * 500, and as much for the log-sum-exps
    assert bool(((total.view(B, beams) - scores.double()).abs() <= 5e-3).all())


@pytest.mark.gpu
def test_beam_search_ends_at_eos():
    """One step, greedy: the K best first tokens; an end-of-sequence id among them ends its beam at once."""
    mcfg, model = _model("tiny_lm")
    dec = Bolt3Decoder(model, kv_cache="int8")
    ids = torch.randint(0, mcfg["vocab_size"], (1, 40), generator=torch.Generator().manual_seed(1)).cuda()
    h, _, _ = dec.prefill(ids)
    best = torch.log_softmax(model.lm_head(h[:, -1]).double(), -1)[0].topk(6)
    toks, scores, lengths = dec.beam_search(ids, 4, 1)
    assert set(toks[0, :, 0].tolist()) == set(best.indices[:4].tolist())
    eos = int(best.indices[0])
    toks, scores, lengths = dec.beam_search(ids, 1, 30, eos_ids=(eos,))
    assert lengths.tolist() == [[1]] and bool((toks == eos).all()) and toks.shape[2] == 16   # looked at after 16
    toks, scores, lengths = dec.beam_search(ids, 4, 20, eos_ids=(eos,))
    ended = lengths[0] < toks.shape[2]
    for j in range(4):
        row, n = toks[0, j].tolist(), int(lengths[0, j])
        assert eos not in row[:n - 1] and all(t == eos for t in row[n:])
        if ended[j]:
            assert row[n - 1] == eos
    assert bool((scores[:, :-1] >= scores[:, 1:]).all())


@pytest.mark.gpu
def test_expanded_state_steps_like_the_original():
    """Every beam of an expanded state continues as the sequence it was copied from, an oversize pending chunk
    included, and the copies are independent."""
    mcfg, model = _model("small_lm")
    dec = Bolt3Decoder(model, kv_cache="int8")
    g = torch.Generator().manual_seed(9)
    B, T, beams = 2, 300, 3
    ids = torch.randint(0, mcfg["vocab_size"], (B, T), generator=g).cuda()
    _, states, kv = dec.prefill(ids)
    extra = torch.randint(0, mcfg["vocab_size"], (B, 100), generator=g).cuda()
    _, states, kv = dec.step(extra, T, states, kv)              # an unaligned slice: a chunk of 144 tokens
    assert any(isinstance(c, Bolt3LayerState) and c.big_prev is not None for c in kv)
    s2, k2 = expand_beams(model, states, kv, beams)
    tok = torch.randint(0, mcfg["vocab_size"], (B, 1), generator=g).cuda()
    h, _, _ = dec.step(tok, T + 100, states, kv)
    h2, _, _ = dec.step(tok.repeat_interleave(beams, 0), T + 100, s2, k2)
    ref = h.repeat_interleave(beams, 0).float()
    assert (h2.float() - ref).abs().amax() <= 0.05 * ref.pow(2).mean().sqrt()
