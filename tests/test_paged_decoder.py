"""Paged anchor caches in the decoder: bookkeeping, prompts and single tokens, budgets, CUDA-graph steps, beams that share
pages, tensor-parallel shards, errors.

Where a step is compared with one whose attention is split elsewhere, the sums' order differs; hidden states are then
held to 0.05 of their RMS, as for the other caches.
"""
import copy

import pytest
import torch

import test_beam_search as beams_of
from test_paged import ref_attend, rounded_within, rows_of, same
from vsa_lm_b200 import AnchorKVPaged, Bolt3Decoder
from vsa_lm_b200.model import Bolt3LM, SoftmaxAttn
from vsa_lm_b200.tp import Bolt3DecoderTP, Bolt3LMTP, shard_softmax_attn
from vsa_lm_b200.workloads import MODEL_SHAPES, make_model_params


def _model(shape, dev="cuda"):
    mcfg = dict(MODEL_SHAPES[shape])
    model = Bolt3LM(**mcfg)
    model.load_state_dict(make_model_params(mcfg, 0), strict=True)
    return mcfg, model.to(device=dev, dtype=torch.bfloat16).eval()


def _ids(mcfg, B, T, seed=1):
    return torch.randint(0, mcfg["vocab_size"], (B, T), generator=torch.Generator().manual_seed(seed)).cuda()


def _anchors(kv):
    return [c for c in kv if isinstance(c, AnchorKVPaged)]


# ------------------------------------------------------------------------------------------- on the CPU

def _write(cache, rows):
    """Rows [2, B, HKV, t, HD] behind the held ones, through the table as the append does."""
    t = rows.shape[3]
    cache.reserve(t)
    for i in range(t):
        r = cache.n + i
        for b in range(cache.B):
            cache.pages[:, int(cache.table[b, r // cache.page]), :, r % cache.page] = rows[:, b, :, i]
    cache.n += t
    cache.seen += t


def test_bookkeeping_on_cpu():
    g = torch.Generator().manual_seed(1)
    c = AnchorKVPaged(2, 3, 100, 64, "cpu", page=16)
    assert c.capacity == 256 and c.page == 16 and c.k.shape == (2, 3, 0, 64)
    rows = torch.randn(2, 2, 3, 700, 64, generator=g).bfloat16()
    for lo, hi in ((0, 250), (250, 251), (251, 300), (300, 700)):
        _write(c, rows[:, :, :, lo:hi])
    assert c.capacity == 1024 and len(set(c.table.flatten().tolist())) == c.table.numel()
    assert torch.equal(c.read(), rows) and torch.equal(c.k, rows[0]) and torch.equal(c.read(40, 300)[1], rows[1][:, :, 40:300])
    assert torch.equal(c.positions[1, 2], torch.arange(700).int())
    with pytest.raises(ValueError):
        c.read(0, 701)
    d = AnchorKVPaged(2, 3, 10 ** 6, 64, "cpu", page=32, budget=100)
    assert d.capacity == 384 and d.recent == 50 and d.weight.shape == d.order.shape == (2, 3, 384)   # 100 + 2 * 128 rows
    d.reserve(384)
    assert d.capacity == 384
    d.reserve(385)
    assert d.capacity == 768 and d.weight.shape == (2, 3, 768)


@pytest.mark.parametrize("page,T", [(16, 37), (16, 32), (64, 5)])
def test_beams_share_pages_on_cpu(page, T):
    """Beams through selections as beam_select makes them (a beam that goes on keeps its slot): every beam reads its own
    past, and no page of the prompt is copied but the last."""
    B, beams, HKV, HD = 2, 4, 2, 64
    g = torch.Generator().manual_seed(2)
    c = AnchorKVPaged(B, HKV, T + 200, HD, "cpu", page=page)
    prompt = torch.randn(2, B, HKV, T, HD, generator=g).bfloat16()
    _write(c, prompt)
    c = c.repeated(beams)
    past = prompt.repeat_interleave(beams, 1)
    full = T // page
    assert len(set(c.table[:, :full].flatten().tolist())) == B * full
    assert torch.equal(c.read(), past)
    for step in range(70):
        pick = torch.randint(0, beams, (B, beams), generator=g)
        if step % 5 == 0:
            pick = torch.arange(beams).expand(B, beams)
        lives = torch.zeros(B, beams, dtype=torch.bool).scatter_(1, pick, True)
        parent = torch.where(lives, torch.arange(beams), pick)
        c.reorder(parent.int())
        past = past[:, (parent + torch.arange(B)[:, None] * beams).view(-1)]
        assert torch.equal(c.read(), past)
        row = torch.randn(2, B * beams, HKV, 1, HD, generator=g).bfloat16()
        _write(c, row)
        past = torch.cat((past, row), 3)
        assert torch.equal(c.read(), past)
    d = AnchorKVPaged(B, HKV, 100, HD, "cpu", page=page, budget=64)
    _write(d, prompt[:, :, :, :5])
    e = d.repeated(2)
    assert torch.equal(e.read(), d.read().repeat_interleave(2, 1)) and e.weight.shape[0] == 4
    with pytest.raises(ValueError):
        e.reorder(torch.zeros(B, 2, dtype=torch.int32))


def test_arguments_are_checked():
    mcfg = dict(MODEL_SHAPES["tiny_lm"])
    model = Bolt3LM(**mcfg)
    for bad in (dict(kv_page=48), dict(kv_budget=0), dict(kv_budget=10, kv_recent=11), dict(kv_recent=3)):
        with pytest.raises(ValueError):
            Bolt3Decoder(model, kv_cache="paged", **bad)
        with pytest.raises(ValueError):
            Bolt3Decoder.blank_state(model, 1, "cpu", kv_cache="paged", **bad)
    for kind in ("bf16", "int8"):
        with pytest.raises(ValueError, match="budget"):
            Bolt3Decoder(model, kv_cache=kind, kv_budget=10)
    with pytest.raises(ValueError, match="paged"):
        Bolt3Decoder(model, kv_cache="pages")
    with pytest.raises(ValueError, match="budget"):
        Bolt3Decoder(model, kv_cache="paged", kv_budget=300).beam_search(torch.zeros(1, 4, dtype=torch.long), 2, 3)
    bf16, paged = Bolt3Decoder.state_bytes(model), Bolt3Decoder.state_bytes(model, kv_cache="paged")
    assert bf16 == paged
    fixed, per = Bolt3Decoder.state_bytes(model, kv_cache="paged", kv_budget=100, kv_page=32)
    kv = [AnchorKVPaged(3, b.attn.HKV, 10 ** 6, b.attn.HD, "cpu", page=32, budget=100) for b in model.blocks if not hasattr(b, "vsa")]
    held = sum(t.numel() * t.element_size() for c in kv for t in (c.pages, c.weight, c.order))
    assert per == 0 and held and held == 3 * (fixed - bf16[0])


# ------------------------------------------------------------------------------------------- on the GPU

@pytest.mark.gpu
@pytest.mark.parametrize("qk_norm,HD,HKV,page,budget", [(False, 64, 2, 16, None), (True, 128, 4, 64, None), (True, 64, 1, 32, 120)])
def test_anchor_attention_over_a_paged_cache(qk_norm, HD, HKV, page, budget):
    """Prompt slices, an odd slice and single tokens through AnchorKVPaged.attention: the rows are the norm and rotation of
    the projections, and the outputs are the softmax over them (tolerances as derived in test_paged.py)."""
    cfg = dict(dim=256, num_heads=8, num_kv_heads=HKV, head_dim=HD, rope_theta=1e4, eps=1e-6, qk_norm=qk_norm)
    torch.manual_seed(1)
    ly = SoftmaxAttn(cfg).to(device="cuda", dtype=torch.bfloat16).eval()
    if qk_norm:
        for m in (ly.q_norm, ly.k_norm):
            m.weight.data.uniform_(0.8, 1.2)
    B, cache = 2, AnchorKVPaged(2, HKV, 200, HD, "cuda", page=page, budget=budget)
    pos, keys = 0, []
    with torch.no_grad():
        for t in (128, 128, 37, 1, 1, 3, 1, 90):
            h = torch.randn(B, t, 256, device="cuda").bfloat16()
            before = copy.deepcopy(cache)
            y = cache.attention(ly, h, pos)
            k = ly.k_norm(ly.k_proj(h).view(B, t, HKV, HD)) if qk_norm else ly.k_proj(h).view(B, t, HKV, HD)
            keys.append(ly.rope(k.transpose(1, 2).float(), pos_start=pos))
            # the same call's queries, on a copy of what was there
            from vsa_lm_b200 import kernels as K
            before.reserve(t)
            q = K.paged_append(q=ly.q_proj(h), k=ly.k_proj(h), v=ly.v_proj(h), pages=before.pages, table=before.table, n=before.n,
                               pos0=pos, inv_freq=ly.rope.inv_freq.float().contiguous(),
                               q_norm=ly.q_norm.weight.float() if qk_norm else None,
                               k_norm=ly.k_norm.weight.float() if qk_norm else None, eps=1e-6, weight=before.weight, order=before.order)
            n = before.n
            ref, mass, err, rec, rec_err = ref_attend(q.cpu(), before.pages.cpu(), before.table.cpu(), [n] * B, HD ** -0.5, HKV)
            few = t * (8 // HKV) <= 16
            tol = mass * (2 * (err + (2 ** -17 if few else 2 ** -9) + 2 ** -21) + (n + t) * 2 ** -23)
            assert rounded_within(y.cpu().view(B, t, 8, HD), ref, tol)
            pos += t
            if budget is None:
                assert cache.n == pos
            else:
                assert cache.n <= budget + 128 + 127 and cache.seen == pos
            # bf16's roundings of a norm, of a product and of a sum in the module, one here
            want = torch.cat(keys, 2).gather(2, cache.positions.long()[..., None].expand(-1, -1, -1, HD))
            assert bool(((cache.k.float() - want).abs() <= 4 * 2 ** -8 * want.abs().amax(-1, keepdim=True)).all())
    cache.check_status()
    if budget is not None:
        assert cache.capacity < 3 * 128 + budget and cache.n < pos


@pytest.mark.gpu
@pytest.mark.parametrize("shape", ["small_lm", "tiny_lm"])
@pytest.mark.parametrize("budget", [None, 150])
def test_paged_step_graph_equals_eager_steps(shape, budget):
    mcfg, model = _model(shape)
    dec = Bolt3Decoder(model, kv_cache="paged", kv_budget=budget, kv_page=32)
    B, T, N = 2, 300, 150
    ids, steps = _ids(mcfg, B, T), _ids(mcfg, B, N, 3)
    h0, st_e, kv_e = dec.prefill(ids)
    h1, st_g, kv_g = dec.prefill(ids)
    assert torch.equal(h0, h1) and _anchors(kv_e)
    if budget is None:                                    # the same model over contiguous caches
        h2, _, _ = Bolt3Decoder(model).prefill(ids)
        assert (h2.float() - h0.float()).abs().mean() <= 0.05 * h2.float().abs().mean()
    runner = dec.step_graph(st_g, kv_g)
    for i in range(N):
        tok = steps[:, i:i + 1]
        he, st_e, kv_e = dec.step(tok, T + i, st_e, kv_e)
        hg = runner.step(tok, T + i)
        err = (hg.float() - he.float()).abs().amax()
        assert err <= 0.05 * he.float().pow(2).mean().sqrt(), (i, float(err))
        assert [c.n for c in _anchors(kv_e)] == [c.n for c in _anchors(kv_g)]
    runner.close()
    Bolt3Decoder.check_status(kv_e)
    Bolt3Decoder.check_status(kv_g)
    for a, b in zip(_anchors(kv_e), _anchors(kv_g)):
        if budget is None:
            assert a.n == T + N
            continue
        # 450 tokens seen, the last chunk's end at 384: 150 rows then, and 66 tokens since
        assert a.n == b.n == budget + 66 and a.seen == T + N
        for c in (a, b):
            pos = c.positions
            assert bool((pos.sort(-1).values.diff(dim=-1) > 0).all())               # no token twice
            assert bool((pos.sort(-1, descending=True).values[..., :141] == torch.arange(T + N - 1, T + N - 142, -1, device="cuda")).all())
            # every head's records add up to what its queries gave the rows that are left: at most one each
            assert bool((c.weight[..., :c.n].sum(-1) <= (T + N) * mcfg["num_heads"] // mcfg["num_kv_heads"] * (1 + 1e-3)).all())
            assert bool((c.weight[..., :c.n] >= 0).all())
        # the records agree but for the sums' order and what followed from it
        assert float((a.weight[..., :a.n].sum(-1) / b.weight[..., :b.n].sum(-1) - 1).abs().max()) < 0.05


@pytest.mark.gpu
def test_kept_rows_are_those_of_a_full_cache():
    """The first anchor sees the same inputs whatever it keeps: its rows are a full cache's rows of their positions, bit for
    bit, and its first eviction is the one of the full records."""
    mcfg, model = _model("small_lm")
    ids = _ids(mcfg, 2, 128 * 2 + 40)
    full = Bolt3Decoder(model, kv_cache="paged")
    wide = Bolt3Decoder(model, kv_cache="paged", kv_budget=10 ** 4)
    dec = Bolt3Decoder(model, kv_cache="paged", kv_budget=100, kv_recent=30)
    hf, _, kvf = full.prefill(ids)
    hw, _, kvw = wide.prefill(ids)
    assert torch.equal(hf, hw)                            # a record changes no output
    _, _, kv = dec.prefill(ids)
    f, c = _anchors(kvf)[0], _anchors(kv)[0]
    at = c.positions.long()[None, ..., None].expand(2, -1, -1, -1, f.pages.shape[-1])
    assert same(c.read(), f.read().gather(3, at).contiguous())
    assert c.n == 100 + 40 and f.n == 296
    # after 128 tokens: the 30 newest and the 70 heaviest of the others
    _, _, kv1 = dec.prefill(ids[:, :128])
    _, _, kv2 = wide.prefill(ids[:, :128])
    w = _anchors(kv2)[0].weight[..., :98].cpu()
    heavy = w.sort(dim=-1, descending=True, stable=True).indices[..., :70].sort(-1).values
    got = _anchors(kv1)[0].positions.cpu().sort(-1).values
    assert torch.equal(got[..., :70], heavy.int()) and bool((got[..., 70:] == torch.arange(98, 128)).all())


@pytest.mark.gpu
def test_generation_at_constant_size():
    mcfg, model = _model("tiny_lm")
    dec = Bolt3Decoder(model, kv_cache="paged", kv_budget=64, kv_page=16)
    ids = _ids(mcfg, 3, 200)
    toks, lengths = dec.generate_batch(ids, 400, temperature=0.0)
    assert toks.shape == (3, 400)
    h, states, kv = dec.prefill(ids)
    cap = [c.capacity for c in _anchors(kv)]
    out, states, kv, pos = dec.continue_generate(_ids(mcfg, 3, 77, 5), states, kv, 200, 300)
    assert pos == 577 and [c.capacity for c in _anchors(kv)] == cap
    assert all(c.seen == 577 and c.n <= 64 + 127 for c in _anchors(kv))
    # a generation whose budget is never reached is the one without
    a = Bolt3Decoder(model, kv_cache="paged", kv_budget=5000).generate_batch(ids, 40, temperature=0.0)[0]
    b = Bolt3Decoder(model, kv_cache="paged").generate_batch(ids, 40, temperature=0.0)[0]
    assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("beams,T,graphs", [(4, 150, True), (3, 128, False), (1, 40, True)])
def test_beam_scores_over_paged_caches(beams, T, graphs):
    beams_of.test_beam_scores_are_those_of_the_returned_tokens("tiny_lm", "paged", beams, T, graphs)


@pytest.mark.gpu
def test_beam_search_over_paged_caches_is_that_over_contiguous_ones():
    """The same tokens as with int8 or bf16 caches need not come out; the same as with unshared pages must: one beam's past
    is read through shared pages bit for bit."""
    mcfg, model = _model("small_lm")
    dec = Bolt3Decoder(model, kv_cache="paged", kv_page=16)
    ids = _ids(mcfg, 2, 70)
    toks, scores, lengths = dec.beam_search(ids, 4, 40)
    one, s1, _ = dec.beam_search(ids, 1, 40)
    greedy, _ = dec.generate_batch(ids, 40, temperature=0.0)
    assert torch.equal(one[:, 0], greedy)
    assert bool((scores[:, 0] >= s1[:, 0] - 1e-3).all())


@pytest.mark.gpu
@pytest.mark.parametrize("world,qk_norm", [(2, True), (4, False)])
def test_shards_of_an_anchor_over_paged_caches(world, qk_norm):
    torch.manual_seed(1)
    cfg = dict(dim=512, num_heads=16, num_kv_heads=4, head_dim=128, rope_theta=1e4, eps=1e-6, qk_norm=qk_norm)
    attn = SoftmaxAttn(cfg).to(device="cuda", dtype=torch.bfloat16).eval()
    shards = [shard_softmax_attn(attn, r, world) for r in range(world)]
    B, cache = 2, AnchorKVPaged(2, 4, 300, 128, "cuda")
    caches = [AnchorKVPaged(B, s.HKV, 300, s.HD, "cuda") for s in shards]
    pos = 0
    with torch.no_grad():
        for t in (128, 40, 1, 1, 3):
            h = torch.randn(B, t, 512, device="cuda").bfloat16()
            ref = Bolt3Decoder._anchor_attention(attn, cache, h, pos).float()
            got = sum(Bolt3Decoder._anchor_attention(s, c, h, pos, partial_fp32=True) for s, c in zip(shards, caches))
            assert got.dtype == torch.float32 and got.shape == ref.shape
            # one rounding to bf16, and the attention's own bf16 output by a split of the keys in another order
            assert bool(((got - ref).abs() <= 2 ** -8 * ref.abs() + 2 ** -8 * ref.pow(2).mean().sqrt()).all())
            pos += t
    assert same(torch.cat([c.read() for c in caches], 2).contiguous(), cache.read())


@pytest.mark.gpu
def test_a_tensor_parallel_decoder_with_a_budget():
    """One rank, no process group: the split model's own step."""
    mcfg, model = _model("small_lm")
    dec = Bolt3DecoderTP(Bolt3LMTP(model), kv_cache="paged", kv_budget=120)
    ids = _ids(mcfg, 2, 290)
    h, states, kv = dec.prefill(ids)
    ref, _, _ = Bolt3Decoder(model, kv_cache="paged", kv_budget=120).prefill(ids)
    assert (h.float() - ref.float()).abs().mean() <= 0.05 * ref.float().abs().mean()
    assert all(c.n == 120 + 34 for c in _anchors(kv))
    toks, _ = dec.generate_batch(ids, 12, temperature=0.0)
    assert toks.shape == (2, 12)


@pytest.mark.gpu
@pytest.mark.parametrize("call", ["generate_batch", "continue_generate", "beam_search", "steps"])
def test_errors_of_the_kernels_reach_the_caller(call):
    """Made on the host: a status word is set as a kernel would set it."""
    mcfg, model = _model("tiny_lm")
    dec = Bolt3Decoder(model, kv_cache="paged")
    ids = _ids(mcfg, 1, 40)
    if call in ("generate_batch", "beam_search"):
        real = dec.prefill

        def prefill(ids, **kw):
            h, states, kv = real(ids, **kw)
            _anchors(kv)[0].status.word.fill_(2)
            return h, states, kv

        dec.prefill = prefill
        with pytest.raises(RuntimeError, match="bounded wait"):
            dec.generate_batch(ids, 3, temperature=0.0) if call == "generate_batch" else dec.beam_search(ids, 2, 3)
        return
    _, states, kv = dec.prefill(ids)
    _anchors(kv)[0].status.word.fill_(2)
    with pytest.raises(RuntimeError, match="bounded wait"):
        if call == "continue_generate":
            dec.continue_generate(ids[:, :5], states, kv, 40, 3)
        else:
            for i in range(300):
                dec.step(ids[:, :1], 40 + i, states, kv)


@pytest.mark.gpu
def test_a_model_of_anchors_alone():
    """No other state in the steps, their graphs and the beams' reordering."""
    torch.manual_seed(3)
    model = Bolt3LM(vocab_size=64, dim=128, num_layers=2, num_heads=4, num_kv_heads=2, head_dim=64, intermediate=128,
                    layer_types=["softmax", "softmax"]).to("cuda", torch.bfloat16).eval()
    ids = torch.randint(0, 64, (2, 150), generator=torch.Generator().manual_seed(4)).cuda()
    for budget in (None, 40):
        dec = Bolt3Decoder(model, kv_cache="paged", kv_page=16, kv_budget=budget)
        (_, st_e, kv_e), (_, st_g, kv_g) = dec.prefill(ids), dec.prefill(ids)
        runner = dec.step_graph(st_g, kv_g)
        for i in range(120):
            tok = ids[:, i:i + 1]
            he, _, _ = dec.step(tok, 150 + i, st_e, kv_e)
            err = (runner.step(tok, 150 + i).float() - he.float()).abs().amax()
            assert err <= 0.05 * he.float().pow(2).mean().sqrt(), (budget, i, float(err))
        runner.close()
        Bolt3Decoder.check_status(kv_g)
        # 270 tokens seen, the last chunk's end at 256
        assert all(c.n == (270 if budget is None else 40 + 14) and c.seen == 270 for c in kv_e + kv_g)
    toks, scores, lengths = Bolt3Decoder(model, kv_cache="paged", kv_page=16).beam_search(ids, 3, 30)
    assert toks.shape == (2, 3, 30) and bool(scores.isfinite().all()) and bool((scores.diff(dim=1) <= 0).all())
