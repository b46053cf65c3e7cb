"""A decoder with 8-bit anchor caches: errors that its kernels report on the device reach the caller, a beam search
pads with the id it was given first, and models that it cannot serve are refused when it is made.

The errors are made on the host: a status word is set as a kernel would set it. No kernel fails here.
"""
import copy

import pytest
import torch

from vsa_lm_b200 import AnchorKV8, Bolt3Decoder, Bolt3LayerState
from vsa_lm_b200.model import Bolt3LM
from vsa_lm_b200.workloads import MODEL_SHAPES, make_model_params


def _decoder(shape="tiny_lm", **kw):
    mcfg = dict(MODEL_SHAPES[shape])
    model = Bolt3LM(**mcfg)
    model.load_state_dict(make_model_params(mcfg, 0), strict=True)
    return mcfg, Bolt3Decoder(model.to(device="cuda", dtype=torch.bfloat16).eval(), kv_cache="int8", **kw)


def _ids(mcfg, B, T, seed=1):
    return torch.randint(0, mcfg["vocab_size"], (B, T), generator=torch.Generator().manual_seed(seed)).cuda()


def _anchor(kv):
    return next(c for c in kv if isinstance(c, AnchorKV8))


def _fail_prefill(dec, kind):
    """dec.prefill as if a kernel of the prompt's last slice had reported an expired wait."""
    real = dec.prefill

    def prefill(ids, **kw):
        h, states, kv = real(ids, **kw)
        next(c for c in kv if isinstance(c, kind)).status.word.fill_(2)
        return h, states, kv

    dec.prefill = prefill


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [AnchorKV8, Bolt3LayerState])
def test_beam_search_reports_errors_of_its_prompt(kind):
    mcfg, dec = _decoder()
    ids = _ids(mcfg, 1, 40)
    dec.beam_search(ids, 2, 3)
    _fail_prefill(dec, kind)
    with pytest.raises(RuntimeError, match="bounded wait"):
        dec.beam_search(ids, 2, 3)


@pytest.mark.gpu
@pytest.mark.parametrize("graphs", [True, False])
@pytest.mark.parametrize("call", ["generate_batch", "generate", "continue_generate"])
def test_generation_reports_errors_of_the_anchors(call, graphs):
    """The last tokens' too: fewer than a chunk are generated."""
    mcfg, dec = _decoder(cuda_graphs=graphs)
    ids = _ids(mcfg, 1, 40)
    if call == "continue_generate":
        _, states, kv = dec.prefill(ids)
        more = _ids(mcfg, 1, 5, 2)
        _, states, kv, pos = dec.continue_generate(more, states, kv, 40, 3)
        _anchor(kv).status.word.fill_(2)
        with pytest.raises(RuntimeError, match="bounded wait"):
            dec.continue_generate(more, states, kv, pos, 3)
        return
    getattr(dec, call)(ids, 3, temperature=0.0)
    _fail_prefill(dec, AnchorKV8)
    with pytest.raises(RuntimeError, match="bounded wait"):
        getattr(dec, call)(ids, 3, temperature=0.0)


@pytest.mark.gpu
@pytest.mark.parametrize("graphs", [True, False])
def test_steps_report_errors_of_the_anchors(graphs):
    """A caller's own loop of steps hears of an error within two chunks of tokens."""
    mcfg, dec = _decoder()
    ids = _ids(mcfg, 2, 40)
    h, states, kv = dec.prefill(ids)
    runner = dec.step_graph(states, kv) if graphs else None
    tok = _ids(mcfg, 2, 1, 3)

    def step(i):
        runner.step(tok, 40 + i) if graphs else dec.step(tok, 40 + i, states, kv)

    for i in range(10):
        step(i)
    _anchor(kv).status.word.fill_(2)
    with pytest.raises(RuntimeError, match="bounded wait"):
        for i in range(10, 10 + 2 * dec.C):
            step(i)
    if runner is not None:
        runner.close()


@pytest.mark.gpu
def test_prompt_slices_report_errors_of_the_anchors():
    mcfg, dec = _decoder()
    _, states, kv = dec.prefill(_ids(mcfg, 1, 128))
    _anchor(kv).status.word.fill_(8)
    more = _ids(mcfg, 1, 128, 4)
    with pytest.raises(RuntimeError, match="outside the range"):
        for i in range(3):
            dec.step(more, 128 * (i + 1), states, kv)


@pytest.mark.gpu
def test_copied_states_keep_their_errors():
    mcfg, dec = _decoder()
    _, states, kv = dec.prefill(_ids(mcfg, 1, 150))       # past a chunk: a status copy is under way
    clean = copy.deepcopy(_anchor(kv))
    _anchor(kv).status.word.fill_(2)
    spoiled = copy.deepcopy(_anchor(kv))
    clean.check_status()
    for c in (spoiled, _anchor(kv)):
        with pytest.raises(RuntimeError, match="bounded wait"):
            c.check_status()


@pytest.mark.gpu
def test_beam_search_pads_with_the_first_of_its_ids():
    mcfg, dec = _decoder()
    ids = _ids(mcfg, 1, 40)
    h, _, _ = dec.prefill(ids)
    best = int(dec.model.lm_head(h[:, -1]).argmax())
    first = best + 1 if best + 1 < mcfg["vocab_size"] else best - 1
    for eos in ((max(best, first), min(best, first)), [min(best, first), max(best, first)]):
        toks, _, lengths = dec.beam_search(ids, 1, 20, eos_ids=eos)
        end = int(lengths[0, 0])
        assert end < toks.shape[2] and int(toks[0, 0, end - 1]) in eos and bool((toks[0, 0, end:] == eos[0]).all())
    toks, _, lengths = dec.beam_search(ids, 1, 20, eos_ids={best, first})       # a set has no first: the lowest
    assert bool((toks[0, 0, int(lengths[0, 0]):] == min(best, first)).all())


def test_models_that_8_bit_caches_cannot_serve_are_refused_at_once():
    def model(**kw):
        cfg = dict(vocab_size=32, dim=64, num_layers=1, num_heads=2, num_kv_heads=1, head_dim=64, intermediate=64,
                   layer_types=["softmax"])
        return Bolt3LM(**{**cfg, **kw})

    Bolt3Decoder(model(), kv_cache="int8")
    Bolt3Decoder.blank_state(model(num_heads=16), 1, "cpu", kv_cache="int8")
    for bad in (model(head_dim=32), model(head_dim=96), model(num_heads=17), model(num_heads=34, num_kv_heads=2)):
        Bolt3Decoder(bad)                                        # bf16 caches hold them
        Bolt3Decoder.blank_state(bad, 1, "cpu")
        with pytest.raises(ValueError, match="8-bit"):
            Bolt3Decoder(bad, kv_cache="int8")
        with pytest.raises(ValueError, match="8-bit"):
            Bolt3Decoder.blank_state(bad, 1, "cpu", kv_cache="int8")


def test_scales_of_rows_without_a_token_are_zero():
    """Whatever the memory held: torch fills new memory with NaN here."""
    torch.use_deterministic_algorithms(True)
    try:
        assert torch.utils.deterministic.fill_uninitialized_memory and bool(torch.empty(3).isnan().all())
        c = AnchorKV8(2, 3, 100, 64, "cpu")
        assert bool((c.scale == 0).all())
        c.scale.uniform_()
        c.n = 250
        c.reserve(7)
        assert c.capacity == 512 and bool((c.scale[:, :, :, 250:] == 0).all())
        assert torch.equal(c.repeated(2).scale[:, 3], c.scale[:, 1])
    finally:
        torch.use_deterministic_algorithms(False)


def _edit(model, how, factor):
    for blk in model.blocks:
        if not hasattr(blk, "vsa"):
            for norm in (blk.attn.q_norm, blk.attn.k_norm):
                w = norm.weight
                if how == "data":
                    w.data.mul_(factor)                       # no version of the parameter changes
                elif how == "in place":
                    with torch.no_grad():
                        w.mul_(factor)
                else:
                    norm.weight = torch.nn.Parameter(w.detach() * factor)


@pytest.mark.gpu
@pytest.mark.parametrize("how,graphs", [("data", True), ("data", False), ("in place", True), ("in place", False),
                                        ("replaced", False)])
def test_edited_norm_weights_are_used_at_once(how, graphs):
    """An edit between two steps, in eager steps and (edits that keep the parameter's memory) in a captured graph."""
    mcfg, dec = _decoder("small_lm")
    ids, tok = _ids(mcfg, 1, 130), _ids(mcfg, 1, 1, 2)

    def run(factor_before, factor_between):
        _, states, kv = dec.prefill(ids)
        runner = dec.step_graph(states, kv) if graphs else None
        step = lambda i: runner.step(tok, 130 + i) if graphs else dec.step(tok, 130 + i, states, kv)
        _edit(dec.model, how, factor_before)
        step(0)
        _edit(dec.model, how, factor_between)
        step(1)
        c = _anchor(kv)
        rows = [t[:, :, :, 130:132].clone() for t in (c.data, c.scale)]
        _edit(dec.model, how, 1.0 / (factor_before * factor_between))
        if runner is not None:
            runner.close()
        return rows

    plain, edited = run(1.0, 1.0), run(1.0, 2.0)
    for a, b in zip(plain, edited):
        assert torch.equal(a[..., 0, :] if a.dim() == 5 else a[..., 0], b[..., 0, :] if b.dim() == 5 else b[..., 0])
    # twice the weights: the key's scale doubles, exactly
    assert torch.equal(edited[1][0, ..., 1], 2 * plain[1][0, ..., 1]) and torch.equal(edited[0], plain[0])
