"""8-bit anchor caches and beam search on models that are split by KV head.

A shard's cache holds its own KV heads' rows, bit for bit those of the whole layer's cache: rows are normed, rotated
and quantised head by head. The shards' fp32 partial outputs sum to the whole layer's output but for the roundings
of that one to bf16 and of its sums' order.
"""
import pytest
import torch

from vsa_lm_b200 import AnchorKV8, Bolt3Decoder
from vsa_lm_b200.model import Bolt3LM, SoftmaxAttn
from vsa_lm_b200.tp import Bolt3DecoderTP, Bolt3LMTP, shard_softmax_attn
from vsa_lm_b200.workloads import MODEL_SHAPES, make_model_params


@pytest.mark.gpu
@pytest.mark.parametrize("world,qk_norm", [(2, True), (4, False)])
def test_shards_of_an_anchor_over_int8_caches(world, qk_norm):
    torch.manual_seed(1)
    cfg = dict(dim=512, num_heads=16, num_kv_heads=4, head_dim=128, rope_theta=1e4, eps=1e-6, qk_norm=qk_norm)
    attn = SoftmaxAttn(cfg).to(device="cuda", dtype=torch.bfloat16).eval()
    shards = [shard_softmax_attn(attn, r, world) for r in range(world)]
    B, cache = 2, AnchorKV8(2, 4, 300, 128, "cuda")
    caches = [AnchorKV8(B, s.HKV, 300, s.HD, "cuda") for s in shards]
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
    assert torch.equal(torch.cat([c.data[:, :, :, :pos] for c in caches], 2), cache.data[:, :, :, :pos])
    assert torch.equal(torch.cat([c.scale[:, :, :, :pos] for c in caches], 2), cache.scale[:, :, :, :pos])


@pytest.mark.gpu
def test_beam_search_on_a_tensor_parallel_decoder():
    """One rank, no process group: the split model's own step, whose partial sums are rounded once."""
    mcfg = dict(MODEL_SHAPES["small_lm"])
    model = Bolt3LM(**mcfg)
    model.load_state_dict(make_model_params(mcfg, 0), strict=True)
    model = model.to(device="cuda", dtype=torch.bfloat16).eval()
    dec = Bolt3DecoderTP(Bolt3LMTP(model), kv_cache="int8")
    ids = torch.randint(0, mcfg["vocab_size"], (2, 150), generator=torch.Generator().manual_seed(1)).cuda()
    h, states, kv = dec.prefill(ids)
    assert any(isinstance(c, AnchorKV8) for c in kv)
    ref, _, _ = Bolt3Decoder(model, kv_cache="int8").prefill(ids)
    assert bool(((h.float() - ref.float()).abs() <= 0.05 * ref.float().pow(2).mean().sqrt()).all())
    toks, scores, lengths = dec.beam_search(ids, 3, 12)
    assert toks.shape == (2, 3, 12) and bool((scores[:, :-1] >= scores[:, 1:]).all()) and bool(scores.isfinite().all())
    best = torch.log_softmax(dec.model.lm_head(h[:, -1]).double(), -1)
    first = dec.beam_search(ids, 1, 1)[0][:, 0, 0]
    assert bool((best.gather(1, first[:, None])[:, 0] >= best.amax(-1) - 1e-6).all())
