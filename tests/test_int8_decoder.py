"""A decoder with 8-bit anchor caches: errors that its kernels report on the device reach the caller.

The errors are made on the host: a status word is set as a kernel would set it. No kernel fails here.
"""
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
