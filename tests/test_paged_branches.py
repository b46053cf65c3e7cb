"""The paged cache's kernels at the sizes that choose among their forms: evictions of more heads than the machine holds large
blocks of, lists of moves that do not fit shared memory, prompt slices over dozens of splits of the keys. The comparisons are
those of test_paged.py."""
import pytest
import torch

import test_paged as paged
from vsa_lm_b200 import AnchorKVPaged, Bolt3Decoder
from vsa_lm_b200.model import Bolt3LM
from vsa_lm_b200.workloads import MODEL_SHAPES, make_model_params


def _lens(B, *rows):
    return tuple(rows[b % len(rows)] for b in range(B))


EVICT = [
    # B, HKV, HD, page, n, keep, recent, lens, weights
    (300, 1, 64, 16, 400, 200, 32, None, "random"),                  # small blocks: more than 296 heads
    (150, 2, 128, 64, 300, 200, 60, _lens(150, 300, -1, 200, 201, 0), "few"),
    (75, 4, 64, 128, 500, 40, 40, _lens(75, 500, 499, 41), "odd"),
    (300, 1, 128, 32, 2100, 1030, 64, _lens(300, 2100, 900, 1031, -1), "random"),   # and moves listed in the workspace
    (148, 1, 128, 16, 2100, 1040, 64, None, "random"),               # listed in the workspace, moved by the head's own block
    (148, 1, 64, 64, 4200, 1030, 100, _lens(148, 4200, 1029, 2000), "few"),   # the same, blocks of 1024 threads
    (149, 1, 64, 64, 4200, 1030, 100, _lens(149, 4200, 1029, 2000), "few"),   # one head more: blocks of 512
    (75, 2, 64, 128, 10300, 10200, 900, _lens(75, 10300, 10201, 500), "random"),   # of 1024 again
    (147, 1, 64, 64, 2100, 1040, 64, _lens(147, 2100, 5, 1041), "random"),    # one head less: moved by a kernel of its own
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", EVICT)
def test_evictions_of_many_heads(case):
    paged.test_evict_matches_its_definition(case)


ATTEND = [
    # B, T, H, HKV, HD, page, n, lens
    (1, 30, 16, 1, 128, 64, 20000, None),                            # 53 splits
    (1, 30, 16, 1, 64, 32, 9000, None),                              # 71 splits of a block each
    (2, 30, 16, 1, 128, 128, 9000, (9000, 40)),                      # 36 splits, most of them empty for the short sequence
    (1, 20, 4, 1, 64, 16, 18000, None),                              # one tile of rows
]


@pytest.mark.gpu
@pytest.mark.parametrize("weigh", [False, True])
@pytest.mark.parametrize("case", ATTEND)
def test_prompt_slices_over_many_splits(case, weigh):
    paged.test_attend_matches_64_bits(case, weigh)


@pytest.mark.gpu
@pytest.mark.parametrize("graphs", [True, False])
@pytest.mark.parametrize("shape,page,T", [("small_lm", 16, 70), ("tiny_lm", 32, 150)])
def test_beams_that_share_pages_are_beams_with_pages_of_their_own(shape, page, T, graphs):
    """The same search with every page copied for every beam, at the start and at every reordering: the same tokens and scores,
    bit for bit."""
    mcfg = dict(MODEL_SHAPES[shape])
    model = Bolt3LM(**mcfg)
    model.load_state_dict(make_model_params(mcfg, 0), strict=True)
    model = model.to(device="cuda", dtype=torch.bfloat16).eval()
    dec = Bolt3Decoder(model, kv_cache="paged", kv_page=page, cuda_graphs=graphs)
    ids = torch.randint(0, mcfg["vocab_size"], (2, T), generator=torch.Generator().manual_seed(1)).cuda()
    shared = dec.beam_search(ids, 4, 40)
    real, moved = AnchorKVPaged.repeated, []

    def repeated(self, times):
        self.budget = 1                                              # a bounded cache shares no page
        new = real(self, times)
        self.budget = new.budget = None
        assert len(set(new.table.flatten().tolist())) == new.table.numel()
        return new

    def reorder(self, parent):
        groups, beams = parent.shape
        src = (parent.long() + torch.arange(groups, device=parent.device)[:, None] * beams).view(-1)
        moved.append(bool((src != torch.arange(groups * beams, device=src.device)).any()))
        self.pages[:, self.own.view(-1).long()] = self.pages[:, self.own[src].view(-1).long()]

    with pytest.MonkeyPatch.context() as m:
        m.setattr(AnchorKVPaged, "repeated", repeated)
        m.setattr(AnchorKVPaged, "reorder", reorder)
        own = dec.beam_search(ids, 4, 40)
    assert sum(moved) > 1
    assert all(torch.equal(a, b) for a, b in zip(shared, own))
