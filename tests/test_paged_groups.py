"""Records of paged attention where a head has more query rows than the record kernel's CTA holds at once (512): they come in
groups, one after another, over the same keys. Against 64 bits, and the same bits at every call. Tolerances as derived in
test_paged.py; a record sums up to T * G terms, at most (64 + 4 + groups) 2^-24 of it in roundings, less than the n 2^-23
that is there for the softmax's sum.
"""
import pytest
import torch

from test_paged import new_pages, put_rows, randn, ref_attend, rounded_within, same
from vsa_lm_b200 import AnchorKVPaged
from vsa_lm_b200 import kernels as K
from vsa_lm_b200.model import SoftmaxAttn


def _inputs(B, T, H, HKV, HD, page, n, lens=None, seed=200):
    pages, table = new_pages(seed, B, HKV, HD, page, n + T)
    for b in range(B):
        m = (n if lens is None else lens[b]) + T
        for h in range(HKV):
            if m >= T:
                put_rows(pages, table, b, h, randn(seed + 1 + 31 * b + h, 2, m, HD, dtype=torch.bfloat16))
    return pages, table, randn(seed + 1000, B, T, H, HD, dtype=torch.bfloat16)


GROUPS = [
    # B, T, H, HKV, HD, page, n, lens
    (1, 128, 5, 1, 64, 64, 128, None),                   # 640 rows: a second group of one tile; a block of keys to a CTA
    (2, 128, 14, 2, 128, 32, 200, None),                 # 7 query heads: 896 rows, the second group one tile short
    (2, 128, 16, 2, 64, 64, 300, (300, 17)),             # 8 of them: two whole groups
    (1, 128, 16, 1, 128, 64, 500, None),                 # 16: four groups
    (1, 128, 7, 1, 64, 16, 9000, None),                  # several blocks of keys to a CTA
    (1, 128, 8, 1, 128, 128, 9000, None),
    (1, 128, 16, 1, 64, 64, 6000, None),
    (1, 67, 16, 1, 128, 64, 5001, None),                 # 1072 rows: the third group a part of a tile
    (40, 90, 12, 2, 64, 32, 400, None),                  # more heads than half the machine: all blocks of a head to a CTA
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", GROUPS)
def test_records_of_several_groups_match_64_bits(case):
    B, T, H, HKV, HD, page, n, lens = case
    L = lens or (n,) * B
    pages, table, q = _inputs(B, T, H, HKV, HD, page, n, lens)
    y, mass, err, rec, rec_err = ref_attend(q, pages, table, L, HD ** -0.5, HKV)
    before = torch.rand(B, HKV, table.shape[1] * page, generator=torch.Generator().manual_seed(7))
    weight = before.cuda()
    status = K.DeviceStatus("cuda")
    got = K.paged_attend(q=q.cuda(), pages=pages.cuda(), table=table.cuda(), n=n, weight=weight, status=status,
                         lens=torch.tensor(lens, dtype=torch.int32).cuda() if lens else None).cpu().view(B, T, H, HD)
    assert int(status.word) == 0
    assert rounded_within(got, y, mass * (2 * (err + 2 ** -9 + 2 ** -21) + (n + T) * 2 ** -23))
    want = before.double() + rec
    assert bool(((weight.cpu().double() - want).abs() <= rec_err + 2 ** -23 * want * (rec > 0)).all())
    assert same(weight.cpu()[rec == 0], before[rec == 0])


@pytest.mark.gpu
@pytest.mark.parametrize("HD", [64, 128])
@pytest.mark.parametrize("B,G,n", [(4, 8, 700), (2, 16, 333), (20, 7, 450), (1, 8, 9000)])
def test_records_of_several_groups_have_the_same_bits_at_every_call(HD, B, G, n):
    T, HKV, page = 128, 4, 64
    pages, table, q = _inputs(B, T, G * HKV, HKV, HD, page, n)
    pages, table, q = pages.cuda(), table.cuda(), q.cuda()
    first = None
    for _ in range(100):
        weight = torch.zeros(B, HKV, table.shape[1] * page, device="cuda")
        y = K.paged_attend(q=q, pages=pages, table=table, n=n, weight=weight)
        first = first or (y, weight)
        assert torch.equal(y, first[0]) and torch.equal(weight, first[1])
    # every query row gives one in all
    assert float((first[1].double().sum(-1) - T * G).abs().max()) <= T * G * (n + T) * 2 ** -22


@pytest.mark.gpu
@pytest.mark.parametrize("heads,HKV,HD", [(8, 1, 64), (16, 1, 128), (14, 2, 64)])
def test_a_layers_records_of_prompt_slices(heads, HKV, HD):
    """Slices through AnchorKVPaged.attention with a budget that is not reached: the records grow by what 64 bits give for the
    same queries and rows."""
    torch.manual_seed(5)
    ly = SoftmaxAttn(dict(dim=256, num_heads=heads, num_kv_heads=HKV, head_dim=HD, rope_theta=1e4, eps=1e-6, qk_norm=True))
    ly = ly.to(device="cuda", dtype=torch.bfloat16).eval()
    B, cache, pos = 2, AnchorKVPaged(2, HKV, 600, HD, "cuda", page=32, budget=5000), 0
    kept = {}
    real = K.paged_append

    def append(**kw):
        kept["q"] = real(**kw)
        kept["before"] = kw["weight"].clone()
        return kept["q"]

    with torch.no_grad(), pytest.MonkeyPatch.context() as m:
        m.setattr(K, "paged_append", append)
        for t in (128, 128, 75, 1, 128):
            h = torch.randn(B, t, 256, device="cuda").bfloat16()
            n = cache.n
            cache.attention(ly, h, pos)
            _, _, _, rec, rec_err = ref_attend(kept["q"].cpu(), cache.pages.cpu(), cache.table.cpu(), [n] * B, HD ** -0.5, HKV)
            want = kept["before"].cpu().double() + rec
            got = cache.weight.cpu().double()
            assert bool(((got - want).abs() <= rec_err + 2 ** -23 * want * (rec > 0))[..., :n + t].all())
            pos += t
    cache.check_status()
