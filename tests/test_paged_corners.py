"""Corners of the paged cache's records and eviction: weights too small to hold, zeros of either sign, outputs in the queries' place.
Tolerances as derived in test_paged.py."""
import pytest
import torch

from test_paged import new_pages, put_rows, randn, ref_attend, ref_evict, same
from vsa_lm_b200 import kernels as K


@pytest.mark.gpu
@pytest.mark.parametrize("HD", [64, 128])
@pytest.mark.parametrize("T", [1, 3, 40, 61, 150])
def test_a_key_without_weight_has_a_record_of_zero(T, HD):
    """Keys whose every weight is below 2^-150 (0 in fp32): their records stay as they were, to the bit, whatever the number of
    query rows; and an eviction by such records keeps the lowest rows."""
    B, H, HKV, page, n = 2, 8, 2, 32, 333
    pages, table = new_pages(300, B, HKV, HD, page, n + T)
    q = randn(301, B, T, H, HD, dtype=torch.bfloat16)
    q[..., 0] = 40.0
    heavy = 5
    for b in range(B):
        for h in range(HKV):
            kv = randn(302 + 2 * b + h, 2, n + T, HD)
            kv[0, :, 0] = -HD ** 0.5 * 2                  # every score about -80, and 80 at the heavy row: 2^-230 of its weight
            kv[0, heavy, 0] = HD ** 0.5 * 2
            put_rows(pages, table, b, h, kv.to(torch.bfloat16))
    _, _, _, rec, _ = ref_attend(q, pages, table, [n] * B, HD ** -0.5, HKV)
    light = rec < 2.0 ** -160
    assert light[..., :heavy].all() and light[..., heavy + 1:].all() and (rec[..., heavy] > 0.99 * T * H // HKV).all()
    gp, gt = pages.cuda(), table.cuda()
    weight = torch.zeros(B, HKV, table.shape[1] * page, device="cuda")
    K.paged_attend(q=q.cuda(), pages=gp, table=gt, n=n, weight=weight)
    assert bool((weight.cpu()[light] == 0).all())
    order = torch.arange(weight.shape[-1], dtype=torch.int32, device="cuda").expand_as(weight).contiguous()
    K.paged_evict(pages=gp, table=gt, weight=weight, order=order, n=n + T, keep=100, recent=0)
    assert bool((order[..., :100].cpu() == torch.arange(100)).all())


@pytest.mark.gpu
@pytest.mark.parametrize("n,keep", [(500, 100), (5000, 3000), (20000, 600)])
def test_zeros_of_either_sign_are_equal_weights(n, keep):
    """Ties go to the lowest row, the signs of zeros notwithstanding; what moves keeps its bits."""
    B, HKV, HD, page = 2, 2, 64, 64
    pages, table = new_pages(310, B, HKV, HD, page, n, poison=0.0)
    pages.view(torch.int16).random_(-2 ** 15, 2 ** 15, generator=torch.Generator().manual_seed(311))
    g = torch.Generator().manual_seed(312)
    shape = (B, HKV, table.shape[1] * page)
    weight = torch.where(torch.rand(shape, generator=g) < 0.5, -0.0, 0.0)
    weight = torch.where(torch.rand(shape, generator=g) < 0.01, torch.rand(shape, generator=g), weight)
    weight[1] = -weight[1]
    order = torch.stack([torch.randperm(shape[-1], generator=g) for _ in range(B * HKV)]).view(shape).int()
    gp, gw, go = pages.cuda(), weight.cuda(), order.cuda()
    K.paged_evict(pages=gp, table=table.cuda(), weight=gw, order=go, n=n, keep=keep, recent=keep // 5)
    ref_evict(pages, table, weight, order, [n] * B, keep, keep // 5)
    assert same(gw.cpu(), weight) and torch.equal(go.cpu(), order) and same(gp.cpu(), pages)


@pytest.mark.gpu
@pytest.mark.parametrize("HD", [64, 128])
@pytest.mark.parametrize("B,T,H,HKV,n,weigh", [
    (2, 1, 8, 2, 100, True),                              # a CTA per head
    (1, 4, 16, 4, 5000, True),                            # runs of several warps, joined
    (160, 1, 4, 1, 333, True),                            # whole heads by a warp
    (2, 37, 8, 2, 100, False),                            # many rows
    (1, 64, 8, 1, 9000, False),                           # and splits of the keys
])
def test_outputs_in_the_place_of_their_queries(HD, B, T, H, HKV, n, weigh):
    pages, table = (x.cuda() for x in new_pages(320, B, HKV, HD, 32, n + T, poison=0.0))
    pages.copy_(randn(321, *pages.shape, dtype=torch.bfloat16))
    q = randn(322, B, T, H, HD, dtype=torch.bfloat16).cuda()
    weight = [torch.zeros(B, HKV, table.shape[1] * 32, device="cuda") if weigh else None for _ in range(2)]
    y = K.paged_attend(q=q, pages=pages, table=table, n=n, weight=weight[0])
    K.paged_attend(q=q, pages=pages, table=table, n=n, weight=weight[1], y=q)
    assert torch.equal(q.view(B, T, H * HD), y)
    assert not weigh or torch.equal(*weight)
