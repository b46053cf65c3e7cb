"""The paged KV cache of a softmax anchor: bolt3_paged_append, bolt3_paged_attend (with and without its record of weights) and
bolt3_paged_evict against plain implementations in 64 bits.

Tolerances, from the arithmetic of include/bolt3.h:
- a bf16 result is rounded once, and rounding is monotone: it lies between the rounded ends of the interval in which
  the value before it may lie (`rounded_within`);
- a norm and a rotation in fp32 are off by a few 2^-24 of the row's largest value, 2e-6 of it here;
- a score t (base 2) is off by HD roundings of the products' absolute sum, times 2 for the tensor cores' truncation,
  and by a few roundings of itself and of the reference it is measured from: 2^-22 (|t| + |reference|). An error d of
  a score changes its weight by a factor of 2^d;
- a weight in the product with the values is two bf16 terms, 2^-17 of it, up to 16 query rows per KV head; one, 2^-9,
  above; ex2 is off by 2^-22; a sum of N terms by N 2^-24.
"""
import math

import pytest
import torch

from vsa_lm_b200 import kernels as K


def randn(seed, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def rounded_within(y, ref, tol):
    """Whether the bf16 `y` is the rounding of a number within `tol` of the 64-bit `ref`. (The ends are
    widened by the fp32 step on the way to bf16.)"""
    tol = tol + 2 ** -23 * ref.abs() + 1e-37
    lo, hi = ((ref + d).float().to(torch.bfloat16).double() for d in (-tol, tol))
    return bool(((y.double() >= lo) & (y.double() <= hi)).all())


def same(a, b):
    """Equal bit for bit (NaN included)."""
    view = {2: torch.int16, 4: torch.int32}[a.element_size()]
    return bool(torch.equal(a.view(view), b.view(view)))


def new_pages(seed, B, HKV, HD, page, rows, spare=2, poison=float("nan")):
    """A pool full of poison, and a table: pages in no order, entries behind what `rows` rows need far out of the pool."""
    W = -(-rows // page)
    P = B * W + spare
    g = torch.Generator().manual_seed(seed)
    table = torch.randperm(P, generator=g)[:B * W].view(B, W).to(torch.int32)
    table = torch.cat((table, torch.full((B, 2), 2 ** 30, dtype=torch.int32)), 1)
    return torch.full((2, P, HKV, page, HD), poison, dtype=torch.bfloat16), table


def rows_of(pages, table, b, h, n):
    """Keys and values [2, n, HD] of the first n rows of a head."""
    page = pages.shape[3]
    r = torch.arange(n)
    return pages[:, table[b].long()[r // page], h, r % page]


def put_rows(pages, table, b, h, kv):
    page = pages.shape[3]
    r = torch.arange(kv.shape[1])
    pages[:, table[b].long()[r // page], h, r % page] = kv


# ------------------------------------------------------------------------------------------- append

APPEND = [
    # B, T, H, HKV, HD, page, n, norm, rope, lens, far
    (1, 1, 4, 2, 64, 16, 0, True, True, None, 0),
    (3, 1, 32, 8, 128, 64, 700, True, True, None, 100000),
    (2, 5, 15, 5, 64, 16, 13, False, True, None, 0),
    (3, 37, 7, 1, 64, 32, 263, True, True, (0, 263, -1), 2 ** 24 + 12345),
    (2, 130, 4, 4, 128, 128, 10, True, False, None, 5),
    (4, 2, 1, 1, 128, 16, 14, False, False, (14, 0, -1, 3), 0),
    (9, 128, 12, 2, 128, 32, 128, True, True, None, 0),
]


@pytest.mark.gpu
@pytest.mark.parametrize("records", [False, True])
@pytest.mark.parametrize("case", APPEND)
def test_append_matches_64_bits(case, records):
    B, T, H, HKV, HD, page, n, norm, rope, lens, far = case
    proj = randn(1, B, T, (H + 2 * HKV) * HD + 8, dtype=torch.bfloat16)
    cut = (8, 8 + H * HD, 8 + (H + HKV) * HD, 8 + (H + 2 * HKV) * HD)
    q, k, v = (proj[..., a:b] for a, b in zip(cut, cut[1:]))
    qw = 1 + 0.2 * randn(2, HD) if norm else None
    kw = 1 + 0.2 * randn(3, HD) if norm else None
    inv = 1e4 ** (-torch.arange(0, HD, 2).float() / HD) if rope else None
    L = torch.tensor(lens if lens else [n] * B)
    own_pos = bool(lens) and records                      # positions per sequence, else pos0 + lens - n
    pos0 = n + far
    start = torch.tensor([far + 3 * b for b in range(B)]) if own_pos else pos0 + (L - n)
    pos = start[:, None] + torch.arange(T)
    pages, table = new_pages(4, B, HKV, HD, page, n + T)
    want = pages.clone()
    cap = table.shape[1] * page
    weight = torch.full((B, HKV, cap), 7.0)
    order = torch.full((B, HKV, cap), -5, dtype=torch.int32)
    cu = lambda t: None if t is None else t.cuda()
    g, gp, gw, go = proj.cuda(), pages.cuda(), weight.cuda(), order.cuda()
    gq, gk, gv = (g[..., a:b] for a, b in zip(cut, cut[1:]))
    status = K.DeviceStatus("cuda")
    q_out = K.paged_append(q=gq, k=gk, v=gv, pages=gp, table=table.cuda(), n=n, pos0=pos0, inv_freq=cu(inv), q_norm=cu(qw),
                           k_norm=cu(kw), eps=1e-5, lens=cu(L.int()) if lens else None,
                           pos=start.int().cuda() if own_pos else None, weight=gw if records else None,
                           order=go if records else None, status=status).cpu()
    assert int(status.word) == 0

    def ref(x, w):
        x = x.double().reshape(B, T, -1, HD)
        if w is not None:
            x = x / (x.pow(2).mean(-1, keepdim=True) + 1e-5).sqrt() * w.double()
        if inv is not None:
            ang = (pos.double()[..., None] * inv.double())[:, :, None]
            c, s, a, b = ang.cos(), ang.sin(), x[..., :HD // 2], x[..., HD // 2:]
            x = torch.cat((a * c - b * s, b * c + a * s), -1)
        return x

    rq, rk = ref(q, qw), ref(k, kw)
    got = gp.cpu()
    for b in range(B):
        if L[b] < 0:
            assert bool((q_out[b] == 0).all())
            continue
        assert rounded_within(q_out[b], rq[b], 2e-6 * rq[b].abs().amax(-1, keepdim=True))
        r = torch.arange(int(L[b]), int(L[b]) + T)
        at = table[b].long()[r // page]
        assert rounded_within(got[0, at, :, r % page], rk[b], 2e-6 * rk[b].abs().amax(-1, keepdim=True))
        want[0, at, :, r % page] = got[0, at, :, r % page]
        want[1, at, :, r % page] = v[b].reshape(T, HKV, HD)
        if records:
            weight[b, :, r] = 0
            order[b, :, r] = pos[b].int()
    assert same(got, want)                                # values as they came, all other rows as they were
    assert torch.equal(gw.cpu(), weight) and torch.equal(go.cpu(), order)


# ------------------------------------------------------------------------------------------- attend

def ref_attend(q, pages, table, L, scale, HKV):
    """64-bit outputs [B, T, H, HD], records [B, HKV, cap], and what their tolerances need."""
    B, T, H, HD = q.shape
    G, cap = H // HKV, table.shape[1] * pages.shape[3]
    y, mass = torch.zeros(B, T, H, HD, dtype=torch.double), torch.zeros(B, T, H, HD, dtype=torch.double)
    err = torch.zeros(B, T, H, 1, dtype=torch.double)
    rec, rec_err = torch.zeros(B, HKV, cap, dtype=torch.double), torch.zeros(B, HKV, cap, dtype=torch.double)
    for b in range(B):
        if L[b] < 0:
            continue
        n = int(L[b]) + T
        late = torch.ones(T, n, dtype=torch.bool).triu(int(L[b]) + 1)
        for h in range(HKV):
            k, v = rows_of(pages, table, b, h, n).double()
            x = q[b, :, h * G:(h + 1) * G].double().transpose(0, 1)              # [G, T, HD]
            t = (x @ k.t()) * scale
            t = t.masked_fill(late, -math.inf)
            p = torch.softmax(t, -1)
            e = (x.abs() @ k.abs().t()) * (scale * HD * 2 ** -23) + t.abs().nan_to_num(posinf=0.0) * 2 ** -22
            e = e.masked_fill(late, 0).amax(-1, keepdim=True) + t.amax(-1, keepdim=True).abs() * 2 ** -22
            y[b, :, h * G:(h + 1) * G] = (p @ v).transpose(0, 1)
            mass[b, :, h * G:(h + 1) * G] = (p @ v.abs()).transpose(0, 1)
            err[b, :, h * G:(h + 1) * G] = e.transpose(0, 1)
            rec[b, h, :n] = p.sum((0, 1))
            rec_err[b, h, :n] = (p * (2 * e + 2 ** -21 + n * 2 ** -23)).sum((0, 1))
    return y, mass, err, rec, rec_err


ATTEND = [
    # B, T, H, HKV, HD, page, n, lens
    (1, 1, 4, 2, 64, 16, 0, None),                       # a first token sees itself alone
    (1, 1, 15, 5, 64, 16, 332, None),                    # a CTA per head
    (3, 1, 7, 1, 64, 32, 700, (0, 699, -1)),             # odd rows, an idle sequence
    (2, 1, 32, 2, 128, 64, 31, None),                    # 16 rows to a head, a block to the row
    (1, 1, 16, 1, 128, 128, 5000, None),                 # runs over one head, 16 rows
    (40, 1, 32, 8, 128, 16, 100, None),                  # more heads than CTAs
    (5, 1, 32, 8, 128, 64, 900, (900, 0, -1, 63, 64)),   # runs over ragged sequences
    (2, 3, 15, 5, 64, 16, 45, (45, -1)),                 # a few tokens, causal among themselves
    (2, 7, 16, 4, 128, 32, 1000, (3, 1000)),             # two column tiles
    (1, 2, 16, 1, 128, 16, 2500, None),                  # 32 rows over runs
    (1, 16, 5, 5, 64, 16, 100, None),                    # 16 rows of as many tokens
    (1, 17, 5, 5, 64, 32, 100, None),                    # the fewest of many rows
    (12, 1, 32, 8, 128, 64, 2500, None),                 # a CTA per head, most of the machine
    (8, 1, 16, 8, 64, 64, 4200, None),                   # longer: its records apart
    (8, 1, 32, 8, 64, 64, 2500, (2500, 3, 0, -1, 64, 63, 65, 1)),   # the same ragged: runs
    (2, 1, 7, 1, 64, 64, 20000, (20000, 5)),             # hundreds of partial sums of a head
    (1, 1, 16, 1, 128, 32, 20000, None),
    (2, 33, 4, 4, 64, 16, 0, None),                      # many rows: a prompt from its start
    (3, 40, 4, 2, 128, 64, 500, (500, 0, -1)),           # one tile of rows, a ragged batch
    (1, 128, 8, 2, 128, 128, 130, None),                 # two tiles
    (2, 128, 32, 8, 64, 32, 77, (77, 1)),                # pages inside a block
    (1, 100, 7, 1, 64, 16, 3000, None),                  # keys split over CTAs
    (1, 300, 12, 2, 128, 64, 200, None),                 # more than one CTA of rows, several groups of 512
    (1, 160, 16, 1, 128, 32, 1500, None),                # 2560 rows: groups over split keys
]


@pytest.mark.gpu
@pytest.mark.parametrize("weigh", [False, True])
@pytest.mark.parametrize("case", ATTEND)
def test_attend_matches_64_bits(case, weigh):
    B, T, H, HKV, HD, page, n, lens = case
    L = lens if lens else [n] * B
    pages, table = new_pages(5, B, HKV, HD, page, n + T)
    for b in range(B):
        if L[b] >= 0:
            for h in range(HKV):
                kv = randn(1000 + 31 * b + h, 2, L[b] + T, HD)
                kv[0, :, 3] *= 6                          # a wide channel
                put_rows(pages, table, b, h, kv.to(torch.bfloat16))
    wide = randn(6, B, T, H * HD + 24, dtype=torch.bfloat16)
    q = wide[..., 16:16 + H * HD].unflatten(-1, (H, HD))
    y, mass, err, rec, rec_err = ref_attend(q, pages, table, L, HD ** -0.5, HKV)
    cap = table.shape[1] * page
    before = torch.rand(B, HKV, cap, generator=torch.Generator().manual_seed(7))
    weight = before.cuda() if weigh else None
    status = K.DeviceStatus("cuda")
    gp = pages.cuda()
    got = K.paged_attend(q=wide.cuda()[..., 16:16 + H * HD], pages=gp, table=table.cuda(), n=n,
                         lens=torch.tensor(L, dtype=torch.int32).cuda() if lens else None, weight=weight, status=status)
    assert int(status.word) == 0
    got = got.cpu().view(B, T, H, HD)
    few = T * (H // HKV) <= 16
    tol = mass * (2 * (err + (2 ** -17 if few else 2 ** -9) + 2 ** -21) + (n + T) * 2 ** -23)
    for b in range(B):
        if L[b] < 0:
            assert bool((got[b] == 0).all())
        else:
            assert rounded_within(got[b], y[b], tol[b])
    assert same(gp.cpu(), pages)
    if weigh:
        want = before.double() + rec
        assert bool(((weight.cpu().double() - want).abs() <= rec_err + 2 ** -23 * want * (rec > 0)).all())
        assert same(weight.cpu()[rec == 0], before[rec == 0])   # rows that no query sees


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 64])
def test_a_key_far_above_the_others_takes_everything(T):
    """Scores of hundreds; a reference that moves late in the cache and in the middle of a block."""
    B, H, HKV, HD, page, n = 1, 4, 1, 128, 32, 2000
    pages, table = new_pages(8, B, HKV, HD, page, n + T)
    kv = randn(9, 2, n + T, HD)
    q = randn(10, B, T, H, HD, dtype=torch.bfloat16)
    kv[0, 1700] = 20 * q[0, 0, 0].float()
    kv[0, 70] = 10 * q[0, 0, 0].float()
    kv = kv.to(torch.bfloat16)
    put_rows(pages, table, 0, 0, kv)
    y, mass, err, rec, rec_err = ref_attend(q, pages, table, [n], HD ** -0.5, HKV)
    weight = torch.zeros(B, HKV, table.shape[1] * page, device="cuda")
    got = K.paged_attend(q=q.cuda(), pages=pages.cuda(), table=table.cuda(), n=n, weight=weight).cpu().view(B, T, H, HD)
    assert rounded_within(got, y, mass * (2 * (err + (2 ** -17 if T * H <= 16 else 2 ** -9) + 2 ** -21) + (n + T) * 2 ** -23))
    assert bool(((weight.cpu().double() - rec).abs() <= rec_err + 2 ** -23 * rec).all())
    assert abs(float(y[0, 0, 0, 0]) - float(kv[1, 1700, 0])) < 1e-3


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 2, 40])
def test_values_that_are_not_finite_spoil_what_sees_them_only(T):
    """A NaN in one sequence's value and an infinite key in another's; the third is as it was."""
    B, H, HKV, HD, page, n = 3, 8, 2, 64, 16, 100
    pages, table = new_pages(11, B, HKV, HD, page, n + T, poison=float("inf"))
    for b in range(B):
        for h in range(HKV):
            put_rows(pages, table, b, h, randn(12 + 2 * b + h, 2, n + T, HD, dtype=torch.bfloat16))
    q = randn(13, B, T, H, HD, dtype=torch.bfloat16).cuda()
    clean = K.paged_attend(q=q, pages=pages.cuda(), table=table.cuda(), n=n).view(B, T, HKV, H // HKV, HD)
    assert bool(clean.isfinite().all())
    pages[1, table[0, 1].long(), 0, 3, 5] = float("nan")         # value of row 19, dimension 5, head 0 of sequence 0
    pages[0, table[1, 2].long(), 1, 0] = float("inf")            # key of row 32, head 1 of sequence 1
    y = K.paged_attend(q=q, pages=pages.cuda(), table=table.cuda(), n=n).view(B, T, HKV, H // HKV, HD)
    assert bool(y[0, :, 0, :, 5].isnan().all())
    keep = torch.ones(HD, dtype=torch.bool)
    keep[5] = False
    assert same(y[0, :, 0][..., keep.cuda()].contiguous(), clean[0, :, 0][..., keep.cuda()].contiguous())
    assert same(y[0, :, 1].contiguous(), clean[0, :, 1].contiguous())
    assert bool(y[1, :, 1].isnan().all())
    assert same(y[1, :, 0].contiguous(), clean[1, :, 0].contiguous()) and same(y[2].contiguous(), clean[2].contiguous())


@pytest.mark.gpu
@pytest.mark.parametrize("T,n", [(1, 40), (1, 3000), (48, 3000)])
def test_sequences_may_share_pages_that_are_read(T, n):
    H, HKV, HD, page = 8, 2, 128, 64
    pages, table = new_pages(14, 1, HKV, HD, page, n + T)
    for h in range(HKV):
        put_rows(pages, table, 0, h, randn(15 + h, 2, n + T, HD, dtype=torch.bfloat16))
    q = randn(16, 1, T, H, HD, dtype=torch.bfloat16).cuda()
    one = K.paged_attend(q=q, pages=pages.cuda(), table=table.cuda(), n=n)
    three = K.paged_attend(q=q.repeat(3, 1, 1, 1), pages=pages.cuda(), table=table.cuda().expand(3, -1), n=n)
    # (another cut into runs: the sums' order differs)
    assert bool(((three.double() - one.double()).abs() <= 2 ** -7 * one.double().abs() + 1e-4).all())


# -------------------------------------------------------------------------------------------- evict

def ref_evict(pages, table, weight, order, L, keep, recent):
    """In place; pages' rows by bits."""
    B, HKV, cap = weight.shape
    page = pages.shape[3]
    for b in range(B):
        n = int(L[b])
        if n <= keep:
            continue
        for h in range(HKV):
            w = [float("inf") if x != x else x for x in weight[b, h, :n].tolist()]
            o = order[b, h, :n].tolist()
            new = max(o) - recent
            rank = sorted(range(n), key=lambda i: (o[i] <= new, -w[i], i))
            kept = set(rank[:keep])
            to = [i for i in range(keep) if i not in kept]
            frm = [i for i in range(keep, n) if i in kept]
            assert len(to) == len(frm)
            at = table[b].long()
            for i, j in zip(to, frm):
                pages[:, at[i // page], h, i % page] = pages[:, at[j // page], h, j % page]
                weight[b, h, i] = weight[b, h, j]
                order[b, h, i] = order[b, h, j]


EVICT = [
    # B, HKV, HD, page, n, keep, recent, lens, weights
    (1, 2, 64, 16, 33, 32, 8, None, "random"),
    (2, 3, 128, 32, 100, 1, 1, None, "random"),
    (2, 3, 128, 32, 100, 1, 0, None, "random"),
    (3, 2, 64, 64, 300, 200, 200, (300, 200, 201), "random"),
    (4, 1, 128, 16, 300, 77, 13, (300, -1, 0, 78), "random"),
    (1, 5, 64, 128, 700, 512, 100, None, "equal"),
    (2, 2, 128, 64, 700, 512, 100, None, "few"),
    (1, 2, 64, 16, 400, 150, 40, None, "odd"),
    (1, 1, 128, 128, 20000, 3000, 500, None, "random"),   # keys beside shared memory, moves by a second kernel
    (1, 2, 64, 64, 20000, 19000, 500, None, "few"),
    (160, 1, 128, 16, 1300, 600, 64, None, "random"),     # more heads than CTAs, many moves each
    (2, 2, 64, 32, 64, 64, 5, None, "random"),            # nothing to drop
    (1, 2, 128, 32, 500, 100, 60, None, "same order"),    # more new rows than fit
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", EVICT)
def test_evict_matches_its_definition(case):
    B, HKV, HD, page, n, keep, recent, lens, kind = case
    L = lens if lens else [n] * B
    pages, table = new_pages(17, B, HKV, HD, page, n, poison=0.0)
    pages.view(torch.int16).random_(-2 ** 15, 2 ** 15, generator=torch.Generator().manual_seed(18))   # NaN rows too: bits move
    cap = table.shape[1] * page
    g = torch.Generator().manual_seed(19)
    weight = torch.rand(B, HKV, cap, generator=g)
    if kind == "equal":
        weight.fill_(0.25)
    elif kind == "few":
        weight = torch.randint(0, 3, weight.shape, generator=g).float()
    elif kind == "odd":                                   # NaN, infinities, both zeros, negative and tiny ones
        values = torch.tensor([float("nan"), math.inf, -math.inf, 0.0, -0.0, -1.5, 1e-42, 3.4e38, 0.5])
        weight = values[torch.randint(0, len(values), weight.shape, generator=g)]
        weight = torch.where(weight == 0, weight.abs(), weight)   # (equal floats of different bits have no order here)
    order = torch.stack([torch.randperm(3 * cap, generator=g)[:cap] for _ in range(B * HKV)]).view(B, HKV, cap).int()
    if kind == "same order":
        order.fill_(9)
    gp, gw, go, gt = pages.cuda(), weight.cuda(), order.cuda(), table.cuda()
    status = K.DeviceStatus("cuda")
    left = K.paged_evict(pages=gp, table=gt, weight=gw, order=go, n=n, keep=keep, recent=recent,
                         lens=torch.tensor(L, dtype=torch.int32).cuda() if lens else None, status=status)
    assert int(status.word) == 0
    if lens:
        assert left.dtype == torch.int32 and left.tolist() == [min(x, keep) for x in L]
    else:
        assert left == min(n, keep)
    ref_evict(pages, table, weight, order, L, keep, recent)
    assert same(gw.cpu(), weight) and torch.equal(go.cpu(), order) and same(gp.cpu(), pages)


# ------------------------------------------------------------------------------ together, graphs, streams

def test_reference_eviction_by_hand():
    """The definition at a size that can be read: rows 1 and 4 are new, 0 has the largest weight, 2 and 3 tie."""
    pages = torch.zeros(2, 1, 1, 16, 64, dtype=torch.bfloat16)
    pages[0, 0, 0, :6, 0] = torch.arange(6.0)
    table = torch.zeros(1, 1, dtype=torch.int32)
    weight = torch.tensor([[[9.0, 0.0, 1.0, 1.0, 0.0, 0.5] + [0.0] * 10]])
    order = torch.tensor([[[0, 8, 1, 2, 9, 3] + [0] * 10]], dtype=torch.int32)
    ref_evict(pages, table, weight, order, [6], 4, 2)
    assert pages[0, 0, 0, :6, 0].tolist() == [0, 1, 2, 4, 4, 5]
    assert order[0, 0, :6].tolist() == [0, 8, 1, 9, 9, 3]
    assert weight[0, 0, :6].tolist() == [9.0, 0.0, 1.0, 0.0, 0.0, 0.5]


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 3, 40])
def test_calls_replayed_from_a_graph_on_another_stream(T):
    """append, attend and evict captured once and replayed at two device positions, and two captured graphs at once, give
    what eager calls give."""
    B, H, HKV, HD, page, n = 2, 8, 2, 64, 16, 200
    cap_rows = n + 2 * T
    pages, table = new_pages(20, B, HKV, HD, page, cap_rows, poison=0.0)
    for b in range(B):
        for h in range(HKV):
            put_rows(pages, table, b, h, randn(21 + 2 * b + h, 2, n, HD, dtype=torch.bfloat16))
    W = -(-cap_rows // page)
    table = table[:, :W].contiguous()
    cap = W * page
    order = torch.arange(cap, dtype=torch.int32).expand(B, HKV, cap).contiguous()
    proj = randn(25, 2, B, T, (H + 2 * HKV) * HD, dtype=torch.bfloat16).cuda()
    inv = (1e4 ** (-torch.arange(0, HD, 2).float() / HD)).cuda()
    cut = (0, H * HD, (H + HKV) * HD, (H + 2 * HKV) * HD)

    def fresh():
        return dict(pages=pages.cuda(), weight=torch.zeros(B, HKV, cap, device="cuda"), order=order.cuda())

    gt = table.cuda()

    def both(st, x, n, **kw):
        q, k, v = (x[..., a:b] for a, b in zip(cut, cut[1:]))
        q = K.paged_append(q=q, k=k, v=v, table=gt, n=n, pos0=n, inv_freq=inv, **st, **kw)
        return K.paged_attend(q=q, pages=st["pages"], table=gt, n=n, weight=st["weight"], **kw)

    want = fresh()
    y0 = both(want, proj[0], n)
    y1 = both(want, proj[1], n + T)
    keep = n // 2
    want_pages = {k: t.clone() for k, t in want.items()}
    K.paged_evict(table=gt, n=n + 2 * T, keep=keep, recent=9, **want)

    got, other, x = fresh(), fresh(), torch.empty_like(proj[0])
    pos = K.DevicePosition("cuda")
    pos.ref, pos.span = n, T + 1
    status = K.DeviceStatus("cuda")
    both(fresh(), proj[0], n)                             # the libraries' lazy state
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    graphs = []
    with torch.cuda.stream(side):
        for st in (got, other):
            gr = torch.cuda.CUDAGraph()
            gr.capture_begin()
            out = both(st, x, n, dev_pos=pos, status=status)
            gr.capture_end()
            graphs.append((gr, out))
        ev = torch.cuda.CUDAGraph()
        ev.capture_begin()
        K.paged_evict(table=gt, n=n + 2 * T, keep=keep, recent=9, status=status, **got)
        ev.capture_end()
        ys = []
        for i in range(2):
            x.copy_(proj[i])
            pos.set(n + i * T)
            for gr, out in graphs:
                gr.replay()
                ys.append(out.clone())
    side.synchronize()
    assert int(status.word) == 0
    assert all(torch.equal(a, b) for a, b in zip(ys, (y0, y0, y1, y1)))
    for st in (got, other):
        assert all(torch.equal(st[k], want_pages[k]) for k in st)
    ev.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(got[k], want[k]) for k in got)


@pytest.mark.gpu
def test_a_bounded_cache_holds_what_a_full_one_weighs_most():
    """Tokens one by one with an eviction every few of them: the kept rows are those of the definition at every eviction,
    and attention over them is attention over those tokens."""
    B, H, HKV, HD, page, keep, step, recent = 2, 6, 2, 64, 16, 40, 8, 12
    pages, table = new_pages(30, B, HKV, HD, page, keep + step, poison=float("nan"))
    W = -(-(keep + step) // page)
    table = table[:, :W].contiguous()
    cap = W * page
    st = dict(pages=pages.cuda(), weight=torch.zeros(B, HKV, cap, device="cuda"),
              order=torch.zeros(B, HKV, cap, dtype=torch.int32, device="cuda"))
    gt = table.cuda()
    n, seen = 0, []
    for i in range(150):
        x = randn(100 + i, B, 1, (H + 2 * HKV) * HD, dtype=torch.bfloat16)
        seen.append(x[:, 0, H * HD:].view(B, 2, HKV, HD))
        g = x.cuda()
        q = K.paged_append(q=g[..., :H * HD], k=g[..., H * HD:(H + HKV) * HD], v=g[..., (H + HKV) * HD:], table=gt, n=n, pos0=i, **st)
        before = {k: t.cpu() for k, t in st.items()}
        y = K.paged_attend(q=q, pages=st["pages"], table=gt, n=n, weight=st["weight"]).cpu().view(B, 1, H, HD)
        n += 1
        for b in range(B):                                # every row is the token that its position names
            for h in range(HKV):
                at = before["order"][b, h, :n].tolist()
                assert len(set(at)) == n and max(at) == i
                want = torch.stack([seen[p][b, :, h] for p in at], 1)
                assert same(rows_of(before["pages"], table, b, h, n).contiguous(), want.contiguous())
        ref, mass, err, rec, rec_err = ref_attend(x[..., :H * HD].view(B, 1, H, HD), before["pages"], table, [n - 1] * B, HD ** -0.5, HKV)
        assert rounded_within(y, ref, mass * (2 * (err + 2 ** -17 + 2 ** -21) + n * 2 ** -23))
        if n == keep + step:
            want = {k: t.cpu() for k, t in st.items()}
            ref_evict(want["pages"], table, want["weight"], want["order"], [n] * B, keep, recent)
            n = K.paged_evict(table=gt, n=n, keep=keep, recent=recent, **st)
            assert n == keep
            assert same(st["weight"].cpu(), want["weight"]) and torch.equal(st["order"].cpu(), want["order"])
            assert same(st["pages"].cpu(), want["pages"])
            newest = st["order"][..., :keep].cpu().sort(-1, descending=True).values[..., :recent]
            assert bool((newest == torch.arange(i, i - recent, -1)).all())


# ----------------------------------------------------------------------------------------- refusals

def _call(**over):
    """Arguments of the three calls on small CUDA tensors; `over` replaces some of them."""
    B, H, HKV, HD, page, W = 2, 4, 2, 64, 16, 3
    d = dict(device="cuda")
    st = dict(q=torch.zeros(B, 1, H * HD, dtype=torch.bfloat16, **d), k=torch.zeros(B, 1, HKV * HD, dtype=torch.bfloat16, **d),
              v=torch.zeros(B, 1, HKV * HD, dtype=torch.bfloat16, **d),
              pages=torch.zeros(2, B * W, HKV, page, HD, dtype=torch.bfloat16, **d),
              table=torch.arange(B * W, dtype=torch.int32, **d).view(B, W), weight=torch.zeros(B, HKV, W * page, **d),
              order=torch.zeros(B, HKV, W * page, dtype=torch.int32, **d), n=5, pos0=5, lens=None, pos=None, keep=3, recent=1,
              sm_scale=None, status=K.DeviceStatus("cuda"))
    st.update(over)
    a = {k: st[k] for k in ("pages", "table", "n", "lens", "status")}
    return (lambda: K.paged_append(q=st["q"], k=st["k"], v=st["v"], pos0=st["pos0"], pos=st["pos"], weight=st["weight"], order=st["order"], **a),
            lambda: K.paged_attend(q=st["q"], weight=st["weight"], sm_scale=st["sm_scale"], **a),
            lambda: K.paged_evict(weight=st["weight"], order=st["order"], keep=st["keep"], recent=st["recent"], **a)), st


def test_cpu_tensors_are_refused():
    z = torch.zeros
    pages, table = z(2, 4, 2, 16, 64, dtype=torch.bfloat16), z(2, 2, dtype=torch.int32)
    q, k = z(2, 1, 256, dtype=torch.bfloat16), z(2, 1, 128, dtype=torch.bfloat16)
    rec = dict(weight=z(2, 2, 32), order=z(2, 2, 32, dtype=torch.int32))
    with pytest.raises((RuntimeError, AssertionError)):
        K.paged_append(q=q, k=k, v=k, pages=pages, table=table, n=0, pos0=0)
    with pytest.raises((RuntimeError, AssertionError)):
        K.paged_attend(q=q, pages=pages, table=table, n=0)
    with pytest.raises((RuntimeError, AssertionError)):
        K.paged_evict(pages=pages, table=table, n=20, keep=4, **rec)


REFUSED = [
    # which of (append, attend, evict) refuse, arguments, error
    ((0, 1, 2), lambda: dict(pages=torch.zeros(2, 6, 2, 16, 64, device="cuda")), TypeError),
    ((0, 1, 2), lambda: dict(pages=torch.zeros(2, 6, 2, 24, 64, dtype=torch.bfloat16, device="cuda")), ValueError),
    ((0, 1, 2), lambda: dict(pages=torch.zeros(2, 6, 2, 16, 80, dtype=torch.bfloat16, device="cuda")), ValueError),
    ((0, 1, 2), lambda: dict(pages=torch.zeros(2, 12, 2, 16, 64, dtype=torch.bfloat16, device="cuda")[:, ::2]), ValueError),
    ((0, 1, 2), lambda: dict(table=torch.zeros(2, 3, dtype=torch.int64, device="cuda")), TypeError),
    ((0, 1, 2), lambda: dict(table=torch.zeros(2, 3, dtype=torch.int32)), RuntimeError),
    ((0, 1, 2), lambda: dict(table=torch.zeros(2, 6, dtype=torch.int32, device="cuda")[:, ::2]), ValueError),
    ((0, 1, 2), lambda: dict(weight=torch.zeros(2, 2, 47, device="cuda")), ValueError),
    ((0, 2), lambda: dict(order=torch.zeros(2, 2, 48, device="cuda")), TypeError),
    ((0, 2), lambda: dict(weight=None), ValueError),
    ((0, 1), lambda: dict(n=48), RuntimeError),                 # no room for the token
    ((2,), lambda: dict(n=49), RuntimeError),
    ((0, 1, 2), lambda: dict(n=-1), RuntimeError),
    ((0, 1, 2), lambda: dict(lens=torch.zeros(3, dtype=torch.int32, device="cuda")), ValueError),
    ((0, 1, 2), lambda: dict(lens=torch.zeros(2, dtype=torch.int64, device="cuda")), TypeError),
    ((0,), lambda: dict(pos=torch.zeros(2, dtype=torch.int32, device="cuda")), ValueError),
    ((0, 1), lambda: dict(q=torch.zeros(2, 1, 100, dtype=torch.bfloat16, device="cuda")), ValueError),
    ((1,), lambda: dict(q=torch.zeros(2, 1, 3 * 64, dtype=torch.bfloat16, device="cuda")), RuntimeError),   # 3 heads on 2
    ((1,), lambda: dict(q=torch.zeros(2, 1, 34 * 64, dtype=torch.bfloat16, device="cuda")), RuntimeError),  # 17 to one
    ((1,), lambda: dict(sm_scale=0.0), RuntimeError),
    ((1,), lambda: dict(sm_scale=float("nan")), RuntimeError),
    ((1,), lambda: dict(sm_scale=-1.0), RuntimeError),
    ((2,), lambda: dict(keep=0), ValueError),
    ((2,), lambda: dict(recent=4), ValueError),
    ((2,), lambda: dict(recent=-1), ValueError),
]


@pytest.mark.gpu
@pytest.mark.parametrize("i", range(len(REFUSED)))
def test_what_does_not_fit_is_refused(i):
    which, over, error = REFUSED[i]
    calls, st = _call(**over())
    for j in which:
        with pytest.raises(error):
            calls[j]()
    torch.cuda.synchronize()
    assert int(st["status"].word) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 40])
def test_lengths_and_pages_on_the_device_that_do_not_fit_are_skipped(T):
    """The kernels' own checks: a length above the bound, a page outside the pool. Nothing is read or written there, and
    the status word says so."""
    B, H, HKV, HD, page, W = 3, 4, 2, 64, 16, 6
    n = 30
    for what in ("length", "page", "negative page"):
        pages = torch.zeros(2, B * W, HKV, page, HD, dtype=torch.bfloat16, device="cuda")
        table = torch.arange(B * W, dtype=torch.int32, device="cuda").view(B, W).clone()
        lens = torch.tensor([n, n, n], dtype=torch.int32, device="cuda")
        if what == "length":
            lens[1] = n + 1
        else:
            table[1, 1] = B * W if what == "page" else -7
        weight = torch.ones(B, HKV, W * page, device="cuda")
        order = torch.arange(W * page, dtype=torch.int32, device="cuda").expand(B, HKV, -1).contiguous()
        x = randn(40, B, T, (H + 2 * HKV) * HD, dtype=torch.bfloat16).cuda()
        status = K.DeviceStatus("cuda")

        def bits():
            status.arm("paged cache")
            with pytest.raises(RuntimeError, match="outside the range"):
                status.check(block=True)

        kw = dict(pages=pages, table=table, lens=lens, status=status)
        q = K.paged_append(q=x[..., :H * HD], k=x[..., H * HD:(H + HKV) * HD], v=x[..., (H + HKV) * HD:], n=n, pos0=n, weight=weight,
                           order=order, **kw)
        bits()                                            # (row 30 lies in page 1)
        assert bool((pages[:, W:2 * W].isfinite()).all())
        y = K.paged_attend(q=q, n=n, weight=weight, **kw)
        bits()
        if what == "length":
            assert bool((y[1] == 0).all()) and bool((weight[1] == 1).all())
        assert bool((y[0] != 0).any()) and bool((y[2] != 0).any())
        was = pages.clone(), weight.clone(), order.clone()
        left = K.paged_evict(weight=weight, order=order, n=n, keep=10, recent=2, **kw)
        bits()
        assert left.tolist()[0::2] == [10, 10] and left.tolist()[1] == (-1 if what == "length" else 10)
        assert torch.equal(pages[:, W:2 * W], was[0][:, W:2 * W])
        assert torch.equal(weight[1], was[1][1]) and torch.equal(order[1], was[2][1])


@pytest.mark.gpu
def test_a_device_position_out_of_its_range_is_skipped():
    calls, st = _call()
    pos = K.DevicePosition("cuda")
    pos.ref, pos.span = 5, 4
    pos.set(9)
    y = K.paged_attend(q=st["q"], pages=st["pages"], table=st["table"], n=5, dev_pos=pos, status=st["status"], weight=st["weight"])
    st["status"].arm("paged cache")
    with pytest.raises(RuntimeError, match="outside the range"):
        st["status"].check(block=True)
    assert bool((y == 0).all()) and bool((st["weight"] == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 40])
def test_a_pool_whose_offsets_pass_32_bits(T):
    """The same rows in pages at the start of a small pool and at the end of one of more than 2^31 values to a side."""
    B, H, HKV, HD, page, n = 2, 4, 1, 128, 128, 300
    W, P = 3, (1 << 31) // (128 * 128) + 9
    x = randn(60, B, n + T, (H + 2 * HKV) * HD, dtype=torch.bfloat16).cuda()
    cut = (0, H * HD, (H + HKV) * HD, (H + 2 * HKV) * HD)
    small = torch.zeros(2, B * W, HKV, page, HD, dtype=torch.bfloat16, device="cuda")
    large = torch.empty(2, P, HKV, page, HD, dtype=torch.bfloat16, device="cuda")
    tables = [torch.arange(B * W, dtype=torch.int32, device="cuda").view(B, W)]
    tables.append(tables[0] + (P - B * W))
    out = []
    for pages, table in zip((small, large), tables):
        pages[:, table.view(-1).long()] = 0
        rec = dict(weight=torch.zeros(B, HKV, W * page, device="cuda"), order=torch.zeros(B, HKV, W * page, dtype=torch.int32, device="cuda"))
        for t0, t1 in ((0, n), (n, n + T)):
            q, k, v = (x[:, t0:t1, a:b] for a, b in zip(cut, cut[1:]))
            q = K.paged_append(q=q, k=k, v=v, pages=pages, table=table, n=t0, pos0=t0, **rec)
        y = K.paged_attend(q=q, pages=pages, table=table, n=n, weight=rec["weight"])
        left = K.paged_evict(pages=pages, table=table, n=n + T, keep=200, recent=9, **rec)
        out.append((q, y, left, pages[:, table.view(-1).long()], rec["weight"], rec["order"]))
    for a, b in zip(*out):
        assert a == b if isinstance(a, int) else torch.equal(a, b)
    assert bool((out[0][1] != 0).any())


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 40])
def test_calls_on_two_streams_at_once(T):
    """Two streams take steps over caches of their own at the same time; each is as it is alone."""
    H, HKV, HD, page, n = 8, 2, 128, 32, 700
    cap = 1024
    x = [randn(70 + i, 3, T, (H + 2 * HKV) * HD, dtype=torch.bfloat16).cuda() for i in range(2)]
    cut = (0, H * HD, (H + HKV) * HD, (H + 2 * HKV) * HD)
    kv = [randn(72 + i, 2, 3 * cap // page, HKV, page, HD, dtype=torch.bfloat16).cuda() for i in range(2)]
    table = torch.arange(3 * cap // page, dtype=torch.int32, device="cuda").view(3, -1)

    def fresh(i):
        return dict(pages=kv[i].clone(), weight=torch.zeros(3, HKV, cap, device="cuda"),
                    order=torch.arange(cap, dtype=torch.int32, device="cuda").expand(3, HKV, cap).contiguous())

    def step(i, st, j):
        q, k, v = (x[i][..., a:b] for a, b in zip(cut, cut[1:]))
        q = K.paged_append(q=q, k=k, v=v, table=table, n=n + j * T, pos0=n + j * T, **st)
        return K.paged_attend(q=q, pages=st["pages"], table=table, n=n + j * T, weight=st["weight"])

    def finish(st):
        K.paged_evict(table=table, n=n + 4 * T, keep=n // 2, recent=3, **st)

    want, ys = [fresh(i) for i in range(2)], [[], []]
    for i in range(2):
        ys[i] = [step(i, want[i], j) for j in range(4)]
        finish(want[i])
    got, zs = [fresh(i) for i in range(2)], [[], []]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for j in range(4):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                zs[i].append(step(i, got[i], j))
    for i, st in enumerate(streams):
        with torch.cuda.stream(st):
            finish(got[i])
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, b) for a, b in zip(ys[i], zs[i]))
        assert all(torch.equal(want[i][k], got[i][k]) for k in got[i])


@pytest.mark.gpu
def test_positions_are_recorded_in_32_bits():
    """The last positions that fit are recorded, later ones refused; positions on the device count as the largest."""
    for pos0 in (2 ** 31 - 1, -(2 ** 31) + 4):
        calls, st = _call(pos0=pos0)
        with pytest.raises(RuntimeError):
            calls[0]()
    calls, st = _call(pos0=2 ** 31 - 2)
    calls[0]()
    assert st["order"][:, :, 5].tolist() == [[2 ** 31 - 2] * 2] * 2
    z = torch.zeros(2, 3, 2 * 64, dtype=torch.bfloat16, device="cuda")
    K.paged_append(q=z, k=z, v=z, pages=st["pages"], table=st["table"], n=5, pos0=0, weight=st["weight"], order=st["order"],
                   lens=torch.tensor([5, 0], dtype=torch.int32, device="cuda"),
                   pos=torch.tensor([2 ** 31 - 2, -7], dtype=torch.int32, device="cuda"))
    assert st["order"][0, 0, 5:8].tolist() == [2 ** 31 - 2, 2 ** 31 - 1, 2 ** 31 - 1]
    assert st["order"][1, 1, 0:3].tolist() == [-7, -6, -5]


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 40])
def test_tables_and_queries_with_strides(T):
    """Rows of a larger table, queries out of a larger tensor, and outputs that the caller gives."""
    B, H, HKV, HD, page, n = 3, 8, 2, 64, 16, 200
    W = -(-(n + T) // page)
    pages = randn(80, 2, B * W, HKV, page, HD, dtype=torch.bfloat16).cuda()
    wide = torch.full((2 * B, W + 5), -3, dtype=torch.int32, device="cuda")
    table = torch.randperm(B * W, generator=torch.Generator().manual_seed(81)).to(torch.int32).view(B, W).cuda()
    wide[::2, 2:W + 2] = table
    q = randn(82, B, T, H, HD, dtype=torch.bfloat16).cuda()
    qs = torch.full((B, 2 * T, H + 3, HD), float("nan"), dtype=torch.bfloat16, device="cuda")
    qs[:, ::2, 1:H + 1] = q
    weight = [torch.zeros(B, HKV, W * page, device="cuda") for _ in range(2)]
    y = K.paged_attend(q=q, pages=pages, table=table, n=n, weight=weight[0])
    out = torch.empty_like(y)
    got = K.paged_attend(q=qs[:, ::2, 1:H + 1], pages=pages, table=wide[::2, 2:W + 2], n=n, weight=weight[1], y=out)
    assert got is out and torch.equal(got, y) and torch.equal(*weight)
