"""The 8-bit KV cache of a softmax anchor: bolt3_kv8_append, bolt3_kv8_read and bolt3_kv8_attend
against plain implementations in 64 bits.

Tolerances, from the arithmetic of include/bolt3.h:
- a bf16 result is rounded once, and rounding is monotone: it lies between the rounded ends of the
  interval in which the value before it may lie (`rounded_within`);
- a norm and a rotation in fp32 are off by a few 2^-24 of the row's largest value, 2e-6 of it here;
- a stored row is off by half a step of its scale, a value row exactly as torch's fp32 division and
  rounding give it;
- attention: weights rounded to f16 (2^-11 each, and 2^-25 of the largest one where they are below f16's
  normal range), and scores summed in fp32 (HD roundings of the products' absolute sum, times 2 for
  the tensor cores' truncation).
"""
import ctypes
import math

import pytest
import torch

from vsa_lm_b200 import _lib
from vsa_lm_b200 import kernels as K

FLOOR = 2.0 ** -40


def randn(seed, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def rounded_within(y, ref, tol):
    """Whether the bf16 `y` is the rounding of a number within `tol` of the 64-bit `ref`. (The ends are
    widened by the fp32 step on the way to bf16.)"""
    tol = tol + 2 ** -23 * ref.abs() + 1e-37
    lo, hi = ((ref + d).float().to(torch.bfloat16).double() for d in (-tol, tol))
    return bool(((y.double() >= lo) & (y.double() <= hi)).all())


def new_cache(B, HKV, cap, HD, dev="cuda"):
    """A cache whose untouched rows are poison: a NaN scale and the largest stored values."""
    return (torch.full((2, B, HKV, cap, HD), 127, dtype=torch.int8, device=dev),
            torch.full((2, B, HKV, cap), float("nan"), device=dev))


def ref_rows(x, w, eps, pos, inv_freq):
    """64-bit norm and rotation of x [B, T, h, HD]; pos [B, T]."""
    x = x.double()
    HD = x.shape[-1]
    if w is not None:
        x = x / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt() * w.double()
    if inv_freq is not None:
        ang = (pos.float()[..., None] * inv_freq).double()[:, :, None]   # the angle is an fp32 product
        c, s, a, b = ang.cos(), ang.sin(), x[..., :HD // 2], x[..., HD // 2:]
        x = torch.cat((a * c - b * s, b * c + a * s), -1)
    return x


def stored(x):
    """Scale and int8 of rows, in fp32 as torch computes them."""
    sc = (x.abs().amax(-1) / 127).clamp_min(FLOOR)
    return torch.round(x / sc[..., None]).clamp(-128, 127).to(torch.int8), sc


APPEND = [
    # B, T, H, HKV, HD, n, cap, norm, rope, lens
    (1, 1, 4, 2, 64, 0, 1, True, True, None),
    (3, 1, 32, 8, 128, 700, 1024, True, True, None),
    (2, 5, 15, 5, 64, 3, 9, False, True, None),
    (3, 37, 7, 1, 64, 100, 300, True, True, (0, 263, -1)),
    (2, 130, 4, 4, 128, 10, 200, True, False, None),
    (4, 2, 1, 1, 128, 9, 16, False, False, (14, 0, -1, 3)),
    (9, 128, 12, 2, 128, 128, 256, True, True, None),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", APPEND)
def test_append_matches_64_bits(case):
    B, T, H, HKV, HD, n, cap, norm, rope, lens = case
    proj = randn(1, B, T, (H + 2 * HKV) * HD + 8, dtype=torch.bfloat16)
    q, k, v = proj[..., 8:8 + H * HD], proj[..., 8 + H * HD:8 + (H + HKV) * HD], proj[..., 8 + (H + HKV) * HD:]
    qw = 1 + 0.2 * randn(2, HD) if norm else None
    kw = 1 + 0.2 * randn(3, HD) if norm else None
    inv = 1e4 ** (-torch.arange(0, HD, 2).float() / HD) if rope else None
    L = torch.tensor(lens if lens else [n] * B)
    pos0 = n + 17
    pos = pos0 + (L[:, None] - n) + torch.arange(T)
    data, scale = new_cache(B, HKV, cap, HD)
    was = data.clone(), scale.clone()
    status = K.DeviceStatus("cuda")
    g = proj.cuda()
    cu = lambda t: None if t is None else t.cuda()
    q_out = K.kv8_append(q=g[..., 8:8 + H * HD], k=g[..., 8 + H * HD:8 + (H + HKV) * HD], v=g[..., 8 + (H + HKV) * HD:],
                         data=data, scale=scale, n=n, pos0=pos0, inv_freq=cu(inv), q_norm=cu(qw), k_norm=cu(kw),
                         eps=1e-5, lens=cu(L.int()) if lens else None, status=status).cpu()
    assert int(status.word) == 0
    rq = ref_rows(q.reshape(B, T, H, HD), qw, 1e-5, pos, inv)
    rk = ref_rows(k.reshape(B, T, HKV, HD), kw, 1e-5, pos, inv)
    v8, vs = stored(v.reshape(B, T, HKV, HD).float())
    touched = torch.zeros(B, cap, dtype=torch.bool)
    for b in range(B):
        if L[b] < 0:
            assert bool((q_out[b] == 0).all())
            continue
        assert rounded_within(q_out[b], rq[b], 2e-6 * rq[b].abs().amax(-1, keepdim=True))
        rows = slice(int(L[b]), int(L[b]) + T)
        touched[b, rows] = True
        ks, k8 = scale[0, b, :, rows].cpu(), data[0, b, :, rows].cpu()
        ref = rk[b].transpose(0, 1)
        top = ref.abs().amax(-1)
        assert bool(((ks.double() - top / 127).abs() <= 2e-6 * top / 127 + FLOOR).all())
        assert bool(((k8.double() * ks.double()[..., None] - ref).abs() <= 0.5 * ks.double()[..., None] + 2e-6 * top[..., None]).all())
        assert torch.equal(data[1, b, :, rows].cpu(), v8[b].transpose(0, 1))
        assert torch.equal(scale[1, b, :, rows].cpu(), vs[b].transpose(0, 1))
    keep = ~touched[None, :, None].expand(2, B, HKV, cap).cuda()
    assert torch.equal(data[keep], was[0][keep]) and bool(scale[keep].isnan().all())


@pytest.mark.gpu
def test_append_zero_nan_and_infinite_rows():
    HD = 64
    x = torch.zeros(1, 5, HD, dtype=torch.bfloat16)
    x[0, 1, 3] = float("nan")
    x[0, 2, 5] = float("-inf")
    x[0, 3] = 1e-30
    x[0, 4] = 3e38
    data, scale = new_cache(1, 1, 8, HD)
    g = x.cuda()
    q = K.kv8_append(q=g, k=g, v=g, data=data, scale=scale, n=0, pos0=0)
    for side in (0, 1):
        s = scale[side, 0, 0].cpu()
        assert s[0] == FLOOR and s[1].isnan() and s[2] == float("inf") and s[3] == FLOOR
        assert s[4] == x[0, 4, 0].float() / 127
        assert bool((data[side, 0, 0, 0] == 0).all()) and bool((data[side, 0, 0, 4] == 127).all())
    assert torch.equal(q[0, 0].cpu(), torch.zeros(1, HD, dtype=torch.bfloat16)) and bool(q[0, 1, 0, 3].isnan())
    back = K.kv8_read(data, scale, 0, 5).cpu()
    assert bool((back[:, 0, 0, 0] == 0).all()) and bool(back[:, 0, 0, 1].isnan().all())


@pytest.mark.gpu
def test_lengths_out_of_range_skip_the_sequence():
    B, HKV, HD, cap, T = 4, 2, 64, 8, 3
    x = randn(4, B, T, HKV * HD, dtype=torch.bfloat16).cuda()
    lens = torch.tensor([6, 5, -2, -1], dtype=torch.int32).cuda()     # 6 + 3 > 8; fits; not a length; idle
    data, scale = new_cache(B, HKV, cap, HD)
    before = data.clone()
    status = K.DeviceStatus("cuda")
    q = K.kv8_append(q=x, k=x, v=x, data=data, scale=scale, n=0, pos0=0, lens=lens, status=status)
    assert int(status.word) == 8
    for b in (0, 2, 3):
        assert torch.equal(data[:, b], before[:, b]) and bool((q[b] == 0).all())
    assert not torch.equal(data[:, 1], before[:, 1])
    for fn in (lambda s: K.kv8_attend(q=x, data=data, scale=scale, n=5, lens=lens, status=s),
               lambda s: K.kv8_read(data, scale, 0, T, lens=lens, status=s)):
        status = K.DeviceStatus("cuda")
        out = fn(status)
        assert int(status.word) == 8
        out = out if out.dim() == 3 else out.transpose(0, 1)
        for b in (0, 2, 3):
            assert bool((out[b] == 0).all())
        assert bool((out[1] != 0).any())


@pytest.mark.gpu
@pytest.mark.parametrize("B,HKV,HD,cap,t0,T,lens", [
    (1, 1, 64, 1, 0, 1, None), (2, 5, 64, 300, 7, 211, None), (3, 8, 128, 1030, 0, 1030, None),
    (3, 2, 128, 40, 0, 9, (31, 0, -1))])
def test_read_is_the_rounded_product(B, HKV, HD, cap, t0, T, lens):
    g = torch.Generator().manual_seed(5)
    data = torch.randint(-128, 128, (2, B, HKV, cap, HD), generator=g, dtype=torch.int8)
    scale = torch.rand(2, B, HKV, cap, generator=g)
    L = torch.tensor(lens, dtype=torch.int32).cuda() if lens else None
    out = K.kv8_read(data.cuda(), scale.cuda(), t0, T, lens=L).cpu()
    for b in range(B):
        s = lens[b] if lens else t0
        ref = torch.zeros(2, HKV, T, HD, dtype=torch.bfloat16)
        if s >= 0:
            ref = (data[:, b, :, s:s + T].float() * scale[:, b, :, s:s + T, None]).to(torch.bfloat16)
        assert torch.equal(out[:, b], ref)


def random_cache(seed, B, HKV, cap, HD, wide=1.0, spread=0.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(2, B, HKV, cap, HD, generator=g)
    x[0, ..., :3] *= wide
    if spread:
        x[1] *= torch.exp2(spread * (2 * torch.rand(B, HKV, cap, 1, generator=g) - 1))
    return stored(x)


def check_attend(q, data, scale, n, lens, sm_scale, y):
    """y against 64 bits with the bound of the module's docstring."""
    B, T, H, HD = q.shape
    HKV, G = data.shape[2], H // data.shape[2]
    y = y.view(B, T, HKV, G, HD).double()
    for b in range(B):
        s = n if lens is None else lens[b]
        if s < 0:
            assert bool((y[b] == 0).all())
            continue
        L = s + T
        k, v = (data[:, b, :, :L].double() * scale[:, b, :, :L, None].double())
        qb = q[b].double().view(T, HKV, G, HD)
        t = torch.einsum("thgd,hld->htgl", qb, k) * sm_scale
        t_abs = torch.einsum("thgd,hld->htgl", qb.abs(), k.abs()).amax(-1, keepdim=True) * abs(sm_scale)
        late = torch.arange(L) > (s + torch.arange(T))[:, None]
        p = torch.softmax(t.masked_fill(late[None, :, None], -math.inf), -1)
        ref = torch.einsum("htgl,hld->thgd", p, v)
        mag = torch.einsum("htgl,hld->thgd", p, v.abs())
        big = v.abs().amax((1, 2)).view(1, HKV, 1, 1)
        slack = (2 ** -11 + 2 ** -18 + 2 * HD * 2 ** -24 * t_abs).permute(1, 0, 2, 3)
        assert rounded_within(y[b], ref, slack * mag + L * 2 ** -25 * big), b


ATTEND = [
    # B, T, H, HKV, HD, n, cap, lens
    (1, 1, 1, 1, 64, 0, 1, None),                       # the first token of all
    (1, 1, 4, 4, 128, 1, 2, None),
    (2, 1, 15, 5, 64, 14, 15, None),                    # 15 rows: one short of a block of 16 keys
    (2, 1, 32, 8, 128, 15, 16, None),
    (2, 1, 14, 2, 128, 16, 17, None),
    (3, 1, 16, 2, 64, 300, 512, (-1, 0, 300)),
    (5, 1, 32, 8, 128, 1000, 1001, (1000, 64, 63, 777, 0)),
    (1, 1, 4, 1, 128, 5000, 5120, None),                # one chain, split over many blocks
    (1, 2, 16, 1, 64, 130, 200, None),
    (2, 3, 8, 2, 128, 70, 100, (70, 5)),                # 12 query rows: two column tiles of 8
    (2, 17, 15, 5, 64, 0, 17, None),                    # a prompt from nothing
    (1, 64, 12, 2, 128, 37, 128, None),
    (3, 128, 8, 2, 128, 200, 330, (200, -1, 3)),
    (2, 129, 4, 4, 128, 127, 256, None),
    (1, 257, 10, 2, 64, 511, 768, None),
    (2, 31, 16, 1, 128, 90, 121, None),
    (2, 128, 32, 8, 128, 384, 512, None),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", ATTEND)
def test_attend_matches_64_bits(case):
    B, T, H, HKV, HD, n, cap, lens = case
    data, scale = random_cache(7, B, HKV, cap, HD)
    # what lies past the rows a sequence holds must not matter
    for b in range(B):
        s = n if lens is None else max(lens[b], -T)
        data[:, b, :, s + T:] = 127
        scale[:, b, :, s + T:] = float("nan")
    q = randn(8, B, T, H, HD, dtype=torch.bfloat16)
    L = torch.tensor(lens, dtype=torch.int32).cuda() if lens else None
    y = K.kv8_attend(q=q.cuda(), data=data.cuda(), scale=scale.cuda(), n=n, lens=L).cpu()
    check_attend(q, data, scale, n, lens, HD ** -0.5, y)


@pytest.mark.gpu
@pytest.mark.parametrize("T,H,HKV,HD", [(1, 8, 2, 128), (1, 4, 1, 64), (128, 8, 2, 128), (40, 8, 2, 64)])
@pytest.mark.parametrize("kind", ["sharp", "flat", "wide queries", "tiny queries", "spread values", "negative scale"])
def test_attend_value_ranges(T, H, HKV, HD, kind):
    """Peaked and flat softmaxes, large and tiny queries, value rows of very different size."""
    n, sm = 600, HD ** -0.5
    data, scale = random_cache(9, 2, HKV, n + T, HD, wide=8.0 if kind == "sharp" else 1.0,
                               spread=14.0 if kind == "spread values" else 0.0)
    q = randn(10, 2, T, H, HD)
    q *= {"sharp": 4.0, "wide queries": 3e4, "tiny queries": 1e-20}.get(kind, 1.0)
    sm *= {"flat": 1e-3, "wide queries": 1e-4, "tiny queries": 1e20, "negative scale": -1.0}.get(kind, 1.0)
    q = q.to(torch.bfloat16)
    y = K.kv8_attend(q=q.cuda(), data=data.cuda(), scale=scale.cuda(), n=n, sm_scale=sm).cpu()
    check_attend(q, data, scale, n, None, sm, y)


@pytest.mark.gpu
@pytest.mark.parametrize("T,HD", [(3, 64), (100, 64), (40, 128)])
def test_attend_rows_of_very_different_sizes(T, HD):
    """Query rows 2^26 times larger than their neighbours leave those as they are."""
    B, H, HKV, n = 2, 8, 2, 300
    data, scale = random_cache(25, B, HKV, n + T, HD)
    q = randn(26, B, T, H, HD)
    q.view(B, T * H, HD)[:, ::3] *= 2.0 ** 26
    q = q.to(torch.bfloat16)
    y = K.kv8_attend(q=q.cuda(), data=data.cuda(), scale=scale.cuda(), n=n).cpu()
    check_attend(q, data, scale, n, None, HD ** -0.5, y)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 100])
def test_attend_nan_stays_in_its_sequence(T):
    """A NaN key or value that a query sees spoils that query; what no query of a sequence sees does not."""
    B, H, HKV, HD, n = 3, 4, 2, 128, 40
    data, scale = random_cache(11, B, HKV, n + T, HD)
    scale[0, 1, 0, 5] = float("nan")          # a key of sequence 1, head 0
    scale[1, 2, 1, 7] = float("nan")          # a value of sequence 2, head 1
    scale[1, 0, 0, n + T - 1] = float("nan")  # only the last query of sequence 0 sees this one
    q = randn(12, B, T, H, HD, dtype=torch.bfloat16)
    y = K.kv8_attend(q=q.cuda(), data=data.cuda(), scale=scale.cuda(), n=n).cpu().view(B, T, HKV, H // HKV, HD)
    spoiled = y.isnan().all(-1)
    want = torch.zeros_like(spoiled)
    want[1, :, 0] = True
    want[2, :, 1] = True
    want[0, T - 1, 0] = True
    assert torch.equal(spoiled, want) and torch.equal(y.isnan().any(-1), want)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 4, 100])
@pytest.mark.parametrize("what", [float("nan"), float("inf"), float("-inf")])
def test_attend_unbounded_query_spoils_its_own_row(T, what):
    B, H, HKV, HD, n = 2, 4, 2, 64, 50
    data, scale = random_cache(21, B, HKV, n + T, HD)
    q = randn(22, B, T, H, HD, dtype=torch.bfloat16)
    clean = K.kv8_attend(q=q.cuda(), data=data.cuda(), scale=scale.cuda(), n=n).cpu().view(B, T, H, HD)
    q[1, T // 2, 3, 7] = what
    y = K.kv8_attend(q=q.cuda(), data=data.cuda(), scale=scale.cuda(), n=n).cpu().view(B, T, H, HD)
    assert bool(y[1, T // 2, 3].isnan().all())
    keep = torch.ones(B, T, H, dtype=torch.bool)
    keep[1, T // 2, 3] = False
    check = y.clone()
    check[1, T // 2, 3] = 0
    assert bool(check.isfinite().all()) and torch.equal(y[keep], clean[keep])


@pytest.mark.gpu
def test_attend_a_long_prompt_at_once():
    """More rows than a grid's second dimension holds: 20000 tokens of 4 heads on one KV head, checked at a few rows."""
    H, HD, T = 4, 64, 20000
    data, scale = random_cache(23, 1, 1, T, HD)
    q = randn(24, 1, T, H, HD, dtype=torch.bfloat16)
    y = K.kv8_attend(q=q.cuda(), data=data.cuda(), scale=scale.cuda(), n=0).cpu()
    for t in (0, 1, 127, 5000, T - 1):
        check_attend(q[:, t:t + 1], data, scale, t, None, HD ** -0.5, y[:, t:t + 1])


@pytest.mark.gpu
def test_attend_rows_past_32_bit_offsets():
    """Rows whose byte offset in the cache passes 2^31 and whose element offset of the values 2^32."""
    HKV, HD, cap = 8, 128, 2_200_000
    data = torch.zeros(2, 1, HKV, cap, HD, dtype=torch.int8, device="cuda")
    scale = torch.ones(2, 1, HKV, cap, device="cuda")
    n, few = cap - 1, 40
    d, s = random_cache(13, 1, HKV, few, HD)
    lo = cap - few
    scale[0] = 1e-3
    # zero keys score 0; the last rows hold keys that outweigh all of them together
    q = randn(14, 1, 1, HKV * 2, HD, dtype=torch.bfloat16)
    data[:, :, :, lo:] = d.cuda()
    scale[:, :, :, lo:] = s.cuda()
    y = K.kv8_attend(q=q.cuda(), data=data, scale=scale, n=n, sm_scale=4.0).cpu().double().view(HKV, 2, HD)
    k, v = d[:, 0].double() * s[:, 0, ..., None].double()
    t = torch.einsum("hgd,hld->hgl", q[0, 0].double().view(HKV, 2, HD), k) * 4.0
    full = torch.cat((torch.zeros(HKV, 2, lo, dtype=torch.float64), t), -1)
    p = torch.softmax(full, -1)[..., lo:]
    ref = torch.einsum("hgl,hld->hgd", p, v)
    assert bool(((y - ref).abs() <= 2 ** -7 * v.abs().amax()).all())
    back = K.kv8_read(data, scale, lo, few).cpu()
    assert torch.equal(back, (d.float() * s[..., None]).to(torch.bfloat16))


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 3, 70])
def test_device_position_equals_the_host_position(T):
    B, H, HKV, HD, cap = 2, 8, 2, 64, 512
    x = randn(15, B, T, (H + 2 * HKV) * HD, dtype=torch.bfloat16).cuda()
    q, k, v = x[..., :H * HD], x[..., H * HD:(H + HKV) * HD], x[..., (H + HKV) * HD:]
    inv = (1e4 ** (-torch.arange(0, HD, 2).float() / HD)).cuda()
    d0, s0 = random_cache(16, B, HKV, cap, HD)
    a, b = (d0.cuda(), s0.cuda()), (d0.cuda(), s0.cuda())
    pos = K.DevicePosition("cuda")
    pos.ref, pos.span = 100, 64
    pos.set(133)
    qa = K.kv8_append(q=q, k=k, v=v, data=a[0], scale=a[1], n=333, pos0=133, inv_freq=inv)
    qb = K.kv8_append(q=q, k=k, v=v, data=b[0], scale=b[1], n=300, pos0=100, inv_freq=inv, dev_pos=pos)
    assert torch.equal(qa, qb) and torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    ya = K.kv8_attend(q=qa, data=a[0], scale=a[1], n=333)
    yb = K.kv8_attend(q=qb, data=b[0], scale=b[1], n=300, dev_pos=pos)
    check_attend(qb.cpu(), b[0].cpu(), b[1].cpu(), 333, None, HD ** -0.5, yb.cpu())
    check_attend(qa.cpu(), a[0].cpu(), a[1].cpu(), 333, None, HD ** -0.5, ya.cpu())
    status = K.DeviceStatus("cuda")
    pos.set(164)                                       # past the span: nothing is written, zeros come back
    before = b[0].clone()
    K.kv8_append(q=q, k=k, v=v, data=b[0], scale=b[1], n=300, pos0=100, inv_freq=inv, dev_pos=pos, status=status)
    y = K.kv8_attend(q=qb, data=b[0], scale=b[1], n=300, dev_pos=pos, status=status)
    assert int(status.word) == 8 and torch.equal(before, b[0]) and bool((y == 0).all())


@pytest.mark.gpu
def test_on_another_stream_and_repeatable():
    B, H, HKV, HD, n = 2, 8, 2, 128, 900
    data, scale = (t.cuda() for t in random_cache(17, B, HKV, n + 1, HD))
    q = randn(18, B, 1, H, HD, dtype=torch.bfloat16).cuda()
    y = K.kv8_attend(q=q, data=data, scale=scale, n=n)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = [K.kv8_attend(q=q, data=data, scale=scale, n=n) for _ in range(3)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(y, z) for z in again)       # no sum depends on the order blocks finish in


@pytest.mark.gpu
def test_strided_queries():
    B, T, H, HKV, HD, n = 2, 4, 8, 4, 64, 30
    data, scale = random_cache(19, B, HKV, n + T, HD)
    wide = randn(20, B, T + 3, H * HD + 64, dtype=torch.bfloat16)
    part = wide[:, 1:1 + T, 64:]
    y = K.kv8_attend(q=wide.cuda()[:, 1:1 + T, 64:], data=data.cuda(), scale=scale.cuda(), n=n).cpu()
    check_attend(part.reshape(B, T, H, HD), data, scale, n, None, HD ** -0.5, y)


@pytest.mark.gpu
def test_refusals():
    B, T, H, HKV, HD, cap = 2, 3, 4, 2, 64, 16
    data, scale = new_cache(B, HKV, cap, HD)
    q = torch.zeros(B, T, H, HD, dtype=torch.bfloat16, device="cuda")
    kv = torch.zeros(B, T, HKV, HD, dtype=torch.bfloat16, device="cuda")
    ok = dict(q=q, k=kv, v=kv, data=data, scale=scale, n=0, pos0=0)
    lens = torch.zeros(B, dtype=torch.int32, device="cuda")

    def refused(exc, fn, base, **change):
        with pytest.raises(exc):
            fn(**{**base, **change})

    app, att = K.kv8_append, K.kv8_attend
    at = dict(q=q, data=data, scale=scale, n=0)
    for fn, base in ((app, ok), (att, at)):
        refused(RuntimeError, fn, base, q=q.cpu())
        refused(TypeError, fn, base, q=q.float())
        refused(ValueError, fn, base, q=q[:, :, :, :32])
        refused(ValueError, fn, base, q=q.transpose(2, 3).contiguous().transpose(2, 3))
        refused(TypeError, fn, base, data=data.to(torch.uint8))
        refused(ValueError, fn, base, data=data[:, :, :, :8])
        refused(ValueError, fn, base, scale=scale[:, :, :, :8].contiguous())
        refused(RuntimeError, fn, base, n=cap - T + 1)         # no room
        refused(RuntimeError, fn, base, n=-1)
        refused(ValueError, fn, base, lens=lens[:1])
        refused(TypeError, fn, base, lens=lens.long())
        refused(ValueError, fn, base, lens=lens, dev_pos=K.DevicePosition("cuda"))
    refused(ValueError, app, ok, k=q)                          # 4 heads for a cache of 2
    refused(TypeError, app, ok, q_norm=torch.ones(HD, device="cuda", dtype=torch.bfloat16))
    refused(ValueError, app, ok, inv_freq=torch.ones(HD // 4, device="cuda"))
    refused(RuntimeError, app, ok, q=torch.zeros(B, T, H * HD + 4, dtype=torch.bfloat16, device="cuda")[..., 4:])
    refused(RuntimeError, att, at, q=torch.zeros(B, T, 3, HD, dtype=torch.bfloat16, device="cuda"))   # 3 heads on 2
    refused(RuntimeError, att, at, q=torch.zeros(B, T, 34, HD, dtype=torch.bfloat16, device="cuda"))  # 17 per KV head
    with pytest.raises(RuntimeError):
        K.kv8_read(data, scale, cap - 2, 3)
    with pytest.raises(RuntimeError):
        K.kv8_read(data, scale, -1, 3)


def test_entry_points_reject_bad_arguments_without_a_gpu():
    """Fake (never dereferenced) addresses: every call returns before a launch."""
    lib = _lib.load()
    for name in ("bolt3_kv8_append", "bolt3_kv8_read", "bolt3_kv8_attend"):
        assert getattr(lib, name)(None, None) == 1
    fake = 1 << 20

    def attend(**kw):
        a = _lib.Kv8AttendArgs(B=1, T=1, H=4, HKV=2, HD=64, q=fake, q_sb=256, q_st=256, data=fake, scale=fake, cap=8,
                               n=7, y=fake, sm_scale=0.1)
        for k, v in kw.items():
            setattr(a, k, v)
        return lib.bolt3_kv8_attend(ctypes.byref(a), None)

    assert attend(q=0) == 1 and attend(lens=fake, pos_dev=fake, pos_span=1) == 1 and attend(pos_dev=fake) == 1
    assert attend(HD=96) == 2 and attend(H=5) == 2 and attend(H=34) == 2 and attend(T=0) == 2 and attend(B=-1) == 2
    assert attend(q=fake + 8) == 3 and attend(q_st=4) == 3
    assert attend(n=8) == 4 and attend(n=-1) == 4 and attend(pos_dev=fake, pos_span=2) == 4
    assert attend(n=7000, cap=8000) == 4                         # the split cache needs a workspace

    def append(**kw):
        a = _lib.Kv8AppendArgs(B=1, T=2, H=4, HKV=2, HD=64, q=fake, k=fake, v=fake, q_out=fake, data=fake, scale=fake,
                               cap=8, n=0)
        for k, v in kw.items():
            setattr(a, k, v)
        return lib.bolt3_kv8_append(ctypes.byref(a), None)

    assert append(v=0) == 1 and append(H=0) == 2 and append(HD=32) == 2 and append(H=4095, HKV=8) == 2
    assert append(n=7) == 4 and append(n=-1) == 4 and append(k_st=12) == 3 and append(q_norm_w=fake + 4) == 3

    def read(**kw):
        a = _lib.Kv8ReadArgs(B=1, HKV=2, HD=64, T=2, data=fake, scale=fake, cap=8, t0=0, out=fake)
        for k, v in kw.items():
            setattr(a, k, v)
        return lib.bolt3_kv8_read(ctypes.byref(a), None)

    assert read(out=0) == 1 and read(T=0) == 2 and read(t0=7) == 4 and read(T=9) == 4 and read(out=fake + 2) == 3
    assert read(B=1 << 30, HKV=4) == 2
    assert lib.bolt3_kv8_attend_workspace(1, 1, 4, 3, 64, 100) == 0
    assert lib.bolt3_kv8_attend_workspace(1, 1, 4, 2, 64, 1 << 50) == 0 and attend(lens=fake, n=9) == 4
    assert attend(T=1 << 23, cap=1 << 24, n=0, H=8) == 2


def test_cpu_tensors_are_refused():
    d, s = new_cache(1, 1, 4, 64, dev="cpu")
    x = torch.zeros(1, 1, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError):
        K.kv8_append(q=x, k=x, v=x, data=d, scale=s, n=0, pos0=0)
    with pytest.raises(RuntimeError):
        K.kv8_attend(q=x, data=d, scale=s, n=0)
    with pytest.raises(RuntimeError):
        K.kv8_read(d, s, 0, 1)
