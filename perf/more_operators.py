"""Paged anchor caches of bounded size: the operators' cases, inputs and plain forms.

Four operators, each in its plain form (elementary torch operations in 32 bits, one rounding at the end)
and through the framework's entry points (`own`):

- append: RMSNorm of every query and key head, rotate-half position rotation, queries out in bf16, keys and
  values into the pages that a table gives each sequence;
- attend: softmax attention of the T newest tokens over the pages, causal among themselves;
- weigh: the same, and the softmax weight that each cached row got from all query rows of its head is added
  to a record;
- evict: T tokens enter a cache that holds up to `keep` rows (append), then every head keeps `keep` of them:
  the newest ones and those with the largest recorded weight. Kept rows from behind `keep` move into the
  places of dropped ones.
"""
import math

import torch

own = False

DEV = "cuda"


# ---------------------------------------------------------------------------------------- cases

def _append(B, T, H, HKV, HD, page, n, pos, norm, ragged):
    return dict(op="append", B=B, T=T, H=H, HKV=HKV, HD=HD, page=page, n=n, pos=pos, norm=norm, ragged=ragged)


def _attend(op, B, T, H, HKV, HD, page, n, ragged):
    return dict(op=op, B=B, T=T, H=H, HKV=HKV, HD=HD, page=page, n=n, ragged=ragged)


def _evict(B, T, H, HKV, HD, page, keep, recent, ragged):
    return dict(op="evict", B=B, T=T, H=H, HKV=HKV, HD=HD, page=page, keep=keep, recent=recent, ragged=ragged)


def listed():
    return [
        # one token of 64 sequences enters an anchor's cache of 2303 rows, far into the text (a generation step)
        dict(name="append_step", **_append(64, 1, 32, 8, 128, 64, 2303, 100000, True, False)),
        # a ragged slice of a prompt, narrow heads without norms, every sequence at its own length and position
        dict(name="append_slice_odd", **_append(37, 101, 15, 5, 64, 16, 700, 700, False, True)),
        # one token of one short conversation: latency
        dict(name="attend_small", **_attend("attend", 1, 1, 15, 5, 64, 16, 332, False)),
        # one token of one conversation of 131072: the cache is split over the whole machine
        dict(name="attend_one_long", **_attend("attend", 1, 1, 32, 8, 128, 64, 131071, False)),
        # one token of 64 sequences of different lengths
        dict(name="attend_step", **_attend("attend", 64, 1, 32, 8, 128, 64, 2303, True)),
        # the largest: a 128-token slice of 64 prompts after 2048 cached tokens
        dict(name="attend_slice", **_attend("attend", 64, 128, 32, 8, 128, 128, 2048, False)),
        # one token of three short conversations, their weights recorded: latency
        dict(name="weigh_small", **_attend("weigh", 3, 1, 7, 1, 64, 32, 700, True)),
        # one token of 64 sequences at a bounded cache, weights recorded (a generation step)
        dict(name="weigh_step", **_attend("weigh", 64, 1, 32, 8, 128, 64, 2175, False)),
        # a 128-token slice of 16 prompts, weights recorded
        dict(name="weigh_slice", **_attend("weigh", 16, 128, 32, 8, 128, 64, 2048, False)),
        # 13 tokens of one conversation with narrow heads go past its bound
        dict(name="evict_small", **_evict(1, 13, 15, 5, 64, 16, 501, 64, False)),
        # a chunk's end of 64 sequences: 128 tokens in, 128 out, at 2048 rows
        dict(name="evict_step", **_evict(64, 128, 32, 8, 128, 64, 2048, 256, False)),
        # a long slice of a few prompts of different lengths goes past the bound at once
        dict(name="evict_long", **_evict(4, 2011, 16, 2, 128, 32, 4096, 512, True)),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


HEADS = ((15, 5, 64), (4, 2, 64), (32, 8, 128), (8, 8, 128), (16, 2, 128), (7, 1, 64), (12, 2, 128), (16, 1, 128))


def draw(rng):
    op = rng.choice(("append", "attend", "attend", "weigh", "weigh", "evict"))
    H, HKV, HD = rng.choice(HEADS)
    page = rng.choice((16, 32, 64, 128))
    ragged = rng.random() < 0.5
    if op == "append":
        T = rng.choice((1, 1, 128, _log(rng, 2, 300)))
        n = _log(rng, 1, 4000) - 1
        return _append(max(1, min(128, _log(rng, 1, 8000) // T)), T, H, HKV, HD, page, n,
                       n + rng.choice((0, _log(rng, 1, 130000))), rng.random() < 0.5, ragged)
    if op == "evict":
        keep, T = _log(rng, 16, 8192), _log(rng, 1, 2048)
        return _evict(max(1, min(64, _log(rng, 1, 64), 150000 // (keep + T))), T, H, HKV, HD, page, keep,
                      rng.randint(0, keep), ragged)
    T = rng.choice((1, 1, 1, 2, _log(rng, 2, 128), 128))
    n = _log(rng, 1, 131072) - 1
    most = 64 * 128 * 2048 if op == "attend" else 16 * 128 * 2048
    B = max(1, min(64, _log(rng, 1, 64), 160000 // (n + T), most // (T * (n + T))))
    return _attend(op, B, T, H, HKV, HD, page, n, ragged)


# ---------------------------------------------------------------------------------------- inputs

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _lens(B, n, g):
    """Rows of every sequence, spread over [n / 2, n]."""
    return torch.randint(n // 2, n + 1, (B,), generator=g, device=DEV, dtype=torch.int32)


def _pages(g, B, HKV, HD, page, rows):
    """(pages bf16 [2, pages, HKV, page, HD] of keys and values, table int32 [B, pages of a sequence]): pages in
    no order, some of the pool unused; a few wide channels in the keys, as trained models have them."""
    W = (rows + page - 1) // page
    P = B * W + 3
    pages = torch.empty(2, P, HKV, page, HD, device=DEV, dtype=torch.bfloat16)
    wide = 1 + 4 * (torch.rand(HKV, 1, HD, generator=g, device=DEV) < 0.04).float()
    step = max(1, (1 << 26) // (HKV * page * HD))
    for p in range(0, P, step):
        pages[0, p:p + step] = _randn(g, *pages[0, p:p + step].shape) * wide
        pages[1, p:p + step] = _randn(g, *pages[1, p:p + step].shape)
    table = torch.randperm(P, generator=g, device=DEV)[:B * W].view(B, W).to(torch.int32)
    return pages, table


def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    s = dict(case)
    B, T, H, HKV, HD, page = (case[k] for k in ("B", "T", "H", "HKV", "HD", "page"))
    n = case["keep"] if op == "evict" else case["n"]
    s["n"] = n
    s["pages"], s["table"] = _pages(g, B, HKV, HD, page, n + T)
    s["lens"] = _lens(B, n, g) if case["ragged"] else None
    s["weight"] = s["order"] = None
    cap = s["table"].shape[1] * page
    if op in ("append", "evict"):
        proj = _randn(g, B, T, (H + 2 * HKV) * HD).to(torch.bfloat16)    # one fused projection of the hidden states
        s.update(q=proj[..., :H * HD], k=proj[..., H * HD:(H + HKV) * HD], v=proj[..., (H + HKV) * HD:],
                 inv_freq=1.0 / (1e6 ** (torch.arange(0, HD, 2, device=DEV).float() / HD)), eps=1e-6,
                 q_norm=None, k_norm=None)
        if case.get("norm", True):
            s["q_norm"] = 1 + 0.1 * _randn(g, HD)
            s["k_norm"] = 1 + 0.1 * _randn(g, HD)
        # positions of the next token: rows that were dropped before count too
        s["pos0"] = case["pos"] if op == "append" else 3 * n + 7
        s["pos"] = None
        if case["ragged"]:
            s["pos"] = s["lens"] + (s["pos0"] - n)
    else:
        s["q"] = _randn(g, B, T, H, HD).to(torch.bfloat16)
        s["sm_scale"] = HD ** -0.5
    if op in ("weigh", "evict"):
        # weights so far: most of it on few rows, none on rows that just came; a record that has just begun where the
        # call's own share is looked at
        x = torch.rand(B, HKV, cap, generator=g, device=DEV)
        s["weight"] = torch.where(x < 0.1, 0.0, (0.05 if op == "evict" else 1e-5) / (1.0001 - x))
    if op == "evict":
        # positions of the held rows, in no order: gaps where rows were dropped before
        gaps = torch.randint(1, 4, (B, HKV, cap), generator=g, device=DEV)
        held = torch.full((B,), n, device=DEV) if s["lens"] is None else s["lens"].long()
        row = torch.arange(cap, device=DEV)
        place = torch.where(row < held[:, None, None], torch.rand(B, HKV, cap, generator=g, device=DEV), 2.0)
        last = torch.full((B,), s["pos0"], device=DEV) if s["pos"] is None else s["pos"].long()
        back = gaps.cumsum(-1).gather(-1, place.argsort(-1).argsort(-1))
        s["order"] = torch.where(row < held[:, None, None], last[:, None, None] - back, 0).to(torch.int32)
    return s


# ---------------------------------------------------------------------------------------- plain forms

def _held(s):
    return s["lens"].long() if s["lens"] is not None else torch.full((s["B"],), s["n"], device=DEV)


def _norm_rotate(x, w, eps, cos, sin):
    """x [B, T, heads, HD] in 32 bits; cos, sin [B, T, 1, HD / 2]."""
    if w is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * w
    a, b = x.chunk(2, dim=-1)
    return torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)


def _plain_append(s):
    B, T, H, HKV, HD, page = (s[k] for k in ("B", "T", "H", "HKV", "HD", "page"))
    t = torch.arange(T, device=DEV)
    row = _held(s)[:, None] + t
    pos = (torch.full((B,), s["pos0"], device=DEV) if s["pos"] is None else s["pos"].long())[:, None] + t
    ang = (pos.double()[..., None] * s["inv_freq"].double())[:, :, None]
    cos, sin = ang.cos().float(), ang.sin().float()
    q = _norm_rotate(s["q"].float().view(B, T, H, HD), s["q_norm"], s["eps"], cos, sin).to(torch.bfloat16)
    k = _norm_rotate(s["k"].float().view(B, T, HKV, HD), s["k_norm"], s["eps"], cos, sin).to(torch.bfloat16)
    pg = s["table"].long().gather(1, row // page)[..., None]
    h, r = torch.arange(HKV, device=DEV), (row % page)[..., None]
    s["pages"][0, pg, h, r] = k
    s["pages"][1, pg, h, r] = s["v"].view(B, T, HKV, HD)
    if s["weight"] is not None:
        b = torch.arange(B, device=DEV)[:, None, None]
        s["weight"][b, h, row[..., None]] = 0.0
        s["order"][b, h, row[..., None]] = pos[..., None].to(torch.int32).expand(B, T, HKV)
    return q


def _plain_attend(s):
    B, T, H, HKV, HD = (s[k] for k in ("B", "T", "H", "HKV", "HD"))
    G = H // HKV
    k, v = s["pages"][:, s["table"].long()].transpose(2, 3).reshape(2, B, HKV, -1, HD).float()
    L = k.shape[2]
    q = s["q"].float().view(B, T, HKV, G, HD).permute(0, 2, 1, 3, 4).reshape(B, HKV, T * G, HD)
    t = (q @ k.transpose(-1, -2)).view(B, HKV, T, G, L) * s["sm_scale"]
    last = _held(s)[:, None] + torch.arange(T, device=DEV)
    seen = torch.arange(L, device=DEV) <= last[..., None]
    t = t.masked_fill_(~seen[:, None, :, None], -math.inf)
    p = torch.exp(t - t.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    y = (p.view(B, HKV, T * G, L) @ v).view(B, HKV, T, G, HD)
    y = y.permute(0, 2, 1, 3, 4).reshape(B, T, H * HD).to(torch.bfloat16)
    if s["weight"] is None:
        return y
    s["weight"] += p.sum((2, 3))
    return dict(y=y, weight=s["weight"])


def _plain_evict(s):
    keep, page = s["keep"], s["page"]
    q = _plain_append(s)
    n = _held(s) + s["T"]
    weight, order = s["weight"], s["order"]
    cap = weight.shape[-1]
    row = torch.arange(cap, device=DEV)
    valid = row < n[:, None, None]
    newest = torch.where(valid, order.long(), -(1 << 40)).amax(-1, keepdim=True)
    first = valid & (order > newest - s["recent"])
    bits = weight.view(torch.int32).long()
    key = torch.where(bits < 0, ~bits & 0xFFFFFFFF, bits | 0x80000000)             # in the order of the weights
    key = ((first.long() << 32 | key) << 21) | (0x1FFFFF - row)                    # ties to the lowest row
    key = torch.where(valid, key, -1)
    least = torch.topk(key, min(keep, cap), dim=-1).values[..., -1:]
    kept = valid & (key >= least)
    hole, mover = (row < keep) & valid & ~kept, (row >= keep) & kept
    src = torch.zeros(*weight.shape[:2], cap + 1, device=DEV, dtype=torch.long)
    src.scatter_(-1, torch.where(mover, mover.cumsum(-1) - 1, cap), row.expand_as(mover))
    b, h, to = hole.nonzero(as_tuple=True)
    frm = src[b, h, (hole.cumsum(-1) - 1)[b, h, to]]
    pg = s["table"].long()
    s["pages"][:, pg[b, to // page], h, to % page] = s["pages"][:, pg[b, frm // page], h, frm % page]
    weight[b, h, to] = weight[b, h, frm]
    order[b, h, to] = order[b, h, frm]
    left = min(s["n"] + s["T"], keep) if s["lens"] is None else n.clamp_max(keep).to(torch.int32)
    return dict(q=q, pages=s["pages"], weight=weight, order=order, left=left)


# ---------------------------------------------------------------------------------------- one pass

def _own_append(s):
    from vsa_lm_b200 import kernels as K

    return K.paged_append(q=s["q"], k=s["k"], v=s["v"], pages=s["pages"], table=s["table"], n=s["n"], pos0=s["pos0"],
                          inv_freq=s["inv_freq"], q_norm=s["q_norm"], k_norm=s["k_norm"], eps=s["eps"], lens=s["lens"],
                          pos=s["pos"], weight=s["weight"], order=s["order"])


def _own_attend(s):
    from vsa_lm_b200 import kernels as K

    y = K.paged_attend(q=s["q"], pages=s["pages"], table=s["table"], n=s["n"], sm_scale=s["sm_scale"], lens=s["lens"],
                       weight=s["weight"])
    return y if s["weight"] is None else dict(y=y, weight=s["weight"])


def _own_evict(s):
    from vsa_lm_b200 import kernels as K

    q = _own_append(s)
    n = s["n"] + s["T"]
    lens = None if s["lens"] is None else s["lens"] + s["T"]
    left = K.paged_evict(pages=s["pages"], table=s["table"], weight=s["weight"], order=s["order"], n=n, keep=s["keep"],
                         recent=s["recent"], lens=lens)
    return dict(q=q, pages=s["pages"], weight=s["weight"], order=s["order"], left=left)


def run(state):
    s = state
    if s["op"] == "append":
        q = _own_append(s) if own else _plain_append(s)
        return dict(q=q, pages=s["pages"])
    if s["op"] == "evict":
        out = _own_evict(s) if own else _plain_evict(s)
        # the text goes on: the next pass's tokens are newer than all that the cache holds
        s["pos0"] += s["T"]
        if s["pos"] is not None:
            s["pos"] += s["T"]
        return out
    return _own_attend(s) if own else _plain_attend(s)


# ---------------------------------------------------------------------------------------- floors and 64 bits

def work(case):
    c = case
    B, T, H, HKV, HD = (c[k] for k in ("B", "T", "H", "HKV", "HD"))
    # projections in, queries out, keys and values into the pages
    into = B * T * (2 * H + 4 * HKV) * HD * 2
    if c["op"] == "append":
        return dict(bytes=into, flops=B * T * (H + HKV) * HD * 10)
    if c["op"] == "evict":
        # weights and positions of all rows read, those of the new ones written; the rows that move, read and written:
        # at most the new ones (a ragged batch is at three quarters of its bound on average, and a quarter of `keep` fits)
        n = c["keep"] * (0.75 if c["ragged"] else 1.0)
        heads, over = B * HKV, max(0, min(n + T - c["keep"], c["keep"]))
        return dict(bytes=into + heads * ((n + T) * 8 + T * 8 + over * (2 * 2 * HD * 2 + 16)), flops=B * T * (H + HKV) * HD * 10)
    n = c["n"] * (0.75 if c["ragged"] else 1.0)
    keys, rows = B * HKV * (n + T), B * T * H
    return dict(bytes=keys * (2 * HD * 2 + (8 if c["op"] == "weigh" else 0)) + rows * HD * 4,
                flops=rows * (n + (T + 1) / 2) * HD * 4)


def exact(case, seed):
    s = prepare(case, seed)
    B, T, H, HKV, HD, page = (s[k] for k in ("B", "T", "H", "HKV", "HD", "page"))
    G = H // HKV
    held = [s["n"]] * B if s["lens"] is None else s["lens"].tolist()

    def in_64_append():
        start = [s["pos0"]] * B if s["pos"] is None else s["pos"].tolist()
        pos = torch.tensor([[p + t for t in range(T)] for p in start], device=DEV, dtype=torch.float64)
        turn = torch.polar(torch.ones(B, T, 1, HD // 2, device=DEV, dtype=torch.float64),
                           (pos[..., None] * s["inv_freq"].double())[:, :, None])

        def heads(x, w):
            x = x.double().reshape(B, T, -1, HD)
            if w is not None:
                x = x / (x.pow(2).sum(-1, keepdim=True) / HD + s["eps"]).sqrt() * w.double()
            z = torch.complex(x[..., :HD // 2], x[..., HD // 2:]) * turn
            return torch.cat((z.real, z.imag), -1)

        k, v = heads(s["k"], s["k_norm"]), s["v"].double().reshape(B, T, HKV, HD)
        pages = s["pages"].double()
        for b in range(B):
            rows = torch.arange(held[b], held[b] + T, device=DEV)
            at = s["table"][b].long()[rows // page]
            pages[0, at, :, rows % page] = k[b]
            pages[1, at, :, rows % page] = v[b]
            if s["order"] is not None:
                s["weight"][b, :, held[b]:held[b] + T] = 0
                s["order"][b, :, held[b]:held[b] + T] = torch.arange(start[b], start[b] + T, device=DEV, dtype=torch.int32)
        return dict(q=heads(s["q"], s["q_norm"]), pages=pages)

    def in_64_attend():
        y = torch.empty(B, T, H, HD, device=DEV, dtype=torch.float64)
        weight = None if s["weight"] is None else s["weight"].double()
        for b in range(B):
            n = held[b] + T
            mine = s["pages"][:, s["table"][b].long()].transpose(1, 2).reshape(2, HKV, -1, HD)[:, :, :n]
            late = torch.ones(T, n, device=DEV, dtype=torch.bool).triu(held[b] + 1)
            for h in range(HKV):
                k, v = mine[:, h].double()
                q = s["q"][b, :, h * G:(h + 1) * G].double()
                t = torch.einsum("tgd,ld->gtl", q, k) * s["sm_scale"]
                p = torch.softmax(t.masked_fill(late, -math.inf), -1)
                y[b, :, h * G:(h + 1) * G] = torch.einsum("gtl,ld->tgd", p, v)
                if weight is not None:
                    weight[b, h, :n] += p.sum((0, 1))
        y = y.view(B, T, H * HD)
        return y if weight is None else dict(y=y, weight=weight)

    def in_64_evict():
        out = in_64_append()
        keep, recent = s["keep"], s["recent"]
        pages, weight = out["pages"], s["weight"].double()
        for b in range(B):
            n = held[b] + T
            if n <= keep:
                continue
            at = s["table"][b].long()
            for h in range(HKV):
                w, o = weight[b, h, :n], s["order"][b, h, :n].long()
                rank = torch.where(o > o.max() - recent, math.inf, w)
                best = torch.sort(rank, descending=True, stable=True).indices[:keep]
                kept = torch.zeros(n, device=DEV, dtype=torch.bool)
                kept[best] = True
                to = (~kept[:keep]).nonzero().view(-1)
                frm = kept[keep:].nonzero().view(-1) + keep
                pages[:, at[to // page], h, to % page] = pages[:, at[frm // page], h, frm % page]
                weight[b, h, to] = weight[b, h, frm]
        return dict(q=out["q"], pages=pages, weight=weight, order=None, left=None)

    return dict(append=in_64_append, attend=in_64_attend, weigh=in_64_attend, evict=in_64_evict)[case["op"]]()
