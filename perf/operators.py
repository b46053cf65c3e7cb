"""Beam decoding over 8-bit anchor caches: the operators' cases, inputs and plain forms.

Five operators, each in its plain form (elementary torch operations in 32 bits, one rounding at the
end) and through the framework's entry points (`own`):

- append: RMSNorm of every query and key head, rotate-half position rotation, queries out in bf16, keys
  and values written to an int8 cache with one fp32 scale per (token, KV head);
- read: a range of that cache back as bf16;
- attend: softmax attention of the T newest tokens over the cache, causal among themselves;
- select: log-softmax over the vocabulary, the K best continuations of K beams, assigned to slots so
  that a surviving beam keeps its slot;
- reorder: every beam's decode state replaced by its parent's, in place.
"""
import math

import torch

own = False

DEV = "cuda"
FLOOR = 2.0 ** -40          # smallest scale of a quantised row
PAD = 7                     # the end-of-sequence id of the select cases


# ---------------------------------------------------------------------------------------- cases

def _append(B, T, H, HKV, HD, n, norm, ragged):
    return dict(op="append", B=B, T=T, H=H, HKV=HKV, HD=HD, n=n, norm=norm, ragged=ragged)


def _read(B, HKV, HD, t0, T, cap):
    return dict(op="read", B=B, HKV=HKV, HD=HD, t0=t0, T=T, cap=cap)


def _attend(B, T, H, HKV, HD, n, ragged):
    return dict(op="attend", B=B, T=T, H=H, HKV=HKV, HD=HD, n=n, ragged=ragged)


def _select(B, K, V, dtype, first):
    return dict(op="select", B=B, K=K, V=V, dtype=dtype, first=first)


def _reorder(B, K, HKV, HD, cap, t0, t1, layer):
    return dict(op="reorder", B=B, K=K, HKV=HKV, HD=HD, cap=cap, t0=t0, t1=t1, layer=layer)


def listed():
    return [
        # one token of 64 sequences enters an anchor's cache after 2303 (a generation step)
        dict(name="append_step", **_append(64, 1, 32, 8, 128, 2303, True, False)),
        # a ragged slice of a prompt, narrow heads without norms, every sequence at its own length
        dict(name="append_slice_odd", **_append(37, 101, 15, 5, 64, 700, False, True)),
        # 16 cached rows back for a look at what one step wrote
        dict(name="read_few", **_read(1, 5, 64, 1001, 16, 1280)),
        # a whole prompt's keys and values exported as bf16
        dict(name="read_prompt", **_read(16, 8, 128, 0, 2047, 2304)),
        # one token of one short conversation: latency
        dict(name="attend_small", **_attend(1, 1, 15, 5, 64, 332, False)),
        # one token of one conversation of 131072: the cache is split over the whole machine
        dict(name="attend_one_long", **_attend(1, 1, 32, 8, 128, 131071, False)),
        # one token of 64 sequences (16 groups of 4 beams) of different lengths
        dict(name="attend_step", **_attend(64, 1, 32, 8, 128, 2303, True)),
        # the largest: a 128-token slice of 64 prompts after 2048 cached tokens
        dict(name="attend_slice", **_attend(64, 128, 32, 8, 128, 2048, False)),
        # the first step of one beam search: three of the four beams are empty
        dict(name="select_first", **_select(1, 4, 32000, "float32", True)),
        # a step of 64 groups of 4 beams over a vocabulary of 151936, some beams finished
        dict(name="select_step", **_select(64, 4, 151936, "bfloat16", False)),
        # one group's anchor cache, only the tokens since the prompt
        dict(name="reorder_small", **_reorder(1, 4, 5, 64, 512, 131, 164, False)),
        # 16 groups of 4: one Bolt-3 layer's whole state and one anchor cache since the prompt
        dict(name="reorder_layer", **_reorder(16, 4, 8, 128, 2560, 2048, 2304, True)),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


HEADS = ((15, 5, 64), (4, 2, 64), (32, 8, 128), (8, 8, 128), (16, 2, 128), (7, 1, 64), (12, 2, 128))


def draw(rng):
    op = rng.choice(("append", "read", "attend", "attend", "select", "reorder"))
    H, HKV, HD = rng.choice(HEADS)
    if op == "append":
        T = rng.choice((1, 1, 128, _log(rng, 2, 300)))
        return _append(max(1, min(128, _log(rng, 1, 8000) // T)), T, H, HKV, HD, _log(rng, 1, 4000) - 1,
                       rng.random() < 0.5, rng.random() < 0.5)
    if op == "read":
        t0, T = _log(rng, 1, 1000) - 1, _log(rng, 1, 4000)
        return _read(_log(rng, 1, 16), HKV, HD, t0, T, (t0 + T + 255) // 256 * 256)
    if op == "attend":
        T = rng.choice((1, 1, 1, 2, _log(rng, 2, 128), 128))
        n = _log(rng, 1, 131072) - 1
        B = max(1, min(64, _log(rng, 1, 64), 160000 // (n + T), 64 * 128 * 2048 // (T * (n + T))))
        return _attend(B, T, H, HKV, HD, n, rng.random() < 0.5)
    if op == "select":
        V = _log(rng, 100, 150000)
        return _select(_log(rng, 1, 64), rng.choice((1, 2, 3, 4, 5, 8, 16)) if V < 35000 else rng.choice((1, 2, 4)), V,
                       rng.choice(("float32", "bfloat16")), rng.random() < 0.25)
    t0, more = _log(rng, 1, 2048) - 1, _log(rng, 1, 256)
    return _reorder(_log(rng, 1, 16), rng.choice((2, 3, 4)), HKV, HD, (t0 + more + 255) // 256 * 256, t0, t0 + more,
                    rng.random() < 0.3)


# ---------------------------------------------------------------------------------------- inputs

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _lens(case, g):
    """The cached length of every sequence: `n` for all of them, or spread over [n / 2, n]."""
    if not case["ragged"]:
        return None
    n = case["n"]
    return torch.randint(n // 2, n + 1, (case["B"],), generator=g, device=DEV, dtype=torch.int32)


def _freqs(HD):
    return 1.0 / (1e6 ** (torch.arange(0, HD, 2, device=DEV).float() / HD))


def _cache(g, B, HKV, cap, HD):
    """An int8 cache [2, B, HKV, cap, HD] of keys and values with its scales [2, B, HKV, cap]: a few wide
    channels in the keys, a small value at the first token, as trained models have them."""
    x = _randn(g, 2, B, HKV, cap, HD)
    x[0] *= 1 + 4 * (torch.rand(HKV, 1, HD, generator=g, device=DEV) < 0.04).float()
    x[1, :, :, 0] *= 0.02
    scale = (x.abs().amax(-1) / 127).clamp_min(FLOOR)
    data = x.div_(scale[..., None]).round_().to(torch.int8)
    return data, scale


def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    s = dict(case)
    if op == "append":
        B, T, H, HKV, HD = (case[k] for k in ("B", "T", "H", "HKV", "HD"))
        cap = (case["n"] + T + 255) // 256 * 256
        proj = _randn(g, B, T, (H + 2 * HKV) * HD).to(torch.bfloat16)    # one fused projection of the hidden states
        s.update(q=proj[..., :H * HD], k=proj[..., H * HD:(H + HKV) * HD], v=proj[..., (H + HKV) * HD:],
                 data=torch.zeros(2, B, HKV, cap, HD, device=DEV, dtype=torch.int8),
                 scale=torch.ones(2, B, HKV, cap, device=DEV), lens=_lens(case, g), inv_freq=_freqs(HD), eps=1e-6,
                 q_norm=None, k_norm=None)
        if case["norm"]:
            s["q_norm"] = 1 + 0.1 * _randn(g, HD)
            s["k_norm"] = 1 + 0.1 * _randn(g, HD)
    elif op == "read":
        s["data"], s["scale"] = _cache(g, case["B"], case["HKV"], case["cap"], case["HD"])
    elif op == "attend":
        B, T, H, HKV, HD = (case[k] for k in ("B", "T", "H", "HKV", "HD"))
        s["data"], s["scale"] = _cache(g, B, HKV, (case["n"] + T + 255) // 256 * 256, HD)
        s.update(q=_randn(g, B, T, H, HD).to(torch.bfloat16), lens=_lens(case, g), sm_scale=HD ** -0.5)
    elif op == "select":
        B, K, V = case["B"], case["K"], case["V"]
        logits = torch.empty(B * K, V, device=DEV, dtype=getattr(torch, case["dtype"]))
        for r in range(0, B * K, 16):
            logits[r:r + 16] = 3 * _randn(g, *logits[r:r + 16].shape)
        scores = -10 * torch.rand(B, K, generator=g, device=DEV)
        finished = torch.rand(B, K, generator=g, device=DEV) < 0.2
        if case["first"]:
            scores[:, 0], scores[:, 1:], finished = 0.0, -math.inf, torch.zeros_like(finished)
        s.update(logits=logits, scores=scores, finished=finished)
    else:
        B, K, HKV, HD, cap = (case[k] for k in ("B", "K", "HKV", "HD", "cap"))
        n, c = B * K, B * K * HKV

        def rows(dtype, *shape):
            raw = torch.randint(-128, 128, (math.prod(shape) * dtype.itemsize,), generator=g, device=DEV, dtype=torch.int8)
            return raw.view(dtype).view(shape) if not dtype.is_floating_point else _randn(g, *shape).to(dtype)

        # (tensor, dimension of the beams, dimension of the tokens or None for all of a beam's rows)
        items = [(rows(torch.int8, 2, n, HKV, cap, HD), 1, 3), (rows(torch.float32, 2, n, HKV, cap), 1, 3)]
        if case["layer"]:
            bf, f32 = torch.bfloat16, torch.float32
            items += [(rows(bf, c, 256, HD), 0, None) for _ in range(3)] + [(rows(f32, c, 256), 0, None)]
            items += [(rows(bf, c, 4, HD), 0, None) for _ in range(2)]
            items += [(rows(bf, c, 128, HD), 0, None) for _ in range(3)] + [(rows(f32, c, 128), 0, None) for _ in range(3)]
            items += [(rows(torch.uint8, c, 128), 0, None), (rows(torch.int32, c), 0, None)]
            items += [(rows(f32, n, HKV, HD, HD), 0, None)]
        # parents as the selection gives them: a beam that lives on keeps its slot
        pick = torch.randint(0, K, (B, K), generator=g, device=DEV)
        lives = torch.zeros(B, K, dtype=torch.bool, device=DEV).scatter_(1, pick, True)
        parent = torch.where(lives, torch.arange(K, device=DEV), pick)
        s.update(items=items, parent=parent.to(torch.int32))
    return s


# ---------------------------------------------------------------------------------------- plain forms

def _starts(s):
    return s["lens"].long() if s["lens"] is not None else torch.full((s["B"],), s["n"], device=DEV)


def _norm_rotate(x, w, eps, ang):
    """x [B, T, heads, HD] in 32 bits; ang [B, T, HD / 2]."""
    if w is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * w
    a, b = x.chunk(2, dim=-1)
    c, d = ang.cos()[:, :, None], ang.sin()[:, :, None]
    return torch.cat((a * c - b * d, b * c + a * d), dim=-1)


def _quantise(x):
    scale = (x.abs().amax(-1) / 127).clamp_min(FLOOR)
    return torch.round(x / scale[..., None]).to(torch.int8), scale


def _plain_append(s):
    B, T, H, HKV, HD = (s[k] for k in ("B", "T", "H", "HKV", "HD"))
    pos = _starts(s)[:, None] + torch.arange(T, device=DEV)
    ang = pos.float()[..., None] * s["inv_freq"]
    q = _norm_rotate(s["q"].float().view(B, T, H, HD), s["q_norm"], s["eps"], ang).to(torch.bfloat16)
    k = _norm_rotate(s["k"].float().view(B, T, HKV, HD), s["k_norm"], s["eps"], ang)
    kv = torch.stack((k, s["v"].float().view(B, T, HKV, HD)))
    x8, scale = _quantise(kv)
    b, h = torch.arange(B, device=DEV)[:, None, None], torch.arange(HKV, device=DEV)
    s["data"][:, b, h, pos[..., None]] = x8
    s["scale"][:, b, h, pos[..., None]] = scale
    back = s["data"][:, b, h, pos[..., None]].float() * s["scale"][:, b, h, pos[..., None]][..., None]
    return dict(q=q, kv=back.transpose(2, 3).to(torch.bfloat16))


def _plain_read(s):
    at = slice(s["t0"], s["t0"] + s["T"])
    return (s["data"][:, :, :, at].float() * s["scale"][:, :, :, at, None]).to(torch.bfloat16)


def _plain_attend(s):
    B, T, H, HKV, HD = (s[k] for k in ("B", "T", "H", "HKV", "HD"))
    L, G = s["n"] + T, H // HKV
    k, v = s["data"][:, :, :, :L].float() * s["scale"][:, :, :, :L, None]
    q = s["q"].float().view(B, T, HKV, G, HD).permute(0, 2, 1, 3, 4).reshape(B, HKV, T * G, HD)
    t = (q @ k.transpose(-1, -2)).view(B, HKV, T, G, L) * s["sm_scale"]
    last = _starts(s)[:, None] + torch.arange(T, device=DEV)
    seen = torch.arange(L, device=DEV) <= last[..., None]
    t = t.masked_fill_(~seen[:, None, :, None], -math.inf)
    p = torch.exp(t - t.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    y = (p.view(B, HKV, T * G, L) @ v).view(B, HKV, T, G, HD)
    return y.permute(0, 2, 1, 3, 4).reshape(B, T, H * HD).to(torch.bfloat16)


def _slots(parent, valid, K):
    """Slot of each chosen continuation [B, K] (best first): its parent's slot for the first child of
    that parent, else the lowest slots that no parent holds, in order."""
    r = torch.arange(K, device=DEV)
    same = (parent[:, :, None] == parent[:, None, :]) & valid[:, None, :] & (r[None, :] < r[:, None])
    first = valid & ~same.any(-1)
    taken = ((parent[:, :, None] == r) & first[:, :, None]).any(1)
    free = torch.argsort(taken.int(), dim=1, stable=True)
    later = valid & ~first
    at = (later.int().cumsum(1) - 1).clamp_min(0)
    return torch.where(first, parent, free.gather(1, at))


def _plain_select(s):
    B, K, V = s["B"], s["K"], s["V"]
    x = s["logits"].float().view(B, K, V)
    top = x.amax(-1, keepdim=True)
    lse = top + torch.log(torch.exp(x - top).sum(-1, keepdim=True))
    cand = s["scores"][..., None] + (x - lse)
    done = s["finished"][..., None]
    only = torch.where(torch.arange(V, device=DEV) == PAD, s["scores"][..., None], -math.inf)
    cand = torch.where(done, only, cand).view(B, K * V)
    bits = cand.view(torch.int32).long()
    key = torch.where(bits < 0, ~bits & 0xFFFFFFFF, bits | 0x80000000) - (1 << 31)      # in the order of the scores
    key = (key << 32) | (0xFFFFFFFF - torch.arange(K * V, device=DEV))                  # ties to the lowest index
    at = 0xFFFFFFFF - (torch.topk(key, K, dim=1).values & 0xFFFFFFFF)
    best = cand.gather(1, at)
    return _by_slot(s, best, at // V, at % V)


def _by_slot(s, best, parent, token):
    B, K = best.shape
    valid = best > -math.inf
    slot = _slots(parent, valid, K)
    slot = torch.where(valid, slot, K)          # what is not chosen falls into a column of its own
    idle = torch.arange(K + 1, device=DEV).expand(B, -1)
    scores = torch.full((B, K + 1), -math.inf, device=DEV, dtype=best.dtype).scatter(1, slot, best)[:, :K]
    parents = idle.scatter(1, slot, parent)[:, :K]
    tokens = torch.full((B, K + 1), PAD, device=DEV).scatter(1, slot, token)[:, :K]
    used = torch.zeros(B, K + 1, device=DEV, dtype=torch.bool).scatter(1, slot, valid)[:, :K]
    finished = ~used | (tokens == PAD)
    return dict(scores=scores, parent=parents.to(torch.int32), token=tokens, finished=finished)


def _plain_reorder(s):
    n = s["B"] * s["K"]
    src = (s["parent"].long() + torch.arange(s["B"], device=DEV)[:, None] * s["K"]).view(-1)
    for t, beams, tokens in s["items"]:
        u = t if tokens is None else t.narrow(tokens, s["t0"], s["t1"] - s["t0"])
        u = u.unflatten(beams, (n, -1))
        u.copy_(u.index_select(beams, src))
    return [t for t, _, _ in s["items"]]


PLAIN = dict(append=_plain_append, read=_plain_read, attend=_plain_attend, select=_plain_select, reorder=_plain_reorder)


# ---------------------------------------------------------------------------------------- one pass

def run(state):
    s = state
    if not own:
        return PLAIN[s["op"]](s)
    from vsa_lm_b200 import kernels as K

    if s["op"] == "append":
        q = K.kv8_append(q=s["q"], k=s["k"], v=s["v"], data=s["data"], scale=s["scale"], n=s["n"], pos0=s["n"],
                         inv_freq=s["inv_freq"], q_norm=s["q_norm"], k_norm=s["k_norm"], eps=s["eps"], lens=s["lens"])
        return dict(q=q, kv=K.kv8_read(s["data"], s["scale"], s["n"], s["T"], lens=s["lens"]))
    if s["op"] == "read":
        return K.kv8_read(s["data"], s["scale"], s["t0"], s["T"])
    if s["op"] == "attend":
        return K.kv8_attend(q=s["q"], data=s["data"], scale=s["scale"], n=s["n"], sm_scale=s["sm_scale"],
                            lens=s["lens"])
    if s["op"] == "select":
        scores, parent, token, finished = K.beam_select(s["logits"], s["scores"], s["finished"], eos_ids=(PAD,))
        return dict(scores=scores, parent=parent, token=token, finished=finished)
    K.beam_reorder(s["items"], s["parent"], t0=s["t0"], t1=s["t1"])
    return [t for t, _, _ in s["items"]]


# ---------------------------------------------------------------------------------------- floors and 64 bits

def work(case):
    c = case
    if c["op"] == "append":
        rows, HD = c["B"] * c["T"], c["HD"]
        kv = 2 * c["HKV"]
        # projections in, queries out, the cache's rows and scales written, and those read back as bf16
        return dict(bytes=rows * ((2 * c["H"] + kv) * HD * 2 + 2 * kv * (HD + 4) + kv * HD * 2),
                    flops=rows * (c["H"] + kv) * HD * 10)
    if c["op"] == "read":
        rows = 2 * c["B"] * c["HKV"] * c["T"]
        return dict(bytes=rows * (c["HD"] * 3 + 4), flops=rows * c["HD"])
    if c["op"] == "attend":
        # a ragged batch holds three quarters of the longest on average
        n = c["n"] * (0.75 if c["ragged"] else 1.0)
        keys, rows = c["B"] * c["HKV"] * (n + c["T"]), c["B"] * c["T"] * c["H"]
        return dict(bytes=keys * 2 * (c["HD"] + 4) + rows * c["HD"] * 4, flops=rows * (n + (c["T"] + 1) / 2) * c["HD"] * 4)
    if c["op"] == "select":
        rows = c["B"] * c["K"] * (1.0 if c["first"] else 0.8)     # a finished beam's logits are not needed
        return dict(bytes=rows * c["V"] * (4 if c["dtype"] == "float32" else 2) + c["B"] * c["K"] * 32,
                    flops=rows * c["V"] * 4)
    K, HKV, HD, span = c["K"], c["HKV"], c["HD"], c["t1"] - c["t0"]
    per = 2 * HKV * span * (HD + 4)
    if c["layer"]:
        per += HKV * (3 * 256 * HD * 2 + 256 * 4 + 8 * HD * 2 + 3 * 128 * HD * 2 + 3 * 512 + 128 + 4 + HD * HD * 4)
    moved = c["B"] * K * (1 - 1 / K) ** K                         # the slots that no parent holds, on average
    kept = c["B"] * K * (1 - (1 - 1 / K) ** K)                    # parents read: at most one for each moved slot
    return dict(bytes=(moved + min(moved, kept)) * per, flops=0)


def exact(case, seed):
    s = prepare(case, seed)

    def in_64_append():
        B, T, HKV, HD = s["B"], s["T"], s["HKV"], s["HD"]
        start = [s["n"]] * B if s["lens"] is None else s["lens"].tolist()
        pos = torch.tensor([[p + t for t in range(T)] for p in start], device=DEV, dtype=torch.float64)
        turn = torch.polar(torch.ones(B, T, 1, HD // 2, device=DEV, dtype=torch.float64),
                           (pos[..., None] * s["inv_freq"].double())[:, :, None])

        def heads(x, w):
            x = x.double().reshape(B, T, -1, HD)
            if w is not None:
                x = x / (x.pow(2).sum(-1, keepdim=True) / HD + s["eps"]).sqrt() * w.double()
            z = torch.complex(x[..., :HD // 2], x[..., HD // 2:]) * turn
            return torch.cat((z.real, z.imag), -1)

        def stored(x):
            step = torch.clamp(x.abs().max(-1, keepdim=True).values / 127, min=FLOOR)
            return (torch.round(x / step) * step).permute(0, 2, 1, 3)

        v = s["v"].double().reshape(B, T, HKV, HD)
        return dict(q=heads(s["q"], s["q_norm"]), kv=torch.stack((stored(heads(s["k"], s["k_norm"])), stored(v))))

    def in_64_attend():
        B, T, H, HKV, HD = (s[k] for k in ("B", "T", "H", "HKV", "HD"))
        y = torch.empty(B, T, H, HD, device=DEV, dtype=torch.float64)
        for b in range(B):
            n = s["n"] if s["lens"] is None else int(s["lens"][b])
            k, v = s["data"][:, b, :, :n + T].double() * s["scale"][:, b, :, :n + T, None].double()
            late = torch.ones(T, n + T, device=DEV, dtype=torch.bool).triu(n + 1)
            for h in range(HKV):
                q = s["q"][b, :, h * (H // HKV):(h + 1) * (H // HKV)].double()
                t = torch.einsum("tgd,ld->gtl", q, k[h]) * s["sm_scale"]
                p = torch.softmax(t.masked_fill(late, -math.inf), -1)
                y[b, :, h * (H // HKV):(h + 1) * (H // HKV)] = torch.einsum("gtl,ld->tgd", p, v[h])
        return y.view(B, T, H * HD)

    def in_64_select():
        B, K, V = s["B"], s["K"], s["V"]
        out = torch.full((B, K), -math.inf, device=DEV, dtype=torch.float64)
        for b in range(B):
            row = torch.log_softmax(s["logits"][b * K:(b + 1) * K].double(), -1) + s["scores"][b, :, None].double()
            row[s["finished"][b]] = -math.inf
            row[s["finished"][b], PAD] = s["scores"][b][s["finished"][b]].double()
            score, at = torch.sort(row.view(-1), descending=True, stable=True)
            chosen = [(float(score[i]), int(at[i]) // V) for i in range(K) if float(score[i]) > -math.inf]
            homes, left = {}, []
            for value, p in chosen:
                if p in homes:
                    left.append(value)
                else:
                    homes[p] = value
            spare = [i for i in range(K) if i not in homes]
            homes.update(zip(spare, left))
            for i, value in homes.items():
                out[b, i] = value
        return dict(scores=out, parent=None, token=None, finished=None)

    def in_64_reorder():
        K, n = s["K"], s["B"] * s["K"]
        out = []
        for t, beams, tokens in s["items"]:
            if not t.is_floating_point():
                out.append(None)
                continue
            u = t.double().movedim(beams, 0).clone()
            r = u.shape[0] // n
            was = u.clone()
            at = slice(None) if tokens is None else slice(s["t0"], s["t1"])
            for i in range(n):
                p = i // K * K + int(s["parent"].view(-1)[i])
                to, frm = u[i * r:(i + 1) * r], was[p * r:(p + 1) * r]
                if tokens is None:
                    to.copy_(frm)
                else:
                    to[..., at].copy_(frm[..., at])
            out.append(u.movedim(0, beams))
        return out

    def in_64_read():
        at = slice(s["t0"], s["t0"] + s["T"])
        return s["data"][:, :, :, at].double() * s["scale"][:, :, :, at, None].double()

    return dict(append=in_64_append, read=in_64_read, attend=in_64_attend, select=in_64_select,
                reorder=in_64_reorder)[case["op"]]()
