"""Attention, rotary positions and paged attention: the calls that are timed,
their plain forms and their values in 64 bits.

`listed()` names the cases, `draw(rng)` gives more of the same ranges,
`prepare(case, seed)` makes a case's inputs on the GPU, `run(state)` makes one
call -- the plain form in 32-bit torch operations, or with `own` set the
package's operator -- and `exact(case, seed)` gives the same outputs from the
definition in 64 bits.

Definitions. Query i stands at position i + Lk - Lq, key j at position j.
    t[i, j] = scale * q[i] . k[j]
    s[i, j] = cap * tanh(t / cap) - slope[h] * |position(i) - j|   (cap > 0, else t)
Key j is seen by query i if (not causal, or j <= position(i), or
j < prefix[b]) and (no documents, or both carry the same id >= 0).
    lse[i] = log sum_j exp(s[i, j]),  out[i] = sum_j exp(s[i, j] - lse[i]) v[j]
over the seen keys; a query that sees none gives out = 0 and lse = -inf.
"""
import math
import random

import numpy as np
import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}


# ------------------------------------------------------------------ cases
def _attention(name, op, dtype, B, H, Hkv, Lq, Lk, D, causal=True, cap=0.0, slopes=False, documents=0, padding=0,
               prefix=False):
    return dict(name=name, op=op, dtype=dtype, B=B, H=H, Hkv=Hkv, Lq=Lq, Lk=Lk, D=D, causal=causal, cap=cap,
                slopes=slopes, documents=documents, padding=padding, prefix=prefix)


def _rotary(name, dtype, B, L, H, Hkv, D, part, interleaved, inverse, scaling, far):
    return dict(name=name, op="rotary", dtype=dtype, B=B, L=L, H=H, Hkv=Hkv, D=D, part=part,
                interleaved=interleaved, inverse=inverse, scaling=scaling, far=far)


def _paged(name, dtype, B, H, Hkv, shortest, longest, page, D, cap=0.0, slopes=False, append=True):
    return dict(name=name, op="paged", dtype=dtype, B=B, H=H, Hkv=Hkv, shortest=shortest, longest=longest, page=page,
                D=D, cap=cap, slopes=slopes, append=append)


def listed():
    bf, fp = "bfloat16", "float32"
    return [
        # the attention of the decoder that the training step is measured on (batch 64 x 256, 6 heads of 64), in its
        # own type, with a bias by distance in place of learnt positions
        _attention("forward decoder", "forward", fp, 64, 6, 6, 256, 256, 64, slopes=True),
        # a long text: capped scores, four query heads to each key-value head
        _attention("forward long capped", "forward", bf, 1, 16, 4, 8192, 8192, 128, cap=50.0),
        # a training batch of several documents packed into each row, of an odd length
        _attention("forward packed", "forward", bf, 3, 12, 12, 4001, 4001, 64, documents=7, padding=33),
        # the gradients of the same three kinds of call; the packed one with a prefix that sees both ways
        _attention("backward decoder", "backward", fp, 64, 6, 6, 256, 256, 64, slopes=True),
        _attention("backward long capped", "backward", bf, 1, 16, 4, 8192, 8192, 128, cap=50.0),
        _attention("backward packed prefix", "backward", bf, 2, 12, 12, 2047, 2047, 64, documents=3, padding=9,
                   prefix=True),
        # one new token for each of 64 running requests at far positions: latency
        _rotary("rotary token", bf, 64, 1, 32, 8, 128, 128, False, False, "parts", 100000),
        # the decoder's batch, part of each head, neighbouring pairs
        _rotary("rotary decoder", fp, 64, 256, 6, 6, 64, 32, True, False, "none", 0),
        # gradients of a long training batch
        _rotary("rotary long gradient", bf, 2, 8192, 32, 8, 128, 128, False, True, "linear", 0),
        # one request's next token: latency
        _paged("paged single", bf, 1, 32, 8, 1000, 1000, 16, 128),
        # the next token of a batch of requests of very different lengths
        _paged("paged ragged batch", bf, 32, 32, 8, 1, 8192, 16, 128, cap=30.0),
        # two requests with very long contexts: work split over the length
        _paged("paged long", fp, 2, 6, 6, 99001, 100003, 64, 64, slopes=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["forward", "forward", "backward", "backward", "rotary", "paged", "paged"])
    heads = rng.choice([(1, 1), (4, 1), (6, 6), (12, 12), (8, 2), (12, 4), (16, 4), (16, 16)])
    if op in ("forward", "backward"):
        dtype = rng.choice(["float32", "bfloat16", "bfloat16"])
        D = rng.choice([32, 64, 64, 80, 96, 128, 128])
        Lk = _log(rng, 1 if op == "forward" else 16, 1200 if dtype == "float32" else 8000)
        Lq = rng.choice([Lk, Lk, Lk, 1, rng.randint(1, Lk)])
        pairs = (100 if dtype == "float32" else 700) * 10 ** 6
        B = _log(rng, 1, max(1, min(64, pairs // (heads[0] * Lq * Lk), 2 ** 24 // (heads[0] * Lk))))
        documents = rng.choice([0, 0, rng.randint(1, 9)]) if Lk >= 64 else 0
        causal = rng.random() < 0.8
        return _attention("", op, dtype, B, heads[0], heads[1], Lq, Lk, D, causal=causal,
                          cap=rng.choice([0.0, 20.0, 50.0]), slopes=rng.random() < 0.4, documents=documents,
                          padding=rng.randint(0, Lk // 8) if documents else 0, prefix=causal and rng.random() < 0.3)
    if op == "rotary":
        D = rng.choice([64, 80, 128])
        L = _log(rng, 1, 8192)
        B = _log(rng, 1, max(1, min(128, 16384 // L)))
        return _rotary("", rng.choice(["float32", "bfloat16"]), B, L, heads[0], heads[1], D,
                       rng.choice([D, D, D // 2, 24]), rng.random() < 0.5, rng.random() < 0.5,
                       rng.choice(["none", "linear", "ntk", "parts"]), rng.choice([0, 5000, 1000000]))
    longest = _log(rng, 1, 60000)
    B = _log(rng, 1, max(1, min(64, 200000 // longest)))
    return _paged("", rng.choice(["float32", "bfloat16", "bfloat16"]), B, heads[0], heads[1],
                  rng.randint(0, longest), longest, rng.choice([1, 8, 16, 24, 64, 256]), rng.choice([64, 96, 128]),
                  cap=rng.choice([0.0, 30.0]), slopes=rng.random() < 0.4, append=rng.random() < 0.7)


# ------------------------------------------------------------------ inputs
def _document_ids(case, seed):
    """[B, Lk] ids: each row is cut into documents of uneven lengths, in an order that goes by the seed, with
    `padding` positions of id -1 at its end."""
    rng = random.Random(seed)
    B, L, n = case["B"], case["Lk"] - case["padding"], case["documents"]
    parts = [1 + (3 * i) % 5 for i in range(n)]
    ids = np.full((B, case["Lk"]), -1, np.int32)
    for b in range(B):
        order = parts[:]
        rng.shuffle(order)
        at, total = 0, sum(order)
        for i, p in enumerate(order):
            end = L if i == n - 1 else min(L, at + L * p // total)
            ids[b, at:end] = i
            at = end
    return ids


def _prefixes(case, seed):
    """[B] lengths of the rows' prefixes, in an order that goes by the seed."""
    B, L = case["B"], case["Lk"]
    lengths = [L * (b + 1) // (2 * B + 1) for b in range(B)]
    random.Random(seed + 1).shuffle(lengths)
    return np.array(lengths, np.int32)


def _slopes(H):
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / H) for h in range(H)], dtype=torch.float32, device="cuda")


def _normal(g, shape, dtype, gain=1.0):
    return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * gain).to(DTYPES[dtype])


def _frequencies(case):
    """Radians a position of each rotated pair, in the scalings that long contexts use."""
    n = case["part"] // 2
    theta, factor, trained = 10000.0, 8.0, 4096.0
    if case["scaling"] == "ntk":
        theta *= factor ** (case["part"] / max(1, case["part"] - 2))
    f = theta ** (-torch.arange(n, dtype=torch.float64) * 2 / case["part"])
    if case["scaling"] == "linear":
        f = f / factor
    if case["scaling"] == "parts":  # slow pairs are stretched, fast ones kept, with a ramp between 1 and 32 turns
        turns = trained * f / (2 * math.pi)
        keep = ((turns - 1.0) / 31.0).clamp(0, 1)
        f = f * keep + f / factor * (1 - keep)
    return f.cuda()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case=case)
    dt = case["dtype"]
    B, H, Hkv, D = case["B"], case["H"], case["Hkv"], case["D"]
    if case["op"] in ("forward", "backward"):
        Lq, Lk = case["Lq"], case["Lk"]
        # views of [B, L, heads * D] activations, as the projections leave them
        s["q"] = _normal(g, (B, Lq, H, D), dt, 3.0 if case["cap"] else 1.0).transpose(1, 2)
        s["k"] = _normal(g, (B, Lk, Hkv, D), dt).transpose(1, 2)
        s["v"] = _normal(g, (B, Lk, Hkv, D), dt).transpose(1, 2)
        s["slopes"] = _slopes(H) if case["slopes"] else None
        s["documents"] = torch.from_numpy(_document_ids(case, seed)).cuda() if case["documents"] else None
        s["prefix"] = torch.from_numpy(_prefixes(case, seed)).cuda() if case["prefix"] else None
        if case["op"] == "backward":
            s["dout"] = _normal(g, (B, Lq, H, D), dt).transpose(1, 2)
            s["out"], s["lse"] = _plain_forward(s)
    elif case["op"] == "rotary":
        L = case["L"]
        s["q"] = _normal(g, (B, L, H, D), dt).transpose(1, 2)
        s["k"] = _normal(g, (B, L, Hkv, D), dt).transpose(1, 2)
        start = torch.randint(0, case["far"] + 1, (B, 1), generator=g, device="cuda")
        s["positions"] = (start + torch.arange(L, device="cuda")).to(torch.int32)
        s["frequencies"] = _frequencies(case)
    else:
        page, longest = case["page"], case["longest"]
        rng = random.Random(seed)
        if B == 1:
            lengths = [longest]
        else:
            lengths = [case["shortest"] + (longest - case["shortest"]) * b // (B - 1) for b in range(B)]
            rng.shuffle(lengths)
        width = -(-longest // page)
        pages = B * width + 3
        order = torch.randperm(pages, generator=g, device="cuda")[:B * width].to(torch.int32)
        s["block_table"] = order.view(B, width)
        s["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        s["k_pages"] = _normal(g, (pages, page, Hkv, D), dt)
        s["v_pages"] = _normal(g, (pages, page, Hkv, D), dt)
        s["q"] = _normal(g, (B, H, D), dt, 3.0 if case["cap"] else 1.0)
        s["slopes"] = _slopes(H) if case["slopes"] else None
        s["k_new"] = _normal(g, (B, Hkv, D), dt) if case["append"] else None
        s["v_new"] = _normal(g, (B, Hkv, D), dt) if case["append"] else None
    return s


# ------------------------------------------------------------------ plain forms
def _seen(case, documents, prefix, device):
    """[B or 1, Lq, Lk] truth values: which keys each query sees."""
    Lq, Lk = case["Lq"], case["Lk"]
    at = torch.arange(Lq, device=device) + (Lk - Lq)
    j = torch.arange(Lk, device=device)
    seen = torch.ones((1, Lq, Lk), dtype=torch.bool, device=device)
    if case["causal"]:
        seen = (j[None, :] <= at[:, None])[None]
        if prefix is not None:
            seen = seen | (j[None, None, :] < prefix[:, None, None])
    if documents is not None:
        mine = documents[:, Lk - Lq:]
        seen = seen & (mine[:, :, None] == documents[:, None, :]) & (mine >= 0)[:, :, None]
    return seen


def _scores(s, q, k, wide):
    """Scores with masked places at -inf, and tanh(t / cap)."""
    case = s["case"]
    t = torch.matmul(q, k.transpose(-1, -2)) * (1.0 / math.sqrt(case["D"]))
    bend = None
    if case["cap"]:
        bend = torch.tanh(t / case["cap"])
        t = bend * case["cap"]
    if s["slopes"] is not None:
        at = torch.arange(case["Lq"], device=t.device) + (case["Lk"] - case["Lq"])
        far = (at[:, None] - torch.arange(case["Lk"], device=t.device)[None, :]).abs().to(wide)
        t = t - s["slopes"].to(wide)[None, :, None, None] * far
    seen = _seen(case, s["documents"], s["prefix"], t.device)[:, None]
    return t.masked_fill(~seen, -math.inf), bend


def _softmax(t):
    """exp(t - lse) and lse of each row, 0 and -inf where nothing is seen."""
    top = t.amax(-1, keepdim=True)
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    e = torch.exp(t - top)
    total = e.sum(-1, keepdim=True)
    p = e / torch.where(total > 0, total, torch.ones_like(total))
    return p, (top + torch.log(total)).squeeze(-1)


def _heads(x, H):
    return x.repeat_interleave(H // x.shape[1], dim=1)


def _plain_forward(s):
    case = s["case"]
    q, k, v = (s[n].float() for n in ("q", "k", "v"))
    t, _ = _scores(s, q, _heads(k, case["H"]), torch.float32)
    p, lse = _softmax(t)
    return torch.matmul(p, _heads(v, case["H"])).to(s["q"].dtype), lse


def _plain_backward(s):
    case = s["case"]
    B, H, Hkv, D = case["B"], case["H"], case["Hkv"], case["D"]
    q, k, v, dout = (s[n].float() for n in ("q", "k", "v", "dout"))
    k, v = _heads(k, H), _heads(v, H)
    t, bend = _scores(s, q, k, torch.float32)
    p, _ = _softmax(t)
    del t
    dv = torch.matmul(p.transpose(-1, -2), dout)
    dp = torch.matmul(dout, v.transpose(-1, -2))
    ds = p * (dp - (p * dp).sum(-1, keepdim=True))
    del dp, p
    if bend is not None:
        ds = ds * (1 - bend * bend)
    ds = ds * (1.0 / math.sqrt(D))
    dq = torch.matmul(ds, k)
    dk = torch.matmul(ds.transpose(-1, -2), q)
    dk, dv = (x.view(B, Hkv, H // Hkv, -1, D).sum(2) for x in (dk, dv))
    return tuple(x.to(s["q"].dtype) for x in (dq, dk, dv))


def _rotate(x, cos, sin, part, interleaved):
    """Pairs of the first `part` of each head turned by the angles, the rest as it is."""
    head, rest = x[..., :part], x[..., part:]
    a, b = (head[..., 0::2], head[..., 1::2]) if interleaved else (head[..., :part // 2], head[..., part // 2:])
    y = (a * cos - b * sin, a * sin + b * cos)
    y = torch.stack(y, -1).flatten(-2) if interleaved else torch.cat(y, -1)
    return torch.cat([y, rest], -1)


def _plain_rotary(s):
    case = s["case"]
    angle = s["positions"].double()[:, None, :, None] * s["frequencies"]
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    if case["inverse"]:
        sin = -sin
    return tuple(_rotate(s[n].float(), cos, sin, case["part"], case["interleaved"]).to(s[n].dtype) for n in ("q", "k"))


def _plain_append(s):
    """Each request's new key and value go to its last position."""
    case, lengths = s["case"], s["lengths"].long()
    live = (lengths > 0).nonzero().squeeze(-1)
    last = lengths[live] - 1
    page = s["block_table"][live, last // case["page"]].long()
    s["k_pages"][page, last % case["page"]] = s["k_new"][live]
    s["v_pages"][page, last % case["page"]] = s["v_new"][live]


def _plain_paged(s):
    case = s["case"]
    B, H, Hkv, D, G = case["B"], case["H"], case["Hkv"], case["D"], case["H"] // case["Hkv"]
    if case["append"]:
        _plain_append(s)
    k, v = (s[n][s["block_table"].long()].flatten(1, 2).float() for n in ("k_pages", "v_pages"))
    q = s["q"].float().view(B, Hkv, G, D)
    t = torch.matmul(q, k.permute(0, 2, 3, 1)) * (1.0 / math.sqrt(D))
    if case["cap"]:
        t = torch.tanh(t / case["cap"]) * case["cap"]
    j = torch.arange(t.shape[-1], device=t.device)
    far = s["lengths"][:, None] - 1 - j[None, :]
    if s["slopes"] is not None:
        t = t - s["slopes"].view(1, Hkv, G, 1) * far.float()[:, None, None, :]
    p, lse = _softmax(t.masked_fill((far < 0)[:, None, None, :], -math.inf))
    out = torch.matmul(p, v.transpose(1, 2)).view(B, H, D).to(s["q"].dtype)
    return _paged_outputs(s, out, lse.view(B, H))


def _paged_outputs(s, out, lse):
    return (out, lse, s["k_pages"], s["v_pages"]) if s["case"]["append"] else (out, lse)


# ------------------------------------------------------------------ one pass
def run(state):
    s, case = state, state["case"]
    if not own:
        return {"forward": _plain_forward, "backward": _plain_backward, "rotary": _plain_rotary,
                "paged": _plain_paged}[case["op"]](s)
    import macrograd_b200 as mg

    if case["op"] == "forward":
        return mg.attention(s["q"], s["k"], s["v"], causal=case["causal"], cap=case["cap"], slopes=s["slopes"],
                            documents=s["documents"], prefix=s["prefix"])
    if case["op"] == "backward":
        return mg.attention_backward(s["dout"], s["q"], s["k"], s["v"], s["out"], s["lse"], causal=case["causal"],
                                     cap=case["cap"], slopes=s["slopes"], documents=s["documents"],
                                     prefix=s["prefix"])
    if case["op"] == "rotary":
        turn = mg.rotary_backward if case["inverse"] else mg.rotary
        return turn(s["q"], s["k"], s["positions"], s["frequencies"], interleaved=case["interleaved"])
    return _paged_outputs(s, *mg.paged_attention(s["q"], s["k_pages"], s["v_pages"], s["block_table"], s["lengths"],
                                                 cap=case["cap"], slopes=s["slopes"], k_new=s["k_new"],
                                                 v_new=s["v_new"]))


# ------------------------------------------------------------------ least work
def _pairs(case):
    """Seen (query, key) pairs of all rows of the batch, for one head."""
    B, Lq, Lk = case["B"], case["Lq"], case["Lk"]
    at = np.arange(Lq, dtype=np.int64) + (Lk - Lq)
    ids = _document_ids(case, 0) if case["documents"] else np.zeros((B, Lk), np.int32)
    prefix = _prefixes(case, 0) if case["prefix"] else np.zeros(B, np.int32)
    total = 0
    for b in range(B):
        for d in np.unique(ids[b]):
            if d < 0:
                continue
            where = np.nonzero(ids[b] == d)[0]
            mine = at[(at >= where[0]) & (at <= where[-1])]
            if not case["causal"]:
                total += len(mine) * len(where)
                continue
            upto = np.maximum(mine + 1, min(int(prefix[b]), Lk))  # keys before this position are seen
            total += int(np.clip(np.minimum(upto, where[-1] + 1) - where[0], 0, None).sum())
    return total


def work(case):
    e = 2 if case["dtype"] == "bfloat16" else 4
    B, H, Hkv, D = case["B"], case["H"], case["Hkv"], case["D"]
    if case["op"] in ("forward", "backward"):
        rows, keys = B * H * case["Lq"], B * Hkv * case["Lk"]
        masks = 4 * (B * case["Lk"] * bool(case["documents"]) + B * case["prefix"] + H * case["slopes"])
        if case["op"] == "forward":  # q, k, v in; out, lse out; two products
            return {"bytes": e * D * (2 * rows + 2 * keys) + 4 * rows + masks, "flops": 4 * D * H * _pairs(case)}
        # q, k, v, out, dout, lse in; dq, dk, dv out; five products
        return {"bytes": e * D * (4 * rows + 4 * keys) + 4 * rows + masks, "flops": 10 * D * H * _pairs(case)}
    if case["op"] == "rotary":
        heads = B * case["L"] * (H + Hkv)
        return {"bytes": 2 * e * D * heads + 4 * B * case["L"] + 4 * case["part"], "flops": 3 * case["part"] * heads}
    span = case["longest"] - case["shortest"]
    keys = case["longest"] if B == 1 else sum(case["shortest"] + span * b // (B - 1) for b in range(B))
    new = 4 * e * D * B * Hkv if case["append"] else 0
    return {"bytes": 2 * e * D * Hkv * keys + 2 * e * D * B * H + 4 * B * H + 4 * (keys // case["page"]) + 4 * B + new,
            "flops": 4 * D * H * keys}


# ------------------------------------------------------------------ values in 64 bits
def _exact_attention(case, s):
    """Head by head in 64 bits, each score from its definition."""
    B, H, Hkv, Lq, Lk, D = (case[n] for n in ("B", "H", "Hkv", "Lq", "Lk", "D"))
    outs = [torch.zeros((B, H, Lq, D), dtype=torch.float64, device="cuda")]
    if case["op"] == "forward":
        outs.append(torch.full((B, H, Lq), -math.inf, dtype=torch.float64, device="cuda"))
    else:
        outs += [torch.zeros((B, Hkv, Lk, D), dtype=torch.float64, device="cuda") for _ in range(2)]
    i = torch.arange(Lk - Lq, Lk, device="cuda").view(-1, 1)
    j = torch.arange(Lk, device="cuda").view(1, -1)
    for b in range(B):
        hidden = (j > i) if case["causal"] else torch.zeros((Lq, Lk), dtype=torch.bool, device="cuda")
        if case["causal"] and case["prefix"]:
            hidden = hidden & ~(j < int(s["prefix"][b]))
        if case["documents"]:
            ids = s["documents"][b]
            hidden = hidden | (ids[Lk - Lq:].view(-1, 1) != ids.view(1, -1)) | (ids.view(1, -1) < 0)
        for h in range(H):
            kv = h * Hkv // H
            q, k, v = s["q"][b, h].double(), s["k"][b, kv].double(), s["v"][b, kv].double()
            x = q @ k.T / math.sqrt(D)
            curve = None
            if case["cap"]:
                x = torch.tanh(x / case["cap"])
                curve = 1 - x ** 2
                x = case["cap"] * x
            if case["slopes"]:
                x = x - s["slopes"][h].double() * (i - j).abs()
            x = torch.where(hidden, torch.full_like(x, -math.inf), x)
            lse = torch.logsumexp(x, -1)
            p = torch.where(hidden, torch.zeros_like(x), torch.exp(x - lse.unsqueeze(-1)))
            if case["op"] == "forward":
                outs[0][b, h], outs[1][b, h] = p @ v, lse
                continue
            g = s["dout"][b, h].double()
            outs[2][b, kv] += p.T @ g
            dx = g @ v.T
            dx = p * (dx - (p * dx).sum(-1, keepdim=True)) / math.sqrt(D)
            if curve is not None:
                dx = dx * curve
            outs[0][b, h] = dx @ k
            outs[1][b, kv] += dx.T @ q
    return tuple(outs)


def _exact_rotary(case, s):
    """Each pair as a complex number times exp(i angle)."""
    angle = s["positions"].double().unsqueeze(-1) * _frequencies(case)
    turn = torch.polar(torch.ones_like(angle), -angle if case["inverse"] else angle).unsqueeze(1)
    got = []
    for x in (s["q"].double(), s["k"].double()):
        part, y = case["part"], x.clone()
        first = slice(0, part, 2) if case["interleaved"] else slice(0, part // 2)
        second = slice(1, part, 2) if case["interleaved"] else slice(part // 2, part)
        z = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * turn
        y[..., first], y[..., second] = z.real, z.imag
        got.append(y)
    return tuple(got)


def _exact_paged(case, s):
    """Request by request in 64 bits."""
    B, H, Hkv, D = (case[n] for n in ("B", "H", "Hkv", "D"))
    out = torch.zeros((B, H, D), dtype=torch.float64, device="cuda")
    lse = torch.full((B, H), -math.inf, dtype=torch.float64, device="cuda")
    for b, n in enumerate(s["lengths"].tolist()):
        if n == 0:
            continue
        rows = s["block_table"][b, :-(-n // case["page"])].long()
        k, v = (s[x][rows].reshape(-1, Hkv, D)[:n].double() for x in ("k_pages", "v_pages"))
        if case["append"]:
            k[-1], v[-1] = s["k_new"][b].double(), s["v_new"][b].double()
            s["k_pages"][rows[-1], (n - 1) % case["page"]] = s["k_new"][b]
            s["v_pages"][rows[-1], (n - 1) % case["page"]] = s["v_new"][b]
        x = torch.einsum("gmd,ngd->gmn", s["q"][b].double().view(Hkv, H // Hkv, D), k) / math.sqrt(D)
        if case["cap"]:
            x = case["cap"] * torch.tanh(x / case["cap"])
        if case["slopes"]:
            back = torch.arange(n - 1, -1, -1, dtype=torch.float64, device="cuda")
            x = x - s["slopes"].double().view(Hkv, -1, 1) * back
        lse[b] = torch.logsumexp(x, -1).view(H)
        out[b] = torch.einsum("gmn,ngd->gmd", torch.softmax(x, -1), v).reshape(H, D)
    return (out, lse, None, None) if case["append"] else (out, lse)


def exact(case, seed):
    s = prepare(case, seed)
    return {"rotary": _exact_rotary, "paged": _exact_paged}.get(case["op"], _exact_attention)(case, s)
