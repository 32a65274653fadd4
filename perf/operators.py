"""Measured cases of the operators of a paged key/value cache: the plan that hands out pages, the norm / rotation / append of new rows,
the attention of ragged chunks over the pages, and the check of drafted tokens.

`own` false: the operators in their plain form (elementary torch operations in 32 bits, or 64 where that matters); `own` true: the
framework's entry points.  Shapes are those of the repository's configurations (head sizes 64 and 128, 8 to 32 heads, vocabularies of 32000
and 50257) or generic.
"""
import math
import random

import torch

own = False

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
SIZE = {"f16": 2, "bf16": 2, "f32": 4}


# ------------------------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # the pages of eight chats that verify five tokens each, and of a thousand requests with prompts among them
        dict(name="plan_8", op="plan", B=8, T=2000, n=5, page=16),
        dict(name="plan_1024", op="plan", B=1024, T=8192, n=120, page=16),
        # new rows on their way into the cache: a step of eight sequences of the 7B-class model, a prompt pass of the 1B-class model, an fp32 model
        dict(name="rope_8", op="rope", dtype="f16", rows=8, H=32, Hkv=8, hd=128, page=16, T=4000, rot=128, style=1, norm=True),
        dict(name="rope_16k", op="rope", dtype="bf16", rows=16384, H=32, Hkv=8, hd=64, page=32, T=16384, rot=64, style=2, norm=True),
        dict(name="rope_f32", op="rope", dtype="f32", rows=2036, H=8, Hkv=8, hd=64, page=16, T=131072, rot=32, style=1, norm=False),
        # one chat of the 7B-class model; 64 requests of different lengths; drafts of four tokens over long contexts of the 1B-class model;
        # two chunks of long prompts; an fp32 model with a window
        dict(name="token_1", op="attention", dtype="f16", B=1, H=32, Hkv=8, hd=128, page=16, T=530, n=1, window=0),
        dict(name="token_64", op="attention", dtype="f16", B=64, H=32, Hkv=8, hd=128, page=16, T=4096, n=1, window=0),
        dict(name="draft_16", op="attention", dtype="bf16", B=16, H=32, Hkv=8, hd=64, page=32, T=16384, n=5, window=0),
        dict(name="chunk_2k", op="attention", dtype="bf16", B=2, H=32, Hkv=8, hd=128, page=16, T=32768, n=2048, window=0),
        dict(name="chunk_f32", op="attention", dtype="f32", B=4, H=8, Hkv=8, hd=64, page=16, T=1000, n=200, window=256),
        # four drafted tokens of one chat; seven of each of 64
        dict(name="verify_1", op="verify", B=1, K=4, V=32000, draft=True),
        dict(name="verify_64", op="verify", B=64, K=7, V=50257, draft=True),
    ]


def _log(rng, a, b):
    return min(b, max(a, int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))))


def draw(rng):
    op = rng.choice(("plan", "rope", "attention", "attention", "attention", "verify"))
    page = rng.choice((8, 16, 16, 32, 64, 128))
    if op == "plan":
        return dict(op=op, B=_log(rng, 1, 1024), T=_log(rng, 40, 8192), n=_log(rng, 1, 120), page=rng.choice((16, 32, 64, 128)))
    if op == "verify":
        return dict(op=op, B=_log(rng, 1, 64), K=rng.randint(1, 7), V=_log(rng, 500, 50257), draft=rng.random() < 0.8)
    dtype = rng.choice(("f16", "bf16", "f16", "bf16", "f32"))
    hd = rng.choice((64, 128))
    Hkv = rng.choice((1, 2, 4, 8))
    H = Hkv * rng.choice((1, 2, 3, 4, 8) if Hkv < 8 else (1, 2, 4))
    if op == "rope":
        style = rng.choice((1, 2))
        return dict(op=op, dtype=dtype, rows=_log(rng, 1, 8000), H=H, Hkv=Hkv, hd=hd, page=page, T=_log(rng, 8000, 131072), rot=rng.choice((hd, hd, hd // 2)),
                    style=style, norm=rng.random() < 0.7)
    kind = rng.choice(("token", "draft", "chunk"))
    if kind == "token":
        B, n, T = _log(rng, 1, 64), 1, _log(rng, 1, 4096)
    elif kind == "draft":
        B, n, T = _log(rng, 1, 16), rng.randint(2, 9), _log(rng, 20, 16384)
    else:
        B, n, T = rng.randint(1, 3), _log(rng, 30, 700), _log(rng, 700, 12000)
        if dtype == "f32":
            T = min(T, 3000)
    return dict(op=op, dtype=dtype, B=B, H=H, Hkv=Hkv, hd=hd, page=page, T=T, n=min(n, T), window=rng.choice((0, 0, 0, _log(rng, 16, 4096))))


def lengths(case):
    """(tokens cached before, new tokens) of every sequence: ragged, the first one is the longest, and the same for every seed."""
    rng = random.Random(case["T"] * 7 + case["B"])
    T, n, B = case["T"], case["n"], case["B"]
    new = [n] + [n if n < 16 else rng.randint(max(1, n // 2), n) for _ in range(B - 1)]
    total = [T] + [rng.randint(max(1, T // 4), T) for _ in range(B - 1)]
    total = [max(t, m) for t, m in zip(total, new)]
    return [t - m for t, m in zip(total, new)], new


def _pages(tokens, page):
    return -(-tokens // page)


def _visible(case):
    """For every sequence the number of (query, key) pairs that see each other, and the keys that some query sees."""
    out = []
    for old, n in zip(*lengths(case)):
        w = case["window"] or (old + n)
        seen = sum(min(old + i + 1, w) for i in range(n))
        out.append((seen, min(old + n, w + n - 1)))
    return out


def work(case):
    op = case["op"]
    if op == "plan":
        old, new = lengths(case)
        grow = sum(_pages(a + b, case["page"]) - _pages(a, case["page"]) for a, b in zip(old, new))
        rows = sum(new)
        # lengths and page counts in and out, both calls; pages moved from the stack to the table and back; slot and position of every row
        return dict(bytes=4 * (2 * (3 * case["B"] + 3 * case["B"] + 1) + 2 * 3 * grow + 2 * rows), flops=rows)
    if op == "rope":
        e = case["rows"] * (case["H"] + 2 * case["Hkv"]) * case["hd"]
        return dict(bytes=2 * e * SIZE[case["dtype"]] + 8 * case["rows"], flops=8 * e)
    if op == "attention":
        rows, seen = sum(lengths(case)[1]), _visible(case)
        es = SIZE[case["dtype"]]
        return dict(bytes=2 * es * case["hd"] * (rows * case["H"] + case["Hkv"] * sum(k for _, k in seen)) + 4 * sum(_pages(k, case["page"]) for _, k in seen),
                    flops=4 * case["hd"] * case["H"] * sum(s for s, _ in seen))
    rows = 2 if case["draft"] else 1
    return dict(bytes=4 * case["B"] * (rows * case["V"] + 5 * case["K"] + 3), flops=3 * case["B"] * case["V"])


# ------------------------------------------------------------------------------------------------------------------ the inputs
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _table(g, case, tokens):
    """Pages of every sequence in random order in a pool that is a little larger than needed: table, pages held, free pages, their number."""
    page, B = case["page"], case["B"]
    held = torch.tensor([_pages(t, page) for t in tokens], dtype=torch.int32, device="cuda")
    width = _pages(case["T"] + 64, page)
    pool = sum(_pages(t + case["n"], page) + 1 for t in tokens) + 3
    order = torch.randperm(pool, generator=g, device="cuda").to(torch.int32)
    at = torch.arange(width, device="cuda")[None]
    first = held.cumsum(0) - held
    table = torch.where(at < held[:, None], order[(first[:, None] + at).clamp(max=pool - 1)], torch.full((B, width), -1, dtype=torch.int32, device="cuda"))
    used = int(sum(_pages(t, page) for t in tokens))
    free = torch.zeros(pool, dtype=torch.int32, device="cuda")
    free[: pool - used] = order[used:]
    return table.contiguous(), held, free, torch.tensor([pool - used], dtype=torch.int32, device="cuda"), pool


def prepare(case, seed):
    g, op = _generator(seed), case["op"]
    s = dict(case=case)
    if op == "plan":
        old, new = lengths(case)
        s["table"], s["held"], s["free"], s["count"], s["pool"] = _table(g, case, old)
        s["cached"], s["fresh"] = (torch.tensor(v, dtype=torch.int32, device="cuda") for v in (old, new))
        s["none"] = torch.zeros_like(s["fresh"])
        s["rows"] = sum(new) + 7   # a step's buffers are a little larger than its rows
        return s
    if op == "rope":
        rows, H, Hkv, hd, page, t = case["rows"], case["H"], case["Hkv"], case["hd"], case["page"], TYPES[case["dtype"]]
        # one row per token of the projection: q | k | v
        s["qkv"] = (torch.randn(rows, (H + 2 * Hkv) * hd, generator=g, device="cuda") * 1.5).to(t)
        s["q_norm"], s["k_norm"] = ((1 + 0.2 * torch.randn(hd, generator=g, device="cuda")).to(t) for _ in range(2))
        pool = _pages(rows, page) + 2
        s["K"], s["V"] = (torch.randn(pool, Hkv, page, hd, generator=g, device="cuda").to(t) for _ in range(2))
        s["positions"] = torch.randint(0, case["T"], (rows,), generator=g, device="cuda", dtype=torch.int32)
        s["slots"] = torch.randperm(pool * page, generator=g, device="cuda")[:rows].to(torch.int32)
        return s
    if op == "attention":
        old, new = lengths(case)
        H, Hkv, hd, page, t = case["H"], case["Hkv"], case["hd"], case["page"], TYPES[case["dtype"]]
        s["table"], _, _, _, pool = _table(g, case, [a + b for a, b in zip(old, new)])
        s["K"], s["V"] = (torch.randn(pool, Hkv, page, hd, generator=g, device="cuda", dtype=torch.float32).to(t) for _ in range(2))
        s["q"] = (torch.randn(sum(new), H, hd, generator=g, device="cuda") * 1.3).to(t)
        s["lens"] = torch.tensor([a + b for a, b in zip(old, new)], dtype=torch.int32, device="cuda")
        starts = [0]
        for m in new:
            starts.append(starts[-1] + m)
        s["starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
        s["most"] = max(new)
        return s
    B, K, V = case["B"], case["K"], case["V"]
    logits = torch.randn(B, K + 1, V, generator=g, device="cuda") * 2.5
    s["p"] = torch.softmax(logits, -1).reshape(B * (K + 1), V)
    near = logits[:, :K] + 0.7 * torch.randn(B, K, V, generator=g, device="cuda")
    q = torch.softmax(near, -1)
    e = torch.rand(B, K, V, generator=g, device="cuda").clamp_(1e-9).log_().neg_()
    s["tokens"] = (q / e).argmax(-1).to(torch.int32)
    s["q"] = q.reshape(B * K, V) if case["draft"] else None
    s["u"] = torch.rand(B, K + 1, generator=g, device="cuda")
    return s


# ------------------------------------------------------------------------------------------------------------------ plain forms
def _plain_plan(s, cached, fresh):
    page, rows = s["case"]["page"], s["rows"]
    table, held, free, count = s["table"], s["held"], s["free"], s["count"]
    width, have = table.shape[1], held.long()
    fits = (cached >= 0) & (fresh >= 0) & (cached.long() + fresh <= width * page)
    old, new = cached.long(), torch.where(fits, fresh, 0).long()
    want = (old + new + page - 1) // page
    need = torch.where(new > 0, (want - have).clamp(min=0), 0)
    granted = (need == 0) | (need.cumsum(0) <= count)
    asked = torch.where(granted, new, 0)
    granted &= asked.cumsum(0) <= rows
    new, need = torch.where(granted, asked, 0), torch.where(granted, need, 0)
    keep = torch.where(new > 0, want, torch.minimum(have, (old + page - 1) // page))
    keep = torch.where(fits, keep, have)
    taken, at = need.cumsum(0), torch.arange(width, device=table.device)[None]
    grow = (at >= have[:, None]) & (at < (have + need)[:, None])
    place = count.long() - 1 - ((taken - need - have)[:, None] + at)
    table.copy_(torch.where(grow, free[place.clamp(0, free.numel() - 1)], table))
    surplus = (have - keep).clamp(min=0)
    back = (at >= keep[:, None]) & (at < have[:, None])
    height = count.long() - taken[-1] + surplus.sum()
    place = height - 1 - ((surplus.cumsum(0) - surplus - keep)[:, None] + at)
    # pages that do not come back write to a place past the end
    wide = torch.cat([free, free.new_zeros(1)])
    wide[torch.where(back, place, free.numel()).reshape(-1)] = table.reshape(-1)
    free.copy_(wide[:-1])
    table.masked_fill_(back, -1)
    held.copy_(keep)
    count.copy_(height)
    starts = torch.cat([new.new_zeros(1), new.cumsum(0)])
    row = torch.arange(rows, device=table.device)
    b = torch.searchsorted(starts[1:], row, right=True).clamp(max=held.numel() - 1)
    there = row < starts[-1]
    pos = torch.where(there, old[b] + row - starts[b], 0)
    entry = table[b, pos // page].long()
    slots = torch.where(there & (entry >= 0), entry * page + pos % page, -1)
    return [(old + new).int(), starts.int(), slots.int(), torch.where(there, pos, -1).int()]


def _rotate(x, cos, sin, rot, style):
    turned, rest = x[..., :rot], x[..., rot:]
    if style == 1:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = turned[..., : rot // 2], turned[..., rot // 2:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, rest], -1)


EPS, BASE = 1e-6, 500000.0


def _split(s):
    c = s["case"]
    H, Hkv, hd = c["H"], c["Hkv"], c["hd"]
    q, k, v = s["qkv"].split([H * hd, Hkv * hd, Hkv * hd], 1)
    return q.unflatten(1, (H, hd)), k.unflatten(1, (Hkv, hd)), v.unflatten(1, (Hkv, hd))


def _plain_rope(s):
    c, t = s["case"], s["qkv"].dtype
    q, k, v = _split(s)
    q, k = q.float(), k.float()
    if c["norm"]:
        q = q * (q.square().mean(-1, keepdim=True) + EPS).rsqrt() * s["q_norm"].float()
        k = k * (k.square().mean(-1, keepdim=True) + EPS).rsqrt() * s["k_norm"].float()
    turn = torch.arange(0, c["rot"], 2, device=q.device, dtype=torch.float64) / c["rot"]
    angle = s["positions"].double()[:, None] * (BASE ** -turn)[None]
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    q, k = (_rotate(x, cos, sin, c["rot"], c["style"]) for x in (q, k))
    page, slot = c["page"], s["slots"].long()
    s["K"][slot // page, :, slot % page] = k.to(t)
    s["V"][slot // page, :, slot % page] = v
    return [q.to(t), s["K"], s["V"]]


def _plain_attention(s):
    c, t = s["case"], s["q"].dtype
    B, H, Hkv, hd, page, T, n = c["B"], c["H"], c["Hkv"], c["hd"], c["page"], c["T"], s["most"]
    G, blocks = H // Hkv, _pages(T, page)
    table = s["table"][:, :blocks].long().clamp(min=0)
    keys, values = (x[table].transpose(2, 3).reshape(B, blocks * page, Hkv, hd).permute(0, 2, 1, 3).float() for x in (s["K"], s["V"]))
    starts, lens = s["starts"].long(), s["lens"].long()
    count = starts[1:] - starts[:-1]
    i = torch.arange(n, device=keys.device)
    row = (starts[:-1, None] + i).clamp(max=s["q"].shape[0] - 1)
    q = s["q"][row].float().reshape(B, n, Hkv, G, hd).permute(0, 2, 3, 1, 4).reshape(B, Hkv, G * n, hd)
    scores = (q @ keys.transpose(2, 3)).mul_(hd ** -0.5).reshape(B, Hkv, G, n, blocks * page)
    pos, j = (lens - count)[:, None, None] + i[None, :, None], torch.arange(blocks * page, device=keys.device)
    hidden = j > pos
    if c["window"]:
        hidden = hidden | (j <= pos - c["window"])
    scores.masked_fill_(hidden[:, None, None], -math.inf)
    # rows that are only there to fill up may see nothing: their largest score is taken for 0
    top = scores.amax(-1, keepdim=True)
    weights = scores.sub_(torch.where(top == -math.inf, 0, top)).exp_()
    total = weights.sum(-1, keepdim=True)
    out = (weights.reshape(B, Hkv, G * n, -1) @ values).reshape(B, Hkv, G, n, hd) / total
    out = out.permute(0, 3, 1, 2, 4).reshape(B, n, H, hd)
    return [out[i[None] < count[:, None]].to(t)]


def _plain_verify(s):
    c = s["case"]
    B, K, V = c["B"], c["K"], c["V"]
    p = s["p"].reshape(B, K + 1, V)
    x = s["tokens"].long()[..., None]
    at = p[:, :K].gather(2, x)[..., 0].double()
    drafted = s["q"].reshape(B, K, V).gather(2, x)[..., 0].double() if c["draft"] else torch.ones_like(at)
    taken = (s["u"][:, :K].double() * drafted < at).long().cumprod(1).sum(1)
    b = torch.arange(B, device=p.device)
    row = p[b, taken].double()
    if c["draft"]:
        less = s["q"].reshape(B, K, V)[b, taken.clamp(max=K - 1)].double()
    else:
        less = torch.zeros_like(row).scatter_(1, x[b, taken.clamp(max=K - 1)], 1.0)
    rest = (row - less).clamp(min=0)
    use = (taken < K)[:, None] & (rest.sum(1, keepdim=True) > 0)
    weights = torch.where(use, rest, row)
    sums = weights.cumsum(1)
    token = (sums <= s["u"][:, K:].double() * sums[:, -1:]).sum(1)
    last = V - 1 - (weights > 0).long().flip(1).argmax(1)
    token = torch.minimum(token, last)
    i = torch.arange(K + 1, device=p.device)[None]
    drafts = torch.cat([s["tokens"].long(), token[:, None]], 1)
    tokens = torch.where(i < taken[:, None], drafts, torch.where(i == taken[:, None], token[:, None], -1))
    return [tokens.int(), (taken + 1).int()]


def run(s):
    c = s["case"]
    op = c["op"]
    if own:
        from seq2seqsharp_b200.ops import Ops
        if op == "plan":
            # a step takes the pages of its rows; all drafts refused, the next one gives them back
            first = Ops.PagedPlan(s["cached"], s["fresh"], s["table"], s["held"], s["free"], s["count"], c["page"], s["rows"])
            Ops.PagedPlan(s["cached"], s["none"], s["table"], s["held"], s["free"], s["count"], c["page"], s["rows"])
            return [*first, s["table"], s["held"], s["free"], s["count"]]
        if op == "rope":
            q, k, v = _split(s)
            q = Ops.QKNormRopePaged(None, q, k, v, s["q_norm"] if c["norm"] else None, s["k_norm"] if c["norm"] else None, EPS, s["positions"], s["slots"],
                                    s["K"], s["V"], ropeStyle=c["style"], ropeDims=c["rot"], base=BASE)
            return [q, s["K"], s["V"]]
        if op == "attention":
            return [Ops.PagedAttention(None, s["q"], s["K"], s["V"], s["table"], s["starts"], s["lens"], s["most"], window=c["window"])]
        return list(Ops.VerifyDraft(s["p"], s["q"], s["tokens"], s["u"]))
    if op == "plan":
        first = _plain_plan(s, s["cached"], s["fresh"])
        _plain_plan(s, s["cached"], s["none"])
        return [*first, s["table"], s["held"], s["free"], s["count"]]
    return {"rope": _plain_rope, "attention": _plain_attention, "verify": _plain_verify}[op](s)


# ------------------------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rope":
        H, Hkv, hd, rot = case["H"], case["Hkv"], case["hd"], case["rot"]
        x = s["qkv"].double().reshape(case["rows"], H + 2 * Hkv, hd)
        heads, v = x[:, : H + Hkv].clone(), x[:, H + Hkv:]
        if case["norm"]:
            gain = torch.cat([s["q_norm"].double().expand(H, hd), s["k_norm"].double().expand(Hkv, hd)])
            heads = heads / torch.sqrt((heads ** 2).sum(-1, keepdim=True) / hd + EPS) * gain
        i = torch.arange(rot // 2, device=x.device)
        rate = torch.exp(i.double() * (-2.0 * math.log(BASE) / rot))
        z = torch.polar(torch.ones(1, 1, device=x.device, dtype=torch.float64), s["positions"].double()[:, None] * rate)[:, None]
        lo, hi = (2 * i, 2 * i + 1) if case["style"] == 1 else (i, i + rot // 2)
        w = torch.complex(heads[..., lo], heads[..., hi]) * z
        heads[..., lo], heads[..., hi] = w.real, w.imag
        K, V = s["K"].double(), s["V"].double()
        for cache, new in ((K, heads[:, H:]), (V, v)):
            flat = cache.transpose(1, 2).reshape(-1, Hkv, hd)
            flat[s["slots"].long()] = new
            cache.copy_(flat.reshape(cache.shape[0], case["page"], Hkv, hd).transpose(1, 2))
        return [heads[:, :H], K, V]
    if case["op"] == "attention":
        G, out = case["H"] // case["Hkv"], torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
        at = 0
        for b, (old, n) in enumerate(zip(*lengths(case))):
            T = old + n
            pages = s["table"][b, : _pages(T, case["page"])].long()
            for h in range(case["Hkv"]):
                k, v = (x[pages, h].reshape(-1, case["hd"])[:T].double() for x in (s["K"], s["V"]))
                for i0 in range(0, n, 512):
                    i1 = min(n, i0 + 512)
                    q = s["q"][at + i0: at + i1, h * G:(h + 1) * G].double()
                    logit = torch.einsum("igd,td->git", q, k) / math.sqrt(case["hd"])
                    ahead = torch.arange(T, device="cuda")[None] - (old + torch.arange(i0, i1, device="cuda"))[:, None]
                    sees = ahead <= 0
                    if case["window"]:
                        sees &= ahead > -case["window"]
                    logit = logit.masked_fill(~sees, -math.inf)
                    out[at + i0: at + i1, h * G:(h + 1) * G] = torch.einsum("git,td->igd", torch.softmax(logit, -1), v)
            at += n
        return [out]
    return None
