"""Measured cases of a model's linears in 8-bit integers and of the log probabilities that show what they change: the norm with the residual's addition and an
output in 8 bits, (gated) activations in 8 bits, the product of 8-bit rows and weights with scales per token and channel, and the log probabilities of given
tokens with entropy, rank and top alternatives.

`own` false: the operators in their plain form (elementary torch operations in 32 bits, or 64 where that matters); `own` true: the
framework's entry points.  Shapes are those of the repository's configurations (widths 2048 and 4096, feed-forward widths 8192 and 11008, vocabularies of 32000
and 50257) or generic.
"""
import math

import torch

own = False

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
SIZE = {"f16": 2, "bf16": 2, "f32": 4}
EPS = 1e-6


# ------------------------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # a token of one chat and a prompt pass of the 7B-class model; rows of an odd width in 32 bits, without a residual
        dict(name="norm_1", op="norm", dtype="f16", rows=1, d=4096, residual=True),
        dict(name="norm_f32", op="norm", dtype="f32", rows=333, d=1001, residual=False),
        dict(name="norm_16k", op="norm", dtype="bf16", rows=16384, d=4096, residual=True),
        # gated products between two linears: a step of eight sequences of the 7B-class model, a prompt pass of the 1B-class one
        dict(name="gated_8", op="rows", dtype="f16", rows=8, F=11008, act="silu", gate=True),
        dict(name="gated_8k", op="rows", dtype="bf16", rows=8192, F=8192, act="silu", gate=True),
        # linears of the 7B-class model: the first of the feed-forward block for one chat, the second for 64; odd sizes; the first for a prompt pass
        dict(name="linear_1", op="linear", dtype="f16", M=1, K=4096, N=22016, bias=False),
        dict(name="linear_64", op="linear", dtype="f16", M=64, K=11008, N=4096, bias=False),
        dict(name="linear_203", op="linear", dtype="f32", M=203, K=1000, N=2047, bias=True),
        dict(name="linear_8k", op="linear", dtype="bf16", M=8192, K=4096, N=22016, bias=False),
        # what one chat's newest token was worth, that of 64 with the 20 best, and a text of 4096 tokens that is only scored
        dict(name="logp_1", op="logp", dtype="f32", rows=1, V=32000, top=5),
        dict(name="logp_64", op="logp", dtype="f32", rows=64, V=50257, top=20),
        dict(name="logp_4k", op="logp", dtype="bf16", rows=4096, V=50257, top=1),
    ]


def _log(rng, a, b):
    return min(b, max(a, int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))))


def _width(rng, a, b):
    """Half of the widths are multiples of 64, as models have them, half are any."""
    n = _log(rng, a, b)
    return max(64, n // 64 * 64) if rng.random() < 0.5 else n


def draw(rng):
    op = rng.choice(("norm", "rows", "linear", "linear", "logp"))
    dtype = rng.choice(("f16", "bf16", "f32"))
    if op == "norm":
        d = _width(rng, 64, 12288)
        return dict(op=op, dtype=dtype, rows=_log(rng, 1, min(16384, 30_000_000 // d)), d=d, residual=rng.random() < 0.7)
    if op == "rows":
        F = _width(rng, 64, 22016)
        return dict(op=op, dtype=dtype, rows=_log(rng, 1, min(8192, 30_000_000 // F)), F=F, act=rng.choice(("none", "relu", "silu", "gelu")), gate=rng.random() < 0.6)
    if op == "linear":
        K, N = _width(rng, 64, 11008), _width(rng, 64, 50257)
        M = _log(rng, 1, max(2, min(8192, int(4e11 / (K * N)))))
        return dict(op=op, dtype=dtype, M=M, K=K, N=N, bias=rng.random() < 0.4)
    V = _log(rng, 1000, 131072)
    return dict(op=op, dtype=dtype, rows=_log(rng, 1, min(4096, 100_000_000 // V)), V=V, top=rng.choice((0, 1, 5, 20, 32)))


def work(case):
    op, es = case["op"], SIZE[case["dtype"]]
    if op == "norm":
        e = case["rows"] * case["d"]
        return dict(bytes=e * (es * (3 if case["residual"] else 1) + 1) + es * case["d"] + 4 * case["rows"], flops=8 * e)
    if op == "rows":
        e = case["rows"] * case["F"]
        return dict(bytes=e * (es * (2 if case["gate"] else 1) + 1) + 4 * case["rows"], flops=8 * e)
    if op == "linear":
        M, K, N = case["M"], case["K"], case["N"]
        return dict(bytes=M * K + N * K + 4 * (M + N) + es * M * N + (es * N if case["bias"] else 0), flops=2 * M * N * K)
    rows, V = case["rows"], case["V"]
    return dict(bytes=rows * V * es + rows * (4 + 12 + 8 * case["top"]), flops=6 * rows * V)


# ------------------------------------------------------------------------------------------------------------------ the inputs
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _bytes(g, rows, cols):
    """Rows of 8-bit integers as the framework's operators leave them: every row starts on a boundary of 16 bytes."""
    wide = torch.randn(rows, -(-cols // 16) * 16, generator=g, device="cuda").mul_(36).round_().clamp_(-127, 127)
    return wide.to(torch.int8)[:, :cols]


def prepare(case, seed):
    g, op, t = _generator(seed), case["op"], TYPES[case["dtype"]]
    s = dict(case=case)
    if op == "norm":
        rows, d = case["rows"], case["d"]
        # a stream with a few loud channels, and what a layer adds to it
        loud = 1 + 12 * (torch.rand(d, generator=g, device="cuda") < 0.01)
        s["x"] = torch.randn(rows, d, generator=g, device="cuda").to(t)
        s["residual"] = (torch.randn(rows, d, generator=g, device="cuda") * 2 * loud).to(t) if case["residual"] else None
        s["gamma"] = (1 + 0.2 * torch.randn(d, generator=g, device="cuda")).to(t)
        return s
    if op == "rows":
        # both projections of a token side by side, as one linear gives them
        wide = (torch.randn(case["rows"], case["F"] * (2 if case["gate"] else 1), generator=g, device="cuda") * 1.5).to(t)
        s["a"], s["gate"] = wide[:, : case["F"]], wide[:, case["F"]:] if case["gate"] else None
        return s
    if op == "linear":
        M, K, N = case["M"], case["K"], case["N"]
        s["q"], s["w"] = _bytes(g, M, K), _bytes(g, N, K)
        s["q_scale"] = (0.5 + torch.rand(M, generator=g, device="cuda")) * 0.03
        s["w_scale"] = (0.5 + torch.rand(N, generator=g, device="cuda")) * (0.9 / 36 / math.sqrt(K))
        s["bias"] = (0.3 * torch.randn(N, generator=g, device="cuda")).to(t) if case["bias"] else None
        return s
    rows, V = case["rows"], case["V"]
    logits = torch.randn(rows, V, generator=g, device="cuda", dtype=torch.float32 if rows * V < 50_000_000 else torch.bfloat16).mul_(2.5)
    s["logits"] = logits.to(t)
    # the tokens of a text: most of them likely ones
    some = torch.randint(0, V, (rows, 64), generator=g, device="cuda")
    s["tokens"] = some.gather(1, logits.gather(1, some).float().argmax(1, keepdim=True))[:, 0].int()
    return s


# ------------------------------------------------------------------------------------------------------------------ plain forms
def _values(q, scale):
    """What bytes with a scale per row stand for, in 16 bits."""
    return torch.mul(q, scale[:, None], out=torch.empty(q.shape, dtype=torch.bfloat16, device=q.device))


def _plain_bytes(y):
    scale = y.abs().amax(-1) / 127
    return (y / scale.clamp(min=1e-38)[:, None]).round(), scale


def _plain_norm(s):
    h = s["x"]
    if s["residual"] is not None:
        h = (h.float() + s["residual"].float()).to(h.dtype)
    x = h.float()
    y = x * (x.square().mean(-1, keepdim=True) + EPS).rsqrt() * s["gamma"].float()
    q, scale = _plain_bytes(y)
    return [_values(q, scale), scale, h]


def _act(a, act):
    if act == "relu":
        return a.clamp(min=0)
    if act == "silu":
        return a / (1 + (-a).exp())
    if act == "gelu":
        return 0.5 * a * (1 + torch.erf(a * math.sqrt(0.5)))
    return a


def _plain_rows(s):
    v = _act(s["a"].float(), s["case"]["act"])
    if s["gate"] is not None:
        v = v * s["gate"].float()
    q, scale = _plain_bytes(v)
    return [_values(q, scale), scale]


def _plain_linear(s):
    y = (s["q"].float() @ s["w"].float().t()) * (s["q_scale"][:, None] * s["w_scale"])
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return [y.to(TYPES[s["case"]["dtype"]])]


def _plain_logp(s):
    # + 0: a zero has one sign, as it has one place in the order
    x, t, top = s["logits"].float() + 0, s["tokens"].long()[:, None], s["case"]["top"]
    V = x.shape[1]
    below = x - x.amax(-1, keepdim=True)
    e = below.exp()
    total = e.sum(-1, dtype=torch.float64)
    log = total.log()
    mean = (e * below.clamp(min=-1e30)).sum(-1, dtype=torch.float64) / total
    at = x.gather(1, t)
    j = torch.arange(V, device=x.device)
    rank = ((x > at) | ((x == at) & (j < t))).sum(-1)
    # one whole number per word that orders by logit, and by index among equal ones
    bits = x.view(torch.int32).long()
    key = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits) * V + (V - 1 - j)
    best = V - 1 - key.topk(top, -1).values % V
    lp = lambda i: (below.gather(1, i).double() - log[:, None]).float()  # noqa: E731
    return [lp(t)[:, 0], (log - mean).float(), rank.int(), best.int(), lp(best)]


def run(s):
    c = s["case"]
    op = c["op"]
    if own:
        from seq2seqsharp_b200 import _native as N
        from seq2seqsharp_b200.ops import Ops
        if op == "norm":
            q, scale, h = Ops.RMSNormInt8(None, s["x"], s["residual"], s["gamma"], EPS)
            return [_values(q, scale), scale, h]
        if op == "rows":
            act = {"none": N.ACT_NONE, "relu": N.ACT_RELU, "silu": N.ACT_SILU, "gelu": N.ACT_GELU}[c["act"]]
            q, scale = Ops.RowsInt8(None, s["a"], s["gate"], act)
            return [_values(q, scale), scale]
        if op == "linear":
            return [Ops.LinearInt8(None, s["q"], s["q_scale"], s["w"], s["w_scale"], s["bias"], dtype=TYPES[c["dtype"]])]
        return list(Ops.TokenLogProbs(s["logits"], s["tokens"], c["top"]))
    return {"norm": _plain_norm, "rows": _plain_rows, "linear": _plain_linear, "logp": _plain_logp}[op](s)


# ------------------------------------------------------------------------------------------------------------------ in 64 bits
def _exact_bytes(y):
    scale = y.abs().max(1).values / 127
    q = torch.where(scale[:, None] > 0, y / scale[:, None], torch.zeros_like(y)).round()
    return [q * scale[:, None], scale]


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "norm":
        h = s["x"] if s["residual"] is None else (s["x"].double() + s["residual"].double()).to(s["x"].dtype)
        d = h.double()
        y = d / torch.sqrt((d ** 2).sum(1, keepdim=True) / case["d"] + EPS) * s["gamma"].double()
        # the sum is what the norm goes by, so it is the rounded one
        return [*_exact_bytes(y), h.double()]
    if op == "rows":
        a = s["a"].double()
        v = {"none": lambda: a, "relu": lambda: torch.maximum(a, torch.zeros_like(a)), "silu": lambda: a * torch.sigmoid(a),
             "gelu": lambda: a * torch.special.ndtr(a)}[case["act"]]()
        return _exact_bytes(v if s["gate"] is None else v * s["gate"].double())
    if op == "linear":
        if case["M"] * case["K"] * case["N"] > 1e11:
            return None
        y = torch.einsum("mk,nk->mn", s["q"].double(), s["w"].double())
        y = y * s["q_scale"].double()[:, None] * s["w_scale"].double()
        return [y if s["bias"] is None else y + s["bias"].double()]
    out, ent, tops = [], [], []
    for r0 in range(0, case["rows"], 256):
        x = s["logits"][r0: r0 + 256].double()
        lp = torch.log_softmax(x, 1)
        out.append(lp.gather(1, s["tokens"][r0: r0 + 256].long()[:, None])[:, 0])
        ent.append(torch.special.entr(lp.exp()).sum(1))
        tops.append(lp.topk(case["top"], 1).values)
    return [torch.cat(out), torch.cat(ent), None, None, torch.cat(tops)]
