"""The operators of a decoder's step beside its cache and its attention, at the
sizes that they run at: products of tokens with weights in 8-bit integers, the
same grouped by expert, attention of many sequences that share a long prefix of
the 8-bit cache, and the next token drawn from the logits.

Every case is a plain dict whose "kind" names the operator:

  linear   tokens [rows, k] times weights [n, k]: 8-bit codes of both, a scale for each token and each output channel
  experts  the same with weights of every expert: rows sorted by expert, ragged, some experts without a row
  prefix   attention over the 8-bit cache: groups of sequences that share a prefix's pages, and each sequence's own pages
  sample   temperature, top-k, top-p and min-p, then a token by a given uniform number

Where `own` is false the same passes run in their plain form: elementary torch
operations in 32 bits (the draw in 64: cumulated weights lie next to a border),
rounded once at the end.
"""
from __future__ import annotations

import math
import os
import sys

import torch

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
TINY = 2.0 ** -126  # smallest scale of a token that holds anything


def _nhip():
    pkg = os.path.join(_ROOT, "ncnn-compiler_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import nhip
    return nhip


def listed():
    return [
        # one new token of each of a small batch of sequences through a square projection: latency and the weights
        dict(name="linear_step", kind="linear", rows=16, k=2048, n=2048, act="none", bias=False, dtype="bf16"),
        # the same tokens of a larger batch against all rows of an odd vocabulary
        dict(name="linear_vocabulary", kind="linear", rows=48, k=2048, n=50021, act="none", bias=False, dtype="f16"),
        # pooled features of a batch of images through the classifier, in the framework's own type
        dict(name="linear_classes", kind="linear", rows=256, k=2048, n=1000, act="none", bias=True, dtype="f32"),
        # all tokens of two pictures through the first product of a block
        dict(name="linear_prompt", kind="linear", rows=6272, k=2048, n=8192, act="silu", bias=True, dtype="bf16"),
        # a step of 64 sequences, two experts a token
        dict(name="experts_step", kind="experts", rows=128, experts=16, k=2048, n=1024, act="none", bias=False, dtype="bf16"),
        # all tokens of two pictures, two experts a token
        dict(name="experts_prompt", kind="experts", rows=12544, experts=32, k=1024, n=4096, act="silu", bias=True, dtype="f16"),
        # five candidates for the caption of one picture
        dict(name="prefix_beams", kind="prefix", groups=1, members=5, lq=1, prefix=197, own=37, heads=12, kv_heads=12, d=64,
             block=16, dtype="f32"),
        # sixteen samples of each of four pictures, a step
        dict(name="prefix_samples", kind="prefix", groups=4, members=16, lq=1, prefix=3136, own=256, heads=32, kv_heads=8,
             d=128, block=64, dtype="bf16"),
        # a batch that shares one long prompt, some tokens of each sequence at a time
        dict(name="prefix_long", kind="prefix", groups=1, members=48, lq=7, prefix=12544, own=1568, heads=32, kv_heads=8, d=128,
             block=64, dtype="f16"),
        # a class for each of a few rows
        dict(name="sample_classes", kind="sample", rows=16, vocab=1000, temperature=1.0, top_k=5, top_p=1.0, min_p=0.0,
             each=False, dtype="f32"),
        # a batch of sequences, each with settings of its own, greedy ones among them
        dict(name="sample_step", kind="sample", rows=64, vocab=131072, temperature=0.8, top_k=50, top_p=0.9, min_p=0.02,
             each=True, dtype="bf16"),
        # many samples by top-p alone, an odd vocabulary
        dict(name="sample_many", kind="sample", rows=256, vocab=50021, temperature=1.1, top_k=0, top_p=0.95, min_p=0.0,
             each=False, dtype="f32"),
    ]


# ------------------------------------------------------------------ drawn cases
def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw(rng):
    kind = rng.choice(["linear", "experts", "prefix", "sample"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if kind in ("linear", "experts"):
        case = dict(kind=kind, rows=_log_int(rng, 1, 16384), k=_log_int(rng, 32, 8192), n=_log_int(rng, 32, 65536),
                    act=rng.choice(["none", "relu", "silu"]), bias=rng.random() < 0.5, dtype=dtype)
        if kind == "experts":
            case.update(experts=_log_int(rng, 2, 64), n=_log_int(rng, 32, 8192))
        if rng.random() < 0.5:  # half of them as widths of layers are, the others as they come
            case.update(k=case["k"] // 32 * 32, n=case["n"] // 32 * 32)
        return case
    if kind == "prefix":
        kv = rng.choice([1, 2, 4, 8, 12])
        own_tokens = _log_int(rng, 1, 2048)
        return dict(kind=kind, groups=rng.choice([1, 1, 2, 4, 8]), members=_log_int(rng, 1, 64),
                    lq=rng.choice([1, 1, min(own_tokens, _log_int(rng, 1, 16))]), prefix=_log_int(rng, 1, 12544),
                    own=own_tokens, heads=kv * rng.choice([1, 2, 4, 8]), kv_heads=kv, d=rng.choice([32, 40, 64, 80, 96, 128]),
                    block=rng.choice([16, 32, 64, 128]), dtype=dtype)
    return dict(kind=kind, rows=_log_int(rng, 1, 256), vocab=_log_int(rng, 100, 131072),
                temperature=rng.choice([0.0, 0.5, 0.8, 1.0, 1.5]), top_k=rng.choice([0, 0, 1, 20, 50, 200, 1000]),
                top_p=rng.choice([1.0, 1.0, 0.5, 0.9, 0.95, 0.99]), min_p=rng.choice([0.0, 0.0, 0.02, 0.1]),
                each=rng.random() < 0.5, dtype=dtype)


def draw(rng):
    """A case of the listed ranges that costs no more than the largest listed one of its kind."""
    while True:
        case = _draw(rng)
        most = [work(c) for c in listed() if c["kind"] == case["kind"]]
        w = work(case)
        if w["bytes"] <= max(m["bytes"] for m in most) and w["flops"] <= max(m["flops"] for m in most):
            return case


# ------------------------------------------------------------------- inputs
def _counts(case):
    """Rows of each expert: uneven, every fifth expert without any (but the first)."""
    e, rows = case["experts"], case["rows"]
    share = [0 if i % 5 == 4 else 1 + (i * 7919) % 11 for i in range(e)]
    ends = [rows * sum(share[:i + 1]) // sum(share) for i in range(e)]
    return [b - a for a, b in zip([0] + ends[:-1], ends)]


def _lengths(n, most, least=0):
    """Ragged lengths: the first is the longest, the others lie between half of it and all of it."""
    return [max(least, most - (i * 7919) % (most // 2 + 1)) for i in range(n)]


def _own_lengths(case):
    return _lengths(case["groups"] * case["members"], case["own"], case["lq"])


def _randn(gen, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


def _pages(gen, shape):
    """Codes and scales of pages [pages, heads, tokens, d] as normal values give them."""
    x = torch.randn(shape, generator=gen, device="cuda")
    s = (x.abs().amax((2, 3)) * (1.0 / 127.0)).clamp_min(TINY)
    return torch.round(x / s[:, :, None, None]).clamp(-127, 127).to(torch.int8), s


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    kind = case["kind"]
    s = dict(case=case)
    if kind in ("linear", "experts"):
        rows, k, n = case["rows"], case["k"], case["n"]
        e = (case["experts"],) if kind == "experts" else ()
        # tokens of different size, a few channels far larger than the others, as blocks leave them
        size = 0.25 + torch.rand((rows, 1), generator=gen, device="cuda") * 4
        large = 1 + 15 * (torch.rand((k,), generator=gen, device="cuda") < 0.01)
        s["x"] = (torch.randn((rows, k), generator=gen, device="cuda") * size * large).to(dt)
        s["codes"] = torch.randn(e + (n, k), generator=gen, device="cuda").mul_(32).round_().clamp_(-127, 127).to(torch.int8)
        s["scale"] = (0.5 + torch.rand(e + (n,), generator=gen, device="cuda")) / (32 * math.sqrt(k))
        s["bias"] = 0.2 * torch.randn(e + (n,), generator=gen, device="cuda") if case["bias"] else None
        if kind == "experts":
            counts = _counts(case)
            s["starts"] = torch.tensor([sum(counts[:i]) for i in range(len(counts) + 1)], dtype=torch.int32, device="cuda")
        if own:
            nhip = _nhip()
            act = {"none": nhip.ACT_NONE, "relu": nhip.ACT_RELU, "silu": nhip.ACT_SILU}[case["act"]]
            s["plan"] = nhip.Linear8(s["codes"], s["scale"], bias=s["bias"], act=act)
    elif kind == "prefix":
        g, m, bt, kv, d = (case[k] for k in ("groups", "members", "block", "kv_heads", "d"))
        s["q"] = _randn(gen, (g * m, case["lq"], case["heads"], d), dt)
        per_prefix, per_own = -(-case["prefix"] // bt), -(-case["own"] // bt)
        pages = g * per_prefix + g * m * per_own
        order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)  # pages in no order
        s["prefix_table"] = order[:g * per_prefix].view(g, per_prefix)
        s["table"] = order[g * per_prefix:].view(g * m, per_own).contiguous()
        s["k"], s["ks"] = _pages(gen, (pages, kv, bt, d))
        s["v"], s["vs"] = _pages(gen, (pages, kv, bt, d))
        s["prefix_lengths"] = torch.tensor(_lengths(g, case["prefix"], 1), dtype=torch.int32, device="cuda")
        s["lengths"] = torch.tensor(_own_lengths(case), dtype=torch.int32, device="cuda")
        if own:
            s["cache"] = _nhip().KvCache8.of(s["k"], s["v"], s["ks"], s["vs"])
    else:
        rows, vocab = case["rows"], case["vocab"]
        s["logits"] = _randn(gen, (rows, vocab), dt, 3.0)
        s["uniform"] = torch.rand((rows,), generator=gen, device="cuda")
        if case["each"]:  # every third row without top-k, every fourth greedy, others a little apart
            i = torch.arange(rows, device="cuda")
            s["temperature"] = torch.where(i % 4 == 3, 0.0, case["temperature"] + 0.01 * (i % 16)).float()
            s["top_k"] = torch.where(i % 3 == 2, 0, case["top_k"] + i % 7).to(torch.int32)
            s["top_p"] = (case["top_p"] - 0.005 * (i % 9)).float()
            s["min_p"] = (case["min_p"] * (i % 2)).float()
    return s


# ------------------------------------------------------------------- a pass
def run(s):
    return (_run_own if own else _run_plain)(s)


def _settings(s):
    given = s if s["case"]["each"] else s["case"]
    return {k: given[k] for k in ("temperature", "top_k", "top_p", "min_p")}


def _run_own(s):
    case = s["case"]
    kind = case["kind"]
    if kind == "linear":
        return s["plan"].forward(s["x"])
    if kind == "experts":
        return s["plan"].forward(s["x"], expert_starts=s["starts"])
    if kind == "prefix":
        return s["cache"].prefix_attention(s["q"], s["prefix_table"], s["prefix_lengths"], s["table"], s["lengths"],
                                           max_prefix=case["prefix"], max_length=case["own"], causal=True)
    return _nhip().sample(s["logits"], s["uniform"], **_settings(s))


def _tokens8(x):
    """Codes of each token as 32-bit values, and its scale: x times the scale's reciprocal to the nearest, halves away
    from zero, each operation rounded to 32 bits, as the codes are defined."""
    x = x.float()
    most = x.abs().amax(1, keepdim=True)
    scale = torch.where(most > 0, (most * (1.0 / 127.0)).clamp_min(TINY), 0.0)
    q = x * torch.where(scale > 0, 1.0 / scale, 0.0)
    return torch.trunc(q + torch.copysign(torch.full_like(q, 0.5), q)).clamp(-127, 127), scale


def _finish(y, bias, act):
    y = y if bias is None else y + bias
    return y.clamp_min(0) if act == "relu" else y / (1 + torch.exp(-y)) if act == "silu" else y


def _softmax_two(qp, kp, vp, keep_p, qo, ko, vo, keep_o):
    """Softmax over two sets of keys: rows of a group [g, kv, m * r, d] on [g, kv, prefix, d], the same rows
    [b, kv, r, d] on [b, kv, own, d]; -> [b, kv, r, d]."""
    b, kv, r, d = qo.shape
    g = qp.shape[0]
    scale = 1.0 / math.sqrt(d)
    sp = torch.where(keep_p, torch.matmul(qp, kp.transpose(2, 3)) * scale, -math.inf)
    so = torch.where(keep_o, torch.matmul(qo, ko.transpose(2, 3)) * scale, -math.inf)

    def apart(t):  # [g, kv, m * r, x] -> [b, kv, r, x]
        return t.view(g, kv, b // g, r, -1).transpose(1, 2).reshape(b, kv, r, -1)

    def together(t):
        return t.view(g, b // g, kv, r, -1).transpose(1, 2).reshape(g, kv, b // g * r, -1)

    top = torch.maximum(apart(sp.amax(-1, keepdim=True)), so.amax(-1, keepdim=True))
    top = torch.where(top == -math.inf, 0.0, top)
    sp = torch.exp(sp - together(top))
    so = torch.exp(so - top)
    total = apart(sp.sum(-1, keepdim=True)) + so.sum(-1, keepdim=True)
    return (apart(torch.matmul(sp, vp)) + torch.matmul(so, vo)) / torch.where(total == 0, 1.0, total)


def _run_plain(s):
    case = s["case"]
    kind = case["kind"]
    dt = DTYPES[case["dtype"]]
    if kind == "linear":
        q, scale = _tokens8(s["x"])
        y = torch.matmul(q, s["codes"].float().t()) * (scale * s["scale"])
        return _finish(y, s["bias"], case["act"]).to(dt)
    if kind == "experts":
        q, scale = _tokens8(s["x"])
        counts = _counts(case)
        # every expert's rows behind each other up to the longest, the rest of them zeros
        starts = s["starts"].long()
        at = starts[:-1, None] + torch.arange(max(counts), device="cuda")
        held = at < starts[1:, None]
        at = torch.where(held, at, 0)
        y = torch.bmm(torch.where(held[..., None], q[at], 0.0), s["codes"].float().transpose(1, 2).contiguous())
        y = y * (scale[at] * s["scale"][:, None])
        y = _finish(y, None if s["bias"] is None else s["bias"][:, None], case["act"])
        return y[held].to(dt)
    if kind == "prefix":
        g, m, lq, kv, d, bt = (case[k] for k in ("groups", "members", "lq", "kv_heads", "d", "block"))
        b, group = g * m, case["heads"] // case["kv_heads"]
        kp, vp, ko, vo = ((codes[table] * scale[table][..., None, None]).transpose(1, 2).reshape(len(table), kv, -1, d)
                          for table in (s["prefix_table"].long(), s["table"].long())
                          for codes, scale in ((s["k"], s["ks"]), (s["v"], s["vs"])))
        qo = s["q"].float().view(b, lq, kv, group, d).permute(0, 2, 1, 3, 4).reshape(b, kv, lq * group, d)
        qp = qo.view(g, m, kv, lq * group, d).transpose(1, 2).reshape(g, kv, m * lq * group, d)
        keep_p = torch.arange(kp.shape[2], device="cuda") < s["prefix_lengths"][:, None]
        last = s["lengths"][:, None] - lq + 1 + torch.arange(lq, device="cuda")
        keep_o = (torch.arange(ko.shape[2], device="cuda") < last[..., None]).repeat_interleave(group, 1)
        o = _softmax_two(qp, kp, vp, keep_p[:, None, None], qo, ko, vo, keep_o[:, None])
        return o.view(b, kv, lq, group, d).transpose(1, 2).reshape(b, lq, kv * group, d).to(dt)
    rows, vocab = case["rows"], case["vocab"]
    t, top_k, top_p, min_p = (torch.as_tensor(v, dtype=torch.float32, device="cuda").double().expand(rows)[:, None]
                              for v in _settings(s).values())
    x = s["logits"].double()
    x, index = torch.sort(x, dim=1, descending=True, stable=True)  # ties: the lowest index first
    rank = torch.arange(vocab, device="cuda")
    w = torch.exp(torch.where(x == x[:, :1], 0.0, (x - x[:, :1]) / torch.where(t > 0, t, 1.0)))
    w = torch.where((rank < torch.where(t > 0, torch.where(top_k > 0, top_k, vocab), 1)), w, 0.0)
    before = torch.cumsum(w, 1) - w
    w = torch.where((before < top_p * w.sum(1, keepdim=True)) & (w >= min_p) | (top_p >= 1) & (w >= min_p) | (rank == 0), w, 0.0)
    w = torch.zeros_like(w).scatter_(1, index, w)
    upto = torch.cumsum(w, 1)
    target = s["uniform"].double()[:, None] * upto[:, -1:]
    token = (upto <= target).sum(1).clamp_max(vocab - 1)
    logprob = torch.log(w.gather(1, token[:, None]) / upto[:, -1:])[:, 0]
    return token.to(torch.int32), logprob.float()


# --------------------------------------------------------- what a pass needs
def work(case):
    kind, size = case["kind"], SIZE[case["dtype"]]
    if kind in ("linear", "experts"):
        rows, k, n = case["rows"], case["k"], case["n"]
        used = sum(c > 0 for c in _counts(case)) if kind == "experts" else 1
        return {"bytes": rows * (k + n) * size + used * n * (k + 4 + (4 if case["bias"] else 0)), "flops": 2 * rows * k * n}
    if kind == "prefix":
        kv, d, lq, bt = case["kv_heads"], case["d"], case["lq"], case["block"]
        shared, lengths = _lengths(case["groups"], case["prefix"], 1), _own_lengths(case)
        pairs = sum(n * lq * case["members"] for n in shared) + sum(sum(n - i for i in range(lq)) for n in lengths)
        return {"bytes": 2 * len(lengths) * lq * case["heads"] * d * size
                + 2 * kv * sum(n * d + -(-n // bt) * 4 for n in shared + lengths), "flops": 4 * pairs * case["heads"] * d}
    return {"bytes": case["rows"] * (case["vocab"] * size + 12), "flops": 4 * case["rows"] * case["vocab"]}


# ------------------------------------------------------- the same in 64 bits
def exact(case, seed):
    """From the definitions, a part of the rows, an expert, a head or a row at a time."""
    s = prepare(case, seed)
    f64 = torch.float64
    if case["kind"] in ("linear", "experts"):
        single = case["kind"] == "linear"
        bounds = [0, case["rows"]] if single else s["starts"].tolist()
        out = torch.empty((case["rows"], case["n"]), dtype=f64, device="cuda")
        for e, (a, b) in enumerate(zip(bounds, bounds[1:])):
            codes, scale, bias = (v if single or v is None else v[e] for v in (s["codes"], s["scale"], s["bias"]))
            codes = codes.to(f64)
            for r in range(a, b, 2048):
                x = s["x"][r:min(b, r + 2048)].to(torch.float32)
                # the codes are defined by their steps in 32 bits; all that follows them is exact
                step = torch.amax(torch.abs(x), 1) * torch.tensor(1 / 127, dtype=torch.float32, device="cuda")
                step[(step > 0) & (step < TINY)] = TINY
                per = (torch.reciprocal(step)[:, None] * x).nan_to_num_(0.0, 0.0, 0.0)
                q = torch.sign(per) * torch.floor(per.abs() + 0.5)
                y = q.clamp(-127, 127).to(f64) @ codes.t() * step.to(f64)[:, None] * scale.to(f64)
                y = y if bias is None else y + bias.to(f64)
                out[r:r + len(x)] = y * torch.sigmoid(y) if case["act"] == "silu" else y.relu() if case["act"] == "relu" else y
        return out
    if case["kind"] == "prefix":
        group, lq = case["heads"] // case["kv_heads"], case["lq"]
        out = torch.zeros(s["q"].shape, dtype=f64, device="cuda")

        def values(codes, scale, pages, h, n):
            pages = pages.long()
            return (codes[pages, h].to(f64) * scale[pages, h, None, None].to(f64)).flatten(0, 1)[:n]

        for gi, np_ in enumerate(s["prefix_lengths"].tolist()):
            for h in range(case["kv_heads"]):
                shared = [values(c, sc, s["prefix_table"][gi], h, np_) for c, sc in ((s["k"], s["ks"]), (s["v"], s["vs"]))]
                for i in range(gi * case["members"], (gi + 1) * case["members"]):
                    n = int(s["lengths"][i])
                    k, v = (torch.cat([a, values(c, sc, s["table"][i], h, n)])
                            for a, (c, sc) in zip(shared, ((s["k"], s["ks"]), (s["v"], s["vs"]))))
                    q = s["q"][i, :, h * group:(h + 1) * group].to(f64)  # [lq, group, d]
                    score = torch.matmul(q, k.t()) / math.sqrt(case["d"])
                    ahead = torch.ones((lq, len(k)), dtype=torch.bool, device="cuda").triu(np_ + n - lq + 1)
                    out[i, :, h * group:(h + 1) * group] = torch.matmul(
                        torch.softmax(score.masked_fill(ahead[:, None], -math.inf), -1), v)
        return out
    rows = []
    settings = {k: (v.tolist() if case["each"] else [torch.tensor(v, dtype=torch.float32).item()] * case["rows"])
                for k, v in _settings(s).items()}
    for i in range(case["rows"]):
        x, t = s["logits"][i].to(f64), settings["temperature"][i]
        if t <= 0:
            rows.append((int(torch.nonzero(x == x.max())[0]), 0.0))
            continue
        order = torch.argsort(-x, stable=True)
        if settings["top_k"][i] > 0:
            order = order[:int(settings["top_k"][i])]
        p = torch.softmax(x[order] / t, 0)
        stay = p >= settings["min_p"][i] * p[0]
        if settings["top_p"][i] < 1:
            stay &= torch.cat([p.new_zeros(1), p.cumsum(0)[:-1]]) < settings["top_p"][i]
        stay[0] = True
        kept, p = torch.sort(order[stay])[0], p[stay][torch.argsort(order[stay])]
        p = p / p.sum()
        at = min(int(torch.searchsorted(p.cumsum(0), s["uniform"][i].to(f64), right=True)), len(p) - 1)
        rows.append((int(kept[at]), math.log(float(p[at]))))
    return (torch.tensor([r[0] for r in rows], dtype=torch.int32), torch.tensor([r[1] for r in rows], dtype=f64))
