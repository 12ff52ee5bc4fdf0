"""The operators between a vision trunk and the decoder that reads it, at the
sizes that they run at: group norm with an activation into channels-last
tokens, rotary positions over several axes, cross attention to an encoder's
states, and attention over a cache held in 8 bits.

Every case is a plain dict whose "kind" names the operator:

  norm    group norm + activation; layout "tokens" ([n, pixels, c]) or "blobs" ([n, c, h, w] in, tokens out)
  rotary  rotary positions with three axes (time, height, width)
  cross   attention of lq tokens to lk encoder states, ragged lengths and a key mask
  cached  attention over the 8-bit cache through a block table, causal or not
  append  tokens quantised into the 8-bit cache, and the blocks that they touch read back as values

Where `own` is false the same passes run in their plain form: elementary
torch operations in 32 bits, rounded once at the end.
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
TINY = 2.0 ** -126  # smallest scale of a block that holds anything


def _nhip():
    pkg = os.path.join(_ROOT, "ncnn-compiler_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import nhip
    return nhip


def listed():
    return [
        # features of one small image, from the trunk's fp32 blobs to tokens: launch latency counts
        dict(name="norm_image_blobs", kind="norm", n=1, h=28, w=28, c=128, groups=32, act="silu", dtype="f32",
             layout="blobs"),
        # a batch of feature maps, already channels last
        dict(name="norm_batch", kind="norm", n=32, h=56, w=56, c=256, groups=32, act="silu", dtype="bf16",
             layout="tokens"),
        # large odd planes, ten channels to a group: the size of a decoder's last layers
        dict(name="norm_large_odd", kind="norm", n=8, h=225, w=223, c=320, groups=32, act="relu", dtype="f16",
             layout="tokens"),
        # one new token for each of a batch of sequences: latency
        dict(name="rotary_step", kind="rotary", b=32, t=1, h=1, w=1, heads=16, d=128, rotary=128, paired="halves",
             dtype="f16"),
        # all tokens of eight frames, twice
        dict(name="rotary_video", kind="rotary", b=2, t=8, h=56, w=56, heads=16, d=128, rotary=128, paired="halves",
             dtype="bf16"),
        # one decoder step of a batch, each sequence reading its own image's states
        dict(name="cross_step", kind="cross", b=32, lq=1, lk=3136, heads=32, kv_heads=8, d=128, dtype="bf16",
             masked=False),
        # image tokens reading a short padded text, in the framework's own type
        dict(name="cross_text_f32", kind="cross", b=4, lq=784, lk=197, heads=12, kv_heads=12, d=64, dtype="f32",
             masked=True),
        # all tokens of one picture reading those of a larger one
        dict(name="cross_large", kind="cross", b=2, lq=3136, lk=12544, heads=16, kv_heads=4, d=128, dtype="bf16",
             masked=False),
        # one decoder step over long 8-bit caches
        dict(name="cached_step", kind="cached", b=16, lq=1, lmax=12544, heads=32, kv_heads=8, d=128, block=64,
             causal=True, dtype="bf16"),
        # a chunk of a prompt over what the cache already holds
        dict(name="cached_chunk", kind="cached", b=2, lq=509, lmax=6272, heads=16, kv_heads=4, d=64, block=32,
             causal=True, dtype="f16"),
        # the new token of every sequence goes into its cache
        dict(name="append_step", kind="append", b=64, tokens=1, start=1001, kv_heads=8, d=128, block=64, dtype="bf16"),
        # an image's states go into the cache behind a few tokens that are there
        dict(name="append_prompt", kind="append", b=4, tokens=3136, start=37, kv_heads=8, d=128, block=64,
             dtype="bf16"),
    ]


# ------------------------------------------------------------------ drawn cases
def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw(rng):
    kind = rng.choice(["norm", "rotary", "cross", "cached", "append"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if kind == "norm":
        groups = rng.choice([1, 4, 8, 16, 32])
        return dict(kind=kind, n=_log_int(rng, 1, 32), h=_log_int(rng, 1, 224), w=_log_int(rng, 1, 224),
                    c=groups * _log_int(rng, 1, 40), groups=groups, act=rng.choice(["none", "relu", "silu"]),
                    dtype=dtype, layout=rng.choice(["tokens", "tokens", "blobs"]))
    if kind == "rotary":
        d = rng.choice([32, 64, 80, 96, 128])
        return dict(kind=kind, b=_log_int(rng, 1, 64), t=_log_int(rng, 1, 32), h=_log_int(rng, 1, 64),
                    w=_log_int(rng, 1, 64), heads=_log_int(rng, 1, 32), d=d, rotary=rng.choice([d, d // 2]),
                    paired=rng.choice(["halves", "neighbours"]), dtype=dtype)
    kv = rng.choice([1, 2, 4, 8, 12])
    d = rng.choice([32, 40, 64, 80, 96, 128])
    if kind == "cross":
        return dict(kind=kind, b=_log_int(rng, 1, 32), lq=rng.choice([1, _log_int(rng, 1, 4096)]),
                    lk=_log_int(rng, 1, 12544), heads=kv * rng.choice([1, 2, 4, 8]), kv_heads=kv, d=d, dtype=dtype,
                    masked=rng.random() < 0.5)
    if kind == "cached":
        lmax = _log_int(rng, 1, 12544)
        return dict(kind=kind, b=_log_int(rng, 1, 32), lq=rng.choice([1, min(lmax, _log_int(rng, 1, 1024))]),
                    lmax=lmax, heads=kv * rng.choice([1, 2, 4, 8]), kv_heads=kv, d=d,
                    block=rng.choice([16, 32, 64, 128]), causal=rng.random() < 0.7, dtype=dtype)
    return dict(kind=kind, b=_log_int(rng, 1, 64), tokens=rng.choice([1, _log_int(rng, 1, 4096)]),
                start=_log_int(rng, 1, 4096) - 1, kv_heads=kv, d=d, block=rng.choice([16, 32, 64, 128]), dtype=dtype)


def draw(rng):
    """A case of the listed ranges that costs no more than the largest listed one of its kind."""
    while True:
        case = _draw(rng)
        most = [work(c) for c in listed() if c["kind"] == case["kind"]]
        w = work(case)
        wide = 2.0 if case["dtype"] == "f32" else 1.0  # 32-bit matrix products run at a fraction of the 16-bit rate
        if w["bytes"] <= max(m["bytes"] for m in most) and w["flops"] * wide <= max(m["flops"] for m in most):
            return case


# ------------------------------------------------------------------- inputs
def _lengths(case, most, least=1):
    """Ragged lengths of a batch: the first is the longest, the others lie between half of it and all of it."""
    return [max(least, most - (i * 7919) % (most // 2 + 1)) for i in range(case["b"])]


def _sections(case):
    """Rotated pairs of each axis: a quarter for the time, the rest for height and width."""
    pairs = case["rotary"] // 2
    t = pairs // 4
    return t, (pairs - t) // 2, pairs - t - (pairs - t) // 2


def _inv_freq(case):
    """One falling series of frequencies for each axis, in 32 bits."""
    return torch.cat([torch.tensor([10000.0 ** (-i / s) for i in range(s)], dtype=torch.float32)
                      for s in _sections(case)])


def _randn(gen, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


def _quantised(x):
    """Blocks of values [blocks, heads, tokens, d] as codes and scales."""
    s = (x.abs().amax((2, 3)) * (1.0 / 127.0)).clamp_min(TINY)
    q = x / s[:, :, None, None]
    return torch.trunc(q + torch.copysign(torch.full_like(q, 0.5), q)).clamp(-127, 127).to(torch.int8), s


def _tables(case, gen, blocks):
    """A block table [b, blocks] over a pool whose pages are in no order, and the pool's pages."""
    pages = case["b"] * blocks
    return torch.randperm(pages, generator=gen, device="cuda").to(torch.int32).view(case["b"], blocks), pages


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    kind = case["kind"]
    s = dict(case=case)
    if kind == "norm":
        n, h, w, c = case["n"], case["h"], case["w"], case["c"]
        # trunk features: channels of different spread and mean, as a ReLU network leaves them
        gain = 0.5 + torch.rand((c,), generator=gen, device="cuda") * 2
        shift = torch.randn((c,), generator=gen, device="cuda")
        x = torch.randn((n, h * w, c), generator=gen, device="cuda") * gain + shift
        if case["layout"] == "blobs":
            x = x.transpose(1, 2).contiguous().view(n, c, h, w)
        s["x"] = x.to(dt)
        s["gamma"] = 1 + 0.2 * torch.randn((c,), generator=gen, device="cuda")
        s["beta"] = 0.2 * torch.randn((c,), generator=gen, device="cuda")
        if own:
            nhip = _nhip()
            act = {"none": nhip.ACT_NONE, "relu": nhip.ACT_RELU, "silu": nhip.ACT_SILU}[case["act"]]
            s["plan"] = nhip.GroupNorm(case["groups"], c, s["gamma"].cpu().numpy(), s["beta"].cpu().numpy(), eps=1e-5,
                                       act=act, blobs=case["layout"] == "blobs")
    elif kind == "rotary":
        b, tokens = case["b"], case["t"] * case["h"] * case["w"]
        s["x"] = _randn(gen, (b, tokens, case["heads"], case["d"]), dt)
        grid = torch.stack(torch.meshgrid(*(torch.arange(case[a], device="cuda", dtype=torch.int32)
                                            for a in ("t", "h", "w")), indexing="ij"), -1).view(1, tokens, 3)
        # each sequence begins where its last frame ended
        first = torch.randint(0, 512, (b, 1, 1), generator=gen, device="cuda", dtype=torch.int32)
        s["positions"] = (grid + first * torch.tensor([1, 0, 0], device="cuda", dtype=torch.int32)).contiguous()
        s["inv_freq"] = _inv_freq(case).cuda()
        s["axis"] = torch.repeat_interleave(torch.arange(3), torch.tensor(_sections(case))).cuda()
        if own:
            s["plan"] = _nhip().Rotary(case["d"], _sections(case), inv_freq=_inv_freq(case).numpy(),
                                       neighbours=case["paired"] == "neighbours")
    elif kind == "cross":
        b, lq, lk, kv, d = (case[k] for k in ("b", "lq", "lk", "kv_heads", "d"))
        s["q"] = _randn(gen, (b, lq, case["heads"], d), dt)
        s["k"] = _randn(gen, (b, lk, kv, d), dt)
        s["v"] = _randn(gen, (b, lk, kv, d), dt)
        s["lengths"] = torch.tensor(_lengths(case, lk), dtype=torch.int32, device="cuda")
        s["mask"] = torch.rand((b, lk), generator=gen, device="cuda") < 0.9 if case["masked"] else None
    elif kind == "cached":
        b, lq, kv, d, bt = (case[k] for k in ("b", "lq", "kv_heads", "d", "block"))
        s["q"] = _randn(gen, (b, lq, case["heads"], d), dt)
        s["table"], pages = _tables(case, gen, -(-case["lmax"] // bt))
        s["k"], s["ks"] = _quantised(torch.randn((pages, kv, bt, d), generator=gen, device="cuda"))
        s["v"], s["vs"] = _quantised(torch.randn((pages, kv, bt, d), generator=gen, device="cuda"))
        s["lengths"] = torch.tensor(_lengths(case, case["lmax"]), dtype=torch.int32, device="cuda")
        if own:
            s["cache"] = _nhip().KvCache8.of(s["k"], s["v"], s["ks"], s["vs"])
    else:
        b, n, kv, d, bt = (case[k] for k in ("b", "tokens", "kv_heads", "d", "block"))
        starts = _lengths(case, case["start"], 0)
        # a page more than is needed, so that the plain form may touch it
        s["table"], pages = _tables(case, gen, -(-(case["start"] + n) // bt) + 1)
        s["k"], s["ks"] = _quantised(torch.randn((pages, kv, bt, d), generator=gen, device="cuda"))
        s["v"], s["vs"] = _quantised(torch.randn((pages, kv, bt, d), generator=gen, device="cuda"))
        s["k_new"] = _randn(gen, (b, n, kv, d), dt)
        s["v_new"] = _randn(gen, (b, n, kv, d), dt)
        s["starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
        # the first token of the first page that each sequence touches, and tokens that cover every page that any does
        s["first"] = torch.tensor([x // bt * bt for x in starts], dtype=torch.int32, device="cuda")
        s["span"] = _span(case)
        if own:
            s["cache"] = _nhip().KvCache8.of(s["k"], s["v"], s["ks"], s["vs"])
    return s


def _span(case):
    """Tokens from the start of the first page touched to the last one written, the longest of the batch."""
    bt = case["block"]
    return max(x % bt + case["tokens"] for x in _lengths(case, case["start"], 0))


# ------------------------------------------------------------------- a pass
def run(s):
    return (_run_own if own else _run_plain)(s)


def _run_own(s):
    nhip = _nhip()
    case = s["case"]
    kind = case["kind"]
    if kind == "norm":
        return s["plan"].forward(s["x"])
    if kind == "rotary":
        return s["plan"].forward(s["x"], s["positions"])
    if kind == "cross":
        return nhip.cross_attention(s["q"], s["k"], s["v"], key_lengths=s["lengths"], key_mask=s["mask"])
    if kind == "cached":
        return s["cache"].attention(s["q"], s["table"], s["lengths"], max_length=case["lmax"], causal=case["causal"])
    s["cache"].append(s["k_new"], s["v_new"], s["table"], s["starts"])
    k, v = s["cache"].read(s["table"], s["first"], s["span"], DTYPES[case["dtype"]])
    return k, v, s["ks"], s["vs"]


def _softmax_products(q, k, v, keep):
    """q [b, kv, rows, d], k and v [b, kv, keys, d] in 32 bits, keep broadcast over [b, kv, rows, keys]."""
    p = torch.matmul(q, k.transpose(2, 3)) * (1.0 / math.sqrt(q.shape[-1]))
    p = torch.where(keep, p, -math.inf)
    top = p.amax(-1, keepdim=True)
    p = torch.exp(p - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    return torch.matmul(p, v) / torch.where(total == 0, 1.0, total)


def _grouped(q, kv):
    """[b, lq, heads, d] -> [b, kv, group * lq, d] in 32 bits, and back by _ungrouped."""
    b, lq, heads, d = q.shape
    return q.float().view(b, lq, kv, heads // kv, d).permute(0, 2, 3, 1, 4).reshape(b, kv, heads // kv * lq, d)


def _ungrouped(o, lq, dtype):
    b, kv, rows, d = o.shape
    return o.view(b, kv, rows // lq, lq, d).permute(0, 3, 1, 2, 4).reshape(b, lq, kv * (rows // lq), d).to(dtype)


def _run_plain(s):
    case = s["case"]
    kind = case["kind"]
    dt = DTYPES[case["dtype"]]
    if kind == "norm":
        n, c, g = case["n"], case["c"], case["groups"]
        x = s["x"].float()
        x = x.view(n, c, -1).transpose(1, 2) if case["layout"] == "blobs" else x
        x = x.reshape(n, -1, g, c // g)
        x = x - x.mean((1, 3), keepdim=True)
        x = x * torch.rsqrt((x * x).mean((1, 3), keepdim=True) + 1e-5)
        y = x.view(n, -1, c) * s["gamma"] + s["beta"]
        y = y.clamp_min(0) if case["act"] == "relu" else y / (1 + torch.exp(-y)) if case["act"] == "silu" else y
        return y.to(dt)
    if kind == "rotary":
        x, r = s["x"].float(), case["rotary"]
        angle = (s["positions"][:, :, s["axis"]] * s["inv_freq"])[:, :, None]
        cos, sin = torch.cos(angle), torch.sin(angle)
        if case["paired"] == "halves":
            a, b = x[..., :r // 2], x[..., r // 2:r]
            y = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
        else:
            a, b = x[..., 0:r:2], x[..., 1:r:2]
            y = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
        return torch.cat([y, x[..., r:]], -1).to(dt)
    if kind == "cross":
        keep = torch.arange(case["lk"], device="cuda") < s["lengths"][:, None]
        keep = keep if s["mask"] is None else keep & s["mask"]
        o = _softmax_products(_grouped(s["q"], case["kv_heads"]), s["k"].float().transpose(1, 2),
                              s["v"].float().transpose(1, 2), keep[:, None, None])
        return _ungrouped(o, case["lq"], dt)
    bt, kv, d, b = case["block"], case["kv_heads"], case["d"], case["b"]
    if kind == "cached":
        lq, table = case["lq"], s["table"].long()
        k, v = ((codes[table] * scale[table][..., None, None]).transpose(1, 2).reshape(b, kv, -1, d)
                for codes, scale in ((s["k"], s["ks"]), (s["v"], s["vs"])))
        last = s["lengths"][:, None]
        if case["causal"]:
            last = last - lq + 1 + torch.arange(lq, device="cuda")
        keep = torch.arange(k.shape[2], device="cuda") < last[..., None]
        keep = keep.repeat(1, case["heads"] // kv if case["causal"] else 1, 1)[:, None]
        return _ungrouped(_softmax_products(_grouped(s["q"], kv), k, v, keep), lq, dt)
    # append: every page that a sequence may touch, [b, pages, tokens of a page]
    n, start = case["tokens"], s["starts"].long()
    pages = (n + bt - 2) // bt + 1
    page = start[:, None] // bt + torch.arange(pages, device="cuda")
    at = page[..., None] * bt + torch.arange(bt, device="cuda")
    new = (at >= start[:, None, None]) & (at < start[:, None, None] + n)
    from_new = (at - start[:, None, None]).clamp(0, n - 1)
    rows = torch.arange(b, device="cuda")[:, None]
    ids = s["table"].long()[rows, page.clamp(max=s["table"].shape[1] - 1)]
    old = (at < start[:, None, None])[:, :, None, :, None]
    begun = (page * bt < start[:, None])[:, :, None]
    fresh = new[:, :, None, :, None]
    out = []
    for codes, scale, x in ((s["k"], s["ks"], s["k_new"]), (s["v"], s["vs"], s["v_new"])):
        x = x.float()[rows[..., None], from_new].transpose(2, 3)  # [b, pages, kv, tokens, d]
        had, had_scale = codes[ids], scale[ids]
        most = torch.where(fresh, x.abs(), 0.0).amax((3, 4))
        want = torch.where(most > 0, (most * (1.0 / 127.0)).clamp_min(TINY), 0.0)
        want = torch.where(begun, torch.maximum(want, had_scale), want)
        touched = new.any(-1)[:, :, None]
        now = torch.where(touched, want, had_scale)
        inv = torch.where(now > 0, 1.0 / torch.where(now > 0, now, 1.0), 0.0)[..., None, None]
        q = torch.where(fresh, x * inv, had * (had_scale[..., None, None] * inv))
        q = torch.trunc(q + torch.copysign(torch.full_like(q, 0.5), q)).clamp(-127, 127).to(torch.int8)
        codes[ids] = torch.where(fresh | (old & touched[..., None, None]), q, had)
        scale[ids] = now
        # read back from the first page touched
        at_read = s["first"].long()[:, None] + torch.arange(s["span"], device="cuda")
        id_read = s["table"].long()[rows, at_read // bt]
        out.append((codes[id_read, :, at_read % bt] * scale[id_read][..., None]).to(dt))
    return out[0], out[1], s["ks"], s["vs"]


# --------------------------------------------------------- what a pass needs
def work(case):
    kind, size = case["kind"], SIZE[case["dtype"]]
    if kind == "norm":
        n = case["n"] * case["h"] * case["w"] * case["c"]
        return {"bytes": 2 * n * size + 8 * case["c"], "flops": 8 * n}
    if kind == "rotary":
        tokens = case["b"] * case["t"] * case["h"] * case["w"]
        return {"bytes": 2 * tokens * case["heads"] * case["d"] * size + 12 * tokens,
                "flops": 3 * tokens * case["heads"] * case["rotary"]}
    kv, d, b = case["kv_heads"], case["d"], case["b"]
    if kind == "cross":
        keys = sum(_lengths(case, case["lk"]))
        rows = case["lq"] * case["heads"]
        return {"bytes": (2 * b * rows + 2 * keys * kv) * d * size + (b * case["lk"] if case["masked"] else 0),
                "flops": 4 * rows * keys * d}
    if kind == "cached":
        lengths, lq = _lengths(case, case["lmax"]), case["lq"]
        pairs = sum(sum(max(0, n - lq + 1 + i) for i in range(lq)) if case["causal"] else n * lq for n in lengths)
        return {"bytes": 2 * b * lq * case["heads"] * d * size
                + 2 * sum(n * d + -(-n // case["block"]) * 4 for n in lengths) * kv,
                "flops": 4 * pairs * case["heads"] * d}
    n = case["tokens"]
    read = b * _span(case)  # values read back, codes and values
    return {"bytes": 2 * kv * d * (b * n * (size + 1) + read * (1 + size)), "flops": 6 * b * n * kv * d}


# ------------------------------------------------------- the same in 64 bits
def exact(case, seed):
    """From the definitions, an image, a head or a page at a time."""
    s = prepare(case, seed)
    kind = case["kind"]
    f64 = torch.float64
    if kind == "norm":
        out = []
        for x in s["x"]:
            x = x.to(f64).reshape(case["c"], -1) if case["layout"] == "blobs" else x.to(f64).t()
            cols = []
            for i, y in enumerate(x.chunk(case["groups"])):
                size = case["c"] // case["groups"]
                y = (y - y.mean()) / math.sqrt(float(y.var(correction=0)) + 1e-5)
                y = y * s["gamma"][i * size:(i + 1) * size, None].to(f64) + s["beta"][i * size:(i + 1) * size, None]
                cols.append(y)
            y = torch.cat(cols).t()
            out.append(y * torch.sigmoid(y) if case["act"] == "silu" else y.relu() if case["act"] == "relu" else y)
        return torch.stack(out).contiguous()
    if kind == "rotary":
        x, y = s["x"].to(f64), s["x"].to(f64)
        pairs = case["rotary"] // 2
        for i in range(pairs):
            j, k = (i, i + pairs) if case["paired"] == "halves" else (2 * i, 2 * i + 1)
            turn = torch.polar(torch.ones((), dtype=f64, device="cuda"),
                               s["positions"][..., int(s["axis"][i])].to(f64) * float(s["inv_freq"][i]))
            z = torch.complex(x[..., j], x[..., k]) * turn[..., None]
            y[..., j], y[..., k] = z.real, z.imag
        return y
    if kind in ("cross", "cached"):
        group = case["heads"] // case["kv_heads"]
        out = torch.zeros(s["q"].shape, dtype=f64, device="cuda")
        lq, d = case["lq"], case["d"]
        for b, n in enumerate(s["lengths"].tolist()):
            for h in range(case["kv_heads"]):
                if kind == "cross":
                    k, v = s["k"][b, :n, h].to(f64), s["v"][b, :n, h].to(f64)
                    if s["mask"] is not None:
                        k, v = k[s["mask"][b, :n]], v[s["mask"][b, :n]]
                else:
                    pages = s["table"][b].long()
                    k, v = ((codes[pages, h].to(f64) * scale[pages, h, None, None]).flatten(0, 1)[:n]
                            for codes, scale in ((s["k"], s["ks"]), (s["v"], s["vs"])))
                if not len(k):
                    continue
                for head in range(h * group, (h + 1) * group):
                    score = s["q"][b, :, head].to(f64) @ k.t() / math.sqrt(d)
                    if kind == "cached" and case["causal"]:
                        ahead = torch.ones_like(score, dtype=torch.bool).triu(n - lq + 1)
                        score = score.masked_fill(ahead, -math.inf)
                    out[b, :, head] = torch.nan_to_num(torch.softmax(score, -1)) @ v
        return out
    bt, n = case["block"], case["tokens"]
    out = []
    for codes, scale, x in ((s["k"], s["ks"], s["k_new"]), (s["v"], s["vs"], s["v_new"])):
        kept, scale = codes.to(f64) * scale[..., None, None], scale.to(f64)
        back = torch.zeros((case["b"], s["span"]) + x.shape[2:], dtype=f64, device="cuda")
        for b, (start, first) in enumerate(zip(s["starts"].tolist(), s["first"].tolist())):
            for i, page in enumerate(s["table"][b].tolist()):
                lo, hi = max(start, i * bt), min(start + n, (i + 1) * bt)
                if lo < hi:
                    y = x[b, lo - start:hi - start].to(f64).transpose(0, 1)
                    step = y.abs().amax((1, 2)) / 127
                    if start > i * bt:
                        step = torch.maximum(step, scale[page])
                        kept[page, :, :start - i * bt] = _steps(kept[page, :, :start - i * bt], step)
                    kept[page, :, lo - i * bt:hi - i * bt] = _steps(y, step)
                    # a page keeps its codes past the last token written, which now stand for steps of this size
                    kept[page, :, hi - i * bt:] *= (step / scale[page])[:, None, None]
                    scale[page] = step
                lo, hi = max(first, i * bt), min(first + s["span"], (i + 1) * bt)
                if lo < hi:
                    back[b, lo - first:hi - first] = kept[page, :, lo - i * bt:hi - i * bt].transpose(0, 1)
        out.append((back, scale))
    return out[0][0], out[1][0], out[0][1], out[1][1]


def _steps(x, step):
    """The nearest whole number of steps, halves away from zero."""
    x = x / step[:, None, None]
    return torch.sign(x) * torch.floor(x.abs() + 0.5) * step[:, None, None]
