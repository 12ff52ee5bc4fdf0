"""Steps of a decoder whose sequences share a prefix: 8-bit products (fused
query, key and value; output; experts; vocabulary), rotary positions, the 8-bit
cache, attention over prefix and own pages, and the draw, one behind the other.
Every operator's result is checked in 64 bits for the inputs that it had; then
the whole step as a recorded graph against the eager one."""
import pytest

torch = pytest.importorskip("torch")

import linear8_reference as lref  # noqa: E402
import nhip  # noqa: E402
import test_gpu_sample as draw  # noqa: E402
import token_reference as ref  # noqa: E402

pytestmark = pytest.mark.gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


class Decoder:
    GROUPS, MEMBERS, HEADS, KV, D, DIM, EXPERTS, WIDE, VOCAB, BLOCK, PREFIX, STEPS = 2, 3, 4, 2, 32, 128, 4, 96, 1003, 16, 70, 20

    def __init__(self, dtype, seed=0):
        gen = torch.Generator().manual_seed(seed)
        self.dtype, self.batch = dtype, self.GROUPS * self.MEMBERS
        self.layers = {}

        def layer(name, n, k, experts=None, act=nhip.ACT_NONE):
            w = torch.randint(-127, 128, ((experts, n, k) if experts else (n, k)), generator=gen, dtype=torch.int8)
            ws = (0.5 + torch.rand(w.shape[:-1], generator=gen)) / (70 * k ** 0.5)
            b = 0.1 * torch.randn(w.shape[:-1], generator=gen)
            self.layers[name] = (w, ws, b, act, nhip.Linear8(w.cuda(), ws.cuda(), b.cuda(), act))

        layer("qkv", (self.HEADS + 2 * self.KV) * self.D, self.DIM)
        layer("out", self.DIM, self.HEADS * self.D)
        layer("router", self.EXPERTS, self.DIM)
        layer("up", self.WIDE, self.DIM, self.EXPERTS, nhip.ACT_SILU)
        layer("down", self.DIM, self.WIDE, self.EXPERTS)
        layer("vocabulary", self.VOCAB, self.DIM)
        self.embedding = torch.randn((self.VOCAB, self.DIM), generator=gen).to(dtype).cuda()
        self.rotary = nhip.Rotary(self.D, (self.D // 2,))
        per_prefix, per_own = -(-self.PREFIX // self.BLOCK), -(-self.STEPS // self.BLOCK)
        pages = self.GROUPS * per_prefix + self.batch * per_own
        order = torch.randperm(pages, generator=gen).int().cuda()
        self.prefix_table = order[:self.GROUPS * per_prefix].view(self.GROUPS, per_prefix)
        self.table = order[self.GROUPS * per_prefix:].view(self.batch, per_own).contiguous()
        self.cache = nhip.KvCache8(pages, self.KV, self.D, self.BLOCK)
        self.prefix_lengths = torch.tensor([self.PREFIX, self.PREFIX - 9], dtype=torch.int32, device="cuda")
        self.settings = [torch.tensor(v, device="cuda") for v in ([0.8, 1.0, 0.0, 1.2, 0.7, 1.0], [0, 40, 0, 5, 300, 0],
                                                                   [0.9, 1.0, 0.5, 0.8, 0.95, 1.0], [0.0, 0.01, 0.0, 0.0, 0.02, 0.0])]
        self.settings[1] = self.settings[1].int()
        self.uniform = torch.rand((self.STEPS, self.batch), generator=gen).cuda()
        self.prompt = torch.randint(0, self.VOCAB, (self.GROUPS, self.PREFIX), generator=gen).cuda()
        self.seen = None  # a list: (operator, inputs, result) of each call, while it is one

    def linear(self, name, x, starts=None):
        y = self.layers[name][4].forward(x, expert_starts=starts)
        self.note(name, x, starts, y)
        return y

    def note(self, *what):
        if self.seen is not None:
            self.seen.append(tuple(t.clone() if isinstance(t, torch.Tensor) else t for t in what))

    def project(self, x, positions):
        """Queries, keys and values: views of one product's result, turned in place."""
        b, n = x.shape[:2]
        y = self.linear("qkv", x.reshape(-1, self.DIM)).view(b, n, self.HEADS + 2 * self.KV, self.D)
        q, k, v = y[:, :, :self.HEADS], y[:, :, self.HEADS:self.HEADS + self.KV], y[:, :, self.HEADS + self.KV:]
        for t in (q, k):
            was = t.clone()
            self.rotary.forward(t, positions, out=t)
            self.note("rotary", was, positions, t)
        return q, k, v

    def read_prompt(self):
        x = self.embedding[self.prompt]
        pos = torch.arange(self.PREFIX, dtype=torch.int32, device="cuda").view(1, -1, 1)
        _, k, v = self.project(x, pos)
        self.cache.append(k, v, self.prefix_table, torch.zeros(self.GROUPS, dtype=torch.int32, device="cuda"), self.prefix_lengths)

    def step(self, tokens, held, uniform):
        """tokens [batch], held int32 [batch]: own tokens so far -> (tokens, logprobs)."""
        x = self.embedding[tokens.long()].view(self.batch, 1, self.DIM)
        pos = (self.prefix_lengths.repeat_interleave(self.MEMBERS) + held).view(self.batch, 1, 1)
        q, k, v = self.project(x, pos)
        self.cache.append(k, v, self.table, held)
        lengths = held + 1
        o = self.cache.prefix_attention(q, self.prefix_table, self.prefix_lengths, self.table, lengths, causal=True)
        if self.seen is not None:
            self.note("attention", q, lengths, o, [t.clone() for t in (self.cache.k, self.cache.v, self.cache.k_scale, self.cache.v_scale)])
        x = x.view(self.batch, self.DIM) + self.linear("out", o.view(self.batch, -1))
        # the two best experts of each token: rows in the experts' order, and back
        best = torch.topk(self.linear("router", x).float(), 2, dim=1)[1].flatten()
        order = torch.argsort(best, stable=True)
        starts = (best[None] < torch.arange(self.EXPERTS + 1, device="cuda")[:, None]).sum(1).int()
        y = self.linear("down", self.linear("up", x[order // 2], starts), starts)
        back = torch.zeros_like(y)
        back[order] = y
        x = x + back.view(self.batch, 2, self.DIM).sum(1)
        logits = self.linear("vocabulary", x)
        tokens, logprob = nhip.sample(logits, uniform, *self.settings)
        self.note("sample", logits, uniform, tokens, logprob)
        return tokens, logprob


def check_product(d, name, x, starts, y):
    w, ws, b, act, _ = d.layers[name]
    bounds = [0, len(x)] if starts is None else starts.tolist()
    for e, (lo, hi) in enumerate(zip(bounds, bounds[1:])):
        if lo < hi:
            want, bound = lref.product(x[lo:hi], *(t if starts is None else t[e] for t in (w, ws, b)), "silu" if act else "none")
            ref.assert_within(y[lo:hi], want, bound, name)


def check_attention(d, q, lengths, o, kept):
    values = []
    for table, rows in ((d.prefix_table, d.MEMBERS), (d.table, 1)):
        ids = table.cpu().long()
        values.append([(c.cpu().double() * s.cpu().double()[:, :, None, None])[ids].transpose(2, 3).flatten(1, 2).repeat_interleave(rows, 0)
                       for c, s in ((kept[0], kept[2]), (kept[1], kept[3]))])
    k, v = (torch.cat([a, b], 1) for a, b in zip(*values))
    np_ = d.prefix_lengths.cpu().repeat_interleave(d.MEMBERS)[:, None]
    wide = values[0][0].shape[1]
    t = torch.arange(k.shape[1])
    keep = (t < np_) & (t < wide) | (t >= wide) & (t - wide < lengths.cpu()[:, None])
    want, bound = ref.attention(q.cpu(), k, v, keep[:, None], d.D ** -0.5, d.dtype)
    ref.assert_within(o, want, bound, "attention")


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_steps(dtype):
    nhip.init(0)
    d = Decoder(dtype)
    d.read_prompt()
    tokens = torch.arange(d.batch, dtype=torch.int32, device="cuda")
    held = torch.zeros(d.batch, dtype=torch.int32, device="cuda")
    operators = set()
    for i in range(d.STEPS):
        d.seen = [] if i % 6 == 0 else None
        if i == 0:
            d.read_prompt()  # (the same into the same pages)
        tokens, logprob = d.step(tokens, held, d.uniform[i])
        held = held + 1
        assert ((tokens >= 0) & (tokens < d.VOCAB)).all()
        for name, *what in d.seen or ():
            operators.add(name)
            if name == "rotary":
                x, positions, y = what
                freq = [10000.0 ** (-j / (d.D // 2)) for j in range(d.D // 2)]
                ref.assert_within(y, *ref.rotary(x, positions, (d.D // 2,), freq, False), name)
            elif name == "attention":
                check_attention(d, *what)
            elif name == "sample":
                logits, uniform, got, lp = what
                draw.check((got, lp), logits, uniform, [s.cpu() for s in d.settings])
            else:
                check_product(d, name, *what)
    assert operators == {"qkv", "rotary", "attention", "out", "router", "up", "down", "vocabulary", "sample"}


def test_recorded():
    """The step as a graph, replayed on its own buffers, draws what the eager one does."""
    nhip.init(0)
    runs = []
    for recorded in (False, True):
        d = Decoder(BF16, seed=2)
        d.read_prompt()
        tokens = torch.arange(d.batch, dtype=torch.int32, device="cuda")
        held, uniform = torch.zeros(d.batch, dtype=torch.int32, device="cuda"), torch.zeros(d.batch, device="cuda")
        if recorded:
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):  # (once before the recording, into pages that the replays write again)
                d.step(tokens, held, uniform)
            torch.cuda.current_stream().wait_stream(side)
            d.cache.k_scale[d.table.long()] = 0
            d.cache.v_scale[d.table.long()] = 0
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                new, logprob = d.step(tokens, held, uniform)
        got = []
        for i in range(d.STEPS):
            uniform.copy_(d.uniform[i])
            if recorded:
                graph.replay()
            else:
                new, logprob = d.step(tokens, held, uniform)
            got.append((new.cpu(), logprob.cpu()))
            tokens.copy_(new)
            held += 1
        runs.append(got)
    for (a, b), (c, e) in zip(*runs):
        assert torch.equal(a, c) and torch.equal(b, e)
