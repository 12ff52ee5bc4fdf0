"""Products of tokens in 8-bit integers (Linear8), single and grouped by expert,
against 64 bits."""
import pytest

torch = pytest.importorskip("torch")

import linear8_reference as ref  # noqa: E402
import nhip  # noqa: E402

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
ACTS = {"none": nhip.ACT_NONE, "relu": nhip.ACT_RELU, "silu": nhip.ACT_SILU}


@pytest.fixture(autouse=True)
def _gpu():
    assert torch.cuda.is_available(), "GPU tests need a HIP device"
    nhip.init(0)


def tokens(gen, rows, k, dtype):
    """Tokens of sizes from 2^-8 to 2^4; the second one zeros."""
    x = torch.randn((rows, k), generator=gen) * torch.exp2(torch.randint(-8, 5, (rows, 1), generator=gen).float())
    if rows > 1:
        x[1] = 0
    return x.to(dtype)


def weights(gen, shape, bias):
    w = torch.randint(-127, 128, shape, generator=gen, dtype=torch.int8)
    ws = (0.5 + torch.rand(shape[:-1], generator=gen)) / (70 * shape[-1] ** 0.5)
    return w, ws, torch.randn(shape[:-1], generator=gen) if bias else None


def check(got, want, what=""):
    y, bound = want
    err = (got.cpu().double() - y).abs()
    assert not got.isnan().any() and (err <= bound).all(), f"{what}: {float((err / bound.clamp_min(1e-300)).max()):.3f} of the bound"


SIZES = [(1, 1, 1), (1, 17, 5), (2, 64, 16), (3, 128, 16), (16, 2048, 48), (17, 130, 33), (31, 96, 100), (33, 1000, 257),
         (64, 129, 300), (65, 640, 1000), (255, 65, 31), (256, 512, 256), (257, 260, 500), (700, 1025, 513)]


@pytest.mark.parametrize("tiles", ["-1", "0", "1"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,k,n", SIZES)
def test_product(nhip_env, rows, k, n, dtype, tiles):
    nhip_env.setenv("NHIP_LINEAR8_TILES", tiles)
    gen = torch.Generator().manual_seed(rows + k + n)
    act = ("none", "relu", "silu")[(rows + k) % 3]
    x, (w, ws, b) = tokens(gen, rows, k, TYPES[dtype]), weights(gen, (n, k), n % 2 == 0)
    plan = nhip.Linear8(w.cuda(), ws.cuda(), None if b is None else b.cuda(), ACTS[act])
    check(plan.forward(x.cuda()), ref.product(x, w, ws, b, act))


@pytest.mark.parametrize("rows,k,n", [(16, 8192, 40), (9, 8200, 17), (1, 4100, 33), (16, 2049, 9000), (7, 33, 20000), (3000, 64, 3000),
                                      (49, 300, 40000), (40, 300, 70000), (700, 8192, 100), (16, 2048, 40), (5, 2000, 8192)])
def test_kernels_of_few_and_many(rows, k, n):
    """Sizes on either side of the rules that choose a kernel."""
    gen = torch.Generator().manual_seed(rows)
    x, (w, ws, b) = tokens(gen, rows, k, torch.bfloat16), weights(gen, (n, k), True)
    plan = nhip.Linear8(w.cuda(), ws.cuda(), b.cuda(), nhip.ACT_RELU)
    check(plan.forward(x.cuda()), ref.product(x, w, ws, b, "relu"))


def test_offsets_past_32_bits():
    """Results of more than 2^32 elements' bytes, weights of as many: their ends."""
    gen = torch.Generator().manual_seed(11)
    w, ws, _ = weights(gen, (4096, 64), False)
    plan = nhip.Linear8(w.cuda(), ws.cuda())
    x = torch.randn((600000, 64), device="cuda").half()  # 4.9 GB of results
    got = plan.forward(x)
    for at in (slice(0, 200), slice(599700, 600000)):
        check(got[at], ref.product(x[at], w, ws, None, "none"))
    del got
    many = torch.randint(-127, 128, (300, 4096, 4096), dtype=torch.int8, device="cuda")  # 5 GB of codes
    plan = nhip.Linear8(many, torch.ones((300, 4096), device="cuda"))
    starts = torch.tensor([0] * 150 + [3] * 150 + [8], dtype=torch.int32, device="cuda")
    x = torch.randn((8, 4096), device="cuda")
    got = plan.forward(x, expert_starts=starts)
    for e, at in ((149, slice(0, 3)), (299, slice(3, 8))):
        check(got[at], ref.product(x[at], many[e], torch.ones(4096), None, "none"))


@pytest.mark.parametrize("rows", [5, 300])
def test_shapes_strides_alignment(rows):
    """Rows further apart than their length, not 16-byte aligned, in three dimensions; plans of host arrays."""
    gen = torch.Generator().manual_seed(3)
    w, ws, b = weights(gen, (70, 96), True)
    plan = nhip.Linear8(w.numpy(), ws.numpy(), b)
    for dtype in TYPES.values():
        x = tokens(gen, rows, 96, dtype)
        want = ref.product(x, w, ws, b, "none")
        wide = torch.full((rows, 131), 1e4, dtype=dtype, device="cuda")
        for at in (0, 1, 8, 35):
            wide.fill_(1e4)[:, at:at + 96] = x.cuda()
            check(plan.forward(wide[:, at:at + 96]), want, f"offset {at}")
        check(plan.forward(x.cuda().view(1, rows, 1, 96)).view(rows, 70), want)
        one = x[:1].cuda().expand(rows, 96)  # one token for all rows
        assert torch.equal(plan.forward(one), plan.forward(one.contiguous()))
        out = torch.full((rows, 70), 7.0, dtype=dtype, device="cuda")
        assert plan.forward(x.cuda(), out=out) is out
        check(out, want)
    assert plan.forward(torch.empty((0, 96), device="cuda")).shape == (0, 70)


@pytest.mark.parametrize("tiles", ["-1", "0", "1"])
@pytest.mark.parametrize("counts", [
    [1], [3, 0, 13], [0, 16], [0, 0, 5], [17, 0, 1, 64, 3], [300, 0, 0, 1, 257], [1] * 70, [0] * 66 + [40, 0, 2], [130, 2, 256, 0, 512, 1]])
def test_experts(nhip_env, counts, tiles):
    """Ragged, some without rows, more experts than a wave has lanes; rows before the first and behind the last stay."""
    nhip_env.setenv("NHIP_LINEAR8_TILES", tiles)
    gen = torch.Generator().manual_seed(sum(counts))
    e, k, n = len(counts), 200, 90
    w, ws, b = weights(gen, (e, n, k), True)
    plan = nhip.Linear8(w.cuda(), ws.cuda(), b.cuda(), nhip.ACT_SILU)
    for dtype, before, behind in (("bf16", 0, 0), ("f32", 3, 20), ("f16", 0, 1)):
        starts = before + torch.tensor([sum(counts[:i]) for i in range(e + 1)], dtype=torch.int32)
        rows = before + sum(counts) + behind
        x = tokens(gen, rows, k, TYPES[dtype])
        out = torch.full((rows, n), 7.0, dtype=TYPES[dtype], device="cuda")
        plan.forward(x.cuda(), expert_starts=starts.cuda(), out=out)
        assert (out[:before] == 7).all() and (out[rows - behind:] == 7).all()
        for i, c in enumerate(counts):
            if c:
                at = slice(int(starts[i]), int(starts[i]) + c)
                check(out[at], ref.product(x[at], w[i], ws[i], b[i], "silu"), f"expert {i}")


@pytest.mark.parametrize("tiles", ["-1", "0", "1"])
def test_starts_out_of_range(nhip_env, tiles):
    """Starts are clamped to the rows there are; one that falls leaves an expert without rows."""
    nhip_env.setenv("NHIP_LINEAR8_TILES", tiles)
    gen = torch.Generator().manual_seed(8)
    w, ws, _ = weights(gen, (3, 40, 64), False)
    plan = nhip.Linear8(w.cuda(), ws.cuda())
    x = tokens(gen, 50, 64, torch.float32)
    out = torch.full((50, 40), 7.0, device="cuda")
    plan.forward(x.cuda(), expert_starts=torch.tensor([-5, 20, 10, 2 ** 31 - 1], dtype=torch.int32, device="cuda"), out=out)
    check(out[:10], tuple(t[:10] for t in ref.product(x[:20], w[0], ws[0], None, "none")))
    check(out[20:], ref.product(x[20:], w[2], ws[2], None, "none"))


@pytest.mark.parametrize("tiles", ["0", "1"])
def test_longest_sum(nhip_env, tiles):
    """The largest sums there can be, of the longest rows and codes of -128, are exact."""
    nhip_env.setenv("NHIP_LINEAR8_TILES", tiles)
    k = 131072
    w = torch.full((17, k), -128, dtype=torch.int8)
    w[1], w[2, ::2] = 127, 127
    plan = nhip.Linear8(w.cuda(), torch.ones(17, device="cuda"))
    x = torch.ones((3, k))
    x[1], x[2, 5] = -1, 0.5
    got = plan.forward(x.cuda())
    check(got, ref.product(x, w, torch.ones(17), None, "none"))


@pytest.mark.parametrize("rows", [12, 20])
@pytest.mark.parametrize("tiles", ["-1", "0", "1"])
def test_values(nhip_env, tiles, rows):
    """Subnormal and huge tokens; one with an infinity or NaN is NaN, the others are not touched by it."""
    nhip_env.setenv("NHIP_LINEAR8_TILES", tiles)
    gen = torch.Generator().manual_seed(1)
    w, ws, b = weights(gen, (33, 300), True)
    plan = nhip.Linear8(w.cuda(), ws.cuda(), b.cuda(), nhip.ACT_RELU)
    x = torch.randn((rows, 300), generator=gen)
    x[3] *= 2.0 ** -140
    x[4] = torch.tensor([2.0 ** -149] * 300)
    x[5] *= 2.0 ** 124 / x[5].abs().max()
    want, bound = ref.product(x, w, ws, b, "relu")
    bad = x.clone()
    bad[7, 299], bad[8, 0], bad[9, 17] = float("inf"), -float("inf"), float("nan")
    got = plan.forward(bad.cuda()).cpu()
    hurt = torch.zeros(rows, dtype=torch.bool)
    hurt[7:10] = True
    assert got[hurt].isnan().all()
    check(got[~hurt], (want[~hurt], bound[~hurt]))


def test_weights_in_fp32():
    """Weights are quantised by channel as tokens are, each to a code's half step; a plan keeps no hold on its tensors."""
    gen = torch.Generator().manual_seed(2)
    w = torch.randn((2, 50, 77), generator=gen) * torch.exp2(torch.randint(-4, 5, (2, 50, 1), generator=gen).float())
    w[1, 3] = 0
    codes, scale = ref.codes(w.view(-1, 77))
    assert ((codes * scale[:, None] - w.view(-1, 77)).abs() <= scale[:, None] * (0.5 + 127 * 4 * ref.E)).all()
    host = w.cuda()
    plan = nhip.Linear8(host)
    host.zero_()
    x = tokens(gen, 12, 77, torch.float32)
    starts = torch.tensor([0, 5, 12], dtype=torch.int32, device="cuda")
    got = plan.forward(x.cuda(), expert_starts=starts)
    for e, at in ((0, slice(0, 5)), (1, slice(5, 12))):
        check(got[at], ref.product(x[at], codes.view(2, 50, 77)[e].to(torch.int8), scale.view(2, 50)[e], None, "none"))


def test_refusals():
    w, ws = torch.zeros((8, 16), dtype=torch.int8, device="cuda"), torch.ones(8, device="cuda")
    for bad in (lambda: nhip.Linear8(w), lambda: nhip.Linear8(w.float(), ws), lambda: nhip.Linear8(w, ws[:4]),
                lambda: nhip.Linear8(w, ws, bias=torch.zeros(9)), lambda: nhip.Linear8(w, ws.double())):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        nhip.Linear8(w.half(), ws)
    with pytest.raises(nhip.NhipError):
        nhip.Linear8(w, ws, act=nhip.ACT_SIGMOID)
    plan, many = nhip.Linear8(w, ws), nhip.Linear8(w[None].expand(2, 8, 16), ws[None].expand(2, 8))
    x = torch.zeros((4, 16), device="cuda")
    starts = torch.tensor([0, 2, 4], dtype=torch.int32, device="cuda")
    for bad in (lambda: plan.forward(x[:, :8]), lambda: many.forward(x), lambda: many.forward(x, expert_starts=starts[:2]),
                lambda: many.forward(x, expert_starts=starts.long()), lambda: many.forward(x, expert_starts=starts.cpu()),
                lambda: plan.forward(x.t().contiguous().t()), lambda: plan.forward(x, out=x),
                lambda: plan.forward(x, out=torch.zeros((4, 8), dtype=torch.float16, device="cuda")),
                lambda: plan.forward(x, workspace=torch.empty(1 << 20, dtype=torch.uint8))):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: plan.forward(x.cpu()), lambda: plan.forward(x.double())):
        with pytest.raises(TypeError):
            bad()
    with pytest.raises(nhip.NhipError):
        plan.forward(x, workspace=torch.empty(16, dtype=torch.uint8, device="cuda"))


@pytest.mark.parametrize("rows", [3, 40])
def test_results_over_tokens(rows):
    """Results that overlap a token's row are refused, whatever the number of rows; those beside or between them are not."""
    gen = torch.Generator().manual_seed(4)
    w, ws, b = weights(gen, (64, 64), True)
    plan = nhip.Linear8(w.cuda(), ws.cuda(), b.cuda())
    x = tokens(gen, rows, 64, torch.float16)
    want = ref.product(x, w, ws, b, "none")
    size = rows * 64
    flat = torch.zeros(3 * size, dtype=torch.float16, device="cuda")

    def at(start):
        return flat[start:start + size].view(rows, 64)

    at(size).copy_(x)
    for start in (size, size - 64, size + 64, 1, 2 * size - 1):
        with pytest.raises(nhip.NhipError):
            plan.forward(at(size), out=at(start))
    assert torch.equal(at(size).cpu(), x)  # refused before anything is launched
    for start in (0, 2 * size):
        check(plan.forward(at(size), out=at(start)), want)
    # the results between two rows that lie apart, and over one of them
    wide = torch.zeros((2, 4 * 64), dtype=torch.float16, device="cuda")
    wide[:, :64] = x[:2].cuda()
    between, over = wide.flatten()[64:192].view(2, 64), wide.flatten()[192:320].view(2, 64)
    check(plan.forward(wide[:, :64], out=between), ref.product(x[:2], w, ws, b, "none"))
    with pytest.raises(nhip.NhipError):
        plan.forward(wide[:, :64], out=over)
    one = x[:1].cuda().expand(rows, 64)
    check(plan.forward(one, out=torch.zeros((rows, 64), dtype=torch.float16, device="cuda")), ref.product(one, w, ws, b, "none"))


def test_plan_not_made_in_a_capture():
    w, ws = torch.zeros((8, 16), dtype=torch.int8, device="cuda"), torch.ones(8, device="cuda")
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side, capture_error_mode="relaxed"):
        with pytest.raises(nhip.NhipError):
            nhip.Linear8(w, ws)
    assert nhip.Linear8(w, ws).forward(torch.ones((1, 16), device="cuda")).abs().max() == 0


@pytest.mark.parametrize("rows", [3, 200])
def test_streams_and_graphs(rows):
    """On another stream, and two graphs with a workspace of their own, replayed between eager calls."""
    gen = torch.Generator().manual_seed(5)
    w, ws, b = weights(gen, (200, 512), True)
    plan = nhip.Linear8(w.cuda(), ws.cuda(), b.cuda(), nhip.ACT_SILU)
    xs = [tokens(gen, rows, 512, torch.bfloat16).cuda() for _ in range(4)]
    want = [plan.forward(x) for x in xs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = plan.forward(xs[0], stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want[0])
    held, graphs = [], []
    for i in range(2):
        x, graph = xs[i].clone(), torch.cuda.CUDAGraph()
        ws_ = torch.empty(plan.workspace_size(nhip.DTYPE_BF16, rows), dtype=torch.uint8, device="cuda")
        out = torch.zeros_like(want[0])
        with torch.cuda.graph(graph):
            plan.forward(x, out=out, workspace=ws_)
        held.append((x, ws_, out))
        graphs.append(graph)
    for r in range(4):
        for i in range(2):
            held[i][0].copy_(xs[(r + i) % 4])
            graphs[i].replay()
            assert torch.equal(plan.forward(xs[3]), want[3])
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(held[i][2], want[(r + i) % 4])
