"""Drawing the next token (sample) against its definition in 64 bits."""
from fractions import Fraction

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import nhip  # noqa: E402

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(autouse=True)
def _gpu():
    assert torch.cuda.is_available(), "GPU tests need a HIP device"
    nhip.init(0)


def f32(v):
    return float(np.float32(v))


def outcomes(x, u, temperature, top_k, top_p, min_p):
    """{token: its log probabilities} of a row x in 64 bits.  More than one only where a border lies within what rounding
    every weight to 2^-44 of the largest moves it (half of that a weight; the 64-bit sums' own error is less)."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    top = x.max()
    if top == -np.inf:
        return {-1: {-np.inf}}
    if not temperature > 0:
        return {int(np.argmax(x)): {0.0}}
    order = np.lexsort((np.arange(len(x)), -x))
    with np.errstate(over="ignore", invalid="ignore"):
        ly = np.where(x == top, 0.0, (x - top) / temperature)[order]
    w = np.exp(ly)
    n = min(top_k, len(x)) if top_k > 0 else len(x)
    eps = int(((w[:n] > 0) & (w[:n] < 1)).sum()) * 2.0 ** -45  # (0 and 1 are not rounded)
    before = np.cumsum(w[:n]) - w[:n]
    total = w[:n].sum()
    found = {}
    for slack in (-eps, 0.0, eps):
        stays = (w[:n] >= min_p + np.sign(slack) * 2.0 ** -45) | (w[:n] == 1)  # (the largest weight is not rounded)
        if top_p < 1:
            stays &= before < top_p * total + slack
        stays[0] = True
        m = int(np.argmin(stays)) if not stays.all() else n
        at = np.argsort(order[:m])
        upto = np.cumsum(w[:m][at])
        for t in {u * upto[-1] - eps, u * upto[-1], u * upto[-1] + eps}:
            i = min(int(np.searchsorted(upto, max(t, 0.0), side="right")), m - 1)
            while w[:m][at][i] < 2.0 ** -46 and i:
                i -= 1
            found.setdefault(int(order[:m][at][i]), set()).add(float(ly[:m][at][i] - np.log(upto[-1])))
    return found


def check(got, logits, uniform, settings):
    """A token is one of the definition's outcomes; its logarithm is rounded to fp32 once."""
    token, logprob = (t.cpu() for t in got)
    assert token.dtype == torch.int32 and logprob.dtype == torch.float32
    x = logits.detach().cpu().float().numpy()
    several = 0
    for r in range(len(x)):
        of = [f32(v[r]) if isinstance(v, torch.Tensor) else f32(v) for v in settings]
        want = outcomes(x[r], float(uniform[r]), of[0], int(of[1]), of[2], of[3])
        several += len(want) > 1
        assert int(token[r]) in want, (r, int(token[r]), want, of)
        got_lp, lps = float(logprob[r]), want[int(token[r])]
        assert any(got_lp == lp or abs(got_lp - lp) <= 2.0 ** -23 * abs(lp) + 1e-9 for lp in lps), (r, got_lp, lps)
    assert several <= max(1, len(x) // 50)  # borders are rarely that near


SETTINGS = [(1.0, 0, 1.0, 0.0), (0.7, 50, 1.0, 0.0), (1.0, 0, 0.9, 0.0), (1.3, 40, 0.8, 0.0), (0.9, 0, 1.0, 0.05),
            (0.8, 20, 0.95, 0.1), (0.0, 0, 1.0, 0.0), (1.0, 1, 1.0, 0.0), (2.5, 3000, 0.99, 0.0), (1.0, 1500, 1.0, 0.001),
            (0.05, 0, 0.5, 0.0), (1.0, 0, 0.0, 0.0), (1.0, 7, 1.0, 1.0)]


@pytest.mark.parametrize("settings", SETTINGS)
@pytest.mark.parametrize("dtype", TYPES)
def test_settings(dtype, settings):
    """Small and large vocabularies, odd ones, whose rows begin at any alignment."""
    gen = torch.Generator().manual_seed(4)
    for vocab, rows in ((1, 3), (2, 9), (5, 9), (63, 9), (100, 9), (1000, 16), (4099, 5), (8192, 5), (8193, 5), (50021, 6),
                        (131072, 3)):
        logits = (torch.randn((rows, vocab), generator=gen) * 3).to(TYPES[dtype])
        u = torch.rand((rows,), generator=gen)
        u[0] = 0
        u[-1] = 1 - 2.0 ** -24
        check(nhip.sample(logits.cuda(), u.cuda(), *settings), logits, u, settings)


@pytest.mark.parametrize("chunks", ["0", "1", "5", "64"])
@pytest.mark.parametrize("settings", SETTINGS + [(1.0, 0, 0.999, 0.0), (1.2, 0, 0.3, 0.0)])
def test_rows_begun_by_several(nhip_env, settings, chunks):
    """Long rows are begun by so many workgroups each, here rows of any length."""
    nhip_env.setenv("NHIP_SAMPLE_CHUNKS", chunks)
    gen = torch.Generator().manual_seed(8)
    for (vocab, rows), dtype in zip(((1, 2), (70, 5), (3001, 6), (20011, 5), (60000, 3)), ("f32", "bf16", "f16", "f32", "bf16")):
        logits = (torch.randn((rows, vocab), generator=gen) * 3).to(TYPES[dtype])
        u = torch.rand((rows,), generator=gen)
        check(nhip.sample(logits.cuda(), u.cuda(), *settings), logits, u, settings)


def test_many_rows_and_many_kept():
    """More rows than CUs; more kept tokens than LDS holds, by one filter and by both; the largest vocabulary."""
    gen = torch.Generator().manual_seed(12)
    for rows, vocab, scale, settings in ((300, 17001, 3.0, (1.0, 0, 0.9, 0.0)), (3, 120011, 1.0, (1.5, 0, 0.95, 0.0)),
                                         (3, 120011, 1.0, (1.5, 60000, 0.9, 0.001)), (2, 120011, 0.5, (2.0, 0, 1.0, 0.05)),
                                         (2, 2 ** 19, 2.0, (1.0, 0, 0.99, 0.0)), (2, 2 ** 19, 0.0, (1.0, 0, 1.0, 0.0))):
        logits, u = torch.randn((rows, vocab), generator=gen) * scale, torch.rand((rows,), generator=gen)
        check(nhip.sample(logits.cuda(), u.cuda(), *settings), logits, u, settings)


@pytest.mark.parametrize("chunks", ["0", "3"])
@pytest.mark.parametrize("dtype", TYPES)
def test_each_row_its_own(nhip_env, dtype, chunks):
    nhip_env.setenv("NHIP_SAMPLE_CHUNKS", chunks)
    gen = torch.Generator().manual_seed(6)
    rows, vocab = 40, 20011
    wide = (torch.randn((rows, vocab + 30), generator=gen) * 4).to(TYPES[dtype])
    logits, u = wide[:, 13:13 + vocab], torch.rand((rows,), generator=gen)
    i = torch.arange(rows)
    settings = [torch.where(i % 4 == 3, 0.0, 0.5 + 0.05 * (i % 16)), torch.where(i % 3 == 2, 0, 5 + 40 * i).to(torch.int32),
                torch.where(i % 5 == 4, 1.0, 0.7 + 0.01 * (i % 25)), torch.where(i % 2 == 1, 0.02, 0.0)]
    got = nhip.sample(wide.cuda()[:, 13:13 + vocab], u.cuda(), *(v.cuda() for v in settings))
    check(got, logits, u, settings)


@pytest.mark.parametrize("chunks", ["0", "-1", "4"])
@pytest.mark.parametrize("spread", [0.0, 1e-3, 30.0, 3000.0])
def test_spreads(nhip_env, spread, chunks):
    """Logits that are all alike, hardly apart (borders lie among thousands of neighbours), or very far apart."""
    nhip_env.setenv("NHIP_SAMPLE_CHUNKS", chunks)
    gen = torch.Generator().manual_seed(7)
    for dtype in TYPES.values():
        logits = (torch.randn((4, 30011), generator=gen) * spread + 5).to(dtype)
        u = torch.rand((4,), generator=gen)
        for settings in SETTINGS:
            if spread and settings[2] < 1 or spread > 1e-3:
                check(nhip.sample(logits.cuda(), u.cuda(), *settings), logits, u, settings)


def test_equal_logits():
    """Of equal ones the lower index comes first, and borders that the sums meet exactly are not passed."""
    for vocab in (8, 1000, 9000, 40000, 262144):
        logits = torch.zeros((64, vocab), device="cuda")
        u = (torch.arange(64, device="cuda") + 0.5) / 64
        for settings, kept in (((1.0, 0, 0.5, 0.0), vocab // 2), ((1.0, vocab // 4, 1.0, 0.0), vocab // 4),
                               ((1.0, vocab // 2, 0.25, 0.0), vocab // 8), ((1.0, 0, 1.0, 1.0), vocab)):
            token, logprob = nhip.sample(logits, u, *settings)
            assert torch.equal(token.cpu(), (u.cpu().double() * kept).int()), (vocab, settings)
            assert torch.allclose(logprob.cpu(), -torch.log(torch.tensor(float(kept))), rtol=2e-7)
    # two values, the border among the lower ones
    logits = torch.zeros((16, 50000), device="cuda")
    logits[:, 25000] = 3.0
    u = (torch.arange(16, device="cuda") + 0.5) / 16
    check(nhip.sample(logits, u, 1.0, 9000, 1.0, 0.0), logits, u, (1.0, 9000, 1.0, 0.0))
    check(nhip.sample(logits, u, 1.0, 0, 0.7, 0.0), logits, u, (1.0, 0, 0.7, 0.0))


def test_shares():
    """Over a grid of uniform numbers every token comes as often as its probability says, to one."""
    logits = torch.randn((1, 50), generator=torch.Generator().manual_seed(2)).cuda()
    n = 8192
    u = (torch.arange(n, device="cuda") + 0.5) / n
    token, logprob = nhip.sample(logits.expand(n, 50), u, 0.8)
    share = torch.softmax(logits[0].double() / f32(0.8), 0)
    counts = torch.bincount(token.long(), minlength=50)
    assert ((counts - share * n).abs() <= 1).all()
    assert (logprob.double() - share[token.long()].log()).abs().max() < 1e-6


@pytest.mark.parametrize("chunks", ["0", "2"])
@pytest.mark.parametrize("vocab", [7, 3000, 20000])
@pytest.mark.parametrize("dtype", TYPES)
def test_infinities_and_nan(nhip_env, dtype, vocab, chunks):
    nhip_env.setenv("NHIP_SAMPLE_CHUNKS", chunks)
    gen = torch.Generator().manual_seed(9)
    logits = (torch.randn((10, vocab), generator=gen) * 2).to(TYPES[dtype])
    lowest = torch.finfo(TYPES[dtype]).min
    logits[0] = -float("inf")
    logits[1] = float("nan")
    logits[2, 1:] = -float("inf")
    logits[3, ::2] = float("nan")
    logits[4, 3] = logits[4, 5] = float("inf")
    logits[5] = float("inf")
    logits[6, 2:] = lowest
    logits[7] = lowest
    logits[8] = -logits[7]
    u = torch.rand((10,), generator=gen)
    for settings in SETTINGS:
        if vocab < 10000 or settings[1] < 1500 or settings[1] == 0:
            check(nhip.sample(logits.cuda(), u.cuda(), *settings), logits, u, settings)


def test_settings_out_of_range():
    """What a row's own setting may not be acts as the nearest that it may, NaN as left out; uniform numbers are clamped."""
    gen = torch.Generator().manual_seed(3)
    nan, inf = float("nan"), float("inf")
    logits = torch.randn((8, 9001), generator=gen) * 3
    u = torch.tensor([0.3, 0.6, -1.0, 2.0, nan, 0.2, 0.9, 0.5])
    given = [torch.tensor([1.0, -1.0, 1.0, 1.0, 1.0, nan, 1.0, inf]), torch.tensor([-5, 0, 0, 2 ** 31 - 1, 0, 0, 9002, 0], dtype=torch.int32),
             torch.tensor([nan, 1.0, -0.5, 7.0, 1.0, 1.0, 0.9, 1.0]), torch.tensor([0.0, 0.0, 0.0, 0.0, nan, 0.0, 5.0, -1.0])]
    means = [torch.tensor([1.0, 0.0, 1.0, 1.0, 1.0, 0.0, 1.0, 1e30]), torch.zeros(8, dtype=torch.int32),
             torch.tensor([1.0, 1.0, 0.0, 1.0, 1.0, 1.0, 0.9, 1.0]), torch.tensor([0.0, 0.0, 0.0, 0.0, 0.0, 0.0, 1.0, 0.0])]
    clamped = torch.tensor([0.3, 0.6, 0.0, 1 - 1e-15, 0.0, 0.2, 0.9, 0.5], dtype=torch.float64)
    check(nhip.sample(logits.cuda(), u.cuda(), *(v.cuda() for v in given)), logits, clamped, means)


@pytest.mark.parametrize("chunks", ["0", "5"])
@pytest.mark.parametrize("vocab", [60, 3000, 20011])
def test_next_to_weightless(nhip_env, vocab, chunks):
    """Tokens as far from the largest as weights are not 0, to a rounding of fp32: fewer than top_k weigh anything."""
    nhip_env.setenv("NHIP_SAMPLE_CHUNKS", chunks)
    for top, near, low, temperature in ((20.0, 16.84999, -50.0, 0.1), (100000.0, 99999.65, 0.0, 0.01), (-7000.0, -7031.5005, -8000.0, 1.0)):
        logits = torch.full((8, vocab), low)
        logits[:, 41] = top
        logits[:4, 7] = near
        logits[4:, 20:40] = near
        u = torch.tensor([0.0, 0.3, 0.9, 0.999] * 2)
        for top_k, top_p, min_p in ((2, 1.0, 0.0), (20, 1.0, 0.0), (50, 1.0, 0.0), (50, 0.9, 0.0), (50, 1.0, 1e-3), (0, 0.9, 0.0), (0, 1.0, 0.0)):
            token, logprob = nhip.sample(logits.cuda(), u.cuda(), temperature, top_k, top_p, min_p)
            assert (token == 41).all() and (logprob.abs() < 1e-9).all(), (top, top_k, top_p, token, logprob)


@pytest.mark.parametrize("chunks", ["0", "5"])
def test_farthest_logits(nhip_env, chunks):
    """Logits at either end of fp32, at temperatures that leave both some weight."""
    nhip_env.setenv("NHIP_SAMPLE_CHUNKS", chunks)
    most = torch.finfo(torch.float32).max
    for vocab in (50, 9001):
        logits = torch.full((6, vocab), -most)
        logits[:, 3] = most
        logits[2:4, 5::2] = 0
        u = torch.tensor([0.2, 0.999, 0.5, 0.99, 0.7, 0.05])
        for settings in ((1e38, 0, 1.0, 0.0), (3e38, 0, 0.999, 0.0), (3e38, 40, 1.0, 0.0), (2e38, 0, 1.0, 0.01), (3e38, 2000, 0.99, 0.0)):
            check(nhip.sample(logits.cuda(), u.cuda(), *settings), logits, u, settings)


def whole(logit):
    """The weight of a logit as a whole multiple of 2^-44, None next to a half: 64 bits leave 2^-7 of it uncertain."""
    w = np.exp(float(logit)) * 2.0 ** 44
    return None if abs(w - np.floor(w) - 0.5) < 0.05 else int(np.rint(w))


def draw_exactly(weights, order, top_p, u):
    """(token, kept) by whole numbers and fractions alone."""
    total, before, kept = sum(weights), 0, []
    for i in order:
        if top_p >= 1 or before < Fraction(top_p) * total or not kept:
            kept.append(i)
        before += weights[i]
    target, upto = Fraction(u) * sum(weights[i] for i in kept), 0
    for i in sorted(kept):
        upto += weights[i]
        if upto > target:
            return i, kept
    raise AssertionError


@pytest.mark.parametrize("chunks", ["0", "3"])
@pytest.mark.parametrize("off", [2, -2, 6])
@pytest.mark.parametrize("spread", [(0.01, 0.01), (0.001, 0.001), (0.02, 0.6)])
def test_borders_of_large_sums(nhip_env, spread, off, chunks):
    """Sums past 2^53 units, off from a border by less than a 64-bit float holds: 1024 logits of 0, the others weigh
    2^54 + off together (chosen one by one to that), so that half of all lies off / 2 beyond the first 1024."""
    nhip_env.setenv("NHIP_SAMPLE_CHUNKS", chunks)
    left, rest = 2 ** 54 + off, []
    low = np.linspace(*spread, 2048).astype(np.float32)
    while left:
        at = min(-low[len(rest)], np.float32(np.log(left * 2.0 ** -44)))
        while whole(at) is None or whole(at) > left:
            at = np.nextafter(at, np.float32(-100))
        rest.append(at)
        left -= whole(at)
    logits = torch.cat([torch.zeros(1024), torch.from_numpy(np.array(rest, dtype=np.float32))])
    weights = [whole(v) for v in logits]
    assert sum(weights) == 2 ** 55 + off
    order = sorted(range(len(weights)), key=lambda i: (-float(logits[i]), i))
    for settings, us in (((1.0, 0, 0.5, 0.0), (0.5, 1 - 2.0 ** -24)), ((1.0, 0, 1.0, 0.0), (0.5, 0.25))):
        u = torch.tensor(us)
        token, logprob = nhip.sample(logits.repeat(2, 1).cuda(), u.cuda(), *settings)
        for r in range(2):
            want, kept = draw_exactly(weights, order, settings[2], us[r])
            assert int(token[r]) == want, (settings, us[r])
            assert abs(float(logprob[r]) - (float(logits[want]) - np.log(sum(weights[i] for i in kept) * 2.0 ** -44))) < 2e-6


@pytest.mark.parametrize("settings,most", [((0.0, 0, 1.0, 0.0), 2), ((0.0, 40, 0.9, 0.0), 2), ((1.0, 1, 0.9, 0.0), 2), ((1.0, 0, 1.0, 0.1), 2),
                                           ((1.0, 0, 1.0, 0.0), 3), ((1.0, 40, 0.9, 0.0), 3), ((1.0, 0, 0.9, 0.0), 4)])
def test_launches(nhip_env, settings, most):
    """No launch where the settings leave all rows nothing for it to do."""
    nhip_env.setenv("NHIP_SAMPLE_CHUNKS", "4")
    gen = torch.Generator().manual_seed(13)
    logits, u = torch.randn((6, 30011), generator=gen) * 3, torch.rand((6,), generator=gen)
    nhip.timer_start()
    got = nhip.sample(logits.cuda(), u.cuda(), *settings)
    torch.cuda.synchronize()
    assert nhip.timer_stop()[0] <= most
    check(got, logits, u, settings)


def test_settings_past_32_bits():
    x, u = torch.zeros((4, 50), device="cuda"), torch.zeros(4, device="cuda")
    for top_k in (-1, -2 ** 31 - 1, -2 ** 32 + 5, -2 ** 40):
        with pytest.raises(nhip.NhipError):
            nhip.sample(x, u, top_k=top_k)
    for top_k in (2 ** 31, 2 ** 32 + 5):  # all of them
        assert torch.allclose(nhip.sample(x, u, top_k=top_k)[1].cpu(), -torch.log(torch.tensor(50.0)))


def test_refusals():
    x, u = torch.zeros((4, 50), device="cuda"), torch.zeros(4, device="cuda")
    for bad in (dict(temperature=-1.0), dict(temperature=float("nan")), dict(top_k=-1), dict(top_p=-0.1), dict(min_p=1.5),
                dict(min_p=-0.1), dict(top_p=float("nan"))):
        with pytest.raises(nhip.NhipError):
            nhip.sample(x, u, **bad)
    for bad in (lambda: nhip.sample(x, u[:3]), lambda: nhip.sample(x, u.double()), lambda: nhip.sample(x, u.cpu()),
                lambda: nhip.sample(x, u, temperature=u[:2]), lambda: nhip.sample(x, u, top_k=u),
                lambda: nhip.sample(x, u, top_p=u.cpu()), lambda: nhip.sample(x.t(), torch.zeros(50, device="cuda")),
                lambda: nhip.sample(x, u, out=(u, u)), lambda: nhip.sample(x[0], u)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        nhip.sample(x.double(), u)
    token, logprob = nhip.sample(x[:0], u[:0])
    assert token.shape == (0,) and logprob.shape == (0,)


def test_streams_and_graphs():
    gen = torch.Generator().manual_seed(5)
    logits = [(torch.randn((7, 30000), generator=gen) * 3).to(torch.bfloat16).cuda() for _ in range(4)]
    u = torch.rand((7,), generator=gen).cuda()
    settings = (0.9, 0, 0.9, 0.01)
    want = [nhip.sample(x, u, *settings) for x in logits]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = nhip.sample(logits[0], u, *settings, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want[0]))
    held, graphs = [], []
    for i in range(2):
        x, out, graph = logits[i].clone(), (torch.zeros(7, dtype=torch.int32, device="cuda"), torch.zeros(7, device="cuda")), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            nhip.sample(x, u, *settings, out=out)
        held.append((x, out))
        graphs.append(graph)
    for r in range(4):
        for i in range(2):
            held[i][0].copy_(logits[(r + i) % 4])
            graphs[i].replay()
            assert torch.equal(nhip.sample(logits[3], u, *settings)[0], want[3][0])
        torch.cuda.synchronize()
        for i in range(2):
            assert all(torch.equal(a, b) for a, b in zip(held[i][1], want[(r + i) % 4]))
