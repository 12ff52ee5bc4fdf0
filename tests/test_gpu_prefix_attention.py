"""Attention over the 8-bit cache of sequences that share a prefix, against 64
bits (tests/token_reference.py derives the bounds)."""
import pytest

torch = pytest.importorskip("torch")

import nhip  # noqa: E402
import token_reference as ref  # noqa: E402

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    assert torch.cuda.is_available(), "GPU tests need a HIP device"
    nhip.init(0)


def randn(seed, shape, dtype=F32):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def filled(pages, hkv, d, block, seed=0):
    """A cache of random codes; scales of pages spread over a factor of 30."""
    cache = nhip.KvCache8(pages, hkv, d, block)
    g = torch.Generator().manual_seed(seed)
    for codes, scales in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        codes.copy_(torch.randint(-127, 128, codes.shape, generator=g, dtype=torch.int8))
        scales.copy_(torch.exp(torch.randn(scales.shape, generator=g)) * 0.015)
    return cache


def values(cache, table):
    """(k, v [rows of the table, tokens, heads, d] in 64 bits, which tokens have a page)."""
    ids = table.cpu().long()
    there = (ids >= 0) & (ids < cache.k.shape[0])
    ids = torch.where(there, ids, 0)
    k, v = ((codes.cpu().double() * scales.cpu().double()[:, :, None, None])[ids].transpose(2, 3).flatten(1, 2)
            for codes, scales in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))
    return k, v, there.repeat_interleave(cache.block_tokens, 1)


def check(cache, q, prefix_table, prefix_lengths, table, lengths, causal, max_prefix=None, max_length=None, scale=None, **kw):
    b, lq, h, d = q.shape
    got = cache.prefix_attention(q, prefix_table, ints(prefix_lengths), table, ints(lengths), max_prefix=max_prefix,
                                 max_length=max_length, causal=causal, scale=scale, **kw)
    members = b // len(prefix_lengths)
    kp, vp, there_p = (t.repeat_interleave(members, 0) for t in values(cache, prefix_table))
    ko, vo, there_o = values(cache, table)
    np_ = torch.as_tensor(prefix_lengths).clamp(0, kp.shape[1] if max_prefix is None else max_prefix).repeat_interleave(members)
    no = torch.as_tensor(lengths).clamp(0, ko.shape[1] if max_length is None else max_length)[:, None]
    last = no - lq + 1 + torch.arange(lq) if causal else no.expand(b, lq)
    keep_p = ((torch.arange(kp.shape[1]) < np_[:, None]) & there_p)[:, None].expand(b, lq, kp.shape[1])
    keep_o = (torch.arange(ko.shape[1]) < torch.minimum(last, no)[..., None]) & there_o[:, None]
    want, bound = ref.attention(q.cpu(), torch.cat([kp, ko], 1), torch.cat([vp, vo], 1), torch.cat([keep_p, keep_o], 2),
                                d ** -0.5 if scale is None else scale, q.dtype)
    ref.assert_within(got, want, bound, f"{tuple(q.shape)} {q.dtype} {causal}")
    return got


SHAPES = [
    # groups, members, lq, heads, kv_heads, d, block, prefix lengths, own lengths
    (1, 1, 1, 1, 1, 64, 16, (1,), (1,)),
    (1, 5, 1, 12, 12, 64, 16, (197,), (37, 20, 1, 0, 36)),
    (2, 3, 1, 8, 2, 128, 64, (700, 0), (70, 0, 33, 5, 0, 64)),   # a group without a prefix, one sequence without a key
    (1, 40, 1, 16, 4, 96, 32, (1500,), None),
    (3, 7, 4, 6, 3, 40, 16, (100, 333, 16), None),
    (1, 48, 3, 8, 1, 128, 64, (2049,), None),
    (2, 9, 130, 4, 2, 64, 32, (411, 130), None),
    (1, 2, 150, 2, 2, 80, 128, (40,), (170, 129)),
    (4, 2, 3, 2, 1, 256, 256, (517, 1, 256, 300), None),
    (1, 3, 5, 2, 1, 8, 16, (90,), (4, 2, 0)),                    # queries before the first own token see the prefix alone
]


@pytest.mark.parametrize("tiles", ["-1", "0", "1"])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("groups,members,lq,h,hkv,d,block,prefix,own", SHAPES)
def test_prefix(nhip_env, groups, members, lq, h, hkv, d, block, prefix, own, causal, dtype, tiles):
    nhip_env.setenv("NHIP_ATTN_TILES", tiles)
    b = groups * members
    own = own or tuple(lq + (i * 37) % 150 for i in range(b))
    pp, po = max(1, -(-max(prefix) // block)), max(1, -(-max(own) // block))
    cache = filled(groups * pp + b * po + 3, hkv, d, block, seed=d)
    order = torch.randperm(groups * pp + b * po + 3, generator=torch.Generator().manual_seed(2)).int().cuda()
    check(cache, randn(7, (b, lq, h, d), dtype).cuda(), order[:groups * pp].view(groups, pp), prefix,
          order[groups * pp:groups * pp + b * po].view(b, po), own, causal)


@pytest.mark.parametrize("workers", ["3", "29"])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_dealt(nhip_env, dtype, workers):
    """Work of many rows dealt to so many workgroups: parts that begin and end inside row tiles."""
    nhip_env.setenv("NHIP_ATTN_TILES", "1")
    nhip_env.setenv("NHIP_ATTN_WORKERS", workers)
    cache = filled(40, 2, 64, 32)
    order = torch.randperm(40, generator=torch.Generator().manual_seed(1)).int().cuda()
    check(cache, randn(3, (6, 60, 4, 64), dtype).cuda(), order[:20].view(2, 10), (320, 250), order[20:38].view(6, 3),
          (90, 60, 70, 96, 61, 80), True)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("tiles", ["0", "1"])
def test_limits_and_missing_pages(nhip_env, dtype, tiles):
    nhip_env.setenv("NHIP_ATTN_TILES", tiles)
    cache = filled(9, 2, 64, 16)
    cache.v_scale[3] = 0
    cache.k_scale[4] = 0
    cache.k_scale[8] = float("nan")  # of a page that no row sees
    shared, table = ints([[0, 1, -1, 2], [3, 4, 99, 8]]), ints([[5], [-1], [6], [7]])
    q = randn(8, (4, 2, 4, 64), dtype).cuda()
    lengths = (16, 3, -4, 9)
    got = check(cache, q, shared, (60, 48), table, lengths, False)
    assert torch.equal(got, check(cache, q, shared, (64, 48), table, lengths, False, max_prefix=60))
    check(cache, q, shared, (30, 20), table, (500, 16, 2, 1), True, max_length=10, scale=-0.3)
    none = ints([[-1], [-1], [-1], [-1]])
    assert (check(cache, q, ints([[-1], [-1]]), (16, 16), none, (16, 16, 16, 16), False) == 0).all()
    # without pages on one side or both
    empty_p, empty_o = ints([[], []]).view(2, 0), ints([]).view(4, 0)
    check(cache, q, empty_p, (5, 5), table, lengths, False)
    check(cache, q, shared, (60, 48), empty_o, (5, 5, 5, 5), False)
    assert (cache.prefix_attention(q, empty_p, ints([1, 1]), empty_o, ints([1, 1, 1, 1])) == 0).all()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_scales_apart(dtype):
    """Value scales of the prefix and the own pages differ by powers that a 16-bit probability times them would not hold."""
    cache = filled(6, 1, 64, 16)
    cache.k_scale.fill_(0.01)
    cache.v_scale[:, 0] = torch.tensor([1e-7, 3e-5, 1e-6, 1e-7, 1e-2, 1e-9])
    for lq in (1, 140):
        q = randn(9, (2, lq, 2, 64), dtype).cuda()
        check(cache, q, ints([[0, 1]]), (31,), ints([[4], [2]]), (16, 5), False)
        check(cache, q, ints([[4, 3]]), (32,), ints([[5], [0]]), (3, 16), False)


def test_as_one_sequence():
    """What the attention over the same pages in one table gives, to the roundings of either."""
    cache = filled(30, 2, 128, 16, seed=3)
    table = torch.arange(30, dtype=torch.int32, device="cuda").view(1, 30)
    q = randn(4, (5, 1, 8, 128), F32).cuda()
    rows = torch.cat([table[:, :24].expand(5, 24), table[0, 24:29].view(5, 1)], 1).contiguous()
    a = cache.prefix_attention(q, table[:, :24].contiguous(), ints([384]), rows[:, 24:].contiguous(), ints([16] * 5), causal=True)
    b = cache.attention(q, rows, ints([400] * 5), causal=True)
    assert (a - b).abs().max() <= 1e-5 * b.abs().max()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("lq", [1, 3, 130])
def test_query_strides(dtype, lq):
    """Queries of a larger tensor: any distance between sequences, tokens and heads that keeps 16 bytes."""
    cache = filled(20, 2, 64, 16)
    shared, table = torch.arange(6, dtype=torch.int32, device="cuda").view(2, 3), torch.arange(8, 20, dtype=torch.int32, device="cuda").view(6, 2)
    wide = randn(5, (6, lq + 2, 3, 4, 80), dtype).cuda()
    lengths = (32, 9, 20, 1, 17, 31)
    for q in (wide[:, 1:1 + lq, 1, :, 8:72], wide[:, 1:1 + lq, 1, :, 8:72].flip(0), wide.transpose(2, 3)[:, :lq, :, 2, :64],
              wide[:1, :lq, 0, :, :64].expand(6, lq, 4, 64)):
        q = q if all(s >= 0 for s in q.stride()) else q.contiguous()
        got = check(cache, q, shared, (48, 30), table, lengths, True)
        assert torch.equal(got, cache.prefix_attention(q.contiguous(), shared, ints([48, 30]), table, ints(lengths), causal=True))


def test_pool_past_32_bits():
    pages, hkv, d, block = 20000, 8, 128, 128  # 2.6 GB of codes each
    cache, small = nhip.KvCache8(pages, hkv, d, block), nhip.KvCache8(5, hkv, d, block)
    k, v = randn(1, (1, 500, hkv, d), F16).cuda(), randn(2, (1, 500, hkv, d), F16).cuda()
    far, near = ints([[pages - 1, 3, pages - 2, 19000]]), ints([[2, 0, 1, 4]])
    cache.append(k, v, far, ints([0]))
    small.append(k, v, near, ints([0]))
    for members, lq in ((2, 1), (2, 150)):
        q = randn(3, (members, lq, hkv, d), F16).cuda()
        a, b = (c.prefix_attention(q, t[:, :2].contiguous(), ints([256]), t[:, 2:].reshape(2, 1).contiguous(), ints([128, 60]))
                for c, t in ((cache, far), (small, near)))
        assert torch.equal(a, b)


def test_streams_graphs_and_bits():
    """Bit for bit again, on another stream, and in two graphs with a workspace of their own."""
    cache = filled(60, 2, 128, 64)
    shared, table = torch.arange(40, dtype=torch.int32, device="cuda").view(2, 20), torch.arange(40, 56, dtype=torch.int32, device="cuda").view(16, 1)
    np_, no = ints([1280, 999]), ints([64 - i for i in range(16)])
    qs = [randn(20 + i, (16, 1, 8, 128), BF16).cuda() for i in range(4)]

    def call(q, **kw):
        return cache.prefix_attention(q, shared, np_, table, no, causal=True, **kw)

    want = [call(q) for q in qs]
    assert all(torch.equal(call(q), w) for q, w in zip(qs, want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = call(qs[0], stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want[0])
    held, graphs = [], []
    for i in range(2):
        q, out, graph = qs[i].clone(), torch.zeros_like(want[0]), torch.cuda.CUDAGraph()
        ws = torch.empty(1 << 24, dtype=torch.uint8, device="cuda")
        with torch.cuda.graph(graph):
            call(q, out=out, workspace=ws)
        held.append((q, out, ws))
        graphs.append(graph)
    for r in range(4):
        for i in range(2):
            held[i][0].copy_(qs[(r + i) % 4])
            graphs[i].replay()
            assert torch.equal(call(qs[3]), want[3])
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(held[i][1], want[(r + i) % 4])


def test_limits_past_32_bits():
    """Limits that 32 bits do not hold are refused, not taken for what is left of them."""
    cache = filled(8, 2, 64, 16)
    q, shared, table = randn(1, (4, 1, 4, 64)).cuda(), ints([[0, 1], [2, 3]]), ints([[4], [5], [6], [7]])
    for name in ("max_prefix", "max_length"):
        for v in (2 ** 31, 2 ** 32 + 1, -2 ** 32 + 5):
            with pytest.raises(ValueError):
                cache.prefix_attention(q, shared, ints([30, 30]), table, ints([1, 2, 3, 4]), **{name: v})
    for v in (2 ** 31, 2 ** 32 + 1, -2 ** 32 + 5):
        with pytest.raises(ValueError):
            cache.attention(q, table, ints([1, 2, 3, 4]), max_length=v)


def test_refusals():
    cache = filled(8, 2, 64, 16)
    q, shared, table = torch.zeros((4, 1, 4, 64), device="cuda"), ints([[0, 1], [2, 3]]), ints([[4], [5], [6], [7]])
    np_, no = ints([30, 30]), ints([1, 2, 3, 4])
    for bad in (lambda: cache.prefix_attention(q[:3], shared, np_, table[:3], no[:3]),
                lambda: cache.prefix_attention(q, shared, no, table, no), lambda: cache.prefix_attention(q, shared, np_, table[:2], no),
                lambda: cache.prefix_attention(q, shared.long(), np_, table, no), lambda: cache.prefix_attention(q, shared, np_, table, np_),
                lambda: cache.prefix_attention(q[..., :32], shared, np_, table, no),
                lambda: cache.prefix_attention(q, shared[:0], np_[:0], table, no),
                lambda: cache.prefix_attention(q, shared, np_, table, no, out=torch.zeros((4, 1, 4, 64), dtype=F16, device="cuda")),
                lambda: cache.prefix_attention(q, shared, np_, table, no, workspace=torch.empty(1 << 20, dtype=torch.uint8))):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: cache.prefix_attention(q[:, :, :3], shared, np_, table, no),
                lambda: cache.prefix_attention(q, shared, np_, table, no, workspace=torch.empty(16, dtype=torch.uint8, device="cuda")),
                lambda: cache.prefix_attention(q, shared, np_, table, no, max_prefix=-1)):
        with pytest.raises(nhip.NhipError):
            bad()
    with pytest.raises(TypeError):
        cache.prefix_attention(q.double(), shared, np_, table, no)
    assert cache.prefix_attention(q[:0], shared, np_, table[:0], no[:0]).shape == (0, 1, 4, 64)
