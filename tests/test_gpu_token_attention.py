"""Cross attention and the 8-bit cache (append, read, attention) on the GPU,
through the C ABI, against their formulas in 64 bits (tests/token_reference.py,
which derives the bounds); codes and scales bit for bit."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import nhip  # noqa: E402
import token_reference as ref  # noqa: E402

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
NAN, INF = float("nan"), float("inf")


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    assert torch.cuda.is_available(), "GPU tests need a HIP device"
    nhip.init(0)


def randn(seed, shape, dtype=F32):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g).to(dtype)


def ints(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def keeps(b, lq, lk, lengths=None, mask=None):
    keep = torch.ones((b, lq, lk), dtype=torch.bool)
    if lengths is not None:
        keep &= torch.arange(lk) < torch.as_tensor(lengths)[:, None, None]
    if mask is not None:
        keep &= mask.cpu().expand(b, lk)[:, None]
    return keep


def check_cross(q, k, v, lengths=None, mask=None, scale=None, **kw):
    b, lq, h, d = q.shape
    got = nhip.cross_attention(q, k, v, None if lengths is None else ints(*lengths), mask, scale=scale, **kw)
    want, bound = ref.attention(q, k, v, keeps(b, lq, k.shape[1], lengths, mask), d ** -0.5 if scale is None else scale)
    ref.assert_within(got, want, bound, f"{tuple(q.shape)} x {tuple(k.shape)} {q.dtype}")
    return got


def qkv(b, lq, lk, h, hkv, d, dtype, seed=0):
    return (randn(seed + 1, (b, lq, h, d), dtype).cuda(), randn(seed + 2, (b, lk, hkv, d), dtype).cuda(),
            randn(seed + 3, (b, lk, hkv, d), dtype).cuda())


SHAPES = [
    # b, lq, lk, heads, kv_heads, d, lengths
    (1, 1, 1, 1, 1, 64, None),              # one token, one key
    (3, 1, 700, 8, 2, 128, (700, 0, 333)),  # a step over ragged lengths, one of them empty
    (2, 1, 5000, 4, 1, 64, (5000, 1)),      # a step over a long sequence: split
    (1, 1, 130, 32, 1, 96, None),           # more rows to a key head than a tile
    (2, 17, 33, 6, 3, 40, (33, 32)),        # channels that are no multiple of 32
    (2, 77, 64, 4, 4, 80, (0, 64)),
    (1, 130, 257, 2, 1, 128, (255,)),       # ends inside every tile
    (1, 300, 1000, 3, 3, 64, None),
    (2, 257, 129, 4, 2, 128, (129, 100)),
    (1, 190, 500, 2, 2, 256, (499,)),
    (1, 70, 300, 1, 1, 200, None),
    (1, 600, 97, 5, 1, 32, (96,)),
    (4, 2, 3, 2, 1, 8, (3, 2, 1, 0)),
]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("b,lq,lk,h,hkv,d,lengths", SHAPES)
def test_cross_attention(b, lq, lk, h, hkv, d, lengths, dtype):
    check_cross(*qkv(b, lq, lk, h, hkv, d, dtype), lengths)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("lq,d", [(1, 128), (150, 64), (150, 128), (9, 33), (140, 33)])
def test_masked_places_hold_anything(lq, d, dtype):
    """NaN and infinities under the mask and past the lengths; rows without a key."""
    b, lk = 4, 203
    q, k, v = qkv(b, lq, lk, 4, 2, d, dtype)
    g = torch.Generator().manual_seed(9)
    mask = torch.rand((b, lk), generator=g) < 0.6
    mask[2] = False
    mask[3, :64] = False
    lengths = (203, 150, 203, 131)
    out = ~keeps(b, 1, lk, lengths, mask)[:, 0]
    at = out.cuda()
    k[at] = NAN
    v[at] = INF
    v[1, 160:] = NAN
    got = check_cross(q, k, v, lengths, mask.cuda())
    assert (got[2] == 0).all()
    # one mask for the batch
    q, k, v = qkv(b, lq, lk, 4, 2, d, dtype)
    check_cross(q, k, v, None, mask[0].cuda())


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("lq", [1, 200])
def test_values_that_count_spread(dtype, lq):
    """NaN and infinite keys and values that are not masked reach the rows that see them, and no other batch."""
    q, k, v = qkv(3, lq, 150, 2, 1, 64, dtype)
    v[0, 77, 0, 5] = NAN
    k[1, 20, 0, 3] = NAN
    got = nhip.cross_attention(q, k, v)
    assert torch.isnan(got[0, ..., 5]).all() and not torch.isnan(got[0, ..., 6:]).any()
    assert torch.isnan(got[1]).all() and not torch.isnan(got[2]).any()
    # every score -infinity: 0 / 0, not a row without keys
    q = torch.ones((1, lq, 1, 64), dtype=dtype, device="cuda")
    k = torch.zeros((1, 50, 1, 64), dtype=dtype, device="cuda")
    k[..., 0] = -INF
    assert torch.isnan(nhip.cross_attention(q, k, torch.ones_like(k))).all()
    # some of them: those keys weigh nothing
    k[:, 10:, :, 0] = 0
    v = randn(4, (1, 50, 1, 64), dtype).cuda()
    want, bound = ref.attention(q, k[:, 10:], v[:, 10:], keeps(1, lq, 40), 0.125)
    ref.assert_within(nhip.cross_attention(q, k, v, scale=0.125), want, bound)


@pytest.mark.parametrize("scale", [0.0, -0.2, 3.0])
@pytest.mark.parametrize("lq", [1, 180])
def test_scales(scale, lq):
    check_cross(*qkv(2, lq, 190, 2, 2, 64, F32), scale=scale)
    check_cross(*qkv(2, lq, 190, 2, 2, 64, BF16), scale=scale)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_scores_that_grow(dtype):
    """The running maximum rises at every tile, by more than any power the sums could hold without it."""
    lk, d = 700, 64
    q = torch.full((1, 150, 1, d), 4.0).to(dtype).cuda()
    k = (torch.arange(lk).float() / 8).view(1, lk, 1, 1).expand(1, lk, 1, d).to(dtype).contiguous().cuda()
    v = randn(5, (1, lk, 1, d), dtype).cuda()
    check_cross(q, k, v)
    check_cross(q, k.flip(1), v)
    check_cross(q[:, :1], k, v)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("lq", [1, 144])
def test_cross_strides_and_alignment(dtype, lq):
    q, k, v = qkv(2, lq, 140, 4, 2, 64, dtype)
    want = check_cross(q, k, v)
    heads_first = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]
    assert torch.equal(nhip.cross_attention(*heads_first), want)
    both = torch.cat([k, v], -1)                     # keys and values side by side
    assert torch.equal(nhip.cross_attention(q, both[..., :64], both[..., 64:]), want)
    odd = [torch.nn.functional.pad(t, (1, 2))[..., 1:65] for t in (q, k, v)]  # rows at odd addresses
    check_cross(*odd)
    check_cross(q, k[:1].expand(2, 140, 2, 64), v[:1].expand(2, 140, 2, 64))  # one encoder for the batch


def test_cross_no_keys_no_rows():
    q, k, v = qkv(2, 5, 0, 4, 2, 64, F16)
    assert (nhip.cross_attention(q, k, v) == 0).all()
    q, k, v = qkv(2, 0, 5, 4, 2, 64, F16)
    assert nhip.cross_attention(q, k, v).shape == (2, 0, 4, 64)
    q, k, v = qkv(0, 5, 5, 4, 2, 64, F16)
    assert nhip.cross_attention(q, k, v).shape == (0, 5, 4, 64)


@pytest.mark.parametrize("lq", [1, 160])
def test_cross_offsets_past_32_bits(lq):
    """Key rows 2^22 elements apart: the last lies past 2^32 elements."""
    lk, step = 1100, 1 << 22
    pool = torch.empty(((lk - 1) * step + 64,), dtype=F16, device="cuda")
    k = pool.as_strided((1, lk, 1, 64), (0, step, 64, 1))
    q, small, v = qkv(1, lq, lk, 2, 1, 64, F16)
    k.copy_(small)
    check_cross(q, k, v)
    assert torch.equal(nhip.cross_attention(q, k, v), nhip.cross_attention(q, small, v))


def test_cross_repeats_bit_for_bit_and_takes_a_workspace():
    q, k, v = qkv(2, 1, 4000, 8, 2, 128, BF16)
    want = nhip.cross_attention(q, k, v)
    ws = torch.empty(64 << 20, dtype=torch.uint8, device="cuda").fill_(255)
    out = torch.empty_like(q)
    assert nhip.cross_attention(q, k, v, out=out, workspace=ws) is out
    assert torch.equal(out, want)
    with pytest.raises(nhip.NhipError) as e:
        nhip.cross_attention(q, k, v, workspace=ws[:64])
    assert e.value.status == 5


# ------------------------------------------------------------------ the cache
def check_append(cache, k, v, table, starts, counts=None):
    n = k.shape[1]
    want = [ref.append(c, s, x, table, starts, [n] * len(starts) if counts is None else counts, cache.block_tokens)
            for c, s, x in ((cache.k, cache.k_scale, k), (cache.v, cache.v_scale, v))]
    cache.append(k, v, table, ints(*starts), None if counts is None else ints(*counts))
    for (codes, scales), c, s in zip(want, (cache.k, cache.v), (cache.k_scale, cache.v_scale)):
        np.testing.assert_array_equal(s.cpu().numpy(), scales)
        np.testing.assert_array_equal(c.cpu().numpy(), codes)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("block,d", [(16, 64), (32, 40), (64, 128), (128, 8), (256, 256)])
def test_append(block, d, dtype):
    """A prompt, then single tokens that grow: begun pages are requantised."""
    b, pages = 3, 6
    cache = nhip.KvCache8(b * pages, 2, d, block)
    table = torch.randperm(b * pages, generator=torch.Generator().manual_seed(1)).int().view(b, pages).cuda()
    n = 2 * block + 5
    starts = [0, 3, block]
    check_append(cache, randn(1, (b, n, 2, d), dtype).cuda(), randn(2, (b, n, 2, d), dtype).cuda(), table, starts)
    for i in range(4):
        at = [s + n + i for s in starts]
        new = randn(10 + i, (b, 1, 2, d), dtype) * (0.5 * 3 ** i)
        check_append(cache, new.cuda(), (new * 0.7).cuda(), table, at)
    # the same tokens again change nothing
    was = [t.clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
    cache.append(new.cuda(), (new * 0.7).to(dtype).cuda(), table, ints(*at))
    assert torch.equal(cache.k, was[0]) and torch.equal(cache.k_scale, was[2])


def test_append_counts_tables_and_odd_values():
    d, block = 64, 16
    cache = nhip.KvCache8(8, 3, d, block)
    cache.k.random_(-127, 128)
    cache.k_scale.fill_(0.01)
    table = ints(0, 1, 2, 3, -1, 99, 4, 5).view(4, 2)[:, :2].contiguous()
    k, v = randn(1, (4, 20, 3, d)), randn(2, (4, 20, 3, d))
    k[0, 0, 0, :3] = torch.tensor([NAN, INF, -INF])
    k[1, :, 1] = 0
    v[0, :, 2] = NAN
    v[3, 2, 0] = 1e-44
    v[3, :, 1] = torch.tensor(1e-43)
    check_append(cache, k.cuda(), v.cuda(), table, [4, 0, 0, 9], [20, 7, 20, 30])  # 30: more than there are
    check_append(cache, k.cuda(), v.cuda(), table, [-1, 25, 31, 40], [20, 0, -3, 20])
    wide = randn(3, (4, 20, 3, 2 * d + 1)).cuda()
    check_append(cache, wide[..., :d], wide[..., d + 1:], table, [1, 2, 3, 4])


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_read(dtype):
    cache = nhip.KvCache8(6, 2, 40, 32)
    for t in (cache.k, cache.v):
        t.random_(-127, 128)
    cache.k_scale.copy_(torch.rand((6, 2)))
    cache.v_scale.copy_(torch.rand((6, 2)) * 1e-3)
    table = ints(5, 2, 0, 7, 1, -1).view(2, 3)
    k, v = cache.read(table, ints(-5, 30), 80, dtype)
    for got, codes, scales in ((k, cache.k, cache.k_scale), (v, cache.v, cache.v_scale)):
        codes, scales = codes.cpu().float(), scales.cpu()
        for b in range(2):
            for i in range(80):
                t = (-5, 30)[b] + i
                page = int(table[b, t // 32]) if 0 <= t < 96 else -1
                want = (codes[page, :, t % 32] * scales[page, :, None]).to(dtype) if 0 <= page < 6 else torch.zeros((2, 40), dtype=dtype)
                assert torch.equal(got[b, i].cpu(), want), (b, i)


def filled(pages, hkv, d, block, seed=0):
    """A cache of random codes; scales of pages spread over a factor of 30."""
    cache = nhip.KvCache8(pages, hkv, d, block)
    g = torch.Generator().manual_seed(seed)
    for codes, scales in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        codes.copy_(torch.randint(-127, 128, codes.shape, generator=g, dtype=torch.int8))
        scales.copy_(torch.exp(torch.randn(scales.shape, generator=g)) * 0.015)
    return cache


def check_cached(cache, q, table, lengths, causal, scale=None, max_length=None, **kw):
    b, lq, h, d = q.shape
    got = cache.attention(q, table, ints(*lengths), max_length=max_length, causal=causal, scale=scale, **kw)
    lk = table.shape[1] * cache.block_tokens
    ids = table.cpu().long()
    there = (ids >= 0) & (ids < cache.k.shape[0])
    ids = torch.where(there, ids, 0)
    k, v = ((codes.cpu().double() * scales.cpu().double()[:, :, None, None])[ids].transpose(2, 3).reshape(b, lk, cache.kv_heads, d)
            for codes, scales in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))
    n = torch.as_tensor(lengths).clamp(0, lk if max_length is None else max_length)[:, None]
    last = n - lq + 1 + torch.arange(lq) if causal else n.expand(b, lq)
    t = torch.arange(lk)
    keep = (t < torch.minimum(last, n)[..., None]) & there.repeat_interleave(cache.block_tokens, 1)[:, None]
    want, bound = ref.attention(q.cpu(), k, v, keep, d ** -0.5 if scale is None else scale, q.dtype)
    ref.assert_within(got, want, bound, f"{tuple(q.shape)} {cache.block_tokens} {q.dtype} {causal}")
    return got


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("b,lq,h,hkv,d,block,lengths", [
    (1, 1, 1, 1, 64, 16, (1,)),
    (3, 1, 8, 2, 128, 64, (700, 0, 333)),
    (2, 1, 4, 4, 96, 32, (3000, 65)),
    (2, 3, 16, 1, 40, 16, (100, 2)),          # rows before the sequence's first token: they see nothing
    (2, 130, 4, 2, 64, 32, (130, 411)),
    (1, 257, 2, 1, 128, 128, (300,)),
    (2, 150, 3, 3, 80, 16, (40, 170)),
    (1, 100, 2, 2, 256, 256, (517,)),
    (1, 140, 1, 1, 8, 64, (200,)),
])
def test_cached_attention(b, lq, h, hkv, d, block, lengths, causal, dtype):
    pages = max(1, -(-max(lengths) // block))
    cache = filled(b * pages + 3, hkv, d, block, seed=d)
    table = torch.randperm(b * pages + 3, generator=torch.Generator().manual_seed(2))[:b * pages].int().view(b, pages).cuda()
    check_cached(cache, randn(7, (b, lq, h, d), dtype).cuda(), table, lengths, causal)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("lq", [1, 140])
def test_cached_attention_missing_pages_and_limits(lq, dtype):
    cache = filled(9, 2, 64, 16)
    cache.v_scale[3] = 0
    cache.k_scale[4] = 0
    table = ints(0, 1, -1, 2, 3, 4, 5, 1000, 8, -7).view(2, 5)
    q = randn(8, (2, lq, 4, 64), dtype).cuda()
    check_cached(cache, q, table, (80, 77), False)
    check_cached(cache, q, table, (500, -3), False)             # past the table; negative
    check_cached(cache, q, table, (80, 77), False, max_length=50)
    check_cached(cache, q, table, (80, 80), True, scale=-0.3)
    assert (check_cached(cache, q, torch.full_like(table, -1), (80, 80), False) == 0).all()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("lq", [1, 140])
def test_cached_attention_small_and_large_scales(dtype, lq):
    """Pages whose value scales differ by powers that a 16-bit probability times them would not hold."""
    cache = filled(6, 1, 64, 16)
    cache.k_scale.fill_(0.01)
    cache.v_scale[:, 0] = torch.tensor([1e-7, 3e-5, 1e-6, 1e-7, 1e-2, 1e-9])
    q = randn(9, (1, lq, 2, 64), dtype).cuda()
    check_cached(cache, q, ints(0, 1, 2).view(1, 3), (41,), False)
    check_cached(cache, q, ints(5, 4, 3).view(1, 3), (48,), False)


def test_cached_attention_pool_past_32_bits():
    pages, hkv, d, block = 20000, 8, 128, 128  # 2.6 GB of codes each
    cache = nhip.KvCache8(pages, hkv, d, block)
    table = ints(pages - 1, 3, pages - 2).view(1, 3)
    k, v = randn(1, (1, 300, hkv, d), F16).cuda(), randn(2, (1, 300, hkv, d), F16).cuda()
    cache.append(k, v, table, ints(0))
    small = nhip.KvCache8(3, hkv, d, block)
    small.append(k, v, ints(2, 0, 1).view(1, 3), ints(0))
    assert torch.equal(cache.read(table, ints(0), 300, F16)[0], small.read(ints(2, 0, 1).view(1, 3), ints(0), 300, F16)[0])
    for lq in (1, 150):
        q = randn(3, (1, lq, hkv, d), F16).cuda()
        assert torch.equal(cache.attention(q, table, ints(300)), small.attention(q, ints(2, 0, 1).view(1, 3), ints(300)))


# -------------------------------------------------- streams, graphs, refusals
def test_side_stream_and_graph():
    q, k, v = qkv(2, 1, 900, 8, 2, 64, F16)
    cache = nhip.KvCache8(32, 2, 64, 64)
    table = torch.arange(32, dtype=torch.int32, device="cuda").view(2, 16)
    starts, lengths = ints(0, 0), ints(900, 900)

    def step(stream=None):
        cache.append(k, v, table, starts, stream=stream)
        return (nhip.cross_attention(q, k, v, stream=stream), cache.attention(q, table, lengths, causal=True, stream=stream),
                *cache.read(table, starts, 900, F16, stream=stream))

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = step(side)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(3):
        for t in (q, k, v):
            t.copy_(randn(40 + i, t.shape, F16))
        expect = [t.clone() for t in step()]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, expect))


def test_wrapper_refusals():
    q, k, v = qkv(2, 3, 5, 4, 2, 64, F16)
    for args in ((q.cpu(), k, v), (q, k.float(), v), (q.int(), k.int(), v.int())):
        with pytest.raises(TypeError):
            nhip.cross_attention(*args)
    for args in ((q, k[:1], v), (q, k, v[:, :4]), (q, k[..., :32], v[..., :32]),
                 (q, k, v.transpose(2, 3).contiguous().transpose(2, 3))):
        with pytest.raises(ValueError):
            nhip.cross_attention(*args)
    with pytest.raises(ValueError):
        nhip.cross_attention(q, k, v, key_lengths=ints(5))
    with pytest.raises(ValueError):
        nhip.cross_attention(q, k, v, key_lengths=torch.tensor([5, 5], device="cuda"))
    with pytest.raises(ValueError):
        nhip.cross_attention(q, k, v, key_mask=torch.ones((2, 5), device="cuda"))
    with pytest.raises(ValueError):
        nhip.cross_attention(q, k, v, key_mask=torch.ones((2, 4), dtype=torch.bool, device="cuda"))
    with pytest.raises(ValueError):
        nhip.cross_attention(q, k, v, out=torch.empty((2, 3, 4, 32), dtype=F16, device="cuda"))
    with pytest.raises(nhip.NhipError):
        nhip.cross_attention(q[:, :, :3], k, v)
    cache = nhip.KvCache8(2, 2, 64, 16)
    table = ints(0, 1).view(2, 1)
    with pytest.raises(ValueError):
        cache.append(k, v, table.long(), ints(0, 0))
    with pytest.raises(ValueError):
        cache.append(k[..., :32], v[..., :32], table, ints(0, 0))
    with pytest.raises(ValueError):
        cache.attention(q[..., :32], table, ints(1, 1))
    with pytest.raises(nhip.NhipError):
        cache.attention(torch.zeros((2, 3, 4, 65), dtype=F16, device="cuda")[..., 1:], table, ints(1, 1))
    with pytest.raises(ValueError):
        nhip.KvCache8.of(cache.k, cache.v[:1], cache.k_scale, cache.v_scale)
    with pytest.raises(nhip.NhipError):
        nhip.KvCache8(2, 2, 64, 24).attention(q, table, ints(1, 1))
