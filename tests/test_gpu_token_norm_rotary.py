"""Group norm into tokens and rotary positions on the GPU, through the C ABI,
against their formulas in 64 bits (tests/token_reference.py, which derives
the bounds)."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import nhip  # noqa: E402
import token_reference as ref  # noqa: E402

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
ACTS = {"none": nhip.ACT_NONE, "relu": nhip.ACT_RELU, "silu": nhip.ACT_SILU}


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    assert torch.cuda.is_available(), "GPU tests need a HIP device"
    nhip.init(0)


def randn(seed, shape, dtype=F32):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g).to(dtype)


def affine(c):
    return 1 + 0.3 * randn(1, (c,)).numpy(), randn(2, (c,)).numpy()


def check_norm(x, groups, act="silu", blobs=False, eps=1e-5, gb=True, **kw):
    c = x.shape[1] if blobs else x.shape[-1]
    gamma, beta = affine(c) if gb else (None, None)
    norm = nhip.GroupNorm(groups, c, gamma, beta, eps=eps, act=ACTS[act], blobs=blobs)
    got = norm.forward(x, **kw)
    tokens = x.reshape(x.shape[0], c, -1).transpose(1, 2) if blobs else x.reshape(x.shape[0], -1, c)
    want, bound = ref.group_norm(tokens, groups, gamma, beta, eps, act)
    ref.assert_within(got.reshape(want.shape), want, bound, f"{tuple(x.shape)} {x.dtype} {act}")
    return got


# one pixel; odd pixels; more channels than a workgroup's columns; one channel to a group; one group; a group over
# several columns' worth; channels that are no whole vector; many chunks of an image
SHAPES = [(1, 1, 32, 4), (2, 7, 33, 3), (1, 784, 128, 32), (3, 57, 320, 32), (2, 5, 4096, 1), (1, 9, 2568, 8),
          (2, 64, 40, 40), (1, 3001, 24, 1), (1, 70000, 16, 2), (5, 130, 65, 65)]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("n,pixels,c,groups", SHAPES)
@pytest.mark.parametrize("blobs", [False, True])
def test_group_norm(n, pixels, c, groups, dtype, blobs):
    x = randn(n + pixels, (n, c, pixels) if blobs else (n, pixels, c), dtype) * 2 + 0.5
    check_norm(x.cuda(), groups, "silu", blobs)


@pytest.mark.parametrize("one", ["0", "1"])
@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("blobs", [False, True])
@pytest.mark.parametrize("n,pixels,c,groups", [(2, 9, 24, 3), (1, 1500, 96, 32), (3, 333, 20, 20), (2, 4097, 64, 1)])
def test_group_norm_one_and_two_launches(n, pixels, c, groups, blobs, dtype, one, nhip_env):
    nhip_env.setenv("NHIP_NORM_ONE", one)
    x = randn(21, (n, c, pixels) if blobs else (n, pixels, c), dtype)
    check_norm(x.cuda(), groups, "silu", blobs)


@pytest.mark.parametrize("act", ["none", "relu"])
@pytest.mark.parametrize("blobs", [False, True])
def test_group_norm_activation_and_no_affine(act, blobs):
    x = randn(3, (2, 48, 15, 13) if blobs else (2, 15, 13, 48), F32).cuda()
    y = check_norm(x, 6, act, blobs, gb=False)
    assert tuple(y.shape) == ((2, 195, 48) if blobs else (2, 15, 13, 48))


@pytest.mark.parametrize("blobs", [False, True])
@pytest.mark.parametrize("pixels", [6, 5000])
def test_group_norm_large_mean(blobs, pixels):
    """A mean of a thousand spreads: E[x^2] - E[x]^2 in fp32 would leave nothing of the variance."""
    x = randn(4, (2, 32, pixels), F32) + 1000.0
    check_norm((x if blobs else x.transpose(1, 2).contiguous()).cuda(), 4, "none", blobs)


def test_group_norm_constant_channels():
    x = torch.full((1, 50, 8), 3.25, device="cuda")
    gamma, beta = affine(8)
    y = nhip.GroupNorm(2, 8, gamma, beta).forward(x)
    assert torch.equal(y.cpu(), torch.from_numpy(beta).float().expand(1, 50, 8))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_group_norm_strides_and_alignment(dtype):
    wide = randn(5, (3, 40, 96), dtype).cuda()
    check_norm(wide[:, :, 16:80], 8)           # aligned slice of wider pixels
    check_norm(wide[:, :, 3:43], 8)            # unaligned slice
    check_norm(wide[:, ::2, :64], 8)           # every second pixel
    check_norm(wide[1:2].expand(2, 40, 96), 8)  # the same image twice
    planes = randn(6, (2, 12, 50), dtype).cuda()
    check_norm(planes[:, :, 1:44], 4, blobs=True)
    check_norm(planes[:, ::3], 2, blobs=True)


def test_group_norm_in_place_and_given_workspace():
    x = randn(7, (2, 3301, 64), F16).cuda()  # large enough for a workspace
    norm = nhip.GroupNorm(8, 64)
    want = norm.forward(x)
    ws = torch.empty(norm.workspace_size(nhip.DTYPE_F16, 2, 3301), dtype=torch.uint8, device="cuda")
    y = x.clone()
    assert norm.forward(y, out=y, workspace=ws) is y
    assert torch.equal(y, want)
    with pytest.raises(nhip.NhipError) as e:
        norm.forward(x, workspace=ws[:-8])
    assert e.value.status == 5


def test_group_norm_empty_and_nan():
    norm = nhip.GroupNorm(4, 16)
    assert norm.forward(torch.empty((0, 5, 16), device="cuda")).shape == (0, 5, 16)
    assert norm.forward(torch.empty((2, 0, 16), device="cuda")).shape == (2, 0, 16)
    x = randn(8, (2, 20, 16), F32)
    x[1, 3, 5] = float("nan")
    y = norm.forward(x.cuda()).cpu()
    assert torch.isnan(y[1, :, 4:8]).all() and torch.isnan(y).sum() == 80  # that image's group and no other


# ------------------------------------------------------------------ rotary
def positions(seed, b, n, axes, lo=0, hi=300):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(lo, hi, (b, n, axes), generator=g, dtype=torch.int32)


def check_rotary(x, pos, sections, neighbours, inverse=False, **kw):
    freq = np.concatenate([10000.0 ** (-np.arange(s) / max(s, 1)) for s in sections]).astype(np.float32)
    rot = nhip.Rotary(x.shape[-1], sections, inv_freq=freq, neighbours=neighbours)
    want, bound = ref.rotary(x, pos, sections, freq, neighbours, inverse)
    got = rot.forward(x, pos.cuda(), inverse=inverse, **kw)
    ref.assert_within(got, want, bound, f"{tuple(x.shape)} {x.dtype} {sections} {neighbours}")
    return got


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("neighbours", [False, True])
@pytest.mark.parametrize("b,n,h,d,sections", [
    (2, 1, 16, 128, (16, 24, 24)),   # one token
    (1, 65, 3, 64, (8, 8)),          # half of the head, two axes
    (2, 33, 5, 40, (5, 7, 3)),       # no whole vectors
    (1, 7, 1, 34, (17,)),            # odd pairs
    (3, 300, 12, 80, (0, 20, 20)),   # an axis without pairs
    (1, 4000, 9, 96, (12, 12, 12, 12)),
])
def test_rotary(b, n, h, d, sections, neighbours, dtype):
    check_rotary(randn(n, (b, n, h, d), dtype).cuda(), positions(n, b, n, len(sections)), sections, neighbours)


@pytest.mark.parametrize("neighbours", [False, True])
def test_rotary_any_position(neighbours):
    """Angles stay exact at every int32 position, negative ones too."""
    pos = positions(9, 2, 50, 2, -2 ** 31, 2 ** 31 - 1)
    pos[0, :4, 0] = torch.tensor([2 ** 31 - 1, -2 ** 31, -1, 0])
    check_rotary(randn(10, (2, 50, 2, 32), F32).cuda(), pos, (8, 8), neighbours)


@pytest.mark.parametrize("neighbours", [False, True])
def test_rotary_strides_in_place_inverse(neighbours):
    sections = (4, 6, 6)
    x = randn(11, (2, 3, 21, 48), BF16).cuda().transpose(1, 2)    # stored [b, h, n, d]
    pos = positions(12, 1, 21, 3)                                 # one for the batch
    check_rotary(x, pos, sections, neighbours)
    check_rotary(randn(13, (2, 21, 3, 50), F32).cuda()[..., 1:49], pos, sections, neighbours)  # unaligned
    y = randn(14, (2, 21, 3, 48), F32).cuda()
    was = y.clone()
    rot = nhip.Rotary(48, sections, neighbours=neighbours)
    turned = rot.forward(y, pos.cuda())
    assert rot.forward(y, pos.cuda(), out=y) is y and torch.equal(y, turned)
    rot.forward(y, pos.cuda(), inverse=True, out=y)
    assert (y - was).abs().max() < 16 * ref.E * was.abs().max() * 2
    check_rotary(was, pos, sections, neighbours, inverse=True)


def test_rotary_empty():
    rot = nhip.Rotary(32, (8, 8))
    for b, n, h in ((0, 3, 2), (2, 0, 2), (2, 3, 0)):
        x = torch.empty((b, n, h, 32), device="cuda")
        assert rot.forward(x, torch.empty((b, n, 2), dtype=torch.int32, device="cuda")).shape == x.shape


def test_rotary_offsets_past_32_bits():
    """Tokens 2^27 elements apart: the last lies past 2^32 elements."""
    n, step = 34, 1 << 27
    pool = torch.empty(((n - 1) * step + 64,), dtype=F16, device="cuda")
    x = pool.as_strided((1, n, 1, 64), (0, step, 64, 1))
    x.copy_(randn(15, (1, n, 1, 64), F16))
    check_rotary(x, positions(16, 1, n, 1), (32,), False)


# -------------------------------------------------- streams, graphs, refusals
def test_side_stream_and_graph():
    x = randn(17, (2, 500, 64), F16).cuda()
    tok = x.view(2, 500, 2, 32)
    pos = positions(18, 1, 500, 2).cuda()
    norm, rot = nhip.GroupNorm(8, 64, act=nhip.ACT_SILU), nhip.Rotary(32, (8, 8))
    want = rot.forward(norm.forward(x).view_as(tok), pos)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = rot.forward(norm.forward(x, stream=side).view_as(tok), pos, stream=side)
    side.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = rot.forward(norm.forward(x).view_as(tok), pos)
    for i in range(3):
        x.copy_(randn(20 + i, x.shape, F16))
        expect = rot.forward(norm.forward(x).view_as(tok), pos)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, expect)


def test_wrapper_refusals():
    norm, rot = nhip.GroupNorm(4, 16), nhip.Rotary(16, (4, 4))
    x = torch.zeros((2, 3, 16), device="cuda")
    for bad, error in ((x.cpu(), TypeError), (x.double(), TypeError), (x[..., :8], ValueError),
                       (torch.zeros((2, 16, 3), device="cuda").transpose(1, 2), ValueError)):
        with pytest.raises(error):
            norm.forward(bad)
    with pytest.raises(ValueError):
        norm.forward(x, out=torch.zeros((2, 3, 15), device="cuda"))
    with pytest.raises(nhip.NhipError):  # rows that overlap
        norm.forward(torch.zeros((1, 1, 16), device="cuda").expand(2, 3, 16))
    t, p = torch.zeros((2, 3, 1, 16), device="cuda"), torch.zeros((2, 3, 2), dtype=torch.int32, device="cuda")
    for bad in (p.long(), p[:, :2], p[..., :1], p.cpu()):
        with pytest.raises(ValueError):
            rot.forward(t, bad)
    with pytest.raises(nhip.NhipError):  # an output whose tokens overlap
        rot.forward(t, p, out=torch.zeros((2, 1, 1, 16), device="cuda").expand(2, 3, 1, 16))


# ------------------------------------------------- past the last-level cache
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_group_norm_past_the_cache(dtype):
    n, pixels, c = 36, 6007, 256 if dtype == BF16 else 128
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn((n, pixels, c), generator=g, device="cuda").to(dtype)
    gamma, beta = affine(c)
    y = nhip.GroupNorm(16, c, gamma, beta, act=nhip.ACT_RELU).forward(x)
    for i in (0, 17, 35):
        want, bound = ref.group_norm(x[i:i + 1], 16, gamma, beta, 1e-5, "relu")
        ref.assert_within(y[i:i + 1], want, bound)


@pytest.mark.parametrize("neighbours", [False, True])
def test_rotary_past_the_cache(neighbours):
    n = 80001
    x = torch.randn((1, n, 8, 128), generator=torch.Generator(device="cuda").manual_seed(4), device="cuda", dtype=F16)
    pos = positions(5, 1, n, 2).cuda()
    rot = nhip.Rotary(128, (20, 20), neighbours=neighbours)
    y = rot.forward(x, pos)
    for a, b in ((0, 777), (40000, 40100), (n - 5, n)):
        assert torch.equal(y[:, a:b], rot.forward(x[:, a:b], pos[:, a:b].contiguous()))
