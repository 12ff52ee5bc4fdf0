"""Group norm whose workgroups hold their groups' values in registers, on the
GPU, against the formula in 64 bits (tests/token_reference.py, which derives
the bounds)."""
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


def check_norm(x, groups, act="silu", **kw):
    c = x.shape[-1]
    gamma, beta = 1 + 0.3 * randn(1, (c,)).numpy(), randn(2, (c,)).numpy()
    got = nhip.GroupNorm(groups, c, gamma, beta, act=ACTS[act]).forward(x, **kw)
    want, bound = ref.group_norm(x, groups, gamma, beta, 1e-5, act)
    ref.assert_within(got, want, bound, f"{tuple(x.shape)} {x.dtype} {act}")
    return got


# one pixel; fewer pixels than a workgroup's rows; rows of 64, 80, 96 and 128 bytes; a last vector that few threads
# have; one group; one channel to a group; the most pixels that 256, 512 and 1024 threads hold of 64 bytes, and one more
SHAPES = [(1, 1, 64, 8), (3, 5, 64, 8), (2, 57, 320, 32), (2, 1023, 80, 2), (3, 784, 128, 32), (5, 197, 256, 1),
          (2, 333, 40, 40), (1, 1024, 32, 4), (2, 1025, 32, 4), (1, 2048, 32, 2), (1, 2049, 32, 1), (1, 4096, 32, 4),
          (1, 4097, 32, 4), (9, 49, 1024, 32), (2, 100, 4096, 2)]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("n,pixels,c,groups", SHAPES)
def test_held(n, pixels, c, groups, dtype, nhip_env):
    nhip_env.setenv("NHIP_NORM_ONE", "2")
    check_norm((randn(n + pixels, (n, pixels, c), dtype) * 2 + 0.5).cuda(), groups)


@pytest.mark.parametrize("act", ["none", "relu"])
@pytest.mark.parametrize("dtype", [F32, F16])
def test_held_large_mean_and_activation(act, dtype, nhip_env):
    nhip_env.setenv("NHIP_NORM_ONE", "2")
    x = randn(4, (2, 1500, 64), dtype)
    check_norm((x + (1000.0 if dtype is F32 else 20.0)).cuda(), 4, act)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_held_strides(dtype, nhip_env):
    nhip_env.setenv("NHIP_NORM_ONE", "2")
    wide = randn(5, (3, 90, 96), dtype).cuda()
    check_norm(wide[:, :, 16:80], 8)            # aligned slice of wider pixels
    check_norm(wide[:, :, 3:67], 8)             # unaligned: two launches
    check_norm(wide[:, ::2, :64], 8)            # every second pixel
    check_norm(wide[1:2].expand(2, 90, 96), 8)  # the same image twice


def test_held_in_place_and_nan(nhip_env):
    nhip_env.setenv("NHIP_NORM_ONE", "2")
    x = randn(7, (4, 700, 64), F16).cuda()
    want = check_norm(x, 8)
    y = x.clone()
    check = nhip.GroupNorm(8, 64, 1 + 0.3 * randn(1, (64,)).numpy(), randn(2, (64,)).numpy(), act=nhip.ACT_SILU)
    assert check.forward(y, out=y) is y
    assert torch.equal(y, want)
    x[1, 3, 5] = float("nan")
    z = check.forward(x)
    assert torch.isnan(z[1, :, :8]).all() and torch.isnan(z).sum() == 700 * 8  # that image's group and no other


@pytest.mark.parametrize("n,pixels,c,groups,dtype", [(200, 784, 256, 32, BF16), (26, 3136, 256, 32, F16),
                                                     (40, 1024, 640, 32, BF16), (30, 1568, 384, 16, F32)])
def test_held_as_two_launches(n, pixels, c, groups, dtype, nhip_env):
    """Large tensors (some past the caches), by the library's own choice: as by two launches, to a rounding."""
    x = randn(9, (n, pixels, c)).cuda().to(dtype)
    norm = nhip.GroupNorm(groups, c, act=nhip.ACT_SILU)
    got = norm.forward(x)
    nhip_env.setenv("NHIP_NORM_ONE", "0")
    want = norm.forward(x)
    unit = {F32: 2.0 ** -20, F16: 2.0 ** -10, BF16: 2.0 ** -7}[dtype]  # fp32: a few roundings; else the result's
    assert ((got.float() - want.float()).abs() <= unit * want.float().abs() + 2.0 ** -20).all()
