"""Group norm where its statistics can go wrong, in every form of the kernel
(NHIP_NORM_ONE=0 / 1 / 2) and both layouts, against the formula in 64 bits
(tests/token_reference.py, which derives the bounds)."""
import pytest

torch = pytest.importorskip("torch")

import nhip  # noqa: E402
import token_reference as ref  # noqa: E402
from test_gpu_token_norm_rotary import check_norm, randn  # noqa: E402

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
ACTS = {"none": nhip.ACT_NONE, "relu": nhip.ACT_RELU, "silu": nhip.ACT_SILU}
FORMS = pytest.mark.parametrize("one", ["0", "1", "2"])  # (blobs have no third form: as "0")
LAYOUTS = pytest.mark.parametrize("blobs", [False, True])


@pytest.fixture(autouse=True)
def _form(one, nhip_env):
    assert torch.cuda.is_available(), "GPU tests need a HIP device"
    nhip.init(0)
    nhip_env.setenv("NHIP_NORM_ONE", one)


def laid(x, blobs):
    """x [n, pixels, c] as the layout has it, on the GPU."""
    return (x.transpose(1, 2).contiguous() if blobs else x).cuda()


@FORMS
@LAYOUTS
@pytest.mark.parametrize("act", ["none", "relu", "silu"])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("value", ["inf", "-inf", "nan"])
@pytest.mark.parametrize("pixel", [0, 7, 301])
def test_not_finite(pixel, value, dtype, act, blobs, one):
    """The mean of a group that holds it is infinite or NaN: NaN throughout that group, and no other."""
    x = randn(1, (3, 302, 32), dtype)
    x[1, pixel, 9] = float(value)
    y = nhip.GroupNorm(4, 32, act=ACTS[act], blobs=blobs).forward(laid(x, blobs))
    assert torch.isnan(y[1, :, 8:16]).all()
    y[1, :, 8:16] = 0
    assert torch.isfinite(y).all()


@FORMS
@LAYOUTS
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("whole", [True, False])  # every channel of the first pixel, or each group's first value alone
@pytest.mark.parametrize("spreads", [30, 1000])
@pytest.mark.parametrize("n,pixels,c,groups", [(2, 900, 64, 8), (1, 6001, 40, 4), (1, 20000, 16, 1)])
def test_first_value_far_off(n, pixels, c, groups, spreads, whole, dtype, blobs, one):
    """A corner or a first token unlike the rest: sums taken from it have to keep the others' digits."""
    x = randn(pixels, (n, pixels, c), dtype)
    x[:, 0, ::1 if whole else c // groups] += spreads
    check_norm(laid(x, blobs), groups, "none", blobs)


@FORMS
@LAYOUTS
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("factor", [1e25, 1e-25])
def test_squares_out_of_range(factor, dtype, blobs, one):
    """Values whose squares fp32 would not hold."""
    x = (randn(2, (2, 700, 32)) * factor).to(dtype)
    check_norm(laid(x, blobs), 4, "none", blobs, eps=0.0)


@FORMS
@LAYOUTS
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_one_value_of_many(dtype, blobs, one):
    """All values alike but one, by the type's last place."""
    x = torch.full((1, 3000, 16), 96.0, dtype=dtype)
    x[0, 1700, 5] += 96.0 * {F32: 2.0 ** -22, F16: 2.0 ** -9, BF16: 2.0 ** -6}[dtype]
    check_norm(laid(x, blobs), 1, "none", blobs, eps=0.0)


@FORMS
@LAYOUTS
@pytest.mark.parametrize("dtype", [F32, F16])
def test_many_images(dtype, blobs, one):
    """More images than fill the GPU: a thread sums many values."""
    n, pixels, c = 600, 5000, 16
    x = torch.randn((n, pixels, c), generator=torch.Generator(device="cuda").manual_seed(3), device="cuda").to(dtype) + 3
    y = nhip.GroupNorm(2, c, blobs=blobs).forward(laid(x, blobs))
    for i in (0, 333, n - 1):
        want, bound = ref.group_norm(x[i:i + 1], 2, None, None, 1e-5, "none")
        ref.assert_within(y[i:i + 1], want, bound)
