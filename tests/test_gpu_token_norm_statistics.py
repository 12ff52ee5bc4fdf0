"""Group norm where its statistics can go wrong, in every form of the kernel
(NHIP_NORM_ONE=0 / 1 / 2) and both layouts, against the formula in 64 bits
(tests/token_reference.py, which derives the bounds)."""
import pytest

torch = pytest.importorskip("torch")

import nhip  # noqa: E402
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
