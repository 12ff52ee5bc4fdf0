"""Appends to the 8-bit cache by workgroups of every width, with infinities and
NaN among the tokens, bit for bit against the CPU's (tests/token_reference.py)."""
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


def ints(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


# a wave; pages of up to 1024, 2048 and more vectors; vectors that are read again; single elements (unaligned tokens)
@pytest.mark.parametrize("tokens,block,d,dtype,gap", [
    (5, 16, 64, F32, 0), (50, 16, 64, BF16, 0), (150, 64, 128, F16, 0), (150, 64, 128, F32, 0), (300, 128, 128, BF16, 0),
    (300, 256, 64, F32, 0), (600, 256, 256, BF16, 0), (600, 256, 256, F32, 0), (40, 16, 40, F16, 1), (150, 64, 128, BF16, 3)])
def test_append_of_infinities(tokens, block, d, dtype, gap):
    b, heads = 2, 2
    pages = -(-(tokens + 2 * block) // block)
    cache = nhip.KvCache8(b * pages, heads, d, block)
    table = torch.randperm(b * pages, generator=torch.Generator().manual_seed(1)).int().view(b, pages).cuda()
    g = torch.Generator().manual_seed(tokens + d)
    k, v = (torch.randn((b, tokens, heads, d + gap), generator=g).to(dtype)[..., gap:] for _ in range(2))
    k[0, tokens // 2, 0, d // 3] = INF      # one, deep inside
    k[1, tokens - 1, 1, d - 1] = -INF       # the very last
    k[0, :, 1] = INF                        # nothing else
    v[0, 0, 0, 0], v[0, 1, 0, 0] = NAN, INF  # both
    v[1, :, 1] = NAN
    starts = [3, block + 1]
    for scale in (1, 4):  # the second time the pages are begun, and grow
        x, y = k * scale, v * scale
        at = [s + (scale - 1) * 5 for s in starts]
        want = [ref.append(c, s, z, table, at, [tokens] * b, block)
                for c, s, z in ((cache.k, cache.k_scale, x), (cache.v, cache.v_scale, y))]
        wide = [torch.zeros((b, tokens, heads, d + gap), dtype=dtype) for _ in range(2)]
        for w, z in zip(wide, (x, y)):
            w[..., gap:] = z
        xs, ys = (w.cuda()[..., gap:] for w in wide)
        cache.append(xs, ys, table, ints(*at))
        for (codes, scales), c, s in zip(want, (cache.k, cache.v), (cache.k_scale, cache.v_scale)):
            np.testing.assert_array_equal(s.cpu().numpy(), scales)
            np.testing.assert_array_equal(c.cpu().numpy(), codes)
