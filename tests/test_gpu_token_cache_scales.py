"""Attention over the 8-bit cache where pages' scales are not numbers: in pages
that no row reaches, and in pages that rows see."""
import pytest

torch = pytest.importorskip("torch")

import nhip  # noqa: E402
import test_gpu_token_attention as base  # noqa: E402

pytestmark = pytest.mark.gpu
F32, F16, BF16 = base.F32, base.F16, base.BF16
FORMS = pytest.mark.parametrize("tiles", ["0", "1"])
TYPES = pytest.mark.parametrize("dtype", [F32, F16, BF16])


@pytest.fixture(autouse=True)
def _form(tiles, nhip_env):
    assert torch.cuda.is_available(), "GPU tests need a HIP device"
    nhip.init(0)
    nhip_env.setenv("NHIP_ATTN_TILES", tiles)


# sequences that end in the first page of a tile of 32 or 64 keys, at a page's end, in its middle, before the first token
@FORMS
@TYPES
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lq,d", [(1, 64), (3, 40), (140, 64), (140, 128), (90, 256)])
@pytest.mark.parametrize("block,lengths", [(16, (5, 16, 0, 70, 97)), (32, (20, 32, 64, 65, 160))])
def test_pages_not_reached(block, lengths, lq, d, causal, dtype, tiles):
    """Pages of the table past a sequence's length, as a pool that was never cleared leaves them."""
    b, pages = len(lengths), 192 // block
    cache = base.filled(b * pages, 2, d, block, seed=d)
    table = torch.arange(b * pages, dtype=torch.int32).view(b, pages)
    odd = torch.tensor([base.NAN, base.INF, -base.INF])
    for i, n in enumerate(lengths):
        for j, page in enumerate(table[i, -(-n // block):].tolist()):
            cache.k_scale[page] = odd[j % 3]
            cache.v_scale[page] = odd[(j + 1) % 3]
    base.check_cached(cache, base.randn(7, (b, lq, 4, d), dtype).cuda(), table.cuda(), lengths, causal)
