"""Attention of many rows with its work dealt to a given number of workgroups
(NHIP_ATTN_WORKERS): runs inside a row tile, runs that end one and begin the
next, runs with whole row tiles and parts of two others, one run of everything."""
import pytest

torch = pytest.importorskip("torch")

import nhip  # noqa: E402
import test_gpu_token_attention as base  # noqa: E402

pytestmark = pytest.mark.gpu
F32, F16, BF16 = base.F32, base.F16, base.BF16
WORKERS = pytest.mark.parametrize("workers", [1, 3, 5, 7, 13, 29, 64, 100000])
TYPES = pytest.mark.parametrize("dtype", [F32, F16, BF16])


@pytest.fixture(autouse=True)
def _dealt(workers, nhip_env):
    assert torch.cuda.is_available(), "GPU tests need a HIP device"
    nhip.init(0)
    nhip_env.setenv("NHIP_ATTN_TILES", "1")
    nhip_env.setenv("NHIP_ATTN_WORKERS", str(workers))


@WORKERS
@TYPES
@pytest.mark.parametrize("b,lq,lk,h,hkv,d,lengths", [
    (2, 390, 300, 2, 1, 64, (300, 130)),         # 14 row tiles of 5 units: workers with whole tiles and two partial ends
    (3, 200, 700, 4, 2, 128, (700, 0, 65)),      # one sequence without a key, one far shorter
    (1, 130, 257, 2, 2, 256, (255,)),
    (5, 20, 3, 2, 2, 40, None),                  # one unit to a row tile
])
def test_cross(b, lq, lk, h, hkv, d, lengths, dtype, workers):
    base.check_cross(*base.qkv(b, lq, lk, h, hkv, d, dtype), lengths)


@WORKERS
@TYPES
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("b,lq,h,hkv,d,block,lengths", [
    (2, 390, 2, 1, 64, 16, (390, 500)), (2, 130, 4, 2, 128, 64, (130, 411)), (3, 260, 1, 1, 80, 32, (300, 0, 40)),
    (1, 300, 1, 1, 256, 64, (300,)),
])
def test_cached(b, lq, h, hkv, d, block, lengths, causal, dtype, workers):
    base.test_cached_attention(b, lq, h, hkv, d, block, lengths, causal, dtype)


@WORKERS
@TYPES
def test_masked_places_and_values_that_spread(dtype, workers):
    base.test_masked_places_hold_anything(150, 64, dtype)
    base.test_values_that_count_spread(dtype, 200)


@WORKERS
def test_values_that_pieces_do_not_hold(workers):
    """fp32 tiles on the fp32 instructions in some workers' runs only."""
    q, k, v = base.qkv(2, 260, 500, 2, 2, 64, F32)
    k[:, 70:75] *= 1e-36
    v[1, 300:310] *= 1e30
    base.check_cross(q, k, v)


@WORKERS
def test_graph_and_repeats(workers):
    base.test_side_stream_and_graph()
    q, k, v = base.qkv(2, 300, 900, 4, 2, 128, BF16)
    want = nhip.cross_attention(q, k, v)
    assert all(torch.equal(nhip.cross_attention(q, k, v), want) for _ in range(3))
