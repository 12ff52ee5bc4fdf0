"""Both attention kernels (few rows, many rows) on the same cases, whichever
of them the library would take: NHIP_ATTN_TILES=0 / 1."""
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
    nhip.init(0)
    nhip_env.setenv("NHIP_ATTN_TILES", tiles)


@FORMS
@TYPES
@pytest.mark.parametrize("b,lq,lk,h,hkv,d,lengths", base.SHAPES + [
    (1, 128, 64, 1, 1, 64, None),        # one whole tile
    (1, 33, 3000, 2, 1, 128, (2999,)),   # parts joined over many workgroups
    (40, 150, 70, 4, 2, 64, None),       # more row tiles than places, a run of them to a worker
    (300, 3, 5, 2, 2, 40, None),
    (1, 1, 40, 3, 1, 256, (17,)),
])
def test_cross(tiles, b, lq, lk, h, hkv, d, lengths, dtype):
    base.check_cross(*base.qkv(b, lq, lk, h, hkv, d, dtype), lengths)


@FORMS
@TYPES
@pytest.mark.parametrize("lq,d", [(1, 128), (150, 64), (150, 128), (30, 200)])
def test_masked_places(tiles, lq, d, dtype):
    base.test_masked_places_hold_anything(lq, d, dtype)


@FORMS
@TYPES
@pytest.mark.parametrize("lq", [1, 200])
def test_values_that_count(tiles, lq, dtype):
    base.test_values_that_count_spread(dtype, lq)


@FORMS
@TYPES
@pytest.mark.parametrize("lq", [1, 200])
def test_infinite_values_that_count(tiles, lq, dtype):
    """An infinite value reaches every row that gives it weight, in its channel alone."""
    q, k, v = base.qkv(2, lq, 150, 2, 1, 64, dtype)
    v[0, 77, 0, 5] = base.INF
    v[1, 3, 0, 9] = -base.INF
    got = nhip.cross_attention(q, k, v).float()
    assert (got[0, ..., 5] == base.INF).all() and (got[1, ..., 9] == -base.INF).all()
    got[0, ..., 5] = 0
    got[1, ..., 9] = 0
    assert torch.isfinite(got).all()


@FORMS
@pytest.mark.parametrize("lq", [1, 200])
def test_small_and_large_numbers(tiles, lq):
    """fp32 values far from 1: tiny keys and values, near the largest, and both in one sequence."""
    for kf, vf in ((1e-30, 1.0), (1.0, 1e-36), (1.0, 1e37), (1e-38, 1e-38)):
        q, k, v = base.qkv(1, lq, 130, 2, 1, 64, F32)
        base.check_cross(q, k * kf, v * vf)
        base.check_cross(q * 1e-20, k * 1e20, v * vf)
        v[:, 5] *= vf
        base.check_cross(q, k, v)


@FORMS
@pytest.mark.parametrize("lq", [1, 180])
@pytest.mark.parametrize("scale", [0.0, -0.2, 3.0])
def test_scales(tiles, scale, lq):
    base.test_scales(scale, lq)


@FORMS
@TYPES
def test_scores_that_grow(tiles, dtype):
    base.test_scores_that_grow(dtype)


@FORMS
@TYPES
@pytest.mark.parametrize("lq", [1, 144])
def test_strides(tiles, lq, dtype):
    base.test_cross_strides_and_alignment(dtype, lq)


@FORMS
def test_no_keys_no_rows(tiles):
    base.test_cross_no_keys_no_rows()


@FORMS
@pytest.mark.parametrize("lq", [1, 160])
def test_offsets_past_32_bits(tiles, lq):
    base.test_cross_offsets_past_32_bits(lq)


@FORMS
@TYPES
def test_rows_too_far_apart_for_a_tile(tiles, dtype):
    """Key rows 2^25 bytes apart, past what the kernels reach with 31 bits: the general form."""
    step, lk = (1 << 25) // torch.empty((), dtype=dtype).element_size(), 70
    pool = torch.empty(((lk - 1) * step + 64,), dtype=dtype, device="cuda")
    k = pool.as_strided((1, lk, 1, 64), (0, step, 64, 1))
    q, small, v = base.qkv(1, 20, lk, 2, 1, 64, dtype)
    k.copy_(small)
    base.check_cross(q, k, v)


@FORMS
@TYPES
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("b,lq,h,hkv,d,block,lengths", [
    (3, 1, 8, 2, 128, 64, (700, 0, 333)), (2, 3, 16, 1, 40, 16, (100, 2)), (2, 130, 4, 2, 64, 32, (130, 411)),
    (1, 257, 2, 1, 128, 128, (300,)), (2, 150, 3, 3, 80, 16, (40, 170)), (1, 100, 2, 2, 256, 256, (517,)),
    (1, 140, 1, 1, 8, 64, (200,)), (30, 70, 6, 3, 64, 32, tuple(range(10, 310, 10))),
])
def test_cached(tiles, b, lq, h, hkv, d, block, lengths, causal, dtype):
    base.test_cached_attention(b, lq, h, hkv, d, block, lengths, causal, dtype)


@FORMS
@TYPES
@pytest.mark.parametrize("lq", [1, 140])
def test_cached_limits_and_scales(tiles, lq, dtype):
    base.test_cached_attention_missing_pages_and_limits(lq, dtype)
    base.test_cached_attention_small_and_large_scales(dtype, lq)


@FORMS
def test_pool_past_32_bits(tiles):
    base.test_cached_attention_pool_past_32_bits()


@FORMS
def test_repeats_and_streams(tiles):
    base.test_side_stream_and_graph()
    q, k, v = base.qkv(2, 70, 900, 8, 2, 128, BF16)
    want = nhip.cross_attention(q, k, v)
    for _ in range(3):
        assert torch.equal(nhip.cross_attention(q, k, v), want)
