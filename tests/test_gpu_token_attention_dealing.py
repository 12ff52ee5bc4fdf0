"""Attention of many rows at sizes where the library deals the work by itself
(fewer workgroups than row tiles, more, and three to a CU over the cache), against
the same with a row tile to a workgroup."""
import pytest

torch = pytest.importorskip("torch")

import nhip  # noqa: E402
import token_reference as ref  # noqa: E402

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def agree(call, magnitudes, row_tiles, nhip_env):
    """Both sides lie within 3 roundings to the type of the weighted magnitudes, and one of the result, of the exact
    value (probabilities and result rounded; scores' and sums' errors in 32 bits stay below a third of that here)."""
    got = call()
    nhip_env.setenv("NHIP_ATTN_WORKERS", str(row_tiles))
    want = call()
    unit = ref.UNIT[got.dtype]
    bound = 2 * unit * (3 * magnitudes().float() + want.float().abs())
    assert ((got.float() - want.float()).abs() <= bound).all()
    assert not torch.equal(got, want)  # (sums in another order: the work was dealt)


@pytest.mark.parametrize("b,lq,lk,h,hkv,d", [(2, 3136, 6272, 16, 4, 128),   # 784 row tiles
                                             (4, 784, 3136, 12, 12, 64)])  # 336
def test_cross(b, lq, lk, h, hkv, d, nhip_env):
    nhip.init(0)
    g = torch.Generator(device="cuda").manual_seed(1)
    q, k, v = (torch.randn(s, generator=g, device="cuda").to(BF16) for s in ((b, lq, h, d), (b, lk, hkv, d), (b, lk, hkv, d)))
    lengths = torch.tensor([lk - 1000 * i for i in range(b)], dtype=torch.int32, device="cuda")
    tiles = b * hkv * -(-lq * (h // hkv) // 128)
    agree(lambda: nhip.cross_attention(q, k, v, lengths), lambda: nhip.cross_attention(q, k, v.abs(), lengths), tiles, nhip_env)


def test_cached(nhip_env):
    nhip.init(0)
    b, lq, n, h, hkv, d, block = 2, 509, 6272, 16, 4, 64, 32
    g = torch.Generator(device="cuda").manual_seed(2)
    cache = nhip.KvCache8(b * n // block, hkv, d, block)
    table = torch.randperm(b * n // block, generator=g, device="cuda").int().view(b, -1)
    q = torch.randn((b, lq, h, d), generator=g, device="cuda").to(F16)
    k, v = (torch.randn((b, n, hkv, d), generator=g, device="cuda").to(F16) for _ in range(2))
    cache.append(k, v, table, torch.zeros((b,), dtype=torch.int32, device="cuda"))
    lengths = torch.tensor([n, n - 1700], dtype=torch.int32, device="cuda")

    def magnitudes():
        both = nhip.KvCache8.of(cache.k, cache.v.abs(), cache.k_scale, cache.v_scale)
        return both.attention(q, table, lengths, causal=True)

    agree(lambda: cache.attention(q, table, lengths, causal=True), magnitudes, b * hkv * -(-lq * (h // hkv) // 128), nhip_env)
