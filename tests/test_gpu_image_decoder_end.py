"""The image decoder example at the end of its cache: refused, nothing changed."""
import pytest

torch = pytest.importorskip("torch")

import image_decoder  # noqa: E402
import nhip  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("max_tokens", [100, 112])  # inside a page, at its end
def test_cache_is_full(max_tokens):
    nhip.init(0)
    m = image_decoder.ImageDecoder(seed=1, max_tokens=max_tokens)
    tokens, extent = m.features(torch.rand((2, 3, 52, 36), device="cuda"))
    with pytest.raises(ValueError):  # 117 tokens
        m.prompt(tokens, extent)
    assert not m.cache.k.any() and not hasattr(m, "held")
    tokens, (h, w) = m.features(torch.rand((2, 3, 44, 36), device="cuda"))
    x = m.prompt(tokens, (h, w))[:, -1:].contiguous()
    lengths = torch.full((2,), h * w, dtype=torch.int32, device="cuda")
    for _ in range(max_tokens - h * w):
        x = m.step(x, lengths)
        x = x / x.norm() * 8
    was = [t.clone() for t in (m.cache.k, m.cache.v, m.cache.k_scale, m.cache.v_scale)]
    with pytest.raises(ValueError):
        m.step(x, lengths)
    assert m.held == max_tokens
    assert all(torch.equal(a, b) for a, b in zip(was, (m.cache.k, m.cache.v, m.cache.k_scale, m.cache.v_scale)))
