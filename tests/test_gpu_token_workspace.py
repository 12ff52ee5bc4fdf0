"""Workspaces that the token operators refuse: a pointer that the kernels could
not write never reaches them."""
import pytest

torch = pytest.importorskip("torch")

import nhip  # noqa: E402

pytestmark = pytest.mark.gpu


def bad(nbytes):
    return [torch.empty(nbytes, dtype=torch.uint8),                             # host memory
            torch.empty((nbytes, 2), dtype=torch.uint8, device="cuda")[:, 0]]  # half of the bytes that its size says


def test_refused(nhip_env):
    nhip.init(0)
    nhip_env.setenv("NHIP_NORM_ONE", "0")
    x = torch.randn((1, 3000, 64), device="cuda")
    norm = nhip.GroupNorm(8, 64)
    q, k = torch.randn((1, 1, 8, 64), device="cuda"), torch.randn((1, 4000, 2, 64), device="cuda")
    cache = nhip.KvCache8(64, 2, 64, 64)
    table = torch.arange(64, dtype=torch.int32, device="cuda").view(1, 64)
    lengths = torch.tensor([4000], dtype=torch.int32, device="cuda")
    for ws in bad(1 << 20):
        for call in (lambda: norm.forward(x, workspace=ws), lambda: nhip.cross_attention(q, k, k, workspace=ws),
                     lambda: cache.attention(q, table, lengths, workspace=ws)):
            with pytest.raises(ValueError):
                call()
    ws = torch.empty(1 << 20, dtype=torch.float32, device="cuda")  # any type will do
    assert torch.equal(norm.forward(x, workspace=ws), norm.forward(x))
