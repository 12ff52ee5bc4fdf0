"""The image decoder example against the same model in 64 bits on the CPU:
trunk, group norm, projections, rotary positions, the 8-bit cache's arithmetic
and both attentions."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import image_decoder  # noqa: E402
import nhip  # noqa: E402
import numerics  # noqa: E402
import token_reference as ref  # noqa: E402

pytestmark = pytest.mark.gpu


class Reference:
    """image_decoder.ImageDecoder's arithmetic in 64 bits, codes included."""

    def __init__(self, m):
        self.m = m
        self.codes = [(c.cpu(), s.cpu()) for c, s in ((m.cache.k, m.cache.k_scale), (m.cache.v, m.cache.v_scale))]

    def features(self, images):
        x = images.cpu().numpy()
        for w, b, _ in self.m.trunk:
            x = np.maximum(numerics.conv_f64(x, w, b, stride=(2, 2)), 0)
        t = torch.from_numpy(x).flatten(2).transpose(1, 2)
        return ref.group_norm(t.float(), 8, self.m.gamma, self.m.beta, 1e-5, "silu")[0]

    def project(self, block, i, x, heads):
        return (x @ torch.from_numpy(block.weights[i]).double().t()).view(*x.shape[:2], heads, block.head_dim)

    def own(self, x, positions, start, causal):
        m, b, n = self.m, x.shape[0], x.shape[1]
        q, k, v = (self.project(m.own, i, x, h) for i, h in ((0, m.own.heads), (1, m.own.kv_heads), (2, m.own.kv_heads)))
        freq = np.concatenate([10000.0 ** (-np.arange(s) / s) for s in m.sections])
        q, k = (ref.rotary(t.float(), positions, m.sections, freq, False)[0] for t in (q, k))
        self.codes = [tuple(map(torch.from_numpy, ref.append(c, s, t.float(), m.table, [start] * b, [n] * b, m.cache.block_tokens)))
                      for (c, s), t in zip(self.codes, (k, v))]
        ids = m.table.cpu().long()
        kk, vv = ((c.double() * s.double()[:, :, None, None])[ids].transpose(2, 3).flatten(1, 2) for c, s in self.codes)
        t = torch.arange(kk.shape[1])
        last = start + n - n + 1 + torch.arange(n) if causal else torch.full((n,), start + n)
        keep = (t < last[:, None]).expand(b, n, len(t))
        o = ref.attention(q, kk, vv, keep, m.own.head_dim ** -0.5, torch.float32)[0]
        return x + o.flatten(2) @ torch.from_numpy(m.own.weights[3]).double().t()

    def cross(self, x, tokens, lengths):
        c = self.m.cross
        q, k, v = self.project(c, 0, x, c.heads), self.project(c, 1, tokens, c.kv_heads), self.project(c, 2, tokens, c.kv_heads)
        keep = (torch.arange(tokens.shape[1]) < torch.as_tensor(lengths)[:, None])[:, None]
        o = ref.attention(q, k, v, keep, c.head_dim ** -0.5, torch.float32)[0]
        return x + o.flatten(2) @ torch.from_numpy(c.weights[3]).double().t()


def test_image_decoder_matches_its_formulas():
    """fp32 layers differ from 64 bits by about 1e-6; a value on the edge of two codes may then take the other, a step
    of a 254th of its page's range in one of many: 1e-3 of the norm holds both."""
    nhip.init(0)
    m = image_decoder.ImageDecoder(seed=3)
    r = Reference(m)
    images = torch.rand((2, 3, 44, 36), generator=torch.Generator().manual_seed(1)) * 2 - 1
    tokens, (h, w) = m.features(images.cuda())
    want_tokens = r.features(images)
    assert numerics.max_rel_err(tokens.cpu(), want_tokens) < 1e-4
    grid = torch.stack(torch.meshgrid(torch.arange(1), torch.arange(h), torch.arange(w), indexing="ij"), -1).view(1, -1, 3).int()
    got, want = m.prompt(tokens, (h, w)), r.own(want_tokens, grid, 0, False)
    assert numerics.max_rel_err(got.cpu(), want) < 1e-3
    lengths = [h * w, h * w - 31]
    x, wx = got[:, -1:].contiguous(), want[:, -1:]
    for i in range(20):  # past a page's end
        x = m.step(x, torch.tensor(lengths, dtype=torch.int32, device="cuda"))
        at = torch.full((1, 1, 3), h * w + i, dtype=torch.int32)
        wx = r.cross(r.own(wx, at, h * w + i, True), want_tokens, lengths)
        assert numerics.max_rel_err(x.cpu(), wx) < 1e-3 * (i + 1), i
        x, wx = x / x.norm() * 8, wx / wx.norm() * 8
