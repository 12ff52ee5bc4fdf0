"""A decoder that reads images: the layers of a convolutional trunk, and the
token operators behind them, as a program runs them.

  features  3x3 convolutions (stride 2) -> group norm + SiLU, straight from the
            blobs into channels-last tokens
  prompt    the image's tokens, one block: rotary positions (time, row,
            column), keys and values into the 8-bit cache, attention over it
  step      one token a sequence: the same block causally, then cross attention
            to the image's features (unquantised), of the length that each
            image has

Weights are random: this shows the calls, their order and the buffers a program
keeps (`python image_decoder.py` runs it and prints what it did).
"""
from __future__ import annotations

import numpy as np

import nhip
import workloads


class Block:
    """Projections of one attention: query, key, value, output."""

    def __init__(self, rng, dim, heads, kv_heads, head_dim):
        self.heads, self.kv_heads, self.head_dim = heads, kv_heads, head_dim
        self.weights = [(rng.standard_normal(s) / np.sqrt(s[1])).astype(np.float32) for s in (
            (heads * head_dim, dim), (kv_heads * head_dim, dim), (kv_heads * head_dim, dim), (dim, heads * head_dim))]
        self.q, self.k, self.v, self.o = (nhip.InnerProductF32(w) for w in self.weights)

    def project(self, layer, x, heads):
        """x [batch, tokens, dim] -> [batch, tokens, heads, head_dim]."""
        return layer.forward(x.reshape(-1, x.shape[-1])).view(*x.shape[:2], heads, self.head_dim)

    def out(self, x, attended):
        """x + the projected heads."""
        return nhip.add(x, self.o.forward(attended.reshape(-1, self.heads * self.head_dim)).view_as(x))


class ImageDecoder:
    def __init__(self, seed=0, channels=(32, 64), heads=4, kv_heads=2, head_dim=32, block_tokens=16, batch=2,
                 max_tokens=256, device="cuda"):
        import torch
        self.torch, self.device = torch, device
        rng = np.random.default_rng(seed)
        dim = channels[-1]
        self.trunk, c = [], 3
        for k in channels:
            w = workloads.he_normal(rng, (k, c, 3, 3), c * 9)
            b = (rng.standard_normal(k) * 0.05).astype(np.float32)
            self.trunk.append((w, b, nhip.Conv2dF32(nhip.conv_desc(c, k, stride=(2, 2), act=nhip.ACT_RELU), w, b)))
            c = k
        self.gamma = (1 + 0.1 * rng.standard_normal(dim)).astype(np.float32)
        self.beta = (0.1 * rng.standard_normal(dim)).astype(np.float32)
        self.norm = nhip.GroupNorm(8, dim, self.gamma, self.beta, act=nhip.ACT_SILU, blobs=True)
        self.own, self.cross = Block(rng, dim, heads, kv_heads, head_dim), Block(rng, dim, heads, kv_heads, head_dim)
        # a quarter of the pairs follow the time, the others the picture's rows and columns
        pairs = head_dim // 2
        self.sections = (pairs // 4, (pairs - pairs // 4) // 2, pairs - pairs // 4 - (pairs - pairs // 4) // 2)
        self.rotary = nhip.Rotary(head_dim, self.sections)
        # pages of the sequences in turn, as an allocator hands them out
        pages = -(-max_tokens // block_tokens)
        self.table = torch.arange(batch * pages, dtype=torch.int32, device=device).view(pages, batch).t().contiguous()
        self.cache = nhip.KvCache8(batch * pages, kv_heads, head_dim, block_tokens, device=device)
        self.max_tokens = max_tokens

    def features(self, images):
        """images [batch, 3, h, w] -> (tokens [batch, h' w', dim], (h', w'))."""
        x = images
        for _, _, conv in self.trunk:
            x = conv.forward(x)
        return self.norm.forward(x), x.shape[2:]

    def _attend_own(self, x, positions, start, causal):
        """The block's attention of new tokens x to all that the cache holds with them."""
        torch, b, n = self.torch, x.shape[0], x.shape[1]
        if start + n > self.max_tokens:  # the cache would leave out what its table has no page for
            raise ValueError(f"{start} + {n} tokens, the cache holds {self.max_tokens}")
        q = self.own.project(self.own.q, x, self.own.heads)
        k = self.own.project(self.own.k, x, self.own.kv_heads)
        v = self.own.project(self.own.v, x, self.own.kv_heads)
        self.rotary.forward(q, positions, out=q)
        self.rotary.forward(k, positions, out=k)
        self.cache.append(k, v, self.table, torch.full((b,), start, dtype=torch.int32, device=self.device))
        lengths = torch.full((b,), start + n, dtype=torch.int32, device=self.device)
        return self.own.out(x, self.cache.attention(q, self.table, lengths, max_length=self.max_tokens, causal=causal))

    def prompt(self, tokens, extent):
        """The image's tokens through the block; every token sees the whole picture.
        Keeps the keys and values of the cross attention."""
        torch = self.torch
        h, w = extent
        grid = torch.stack([torch.zeros((h * w,), dtype=torch.int32, device=self.device),
                            torch.arange(h, dtype=torch.int32, device=self.device).repeat_interleave(w),
                            torch.arange(w, dtype=torch.int32, device=self.device).repeat(h)], -1)[None]
        y = self._attend_own(tokens, grid.contiguous(), 0, causal=False)
        self.image_k = self.cross.project(self.cross.k, tokens, self.cross.kv_heads)
        self.image_v = self.cross.project(self.cross.v, tokens, self.cross.kv_heads)
        self.held = h * w
        return y

    def step(self, x, image_lengths):
        """One new token a sequence, x [batch, 1, dim]; image_lengths int32 [batch]: features of each image that
        count (the others are padding).  Returns the block's output."""
        t = self.torch.full((1, 1, 3), self.held, dtype=self.torch.int32, device=self.device)
        y = self._attend_own(x, t, self.held, causal=True)
        self.held += 1
        q = self.cross.project(self.cross.q, y, self.cross.heads)
        return self.cross.out(y, nhip.cross_attention(q, self.image_k, self.image_v, key_lengths=image_lengths))


def main():
    import torch
    nhip.init(0)
    model = ImageDecoder()
    images = torch.rand((2, 3, 48, 40), device="cuda") * 2 - 1
    tokens, extent = model.features(images)
    y = model.prompt(tokens, extent)
    print(f"{tuple(images.shape)} -> {tuple(tokens.shape)} tokens of a {tuple(extent)} picture, block {tuple(y.shape)}")
    lengths = torch.tensor([extent[0] * extent[1], extent[0] * extent[1] // 2], dtype=torch.int32, device="cuda")
    x = y[:, -1:].contiguous()
    for i in range(4):
        x = model.step(x, lengths)
        print(f"step {i}: cache of {model.held} tokens, |x| {float(x.norm()):.4f}")


if __name__ == "__main__":
    main()
