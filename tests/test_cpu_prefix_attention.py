"""Refusals of the attention over a shared prefix that need no GPU."""
import ctypes

import pytest

import nhip

ONE = 4096  # stands for a device pointer: none of these calls gets as far as using it


def strides(*v):
    return (ctypes.c_int64 * 3)(*v)


def desc(**kw):
    v = dict(dtype=nhip.DTYPE_F16, batch=4, queries=1, keys=64, heads=8, kv_heads=2, head_dim=64, scale=0.125)
    v.update(kw)
    return nhip.AttentionDesc(**v)


def cache(**kw):
    v = dict(k=ONE, v=ONE, k_scale=ONE, v_scale=ONE, pages=4, kv_heads=2, head_dim=64, block_tokens=64)
    v.update(kw)
    return nhip.Kv8Desc(**v)


def call(d=None, c=None, groups=2, keys=64, q=ONE, qs=strides(512, 512, 64), pt=ONE, pages=1, pl=ONE, t=ONE, lengths=ONE, out=ONE,
         ws=ONE, nbytes=1 << 30):
    return nhip.load().nhip_kv8_prefix_attention_forward(d or desc(), groups, keys, c or cache(), q, qs, pt, pages, pl, t, 1, lengths,
                                                         1, out, ws, nbytes, None)


@pytest.mark.parametrize("change,status", [
    (dict(dtype=nhip.DTYPE_I8), 7), (dict(batch=-2), 2), (dict(batch=3), 2), (dict(queries=-1), 2), (dict(keys=-1), 2),
    (dict(kv_heads=3), 2), (dict(head_dim=257), 2), (dict(scale=float("nan")), 3), (dict(keys=2 ** 31 - 1), 4),
    (dict(queries=2 ** 27), 4), (dict(queries=2 ** 30), 4)])
def test_descriptor(change, status):
    n = ctypes.c_uint64()
    assert nhip.load().nhip_kv8_prefix_attention_workspace_size(desc(**change), 2, 64, cache(), ctypes.byref(n)) == status
    assert call(desc(**change)) == status
    assert nhip.load().nhip_last_error()


def test_arguments():
    n = ctypes.c_uint64()
    size = nhip.load().nhip_kv8_prefix_attention_workspace_size
    assert size(desc(), 0, 64, cache(), ctypes.byref(n)) == 2 and size(desc(), 2, -1, cache(), ctypes.byref(n)) == 2
    assert size(desc(), 2, 64, cache(), None) == 1 and size(desc(), 2, 64, None, ctypes.byref(n)) == 1
    assert size(desc(), 2, 64, cache(), ctypes.byref(n)) == 0 and n.value > 0
    assert call(groups=0) == 2 and call(groups=3) == 2 and call(keys=-1) == 2 and call(keys=2 ** 31 - 1) == 4
    for name in ("q", "qs", "pt", "pl", "t", "lengths", "out", "ws"):
        assert call(**{name: None}) == 1, name
    assert call(c=cache(kv_heads=4)) == 2 and call(c=cache(block_tokens=8)) == 2 and call(pages=-1) == 2
    assert call(q=ONE + 2) == 3 and call(out=ONE + 8) == 3 and call(pl=ONE + 1) == 3 and call(lengths=ONE + 2) == 3
    assert call(qs=strides(512, -8, 64)) == 2 and call(qs=strides(511, 512, 64)) == 3
    assert call(nbytes=n.value - 1) == 5 and call(ws=ONE + 8) == 5
    assert call(desc(batch=0)) == 0 and call(desc(queries=0)) == 0
