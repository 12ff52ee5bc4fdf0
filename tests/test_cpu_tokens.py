"""Refusals of the token operators that need no GPU: the C ABI checks its
arguments before any device work."""
import ctypes

import numpy as np
import pytest

import nhip

P = ctypes.c_void_p
ONE = 4096  # stands for a device pointer: none of these calls gets as far as using it


def strides(*v):
    return (ctypes.c_int64 * 3)(*v)


@pytest.mark.parametrize("channels,groups,eps,act,status", [
    (0, 1, 1e-5, 0, 2), (10, 4, 1e-5, 0, 2), (8, 0, 1e-5, 0, 2), (4100, 4, 1e-5, 0, 2),
    (8, 4, -1.0, 0, 3), (8, 4, float("nan"), 0, 3), (8, 4, float("inf"), 0, 3), (8, 4, 1e-5, nhip.ACT_SIGMOID, 7),
])
def test_group_norm_create(channels, groups, eps, act, status):
    h = P()
    assert nhip.load().nhip_group_norm_create(channels, groups, None, None, eps, act, ctypes.byref(h)) == status
    assert not h.value and nhip.load().nhip_last_error()


def test_group_norm_nulls():
    lib, h = nhip.load(), P()
    one = np.ones(8, np.float32)
    assert lib.nhip_group_norm_create(8, 4, None, None, 1e-5, 0, None) == 1
    assert lib.nhip_group_norm_create(8, 4, one.ctypes.data, None, 1e-5, 0, ctypes.byref(h)) == 1
    assert lib.nhip_group_norm_forward(None, ONE, 0, 0, 1, 1, 8, 8, ONE, ONE, 64, None) == 1
    n = ctypes.c_uint64()
    assert lib.nhip_group_norm_workspace_size(None, 0, 0, 1, 1, ctypes.byref(n)) == 1
    assert lib.nhip_norm_destroy(None) == 0


@pytest.mark.parametrize("head_dim,sections,freq,status", [
    (0, (1,), 1.0, 2), (16, (), 1.0, 2), (16, (1, 1, 1, 1, 1), 1.0, 2), (16, (-1, 4), 1.0, 2), (16, (9,), 1.0, 2),
    (16, (0, 0), 1.0, 2), (16, (4, 4), float("nan"), 3), (16, (4, 4), float("inf"), 3),
])
def test_rotary_create(head_dim, sections, freq, status):
    h = P()
    s = np.array(sections or (1,), np.int32)
    f = np.full(16, freq, np.float32)
    st = nhip.load().nhip_rotary_create(head_dim, len(sections), s.ctypes.data, f.ctypes.data, 0, ctypes.byref(h))
    assert st == status and not h.value


def test_rotary_nulls():
    lib, h = nhip.load(), P()
    s = np.array([1], np.int32)
    assert lib.nhip_rotary_create(16, 1, None, s.ctypes.data, 0, ctypes.byref(h)) == 1
    assert lib.nhip_rotary_create(16, 1, s.ctypes.data, None, 0, ctypes.byref(h)) == 1
    assert lib.nhip_rotary_create(16, 1, s.ctypes.data, s.ctypes.data, 0, None) == 1
    assert lib.nhip_rotary_forward(None, ONE, 0, 1, 1, 1, strides(1, 1, 1), ONE, 0, 0, ONE, strides(1, 1, 1), None) == 1


def desc(**kw):
    v = dict(dtype=nhip.DTYPE_F16, batch=1, queries=1, keys=64, heads=8, kv_heads=2, head_dim=64, scale=0.125)
    v.update(kw)
    return nhip.AttentionDesc(**v)


BAD_DESC = [(dict(dtype=nhip.DTYPE_I8), 7), (dict(dtype=9), 7), (dict(batch=-1), 2), (dict(queries=-1), 2),
            (dict(keys=-1), 2), (dict(heads=0), 2), (dict(kv_heads=3), 2), (dict(kv_heads=0), 2), (dict(head_dim=0), 2),
            (dict(head_dim=257), 2), (dict(scale=float("nan")), 3), (dict(scale=float("inf")), 3),
            (dict(keys=2 ** 31 - 1), 4), (dict(queries=2 ** 30), 4)]


def cross(d, q=ONE, qs=strides(512, 512, 64), k=ONE, ks=strides(8192, 128, 64), v=ONE, out=ONE, ws=ONE, nbytes=1 << 30,
          mask_stride=0):
    return nhip.load().nhip_cross_attention_forward(d, q, qs, k, ks, v, ks, None, None, mask_stride, out, ws, nbytes,
                                                    None)


@pytest.mark.parametrize("change,status", BAD_DESC)
def test_attention_descriptor(change, status):
    n = ctypes.c_uint64()
    assert nhip.load().nhip_cross_attention_workspace_size(desc(**change), ctypes.byref(n)) == status
    assert cross(desc(**change)) == status
    assert nhip.load().nhip_last_error()


def test_cross_attention_arguments():
    n = ctypes.c_uint64()
    assert nhip.load().nhip_cross_attention_workspace_size(None, ctypes.byref(n)) == 1
    assert nhip.load().nhip_cross_attention_workspace_size(desc(), None) == 1
    for bad in ("q", "k", "v", "out", "qs", "ks"):
        assert cross(desc(), **{bad: None}) == 1, bad
    assert cross(desc(), q=ONE + 1) == 3
    assert cross(desc(), k=ONE + 1) == 3
    assert cross(desc(), qs=strides(512, -1, 64)) == 2
    assert cross(desc(), ks=strides(-1, 128, 64)) == 2
    assert cross(desc(), mask_stride=-1) == 2
    assert cross(desc(batch=0)) == 0 and cross(desc(queries=0)) == 0


def cache(**kw):
    v = dict(k=ONE, v=ONE, k_scale=ONE, v_scale=ONE, pages=4, kv_heads=2, head_dim=64, block_tokens=64)
    v.update(kw)
    return nhip.Kv8Desc(**v)


BAD_CACHE = [(dict(k=None), 1), (dict(v_scale=None), 1), (dict(pages=-1), 2), (dict(kv_heads=0), 2),
             (dict(head_dim=60), 2), (dict(head_dim=264), 2), (dict(block_tokens=8), 2), (dict(block_tokens=48), 2),
             (dict(block_tokens=512), 2), (dict(k=ONE + 8), 3), (dict(k_scale=ONE + 2), 3)]


@pytest.mark.parametrize("change,status", BAD_CACHE)
def test_cache_descriptor(change, status):
    lib, c, s = nhip.load(), cache(**change), strides(128, 128, 64)
    assert lib.nhip_kv8_append(c, nhip.DTYPE_F16, ONE, s, ONE, s, 1, 1, ONE, 1, ONE, None, None) == status
    assert lib.nhip_kv8_read(c, nhip.DTYPE_F16, 1, 1, ONE, 1, ONE, ONE, ONE, None) == status
    assert lib.nhip_kv8_attention_forward(desc(), c, ONE, strides(512, 512, 64), ONE, 1, ONE, 0, ONE, ONE, 1 << 30,
                                          None) == status


def test_cache_calls():
    lib, c, s = nhip.load(), cache(), strides(128, 128, 64)
    append = lambda **k: lib.nhip_kv8_append(  # noqa: E731
        c, k.get("dtype", nhip.DTYPE_F16), k.get("key", ONE), k.get("ks", s), ONE, s, k.get("batch", 1),
        k.get("tokens", 1), k.get("table", ONE), k.get("pages", 1), k.get("starts", ONE), None, None)
    assert append(dtype=nhip.DTYPE_I8) == 7 and append(batch=-1) == 2 and append(tokens=-1) == 2
    assert append(key=None) == 1 and append(starts=None) == 1 and append(table=None) == 1 and append(ks=None) == 1
    assert append(key=ONE + 1) == 3 and append(ks=strides(1, -1, 1)) == 2 and append(pages=-1) == 2
    assert append(batch=2 ** 31 - 1, tokens=2 ** 20) == 4
    assert append(batch=0) == 0 and append(tokens=0) == 0
    assert lib.nhip_kv8_append(None, nhip.DTYPE_F16, ONE, s, ONE, s, 1, 1, ONE, 1, ONE, None, None) == 1
    read = lambda dtype, b, t, k, v: lib.nhip_kv8_read(c, dtype, b, t, ONE, 1, ONE, k, v, None)  # noqa: E731
    assert read(nhip.DTYPE_I8, 1, 1, ONE, ONE) == 7 and read(nhip.DTYPE_F16, -1, 1, ONE, ONE) == 2
    assert read(nhip.DTYPE_F16, 1, 1, None, ONE) == 1 and read(nhip.DTYPE_F16, 1, 1, ONE + 2, ONE) == 3
    assert read(nhip.DTYPE_F16, 0, 1, None, None) == 0
    attend = lambda d, lengths=ONE, q=ONE: lib.nhip_kv8_attention_forward(  # noqa: E731
        d, c, q, strides(512, 512, 64), ONE, 1, lengths, 1, ONE, ONE, 1 << 30, None)
    assert attend(desc(kv_heads=4)) == 2 and attend(desc(head_dim=32)) == 2
    assert attend(desc(), lengths=None) == 1 and attend(desc(), lengths=ONE + 1) == 3 and attend(desc(), q=ONE + 2) == 3
    assert attend(desc(batch=0)) == 0 and attend(desc(queries=0), q=None) == 0
