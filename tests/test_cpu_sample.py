"""Refusals of the draw of a token that need no GPU."""
import ctypes

import pytest

import nhip

ONE = 4096  # stands for a device pointer: none of these calls gets as far as using it


def desc(**kw):
    v = dict(dtype=nhip.DTYPE_F16, rows=2, vocab=100, row_stride=100, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0)
    v.update(kw)
    return nhip.SampleDesc(**v)


def forward(d, logits=ONE, uniform=ONE, token=ONE, logprob=ONE, ws=None, nbytes=0):
    return nhip.load().nhip_sample_forward(d, logits, uniform, token, logprob, ws, nbytes, None)


@pytest.mark.parametrize("change,status", [
    (dict(dtype=nhip.DTYPE_I8), 7), (dict(rows=-1), 2), (dict(vocab=0), 2), (dict(vocab=2 ** 19 + 1), 4), (dict(rows=2 ** 22), 4), (dict(row_stride=-1), 2),
    (dict(temperature=-0.5), 3), (dict(temperature=float("nan")), 3), (dict(top_k=-1), 3), (dict(top_p=-1.0), 3),
    (dict(top_p=float("nan")), 3), (dict(min_p=-0.1), 3), (dict(min_p=1.1), 3), (dict(min_p=float("nan")), 3),
    (dict(temperature_each=ONE + 2), 3), (dict(top_k_each=ONE + 1), 3), (dict(top_p_each=ONE + 3), 3), (dict(min_p_each=ONE + 2), 3)])
def test_descriptor(change, status):
    n = ctypes.c_uint64()
    assert nhip.load().nhip_sample_workspace_size(desc(**change), ctypes.byref(n)) == status
    assert forward(desc(**change)) == status
    assert nhip.load().nhip_last_error()


def test_arguments():
    lib, n = nhip.load(), ctypes.c_uint64()
    assert lib.nhip_sample_workspace_size(None, ctypes.byref(n)) == 1 and lib.nhip_sample_workspace_size(desc(), None) == 1
    assert forward(None) == 1
    for name in ("logits", "uniform", "token", "logprob"):
        assert forward(desc(), **{name: None}) == 1, name
        assert forward(desc(), **{name: ONE + 1}) == 3, name
    assert forward(desc(rows=0)) == 0


def test_workspace():
    d, n = desc(vocab=100000), ctypes.c_uint64()
    assert nhip.load().nhip_sample_workspace_size(d, ctypes.byref(n)) == 0 and n.value > 0
    assert forward(d) == 1 and forward(d, ws=ONE, nbytes=n.value - 1) == 5 and forward(d, ws=ONE + 8, nbytes=n.value) == 5
    assert nhip.load().nhip_sample_workspace_size(desc(), ctypes.byref(n)) == 0 and n.value == 0


@pytest.mark.parametrize("change,listed", [
    (dict(), False), (dict(min_p=0.1), False), (dict(top_k=1), False), (dict(temperature=0.0, top_k=40, top_p=0.9), False),
    (dict(top_k=40), True), (dict(top_k=3000), True), (dict(top_p=0.9), True), (dict(top_k_each=ONE), True), (dict(top_p_each=ONE), True),
    (dict(temperature=0.0, temperature_each=ONE, top_p=0.9), True), (dict(top_k=1, top_k_each=ONE), True), (dict(top_k=2 ** 18), False)])
def test_workspace_of_lists(nhip_env, change, listed):
    """Rows begun by several workgroups: 64 KB each for a list of tokens, only where a row can have one."""
    nhip_env.setenv("NHIP_SAMPLE_CHUNKS", "4")
    n = ctypes.c_uint64()
    assert nhip.load().nhip_sample_workspace_size(desc(vocab=100000, rows=1000, **change), ctypes.byref(n)) == 0
    assert (n.value >= 1000 * 65536) == listed and n.value >= 1000 * (1024 * 8 + 4 * 8)
