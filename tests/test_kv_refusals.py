"""Refusals of the rotary, cache and attention entry points that need no GPU:
arguments are checked before the library touches a device."""
import ctypes as C

import pytest

from conftest import load_package


@pytest.fixture(scope="module")
def m():
    return load_package()


def refused(m, fn, *a, code=-1, **kw):
    with pytest.raises(m.MoeError) as e:
        fn(*a, **kw)
    assert e.value.code == code, str(e.value)


@pytest.mark.parametrize("kw", [
    dict(rot=0), dict(rot=3), dict(rot=-2), dict(rot=4098), dict(max_position=0),
    dict(max_position=(1 << 24) + 1), dict(theta=1.0), dict(theta=float("nan")),
    dict(theta=float("inf")), dict(layout=2), dict(scaling=4), dict(scaling=-1),
    dict(scaling=1, factor=0.5), dict(scaling=1, factor=float("nan")), dict(scaling=2, factor=2.0),
    dict(scaling=2, factor=2.0, orig_context=100, beta_fast=1.0, beta_slow=2.0),
    dict(scaling=3, factor=2.0, orig_context=100, low_freq=4.0, high_freq=4.0),
    dict(magnitude=-1.0), dict(magnitude=float("nan")), dict(freq_divisors=[1.0] * 3),
    dict(freq_divisors=[1.0, 0.0, 1.0, 1.0]), dict(freq_divisors=[1.0, float("nan"), 1.0, 1.0])])
def test_rope_description(m, kw):
    refused(m, m.Rope, **(dict(rot=8, theta=1e4, max_position=100) | kw))


@pytest.mark.parametrize("kw,code", [
    (dict(n_pages=0), -1), (dict(n_pages=1 << 31), -1), (dict(page_size=8), -1), (dict(page_size=48), -1),
    (dict(page_size=512), -1), (dict(n_kv_heads=0), -1), (dict(n_kv_heads=4097), -1),
    (dict(head_len=32), -1), (dict(head_len=96), -1), (dict(qtype=1), -2), (dict(qtype=0), -2),
    (dict(pages=4104), -1)])
def test_cache_description(m, kw, code):
    refused(m, m.KVCache, code=code, **(dict(n_pages=4, page_size=16, n_kv_heads=2, head_len=64) | kw))


def test_page_bytes(m):
    assert m.kv_page_bytes(16, 1, 64) == 16 * 2 * 36
    assert m.kv_page_bytes(64, 8, 128) == 64 * 8 * 2 * 72
    assert m.kv_page_bytes(256, 3, 256) == 256 * 3 * 2 * 144
    for bad in [(0, 1, 64), (17, 1, 64), (16, 0, 64), (16, 1, 65), (16, -1, 64)]:
        assert m.kv_page_bytes(*bad) == 0
    assert m.kv_page_bytes(16, 1, 64, m.Q8_0) == 0


def test_null_handles(m):
    L = m.lib()
    b, r = m.KVBatch(), m.Rows()
    for rc in (L.moe_rope_create(None, None), L.moe_kv_create(None, None),
               L.moe_rope_forward(None, 1, 64, None, C.byref(r), C.byref(r), None, None, None),
               L.moe_rope_status(None), L.moe_kv_status(None),
               L.moe_kv_append(None, C.byref(b), None, None, C.byref(r), C.byref(r), None, None, None),
               L.moe_kv_gather(None, C.byref(b), C.byref(r), None, None),
               L.moe_kv_attention(None, C.byref(b), C.byref(r), C.byref(r), None, 1.0, 1, 0, None, 0, None),
               L.moe_kv_attention_workspace(None, C.byref(b), 8)):
        assert rc == -1
        assert L.moe_last_error()
    assert L.moe_kv_pages(None) is None
    assert L.moe_rope_destroy(None) == 0 and L.moe_kv_destroy(None) == 0
