"""Argument checks of the paged cache's C entries and binding; no kernel is launched."""
import ctypes

import pytest

from bmo_jetson_b200 import engine

torch = pytest.importorskip("torch")

from bmo_jetson_b200 import paged  # noqa: E402

P = 1 << 20  # an address that is never followed


def cache(**kw):
    b = paged._Book(P, P, P, P, 4, 8, 32, 16, 0)
    c = paged._Cache(b, P, P, None, None, 2, 4, 128, 0)
    for n, x in kw.items():
        setattr(c.book if n in dict(paged._Book._fields_) else c, n, x)
    return c


def attention(c, **kw):
    a = dict(layer=0, n=4, q=P, qs=2048, heads=16, rows=None, lens=None, scale=0.0, out=P, os=2048, lse=None, act=0,
             status=None, scratch=P, nbytes=1 << 30, stream=None) | kw
    return engine.lib().bmo_k_paged_attention(ctypes.byref(c) if c is not None else None, *a.values())


def append(c, **kw):
    a = dict(layer=0, n=4, k=P, ks=512, v=P, vs=512, slot=P, pos=P, theta=1e4, q=P, qs=2048, heads=16, qo=P, qos=2048,
             act=0, status=None, stream=None) | kw
    return engine.lib().bmo_k_paged_append(ctypes.byref(c) if c is not None else None, *a.values())


def read(c, **kw):
    a = dict(layer=0, n=4, slot=P, k=P, v=P, act=0, status=None, stream=None) | kw
    return engine.lib().bmo_k_paged_read(ctypes.byref(c) if c is not None else None, *a.values())


def plan(b, **kw):
    a = dict(new=P, most=8, slot=P, pos=P, req=P, offs=P, lens=P, state=P, stream=None) | kw
    return engine.lib().bmo_k_paged_plan(ctypes.byref(b) if b is not None else None, *a.values())


BAD_CACHES = [dict(head_dim=96), dict(head_dim=0), dict(n_kv_heads=0), dict(n_layers=0), dict(kv_type=2), dict(k=None),
              dict(v=P + 8), dict(kv_type=1), dict(page_size=0), dict(page_size=70000), dict(n_pages=0),
              dict(n_pages=1 << 28), dict(window=-1), dict(n_pages=(1 << 27) - 1, n_kv_heads=32)]


@pytest.mark.parametrize("kw", BAD_CACHES)
def test_bad_caches(kw):
    c = cache(**kw)
    assert attention(c) and append(c) and read(c)
    assert engine.lib().bmo_k_paged_attention_scratch_bytes(ctypes.byref(c), 16) == 0


def test_null_cache():
    assert attention(None) and append(None) and read(None) and plan(None)
    assert engine.lib().bmo_k_paged_attention_scratch_bytes(None, 16) == 0


@pytest.mark.parametrize("kw", [dict(layer=2), dict(layer=-1), dict(n=-1), dict(n=4097), dict(n=5), dict(q=None),
                                dict(q=P + 2), dict(qs=2047), dict(os=100), dict(heads=15), dict(heads=0), dict(out=None),
                                dict(act=3), dict(act=-1), dict(scratch=None), dict(scratch=P + 4),
                                dict(scale=float("inf"))])
def test_attention_arguments(kw):
    assert attention(cache(), **kw) != 0


@pytest.mark.parametrize("kw", [dict(table=None), dict(lens=None), dict(n_req=0), dict(max_blocks=0),
                                dict(max_blocks=1 << 28)])
def test_attention_tables(kw):
    assert attention(cache(**kw)) != 0


@pytest.mark.parametrize("kw", [dict(layer=2), dict(n=-1), dict(k=None), dict(v=None), dict(k=P + 2), dict(ks=511),
                                dict(slot=None), dict(pos=None), dict(theta=-1.0), dict(theta=float("nan")),
                                dict(theta=float("inf")), dict(theta=0.0), dict(heads=0), dict(qo=None), dict(qos=5),
                                dict(act=7)])
def test_append_arguments(kw):
    assert append(cache(), **kw) != 0


@pytest.mark.parametrize("kw", [dict(layer=2), dict(n=-1), dict(slot=None), dict(k=None), dict(v=P + 8), dict(act=9)])
def test_read_arguments(kw):
    assert read(cache(), **kw) != 0


@pytest.mark.parametrize("kw", [dict(new=None), dict(most=-1), dict(slot=None), dict(pos=None), dict(req=None),
                                dict(offs=None), dict(lens=None), dict(state=None)])
def test_plan_arguments(kw):
    assert plan(cache().book, **kw) != 0


@pytest.mark.parametrize("kw", [dict(table=None), dict(lens=None), dict(free_pages=None), dict(state=None), dict(n_req=0),
                                dict(n_req=65537), dict(max_blocks=0), dict(page_size=0), dict(window=-3),
                                dict(max_blocks=1 << 28)])
def test_plan_books(kw):
    assert plan(cache(**kw).book) != 0


def test_nothing_to_do():
    assert attention(cache(), n=0) == 0 and append(cache(), n=0) == 0 and read(cache(), n=0) == 0


def test_book_needs_a_gpu():
    with pytest.raises(ValueError):
        paged.PageBook.empty(2, 4, 16, 2, device="cpu")
