"""Host-side checks of the cache and log-probability entry points: arguments are refused, and calls without work return, before any CUDA call
(the pointers are never followed)."""
import ctypes

import pytest

from helpers import pkg

P = ctypes.cast((ctypes.c_float * 64)(), ctypes.c_void_p)
OTHER = ctypes.cast((ctypes.c_float * 64)(), ctypes.c_void_p)


@pytest.fixture
def lib():
    L = pkg().lib()
    L.df_attn_last_status()
    yield L
    L.df_attn_last_status()


def append(L, n_tokens=1, heads=2, d=64, page=16, pages=4, ks=128, vs=128, fmt=0, k=P, slots=P):
    return L.df_cache_append(k, P, slots, P, P, P, P, n_tokens, heads, d, page, pages, ks, vs, 0, fmt, None)


def attend(L, q=P, ws=P, ws_bytes=1 << 25, requests=1, tokens=1, heads=4, kv=2, d=64, page=16, pages=4, stride=256, scale=1.0, fmt=0, table=P):
    return L.df_cache_attention(q, P, P, P, P, table, P, P, P, None, ws, ws_bytes, requests, tokens, heads, kv, d, page, pages, 4, stride, scale, 0, fmt, None)


def plan(L, lens=P, out=OTHER, requests=1, tokens=1, page=16, pages=4, slots=P):
    return L.df_cache_plan(lens, P, P, P, P, out, P, slots, P, P, requests, tokens, 4, page, pages, None)


def score(L, rows=1, cols=8, stride=8, top=0, scale=1.0, logits=P, ids=P):
    return L.df_token_logprobs(logits, P, P, P, P, ids, P, rows, cols, stride, top, scale, 0, None)


def test_append_refuses_on_the_host(lib):
    p = pkg()
    for kw in (dict(heads=0), dict(d=0), dict(page=0), dict(pages=1 << 27), dict(fmt=2), dict(n_tokens=2, ks=127), dict(n_tokens=2, vs=127), dict(k=None), dict(slots=None)):
        assert append(lib, **kw) == p.DF_ERR_INVALID_ARG, kw
    for kw in (dict(d=24), dict(d=144), dict(d=8), dict(page=8), dict(page=40), dict(page=272)):
        assert append(lib, **kw) == p.DF_ERR_UNSUPPORTED, kw
    assert append(lib, n_tokens=0, k=None) == p.DF_OK
    lib.df_attn_last_status()


def test_attention_refuses_on_the_host(lib):
    p = pkg()
    for kw in (dict(heads=3), dict(heads=0), dict(kv=0), dict(scale=float("nan")), dict(scale=float("inf")), dict(fmt=7), dict(q=None), dict(ws=None), dict(table=None),
               dict(tokens=2, stride=255), dict(pages=1 << 27), dict(ws=ctypes.c_void_p(P.value + 4))):
        assert attend(lib, **kw) == p.DF_ERR_INVALID_ARG, kw
    assert attend(lib, ws_bytes=1 << 20) == p.DF_ERR_WORKSPACE
    for kw in (dict(d=24), dict(d=144), dict(page=24), dict(page=512)):
        assert attend(lib, **kw) == p.DF_ERR_UNSUPPORTED, kw
    assert attend(lib, tokens=0, q=None) == p.DF_OK and attend(lib, requests=0, q=None) == p.DF_OK


def test_plan_and_release_refuse_on_the_host(lib):
    p = pkg()
    for kw in (dict(page=0), dict(pages=1 << 27), dict(lens=None), dict(out=P), dict(slots=None), dict(tokens=1 << 31)):
        assert plan(lib, **kw) == p.DF_ERR_INVALID_ARG, kw
    assert plan(lib, requests=16385) == p.DF_ERR_UNSUPPORTED
    assert lib.df_cache_release(P, P, P, P, P, P, OTHER, 1, 4, 16, 4, None) == p.DF_ERR_INVALID_ARG      # lens_out is lens
    assert lib.df_cache_release(P, P, P, P, P, OTHER, P, 1, 4, 16, 4, None) == p.DF_ERR_INVALID_ARG      # count_out is free_count
    assert lib.df_cache_release(P, P, P, P, P, OTHER, OTHER, 16385, 4, 16, 4, None) == p.DF_ERR_UNSUPPORTED


def test_logprobs_refuse_on_the_host(lib):
    p = pkg()
    for kw in (dict(cols=0), dict(top=33), dict(top=9), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(rows=2, stride=7), dict(logits=None),
               dict(top=1, ids=None)):
        assert score(lib, **kw) == p.DF_ERR_INVALID_ARG, kw
    assert score(lib, rows=0, logits=None) == p.DF_OK
    grad = lambda rows=1, cols=8, s=8, ds=8, scale=1.0, x=P, d=OTHER: lib.df_token_logprobs_backward(x, P, P, P, P, P, d, rows, cols, s, ds, scale, 0, None)  # noqa: E731
    for kw in (dict(cols=0), dict(scale=0.0), dict(rows=2, s=7), dict(rows=2, ds=7), dict(x=None), dict(d=None), dict(rows=2, d=P, ds=9)):
        assert grad(**kw) == p.DF_ERR_INVALID_ARG, kw
    assert grad(rows=0, x=None) == p.DF_OK


def test_the_python_functions_have_no_cpu_path():
    p = pkg()
    import torch
    x, n = torch.zeros((2, 8)), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(p.AttentionError):
        p.token_logprobs(x, n)
    with pytest.raises(p.AttentionError):
        p.cache_plan(n, n, torch.zeros((2, 2), dtype=torch.int32), n, n[:1], 16, 2)
    with pytest.raises(p.AttentionError):
        p.cache_append(x, x, n, *(torch.zeros((1, 1, 16, 16), dtype=torch.int8),) * 2, *(torch.ones((1, 1)),) * 2)
