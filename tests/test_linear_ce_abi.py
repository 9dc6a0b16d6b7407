"""Host-side checks of the loss from hidden states, the orthogonalised updates and the optimiser step: arguments are refused, and calls without work return, before any
CUDA call (the pointers are never followed)."""
import ctypes

import pytest

from helpers import pkg

N = 1 << 16
BUFFERS = [(ctypes.c_float * N)() for _ in range(8)]


def at(i, offset=0):
    return ctypes.c_void_p(ctypes.addressof(BUFFERS[i]) + offset)


def aligned(i):
    a = ctypes.addressof(BUFFERS[i])
    return ctypes.c_void_p((a + 255) // 256 * 256)


@pytest.fixture
def lib():
    L = pkg().lib()
    L.df_attn_last_status()
    yield L
    L.df_attn_last_status()


def loss(L, x=at(0), w=at(1), t=at(2), loss=at(3), lse=at(4), ws=aligned(5), ws_bytes=1 << 40, rows=2, vocab=8, width=8, xs=8, wst=8, scale=1.0, bf16=0):
    return L.df_linear_cross_entropy(x, w, t, loss, lse, ws, ws_bytes, rows, vocab, width, xs, wst, scale, bf16, None)


def grad(L, x=at(0), w=at(1), t=at(2), lse=at(3), g=at(4), dx=at(6), dw=at(7), ws=aligned(5), ws_bytes=1 << 40, rows=2, vocab=8, width=8, xs=8, wst=8, dxs=8, dws=8,
         scale=1.0, bf16=0):
    return L.df_linear_cross_entropy_backward(x, w, t, lse, g, dx, dw, ws, ws_bytes, rows, vocab, width, xs, wst, dxs, dws, scale, bf16, None)


def orth(L, u=at(0), out=at(1), ws=aligned(5), ws_bytes=1 << 40, n=1, rows=4, cols=8, um=32, ur=8, om=32, orow=8, steps=5, a=3.4445, b=-4.775, c=2.0315, eps=1e-7, bf16=0):
    return L.df_orthogonalize(u, out, ws, ws_bytes, n, rows, cols, um, ur, om, orow, steps, a, b, c, eps, bf16, None)


def table(*tensors):
    return ctypes.cast((ctypes.c_void_p * (3 * len(tensors)))(*[p.value if p else None for t in tensors for p in t]), ctypes.c_void_p)


GOOD = (at(0), at(1), at(2))


def muon(L, tensors=None, n=1, rows=4, cols=8, lr=0.1, beta=0.9, decay=0.0, scale=1.0, steps=5, a=3.4445, eps=1e-7, ws=aligned(5), ws_bytes=1 << 40):
    return L.df_muon_update(table(GOOD) if tensors is None else tensors, n, rows, cols, lr, beta, decay, 1, scale, steps, a, -4.775, 2.0315, eps, ws, ws_bytes, None)


NAN, INF = float("nan"), float("inf")


@pytest.mark.parametrize("kw", [dict(vocab=0), dict(width=0), dict(vocab=1 << 30), dict(width=1 << 24), dict(rows=1 << 30), dict(xs=7), dict(wst=7), dict(scale=0.0), dict(scale=-1.0),
                                dict(scale=NAN), dict(scale=INF), dict(x=None), dict(w=None), dict(t=None), dict(xs=1 << 32), dict(wst=1 << 32)])
def test_both_directions_refuse(lib, kw):
    assert loss(lib, **kw) == pkg().DF_ERR_INVALID_ARG and grad(lib, **kw) == pkg().DF_ERR_INVALID_ARG


@pytest.mark.parametrize("kw", [dict(loss=None), dict(lse=None), dict(lse=at(3)), dict(loss=at(0, 4)), dict(lse=at(1, 60)), dict(loss=at(2)), dict(loss=aligned(5))])
def test_loss_refuses(lib, kw):
    assert loss(lib, **kw) == pkg().DF_ERR_INVALID_ARG


@pytest.mark.parametrize("kw", [dict(lse=None), dict(g=None), dict(dxs=7), dict(dws=7), dict(dx=at(0)), dict(dx=at(1, 32)), dict(dw=at(1)), dict(dw=at(6, 32)), dict(dx=at(3)), dict(dw=at(4)),
                                dict(dx=at(2)), dict(dx=aligned(5)), dict(dws=1 << 32)])
def test_gradient_refuses(lib, kw):
    assert grad(lib, **kw) == pkg().DF_ERR_INVALID_ARG


@pytest.mark.parametrize("call", [loss, grad, orth, muon])
def test_workspaces(lib, call):
    p = pkg()
    size = dict(loss=lib.df_linear_cross_entropy_workspace_bytes(2, 8, 8, 0, 0), grad=lib.df_linear_cross_entropy_workspace_bytes(2, 8, 8, 0, 1),
                orth=lib.df_orthogonalize_workspace_bytes(1, 4, 8), muon=lib.df_orthogonalize_workspace_bytes(1, 4, 8))[call.__name__]
    assert size > 0
    for kw in (dict(ws=None), dict(ws_bytes=size - 1), dict(ws=ctypes.c_void_p(aligned(5).value + 128))):
        assert call(lib, **kw) == p.DF_ERR_WORKSPACE, kw


def test_workspace_sizes(lib):
    size = lib.df_linear_cross_entropy_workspace_bytes
    assert size(0, 8, 8, 0, 0) == 0 and size(8, 0, 8, 0, 0) == 0 and size(8, 8, 0, 0, 1) == 0
    # the logits of 8192 x 50257 rows in fp32 are 1647 MB; what is held is a piece of their gradient, and of the weight in fp16
    assert size(8192, 50257, 768, 1, 0) < 200 << 20 and size(8192, 50257, 768, 1, 1) < 700 << 20
    for rows in (1, 7, 300, 5000):
        for vocab in (1, 255, 257, 50257):
            for width in (1, 64, 65, 1000):
                for bf16 in (0, 1):
                    for backward in (0, 1):
                        assert size(rows, vocab, width, bf16, backward) % 256 == 0
    more = lib.df_orthogonalize_workspace_bytes
    assert more(0, 8, 8) == 0 and more(1, 0, 8) == 0 and more(1, 65537, 8) == 0 and more(1, 65536, 65536) == 0
    assert more(1000, 768, 768) <= 193 << 20


def test_calls_without_work(lib):
    p = pkg()
    assert loss(lib, rows=0, x=None, t=None) == p.DF_OK and grad(lib, rows=0, x=None, t=None, dw=None) == p.DF_OK
    assert grad(lib, dx=None, dw=None) == p.DF_OK
    assert orth(lib, n=0, u=None) == p.DF_OK and muon(lib, n=0) == p.DF_OK


@pytest.mark.parametrize("kw", [dict(rows=0), dict(cols=0), dict(rows=65537), dict(cols=65537), dict(rows=65536, cols=32768), dict(steps=0), dict(steps=65), dict(a=NAN), dict(eps=-1.0),
                                dict(eps=NAN), dict(eps=INF)])
def test_orthogonalising_refuses(lib, kw):
    assert orth(lib, **kw) == pkg().DF_ERR_INVALID_ARG and muon(lib, **kw) == pkg().DF_ERR_INVALID_ARG


def test_strides_and_overlaps_of_matrices(lib):
    p = pkg()
    for kw in (dict(u=None), dict(out=None), dict(ur=7), dict(orow=7), dict(n=2, om=31), dict(out=at(0, 4)), dict(out=at(0), orow=9), dict(n=2, out=at(0), om=33), dict(um=1 << 40)):
        assert orth(lib, **kw) == p.DF_ERR_INVALID_ARG, kw
    assert orth(lib, a=12.0) == p.DF_ERR_UNSUPPORTED


def test_optimiser_refuses(lib):
    p = pkg()
    bytes_ = 4 * 8 * 4
    for t in ((None, at(1), at(2)), (at(0), None, at(2)), (at(0), at(1), None), (at(0), at(0, bytes_ - 4), at(2)), (at(0), at(1), at(0)), (at(0), at(1), at(1, 4))):
        assert muon(lib, tensors=table(t)) == p.DF_ERR_INVALID_ARG
    two = lambda second: muon(lib, tensors=table(GOOD, second), n=2)  # noqa: E731
    for t in ((at(0), at(3), at(4)), (at(3), at(1), at(4)), (at(3), at(4), at(0)), (at(3), at(4), at(1)), (at(2), at(3), at(4)), (at(0, bytes_ - 4), at(3), at(4))):
        assert two(t) == p.DF_ERR_INVALID_ARG
    for kw in (dict(lr=NAN), dict(beta=INF), dict(decay=NAN), dict(scale=INF)):
        assert muon(lib, **kw) == p.DF_ERR_INVALID_ARG, kw
    assert muon(lib, n=1025) == p.DF_ERR_UNSUPPORTED
    assert lib.df_muon_update(None, 1, 4, 8, 0.1, 0.9, 0.0, 1, 1.0, 5, 3.0, -4.0, 2.0, 1e-7, aligned(5), 1 << 40, None) == p.DF_ERR_INVALID_ARG


def test_matrices_in_the_workspace(lib):
    p = pkg()
    inside = ctypes.c_void_p(aligned(5).value + 128)  # 4 x 8 in fp32 need more than that of it
    assert orth(lib, u=inside) == p.DF_ERR_INVALID_ARG and orth(lib, out=inside) == p.DF_ERR_INVALID_ARG and orth(lib, u=inside, out=inside) == p.DF_ERR_INVALID_ARG
    for t in ((inside, at(1), at(2)), (at(0), inside, at(2)), (at(0), at(1), inside)):
        assert muon(lib, tensors=table(t)) == p.DF_ERR_INVALID_ARG


def test_overlaps_among_many_tensors(lib):
    p = pkg()
    n, each = 341, 4 * 8 * 4
    places = [ctypes.c_void_p(at(0).value + i * each) for i in range(3 * n)]
    for i, j in ((0, 3 * n - 1), (3 * n - 1, 1), (4, 600), (302, 301)):  # a parameter or momentum moved onto the end of another tensor
        moved = list(places)
        k = i if i % 3 != 2 else j
        moved[k] = ctypes.c_void_p(places[j if k == i else i].value + each - 4)
        assert muon(lib, tensors=table(*[tuple(moved[3 * x:3 * x + 3]) for x in range(n)]), n=n) == p.DF_ERR_INVALID_ARG
    # the same gradient for two parameters is none: what is refused is only the missing workspace
    shared = [tuple(places[3 * x:3 * x + 3]) for x in range(n)]
    shared[7] = shared[7][:2] + (shared[200][2],)
    assert muon(lib, tensors=table(*shared), n=n, ws=None) == p.DF_ERR_WORKSPACE


def test_a_weight_that_has_to_be_copied_is_so_in_pieces(lib):
    size = lib.df_linear_cross_entropy_workspace_bytes
    assert size(64, 1 << 18, 16384, 1, 0) < 300 << 20 and size(64, 1 << 18, 16384, 0, 0) < 300 << 20
