"""Refusals of the knet_linear_nll_* and global-norm entry points: status codes before anything is
launched, so they run without a GPU."""
import ctypes as C

import pytest

V, H, N = 100, 32, 16
P = 4096          # an address that is never read: every call below is refused first


@pytest.fixture(scope="module")
def lib():
    from knet_sm100 import lib
    return lib.libknet


def fwd(lib, S="32", w=P, trans=0, b=None, x=P, labels=P, V=V, H=H, N=N, total=P, count=P, lse=P, per=P, ws=P, nbytes=1 << 40):
    return getattr(lib, f"knet_linear_nll_fwd_{S}")(w, trans, b, x, labels, V, H, N, total, count, lse, per, ws, nbytes, None)


def bwd(lib, S="32", w=P, trans=0, b=None, x=P, labels=P, V=V, H=H, N=N, lse=P, average=1, dy=1.0, count=P, dw=P, db=None, dx=P,
        ws=P, nbytes=1 << 40):
    return getattr(lib, f"knet_linear_nll_bwd_{S}")(w, trans, b, x, labels, V, H, N, lse, average, dy, count, dw, db, dx, ws, nbytes,
                                                   None)


@pytest.mark.parametrize("S", ["32", "64"])
def test_linear_nll_arguments(lib, S):
    for f in (fwd, bwd):
        for bad in (dict(V=0), dict(V=-1), dict(H=0), dict(N=-1), dict(trans=2), dict(w=None), dict(x=None), dict(labels=None),
                    dict(lse=None)):
            assert f(lib, S, **bad) == -1, (f.__name__, bad)
        for big in (dict(V=1 << 22), dict(H=1 << 22), dict(N=1 << 22), dict(V=1 << 40)):
            assert f(lib, S, **big) == -2, (f.__name__, big)
        need = getattr(lib, f"knet_linear_nll_workspace_{S}")(V, H, N, int(f is bwd))
        assert need > 0
        assert f(lib, S, nbytes=need - 1) == -3 and f(lib, S, ws=None) == -3
        for odd in (dict(w=P + 2), dict(x=P + 2), dict(b=P + 1), dict(labels=P + 2), dict(ws=P + 16), dict(lse=P + 2)):
            assert f(lib, S, **odd) == -4, (f.__name__, odd)
    assert fwd(lib, S, total=None) == -1 and fwd(lib, S, count=None) == -1 and fwd(lib, S, per=None) == -1
    assert bwd(lib, S, count=None) == -1 and bwd(lib, S, dw=P + 2) == -4 and bwd(lib, S, db=P + 1) == -4 and bwd(lib, S, dx=P + 1) == -4


def test_workspace_sizes(lib):
    for S in ("32", "64"):
        q = getattr(lib, f"knet_linear_nll_workspace_{S}")
        assert q(0, 4, 4, 0) == 0 and q(4, 0, 4, 1) == 0 and q(4, 4, 0, 1) == 0 and q(1 << 22, 4, 4, 0) == 0
        for back in (0, 1):
            assert q(50257, 1024, 4096, back) < (768 << 20)          # far below a score matrix and its gradient
            assert q(1, 1, 1, back) % 256 == 0


def test_global_norm_arguments(lib):
    for S in ("32", "64"):
        g = lambda *a: getattr(lib, f"knet_gnorm_{S}")(*a, None)
        c = lambda *a: getattr(lib, f"knet_gclip_global_{S}")(*a, None)
        assert g(P, -1, 1, 1.0, P, P) == -1 and g(P, 1, -1, 1.0, P, P) == -1 and g(None, 1, 1, 1.0, P, P) == -1
        assert g(P, 1, 1, 1.0, None, P) == -1 and g(P, 1, 1, 1.0, P, None) == -1 and g(P, 1, 1, 1.0, P + 4, P) == -4
        assert g(P, 1, 1 << 31, 1.0, P, P) == -2
        assert c(P, 1, 1, 0.0, 1.0, P, P, P) == -1 and c(P, 1, 1, float("nan"), 1.0, P, P, P) == -1
        assert c(P, 1, 1, 1.0, 1.0, P, P, None) == -1 and c(P, 1, 1, 1.0, 1.0, P, P, P + 4) == -4
        a = getattr(lib, f"knet_gclip_apply_{S}")
        assert a(P, 1, 1, None, None) == -1 and a(None, 1, 1, P, None) == -1 and a(P, 0, 0, None, None) == 0
        assert getattr(lib, f"knet_sgd_multi_gc_{S}")(P, 1, 1, 0.1, 1.0, None, None) == -1
        assert getattr(lib, f"knet_adam_multi_gc_{S}")(P, 1, 1, 0.1, 0.9, 0.99, 1e-8, 0, 1.0, P, None) == -1
        assert getattr(lib, f"knet_adam_multi_gcg_{S}")(P, 1, 1, 0.1, 0.9, 0.99, 1e-8, None, 1.0, P, None) == -1


def test_workspace_holds_no_room_that_nothing_uses(lib):
    """Few classes, many instances: dx is written where it belongs, not by way of the workspace."""
    scores = 10 * 100_000
    assert lib.knet_linear_nll_workspace_64(10, 4096, 100_000, 1) < 2 * 8 * scores + (64 << 20) + (1 << 20)
    assert lib.knet_linear_nll_workspace_32(10, 64, 100_000, 1) < 4 * scores + (1 << 20)


def test_the_forms_that_hand_maxima_over(lib):
    """knet_linear_nll_*_max_S refuse what the forms without `class_max` refuse, and one of odd alignment."""
    for S in ("32", "64"):
        f = lambda class_max=P, V=V, ws=P, need=1 << 40: getattr(lib, f"knet_linear_nll_fwd_max_{S}")(
            P, 0, None, P, P, V, H, N, P, P, P, P, class_max, ws, need, None)
        b = lambda class_max=P, V=V, ws=P, need=1 << 40: getattr(lib, f"knet_linear_nll_bwd_max_{S}")(
            P, 0, None, P, P, V, H, N, P, class_max, 1, 1.0, P, P, None, P, ws, need, None)
        for g in (f, b):
            assert g(V=0) == -1 and g(V=1 << 22) == -2 and g(ws=None) == -3 and g(need=0) == -3 and g(class_max=P + 2) == -4
