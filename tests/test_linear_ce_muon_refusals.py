"""CPU: what odl_linear_cross_entropy, odl_newton_schulz and odl_muon_step refuse, before anything reaches a device."""
import pytest
import torch

from origindl_b200 import build, capi, ops

INVALID, TOO_LARGE, NOT_INITIALIZED = 1, 5, 6
SOME = 256  # an address that no refused call follows


@pytest.fixture(scope="module")
def lib():
    build.build()
    return capi.lib()


def lce(lib, x=SOME, w=SOME, b=None, labels=SOME, M=4, N=8, K=16, layout=0, loss=SOME, lse=None, dx=None, dw=None, db=None,
        precision=0):
    return lib.odl_linear_cross_entropy(x, w, b, labels, 1, -100, M, N, K, layout, loss, lse, dx, dw, db, 1.0, precision, None)


@pytest.mark.parametrize("bad", [dict(x=None), dict(w=None), dict(labels=None), dict(loss=None), dict(M=0), dict(N=0), dict(K=0),
                                 dict(M=-1), dict(layout=2), dict(layout=-1), dict(precision=2), dict(precision=-1)])
def test_linear_cross_entropy_refuses(lib, bad):
    assert lce(lib, **bad) == INVALID
    assert b"linear_cross_entropy" in lib.odl_last_error()


@pytest.mark.parametrize("bad", [dict(M=1 << 31), dict(N=1 << 31), dict(K=1 << 40)])
def test_linear_cross_entropy_refuses_sizes(lib, bad):
    assert lce(lib, **bad) == TOO_LARGE


def ns(lib, g=SOME, out=SOME, batch=1, rows=4, cols=8, steps=5, eps=1e-7, precision=0):
    return lib.odl_newton_schulz(g, out, batch, rows, cols, steps, eps, precision, None)


@pytest.mark.parametrize("bad", [dict(g=None), dict(out=None), dict(batch=0), dict(rows=0), dict(cols=-3), dict(steps=-1),
                                 dict(steps=101), dict(eps=0.0), dict(eps=float("nan")), dict(precision=7)])
def test_newton_schulz_refuses(lib, bad):
    assert ns(lib, **bad) == INVALID
    assert b"newton_schulz" in lib.odl_last_error()


@pytest.mark.parametrize("bad", [dict(rows=1 << 31), dict(cols=1 << 31), dict(batch=1 << 16)])
def test_newton_schulz_refuses_sizes(lib, bad):
    assert ns(lib, **bad) == TOO_LARGE


def muon(lib, p=SOME, g=SOME, buf=SOME, batch=1, rows=4, cols=8, layout=0, momentum=0.95, steps=5, eps=1e-7, precision=0):
    return lib.odl_muon_step(p, g, buf, None, batch, rows, cols, layout, 0.02, momentum, 0.0, 1, 0.0, 1.0, steps, eps, precision,
                             None)


@pytest.mark.parametrize("bad", [dict(p=None), dict(g=None), dict(buf=None), dict(layout=3), dict(momentum=-0.5),
                                 dict(momentum=float("nan")), dict(batch=-1), dict(rows=0), dict(eps=-1.0), dict(precision=2)])
def test_muon_refuses(lib, bad):
    assert muon(lib, **bad) == INVALID
    assert b"muon" in lib.odl_last_error()


def test_nothing_runs_without_a_device(lib):
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    assert lce(lib) == NOT_INITIALIZED and ns(lib) == NOT_INITIALIZED and muon(lib) == NOT_INITIALIZED


def test_front_end_refuses_host_tensors():
    x, w, t = torch.zeros(4, 8), torch.zeros(5, 8), torch.zeros(4, dtype=torch.int64)
    with pytest.raises(ValueError):
        ops.linear_cross_entropy(x, w, t)
    with pytest.raises(ValueError):
        ops.newton_schulz(x)
    with pytest.raises(ValueError):
        ops.muon_step(x, x, x)
