"""Refusals of the layer normalisation, without a GPU: the Python entry point's and the C entry points' argument checks."""
import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def lib_():
    import __graft_entry__ as g

    g.build()
    from taming_event_flow_amd import _lib

    return _lib


def test_python_refusals(lib_, monkeypatch):
    from taming_event_flow_amd.models import norm

    x = torch.zeros(2, 8, 4, 4)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        norm.layer_norm(x)
    monkeypatch.setattr(norm._lib, "require_device_tensor", lambda t, name: t)      # the other checks need no device
    monkeypatch.setattr(norm._LayerNormFn, "apply", lambda *a: pytest.fail("not refused"))
    f = norm.layer_norm
    for call, error in ((lambda: f(x.double()), TypeError), (lambda: f(x.long()), TypeError), (lambda: f(x, dim=4), IndexError),
                        (lambda: f(x, dim=-5), IndexError), (lambda: f(torch.zeros(())), IndexError), (lambda: f(torch.zeros(3, 0)), ValueError),
                        (lambda: f(x, eps=-1.0), ValueError), (lambda: f(x, eps=float("nan")), ValueError),
                        (lambda: f(x, eps=float("inf")), ValueError), (lambda: f(x, activation="gelu"), NotImplementedError),
                        (lambda: f(x, torch.ones(7)), ValueError), (lambda: f(x, None, torch.ones(8, 1)), ValueError),
                        (lambda: f(x, torch.ones(8, dtype=torch.float16)), TypeError),
                        (lambda: f(x.half(), torch.ones(8), torch.ones(8, dtype=torch.float16)), TypeError),
                        (lambda: f(x, torch.ones(8, device="meta")), RuntimeError),
                        (lambda: f(x, residual=x[:1]), ValueError), (lambda: f(x, residual=x.half()), ValueError)):
        with pytest.raises(error):
            call()


def test_c_refusals(lib_):
    lib = lib_.lib()
    good = dict(outer=2, inner=4, channels=8, dtype=0, wdtype=0, act=0, eps=1e-5)
    buf = ctypes.create_string_buffer(16)
    p = ctypes.addressof(buf)      # (never dereferenced: every call below is refused before a launch)

    def desc(**kw):
        return ctypes.byref(lib_.NormDesc(**dict(good, **kw)))

    for bad in (dict(channels=0), dict(outer=-1), dict(inner=0), dict(dtype=3), dict(wdtype=1), dict(dtype=1, wdtype=2), dict(act=4),
                dict(eps=-1.0), dict(eps=float("nan")), dict(outer=2 ** 40, inner=2 ** 30)):
        assert lib.tef_layer_norm_forward(desc(**bad), p, None, None, None, p, None, None, None) == -1, bad
        assert lib.tef_layer_norm_workspace_bytes(desc(**bad)) == 0
        assert b"layer norm" in lib.tef_last_error()
    assert lib.tef_layer_norm_forward(None, p, None, None, None, p, None, None, None) == -1
    assert lib.tef_layer_norm_forward(desc(), None, None, None, None, p, None, None, None) == -1
    assert lib.tef_layer_norm_forward(desc(), p, None, None, None, p, p, None, None) == -1      # mean without rstd
    need = lib.tef_layer_norm_workspace_bytes(desc())
    assert need > 0
    args = [p, None, None, None, p, p, p, p, None, p, p]
    assert lib.tef_layer_norm_backward(desc(), *args, p, need - 1, None) == -2
    assert lib.tef_layer_norm_backward(desc(), *args, None, need, None) == -2
    args[4] = None
    assert lib.tef_layer_norm_backward(desc(), *args, p, need, None) == -1
