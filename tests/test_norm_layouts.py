"""What layer_norm returns as a tensor: memory order, and that it can be changed in place.  On the CPU, with the library's calls replaced by
ones that fill the result with a number; the values are checked on the device in test_norm_gpu.py::test_layouts."""
import ctypes

import pytest
import torch


@pytest.fixture
def fake(monkeypatch):
    from taming_event_flow_amd.models import norm

    class Lib:
        def __init__(self):
            self.saved = []

        def tef_layer_norm_forward(self, d, x, w, b, r, y, mean, rstd, stream):
            self.saved.append(mean)
            n = d._obj.outer * d._obj.inner * d._obj.channels
            (ctypes.c_float * n).from_address(y)[:] = [1.0] * n
            return 0

        def tef_layer_norm_workspace_bytes(self, d):
            return 16

        def tef_layer_norm_backward(self, d, x, w, b, r, mean, rstd, dy, dx, dr, dw, db, ws, nbytes, stream):
            n = d._obj.outer * d._obj.inner * d._obj.channels
            (ctypes.c_float * n).from_address(dx)[:] = [2.0] * n
            return 0

    lib = Lib()
    monkeypatch.setattr(norm._lib, "require_device_tensor", lambda t, name: t)
    monkeypatch.setattr(norm._lib, "lib", lambda: lib)
    monkeypatch.setattr(norm._lib, "stream_ptr", lambda: None)
    return lib


LAYOUTS = {"contiguous": lambda: torch.zeros(2, 6, 3, 4), "channels_last": lambda: torch.zeros(2, 6, 3, 4).contiguous(memory_format=torch.channels_last),
           "one_sample_channels_last": lambda: torch.zeros(1, 6, 3, 4).contiguous(memory_format=torch.channels_last),
           "one_channel": lambda: torch.zeros(2, 1, 3, 4).contiguous(memory_format=torch.channels_last),
           "odd_stride_of_one_sample": lambda: torch.zeros(72).as_strided((1, 6, 3, 4), (7, 1, 24, 6)),
           "gaps": lambda: torch.zeros(2, 6, 3, 8)[..., ::2], "sequence": lambda: torch.zeros(5, 2, 6).permute(1, 2, 0)}


@pytest.mark.parametrize("name", LAYOUTS)
def test_result_may_be_changed_in_place(fake, name):
    from taming_event_flow_amd.models.norm import layer_norm

    x = LAYOUTS[name]().requires_grad_(True)
    y = layer_norm(x)
    assert y.shape == x.shape and not y._is_view() and y.grad_fn is not None
    y.mul_(2).clamp_(min=0)      # refused for a view made inside the function
    assert bool((y == 2).all())
    y.sum().backward()
    assert x.grad.shape == x.shape and bool((x.grad == 2).all())


def test_memory_order(fake):
    from taming_event_flow_amd.models.norm import layer_norm

    for name, make in LAYOUTS.items():
        x = make()
        y = layer_norm(x)
        dense = x.is_contiguous() or x.movedim(1, -1).is_contiguous()
        assert y.stride() == (x.stride() if dense else x.contiguous().stride()), name


def test_statistics_are_kept_for_a_backward_pass_only(fake):
    from taming_event_flow_amd.models.norm import LayerNorm

    m, x = LayerNorm(6), LAYOUTS["contiguous"]()
    with torch.no_grad():
        m(x)
    m(x)
    m.requires_grad_(False)
    m(x)
    m(x.requires_grad_(True))
    assert [s is not None for s in fake.saved] == [False, True, False, True]


def test_more_channels_than_32_bits_hold(fake):
    """A size that a 32-bit number of channels would cut down to 8 is refused, by both entry points."""
    from taming_event_flow_amd import _lib
    from taming_event_flow_amd.models import norm

    for n in (2 ** 32 + 8, 2 ** 31, 2 ** 30 + 1):
        x = torch.zeros((), dtype=torch.bfloat16).expand(1, n)
        with pytest.raises(ValueError, match="at most"):
            norm.layer_norm(x, dim=-1)


def test_channel_limit_of_the_library():
    import __graft_entry__ as g

    g.build()
    from taming_event_flow_amd import _lib

    lib = _lib.lib()
    for n, ok in ((2 ** 30, True), (2 ** 30 + 1, False), (2 ** 31 - 1, False)):
        d = _lib.NormDesc(1, 1, n, 2, 0, 0, 1e-5)
        assert (lib.tef_layer_norm_workspace_bytes(ctypes.byref(d)) == 8 * n) == ok
