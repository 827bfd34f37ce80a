"""Refusals of the orthogonalisation and its optimiser, without a GPU, and the workspace query's arithmetic."""
import ctypes

import pytest
import torch

ABC = (3.4445, -4.7750, 2.0315)


@pytest.fixture(scope="module")
def lib_():
    import __graft_entry__ as g

    g.build()
    from taming_event_flow_amd import _lib

    return _lib


def test_python_refusals(lib_, monkeypatch):
    from taming_event_flow_amd import optim

    f, u = optim.orthogonalize, torch.zeros(4, 6)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        f(u)
    for kw in (dict(steps=0), dict(steps=33), dict(steps=2.5), dict(eps=0.0), dict(eps=-1.0), dict(eps=float("nan")), dict(coefficients=(1.0, 2.0)),
               dict(coefficients=(1.0, 2.0, float("inf")))):
        with pytest.raises(ValueError):
            f(u, **kw)
    monkeypatch.setattr(optim._lib, "require_device_tensor", lambda t, name: t)
    monkeypatch.setattr(optim._lib, "lib", lambda: pytest.fail("not refused"))
    for bad, error in ((u.double(), TypeError), (u.long(), TypeError), (u[0], ValueError), ([u, u.half()], ValueError),
                       ([u, torch.zeros(2, 2, device="meta")], ValueError)):
        with pytest.raises(error):
            f(bad)


def test_optimiser_refusals(lib_):
    from taming_event_flow_amd import optim, parallel

    bucket = parallel.FlatGradBucket([torch.nn.Parameter(torch.zeros(4, 6))])
    for kw in (dict(adjust_lr="x"), dict(momentum=1.0), dict(momentum=-0.1), dict(weight_decay=-1.0), dict(lr=float("nan")), dict(steps=0),
               dict(coefficients=(9.0, 0.0, 0.0, 1.0)), dict(eps=0.0)):
        with pytest.raises(ValueError):
            optim.FusedMuon(bucket, **dict(dict(lr=0.1), **kw))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        optim.FusedMuon(bucket, 0.1)
    with pytest.raises(TypeError):
        optim.FusedMuon(parallel.FlatGradBucket([torch.nn.Parameter(torch.zeros(4, 6).double())]), 0.1)


def test_c_refusals(lib_):
    lib = lib_.lib()
    buf = ctypes.create_string_buffer(1024)
    p = (ctypes.addressof(buf) + 255) & ~255      # (never dereferenced: every call below is refused before a launch)
    good = dict(src=p, dst=p, rows=4, cols=6, src_ld=6, dst_ld=6, batch=1, src_stride=24, dst_stride=24)

    def mats(**kw):
        return (lib_.OrthoMatrix * 1)(lib_.OrthoMatrix(**dict(good, **kw)))

    need = lib.tef_orthogonalize_workspace_bytes(mats(), 1)
    assert need > 0

    def call(m=None, n=1, dtype=0, steps=5, abc=ABC, eps=1e-7, ws=p, nbytes=need):
        return lib.tef_orthogonalize(mats() if m is None else m, n, dtype, steps, *abc, eps, ws, nbytes, None)

    for kw in (dict(rows=0), dict(cols=0), dict(batch=0), dict(rows=-1), dict(src_ld=5), dict(dst_ld=5), dict(rows=2 ** 16, cols=2 ** 16),
               dict(cols=2 ** 25, src_ld=2 ** 25, dst_ld=2 ** 25)):
        assert lib.tef_orthogonalize_workspace_bytes(mats(**kw), 1) == 0, kw
        assert call(mats(**kw)) == -1, kw
    assert call(mats(src=None)) == -1 and call(mats(dst=None)) == -1
    assert call(n=-1) == -1 and call(dtype=3) == -1 and call(dtype=-1) == -1
    assert call(steps=0) == -1 and call(steps=33) == -1 and call(eps=0.0) == -1 and call(eps=1e-300) == -1 and call(eps=float("nan")) == -1
    for abc in ((float("nan"), 0, 0), (16.0, 0, 0), (4.0, 0.0, 0.0), (0.0, 0.0, 5.0), (-20.0, 0.0, 0.0)):
        assert call(abc=abc) == -1, abc
        assert b"coefficients" in lib.tef_last_error()
    assert call(nbytes=need - 1) == -2 and call(ws=None) == -2 and call(ws=p + 16) == -2
    assert call(n=0) == 0      # nothing to do, nothing launched
    bm = (lib_.MuonMatrix * 1)(lib_.MuonMatrix(0, 4, 6, 1.0))
    bv = (lib_.MuonVector * 1)(lib_.MuonVector(24, 3))
    mneed = lib.tef_muon_workspace_bytes(bm, 1)
    assert mneed > 0

    def muon(m=bm, nm=1, v=bv, nv=1, ptr=p, vptr=p, ws=p, nbytes=mneed, steps=5):
        return lib.tef_muon_step(ptr, p, p, vptr, m, nm, v, nv, p, p, p, 1, steps, *ABC, 1e-7, ws, nbytes, None)

    assert muon(ptr=None) == -1 and muon(vptr=None) == -1 and muon(nv=-1) == -1 and muon(steps=0) == -1 and muon(nm=-1) == -1
    assert muon(v=(lib_.MuonVector * 1)(lib_.MuonVector(0, 0))) == -1 and muon(v=(lib_.MuonVector * 1)(lib_.MuonVector(-1, 3))) == -1
    assert muon(m=(lib_.MuonMatrix * 1)(lib_.MuonMatrix(-4, 4, 6, 1.0))) == -1
    assert muon(nbytes=mneed - 1) == -2 and muon(ws=None) == -2


def test_workspace_of_many_matrices(lib_):
    """The list is worked through in groups: the workspace is the largest group's, not the sum."""
    lib = lib_.lib()
    one = lib_.OrthoMatrix(1, 1, 80, 80, 80, 80, 1, 0, 0)
    size = lambda n: lib.tef_orthogonalize_workspace_bytes((lib_.OrthoMatrix * n)(*[one] * n), n)  # noqa: E731
    assert size(1) < size(64) == size(128) == size(1000)
    big = lib_.OrthoMatrix(1, 1, 2 ** 15, 2 ** 17, 2 ** 17, 2 ** 17, 1, 0, 0)
    assert lib.tef_orthogonalize_workspace_bytes((lib_.OrthoMatrix * 1)(big), 1) > 2 * 4 * 2 ** 32      # 64-bit sizes
    small = lib_.OrthoMatrix(1, 1, 64, 320, 320, 320, 1 << 20, 0, 0)      # one workgroup each: nothing in memory
    assert lib.tef_orthogonalize_workspace_bytes((lib_.OrthoMatrix * 1)(small), 1) == 256
