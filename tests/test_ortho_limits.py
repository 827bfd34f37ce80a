"""Calls that are too large are refused by the workspace query, before any part of a list has been worked on."""
import ctypes

import pytest

ABC = (3.4445, -4.7750, 2.0315)


@pytest.fixture(scope="module")
def lib_():
    import __graft_entry__ as g

    g.build()
    from taming_event_flow_amd import _lib

    return _lib


def test_tiles_of_a_launch(lib_):
    lib = lib_.lib()
    fine = lib_.OrthoMatrix(1, 1, 65, 65, 65, 65, 1 << 20, 0, 0)
    many = lib_.OrthoMatrix(1, 1, 128, 128, 128, 128, 1 << 20, 0, 0)      # 8 workgroups each to normalise and split: 2^23
    small = lib_.OrthoMatrix(1, 1, 64, 64, 64, 64, 1 << 20, 0, 0)
    assert lib.tef_orthogonalize_workspace_bytes((lib_.OrthoMatrix * 2)(small, fine), 2) > 256
    for bad in ([many], [small, many], [fine] * 70 + [many]):
        arr = (lib_.OrthoMatrix * len(bad))(*bad)
        assert lib.tef_orthogonalize_workspace_bytes(arr, len(bad)) == 0 and b"too many tiles" in lib.tef_last_error()
        # (null workspace: a call that got as far as it would say so; nothing is launched)
        assert lib.tef_orthogonalize(arr, len(bad), 0, 5, *ABC, 1e-7, None, 0, None) == -1


def test_optimiser_list(lib_):
    lib = lib_.lib()
    ok = lib_.MuonMatrix(0, 100, 200, 1.0)
    huge = lib_.MuonMatrix(20000, 2 ** 15, 2 ** 20, 1.0)
    for n in (1, 80):
        arr = (lib_.MuonMatrix * (n + 1))(*[ok] * n, huge)
        assert lib.tef_muon_workspace_bytes(arr, n) > 0
        assert lib.tef_muon_workspace_bytes(arr, n + 1) == 0 and b"too many tiles" in lib.tef_last_error()
        buf = ctypes.create_string_buffer(1024)
        p = (ctypes.addressof(buf) + 255) & ~255
        assert lib.tef_muon_step(p, p, p, None, arr, n + 1, None, 0, p, p, p, 1, 5, *ABC, 1e-7, p, 2 ** 60, None) == -1
