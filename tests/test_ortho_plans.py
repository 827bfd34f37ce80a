"""Which kernels the cases of the tile tests go through, asked of the library without a device: every one of them, every way a product is cut."""
import ctypes

import pytest
from test_ortho_tiles_gpu import CASES, MUON


@pytest.fixture(scope="module")
def lib_():
    import __graft_entry__ as g

    g.build()
    from taming_event_flow_amd import _lib

    return _lib


def plans(lib_, shapes, optimiser):
    arr = (lib_.OrthoMatrix * len(shapes))(*[lib_.OrthoMatrix(1, 1, r, c, c, c, b, r * c, r * c) for b, r, c in shapes])
    for i in range(len(shapes)):
        p = lib_.OrthoPlan()
        assert lib_.lib().tef_orthogonalize_plan(arr, len(shapes), i, optimiser, ctypes.byref(p)) == 0
        yield p


def kernels(p, dtype, to):
    if p.form == 3:
        deep = lambda n: "deep" if n <= 256 else "wide"  # noqa: E731
        yield f"symmetric {p.gram_tile} {deep(p.gram_items)}"
        if p.gram_joins:
            yield f"join {p.gram_tile}"
        for k in range(2):
            yield f"symmetric {p.chain_tile} {deep(p.chain_items[k])}" if p.chain_tile > 32 else "symmetric 32"
            if p.chain_joins[k]:
                yield f"join {p.chain_tile}"
        yield f"apply {p.apply_tile} to X"
        yield f"apply {p.apply_tile} to {to} {dtype}"


def test_every_tiled_kernel_is_reached(lib_):
    seen = set()
    for shapes, dtype in CASES.values():
        for p in plans(lib_, shapes, 0):
            assert p.form == 3
            seen |= set(kernels(p, dtype, "result"))
    for shapes in MUON.values():
        for (r, c), p in zip(shapes, plans(lib_, [(1, r, c) for r, c in shapes], 1)):
            assert p.form == (0 if min(r, c) <= 8 else 3)
            seen |= set(kernels(p, "f32", "parameters"))
    every = {f"symmetric {t} {d}" for t in (64, 128) for d in ("deep", "wide")} | {"symmetric 32", "join 64", "join 128"}
    every |= {f"apply {t} to X" for t in (64, 128)} | {f"apply {t} to parameters f32" for t in (64, 128)}
    every |= {f"apply {t} to result {d}" for t in (64, 128) for d in ("f32", "bf16", "f16")}
    assert seen == every, (every - seen, seen - every)


def test_cuts(lib_):
    """The ways in which a launch's tiles are cut along k: none, all, the last ones only, pieces of a list."""
    one = lambda *s: next(plans(lib_, [s], 0))  # noqa: E731
    p = one(1, 2048, 2048)      # 136 tiles of 128, all in three pieces; two products: 272, of them the last 16 in eight
    assert (p.gram_tile, p.gram_items, p.gram_joins) == (128, 136 * 3, 136)
    assert (p.chain_tile, p.chain_items[0], p.chain_items[1], p.chain_joins[1]) == (128, 136 * 3, 256 + 16 * 8, 16)
    p = one(3, 256, 4608)       # a batch: 30 tiles of 64 in eight pieces, the short products in 32 x 32 tiles
    assert (p.gram_tile, p.gram_items, p.gram_joins, p.chain_tile, p.apply_tile) == (64, 240, 30, 32, 128)
    p = one(1, 130, 50000)
    assert (p.gram_tile, p.gram_items) == (128, 3 * 64)
    p = list(plans(lib_, [(1, 512, 4608)] * 9, 1))[0]
    assert (p.gram_tile, p.chain_tile, p.apply_tile) == (128, 64, 128) and p.gram_joins == 90 and p.gram_items > 90


def test_forms(lib_):
    for shape, optimiser, form in (((1, 2, 3), 0, 0), ((5, 1024, 8), 0, 0), ((1, 8, 1025), 0, 1), ((1, 9, 9), 0, 2), ((7, 320, 64), 0, 2), ((1, 64, 321), 0, 3),
                                   ((1, 65, 65), 0, 3), ((1, 9, 9), 1, 3), ((1, 8, 9), 1, 0), ((1, 3000, 3), 1, 1)):
        assert next(plans(lib_, [shape], optimiser)).form == form, shape
    # the form is a matrix's own, whatever stands beside it
    assert [p.form for p in plans(lib_, [(1, 2, 3), (1, 500, 500), (1, 40, 40), (1, 3, 9999)] * 40, 0)] == [0, 3, 2, 1] * 40


def test_refusals(lib_):
    lib, p = lib_.lib(), lib_.OrthoPlan()
    arr = (lib_.OrthoMatrix * 1)(lib_.OrthoMatrix(1, 1, 4, 6, 6, 6, 1, 24, 24))
    assert lib.tef_orthogonalize_plan(arr, 1, 1, 0, ctypes.byref(p)) == -1 and lib.tef_orthogonalize_plan(arr, 1, -1, 0, ctypes.byref(p)) == -1
    assert lib.tef_orthogonalize_plan(arr, 1, 0, 0, None) == -1 and lib.tef_orthogonalize_plan(None, 1, 0, 0, ctypes.byref(p)) == -1
    arr[0].rows = 0
    assert lib.tef_orthogonalize_plan(arr, 1, 0, 0, ctypes.byref(p)) == -1
