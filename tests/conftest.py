import os
import sys

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)

GOLDEN = os.path.join(ROOT, "tests", "golden")


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a real MI355X (run with -m gpu on the GPU box)")


# Never run, whatever their own conditions say: destroying captured multi-stream graphs has ended the interpreter on this stack.
NEVER = {"test_destroying_retired_graphs_diagnostic": "destroying captured multi-stream graphs has taken the interpreter down on this stack"}


def pytest_collection_modifyitems(items):
    for item in items:
        reason = NEVER.get(getattr(item, "originalname", item.name))
        if reason:
            item.add_marker(pytest.mark.skip(reason=reason), append=False)


# (Rounds 3-4 had an autouse fixture here that ran gc.collect() + torch.cuda.synchronize() after every test: it hid an
# intermittent corruption whose cause round 4 found — destroying a captured multi-stream hipGraph leaves late device-side
# writes behind, which land in whatever the freed memory has become.  train.CapturedWindow.close() now
# waits for the device AFTER its graphs are gone, Trainer / CapturedWindow are released by reference count (no cycles) and
# tests/test_train_gpu.py::test_graph_teardown_leaves_no_late_writes holds the line; the fixture is gone.)


def load_case(name):
    """Load a golden loss case -> (meta dict, window lists, loss, dflows)."""
    import json

    z = np.load(os.path.join(GOLDEN, name + ".npz"))
    meta = json.loads(str(z["meta"]))
    P, F = meta["P"], meta["F"]
    if meta.get("seeded"):      # inputs regenerated from the seed (tests/golden/make_golden.py::save_seeded_case)
        import hashlib

        from taming_event_flow_amd import synth

        rng = np.random.default_rng(meta["seed"])
        win = synth.make_window(rng, meta["B"], meta["H"], meta["W"], P, F, meta["n_grad"], meta["n_det"], meta["sigma"],
                                "smooth", True, True)
        h = hashlib.sha256()
        for t in range(P):
            for f in win["flows"][t]:
                h.update(np.ascontiguousarray(f).tobytes())
            for k in ("ev", "pm", "dev", "dpm"):
                h.update(np.ascontiguousarray(win[k][t]).tobytes())
        assert h.hexdigest() == meta["digest"], "regenerated inputs differ from the ones the reference was run on"
        return meta, win, np.float32(z["loss"]), z["dflows"]
    win = {
        "flows": [[z["flows"][t, i] for i in range(F)] for t in range(P)],
        "ev": [z[f"ev{t}"] for t in range(P)],
        "pm": [z[f"pm{t}"] for t in range(P)],
        "dev": [z[f"dev{t}"] for t in range(P)],
        "dpm": [z[f"dpm{t}"] for t in range(P)],
    }
    return meta, win, np.float32(z["loss"]), z["dflows"]


ITERATIVE_CASES = [
    "it_two_s1_p6", "it_one_s1_p4", "it_two_s2_p8", "it_two_s3_p8", "it_two_s1_p10_f4", "it_two_iid",
    "it_two_zero_flow", "it_two_smooth_terms", "it_two_round_ts", "it_two_float_xy", "it_two_p5_odd", "it_two_unscaled",
    "it_two_nocomp", "it_one_nocomp_s2",      # border_compensation=False (set after construction, as the reference allows)
    # passes_loss not a multiple of 2^(scales_loss - 1): trailing passes outside every window of the finer scales
    "it_two_p10_s3", "it_two_nocomp_p10_s3", "it_two_nocomp_p5_s2",
]
LINEAR_CASES = ["lin_s1_p6", "lin_s2_p8", "lin_smooth_terms", "lin_zero_flow", "lin_unscaled", "lin_nocomp_s2",
                "lin_nocomp_p5_s2", "lin_p10_s3"]
FULL_RES_CASES = ["it_two_128_p10", "lin_128_p10"]      # BASELINE resolution, inputs regenerated from a seed
# the exact windows bench.py times (B = 8, F = 4, P = 10, 10 000 events), run through the reference
BENCH_WINDOW_CASES = ["bench_window_0", "bench_window_1"]


def load_bench_window(name):
    """A reference-recorded bench window (tests/golden/make_golden.py::save_bench_window) -> (meta, window, golden
    arrays).  The inputs are regenerated exactly as bench.py makes them and checked against the recorded digest."""
    import hashlib
    import json

    from taming_event_flow_amd import synth

    z = np.load(os.path.join(GOLDEN, name + ".npz"))
    meta = json.loads(str(z["meta"]))
    rng = np.random.default_rng(meta["seed"])
    win = synth.make_window(rng, meta["B"], meta["H"], meta["W"], meta["P"], meta["F"], meta["n_grad"], meta["n_det"],
                            sigma=meta["sigma"], kind="smooth")
    h = hashlib.sha256()
    for t in range(meta["P"]):
        for f in win["flows"][t]:
            h.update(np.ascontiguousarray(f).tobytes())
        for k in ("ev", "pm", "dev", "dpm"):
            h.update(np.ascontiguousarray(win[k][t]).tobytes())
    assert h.hexdigest() == meta["digest"], "regenerated inputs differ from the ones the reference was run on"
    return meta, win, {k: z[k] for k in z.files if k != "meta"}


def check_bench_window(meta, gold, loss, g, tol, lattice_tol=None):
    """loss and d loss / d flow [P, F, B, 2, H, W] of a bench window against what the reference recorded: the loss, the
    stride-s lattice of the gradient in max-norm (globally and per map), and per map the float64 sum / sum of squares
    over ALL pixels relative to the map's sum of magnitudes (covers the pixels the lattice skips)."""
    s = meta["stride"]
    assert abs(loss - float(gold["loss"])) <= tol * abs(float(gold["loss"])), (loss, float(gold["loss"]))
    lat = g[..., ::s, ::s]
    ref = gold["dflows_lattice"]
    assert lat.shape == ref.shape
    e_lat = rel_err(lat, ref)
    assert e_lat <= (lattice_tol or tol), e_lat
    gmax = gold["dflows_max"]                                  # [P, F, B, 2] max |g| of every map over ALL its pixels
    e_map = float((np.abs(lat.astype(np.float64) - ref).max(axis=(-1, -2)) / np.maximum(gmax, 1e-30)).max())
    assert e_map <= 20 * tol, e_map
    g64 = g.astype(np.float64)
    e_sum = float((np.abs(g64.sum(axis=(-1, -2)) - gold["dflows_sum"]) / gold["dflows_abs_sum"]).max())
    e_abs = float((np.abs(np.abs(g64).sum(axis=(-1, -2)) - gold["dflows_abs_sum"]) / gold["dflows_abs_sum"]).max())
    e_sq = float((np.abs((g64 * g64).sum(axis=(-1, -2)) - gold["dflows_sq_sum"]) / gold["dflows_sq_sum"]).max())
    e_max = float((np.abs(np.abs(g).max(axis=(-1, -2)) - gmax) / gmax).max())
    assert e_sum <= tol and e_abs <= tol and e_sq <= 2 * tol and e_max <= 20 * tol, (e_sum, e_abs, e_sq, e_max)
    return dict(loss=abs(loss - float(gold["loss"])) / abs(float(gold["loss"])), lattice=e_lat, per_map=e_map, sum=e_sum,
                abs_sum=e_abs, sq_sum=e_sq, max=e_max)


def rel_err(a, b):
    """max-norm relative error of arrays (or scalars)."""
    a = np.asarray(a, np.float64)
    b = np.asarray(b, np.float64)
    return float(np.abs(a - b).max() / max(np.abs(b).max(), 1e-30))


def elementwise_error(a, b, rtol=1e-4, floor=1e-6):
    """Element-wise parity of two flow-gradient arrays in its plain form: max over the elements of
    |a - b| / (rtol * |b| + floor * max|b|) and where it is attained -> (error, index, a[index], b[index]); parity holds
    when error <= 1: every pixel within 1e-4 of ITS OWN reference value, with a floor of 1e-6 of the largest gradient for
    pixels that are (nearly) zero.  (Rounds 1-3 held pixels to 1e-4 x a builder-defined "gradient mass" instead, because
    neither the oracle nor the HIP path could meet this form: their bilinear lookups differed from ATen's by an ulp in a
    third of the cases and the backward used the closed form 2 A (tau - A) / (C + eps) where autograd forms dC + dT * tau.
    With both fixed in round 4 the oracle meets it 40-fold and the HIP path on every recorded case.)"""
    a = np.asarray(a, np.float64)
    b = np.asarray(b, np.float64)
    r = np.abs(a - b) / (rtol * np.abs(b) + floor * np.abs(b).max() + 1e-300)
    i = np.unravel_index(int(r.argmax()), r.shape)
    return float(r[i]), tuple(int(v) for v in i), float(a[i]), float(b[i])


@pytest.fixture(scope="session")
def golden_dir():
    return GOLDEN
