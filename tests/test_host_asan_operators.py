"""tests/asan/operators_driver.py: the host side of the normalisation and orthogonalisation under AddressSanitizer and UBSan, without a GPU."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

pytestmark = pytest.mark.skipif(shutil.which("hipcc") is None, reason="needs hipcc to build the instrumented library")


def test_operators_clean_under_asan_ubsan():
    env = {k: v for k, v in os.environ.items() if k not in ("TEF_HIP_LIB", "LD_PRELOAD")}
    r = subprocess.run([os.path.join(ROOT, "tests", "asan", "run_host_asan.sh")], env=dict(env, TEF_ASAN_DRIVER="operators_driver"), capture_output=True,
                       text=True, timeout=1500)
    out = r.stdout + r.stderr
    assert r.returncode == 0 and "HOST SANITIZER RUN CLEAN (operators)" in out, out[-3000:]
    assert "AddressSanitizer" not in out and "runtime error" not in out, out[-3000:]
