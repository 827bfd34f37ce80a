"""What has ended a process on this stack before does not run, whatever is asked for."""
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_graph_destruction_diagnostic_has_no_switch(monkeypatch):
    """Asked for by its old switch, the test that destroys captured multi-stream graphs is still skipped (seen on the collected item:
    nothing is run)."""
    code = ("import sys, pytest\n"
            "class P:\n"
            "    def pytest_collection_finish(self, session):\n"
            "        for i in session.items:\n"
            "            print('ITEM', i.name, [m.name for m in i.iter_markers()][:1])\n"
            "sys.exit(pytest.main(['--collect-only', '-q', 'tests/test_train_gpu.py', '-k', 'destroying_retired'], plugins=[P()]))\n")
    env = dict(os.environ, TEF_RUN_DESTROY_DIAGNOSTIC="1")
    out = subprocess.run([sys.executable, "-c", code], cwd=ROOT, env=env, capture_output=True, text=True, timeout=300)
    assert "ITEM test_destroying_retired_graphs_diagnostic ['skip']" in out.stdout, out.stdout + out.stderr
