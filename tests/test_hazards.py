"""What has ended a process on this stack before does not run, whatever is asked for."""
import os
import subprocess
import sys
from types import SimpleNamespace

import pytest
import torch

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


def test_capture_refused_while_an_eager_graph_is_alive():
    """Trainer.capture_window's first check, on the CPU: outputs of an eager pass that somebody still holds, then dropped."""
    from taming_event_flow_amd import train

    net = torch.nn.Sequential(torch.nn.Linear(3, 4), torch.nn.LayerNorm(4))
    net[0].bias.requires_grad_(False)
    assert train._held_by_a_graph(net.parameters()) == []
    y = net(torch.ones(2, 3)).sum()
    assert len(train._held_by_a_graph(net.parameters())) == len(train._held_by_a_graph(net.parameters())) == 3
    y.backward()
    tr = train.Trainer.__new__(train.Trainer)
    tr.cfg = {"data": {"passes_loss": 1}, "loss": {}}
    tr.loss_function, tr._win_inputs, tr._parked, tr.model, tr.optimizer, tr.device = SimpleNamespace(num_passes=0), [], {}, net, None, "cpu"
    tr.dec_stream = tr.wgrad_stream = tr.comm_stream = tr._dp_split = None
    tr.deferred_wgrad, tr.window_decode = False, False
    with pytest.raises(RuntimeError, match="autograd graph over 3 of the model's parameters"):
        tr.capture_window([{}])
    view = net[0].weight.view(-1)      # a view refers to its base's accumulator as well
    del y
    assert len(train._held_by_a_graph(net.parameters())) == 1
    del view
    assert train._held_by_a_graph(net.parameters()) == []
