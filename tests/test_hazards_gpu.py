"""Calls that have ended the process on this stack, refused on the host before anything reaches the device."""
import copy

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available()
    import __graft_entry__ as g

    g.build()
    return torch.device("cuda:0")


@pytest.mark.parametrize("norm", [None, "LN"])
def test_capture_after_eager_outputs(dev, norm):
    """Flows of an eager pass still held: refused, and the trainer is as it was.  Dropped: captured and replayed."""
    from taming_event_flow_amd import train

    cfg = copy.deepcopy(train.DEFAULT_CONFIG)
    cfg["data"]["passes_loss"] = 2
    cfg["loader"].update(batch_size=1, resolution=[32, 32], max_num_grad_events=200)
    cfg["model"].update(base_channels=8, norm=norm)
    torch.manual_seed(0)
    tr = train.Trainer(cfg, dev)
    src = train.SyntheticSequences(cfg, dev, 300, seq_len=10 ** 9)
    batches = [src.next() for _ in range(2)]
    tr.reset()
    flows = tr.model(batches[0]["net_input"])["flow"]
    before = [p.detach().clone() for p in tr.model.parameters()]
    with pytest.raises(RuntimeError, match="autograd graph over"):
        tr.capture_window(batches, warmup=1)
    assert all(torch.equal(p.detach(), b) for p, b in zip(tr.model.parameters(), before))
    del flows
    tr.reset()      # (the pass's recurrent states)
    win = tr.capture_window(batches, warmup=1)
    win()
    assert torch.isfinite(tr.last_loss).item()
    win.close()
    tr.close()
