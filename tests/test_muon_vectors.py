"""Which matrices the optimiser leaves to Adam: parameters, or names in a Trainer's config; anything else is an error, not ignored."""
import pytest
import torch


def test_entries_that_are_no_parameters():
    import __graft_entry__ as g

    g.build()
    from taming_event_flow_amd import optim, parallel

    params = [torch.nn.Parameter(torch.zeros(4, 6)), torch.nn.Parameter(torch.zeros(3))]
    bucket = parallel.FlatGradBucket(params)
    for bad in (["preds"], "preds", [torch.nn.Parameter(torch.zeros(4, 6))], [params[0], None]):
        with pytest.raises(ValueError, match="vectors"):
            optim.FusedMuon(bucket, 0.1, vectors=bad)
    with pytest.raises(RuntimeError, match="no CPU fallback"):      # (the next check)
        optim.FusedMuon(bucket, 0.1, vectors=params[:1])


def test_named_tuples_of_matrices(monkeypatch):
    """A named tuple is a tuple: empty matrices need no device."""
    from collections import namedtuple

    from taming_event_flow_amd import optim

    monkeypatch.setattr(optim._lib, "require_device_tensor", lambda t, name: t)
    pair = namedtuple("pair", "a b")(torch.zeros(0, 3), torch.zeros(2, 0))
    got = optim.orthogonalize(pair)
    assert isinstance(got, tuple) and [tuple(t.shape) for t in got] == [(0, 3), (2, 0)]
    assert isinstance(optim.orthogonalize(list(pair)), list)


def test_names_in_a_config():
    from taming_event_flow_amd import train

    net = torch.nn.Module()
    net.arch = torch.nn.Module()
    net.arch.preds = torch.nn.ModuleList([torch.nn.Conv2d(3, 2, 1), torch.nn.Conv2d(4, 2, 1)])
    net.arch.predshead = torch.nn.Linear(2, 2)
    args = lambda **kw: train._muon_arguments(net, dict(name="Muon", lr=0.1, capturable=True, momentum=0.9, **kw))  # noqa: E731
    assert args() == dict(momentum=0.9, vectors=[]) == args(vectors=None)
    got = args(vectors=["arch.preds"])["vectors"]
    assert [id(p) for p in got] == [id(p) for p in net.arch.preds.parameters()]
    got = args(vectors=["arch.preds.1.weight", "arch.predshead"])["vectors"]
    assert [id(p) for p in got] == [id(p) for p in (net.arch.preds[1].weight, net.arch.predshead.weight, net.arch.predshead.bias)]
    net.arch.predshead.bias.requires_grad_(False)      # not trained: in no optimiser
    assert [id(p) for p in args(vectors=["arch.predshead"])["vectors"]] == [id(net.arch.predshead.weight)]
    for bad in (["arch.pred"], ["preds"], ["arch.preds.1.weigh"], "arch.preds"):
        with pytest.raises(ValueError, match="no parameter or module named"):
            args(vectors=bad)
