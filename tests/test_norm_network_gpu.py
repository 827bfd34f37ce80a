"""The layer-normalised network end to end: two recurrent passes, flows and every gradient against the same network written out in 64 bits on the
CPU, and against differences of it.

Tolerance: 1e-4 of a tensor's norm, the package's bar for the network: a chain of some thirty convolutions of up to 1152 products summed in
fp32 (2^-24 sqrt(1152) = 2e-6 each, independent) whose errors the normalisations rescale with the features."""
import copy

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available()
    import __graft_entry__ as g

    g.build()
    return torch.device("cuda:0")


def conv(c, x, stride=1):
    return F.conv2d(x, c.weight, c.bias, stride=stride, padding=c.kernel_size[0] // 2)


def norm(m, x):
    mean = x.mean(1, keepdim=True)
    var = ((x - mean) ** 2).mean(1, keepdim=True)
    v = [1, -1, 1, 1]
    return (x - mean) / (var + m.eps).sqrt() * m.weight.view(v) + m.bias.view(v)


def up(x, s):
    return F.interpolate(x, scale_factor=s, mode="bilinear", align_corners=False)


def network64(arch, x, states):
    feats, new = [], []
    for enc, prev in zip(arch.encoders, states):
        x = torch.relu(norm(enc.conv.norm_layer, conv(enc.conv.conv2d, x, 2)))
        g = enc.recurrent_block
        prev = torch.zeros_like(x) if prev is None else prev
        z = torch.sigmoid(conv(g.update_gate, torch.cat([x, prev], 1)))
        r = torch.sigmoid(conv(g.reset_gate, torch.cat([x, prev], 1)))
        o = torch.tanh(conv(g.out_gate, torch.cat([x, prev * r], 1)))
        x = prev * (1 - z) + o * z
        new.append(x)
        feats.append(x)
    for rb in arch.resblocks:
        y = torch.relu(norm(rb.norm1, conv(rb.conv1, x)))
        x = torch.relu(norm(rb.norm2, conv(rb.conv2, y)) + x)
    flows, pred = [], None
    for k, (dec, head) in enumerate(zip(arch.decoders, arch.preds)):
        x = up(x + feats[-1 - k], 2)
        if pred is not None:
            x = torch.cat([up(pred, 2), x], 1)
        x = torch.relu(norm(dec.norm_layer, conv(dec.conv2d, x)))
        pred = conv(head.conv2d, x)
        if head.activation is not None:
            pred = getattr(torch, head.activation)(pred)
        s = 2 ** (len(arch.encoders) - 1 - k)
        flows.append(s * up(pred, s) if s > 1 else pred)
    return flows, new


def test_flows_and_gradients(dev):
    from taming_event_flow_amd.models.model import RecEVFlowNet

    torch.manual_seed(0)
    net = RecEVFlowNet({"name": "RecEVFlowNet", "base_channels": 8, "norm": "LN"}, 2)
    with torch.no_grad():
        for n, p in net.named_parameters():
            if "norm" in n:
                p.add_(0.2 * torch.randn_like(p))
    twin = copy.deepcopy(net).double()
    net = net.to(dev)
    xs = [torch.randn(2, 2, 32, 48) for _ in range(2)]
    ws = [[torch.randn(2, 2, 32, 48) for _ in range(4)] for _ in range(2)]
    got, total = [], 0.0
    for x, w in zip(xs, ws):
        flows = net(x.to(dev))["flow"]
        got.append(flows)
        total = total + sum((f * v.to(dev)).sum() for f, v in zip(flows, w))
    total.backward()

    def loss64():
        states, out, want = [None] * 4, 0.0, []
        for x, w in zip(xs, ws):
            flows, states = network64(twin.arch, x.double(), states)
            want.append(flows)
            out = out + sum((f * v.double()).sum() for f, v in zip(flows, w))
        return out, want

    ref, want = loss64()
    ref.backward()
    for a, b in zip(got, want):
        for f, g in zip(a, b):
            assert (f.detach().double().cpu() - g.detach()).norm() <= 1e-4 * g.detach().norm()
    for (n, p), q in zip(net.named_parameters(), twin.parameters()):
        assert (p.grad.double().cpu() - q.grad).norm() <= 1e-4 * q.grad.norm() + 1e-7, n
    gen = torch.Generator().manual_seed(3)
    for kind in ("norm", "conv2d.weight", "recurrent_block", "bias"):      # a direction in the parameters of one kind
        dirs = [torch.randn(q.shape, generator=gen, dtype=torch.float64) if kind in n else None for n, q in twin.named_parameters()]
        h, ends = 1e-7, []
        for sign in (1, -1):
            with torch.no_grad():
                for q, v in zip(twin.parameters(), dirs):
                    if v is not None:
                        q.add_(sign * h * v)
                ends.append(loss64()[0].item())
                for q, v in zip(twin.parameters(), dirs):
                    if v is not None:
                        q.sub_(sign * h * v)
        terms = [(p.grad.double().cpu() * v) for p, v in zip(net.parameters(), dirs) if v is not None]
        slope, size = sum(t.sum().item() for t in terms), sum(t.norm().item() for t in terms)
        # rounding of the two losses, 2^-52 |loss| / h, and the gradient's bar along a random direction
        assert abs((ends[0] - ends[1]) / (2 * h) - slope) <= 2.0 ** -50 * abs(ref.item()) / h + 1e-3 * size, kind
