"""The 8-bit checkpoints and the recurrence as they are used: NeRF trained on packed activations, and a feature field composited along rays.

References run in float64 on the CPU with the formula's weight gradient, dy^T q(x).  The kernels' fp32 activations differ from them by some d, and
where x lies within d of a rounding border its code may fall on either side: a weight gradient may therefore differ by
|dy|^T (|q(x + d) - q(x - d)|), and by fp32 rounding.  d = 2^-16 of a row's largest magnitude: 256 u, for layers of at most 454 products whose errors
add up like their square root."""
import pytest
import torch

from act8_definition import quantised

pytestmark = pytest.mark.gpu
D = 2.0 ** -16


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    return torch.device("cuda:0")


class QLinear(torch.autograd.Function):
    """x W^T + b with dW = dy^T q(x); notes (weight, |dy|^T (border term + D of everything)) in `notes`."""

    @staticmethod
    def forward(ctx, x, w, b, notes):
        ctx.save_for_backward(x, w)
        ctx.notes = notes
        return x @ w.t() + b

    @staticmethod
    def backward(ctx, g):
        x, w = ctx.saved_tensors
        d = D * x.abs().amax(1, keepdim=True)
        border = (quantised(x + d) - quantised(x - d)).abs()
        ctx.notes.append((w.shape, g.abs().t() @ (border + 16 * d + D * x.abs()), g.abs().sum(0)))
        return g @ w, g.t() @ quantised(x), g.sum(0), None


def test_nerf_trains_on_packed_activations(dev):
    from neurofluid_amd.nerf import NeRF
    torch.manual_seed(0)
    ref = NeRF(in_channels_xyz=198, in_channels_dir=54)
    net = NeRF(in_channels_xyz=198, in_channels_dir=54, act_checkpoint="e4m3")
    net.load_state_dict(ref.state_dict(), strict=True)
    net, ref = net.to(dev), ref.to(dev)
    g = torch.Generator().manual_seed(1)
    for n in (200, 33, 1):
        x, gy = torch.randn(n, 252, generator=g), torch.randn(n, 4, generator=g)
        grads = {}
        for name, m in (("e4m3", net), ("fp32", ref)):
            xd = x.to(dev).requires_grad_()
            out = m(xd)
            ps = [l.weight for l in m.linear_layers()] + [l.bias for l in m.linear_layers()]
            grads[name] = (out.detach().cpu(), [q.cpu().double() for q in torch.autograd.grad(out, [xd] + ps, gy.to(dev))])
        assert (grads["e4m3"][0] - grads["fp32"][0]).abs().max() <= 2e-6 * max(1.0, float(grads["fp32"][0].abs().max()))
        # the reference: the network of models/nerf.py:83-124 in float64
        ls = net.linear_layers()
        W = [l.weight.detach().cpu().double().requires_grad_() for l in ls]
        B = [l.bias.detach().cpu().double().requires_grad_() for l in ls]
        notes = []
        x64 = x.double().requires_grad_()
        px, pd = x64[:, :198], x64[:, 198:]
        hh = px
        lin = lambda i, v: QLinear.apply(v, W[i], B[i], notes)

        def split(i, a, b):          # layers of two inputs, each with its own scales: two products
            k = a.shape[1]
            wa, wb = W[i][:, :k], W[i][:, k:]
            return QLinear.apply(a, wa, B[i], notes) + QLinear.apply(b, wb, torch.zeros_like(B[i]), notes)
        for i in range(8):
            hh = torch.relu(split(i, px, hh) if i == 4 else lin(i, hh))
        sigma = lin(10, hh)
        view = torch.relu(split(9, lin(8, hh), pd))
        out = torch.cat([torch.sigmoid(lin(11, view)), sigma], 1)
        assert (grads["e4m3"][0].double() - out.detach()).abs().max() <= 1e-4
        want = torch.autograd.grad(out, [x64] + W + B, gy.double())
        slack = {}
        for shape, wb, bb in notes:
            slack.setdefault(tuple(shape), []).append((wb, bb))
        got = grads["e4m3"][1]
        rel = lambda a, b: float((a - b).norm() / b.norm())
        assert rel(got[0], want[0]) <= 1e-4                     # dL/dx does not see the 8 bits
        for i in range(12):
            shape = tuple(W[i].shape)
            if i in (4, 9):
                k = 198 if i == 4 else 256
                parts = [max(float(s[0].max()) for s in slack[(shape[0], c)]) for c in (k, shape[1] - k)]
                bound = torch.cat([torch.full((shape[0], c), p).double() for c, p in zip((k, shape[1] - k), parts)], 1)
            else:
                bound = torch.full(shape, max(float(s[0].max()) for s in slack[shape])).double()
            assert ((got[1 + i] - want[1 + i]).abs() <= bound).all(), i
            assert rel(got[1 + i], want[1 + i]) <= 5e-3, (i, rel(got[1 + i], want[1 + i]))           # (a wrong layer or column is off by 1)
            assert rel(got[13 + i], want[13 + i]) <= 1e-4, i
            # against the exact weight gradient: a code is off by at most 1/16, independently from row to row
            assert rel(got[1 + i], grads["fp32"][1][1 + i]) <= 1 / 16, i
    # density only, no rows, and what is kept
    x = torch.randn(50, 198, generator=g).to(dev).requires_grad_()
    for m in (net, ref):
        m.zero_grad()
        m(x, sigma_only=True).sum().backward()
    assert net.xyz_encoding_final.weight.grad is None and net.rgb[0].weight.grad is None
    a, b = net.xyz_encoding_3[0].weight.grad, ref.xyz_encoding_3[0].weight.grad
    assert (a - b).norm() <= b.norm() / 16
    z = torch.zeros(0, 252, device=dev, requires_grad=True)
    net.zero_grad()
    net(z).sum().backward()
    assert not net.sigma.weight.grad.any() and z.grad.shape == (0, 252)


def test_nerf_keeps_less(dev):
    from neurofluid_amd.nerf import NeRF
    kept = []

    def requested():         # (what memory_allocated counts depends on the free blocks that earlier tests left: up to 1 MB more a tensor)
        return torch.cuda.memory_stats()["requested_bytes.all.current"]
    for ck in (None, "e4m3"):
        net = NeRF(in_channels_xyz=198, in_channels_dir=54, act_checkpoint=ck).to(dev)
        x = torch.randn(40000, 252, device=dev)
        out = net(x[:64])
        del out
        torch.cuda.synchronize()
        before = requested()
        out = net(x)
        kept.append((requested() - before) / 40000)
        del out
    # 2432 + 252 floats a row, against codes and scales of 2432 + 224 + 64 features (2 805 B), ten mask words of four waves x 64 lanes a
    # 32-row tile (320 B), output and index (20 B); either way two weight blobs of 0.67 M floats and three weights of 0.21 M: 155 B a row of 40 000
    assert kept[0] > 4 * (2432 + 252) and kept[1] < 2805 + 320 + 20 + 160 + 20, kept


def test_nerf_frees_what_it_kept(dev):
    """A loss that is still held after its backward holds none of the packed activations."""
    from neurofluid_amd.nerf import NeRF
    net = NeRF(in_channels_xyz=198, in_channels_dir=54, act_checkpoint="e4m3").to(dev)
    x = torch.randn(20000, 252, device=dev)
    net(x).sum().backward()
    before = torch.cuda.memory_allocated()
    loss = net(x).sum()
    assert torch.cuda.memory_allocated() - before >= 20000 * 2432
    loss.backward()
    assert torch.cuda.memory_allocated() - before < 20000 * 2432 // 4


def test_feature_field_along_rays(dev):
    """Rows of a small field (linear layers on 8-bit checkpoints) composited along rays by the recurrence, loss, all gradients."""
    from neurofluid_amd import act8, scan
    g = torch.Generator().manual_seed(5)
    R, S, F, H, C = 40, 24, 36, 64, 8
    x, target = torch.randn(R * S, F, generator=g), torch.randn(R, C, generator=g)
    shapes = [(H, F), (H, H), (C + 1, H)]
    ws = [torch.randn(*s, generator=g) / s[1] ** 0.5 for s in shapes]
    bs = [torch.randn(s[0], generator=g) * 0.1 for s in shapes]
    delta = torch.rand(R, S, 1, generator=g) * 0.2

    def render(out, delta, comp):
        out = out.view(R, S, C + 1)
        lg = -torch.relu(out[..., :1]) * delta
        return comp(lg, -torch.expm1(lg) * torch.tanh(out[..., 1:]))

    def on_gpu():
        ps = [p.to(dev).requires_grad_() for p in ws + bs]
        xd = x.to(dev).requires_grad_()
        h = xd
        for i in range(3):
            h = act8.linear(h, ps[i], ps[3 + i])
            if i < 2:
                h = torch.relu(h)
        img = render(h, delta.to(dev), lambda lg, f: scan.gated_scan(lg, f, log_gate=True, reverse=True)[1])
        loss = ((img - target.to(dev)) ** 2).sum()
        return img.detach(), torch.autograd.grad(loss, [xd] + ps)

    img, grads = on_gpu()
    img2, grads2 = on_gpu()
    assert torch.equal(img, img2) and all(torch.equal(a, b) for a, b in zip(grads, grads2))
    notes = []
    ps = [p.double().requires_grad_() for p in ws + bs]
    x64 = x.double().requires_grad_()
    h = x64
    for i in range(3):
        h = QLinear.apply(h, ps[i], ps[3 + i], notes)
        if i < 2:
            h = torch.relu(h)

    def comp(lg, f):
        s = torch.zeros(R, C).double()
        for t in range(S - 1, -1, -1):
            s = torch.exp(lg[:, t]) * s + f[:, t]
        return s
    want_img = render(h, delta.double(), comp)
    want = torch.autograd.grad(((want_img - target.double()) ** 2).sum(), [x64] + ps)
    assert (img.cpu().double() - want_img.detach()).abs().max() <= 1e-5
    rel = lambda a, b: float((a.cpu().double() - b).norm() / b.norm())
    assert rel(grads[0], want[0]) <= 1e-4
    for i in range(3):
        bound = notes[2 - i][1]                    # (the backward met the layers from the last to the first)
        assert ((grads[1 + i].cpu().double() - want[1 + i]).abs() <= bound).all(), i
        assert rel(grads[4 + i], want[4 + i]) <= 1e-4


def test_what_is_saved_may_leave_the_gpu_in_between(dev):
    """Saved tensors that autograd's hooks keep in host memory, and passes that are run again for the backward, give the same gradients."""
    from torch.utils.checkpoint import checkpoint
    from neurofluid_amd import act8, scan
    g = torch.Generator().manual_seed(31)
    x, w, b = torch.randn(600, 20, generator=g), torch.randn(16, 20, generator=g), torch.randn(16, generator=g)
    h0, rs = torch.randn(3, 16, generator=g), torch.tensor([0, 250, 250, 590])
    lg = -torch.rand(600, 17, generator=g)[:, 1:]              # (rows of 17: read one by one)

    def run(how):
        ins = [q.to(dev).requires_grad_() for q in (x, w, b, h0)]
        gate = torch.empty(600, 17, device=dev)[:, 1:].copy_(lg).detach().requires_grad_()

        def f(x, w, b, h0, gate):
            y = act8.linear(x, w, b)
            h, last = scan.gated_scan(gate, y, h0, log_gate=True, row_splits=rs.to(dev))
            z, _ = scan.gated_scan(gate.view(1, 600, 16) if gate.is_contiguous() else gate[None], h[None], log_gate=True, reverse=True)
            return z.square().sum() + last.square().sum()
        if how == "host":
            with torch.autograd.graph.save_on_cpu():
                loss = f(*ins, gate)
        elif how == "again":
            loss = checkpoint(f, *ins, gate, use_reentrant=False)
        else:
            loss = f(*ins, gate)
        return torch.autograd.grad(loss, ins + [gate])
    want = run("")
    assert all(q.abs().sum() > 0 for q in want)
    for how in ("host", "again"):
        assert all(torch.equal(a, b) for a, b in zip(run(how), want)), how
