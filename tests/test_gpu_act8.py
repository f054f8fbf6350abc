"""8-bit activation checkpoints (csrc/nf_act8.hip) against their definition in 64 bits.

Codes have one right value, so unpacked values are compared for equality.  A weight gradient's products are exact (a code's value has four
significant bits, dy 24); its sums are fp32: with n terms, each split into up to three parts, at most 3 n + 64 additions stand between a term and the
result, each off by at most one ulp, 2 u = 2^-23, of a partial sum that the magnitudes' sum S bounds:  |error| <= (3 n + 64) 2^-23 S.  That no part of
dy is lost is tested apart, where sums are exact."""
import pytest
import torch

from act8_definition import quantised

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    return torch.device("cuda:0")


def same(a, b):
    return bool((((a == b) | (torch.isnan(a) & torch.isnan(b)))).all())


@pytest.mark.parametrize("rows", [0, 1, 3, 63, 64, 65, 200])
@pytest.mark.parametrize("K", [1, 7, 8, 31, 32, 33, 100, 128, 252, 300])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_pack_unpack(dev, rows, K, dtype):
    from neurofluid_amd import act8
    g = torch.Generator().manual_seed(rows * 1000 + K)
    x = (torch.randn(rows, K, generator=g) * torch.exp(2 * torch.randn(rows, 1, generator=g))).to(dtype)
    c = act8.pack(x.to(dev))
    assert c.shape == (rows, K) and c.dtype == dtype and c.rows == rows
    want = quantised(x)
    for dt in (F32, BF16):          # both hold every value exactly
        assert same(c.unpack(dt).cpu().double(), want)
    assert same(c.unpack().cpu(), want.to(dtype))
    if rows and K:
        codes = c.codes.view(rows, -1).cpu()
        assert (codes[:, K:] == 0).all()
        err = (want - x.double()).abs()
        assert (err <= x.double().abs() / 16 + x.double().abs().amax(1, keepdim=True) * 2.0 ** -17).all()


def test_special_values(dev):
    from neurofluid_amd import act8
    inf, nan, big = float("inf"), float("nan"), torch.finfo(F32).max
    rows = [
        [0.0] * 40, [-0.0, 1e-45, -1e-40, 2.0 ** -120, 2.0 ** -119, 2.0 ** -118.5, 3 * 2.0 ** -120, 5 * 2.0 ** -121], [2.0 ** -110 * 448, 2.0 ** -119, 2.0 ** -120],
        [448.0, 447.9, 1.0, 2.0 ** -10, 2.0 ** -9, 3 * 2.0 ** -10, 2.0 ** -10 * 1.0001, -17.0, 18.0, 19.0, 20.0, 21.0], [448.00003, 1.0, 0.001],
        [1.75, 1.0, 0.0302734375, 0.03125], [1.7500001, 0.99], [big, -big, 1.0, big / 3], [inf, 2.0, -3.0, 1e-3], [nan, -inf, 0.1, 0.2], [inf] * 40, [1.0] * 31 + [nan] + [2.0] * 8,
        [9.0 + i for i in range(40)], [2.0 ** i for i in range(-20, 20)], [272.0, 288.0, 304.0, 17.0, 1.0625, 1.1875],
    ]
    for fill in (0.5, 0.0):
        x = torch.tensor([r + [fill] * (40 - len(r)) for r in rows])
        assert same(act8.pack(x.to(dev)).unpack().cpu().double(), quantised(x))


def test_layouts(dev):
    """Rows apart, odd offsets, transposed, more axes; packing does not read beside its rows."""
    from neurofluid_amd import act8
    g = torch.Generator().manual_seed(3)
    buf = torch.full((70, 150), float("nan"))
    buf[:, 5:105] = torch.randn(70, 100, generator=g)
    for dt in (F32, BF16, F16):
        b = buf.to(dt).to(dev)
        want = quantised(buf.to(dt)[:, 5:105]).to(dt)
        assert same(act8.pack(b[:, 5:105]).unpack().cpu(), want)
        assert same(act8.pack(b[:, 5:105].t().contiguous().t()).unpack().cpu(), want)
        assert same(act8.pack(b[:, 5:105].reshape(7, 10, 100)).unpack().cpu(), want.view(7, 10, 100))
        assert same(act8.pack(b[3, 5:105]).unpack().cpu(), want[3])
        assert same(act8.pack(b[::3, 5:105]).unpack().cpu(), want[::3])
    assert act8.pack(torch.zeros(4, 0, device=dev)).unpack().shape == (4, 0)


def check_wgrad(dev, x, dy, dyd=None):
    from neurofluid_amd import act8
    q = quantised(x)
    ck = act8.pack(x.to(dev))
    dW, db = act8.wgrad(dy.to(dev) if dyd is None else dyd, ck)
    assert dW.dtype == db.dtype == F32 and dW.shape == (dy.shape[1], x.shape[1])
    d64 = dy.double()
    n = (3 * x.shape[0] + 64) * 2.0 ** -23
    assert ((dW.cpu().double() - d64.t() @ q).abs() <= n * (d64.abs().t() @ q.abs())).all()
    assert ((db.cpu().double() - d64.sum(0)).abs() <= n * d64.abs().sum(0)).all()
    return dW, db


@pytest.mark.parametrize("rows, M, K", [(1, 1, 1), (5, 3, 7), (64, 128, 128), (65, 129, 130), (63, 4, 256), (257, 256, 256), (1000, 100, 300), (511, 130, 33),
                                        (2048, 64, 40), (4100, 7, 260)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_wgrad(dev, rows, M, K, dtype):
    g = torch.Generator().manual_seed(rows + M + K)
    x = torch.relu(torch.randn(rows, K, generator=g)) * torch.exp(torch.randn(rows, 1, generator=g))
    dy = (torch.randn(rows, M, generator=g) * 0.01).to(dtype)
    check_wgrad(dev, x.to(dtype), dy)


def test_wgrad_large_slices(dev):
    g = torch.Generator().manual_seed(1)
    x, dy = torch.randn(33000, 64, generator=g), torch.randn(33000, 96, generator=g)
    a = check_wgrad(dev, x, dy)
    b = check_wgrad(dev, x, dy)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])          # bit for bit


def test_wgrad_no_rows(dev):
    from neurofluid_amd import act8
    dW, db = act8.wgrad(torch.zeros(0, 5, device=dev), act8.pack(torch.zeros(0, 40, device=dev)))
    assert dW.shape == (5, 40) and not dW.any() and not db.any()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_wgrad_loses_no_bit_of_dy(dev, dtype):
    """One row of dy per output and power-of-two activations: the gradient is dy times a power of two, to the bit.  Only what of dy
    lies below 2^-133, bf16's smallest number, is no sum of bf16 numbers: |error| < 2^-133 x, less than an ulp of anything above 2^-110."""
    from neurofluid_amd import act8
    g = torch.Generator().manual_seed(2)
    rows, M, K = 150, 140, 70
    vals = torch.randn(M, generator=g) * torch.exp(5 * torch.randn(M, generator=g))
    vals[:6] = torch.tensor([16777215.0, -12345677.0, 1 / 3, 0.1, 65504.0, 1e-5])
    if dtype == F32:
        vals[6:9] = torch.tensor([torch.finfo(F32).max, -1.17549449e-38, 8388607.0 * 2.0 ** 100])
    vals = vals.to(dtype)
    dy = torch.zeros(rows, M, dtype=dtype)
    r = torch.randint(0, rows, (M,), generator=g)
    dy[r, torch.arange(M)] = vals
    x = torch.ones(rows, K)                    # every entry a power of two
    x[:, 1::2] = 0.5
    dW, db = act8.wgrad(dy.to(dev), act8.pack(x.to(dev)))
    want = vals.double()[:, None] * x[0].double()[None]
    got = dW.cpu().double()                    # (the two largest are infinite in fp16, and stay so)
    assert ((got == want) | ((got - want).abs() <= 2.0 ** -133 * x[0].double()[None])).all()
    assert torch.equal(dW.cpu()[vals.float().abs() >= 2.0 ** -102], want.float()[vals.float().abs() >= 2.0 ** -102])
    assert torch.equal(db.cpu(), vals.float())


def test_wgrad_not_finite(dev):
    """Infinities and NaN of dy reach their output's row, those of an activation (NaN in 8 bits) its feature's column; nothing else."""
    from neurofluid_amd import act8
    g = torch.Generator().manual_seed(4)
    x, dy = torch.rand(300, 70, generator=g) + 0.5, torch.randn(300, 20, generator=g)
    for dt in (F32, BF16, F16):
        d = dy.to(dt)
        want, wb = act8.wgrad(d.to(dev), act8.pack(x.to(dev)))
        d2, x2 = d.clone(), x.clone()
        d2[100, 3], d2[299, 5], d2[7, 6] = float("inf"), float("nan"), float("-inf")
        x2[200, 40] = float("inf")
        got, gb = act8.wgrad(d2.to(dev), act8.pack(x2.to(dev)))
        cols = [c for c in range(70) if c != 40]
        assert (got[3, cols] == float("inf")).all() and (got[6, cols] == float("-inf")).all() and torch.isnan(got[5]).all() and torch.isnan(got[:, 40]).all()
        assert gb[3] == float("inf") and gb[6] == float("-inf") and torch.isnan(gb[5])
        rows = [m for m in range(20) if m not in (3, 5, 6)]
        cols = [c for c in cols if c // 32 != 1]              # (the block of 40 has lost no value, but may have another largest one)
        assert torch.equal(got[rows][:, cols], want[rows][:, cols]) and torch.equal(gb[rows], wb[rows])


def test_wgrad_layouts_and_jobs(dev):
    from neurofluid_amd import act8
    g = torch.Generator().manual_seed(6)
    x, big = torch.randn(700, 160, generator=g), torch.randn(700, 90, generator=g)
    ck = act8.pack(x.to(dev))
    bd = big.to(dev)
    base = act8.wgrad(bd, ck)
    dtr = bd.t().contiguous().t()
    assert torch.equal(act8.wgrad(dtr, ck)[0], base[0])
    assert torch.equal(act8.wgrad(bd.view(7, 100, 90), act8.pack(x.to(dev).view(7, 100, 160)))[0], base[0])
    off = torch.zeros(700, 97, device=dev)
    off[:, 3:93] = bd
    check_wgrad(dev, x, big, off[:, 3:93])
    one = act8.wgrad(bd[:1].expand(700, 90), ck)              # a gradient with stride 0
    q = quantised(x)
    assert ((one[0].cpu().double() - big[0].double()[:, None] * q.sum(0)[None]).abs() <= (3 * 700 + 64) * 2.0 ** -23 * big[0].double().abs()[:, None] * q.abs().sum(0)).all()
    jobs = [(0, 90, 0, 160, True), (3, 1, 32, 70, True), (89, 1, 128, 32, False), (4, 64, 64, 96, True)]
    res = act8.wgrad_jobs(bd, ck, jobs)
    d64, n = big.double(), (3 * 700 + 64) * 2.0 ** -23
    for (a, M, c, K, b), (dW, db) in zip(jobs, res):
        dd, qq = d64[:, a:a + M], q[:, c:c + K]
        assert ((dW.cpu().double() - dd.t() @ qq).abs() <= n * (dd.abs().t() @ qq.abs())).all()
        assert (db is not None) == b
        if b:
            assert ((db.cpu().double() - dd.sum(0)).abs() <= n * dd.abs().sum(0)).all()
    with pytest.raises(RuntimeError):
        act8.wgrad_jobs(bd, ck, [(0, 90, 16, 32, True)])
    with pytest.raises(RuntimeError):
        act8.wgrad_jobs(bd, ck, [(1, 90, 0, 32, True)])


def test_linear(dev):
    """Forward and dx are the exact layer's; dW is the formula's on the packed input.  Compared with differences, too: the loss is linear in x."""
    from neurofluid_amd import act8
    g = torch.Generator().manual_seed(9)
    x, w, b, gy = (torch.randn(*s, generator=g) for s in ((6, 50, 72), (40, 72), (40,), (6, 50, 40)))
    xd, wd, bd = (q.to(dev).requires_grad_() for q in (x, w, b))
    y = act8.linear(xd, wd, bd)
    assert y.shape == (6, 50, 40)
    # 72 products and the bias: at most 80 additions of one ulp
    bound = 80 * 2.0 ** -23 * (x.double().abs() @ w.double().abs().t() + b.double().abs())
    assert ((y.detach().cpu().double() - (x.double() @ w.double().t() + b.double())).abs() <= bound).all()
    dx, dw, db = torch.autograd.grad(y, [xd, wd, bd], gy.to(dev))
    d2 = gy.double().reshape(-1, 40)
    assert ((dx.cpu().double() - gy.double() @ w.double()).abs() <= 80 * 2.0 ** -23 * (gy.double().abs() @ w.double().abs())).all()
    q = quantised(x.reshape(-1, 72))
    n = (3 * 300 + 64) * 2.0 ** -23
    assert ((dw.cpu().double() - d2.t() @ q).abs() <= n * (d2.abs().t() @ q.abs())).all()
    assert ((db.cpu().double() - d2.sum(0)).abs() <= n * d2.abs().sum(0)).all()
    # the exact dW differs by what the codes differ: at most 2^-4 of every activation, and 2^-10 of a block's scale (2^-18 of its maximum, doubled)
    exact = d2.t() @ x.double().reshape(-1, 72)
    slack = d2.abs().t() @ (x.double().abs().reshape(-1, 72) / 16 + x.abs().max().double() * 2.0 ** -17)
    assert ((dw.cpu().double() - exact).abs() <= slack + n * slack).all()
    d = torch.randn(x.shape, generator=g)
    with torch.no_grad():
        diff = ((act8.linear((x + d).to(dev), wd, bd).double() - act8.linear((x - d).to(dev), wd, bd).double()) * gy.to(dev)).sum() / 2
    assert abs(float(diff) - float((dx.cpu().double() * d).sum())) <= 160 * 2.0 ** -23 * float((gy.double().abs().reshape(-1, 40) * (bound * 2.0 ** 23 / 80 * 3).reshape(-1, 40)).sum())
    # only what is asked for
    with torch.no_grad():
        assert torch.equal(act8.linear(x.to(dev), wd, bd), y)
    y2 = act8.linear(xd, wd.detach(), bd.detach())
    assert torch.equal(torch.autograd.grad(y2, xd, gy.to(dev))[0], dx)
    y3 = act8.linear(xd.detach(), wd)
    assert torch.equal(torch.autograd.grad(y3, wd, gy.to(dev))[0], dw)
    y4 = act8.linear(xd.detach(), wd.detach(), bd)
    assert torch.allclose(torch.autograd.grad(y4, bd, gy.to(dev))[0], db, rtol=0, atol=float(n * d2.abs().sum(0).max()))
    for lead in ((0,), (1,), (3, 0)):
        z = torch.zeros(*lead, 72, device=dev, requires_grad=True)
        o = act8.linear(z, wd, bd)
        gz, gw, gb = torch.autograd.grad(o, [z, wd, bd], torch.ones_like(o))
        assert o.shape == lead + (40,) and gz.shape == z.shape and not gw.any()


def test_linear_packs_for_a_backward_only(dev, monkeypatch):
    from neurofluid_amd import act8
    x, w, b = torch.randn(70, 33, device=dev), torch.randn(5, 33, device=dev, requires_grad=True), torch.randn(5, device=dev, requires_grad=True)
    want = act8.linear(x, w, b)

    def never(x):
        raise AssertionError("packed")
    monkeypatch.setattr(act8, "pack", never)
    with torch.no_grad():
        assert torch.equal(act8.linear(x, w, b), want)
    assert torch.equal(act8.linear(x, w.detach(), b.detach()), want)
    assert torch.equal(act8.linear(x, w.detach(), b), want)


def test_linear_frees_what_it_kept(dev):
    """A loss that is still held after its backward holds none of the packed inputs."""
    from neurofluid_amd import act8
    x, w = torch.randn(20000, 512, device=dev), torch.randn(8, 512, device=dev, requires_grad=True)
    act8.linear(x, w).sum().backward()
    before = torch.cuda.memory_allocated()
    loss = act8.linear(x, w).sum()
    assert torch.cuda.memory_allocated() - before >= 20000 * 512
    loss.backward()
    assert torch.cuda.memory_allocated() - before < 20000 * 512 // 8


def test_linear_layouts(dev):
    """Operands as a model may hold them: expanded rows, a transposed weight, a gradient of one value; the bias alone over many rows, captured."""
    from neurofluid_amd import act8
    g = torch.Generator().manual_seed(13)
    w, b = torch.randn(40, 24, generator=g), torch.randn(40, generator=g)
    n = (3 * 9000 + 64) * 2.0 ** -23
    for base, view in ((torch.randn(1, 24, generator=g), lambda t: t.expand(500, 24)), (torch.randn(24, 300, generator=g), lambda t: t.t()),
                       (torch.randn(500, 1, generator=g), lambda t: t.expand(500, 24)), (torch.randn(9, 7, 30, generator=g), lambda t: t[:, 1:, 2:26])):
        for turned in (False, True):
            x, bd = view(base), b.to(dev).requires_grad_()
            wd = (w.to(dev).t().contiguous().t() if turned else w.to(dev)).requires_grad_()
            y = act8.linear(view(base.to(dev)), wd, bd)
            x2 = x.double().reshape(-1, 24)
            bound = 32 * 2.0 ** -23 * (x2.abs() @ w.double().abs().t() + b.double().abs())
            assert ((y.detach().cpu().double().reshape(-1, 40) - (x2 @ w.double().t() + b.double())).abs() <= bound).all()
            y.sum().backward()          # the gradient comes as one expanded value
            q = quantised(x.reshape(-1, 24).contiguous())
            assert ((wd.grad.cpu().double() - q.sum(0).expand(40, 24)).abs() <= n * q.abs().sum(0)).all()
            assert torch.equal(bd.grad.cpu(), torch.full((40,), float(x2.shape[0])))
    one = [torch.full(k, v, device=dev, requires_grad=True) for k, v in (((3, 1), 2.0), ((1, 1), 5.0), ((1,), 0.25))]
    act8.linear(*one).sum().backward()
    assert [float(t.grad.sum()) for t in one] == [15.0, 6.0, 3.0]
    x, gy = torch.randn(9000, 24, generator=g).to(dev), torch.randn(9000, 40, generator=g).to(dev)
    leaf = b.to(dev).requires_grad_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(act8.linear(x, w.to(dev), leaf), leaf, gy)
    torch.cuda.current_stream().wait_stream(side)
    wd, gr = w.to(dev), torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        db, = torch.autograd.grad(act8.linear(x, wd, leaf), leaf, gy)
    for it in range(4):
        gy.mul_(-1.5)
        gr.replay()
        torch.cuda.synchronize()
        g2 = gy.cpu().double()
        assert ((db.cpu().double() - g2.sum(0)).abs() <= n * g2.abs().sum(0)).all()


def test_streams_and_graphs(dev):
    from neurofluid_amd import act8
    g = torch.Generator().manual_seed(11)
    x, dy = torch.randn(5000, 96, generator=g).to(dev), torch.randn(5000, 64, generator=g).to(dev)

    def both(x, dy):
        c = act8.pack(x)
        return (c.unpack(),) + act8.wgrad(dy, c)
    want = both(x, dy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = both(x, dy)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    bufs = [(x.clone(), dy.clone()) for _ in range(2)]
    graphs, outs = [], []
    for b in bufs:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(both(*b))
        graphs.append(gr)
    for it in range(4):
        for k in (0, 1):
            bufs[k][0].copy_(x * (1 + it + 3 * k))
            graphs[k].replay()
        for k in (0, 1):
            eager = both(x * (1 + it + 3 * k), dy)
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(eager, outs[k]))


def test_long_rows(dev):
    """More rows than one launch's grid takes, more than 2^31 elements behind the first: the last rows equal themselves packed alone."""
    from neurofluid_amd import act8
    rows, K = 4_300_000, 520
    x = torch.zeros(rows, K, dtype=BF16, device=dev)
    x[-1000:].normal_()
    x[:10].normal_()
    c = act8.pack(x)
    out = c.unpack()
    assert torch.equal(out[-1000:], act8.pack(x[-1000:]).unpack()) and torch.equal(out[:10], act8.pack(x[:10]).unpack()) and not out[10:-1000].any()
    dy = torch.zeros(rows, 8, dtype=BF16, device=dev)
    dy[-1000:].normal_()
    dW, db = act8.wgrad(dy, c)
    small, sb = act8.wgrad(dy[-1000:].contiguous(), act8.pack(x[-1000:]))
    s = dy[-1000:].double().abs().t() @ out[-1000:].double().abs()
    assert ((dW - small).abs() <= 2 * 3064 * 2.0 ** -23 * s).all()
