"""The gated recurrence (csrc/nf_scan*.hip) against its definition in 64 bits, step by step on the CPU.

Tolerances are running error bounds, made before the first run.  One fp32 operation is off by u = 2^-24 of its result.  A step of
the kernel is one fused multiply-add on the state (u), and what carries a state across stretches multiplies products of gates (u a gate) and
adds a few more operations a tile; a log gate adds exp, at most one ulp (2 u).  With eight roundings a step allowed for, the error of h_t obeys
    E_t <= |A_t| E_(t-1) + 8 u M_t,      M_t = |A_t| M_(t-1) + |x_t|
(M: the recurrence of the magnitudes).  The same recurrence bounds dx; a product's bound follows from its factors', a sum over D channels adds D u of the
sum of magnitudes; a value stored in 16 bits is off by eps / 2 of itself more."""
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    return torch.device("cuda:0")


def half_step(v, dtype):
    """What rounding v to dtype may cost (the smallest subnormal's half included)."""
    i = torch.finfo(dtype)
    return v.abs() * (i.eps / 2) + i.smallest_normal * i.eps / 2


def seq64(A, x, h0):
    """States of one run over dim 0, magnitudes M and error bound E."""
    h, m, e = h0.clone(), h0.abs(), torch.zeros_like(h0)
    H, M, E = [], [], []
    for t in range(x.shape[0]):
        h = A[t] * h + x[t]
        m = A[t].abs() * m + x[t].abs()
        e = A[t].abs() * e + 8 * U * m
        H.append(h); M.append(m); E.append(e)
    st = lambda q: torch.stack(q) if q else x.new_zeros(x.shape)
    return st(H), st(M), st(E), (h, e)


def oracle(gate, x, h0, g, g_last, log_gate, reverse):
    """One sequence: gate (T, D or 1), x (T, D), ... in float64.  Returns values and bounds (before storage rounding)."""
    T, D = x.shape
    fl = (lambda q: q.flip(0)) if reverse else (lambda q: q)
    A = fl((torch.exp(gate) if log_gate else gate).expand(T, D))
    xs, gs = fl(x), fl(g)
    h, M, E, (last, e_last) = seq64(A, xs, h0)
    before = torch.cat([h0[None], h[:-1]]) if T else h
    e_before = torch.cat([torch.zeros_like(h0)[None], E[:-1]]) if T else E
    # dx_t = g_t + A_(t+1) dx_(t+1): the same recurrence, g_last (with a factor of 1) the state that enters behind the last step.  Its magnitudes
    # are those of the terms, not of sums that have cancelled: the kernel adds them in another order.
    Anext = torch.cat([A[1:], torch.ones(1, D, dtype=A.dtype)]) if T else A
    rdx, rM, rE, _ = seq64(Anext.flip(0), gs.flip(0), g_last)
    dx, M_dx, e_dx = rdx.flip(0), rM.flip(0), rE.flip(0)
    u, e_u = A * dx, A.abs() * e_dx + 4 * U * A.abs() * M_dx
    f, e_f = (u, e_u) if log_gate else (dx, e_dx)
    dg = f * before
    e_dg = e_f * before.abs() + f.abs() * e_before + e_f * e_before + 2 * U * dg.abs()
    if gate.shape[1] == 1 and D > 0:
        e_dg = e_dg.sum(1, keepdim=True) + D * U * dg.abs().sum(1, keepdim=True)
        dg = dg.sum(1, keepdim=True)
    dh0 = u[0] if T else g_last
    e_dh0 = e_u[0] if T else torch.zeros_like(g_last)
    return dict(h=(fl(h), fl(E)), last=(last, e_last), dgate=(fl(dg), fl(e_dg)), dx=(fl(dx), fl(e_dx)), dh0=(dh0, e_dh0))


def check(name, got, want, bound, dtype):
    got = got.detach().cpu().double()
    assert got.shape == want.shape, (name, got.shape, want.shape)
    if not got.numel():
        return
    tol = bound + half_step(want.abs() + bound, dtype)
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), (name, int(bad.sum()), got[bad][:4].tolist(), want[bad][:4].tolist(), tol[bad][:4].tolist())


def make(shape, gate_shape, dtype, gate_dtype, log_gate, seed):
    g = torch.Generator().manual_seed(seed)
    u = torch.rand(gate_shape, generator=g)
    gate = -torch.relu(torch.randn(gate_shape, generator=g)) * u if log_gate else torch.sigmoid(6 * u - 1) * torch.where(torch.rand(gate_shape, generator=g) < 0.1, -1.0, 1.0)
    return gate.to(gate_dtype), torch.randn(shape, generator=g).to(dtype), torch.randn(shape, generator=g).to(dtype), g


def run_dense(dev, B, T, D, dtype, gate_kind, log_gate, reverse, with_h0, seed=0, view=None):
    from neurofluid_amd import scan
    gdt = F32 if gate_kind == "full32" else dtype
    gate, x, gy, gen = make((B, T, D), (B, T, 1 if gate_kind == "shared" else D), dtype, gdt, log_gate, seed)
    h0, gl = torch.randn(B, D, generator=gen), torch.randn(B, D, generator=gen)
    dv = view or (lambda q: q.to(dev))
    gd, xd, yd = dv(gate), dv(x), dv(gy)
    hd = h0.to(dev) if with_h0 else None
    leaves = [q.requires_grad_() for q in (gd, xd, hd) if q is not None]
    h, last = scan.gated_scan(gd, xd, hd, log_gate=log_gate, reverse=reverse)
    assert h.dtype == dtype and last.dtype == F32
    grads = torch.autograd.grad([h, last], leaves, [yd, gl.to(dev)])
    z = torch.zeros(B, D, dtype=torch.float64)
    for b in range(B) if B <= 4 else [0, 1, B // 2, B - 1]:
        want = oracle(gate[b].double(), x[b].double(), h0[b].double() if with_h0 else z[b], gy[b].double(), gl[b].double(), log_gate, reverse)
        check("h", h[b], *want["h"], dtype)
        check("last", last[b], *want["last"], F32)
        check("dgate", grads[0][b], *want["dgate"], gdt)
        check("dx", grads[1][b], *want["dx"], dtype)
        if with_h0:
            check("dh0", grads[2][b], *want["dh0"], F32)
    return h, last, grads


@pytest.mark.parametrize("T", [0, 1, 2, 7, 8, 9, 16, 17, 64, 65, 129, 257, 1030])
@pytest.mark.parametrize("D", [1, 2, 3, 5, 16, 33, 64, 130])
def test_lengths_and_widths(dev, T, D):
    k = (T * 7 + D) % 8
    run_dense(dev, 2, T, D, [F32, BF16, F16][(T + D) % 3], ["full", "shared"][k & 1], bool(k & 2), bool(k & 4), bool((T + D) & 1), seed=T * 131 + D)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("gate_kind", ["full", "full32", "shared"])
@pytest.mark.parametrize("log_gate", [False, True])
@pytest.mark.parametrize("reverse", [False, True])
def test_types_gates_directions(dev, dtype, gate_kind, log_gate, reverse):
    run_dense(dev, 3, 203, 96, dtype, gate_kind, log_gate, reverse, True, seed=5)
    run_dense(dev, 2, 77, 31, dtype, gate_kind, log_gate, reverse, False, seed=6)


@pytest.mark.parametrize("B, T, D, dtype", [(1, 5003, 64, F32), (1, 3001, 7, BF16), (2, 2050, 192, F16), (1, 2600, 1, F32), (1, 4097, 34, BF16)])
@pytest.mark.parametrize("gate_kind", ["full", "shared"])
def test_long_axis_is_cut(dev, B, T, D, dtype, gate_kind):
    run_dense(dev, B, T, D, dtype, gate_kind, True, False, True, seed=T)
    run_dense(dev, B, T, D, dtype, gate_kind, False, True, True, seed=T + 1)


@pytest.mark.parametrize("B, T, D, dtype, gate_kind", [(4100, 40, 4, F32, "shared"), (4099, 600, 1, F32, "full"), (700, 192, 32, F32, "shared"), (2049, 33, 128, BF16, "full")])
def test_many_chains(dev, B, T, D, dtype, gate_kind):
    run_dense(dev, B, T, D, dtype, gate_kind, True, True, False, seed=B)


def test_strided_inputs(dev):
    def padded(q):          # a column slice of a wider buffer, odd offset: rows unaligned for pairs
        buf = torch.full(q.shape[:-1] + (q.shape[-1] + 5,), float("nan"), dtype=q.dtype, device=dev)
        v = buf[..., 3:3 + q.shape[-1]]
        v.copy_(q)
        return v.detach()

    def time_major(q):      # (T, B, D) seen as (B, T, D)
        return q.to(dev).transpose(0, 1).contiguous().transpose(0, 1).detach()

    def channels_apart(q):
        return q.to(dev).transpose(1, 2).contiguous().transpose(1, 2).detach()
    for i, view in enumerate((padded, time_major, channels_apart)):
        for D in (6, 64):
            a = run_dense(dev, 3, 130, D, BF16, "full", False, False, True, seed=i, view=view)
            if view is padded:      # read element by element: stretches of other lengths, so within the bounds (checked above), not to the bit
                continue
            b = run_dense(dev, 3, 130, D, BF16, "full", False, False, True, seed=i)
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and all(torch.equal(p, q) for p, q in zip(a[2], b[2]))


def test_broadcast_inputs_and_expanded_gradient(dev):
    """A gate expanded over the batch (stride 0) and a gradient that is one number (sum().backward())."""
    from neurofluid_amd import scan
    gate, x, _, _ = make((3, 100, 16), (1, 100, 16), F32, F32, False, 9)
    gd, xd = gate.to(dev).requires_grad_(), x.to(dev).requires_grad_()
    h, _ = scan.gated_scan(gd.expand(3, 100, 16), xd)
    h.sum().backward()
    total, bound = 0, 0
    for b in range(3):
        w = oracle(gate[0].double(), x[b].double(), torch.zeros(16).double(), torch.ones(100, 16).double(), torch.zeros(16).double(), False, False)
        check("dx", xd.grad[b], *w["dx"], F32)
        total, bound = total + w["dgate"][0], bound + w["dgate"][1] + half_step(w["dgate"][0], F32)
    check("dgate", gd.grad[0], total, bound + 3 * U * total.abs() + bound, F32)


def splits_of(lens, lead=0):
    return torch.tensor([lead] + lens).cumsum(0)


PACKED = [
    ([5, 0, 1, 64, 0, 0, 130, 7], 0, 3), ([0, 0, 0], 0, 4), ([1] * 40, 0, 0), ([900, 3, 0, 700, 2], 0, 11), ([300], 0, 0), ([12, 9], 4, 2), ([], 0, 6),
]


@pytest.mark.parametrize("lens, lead, tail", PACKED)
@pytest.mark.parametrize("D, dtype, gate_kind", [(3, F32, "shared"), (34, BF16, "full"), (96, F16, "shared"), (1, F32, "full")])
@pytest.mark.parametrize("reverse", [False, True])
def test_packed(dev, lens, lead, tail, D, dtype, gate_kind, reverse):
    """Sequences behind one another, empty ones among them, rows before the first and behind the last (filled with NaN and infinities):
    zero there, and nothing leaks."""
    from neurofluid_amd import scan
    rs = splits_of(lens, lead)
    N, S = int(rs[-1]) + tail, len(lens)
    log_gate = bool(len(lens) & 1)
    gate, x, gy, gen = make((N, D), (N, 1 if gate_kind == "shared" else D), dtype, dtype, log_gate, N + D)
    for q in (gate, x, gy):
        q[:lead] = float("nan")
        q[int(rs[-1]):] = float("inf")
    h0, gl = torch.randn(S, D, generator=gen), torch.randn(S, D, generator=gen)
    for with_h0 in (True, False):
        gd, xd = gate.to(dev).requires_grad_(), x.to(dev).requires_grad_()
        hd = h0.to(dev).requires_grad_() if with_h0 else None
        h, last = scan.gated_scan(gd, xd, hd, log_gate=log_gate, reverse=reverse, row_splits=rs.to(dev))
        gr = torch.autograd.grad([h, last], [gd, xd] + ([hd] if with_h0 else []), [gy.to(dev), gl.to(dev)])
        assert last.shape == (S, D)
        outside = torch.ones(N, dtype=torch.bool)
        for s in range(S):
            a, b = int(rs[s]), int(rs[s + 1])
            outside[a:b] = False
            start = h0[s].double() if with_h0 else torch.zeros(D).double()
            w = oracle(gate[a:b].double(), x[a:b].double(), start, gy[a:b].double(), gl[s].double(), log_gate, reverse)
            check("h", h[a:b], *w["h"], dtype)
            check("last", last[s], *w["last"], F32)
            check("dgate", gr[0][a:b], *w["dgate"], dtype)
            check("dx", gr[1][a:b], *w["dx"], dtype)
            if with_h0:
                check("dh0", gr[2][s], *w["dh0"], F32)
        for q in (h, gr[0], gr[1]):
            assert (q.detach().cpu()[outside] == 0).all()


def test_bad_row_splits_stay_in_bounds(dev):
    """Splits that descend or leave the tensor give some numbers, and every access stays inside."""
    from neurofluid_amd import scan
    x = torch.randn(300, 40, device=dev, requires_grad=True)
    gate = torch.rand(300, 40, device=dev, requires_grad=True)
    h0 = torch.randn(4, 40, device=dev, requires_grad=True)
    for rs in ([0, 200, 100, 300, 250], [-50, 10, 10 ** 12, -(10 ** 12), 300], [400, 500, 600, 700, 800], [5, 4, 3, 2, 1]):
        h, last = scan.gated_scan(gate, x, h0, row_splits=torch.tensor(rs, device=dev))
        torch.autograd.grad([h, last], [gate, x, h0], [torch.ones_like(h), torch.ones_like(last)])
        torch.cuda.synchronize()


def test_not_finite_values_stay_in_their_chain(dev):
    """NaN and infinity in one channel of one batch reach later steps of that channel only; a log gate of -inf or of the type's
    lowest value is a gate of 0."""
    from neurofluid_amd import scan
    gate, x, gy, _ = make((3, 400, 64), (3, 400, 64), F32, F32, True, 3)
    gd, xd = gate.to(dev), x.to(dev)
    want, _ = scan.gated_scan(gd, xd, log_gate=True)
    x2 = xd.clone()
    x2[1, 150, 7] = float("nan")
    x2[2, 300, 8] = float("inf")
    got, last = scan.gated_scan(gd, x2, log_gate=True)
    assert torch.isnan(got[1, 150:, 7]).all() and torch.isnan(last[1, 7])
    assert not torch.isfinite(got[2, 300:, 8]).any()
    keep = torch.ones_like(got, dtype=torch.bool)
    keep[1, 150:, 7] = False
    keep[2, 300:, 8] = False
    assert torch.equal(got[keep], want[keep])
    for low in (float("-inf"), torch.finfo(F32).min):
        g3 = gate.clone()
        g3[:, 100] = low
        g3[:, 201:203] = low
        w = oracle(g3[0].double(), x[0].double(), torch.zeros(64).double(), gy[0].double(), torch.zeros(64).double(), True, False)
        a, b = g3.to(dev).requires_grad_(), xd.clone().requires_grad_()
        h, _ = scan.gated_scan(a, b, log_gate=True)
        da, db = torch.autograd.grad(h, [a, b], gy.to(dev))
        check("h", h[0], *w["h"], F32)
        check("dgate", da[0], *w["dgate"], F32)
        check("dx", db[0], *w["dx"], F32)
        assert torch.equal(h[:, 100], xd[:, 100])


def test_long_offsets(dev):
    """A tensor of more than 2^31 elements: the last batch equals the same data on its own."""
    from neurofluid_amd import scan
    B, T, D = 33, 65536, 1024
    x = torch.empty(B, T, D, dtype=BF16, device=dev)
    x.fill_(0.5)
    x[-1].normal_()
    gate = torch.rand(T, 1, device=dev).to(BF16).expand(B, T, 1)
    with torch.no_grad():
        h, last = scan.gated_scan(gate, x)
        h1, last1 = scan.gated_scan(gate[:1].expand(33, T, 1)[-1:], x[-1:])
    assert torch.equal(last[:-1], last[:1].expand(B - 1, D))
    # cut differently, the carries round differently: 8 u M a step over the few steps that a gate's mean of 1/2 remembers (M < 64, 64 steps
    # at the most), and two bf16 values next to each other are a whole step, eps, apart
    e = 64 * 8 * U * 64
    assert ((h[-1].float() - h1[0].float()).abs() <= 2 * e + torch.finfo(BF16).eps * h1[0].float().abs()).all()
    assert (last[-1] - last1[0]).abs().max() <= 2 * e


def test_far_apart_and_widest_rows(dev):
    """The widest rows that are taken, packed (a tile's rows span 2 GiB), and steps that lie as far apart as a view may have them."""
    from neurofluid_amd import scan
    D, cuts = 1 << 20, (0, 1, 4)
    g = torch.Generator(device=dev).manual_seed(3)
    gate, x = torch.rand(4, D, device=dev, generator=g), torch.randn(4, D, device=dev, generator=g)
    rs = torch.tensor(cuts, device=dev)
    for reverse in (False, True):
        gd, xd = gate.clone().requires_grad_(), x.clone().requires_grad_()
        h, last = scan.gated_scan(gd, xd, row_splits=rs, reverse=reverse)
        h.sum().backward()
        want, dx = torch.empty_like(x, dtype=torch.float64), torch.empty_like(x, dtype=torch.float64)
        for a, b in zip(cuts, cuts[1:]):
            order = list(range(a, b))[::-1] if reverse else list(range(a, b))
            s = torch.zeros(D, dtype=torch.float64, device=dev)
            for j in order:
                s = gate[j].double() * s + x[j].double()
                want[j] = s
            u = torch.zeros_like(s)
            for j in order[::-1]:
                dx[j] = 1 + u
                u = gate[j].double() * dx[j]
        # at most three steps: a rounding each of the product, the sum and the carry, of sums below 3 max |x|
        assert (h.detach().double() - want).abs().max() <= 9 * 2.0 ** -24 * 3 * float(x.abs().max())
        assert (xd.grad.double() - dx).abs().max() <= 9 * 2.0 ** -24 * 3
    T, far = 8300, 150000          # two channels of rows that are 150 000 wide; more than two tiles of 4 096 steps
    for width in (far, 1 << 17, (1 << 17) + 1):
        wide = torch.zeros(T, width, dtype=torch.bfloat16, device=dev)
        wide[:, 1:3] = torch.randn(T, 2, device=dev, generator=g).bfloat16()
        gt = torch.rand(1, T, 1, device=dev, generator=g)
        view = wide[None, :, 1:3]
        a, b = scan.gated_scan(gt, view), scan.gated_scan(gt, view.contiguous())
        s = torch.zeros(2, dtype=torch.float64)
        gc, xc, want = gt.cpu().double().view(-1), view[0].cpu().double(), []
        for t in range(T):
            s = gc[t] * s + xc[t]
            want.append(s)
        want = torch.stack(want)
        # gates below one, uniform: what is kept is the sum of a few values; 64 fp32 roundings of the largest and bf16's half step
        tol = 64 * 2.0 ** -24 * want.abs().max() + want.abs() * 2.0 ** -8
        assert ((a[0][0].cpu().double() - want).abs() <= tol).all() and ((b[0][0].cpu().double() - want).abs() <= tol).all()
        del wide, view


def test_more_chains_than_a_launch_takes(dev):
    from neurofluid_amd import scan
    B = (1 << 26) + 5
    x, gate = torch.ones(B, 1, 1, dtype=torch.bfloat16, device=dev), torch.full((B, 1, 1), 0.5, dtype=torch.bfloat16, device=dev)
    h0 = torch.full((B, 1), 4.0, device=dev)
    h0[-1] = 8.0
    xr = x.requires_grad_()
    h, last = scan.gated_scan(gate, xr, h0)
    hd, ld = h.detach(), last.detach()
    assert float(ld[-1]) == 5.0 and bool((ld[:-1] == 3.0).all()) and float(hd[-1]) == 5.0 and bool((hd[:-1] == 3.0).all())
    dx, = torch.autograd.grad(h, xr, gate)
    assert bool((dx == 0.5).all())


def test_differences(dev):
    """Directional derivative by central differences; f = <w, h> + <v, h_last> is linear in x and h0, smooth in the gate."""
    from neurofluid_amd import scan
    gate, x, w, gen = make((2, 90, 40), (2, 90, 40), F32, F32, True, 12)
    h0, v = torch.randn(2, 40, generator=gen), torch.randn(2, 40, generator=gen)
    ins = [q.to(dev).requires_grad_() for q in (gate, x, h0)]
    wd, vd = w.to(dev), v.to(dev)

    def f(a):
        h, last = scan.gated_scan(*a, log_gate=True)
        return (h.double() * wd).sum() + (last.double() * vd).sum()
    grads = torch.autograd.grad(f(ins), ins)
    for i, q in enumerate(ins):
        d = torch.randn(q.shape, generator=gen).to(dev)
        e = 2.0 ** -7
        plus, minus = list(ins), list(ins)
        plus[i], minus[i] = q.detach() + e * d, q.detach() - e * d
        with torch.no_grad():
            num = float((f(plus) - f(minus)) / (2 * e))
        ana = float((grads[i].double() * d).sum())
        scale = float((grads[i].double() * d).norm()) + 1
        # third derivative e^2 / 6 of a direction of unit variance, and fp32 noise 2^-24 * 90 steps / e on sums of 7200 terms
        assert abs(num - ana) <= 2e-2 * scale, (i, num, ana)


def test_partial_gradients_and_refusal_of_a_second_one(dev):
    from neurofluid_amd import scan
    gate, x, gy, _ = make((2, 70, 12), (2, 70, 1), F32, F32, False, 4)
    full = [q.to(dev).requires_grad_() for q in (gate, x)]
    h, last = scan.gated_scan(*full)
    dg, dx = torch.autograd.grad(h, full, gy.to(dev))
    a, b = gate.to(dev).requires_grad_(), x.to(dev)
    assert torch.equal(torch.autograd.grad(scan.gated_scan(a, b)[0], a, gy.to(dev))[0], dg)
    a, b = gate.to(dev), x.to(dev).requires_grad_()
    assert torch.equal(torch.autograd.grad(scan.gated_scan(a, b)[0], b, gy.to(dev))[0], dx)
    h0 = torch.zeros(2, 12, device=dev, requires_grad=True)
    h, last = scan.gated_scan(gate.to(dev), x.to(dev), h0)
    d, = torch.autograd.grad(last, h0, torch.ones_like(last))       # the final state alone
    check("dh0", d, gate.double().expand(2, 70, 12).prod(1), 200 * U * torch.ones(2, 12).double(), F32)
    h, _ = scan.gated_scan(*full)
    g1, = torch.autograd.grad(h.sum(), full[1], create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g1.sum(), full[0])


def test_repeats_bit_for_bit_on_another_stream_and_in_a_graph(dev):
    from neurofluid_amd import scan
    gate, x, gy, gen = make((2, 1500, 40), (2, 1500, 1), BF16, BF16, True, 8)
    g0, x0, y0 = gate.to(dev), x.to(dev), gy.to(dev)
    h00 = torch.randn(2, 40, generator=gen).to(dev)

    def both(g, xx, hh, yy):
        ins = [q.detach().requires_grad_() for q in (g, xx, hh)]
        h, last = scan.gated_scan(*ins, log_gate=True, reverse=True)
        return (h.detach(), last.detach()) + torch.autograd.grad([h, last], ins, [yy, torch.ones_like(last)])
    want = both(g0, x0, h00, y0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = both(g0, x0, h00, y0)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(want, got))
    # two graphs, each with its own workspace, replayed in turns with eager work between
    bufs = [[q.clone() for q in (g0, x0, h00, y0)] for _ in range(2)]
    graphs, outs = [], []
    for b in bufs:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(both(*b))
        graphs.append(gr)
    for it in range(4):
        for k in (0, 1):
            for q in bufs[k][1:2]:
                q.copy_(x0 * (1 + it + 2 * k))
            graphs[k].replay()
        for k in (0, 1):
            eager = both(g0, x0 * (1 + it + 2 * k), h00, y0)
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(eager, outs[k])), (it, k)


@pytest.mark.parametrize("rows, D", [(1, 1), (3, 5), (257, 64), (1000, 33), (0, 4)])
@pytest.mark.parametrize("dtype, gate_kind, log_gate", [(F32, "full", True), (BF16, "full32", False), (F16, "shared", True), (BF16, "shared", False)])
def test_step(dev, rows, D, dtype, gate_kind, log_gate):
    from neurofluid_amd import scan
    gdt = F32 if gate_kind == "full32" else dtype
    gate, x, _, gen = make((rows, D), (rows, 1 if gate_kind == "shared" else D), dtype, gdt, log_gate, rows + D)
    s0 = torch.randn(rows, D, generator=gen)
    A = (torch.exp(gate.double()) if log_gate else gate.double()).expand(rows, D)
    want = A * s0.double() + x.double()
    bound = 4 * U * ((A * s0.double()).abs() + x.double().abs())
    state, out = s0.to(dev), torch.full((rows, D + 3), 7.0, device=dev)
    h = scan.gated_scan_step(gate.to(dev), x.to(dev), state, log_gate=log_gate, out=out[:, :D])
    check("h", h, want, bound, dtype)
    check("out", out[:, :D], want, bound, F32)
    assert torch.equal(state.cpu(), s0) and (out[:, D:] == 7).all()
    h2 = scan.gated_scan_step(gate.to(dev), x.to(dev), state, log_gate=log_gate)
    assert torch.equal(h2, h) and torch.equal(state, out[:, :D])


def test_step_reads_what_it_overwrites(dev):
    """Inputs that lie among the states that are written: the gates a column of theirs, x the states themselves, shifted, or between them."""
    from neurofluid_amd import scan
    g = torch.Generator().manual_seed(21)
    base = torch.rand(300, 3 * 64 + 8, generator=g)

    def views(b):
        s = b[:, :64]
        yield s, b[:, 8:9], b[:, 70:134]              # one gate a row, from the state's own row
        yield s, b[:, 64:128], s                      # x is the state
        yield s, s, s
        yield s, b[:, 4:68], b[:, 1:65]               # shifted
        yield s, b[:, 64:128], b[:, 128:192]          # in the same rows, beside it
        yield b[1:, :64], b[:-1, :64], b[:-1, 64:128]       # a row later
    for k in range(6):
        want = [t.double() for t in list(views(base))[k]]
        want = want[1] * want[0] + want[2]
        state, gate, x = list(views(base.to(dev)))[k]
        keep = state.clone()
        h = scan.gated_scan_step(gate, x, state)
        assert torch.equal(h, state) and not torch.equal(state, keep)
        assert ((h.cpu().double() - want).abs() <= 2.0 ** -23 * want.abs()).all(), k


def test_two_at_once(dev):
    """Chained scans that wait for one another's tiles, on two streams together and with one thread's gradients beside another's."""
    from neurofluid_amd import scan
    g = torch.Generator().manual_seed(22)
    data = [(torch.rand(1, 40000, 96, generator=g).to(dev), torch.randn(1, 40000, 96, generator=g).to(dev)) for _ in range(2)]

    def work(gate, x):
        gate, x = gate.clone().requires_grad_(), x.clone().requires_grad_()
        h, _ = scan.gated_scan(gate, x)
        return (h,) + torch.autograd.grad(h, [gate, x], x.detach())
    want = [work(*d) for d in data]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in data]
    got = [[], []]
    for _ in range(6):
        for k, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[k].append(work(*data[k]))
    torch.cuda.synchronize()
    for k in (0, 1):
        for r in got[k]:
            assert all(torch.equal(a, b) for a, b in zip(r, want[k]))


def test_steps_make_a_scan(dev):
    """Steps on a kept state are the scan (the same fused multiply-adds in the same order inside a stretch: equal up to the carries)."""
    from neurofluid_amd import scan
    gate, x, _, gen = make((5, 50, 24), (5, 50, 24), F32, F32, False, 2)
    h0 = torch.randn(5, 24, generator=gen).to(dev)
    with torch.no_grad():
        h, last = scan.gated_scan(gate.to(dev), x.to(dev), h0)
    s = h0.clone()
    bound = [seq64(gate[b].double(), x[b].double(), h0[b].cpu().double())[2] for b in range(5)]
    for t in range(50):
        o = scan.gated_scan_step(gate[:, t].to(dev), x[:, t].to(dev), s)
        for b in range(5):
            assert ((o[b] - h[b, t]).abs().cpu() <= 2 * bound[b][t]).all()      # either side within E of the exact state
    for b in range(5):
        assert ((s[b] - last[b]).abs().cpu() <= 2 * bound[b][-1]).all()


def test_composites_like_the_renderer(dev):
    """Features composited along rays, towards the eye, equal the volume rendering sum (models/renderer.py:182-208): weights
    alpha_i prod_(j<i) (1 - alpha_j), alpha = 1 - exp(-sigma delta)."""
    from neurofluid_amd import scan
    g = torch.Generator().manual_seed(1)
    R, S, C = 65, 192, 7
    sd = torch.relu(torch.randn(R, S, 1, generator=g)) * 0.3
    f = torch.randn(R, S, C, generator=g)
    alpha = 1 - torch.exp(-sd.double())
    trans = torch.cumprod(torch.cat([torch.ones(R, 1, 1).double(), 1 - alpha[:, :-1]], 1), 1)
    want = (alpha * trans * f.double()).sum(1)
    lg = -sd.to(dev)
    with torch.no_grad():
        h, last = scan.gated_scan(lg, -torch.expm1(lg) * f.to(dev), log_gate=True, reverse=True)
    # 192 samples of magnitude <= 5 with weights that sum to <= 1; 8 u a step as above
    assert (h[:, 0].cpu().double() - want).abs().max() <= 8 * 192 * U * 5
    assert torch.equal(h[:, 0], last)


def test_a_step_behind_a_recorded_scan_is_noticed(dev):
    """The scan's backward reads h0 again: a step that writes there in between makes it refuse, a step into memory of its own does not."""
    from neurofluid_amd import scan
    gate, x, gy, gen = make((2, 40, 8), (2, 40, 8), F32, F32, False, 6)
    g0, x0, y0, s0 = gate.to(dev).requires_grad_(), x.to(dev), gy.to(dev), torch.randn(2, 8, generator=gen).to(dev)

    def run(step):
        s = s0.clone()
        h, last = scan.gated_scan(g0, x0, s)
        with torch.no_grad():
            step(s)
        return torch.autograd.grad(h, g0, y0)[0]
    want = run(lambda s: None)
    assert torch.equal(run(lambda s: scan.gated_scan_step(x0[:, 0], x0[:, 1], s, out=torch.empty_like(s))), want)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        run(lambda s: scan.gated_scan_step(x0[:, 0], x0[:, 1], s))


def test_step_into_the_columns_beside_the_state(dev):
    """State and out as column ranges of one buffer, either way round; what lies between and behind them stays."""
    from neurofluid_amd import scan
    g = torch.Generator().manual_seed(23)
    for D, width, first, second in ((64, 128, 0, 64), (5, 13, 8, 1), (64, 136, 68, 0)):
        base, x = torch.randn(300, width, generator=g), torch.randn(300, D, generator=g)
        gate = torch.rand(300, D, generator=g)
        buf = base.to(dev)
        h = scan.gated_scan_step(gate.to(dev), x.to(dev), buf[:, first:first + D], out=buf[:, second:second + D])
        state = base[:, first:first + D].double()
        assert ((h.cpu().double() - (gate.double() * state + x.double())).abs() <= 4 * U * ((gate * state).abs() + x.abs())).all()
        assert torch.equal(buf[:, second:second + D], h)
        rest = torch.ones(width, dtype=torch.bool)
        rest[second:second + D] = False
        assert torch.equal(buf.cpu()[:, rest], base[:, rest])


def plan_of(B, T, D, dtype, gate32=False, shared=False, packed=False):
    """Mode (0 a wave a chain, 1 chained tiles, 2 a workgroup a chain) and tiles a chain of contiguous tensors of these sizes."""
    import ctypes
    from neurofluid_amd import _lib
    gs = 1 if shared else D
    s = _lib.Scan(dtype=[F32, BF16, F16].index(dtype), gate32=int(gate32), shared=int(shared), B=B, T=T, D=D, x_sb=T * D, x_st=D, gate_sb=T * gs, gate_st=gs,
                  row_splits=8 if packed else None)
    n = ctypes.c_size_t()
    assert _lib.load().nf_scan_plan(ctypes.byref(s), ctypes.byref(n)) == 0
    return s.mode, n.value // (B * D)


def growing(T, D, shared, reverse, gen):
    """Gates of magnitude 2 whose products pass fp32's range many times over, in a sequence whose states and gradients do not: in processing order a gate of
    zero in the first, middle and last third, x in the 20 steps in front of the last two of them and in the last 20, gradients in the first 20 steps
    behind the first and the middle one."""
    gate = torch.where(torch.rand(T, 1 if shared else D, generator=gen) < 0.5, 2.0, -2.0)
    x, g = torch.zeros(T, D), torch.zeros(T, D)
    cuts = [0, T // 2 + 3, T - 25]
    gate[cuts] = 0.0
    for a, b in ((cuts[1] - 20, cuts[1]), (cuts[2] - 20, cuts[2]), (T - 20, T)):
        x[a:b] = torch.randn(b - a, D, generator=gen)
    for a in cuts[:2]:
        g[a:a + 20] = torch.randn(20, D, generator=gen)
    return [q.flip(0) if reverse else q for q in (gate, x, g)]


@pytest.mark.parametrize("B, T, D, dtype, mode", [(4100, 400, 4, F32, 0), (2, 700, 16, BF16, 1), (1, 9001, 64, BF16, 1), (1, 20003, 34, F32, 1), (8, 1030, 1024, BF16, 2)])
@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("reverse", [False, True])
def test_products_of_gates_that_overflow(dev, B, T, D, dtype, mode, shared, reverse):
    """A zero state stays zero under gates above 1, and behind a gate of zero nothing is left, whatever the products of the stretches have become."""
    from neurofluid_amd import scan
    assert plan_of(B, T, D, dtype, shared=shared)[0] == mode
    gen = torch.Generator().manual_seed(T + D)
    ones = [growing(T, D, shared, reverse, gen) for _ in range(2)]
    gate, x, gy = (torch.stack([ones[b % 2][k] for b in range(2)]).to(dtype) for k in range(3))
    idx = torch.arange(B) % 2
    h0 = torch.randn(B, D, generator=gen)
    gd, xd, hd = gate.to(dev)[idx].requires_grad_(), x.to(dev)[idx].requires_grad_(), h0.to(dev).requires_grad_()
    h, last = scan.gated_scan(gd, xd, hd, reverse=reverse)
    gr = torch.autograd.grad([h, last], [gd, xd, hd], [gy.to(dev)[idx], torch.zeros_like(last)])
    for b in sorted({0, min(1, B - 1), B - 1}):
        w = oracle(gate[b % 2].double(), x[b % 2].double(), h0[b].double(), gy[b % 2].double(), torch.zeros(D).double(), False, reverse)
        for name, got, dt in (("h", h, dtype), ("last", last, F32), ("dgate", gr[0], dtype), ("dx", gr[1], dtype), ("dh0", gr[2], F32)):
            check(name, got[b], *w[name], dt)


def test_products_that_overflow_in_packed_rows(dev):
    from neurofluid_amd import scan
    gen = torch.Generator().manual_seed(7)
    lens, D = [700, 0, 3000, 90, 5000], 40
    rs = splits_of(lens)
    parts = [growing(n, D, False, False, gen) if n else [torch.zeros(0, D)] * 3 for n in lens]
    gate, x, gy = (torch.cat([p[k] for p in parts]) for k in range(3))
    h0 = torch.randn(len(lens), D, generator=gen)
    ins = [q.to(dev).requires_grad_() for q in (gate, x, h0)]
    h, last = scan.gated_scan(*ins, row_splits=rs.to(dev))
    gr = torch.autograd.grad([h, last], ins, [gy.to(dev), torch.zeros_like(last)])
    for s, n in enumerate(lens):
        a, b = int(rs[s]), int(rs[s + 1])
        w = oracle(gate[a:b].double(), x[a:b].double(), h0[s].double(), gy[a:b].double(), torch.zeros(D).double(), False, False)
        for name, got in (("h", h[a:b]), ("last", last[s]), ("dgate", gr[0][a:b]), ("dx", gr[1][a:b]), ("dh0", gr[2][s])):
            check(name, got, *w[name], F32)


@pytest.mark.parametrize("B, T, D, dtype, gate_kind, reverse, mode, tiles", [
    (1, 66000, 64, BF16, "full", False, 1, 258), (1, 66000, 64, F16, "shared", True, 1, 258),        # a second set of 256 tiles
    (1, 131500, 9, F32, "full", True, 1, 514), (1, 131500, 9, BF16, "shared", False, 1, 514),         # a third
    (8, 1030, 1024, BF16, "full", False, 2, 5), (8, 1030, 1024, F16, "shared", True, 2, 5), (9, 1100, 1030, F32, "full", False, 2, 5),
    (8, 1030, 1024, BF16, "full32", True, 2, 5)])
def test_many_tiles(dev, B, T, D, dtype, gate_kind, reverse, mode, tiles):
    """Groups of 16 tiles and sets of 16 groups, and the states that sets hand on; workgroups that walk over several tiles.  Both passes."""
    assert plan_of(B, T, D, dtype, gate32=gate_kind == "full32", shared=gate_kind == "shared") == (mode, tiles)
    run_dense(dev, B, T, D, dtype, gate_kind, bool(T & 1) or reverse, reverse, True, seed=T + D)


INTO_GROUPS = ([2500, 0, 7, 900, 1, 64, 1500, 300], 11, 21)                                      # sequences over, into and inside groups
INTO_SETS = ([30000, 0, 5, 700, 1, 20000, 256, 300, 0, 3000, 13000, 17, 1200, 2], 90, 268)        # ... and sets: one crosses row 65 536, three begin behind it


@pytest.mark.parametrize("lens, tail, tiles, dtype, gate_kind, reverse", [
    INTO_GROUPS + (F32, "shared", False), INTO_GROUPS + (F32, "shared", True), INTO_GROUPS + (BF16, "full", False), INTO_GROUPS + (BF16, "full", True),
    INTO_SETS + (F32, "shared", True), INTO_SETS + (BF16, "full", False)])
def test_packed_over_many_tiles(dev, lens, tail, tiles, dtype, gate_kind, reverse):
    from neurofluid_amd import scan
    D, rs = 9, splits_of(lens)
    N, S = int(rs[-1]) + tail, len(lens)
    assert plan_of(1, N, D, dtype, shared=gate_kind == "shared", packed=True) == (1, tiles)
    gate, x, gy, gen = make((N, D), (N, 1 if gate_kind == "shared" else D), dtype, dtype, reverse, N + D)
    h0, gl = torch.randn(S, D, generator=gen), torch.randn(S, D, generator=gen)
    ins = [q.to(dev).requires_grad_() for q in (gate, x, h0)]
    h, last = scan.gated_scan(*ins, log_gate=reverse, reverse=reverse, row_splits=rs.to(dev))
    gr = torch.autograd.grad([h, last], ins, [gy.to(dev), gl.to(dev)])
    h, last, gr = h.detach().cpu(), last.detach().cpu(), [q.cpu() for q in gr]
    for s in range(S):
        a, b = int(rs[s]), int(rs[s + 1])
        w = oracle(gate[a:b].double(), x[a:b].double(), h0[s].double(), gy[a:b].double(), gl[s].double(), reverse, reverse)
        check("h", h[a:b], *w["h"], dtype)
        check("last", last[s], *w["last"], F32)
        check("dgate", gr[0][a:b], *w["dgate"], dtype)
        check("dx", gr[1][a:b], *w["dx"], dtype)
        check("dh0", gr[2][s], *w["dh0"], F32)
    for q in (h, gr[0], gr[1]):
        assert (q[int(rs[-1]):] == 0).all()


@pytest.mark.parametrize("B, T, D, dtype, reverse", [(3, 203, 96, BF16, False), (2, 77, 31, F16, True), (1, 3001, 200, BF16, True)])
def test_one_gate_a_step_in_32_bits_beside_16_bit_rows(dev, B, T, D, dtype, reverse):
    from neurofluid_amd import scan
    gate, x, gy, gen = make((B, T, D), (B, T, 1), dtype, F32, True, T + D)
    h0, gl = torch.randn(B, D, generator=gen), torch.randn(B, D, generator=gen)
    ins = [q.to(dev).requires_grad_() for q in (gate, x, h0)]
    h, last = scan.gated_scan(*ins, log_gate=True, reverse=reverse)
    gr = torch.autograd.grad([h, last], ins, [gy.to(dev), gl.to(dev)])
    assert h.dtype == dtype and [q.dtype for q in gr] == [F32, dtype, F32]
    for b in range(B):
        w = oracle(gate[b].double(), x[b].double(), h0[b].double(), gy[b].double(), gl[b].double(), True, reverse)
        for name, got, dt in (("h", h, dtype), ("last", last, F32), ("dgate", gr[0], F32), ("dx", gr[1], dtype), ("dh0", gr[2], F32)):
            check(name, got[b], *w[name], dt)


def test_packed_rows_in_a_graph(dev):
    """Captured forward and backward of packed rows, replayed over other splits, values and eager work of their own."""
    from neurofluid_amd import scan
    gate, x, gy, gen = make((6000, 40), (6000, 40), BF16, BF16, False, 15)
    cuts = [torch.tensor(c, device=dev) for c in ([0, 100, 100, 5000, 6000], [7, 8, 3000, 3000, 5990], [0, 0, 0, 6000, 6000], [5, 2000, 4000, 4001, 4002])]
    xs = [(x * k).to(dev) for k in (1, 2, 3, 4)]
    g0, y0, h0 = gate.to(dev), gy.to(dev), torch.randn(4, 40, generator=gen).to(dev)

    def both(rs, xx):
        ins = [q.detach().requires_grad_() for q in (g0, xx, h0)]
        h, last = scan.gated_scan(*ins, row_splits=rs)
        return (h.detach(), last.detach()) + torch.autograd.grad([h, last], ins, [y0, torch.ones_like(last)])
    rs, xx = cuts[0].clone(), xs[0].clone()
    both(rs, xx)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both(rs, xx)
    for it in range(6):
        rs.copy_(cuts[it % 4])
        xx.copy_(xs[(it + 1) % 4])
        graph.replay()
        want = both(cuts[it % 4], xs[(it + 1) % 4])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), it


@pytest.mark.parametrize("B, T, D, mode", [(1, 4_200_000, 520, 1), (33, 65536, 1024, 2), (2_200_000, 16, 64, 0)])
def test_gradients_past_32_bit_offsets(dev, B, T, D, mode):
    """Both passes over more than 2^31 elements.  The gradients that enter are zero but for the last rows of the last batch, and gates of
    1/2 forget: there the results are those of the same rows on their own, and in front of them no gradient is left."""
    from neurofluid_amd import scan
    assert B * T * D > 2 ** 31 and plan_of(B, T, D, BF16, shared=True)[0] == mode
    n = min(T, 300)
    x = torch.zeros(B, T, D, dtype=BF16, device=dev)
    x[-1, T - n:].normal_()
    g = torch.zeros_like(x)
    g[-1, T - n + n // 2:].normal_()
    gate = torch.full((B, T, 1), 0.5, dtype=BF16, device=dev).requires_grad_()
    x.requires_grad_()
    h, last = scan.gated_scan(gate, x)
    dgate, dx = torch.autograd.grad(h, [gate, x], g)
    tail = x[-1, T - n:].detach().cpu().double()
    w = oracle(torch.full((n, 1), 0.5).double(), tail, torch.zeros(D).double(), g[-1, T - n:].cpu().double(), torch.zeros(D).double(), False, False)
    check("h", h[-1, T - n:], *w["h"], BF16)
    check("last", last[-1], *w["last"], F32)
    check("dx", dx[-1, T - n:], *w["dx"], BF16)
    check("dgate", dgate[-1, T - n:], *w["dgate"], BF16)
    assert not h[-1, :T - n].any() and not dx[-1, :max(T - 1000, 0)].any() and not dgate[-1, :T - n].any()
    if B > 1:
        assert not h[:-1].any() and not dx[:-1].any() and not last[:-1].any()
