"""The recurrence and 8-bit checkpoint operators: what is measured of them, and their plain forms.

  step        one step of the gated recurrence on a state that is kept between calls     (scan.gated_scan_step)
  scan        the gated recurrence h_t = A_t h_(t-1) + x_t over whole sequences           (scan.gated_scan)
  scan_train  the same with its backward pass                                             (scan.gated_scan under autograd)
  checkpoint  activations to 8 bits and back                                              (act8.pack, Act8.unpack)
  wgrad       a linear layer's weight and bias gradient from its checkpointed input       (act8.pack, act8.wgrad)

Sizes: rays and samples are the renderer's (1024-ray chunks, 64 / 192 samples, 400 x 400 images, 256-wide layers, 2432
activations a row, 252 features a row); the longer sequences and wider layers are generic.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


# ------------------------------------------------------------------------------------------------
# cases
# ------------------------------------------------------------------------------------------------
def _scan_case(kind, B, T, D, dtype, gate, log, reverse=False, h0=True, splits=0, name=None):
    """gate: "full" (a gate per channel), "full32" (the same, in 32 bits beside 16-bit inputs), "shared" (one gate a step).
    splits > 0: B is 1 and the T rows hold that many sequences of uneven length behind one another."""
    case = dict(kind=kind, B=B, T=T, D=D, dtype=dtype, gate=gate, log=log, reverse=reverse, h0=h0, splits=splits)
    return dict(case, name=name) if name else case


def listed():
    return [
        # one more sample for every ray of a 1024-ray chunk, a small feature field: latency
        dict(name="step_chunk", kind="step", rows=1024, D=32, dtype="f32", log=True),
        # one more sample for every pixel of a 400 x 400 image
        dict(name="step_image", kind="step", rows=160000, D=64, dtype="bf16", log=False),
        # an image's rays composited back to front: rgb + one feature, one transmittance a sample, 64 + 128 samples
        _scan_case("scan", 40000, 192, 4, "f32", "shared", True, reverse=True, h0=False, name="composite_image"),
        # hidden states of a few long sequences, inference
        _scan_case("scan", 4, 4096, 1024, "bf16", "full", False, name="sequences"),
        # a training step's rays (4 views x 1024), 32 feature channels composited, with the gradients
        _scan_case("scan_train", 4096, 192, 32, "f32", "shared", True, reverse=True, h0=False, name="composite_train"),
        # a batch of sequences in training, decay in 32 bits as such models keep it
        _scan_case("scan_train", 8, 2048, 2048, "bf16", "full32", True, name="sequences_train"),
        # one very long sequence, few channels: nothing but the length to split
        _scan_case("scan_train", 1, 65537, 256, "f16", "full", False, name="long_train"),
        # sequences of uneven length packed behind one another (empty ones among them), run backwards
        _scan_case("scan_train", 1, 50001, 200, "bf16", "full", False, reverse=True, splits=37, name="packed_train"),
        # the feature rows of one 1024-ray chunk's coarse pass
        dict(name="checkpoint_features", kind="checkpoint", rows=6001, K=252, dtype="f32"),
        # all saved activations of a training pass
        dict(name="checkpoint_activations", kind="checkpoint", rows=63001, K=2432, dtype="f32"),
        # one 256-wide layer of that pass
        dict(name="wgrad_layer", kind="wgrad", rows=63001, M=256, K=256, dtype="f32"),
        # a wide layer in 16 bits
        dict(name="wgrad_wide", kind="wgrad", rows=32768, M=2048, K=2048, dtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["step", "scan", "scan", "scan_train", "scan_train", "scan_train", "checkpoint", "wgrad", "wgrad"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if kind == "step":
        D = _log_int(rng, 1, 2048)
        return dict(kind=kind, rows=_log_int(rng, 1, max(1, min(160000, 10_000_000 // D))), D=D, dtype=dtype, log=rng.random() < 0.5)
    if kind in ("scan", "scan_train"):
        T = _log_int(rng, 1, 65537)
        D = _log_int(rng, 1, 2048)
        most = 30_000_000 if kind == "scan" else 16_000_000
        D = max(1, min(D, most // T))
        B = _log_int(rng, 1, max(1, min(40000, most // (T * D))))
        gate = rng.choice(["full", "shared"] if dtype == "f32" else ["full", "full32", "shared"])
        splits = 0
        if rng.random() < 0.3:
            B, T = 1, max(64, min(B * T, 65537))
            splits = _log_int(rng, 1, 2000)
        return _scan_case(kind, B, T, D, dtype, gate, rng.random() < 0.5, rng.random() < 0.5, rng.random() < 0.5, splits)
    if kind == "checkpoint":
        K = _log_int(rng, 1, 4096)
        return dict(kind=kind, rows=_log_int(rng, 1, 150_000_000 // K), K=K, dtype=dtype)
    M, K = _log_int(rng, 1, 2048), _log_int(rng, 1, 2048)
    return dict(kind=kind, rows=_log_int(rng, 1, min(65536, 130_000_000_000 // (M * K))), M=M, K=K, dtype=dtype)


# ------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------
def _gate(g, shape, dtype, log, dev):
    """Decays from almost none to almost all.  A log gate is -sigma * delta of a field that is empty in most places."""
    u = torch.rand(shape, generator=g, device=dev)
    if log:
        v = -torch.relu(torch.randn(shape, generator=g, device=dev)) * u * 1.5
    else:
        v = torch.sigmoid(6.0 * u - 1.0)
    return v.to(dtype)


def _splits(case, seed):
    """Row splits of `splits` sequences over about 97 % of the rows (the rest lies behind the last one); every fifth is empty."""
    g = torch.Generator().manual_seed(seed + 7)
    n = case["splits"]
    w = torch.rand(n, generator=g, dtype=torch.float64) ** 3 + 1e-3
    if n > 4:
        w[4::5] = 0.0
    ends = torch.floor(torch.cumsum(w, 0) / w.sum() * math.floor(case["T"] * 0.97)).to(torch.int64)
    return torch.cat([torch.zeros(1, dtype=torch.int64), ends])


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    s = dict(case=case)
    if case["kind"] == "step":
        shape = (case["rows"], case["D"])
        s["gate"] = _gate(g, shape, dt, case["log"], dev)
        s["x"] = torch.randn(shape, generator=g, device=dev).to(dt)
        s["state"] = torch.randn(shape, generator=g, device=dev)
        s["next"] = torch.empty_like(s["state"])
    elif case["kind"] in ("scan", "scan_train"):
        B, T, D = case["B"], case["T"], case["D"]
        gdt = torch.float32 if case["gate"] == "full32" else dt
        lead = (T,) if case["splits"] else (B, T)
        nseq = case["splits"] or B
        s["gate"] = _gate(g, lead + ((1,) if case["gate"] == "shared" else (D,)), gdt, case["log"], dev)
        s["x"] = torch.randn(lead + (D,), generator=g, device=dev).to(dt)
        s["h0"] = torch.randn((nseq, D), generator=g, device=dev) if case["h0"] else None
        s["splits"] = _splits(case, seed).to(dev) if case["splits"] else None
        if case["kind"] == "scan_train":
            s["g"] = torch.randn(lead + (D,), generator=g, device=dev).to(dt)
            s["g_last"] = torch.randn((nseq, D), generator=g, device=dev)
            if own:
                for k in ("gate", "x", "h0"):
                    if s[k] is not None:
                        s[k].requires_grad_(True)
    else:
        x = torch.randn((case["rows"], case["K"]), generator=g, device=dev)
        s["x"] = (torch.relu(x) * torch.exp(torch.randn((case["rows"], 1), generator=g, device=dev))).to(dt)
        if case["kind"] == "wgrad":
            s["dy"] = (torch.randn((case["rows"], case["M"]), generator=g, device=dev) * 1e-2).to(dt)
    return s


# ------------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------------
def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    from neurofluid_amd import act8, scan
    case = s["case"]
    kind = case["kind"]
    if kind == "step":
        h = scan.gated_scan_step(s["gate"], s["x"], s["state"], log_gate=case["log"], out=s["next"])
        return h, s["next"]
    if kind == "scan":
        with torch.no_grad():
            return scan.gated_scan(s["gate"], s["x"], s["h0"], log_gate=case["log"], reverse=case["reverse"], row_splits=s["splits"])
    if kind == "scan_train":
        h, last = scan.gated_scan(s["gate"], s["x"], s["h0"], log_gate=case["log"], reverse=case["reverse"], row_splits=s["splits"])
        leaves = [s["gate"], s["x"]] + ([s["h0"]] if s["h0"] is not None else [])
        grads = torch.autograd.grad([h, last], leaves, [s["g"], s["g_last"]])
        return (h.detach(), last.detach()) + tuple(grads)
    if kind == "checkpoint":
        return act8.pack(s["x"]).unpack(s["x"].dtype)
    return act8.wgrad(s["dy"], act8.pack(s["x"]))


def _doubling(A, x, h0, segment):
    """All states of h_t = A_t h_(t-1) + x_t along dim 1, by combining ever longer stretches: (A, x) of the last 2^k steps.
    segment: the sequence that each row of a packed tensor belongs to (h0 has one row for each), or None."""
    T = x.shape[1]
    A = A.expand_as(x)
    if h0 is not None or segment is not None:
        first = torch.zeros(T, dtype=torch.bool, device=x.device)
        if T:
            first[0] = True
        if segment is not None:
            first[1:] = segment[1:] != segment[:-1]
        init = torch.zeros_like(x)
        if h0 is not None and T:
            init = torch.where(first[None, :, None], h0[segment][None] if segment is not None else h0[:, None], init)
        x = x + A * init
        A = torch.where(first[None, :, None], torch.zeros_like(A), A)
    k = 1
    while k < T:
        x = torch.cat([x[:, :k], x[:, k:] + A[:, k:] * x[:, :-k]], 1)
        A = torch.cat([A[:, :k], A[:, k:] * A[:, :-k]], 1)
        k *= 2
    return x


def _plain_scan(s, grads):
    case = s["case"]
    packed = s["splits"] is not None
    gate, x = s["gate"].float(), s["x"].float()
    g = s["g"].float() if grads else None
    h0, g_last = s["h0"], s["g_last"] if grads else None
    N = x.shape[0] if packed else x.shape[1]
    segment = None
    if packed:
        splits = s["splits"]
        rows = torch.arange(N, device=x.device)
        segment = torch.bucketize(rows, splits[1:], right=True)
        n = int((segment < case["splits"]).sum())
        gate, x, segment = gate[None, :n], x[None, :n], segment[:n]
        g = g[None, :n] if grads else None
    if case["reverse"]:
        gate, x = gate.flip(1), x.flip(1)
        g = g.flip(1) if grads else None
        segment = segment.flip(0) if packed else None
    A = torch.exp(gate) if case["log"] else gate
    T = x.shape[1]
    h = _doubling(A, x, h0, segment)
    if packed:
        ends = torch.ones(T, dtype=torch.bool, device=x.device)
        ends[:-1] = segment[1:] != segment[:-1]
        last = h0.clone() if h0 is not None else torch.zeros(case["splits"], x.shape[2], device=x.device)
        last[segment[ends]] = h[0, ends]
    else:
        last = h[:, -1].clone()
    back = (lambda t: t.flip(1)) if case["reverse"] else (lambda t: t)

    def whole(t, dtype):
        t = back(t).to(dtype)
        if packed:
            out = torch.zeros((N,) + t.shape[2:], dtype=dtype, device=t.device)
            out[:t.shape[1]] = t[0]
            return out
        return t

    if not grads:
        return whole(h, s["x"].dtype), last
    # dx_t = g_t + A_(t+1) dx_(t+1), the last step of a sequence with the gradient of its final state
    first = torch.zeros(T, dtype=torch.bool, device=x.device)
    first[0] = True
    g = g.clone()
    if packed:
        first[1:] = segment[1:] != segment[:-1]
        g[0, ends] += g_last[segment[ends]]
        start = h0[segment][None] if h0 is not None else torch.zeros_like(x)
    else:
        g[:, -1] += g_last
        start = h0[:, None].expand_as(x) if h0 is not None else torch.zeros_like(x)
    after = torch.cat([A[:, 1:], torch.zeros_like(A[:, :1])], 1)
    after = torch.where(torch.cat([first[1:], first[:1]])[None, :, None], torch.zeros_like(after), after)
    dx = _doubling(after.flip(1), g.flip(1), None, None).flip(1)
    before = torch.where(first[None, :, None], start, torch.cat([torch.zeros_like(h[:, :1]), h[:, :-1]], 1))
    dgate = dx * before
    if case["log"]:
        dgate = dgate * A
    if case["gate"] == "shared":
        dgate = dgate.sum(2, keepdim=True)
    out = [whole(h, s["x"].dtype), last, whole(dgate, s["gate"].dtype), whole(dx, s["x"].dtype)]
    if h0 is not None:
        if packed:
            dh0 = g_last.clone()
            dh0[segment[first]] = (A * dx)[0, first]
        else:
            dh0 = (A * dx)[:, 0]
        out.append(dh0)
    return tuple(out)


def _plain_codes(x):
    """The values that the 8-bit form of x stands for: e4m3 with one power-of-two scale for every 32 features of a row, the
    smallest that brings the largest finite magnitude to 448 or less, and 2^-110 at least; what is not finite becomes NaN."""
    rows, K = x.shape
    pad = -K % 32
    v = torch.cat([x.float(), x.new_zeros(rows, pad, dtype=torch.float32)], 1).view(rows, -1, 32)
    ok = torch.isfinite(v)
    m, e = torch.frexp(torch.where(ok, v.abs(), torch.zeros_like(v)).amax(2, keepdim=True))
    k = torch.where(m > 0.875, e - 8, e - 9)
    k = torch.where(m == 0, torch.full_like(k, -110), k).clamp(min=-110)
    scale = ((k + 127) << 23).view(torch.float32)        # 2^k by its bits: a power function need not be exact
    q = (torch.where(ok, v, torch.zeros_like(v)) / scale).to(torch.float8_e4m3fn).float() * scale
    q = torch.where(ok, q, torch.full_like(q, float("nan")))
    return q.view(rows, K + pad)[:, :K]


def _run_plain(s):
    case = s["case"]
    kind = case["kind"]
    if kind == "step":
        A = s["gate"].float()
        A = torch.exp(A) if case["log"] else A
        torch.add(A * s["state"], s["x"].float(), out=s["next"])
        return s["next"].to(s["x"].dtype), s["next"]
    if kind in ("scan", "scan_train"):
        return _plain_scan(s, kind == "scan_train")
    q = _plain_codes(s["x"])
    if kind == "checkpoint":
        return q.to(s["x"].dtype)
    dy = s["dy"].float()
    return dy.t() @ q, dy.sum(0)


# ------------------------------------------------------------------------------------------------
# the definition, in 64 bits
# ------------------------------------------------------------------------------------------------
def _pow2(k):
    return ((k.to(torch.int64) + 1023) << 52).view(torch.float64)


def _exact_codes(x):
    rows, K = x.shape
    v = x.double()
    out = torch.empty_like(v)
    for c in range(0, K, 32):
        b = v[:, c:c + 32]
        top = torch.where(torch.isfinite(b), b.abs(), 0.0).amax(1, keepdim=True)
        k = torch.full_like(top, -110.0)
        some = top > 0
        k[some] = torch.ceil(torch.log2(top[some] / 448.0))
        for shift in (-1.0, 1.0):        # (log2 may be off by a rounding next to a whole number)
            k = torch.where(some & (top <= 448.0 * _pow2(k - 1)), k - 1, k) if shift < 0 else torch.where(top > 448.0 * _pow2(k), k + 1, k)
        k = k.clamp(min=-110.0)
        w = b / _pow2(k)
        fine = _pow2(torch.floor(torch.log2(w.abs().nan_to_num(1.0, 1.0, 1.0).clamp(min=2.0 ** -6))) - 3)
        q = torch.round(w / fine) * fine * _pow2(k)
        out[:, c:c + 32] = torch.where(torch.isfinite(b), q, float("nan"))
    return out


def _exact_one(A, x, h0, g, g_last):
    """One batch (n, T, D) of equally long sequences, step by step.  A: (n, T, D)."""
    n, T, D = x.shape
    h = torch.zeros(n, D, dtype=torch.float64, device=x.device) if h0 is None else h0.double()
    start, hs = h, torch.empty(T, n, D, dtype=torch.float64, device=x.device)
    At, xt = A.transpose(0, 1), x.transpose(0, 1)
    for t in range(T):
        torch.addcmul(xt[t], At[t], h, out=hs[t])
        h = hs[t]
    if g is None:
        return hs.transpose(0, 1), h.clone()
    dx = torch.empty_like(hs)
    gt = g.transpose(0, 1)
    u = g_last.double()
    for t in range(T - 1, -1, -1):
        torch.add(gt[t], u, out=dx[t])
        u = At[t] * dx[t]
    before = torch.cat([start[None], hs[:-1]], 0)
    return hs.transpose(0, 1), h.clone(), (dx * before).transpose(0, 1), dx.transpose(0, 1), u


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    s = {k: (v.detach() if torch.is_tensor(v) else v) for k, v in s.items()}
    if kind == "step":
        A = s["gate"].double()
        h = (torch.exp(A) if case["log"] else A) * s["state"].double() + s["x"].double()
        return h, h
    if kind == "checkpoint":
        return _exact_codes(s["x"])
    if kind == "wgrad":
        dy = s["dy"].double()
        return dy.t() @ _exact_codes(s["x"]), dy.sum(0)
    grads = kind == "scan_train"
    gate = s["gate"].double()
    A = torch.exp(gate) if case["log"] else gate
    x = s["x"].double()
    A = A.expand_as(x)
    g = s["g"].double() if grads else None
    flip = (lambda t, d: t.flip(d) if t is not None else None) if case["reverse"] else (lambda t, d: t)
    if s["splits"] is None:
        r = _exact_one(flip(A, 1), flip(x, 1), s["h0"], flip(g, 1), s.get("g_last"))
        r = list(r)
        for i in (0, 2, 3) if grads else (0,):
            r[i] = flip(r[i], 1)
    else:
        splits = s["splits"].tolist()
        n, D = len(splits) - 1, x.shape[1]
        r = [torch.zeros_like(x), torch.zeros(n, D, dtype=torch.float64, device=x.device)]
        r += [torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(r[1])] if grads else []
        # sequences side by side, the shorter ones frozen behind their end: A = 1, x = 0 there changes no state and passes the gradient on
        lens = [b - a for a, b in zip(splits, splits[1:])]
        order = sorted(range(n), key=lambda q: lens[q])
        groups, cur = [], []
        for q in order:
            if cur and (len(cur) + 1) * lens[q] > 2 * sum(lens[p] for p in cur) + lens[q] + 4096:
                groups.append(cur)
                cur = []
            cur.append(q)
        groups.append(cur)
        for qs in groups:
            L = max(lens[q] for q in qs)
            Ag = torch.ones(len(qs), L, D, dtype=torch.float64, device=x.device)
            xg, gg = torch.zeros_like(Ag), torch.zeros_like(Ag)
            for i, q in enumerate(qs):
                a, b = splits[q], splits[q + 1]
                Ag[i, :b - a], xg[i, :b - a] = flip(A[a:b], 0), flip(x[a:b], 0)
                if grads:
                    gg[i, :b - a] = flip(g[a:b], 0)
            h0 = s["h0"][qs] if s["h0"] is not None else None
            if grads:
                # the gradient of the final state enters behind the padding and passes through it unchanged
                part = _exact_one(Ag, xg, h0, gg, s["g_last"][qs])
            else:
                part = _exact_one(Ag, xg, h0, None, None)
            for i, q in enumerate(qs):
                a, b = splits[q], splits[q + 1]
                r[0][a:b] = flip(part[0][i, :b - a], 0)
                r[1][q] = part[1][i]
                if grads:
                    r[2][a:b], r[3][a:b] = flip(part[2][i, :b - a], 0), flip(part[3][i, :b - a], 0)
                    r[4][q] = part[4][i]
    if grads:
        dg = r[2] * A if case["log"] else r[2]
        r[2] = dg.sum(-1, keepdim=True) if case["gate"] == "shared" else dg
        if s["h0"] is None:
            r = r[:4]
    return tuple(r)


# ------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ------------------------------------------------------------------------------------------------
def work(case):
    e = 4 if case["dtype"] == "f32" else 2
    kind = case["kind"]
    if kind == "step":
        n = case["rows"] * case["D"]
        return dict(bytes=n * (3 * e + 8), flops=2 * n)
    if kind in ("scan", "scan_train"):
        n = case["B"] * case["T"] * case["D"]
        ge = 4 if case["gate"] == "full32" else e
        gates = (case["B"] * case["T"] if case["gate"] == "shared" else n) * ge
        state = (case["splits"] or case["B"]) * case["D"] * 4 * (2 if case["h0"] else 1)
        if kind == "scan":
            return dict(bytes=gates + 2 * n * e + state, flops=2 * n)
        return dict(bytes=2 * gates + 4 * n * e + 2 * state, flops=7 * n)
    if kind == "checkpoint":
        n = case["rows"] * case["K"]
        return dict(bytes=2 * n * e, flops=2 * n)
    r, M, K = case["rows"], case["M"], case["K"]
    return dict(bytes=r * (M + K) * e + 4 * M * (K + 1), flops=2 * r * M * K + r * M)
