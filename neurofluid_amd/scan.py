"""Gated linear recurrence over sequences (csrc/nf_scan.hip): h_t = A_t h_{t-1} + x_t.

The renderer's compositing (models/renderer.py:182-208; nf_composite_fwd / _bwd) is this recurrence for three channels, run towards the eye with
the gate 1 - alpha.  Here channels, gates and direction are the caller's: features of any width composited along rays
(``reverse=True, log_gate=True``, gate = -sigma * delta, x = (1 - exp(gate)) * feature: ``h[:, 0]`` is the ray's value), or states carried
over the frames of a sequence.  There is no torch fallback: CPU tensors raise.
"""
import ctypes
import struct

import torch
from torch.autograd.function import once_differentiable

from . import _lib, ops
from ._lib import check

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_MAX_STEPS, _MAX_CHANNELS, _MAX_STRIDE = 1 << 30, 1 << 20, 1 << 17
_INT_MAX = (1 << 31) - 1            # what the C entry takes (ctypes would keep a larger number's low 32 bits)


def _rows(t):
    """t with adjacent channels and steps that are not too far apart (a copy if they are)."""
    if (t.shape[-1] == 1 or t.stride(-1) == 1) and (t.stride(-2) <= _MAX_STRIDE or t.shape[-2] <= 1):
        return t
    return t.contiguous()


def _check(gate, x, what):
    dtype, shape = x.dtype, x.shape
    if dtype not in _DTYPES:
        raise TypeError(f"{what}: x must be float32, bfloat16 or float16, not {dtype}")
    if len(shape) < 2:
        raise ValueError(f"{what}: x needs an axis of steps or rows and one of channels, got {tuple(shape)}")
    if gate.dtype is not dtype and gate.dtype is not torch.float32:
        raise TypeError(f"{what}: the gate must have x's dtype or float32, not {gate.dtype}")
    if gate.shape != shape and (gate.dim() != len(shape) or gate.shape[:-1] != shape[:-1] or gate.shape[-1] != 1):
        raise ValueError(f"{what}: gate {tuple(gate.shape)} does not fit x {tuple(shape)} (same shape, or one gate a step: last axis 1)")
    if shape[-1] < 1:
        raise ValueError(f"{what}: x has no channels")
    if gate.device != x.device:
        raise ValueError(f"{what}: gate and x are on different devices")


def _check_state(t, shape, x, what, name):
    if t.dtype is not torch.float32 or t.shape != shape or t.device != x.device:
        raise ValueError(f"{what}: {name} must be float32 {shape} on {x.device}, got {t.dtype} {tuple(t.shape)} on {t.device}")


_PACK = struct.Struct("9i4x6P6q7P3i4xPN")          # nf_scan_t's fields, in order


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _describe(gate, x, row_splits, opts, plan, **p):
    """nf_scan_t, packed in one go (35 ctypes fields one by one take longer than the launch)."""
    log_gate, reverse = opts
    if row_splits is None:
        B, T, D = x.shape
        n_seq, splits = 0, 0
        (gsb, gst, _), (xsb, xst, _) = gate.stride(), x.stride()
    else:
        B, (T, D) = 1, x.shape
        n_seq, splits = row_splits.numel() - 1, row_splits.data_ptr()
        gsb = xsb = 0
        gst, xst = gate.stride(0), x.stride(0)
    get = p.get
    ysb, yst = get("strides", (0, 0))
    buf = bytearray(_PACK.size)
    _PACK.pack_into(buf, 0, _DTYPES[x.dtype], gate.dtype is torch.float32, gate.shape[-1] == 1, log_gate, reverse, B, T, D, n_seq, splits, gate.data_ptr(),
                    x.data_ptr(), get("g", 0), get("h0", 0), get("g_last", 0), gsb, gst, xsb, xst, ysb, yst, get("h", 0), get("h_last", 0), get("states", 0),
                    get("sid", 0), get("dgate", 0), get("dx", 0), get("dh0", 0), *plan, 0, 0)
    return _lib.Scan.from_buffer(buf)


def _run(lib, s, backward, x):
    n = lib.nf_scan_workspace_bytes(s, backward)
    if n:
        ws = torch.empty(n, dtype=torch.uint8, device=x.device)          # (alive until the launches are enqueued)
        s.workspace, s.workspace_bytes = ws.data_ptr(), n
    if backward:
        check(lib.nf_scan_bwd(s, _lib.raw_stream(x)), "nf_scan_bwd")
    else:
        check(lib.nf_scan_fwd(s, _lib.raw_stream(x)), "nf_scan_fwd")


@_lib.on_device
def _forward(x, gate, h0, row_splits, opts, keep):
    """-> h, h_last and what the backward needs besides the inputs: (states, sid, plan)."""
    lib = _lib.load()
    dev = x.device
    x, gate = _rows(x), _rows(gate)
    if h0 is not None:
        h0 = h0.contiguous()
    packed = row_splits is not None
    D = x.shape[-1]
    n_state = row_splits.numel() - 1 if packed else x.shape[0]
    h = torch.empty(x.shape, dtype=x.dtype, device=dev)
    if not packed and x.shape[0] * x.shape[1] == 0:
        last = torch.zeros(n_state, D, dtype=torch.float32, device=dev) if h0 is None else h0.clone()
        return h, last, (None, None, (0, 0, 0))
    last = torch.empty((n_state, D), dtype=torch.float32, device=dev)
    sid = torch.empty(x.shape[0], dtype=torch.int32, device=dev) if packed else None
    s = _describe(gate, x, row_splits, opts, (0, 0, 0), h=h.data_ptr(), h_last=last.data_ptr(), h0=_ptr(h0), sid=_ptr(sid))
    n_states = ctypes.c_size_t()
    check(lib.nf_scan_plan(s, n_states), "nf_scan_plan")
    states = None
    if keep:
        states = torch.empty(n_states.value, dtype=torch.float32, device=dev)
        s.states = states.data_ptr()
    _run(lib, s, 0, x)
    return h, last, (states, sid, (s.vec, s.cg, s.mode))


class _ScanFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gate, x, h0, row_splits, opts):
        ctx.set_materialize_grads(False)
        h, last, (states, sid, plan) = _forward(x, gate, h0, row_splits, opts, True)
        ctx.save_for_backward(gate, x, h0, row_splits, states, sid)
        ctx.opts, ctx.plan = opts, plan
        return h, last

    @staticmethod
    @once_differentiable
    def backward(ctx, g, g_last):
        ops._refuse_tangents("gated_scan's backward", g, g_last)
        gate, x, h0, row_splits, states, sid = ctx.saved_tensors
        return _backward(x, gate, h0, row_splits, states, sid, g, g_last, ctx.opts, ctx.plan, ctx.needs_input_grad) + (None, None)


@_lib.on_device
def _backward(x, gate, h0, row_splits, states, sid, g, g_last, opts, plan, need):
    lib = _lib.load()
    dev = x.device
    x, gate = _rows(x), _rows(gate)
    h0 = None if h0 is None else h0.contiguous()
    g_last = None if g_last is None else g_last.contiguous()
    packed = row_splits is not None
    n_state = row_splits.numel() - 1 if packed else x.shape[0]
    dgate = torch.empty(gate.shape, dtype=gate.dtype, device=dev) if need[0] else None
    dx = torch.empty(x.shape, dtype=x.dtype, device=dev) if need[1] else None
    dh0 = torch.empty((n_state, x.shape[-1]), dtype=torch.float32, device=dev) if need[2] else None
    if not packed and x.shape[0] * x.shape[1] == 0:
        if dh0 is not None:
            dh0.copy_(g_last) if g_last is not None else dh0.zero_()
        return dgate, dx, dh0
    strides = (0, 0)
    if g is not None:
        g, vec = _rows(g), plan[0]
        if vec > 1 and (g.data_ptr() % (vec * g.element_size()) or any(v % vec for v in g.stride()[:-1])):
            g = g.clone(memory_format=torch.contiguous_format)
        strides = (0, g.stride(0)) if packed else g.stride()[:2]
    s = _describe(gate, x, row_splits, opts, plan, g=_ptr(g), strides=strides, g_last=_ptr(g_last), h0=_ptr(h0), states=_ptr(states), sid=_ptr(sid),
                  dgate=_ptr(dgate), dx=_ptr(dx), dh0=_ptr(dh0))
    _run(lib, s, 1, x)
    return dgate, dx, dh0


def gated_scan(gate, x, h0=None, *, log_gate=False, reverse=False, row_splits=None):
    """Every state of h_t = A_t h_{t-1} + x_t and the final ones: (h like x, h_last float32).

    x: (B, T, D) float32 / bfloat16 / float16.  gate: x's shape, or (B, T, 1) for one gate a step; x's dtype or float32.  A = gate, or exp(gate)
    with ``log_gate``.  h0: (B, D) float32 initial states (zeros if None).  ``reverse`` runs t from T - 1 to 0 (h_last is then the
    state at t = 0).  ``row_splits`` (n_seq + 1 int64, ascending, on the device; the CSR row splits of fixed_radius_search): x is (N, D), its rows
    row_splits[s] : row_splits[s + 1] are sequence s, h0 and h_last are (n_seq, D); an empty sequence hands its h0 through, and h is zero on
    rows that belong to no sequence.

    Sums, states and the carries between stretches are float32; h is rounded once.  Gates are meant to be decays, |A| <= 1.  States are carried over long
    stretches by the product of the gates: where that passes float32's range, a state that is not zero goes on as infinite even if step by step it would
    not; where it has reached zero, an infinite state goes on as NaN.  Differentiable once, in reverse mode, in gate, x and h0; the backward reads gate and x again (they are kept), not h."""
    what = "gated_scan"
    _check(gate, x, what)
    packed = row_splits is not None
    if x.dim() != (2 if packed else 3):
        raise ValueError(f"{what}: x must be {'(N, D) with row_splits' if packed else '(B, T, D)'}, got {tuple(x.shape)}")
    if packed:
        if row_splits.dtype != torch.int64 or row_splits.dim() != 1 or row_splits.numel() < 1 or row_splits.device != x.device:
            raise ValueError(f"{what}: row_splits must be a non-empty 1-d int64 tensor on {x.device}")
        row_splits = row_splits.contiguous()
        if row_splits.numel() > _MAX_STEPS:
            raise ValueError(f"{what}: more than {_MAX_STEPS} sequences")
    if x.shape[-2] > _MAX_STEPS or (not packed and x.shape[0] > _MAX_STEPS) or x.shape[-1] > _MAX_CHANNELS:
        raise ValueError(f"{what}: more than {_MAX_STEPS} steps or sequences, or than {_MAX_CHANNELS} channels")
    if h0 is not None:
        _check_state(h0, (row_splits.numel() - 1 if packed else x.shape[0], x.shape[-1]), x, what, "h0")
    ops._require_cuda(gate, x)
    ops._refuse_tangents(what, gate, x, h0)
    opts = (bool(log_gate), bool(reverse))
    if torch.is_grad_enabled() and (gate.requires_grad or x.requires_grad or (h0 is not None and h0.requires_grad)):
        return _ScanFn.apply(gate, x, h0, row_splits, opts)
    return _forward(x, gate, h0, row_splits, opts, False)[:2]


def gated_scan_step(gate, x, state, *, log_gate=False, out=None):
    """One step for every row: the new state A * state + x goes to ``out`` (by default into ``state`` itself), its value in x's dtype is returned.

    x: (rows, D); gate: x's shape or (rows, 1); state, out: (rows, D) float32 with adjacent channels.  x and gate may lie in the same memory.  For inference: no gradients.
    What is written counts as changed in place: a backward that still needs the old state refuses to run."""
    what = "gated_scan_step"
    _check(gate, x, what)
    if x.dim() != 2:
        raise ValueError(f"{what}: x must be (rows, D), got {tuple(x.shape)}")
    if torch.is_grad_enabled() and (gate.requires_grad or x.requires_grad or state.requires_grad or (out is not None and out.requires_grad)):
        raise RuntimeError(f"{what} carries no gradients (use gated_scan, or torch.no_grad())")
    shape = x.shape
    rows, D = shape
    if rows > _INT_MAX or D > _INT_MAX:
        raise ValueError(f"{what}: more than {_INT_MAX} rows or channels")
    a, sa, na = _states(state, shape, rows, D, x, what, "state")
    b, sb, nb = (a, sa, na) if out is None else _states(out, shape, rows, D, x, what, "out")
    if (a != b or (sa != sb and rows > 1)) and a < b + nb and b < a + na and not (rows > 1 and sa == sb and 4 * D <= (b - a) % (4 * sa) <= 4 * (sa - D)):
        # (the last: rows equally far apart, out's columns beside the state's in every one of them)
        raise ValueError(f"{what}: out overlaps state without being it")
    ops._require_cuda(gate, x)
    ops._refuse_tangents(what, gate, x, state, out)
    h = _step(x, gate, a, sa, b, sb, rows, D, bool(log_gate))
    # the kernel writes through the pointer, which autograd's check of saved tensors and caches keyed on the version would not see
    torch.autograd.graph.increment_version(state if out is None else out)
    return h


def _states(t, shape, rows, D, x, what, name):
    _check_state(t, shape, x, what, name)
    s0, s1 = t.stride()
    if (D > 1 and s1 != 1) or (rows > 1 and s0 < D):
        raise ValueError(f"{what}: {name} needs adjacent channels and rows that do not overlap")
    return t.data_ptr(), s0, 4 * ((rows - 1) * s0 + D)


def _apart(t, out, out_stride, rows, D):
    """A copy of an input that lies among the states that are written, unless it is them, element for element."""
    p, s = t.data_ptr(), t.stride(0)
    if p >= out + 4 * ((rows - 1) * out_stride + D) or out >= p + t.element_size() * ((rows - 1) * s + t.shape[1]):
        return t
    if p == out and t.shape[1] == D and t.dtype is torch.float32 and (s == out_stride or rows == 1):
        return t
    return t.clone(memory_format=torch.contiguous_format)


@_lib.on_device
def _step(x, gate, state, state_stride, out, out_stride, rows, D, log_gate):
    (gs, g1), (xs, x1) = gate.stride(), x.stride()
    shared = gate.shape[1] == 1
    if (g1 != 1 and not shared) or gs > _MAX_STRIDE:
        gate = _rows(gate)
        gs = gate.stride(0)
    if x1 != 1 or xs > _MAX_STRIDE:
        x = _rows(x)
        xs = x.stride(0)
    gp, xp = gate.data_ptr(), x.data_ptr()
    end = out + 4 * (rows * out_stride + D)            # (generous bounds; _apart looks closer)
    if gp < end and out < gp + 4 * (rows * gs + D):
        gate = _apart(gate, out, out_stride, rows, D)
        gp, gs = gate.data_ptr(), gate.stride(0)
    if xp < end and out < xp + 4 * (rows * xs + D):
        x = _apart(x, out, out_stride, rows, D)
        xp, xs = x.data_ptr(), x.stride(0)
    dtype = x.dtype
    h = torch.empty_like(x) if xs == D and x1 == 1 else torch.empty((rows, D), dtype=dtype, device=x.device)       # (the former in half the time)
    if rows:
        check(_lib.load().nf_scan_step(_DTYPES[dtype], gate.dtype is torch.float32, shared, log_gate, rows, D, gp, gs, xp, xs, state, state_stride,
                                       out, out_stride, h.data_ptr(), _lib.raw_stream(x)), "nf_scan_step")
    return h
