"""Gated linear recurrence over sequences (csrc/nf_scan.hip): h_t = A_t h_{t-1} + x_t.

The renderer's compositing (models/renderer.py:182-208; nf_composite_fwd / _bwd) is this recurrence for three channels, run towards the eye with
the gate 1 - alpha.  Here channels, gates and direction are the caller's: features of any width composited along rays
(``reverse=True, log_gate=True``, gate = -sigma * delta, x = (1 - exp(gate)) * feature: ``h[:, 0]`` is the ray's value), or states carried
over the frames of a sequence.  There is no torch fallback: CPU tensors raise.
"""
import ctypes

import torch
from torch.autograd.function import once_differentiable

from . import _lib, ops
from ._lib import check, ptr

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_MAX_STEPS, _MAX_CHANNELS, _MAX_STRIDE = 1 << 30, 1 << 20, 1 << 18


def _rows(t):
    """t with adjacent channels and steps that are not too far apart (a copy if they are)."""
    if (t.shape[-1] == 1 or t.stride(-1) == 1) and (t.stride(-2) <= _MAX_STRIDE or t.shape[-2] <= 1):
        return t
    return t.contiguous()


def _check(gate, x, what):
    if x.dtype not in _DTYPES:
        raise TypeError(f"{what}: x must be float32, bfloat16 or float16, not {x.dtype}")
    if gate.dtype not in (x.dtype, torch.float32):
        raise TypeError(f"{what}: the gate must have x's dtype or float32, not {gate.dtype}")
    if gate.shape != x.shape and (gate.dim() != x.dim() or gate.shape[:-1] != x.shape[:-1] or gate.shape[-1] != 1):
        raise ValueError(f"{what}: gate {tuple(gate.shape)} does not fit x {tuple(x.shape)} (same shape, or one gate a step: last axis 1)")
    if x.shape[-1] < 1:
        raise ValueError(f"{what}: x has no channels")
    if gate.device != x.device:
        raise ValueError(f"{what}: gate and x are on different devices")


def _check_state(t, shape, x, what, name):
    if t.dtype is not torch.float32 or t.shape != shape or t.device != x.device:
        raise ValueError(f"{what}: {name} must be float32 {shape} on {x.device}, got {t.dtype} {tuple(t.shape)} on {t.device}")


def _describe(gate, x, row_splits, log_gate, reverse):
    s = _lib.Scan()
    packed = row_splits is not None
    s.dtype, s.gate32 = _DTYPES[x.dtype], int(gate.dtype == torch.float32)
    s.shared, s.log_gate, s.reverse = int(gate.shape[-1] == 1), int(log_gate), int(reverse)
    s.B, s.T, s.D = (1,) + tuple(x.shape) if packed else tuple(x.shape)
    s.n_seq = row_splits.numel() - 1 if packed else 0
    s.row_splits, s.gate, s.x = ptr(row_splits), ptr(gate), ptr(x)
    s.gate_sb, s.gate_st = (0, gate.stride(0)) if packed else (gate.stride(0), gate.stride(1))
    s.x_sb, s.x_st = (0, x.stride(0)) if packed else (x.stride(0), x.stride(1))
    return s


def _workspace(lib, s, backward, dev):
    s.workspace_bytes = lib.nf_scan_workspace_bytes(s, backward)
    ws = torch.empty(s.workspace_bytes, dtype=torch.uint8, device=dev) if s.workspace_bytes else None
    s.workspace = ptr(ws)
    return ws


@_lib.on_device
def _forward(x, gate, h0, row_splits, log_gate, reverse, keep):
    """-> h, h_last and what the backward needs besides the inputs: (states, sid, plan)."""
    lib = _lib.load()
    dev = x.device
    s = _describe(gate, x, row_splits, log_gate, reverse)
    n_state = s.n_seq if row_splits is not None else s.B
    h = torch.empty(x.shape, dtype=x.dtype, device=dev)
    if s.B == 0 or (s.T == 0 and row_splits is None):
        last = torch.zeros(n_state, s.D, dtype=torch.float32, device=dev) if h0 is None else h0.clone()
        return h, last, (None, None, (0, 0, 0))
    last = torch.empty(n_state, s.D, dtype=torch.float32, device=dev)
    n_states = ctypes.c_size_t()
    check(lib.nf_scan_plan(s, n_states), "nf_scan_plan")
    states = torch.empty(n_states.value, dtype=torch.float32, device=dev) if keep else None
    sid = torch.empty(s.T, dtype=torch.int32, device=dev) if row_splits is not None else None
    s.h0, s.h, s.h_last, s.states, s.sid = ptr(h0), h.data_ptr(), last.data_ptr(), ptr(states), ptr(sid)
    ws = _workspace(lib, s, 0, dev)              # noqa: F841  (alive until the launches are enqueued)
    check(lib.nf_scan_fwd(s, _lib.raw_stream(x)), "nf_scan_fwd")
    return h, last, (states, sid, (s.vec, s.cg, s.mode))


class _ScanFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gate, x, h0, row_splits, log_gate, reverse):
        ctx.set_materialize_grads(False)
        h, last, (states, sid, plan) = _forward(_rows(x.detach()), _rows(gate.detach()), None if h0 is None else h0.detach().contiguous(),
                                                row_splits, log_gate, reverse, True)
        ctx.save_for_backward(gate, x, h0, row_splits, states, sid)
        ctx.opts, ctx.plan = (log_gate, reverse), plan
        return h, last

    @staticmethod
    @once_differentiable
    def backward(ctx, g, g_last):
        gate, x, h0, row_splits, states, sid = ctx.saved_tensors
        return _backward(_rows(x.detach()), _rows(gate.detach()), None if h0 is None else h0.detach().contiguous(), row_splits, states, sid, g, g_last,
                         ctx.opts, ctx.plan, ctx.needs_input_grad) + (None, None, None)


@_lib.on_device
def _backward(x, gate, h0, row_splits, states, sid, g, g_last, opts, plan, need):
    lib = _lib.load()
    dev = x.device
    gl = None if g_last is None else g_last.detach().contiguous()
    s = _describe(gate, x, row_splits, *opts)
    s.vec, s.cg, s.mode = plan
    n_state = s.n_seq if row_splits is not None else s.B
    dgate = torch.empty(gate.shape, dtype=gate.dtype, device=dev) if need[0] else None
    dx = torch.empty(x.shape, dtype=x.dtype, device=dev) if need[1] else None
    dh0 = torch.empty(n_state, s.D, dtype=torch.float32, device=dev) if need[2] else None
    if s.B == 0 or (s.T == 0 and row_splits is None):
        if dh0 is not None:
            dh0.copy_(gl) if gl is not None else dh0.zero_()
        return dgate, dx, dh0
    y = None
    if g is not None:
        y = _rows(g.detach())
        if y.data_ptr() % (s.vec * y.element_size()) or any(v % s.vec for v in y.stride()[:-1]):
            y = y.clone(memory_format=torch.contiguous_format)
        s.g_sb, s.g_st = (0, y.stride(0)) if row_splits is not None else (y.stride(0), y.stride(1))
    s.g, s.h0, s.g_last, s.states, s.sid = ptr(y), ptr(h0), ptr(gl), ptr(states), ptr(sid)
    s.dgate, s.dx, s.dh0 = ptr(dgate), ptr(dx), ptr(dh0)
    ws = _workspace(lib, s, 1, dev)              # noqa: F841
    check(lib.nf_scan_bwd(s, _lib.raw_stream(x)), "nf_scan_bwd")
    return dgate, dx, dh0


def gated_scan(gate, x, h0=None, *, log_gate=False, reverse=False, row_splits=None):
    """Every state of h_t = A_t h_{t-1} + x_t and the final ones: (h like x, h_last float32).

    x: (B, T, D) float32 / bfloat16 / float16.  gate: x's shape, or (B, T, 1) for one gate a step; x's dtype or float32.  A = gate, or exp(gate)
    with ``log_gate``.  h0: (B, D) float32 initial states (zeros if None).  ``reverse`` runs t from T - 1 to 0 (h_last is then the
    state at t = 0).  ``row_splits`` (n_seq + 1 int64, ascending, on the device; the CSR row splits of fixed_radius_search): x is (N, D), its rows
    row_splits[s] : row_splits[s + 1] are sequence s, h0 and h_last are (n_seq, D); an empty sequence hands its h0 through, and h is zero on
    rows that belong to no sequence.

    Sums, states and the carries between stretches are float32; h is rounded once.  Gates are meant to be decays, |A| <= 1: products of larger ones over long
    stretches overflow.  Differentiable once in gate, x and h0; the backward reads gate and x again (they are kept), not h."""
    what = "gated_scan"
    _check(gate, x, what)
    packed = row_splits is not None
    if x.dim() != (2 if packed else 3):
        raise ValueError(f"{what}: x must be {'(N, D) with row_splits' if packed else '(B, T, D)'}, got {tuple(x.shape)}")
    if packed:
        if row_splits.dtype != torch.int64 or row_splits.dim() != 1 or row_splits.numel() < 1 or row_splits.device != x.device:
            raise ValueError(f"{what}: row_splits must be a non-empty 1-d int64 tensor on {x.device}")
        row_splits = row_splits.contiguous()
    if x.shape[-2] > _MAX_STEPS or (not packed and x.shape[0] > _MAX_STEPS) or x.shape[-1] > _MAX_CHANNELS:
        raise ValueError(f"{what}: more than {_MAX_STEPS} steps or sequences, or than {_MAX_CHANNELS} channels")
    if h0 is not None:
        _check_state(h0, (row_splits.numel() - 1 if packed else x.shape[0], x.shape[-1]), x, what, "h0")
    ops._require_cuda(gate, x)
    if torch.is_grad_enabled() and (gate.requires_grad or x.requires_grad or (h0 is not None and h0.requires_grad)):
        return _ScanFn.apply(gate, x, h0, row_splits, bool(log_gate), bool(reverse))
    return _forward(_rows(x.detach()), _rows(gate.detach()), None if h0 is None else h0.detach().contiguous(), row_splits, log_gate, reverse, False)[:2]


def gated_scan_step(gate, x, state, *, log_gate=False, out=None):
    """One step for every row: the new state A * state + x goes to ``out`` (by default into ``state`` itself), its value in x's dtype is returned.

    x: (rows, D); gate: x's shape or (rows, 1); state, out: (rows, D) float32 with adjacent channels.  For inference: no gradients."""
    what = "gated_scan_step"
    _check(gate, x, what)
    if x.dim() != 2:
        raise ValueError(f"{what}: x must be (rows, D), got {tuple(x.shape)}")
    if torch.is_grad_enabled() and (gate.requires_grad or x.requires_grad or state.requires_grad):
        raise RuntimeError(f"{what} carries no gradients (use gated_scan, or torch.no_grad())")
    rows, D = x.shape
    span = []
    for t, name in ((state, "state"),) if out is None else ((state, "state"), (out, "out")):
        _check_state(t, x.shape, x, what, name)
        s0, s1 = t.stride()
        if (D > 1 and s1 != 1) or (rows > 1 and s0 < D):
            raise ValueError(f"{what}: {name} needs adjacent channels and rows that do not overlap")
        span.append((t.data_ptr(), s0, 4 * ((rows - 1) * s0 + D)))
    (a, sa, na), (b, sb, nb) = span[0], span[-1]
    if (a != b or (sa != sb and rows > 1)) and a < b + nb and b < a + na:
        raise ValueError(f"{what}: out overlaps state without being it")
    ops._require_cuda(gate, x)
    return _step(x, gate, a, sa, b, sb, log_gate)


@_lib.on_device
def _step(x, gate, state, state_stride, out, out_stride, log_gate):
    g_, x_ = _rows(gate), _rows(x)
    rows, D = x.shape
    h = torch.empty((rows, D), dtype=x.dtype, device=x.device)
    if rows:
        check(_lib.load().nf_scan_step(_DTYPES[x.dtype], gate.dtype is torch.float32, gate.shape[1] == 1, bool(log_gate), rows, D, g_.data_ptr(),
                                       g_.stride(0), x_.data_ptr(), x_.stride(0), state, state_stride, out, out_stride, h.data_ptr(),
                                       _lib.raw_stream(x)), "nf_scan_step")
    return h
