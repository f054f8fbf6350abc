"""Activations kept in 8 bits between forward and backward (csrc/nf_act8.hip), and the weight gradients that read them.

What torch autograd keeps for the linear layers of models/nerf.py:55-81 are their inputs, in 32 bits.  ``pack`` keeps them as e4m3 codes with one
power-of-two scale for every 32 features of a row (1.03 bytes a value, off by at most 2^-4 of itself), ``wgrad`` computes dW = dy^T x^ and
db = sum dy from the codes as they are, ``linear`` is the layer that does both, and the module ``NeRF(..., act_checkpoint="e4m3")`` trains on it.
Forward values and the gradients of the inputs are those of the exact activations; only the weights' gradients see the 8 bits.  Codes, what is
unpacked from them and ``wgrad``'s results carry no gradients of their own.
There is no torch fallback: CPU tensors raise.
"""
import ctypes
import math

import torch
from torch.autograd.function import once_differentiable

from . import _lib, ops
from ._lib import check, ptr

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_MAX = 1 << 30
_INT_MAX = (1 << 31) - 1            # what the C entries take (ctypes would keep a larger number's low 32 bits)


def _matrix(t):
    """t's last axis as columns, everything before as rows; columns adjacent (a copy where the layout asks for one)."""
    m = t if t.dim() == 2 else t.reshape(-1, t.shape[-1])
    return m if m.shape[1] <= 1 or m.stride(1) == 1 else m.contiguous()


def _sizes(rows, features):
    """Bytes of the codes and of the scales (nf_act8_code_bytes, nf_act8_scale_bytes)."""
    blocks = (features + 31) // 32
    return 32 * rows * blocks, (rows + 63) // 64 * 64 * blocks


class Act8:
    """A matrix in 8 bits: ``codes`` and ``scales`` (uint8, the layout of nf_act8_pack), ``shape`` and ``dtype`` of what was packed."""

    def __init__(self, codes, scales, shape, dtype):
        self.codes, self.scales, self.shape, self.dtype = codes, scales, tuple(shape), dtype

    @property
    def features(self):
        return self.shape[-1]

    @property
    def rows(self):
        return math.prod(self.shape[:-1])

    @property
    def device(self):
        return self.codes.device

    def _whole(self, what):
        """The kernels read what the shape says: refuse less."""
        codes, scales = self.codes, self.scales
        if self.rows > _MAX or self.shape[-1] > _MAX:
            raise ValueError(f"{what}: more than {_MAX} rows or features")
        sizes = _sizes(self.rows, self.shape[-1])
        if codes.dtype is not torch.uint8 or scales.dtype is not torch.uint8 or codes.numel() < sizes[0] or scales.numel() < sizes[1] or \
                not codes.is_contiguous() or not scales.is_contiguous() or codes.device != scales.device:
            raise ValueError(f"{what}: codes and scales of {self.shape} must be {sizes} adjacent bytes (uint8) on one device, got {codes.dtype} "
                             f"{tuple(codes.shape)} and {scales.dtype} {tuple(scales.shape)}")

    @property
    def tensors(self):
        return self.codes, self.scales

    @property
    def nbytes(self):
        return self.codes.numel() + self.scales.numel()

    def unpack(self, dtype=None):
        """The values that the codes stand for, in ``dtype`` (default: what was packed)."""
        dtype = dtype or self.dtype
        if dtype not in _DTYPES:
            raise TypeError(f"Act8.unpack: float32, bfloat16 or float16, not {dtype}")
        self._whole("Act8.unpack")
        ops._require_cuda(self.codes)
        return _unpack(self.codes, self, dtype)


def pack(x):
    """x (..., K) float32 / bfloat16 / float16 -> Act8.  The scale of a block of 32 features is the smallest power of two (2^-110 at least) that
    brings its largest finite magnitude to 448 or less; codes are rounded to nearest even; values that are not finite become NaN."""
    if x.dtype not in _DTYPES:
        raise TypeError(f"act8.pack: x must be float32, bfloat16 or float16, not {x.dtype}")
    if x.dim() < 1:
        raise ValueError("act8.pack: x needs at least one axis")
    rows = x.numel() // x.shape[-1] if x.shape[-1] else 0
    if rows > _MAX or x.shape[-1] > _MAX:
        raise ValueError(f"act8.pack: more than {_MAX} rows or features")
    ops._require_cuda(x)
    ops._refuse_tangents("act8.pack", x)
    return _pack(x, rows)


@_lib.on_device
def _pack(x, rows):
    shape = x.shape
    K, sizes = shape[-1], _sizes(rows, shape[-1])
    n_codes, n_scales = sizes                         # (multiples of 32)
    both = torch.empty(n_codes + n_scales, dtype=torch.uint8, device=x.device)
    if n_codes:
        m = x if len(shape) == 2 and x.stride(1) == 1 else _matrix(x.detach())
        p = both.data_ptr()
        check(_lib.load().nf_act8_pack(_DTYPES[x.dtype], m.data_ptr(), m.stride(0), rows, K, p, p + n_codes, _lib.raw_stream(x)), "nf_act8_pack")
    codes, scales = both.split_with_sizes(sizes)
    return Act8(codes, scales, shape, x.dtype)


@_lib.on_device
def _unpack(codes, ck, dtype):
    out = torch.empty(ck.shape, dtype=dtype, device=codes.device)
    K = ck.shape[-1]
    check(_lib.load().nf_act8_unpack(_DTYPES[dtype], codes.data_ptr(), ck.scales.data_ptr(), ck.rows, K, out.data_ptr(), K,
                                     _lib.raw_stream(codes)), "nf_act8_unpack")
    return out


def wgrad_jobs(dy, ckpt, jobs):
    """Weight gradients of up to 16 layers that read column ranges of one packed matrix, in one launch: jobs = [(first column of dy, outputs, first
    feature (a multiple of 32), features, with bias)] -> [(dW (outputs, features), db (outputs) or None)], float32."""
    if dy.dtype not in _DTYPES:
        raise TypeError(f"act8.wgrad: dy must be float32, bfloat16 or float16, not {dy.dtype}")
    if not isinstance(ckpt, Act8):
        raise TypeError("act8.wgrad: the activations must be an Act8 (act8.pack)")
    if any(abs(int(v)) > _MAX for job in jobs for v in job[:4]):
        raise ValueError(f"act8.wgrad: a job's numbers pass {_MAX}")
    if dy.dim() < 1 or dy.shape[-1] < 1 or ckpt.features < 1 or dy.numel() // dy.shape[-1] != ckpt.rows:
        raise ValueError(f"act8.wgrad: dy {tuple(dy.shape)} does not fit activations {ckpt.shape}")
    if dy.shape[-1] > _MAX:
        raise ValueError(f"act8.wgrad: more than {_MAX} columns of dy")
    if not 1 <= len(jobs) <= 16:
        raise ValueError("act8.wgrad: 1 to 16 jobs")
    ops._require_cuda(dy)
    ops._refuse_tangents("act8.wgrad", dy)
    if dy.device != ckpt.device:
        raise ValueError("act8.wgrad: dy and the activations are on different devices")
    ckpt._whole("act8.wgrad")
    return _wgrad(dy, ckpt, jobs)


@_lib.on_device
def _wgrad(dy, ckpt, jobs):
    lib = _lib.load()
    m = _matrix(dy.detach())
    js = (_lib.Act8Job * len(jobs))(*[(int(a), int(b), int(c), int(d), int(bool(e))) for a, b, c, d, e in jobs])
    rows, cols, features = ckpt.rows, dy.shape[-1], ckpt.features
    n_dw, n_db = sum(b * d for _, b, _, d, _ in jobs), sum(b for _, b, _, _, e in jobs if e)
    n_ws = lib.nf_act8_wgrad_workspace_floats(rows, cols, features, len(jobs), js)
    ws = torch.empty(n_ws, dtype=torch.float32, device=dy.device) if n_ws else None
    both = torch.empty(n_dw + n_db, dtype=torch.float32, device=dy.device)
    dw, db = both[:n_dw], both[n_dw:]
    check(lib.nf_act8_wgrad(_DTYPES[dy.dtype], m.data_ptr(), m.stride(0), cols, ckpt.codes.data_ptr(), ckpt.scales.data_ptr(), features, rows, len(jobs), js,
                            ptr(ws), dw.data_ptr(), db.data_ptr(), _lib.raw_stream(dy)), "nf_act8_wgrad")
    out, o, q = [], 0, 0
    for _, b, _, d, e in jobs:
        out.append((dw[o:o + b * d].view(b, d), db[q:q + b] if e else None))
        o += b * d
        q += b if e else 0
    return out


def wgrad(dy, ckpt, bias=True):
    """dW = dy^T x^ (M, K) and db = the sum of dy's rows (M) of a linear layer whose input is kept as ``ckpt``, both float32 (db None without
    ``bias``).  dy: (..., M) float32 / bfloat16 / float16, as many rows as were packed.  Products are exact, sums float32 in a fixed order."""
    return wgrad_jobs(dy, ckpt, [(0, dy.shape[-1] if dy.dim() else 0, 0, ckpt.features if isinstance(ckpt, Act8) else 0, bias)])[0]


@_lib.on_device
def _linear(x, weight, bias):
    m, w = _matrix(x.detach()), weight.detach()
    y = torch.empty(m.shape[0], w.shape[0], dtype=torch.float32, device=x.device)
    if bias is not None:
        y.copy_(bias.detach().expand_as(y))
    if m.shape[0]:
        ops.gemm(m, w.t(), out=y, accumulate=bias is not None)
    return y.view(x.shape[:-1] + (w.shape[0],)), m


class _LinearFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias):
        y, m = _linear(x, weight, bias)
        ckpt = pack(m) if ctx.needs_input_grad[1] else None
        ctx.form = ckpt.shape if ckpt is not None else None
        ctx.save_for_backward(weight, *(ckpt.tensors if ckpt is not None else ()))       # (what is saved goes with the backward, not with ctx)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        ops._refuse_tangents("act8.linear's backward", g)
        weight, *kept = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx = dw = db = None
        with torch.cuda.device(g.device):
            m = _matrix(g.detach())
            if need[0]:
                dx = torch.empty(m.shape[0], weight.shape[1], dtype=torch.float32, device=g.device)
                if m.shape[0]:
                    ops.gemm(m, weight.detach(), out=dx)
                dx = dx.view(g.shape[:-1] + (weight.shape[1],))
            if need[1]:
                dw, db = wgrad(m, Act8(*kept, ctx.form, torch.float32), bias=need[2])
            elif need[2]:
                # (a sum by the framework's own product: torch's, over many rows, would leave a memset in a captured graph)
                db = ops.gemm(torch.ones(1, m.shape[0], device=g.device), m)[0] if m.shape[0] else torch.zeros_like(weight[:, 0])
        return dx, dw, db


def linear(x, weight, bias=None):
    """torch.nn.functional.linear on float32 whose input is kept in 8 bits for the backward (4.1 times fewer bytes): y = x W^T + b and dx = dy W run
    on the fp32 matrix pipe (ops.gemm), dW and db are ``wgrad`` of the packed input.  Differentiable once, in reverse mode."""
    for t, name, dims in ((x, "x", None), (weight, "weight", 2), (bias, "bias", 1)):
        if t is None:
            continue
        if t.dtype != torch.float32:
            raise TypeError(f"act8.linear: {name} must be float32, not {t.dtype}")
        if dims is not None and t.dim() != dims:
            raise ValueError(f"act8.linear: {name} must have {dims} axes, got {tuple(t.shape)}")
    if x.dim() < 1 or x.shape[-1] != weight.shape[1] or weight.numel() == 0 or (bias is not None and bias.shape[0] != weight.shape[0]):
        raise ValueError(f"act8.linear: x {tuple(x.shape)}, weight {tuple(weight.shape)}"
                         + (f", bias {tuple(bias.shape)}" if bias is not None else "") + " do not fit")
    if max(x.numel() // x.shape[-1], *weight.shape) > _INT_MAX:
        raise ValueError(f"act8.linear: more than {_INT_MAX} rows or features")
    if any(t is not None and t.device != x.device for t in (weight, bias)):
        raise ValueError("act8.linear: x, weight and bias are on different devices")
    ops._require_cuda(x)
    ops._refuse_tangents("act8.linear", x, weight, bias)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias)):
        return _LinearFn.apply(x, weight, bias)
    return _linear(x, weight, bias)[0]
