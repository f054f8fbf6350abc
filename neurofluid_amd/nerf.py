"""Host-side mirror of /root/reference/models/nerf.py (Embedding :4-38, NeRF :42-124).

Same constructors, parameter names and shapes as the reference (released checkpoints load with ``strict=True``), same
``forward`` signatures and results.  Inside RenderNet the two modules are fused away (nf_render_features emits the
encodings straight into the MLP operand layout, nf_nerf_mlp_fwd* consume it); called on their own — a caller that keeps the
reference's ``models/renderer.py`` and swaps only the modules (INTEGRATION.md level 2) — they run the SAME HIP kernels on
row-major tensors: ``nf_embed_fwd`` / ``nf_embed_bwd`` and the fp32-MFMA MLP (``nf_nerf_mlp_fwd`` / ``nf_nerf_mlp_bwd`` /
``nf_nerf_wgrad`` / ``nf_gemm_f32``), with autograd.  There is no torch fallback: CPU tensors raise.
"""
import ctypes

import torch
from torch import nn

from . import _lib, ops
from ._lib import check, ptr


class _EmbedFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, n_freqs):
        lib = _lib.load()
        ops._require_cuda(x)
        C = x.shape[-1]
        xc = x.detach().contiguous().float()
        rows = xc.numel() // max(C, 1)
        out = torch.empty(*x.shape[:-1], C * (2 * n_freqs + 1), dtype=torch.float32, device=x.device)
        check(lib.nf_embed_fwd(ptr(xc), rows, C, n_freqs, ptr(out), _lib.stream()), "nf_embed_fwd")
        ctx.save_for_backward(xc)
        ctx.n_freqs = n_freqs
        return out

    @staticmethod
    def backward(ctx, g):
        (xc,) = ctx.saved_tensors
        lib = _lib.load()
        C = xc.shape[-1]
        gc = g.detach().contiguous().float()
        dx = torch.empty_like(xc)
        check(lib.nf_embed_bwd(ptr(xc), ptr(gc), xc.numel() // max(C, 1), C, ctx.n_freqs, ptr(dx), _lib.stream()), "nf_embed_bwd")
        return dx, None


class Embedding(nn.Module):
    """x -> (x, sin(2^k x), cos(2^k x), ...), k < N_freqs   (models/nerf.py:21-38)."""

    def __init__(self, in_channels, N_freqs, logscale=True):
        super().__init__()
        if not logscale:
            raise NotImplementedError("only logscale=True is used by the hot path (models/nerf.py:16-17)")
        self.N_freqs = N_freqs
        self.in_channels = in_channels
        self.out_channels = in_channels * (2 * N_freqs + 1)
        self.freq_bands = 2 ** torch.linspace(0, N_freqs - 1, N_freqs)

    def forward(self, x):
        """x: (B, in_channels) -> (B, out_channels), column order of models/nerf.py:33-38."""
        if x.shape[-1] != self.in_channels:
            raise ValueError(f"expected {self.in_channels} channels, got {x.shape[-1]}")
        return _EmbedFn.apply(x, self.N_freqs)


def _nerf_param_struct(layers):
    P = _lib.NerfParams()
    keep = []
    for i, l in enumerate(layers):
        w, b = l.weight.detach().contiguous().float(), l.bias.detach().contiguous().float()
        keep += [w, b]
        P.w[i], P.b[i] = w.data_ptr(), b.data_ptr()
    return P, keep


class _NerfFn(torch.autograd.Function):
    """NeRF.forward on (n, cx + cd) row-major rows: forward on the fp32-MFMA kernel with saved activations, backward =
    nf_nerf_mlp_bwd (data gradient) + nf_nerf_wgrad (15 weight GEMMs + bias sums) + three nf_gemm_f32 for dL/dx."""

    @staticmethod
    def forward(ctx, net, x, sigma_only, *params):
        lib = _lib.load()
        cx, cd = net.in_channels_xyz, net.in_channels_dir
        layers = net.linear_layers()
        dev = x.device
        n = x.shape[0]
        xf = x.detach().float()
        if sigma_only:          # models/nerf.py:100-113: only the position features are given; the view branch is not evaluated
            xf = torch.cat([xf, torch.zeros(n, cd, dtype=torch.float32, device=dev)], 1)
        P, keep = _nerf_param_struct(layers)
        packed = torch.empty(lib.nf_nerf_packed_floats(cx, cd), dtype=torch.float32, device=dev)
        check(lib.nf_nerf_pack(ctypes.byref(P), cx, cd, ptr(packed), _lib.stream()), "nf_nerf_pack")
        need = any(ctx.needs_input_grad)          # (grad mode is off inside Function.forward: ask the ctx, not torch)
        X = ops.rows_to_tiles(xf, cx, cd)
        n_rows = torch.tensor([n], dtype=torch.int32, device=dev)
        row_sample = torch.arange(n, dtype=torch.int32, device=dev)
        out = torch.zeros(max(n, 1), 4, dtype=torch.float32, device=dev)[:n]
        acts = torch.empty(max(n, 1) * 2432, dtype=torch.float32, device=dev) if need else None
        ctx.act8 = None
        if need and net.act_checkpoint is not None:
            return _NerfFn._forward_act8(ctx, net, xf, sigma_only, packed, X, n_rows, row_sample, out, acts)
        if n > 0:
            check(lib.nf_nerf_mlp_fwd(ptr(packed), cx, cd, ptr(X), ptr(n_rows), n, ptr(row_sample), ptr(out), ptr(acts),
                                      _lib.stream()), "nf_nerf_mlp_fwd")
        ctx.net, ctx.sigma_only, ctx.n = net, sigma_only, n
        ctx.x_needs_grad = bool(ctx.needs_input_grad[1])
        if need:
            # the transposed blob of the backward is packed NOW, from the weights this forward used: an optimiser step between
            # forward and backward must not pair forward-time activations with newer weights
            from .autograd_bwd import _pack_bwd
            packed_t = _pack_bwd(net, cx, cd, dev)
            ctx.save_for_backward(packed, packed_t, X, n_rows, row_sample, out, acts,
                                  layers[0].weight.detach().clone(), layers[4].weight.detach().clone(), layers[9].weight.detach().clone())
        return out[:, 3:4].clone() if sigma_only else out

    @staticmethod
    def _forward_act8(ctx, net, xf, sigma_only, packed, X, n_rows, row_sample, out, acts):
        """The training forward with what the backward keeps in 8 bits: the activations (2 432 a row) and the feature row as act8, the ReLU masks
        as bits.  `acts` and X go back to the allocator when this returns."""
        from . import act8
        from .autograd_bwd import _pack_bwd
        lib = _lib.load()
        cx, cd, n, dev = net.in_channels_xyz, net.in_channels_dir, xf.shape[0], xf.device
        layers = net.linear_layers()
        amask = torch.empty(max(lib.nf_nerf_amask_words(n), 1), dtype=torch.int32, device=dev)
        if n > 0:
            packed_n = ops.pack_nerf_n(packed, cx, cd)
            check(lib.nf_nerf_mlp_fwd_n2(ptr(packed_n), cx, cd, ptr(X), ptr(n_rows), n, ptr(row_sample), ptr(out), ptr(acts), ptr(amask), _lib.stream()),
                  "nf_nerf_mlp_fwd_n2")
        kept = [act8.pack(acts[:n * 2432].view(n, 2432)), act8.pack(xf[:, :cx]), act8.pack(xf[:, cx:])]
        ctx.act8 = [(k.shape, k.dtype) for k in kept]
        ctx.net, ctx.sigma_only, ctx.n, ctx.x_needs_grad = net, sigma_only, n, bool(ctx.needs_input_grad[1])
        ctx.save_for_backward(packed, _pack_bwd(net, cx, cd, dev), amask, n_rows, row_sample, out, None,
                              layers[0].weight.detach().clone(), layers[4].weight.detach().clone(), layers[9].weight.detach().clone(),
                              *[t for k in kept for t in k.tensors])
        return out[:, 3:4].clone() if sigma_only else out

    @staticmethod
    def _wgrad_act8(ctx, dpre, kept):
        """The 12 weight and 12 bias gradients from the packed activations (first column of dpre, outputs, first feature, features, bias)."""
        from . import act8
        cx, cd = ctx.net.in_channels_xyz, ctx.net.in_channels_dir
        acts8, xyz8, dir8 = [act8.Act8(kept[2 * i], kept[2 * i + 1], *form) for i, form in enumerate(ctx.act8)]
        hidden = [1, 2, 3, 4, 5, 6, 7]
        jobs = [(256 * l, 256, 256 * (l - 1), 256, True) for l in hidden]
        jobs += [(8 * 256, 256, 7 * 256, 256, True), (9 * 256, 128, 8 * 256, 256, True), (2435, 1, 7 * 256, 256, True), (2432, 3, 9 * 256, 128, True)]
        r = act8.wgrad_jobs(dpre, acts8, jobs)
        first, skip = act8.wgrad_jobs(dpre, xyz8, [(0, 256, 0, cx, True), (4 * 256, 256, 0, cx, False)])
        view, = act8.wgrad_jobs(dpre, dir8, [(9 * 256, 128, 0, cd, False)])
        gw = [first[0]] + [q[0] for q in r[:7]] + [q[0] for q in r[7:]]
        gw[4] = torch.cat([skip[0], gw[4]], 1)
        gw[9] = torch.cat([gw[9], view[0]], 1)
        gb = [first[1]] + [q[1] for q in r]
        return gw, gb

    @staticmethod
    def backward(ctx, g):
        from .autograd_bwd import DPRE
        lib = _lib.load()
        st = _lib.stream()
        net, n = ctx.net, ctx.n
        cx, cd = net.in_channels_xyz, net.in_channels_dir
        layers = net.linear_layers()
        packed, packed_t, X, n_rows, row_sample, out, acts, W1, W5, Wd, *kept = ctx.saved_tensors
        dev = out.device
        # sigma_only (models/nerf.py:100-113) never touches xyz_encoding_final / dir_encoding / rgb: the reference leaves their
        # .grad at None (an optimiser with weight decay or moment decay must not step them), so do we
        unused = (8, 9, 11) if ctx.sigma_only else ()
        if n == 0:
            zeros = [None if i in unused else torch.zeros_like(l.weight) for i, l in enumerate(layers)] + \
                    [None if i in unused else torch.zeros_like(l.bias) for i, l in enumerate(layers)]
            return (None, torch.zeros(0, cx if ctx.sigma_only else cx + cd, device=dev) if ctx.x_needs_grad else None, None) + tuple(zeros)
        d_rs = torch.zeros(n, 4, dtype=torch.float32, device=dev)
        if ctx.sigma_only:
            d_rs[:, 3:4] = g.detach().float()
        else:
            d_rs.copy_(g.detach().float())
        dpre = torch.empty(n, DPRE, dtype=torch.float32, device=dev)
        if ctx.act8 is not None:         # X holds the mask words here
            check(lib.nf_nerf_mlp_bwd_n2(ptr(packed), ptr(packed_t), cx, cd, ptr(X), ptr(n_rows), n, ptr(row_sample), ptr(out), ptr(d_rs),
                                         ptr(dpre), st), "nf_nerf_mlp_bwd_n2")
            gw, gb = _NerfFn._wgrad_act8(ctx, dpre, kept)
        else:
            check(lib.nf_nerf_mlp_bwd_n(ptr(packed), ptr(packed_t), cx, cd, ptr(acts), ptr(n_rows), n, ptr(row_sample), ptr(out),
                                        ptr(d_rs), ptr(dpre), st), "nf_nerf_mlp_bwd_n")
            gw, gb = _NerfFn._wgrad(lib, st, layers, dpre, acts, X, cx, cd, n)
        dx = None
        for i in unused:
            gw[i] = gb[i] = None
        if ctx.x_needs_grad:
            dx = torch.empty(n, cx + cd, dtype=torch.float32, device=dev)
            ops.gemm(dpre[:, 0:256], W1, out=dx[:, :cx])
            ops.gemm(dpre[:, 4 * 256:5 * 256], W5[:, :cx], out=dx[:, :cx], accumulate=True)
            ops.gemm(dpre[:, 9 * 256:9 * 256 + 128], Wd[:, 256:], out=dx[:, cx:])
            if ctx.sigma_only:
                dx = dx[:, :cx].contiguous()
        return (None, dx, None) + tuple(gw) + tuple(gb)

    @staticmethod
    def _wgrad(lib, st, layers, dpre, acts, X, cx, cd, n):
        from .autograd_bwd import DPRE
        dev = dpre.device
        nsl = 22          # 46 tiles x 22 row slices = 1 012 waves: one 128 x 128 tile per wave, one wave per SIMD
        blob = torch.empty(lib.nf_nerf_wgrad_floats(cx, cd), dtype=torch.float32, device=dev)
        wsp = torch.empty(lib.nf_nerf_wgrad_workspace_floats(cx, cd, nsl), dtype=torch.float32, device=dev)
        colsum = torch.empty(DPRE, dtype=torch.float32, device=dev)
        check(lib.nf_nerf_wgrad(ptr(dpre), ptr(acts), ptr(X), cx, cd, n, nsl, ptr(wsp), ptr(blob), ptr(colsum), st), "nf_nerf_wgrad")
        gw, o = [], 0
        for l in layers:
            k = l.weight.numel()
            gw.append(blob[o:o + k].view_as(l.weight))
            o += k
        gb = [colsum[k * 256:(k + 1) * 256] for k in range(8)]
        gb += [colsum[8 * 256:9 * 256], colsum[9 * 256:9 * 256 + 128], colsum[2435:2436], colsum[2432:2435]]
        return gw, gb


class NeRF(nn.Module):
    """models/nerf.py:42-124 (D = 8, W = 256, skips = [4]): parameters with the reference's layer names; forward on the
    fp32-MFMA kernels.

    act_checkpoint="e4m3" (not in the reference): what a training forward keeps for the weight gradients — the activations and the feature row — is
    kept in 8 bits (act8): 3.1 KB a row (masks included) instead of 10.8 KB.  Within one call the fp32 activations are there whole until they are
    packed, so the forward's own peak is 14.1 KB a row instead of 10.9: what falls is what several calls, or other layers, hold until the
    backward.  It is this module's own forward that does so; RenderNet's fused passes keep fp32 whatever its networks say.  Outputs and dL/dx are the fp32 path's (heads summed in another
    order: equal to the last bits); the weight gradients are those of the rounded activations.  For the default feature row (198 + 54 features)."""

    act_checkpoint = None            # (modules pickled before there was a choice have none of their own)

    def __init__(self, D=8, W=256, in_channels_xyz=63, in_channels_dir=27, skips=(4,), act_checkpoint=None):
        super().__init__()
        if act_checkpoint not in (None, "e4m3"):
            raise ValueError(f"act_checkpoint must be None or 'e4m3', not {act_checkpoint!r}")
        if act_checkpoint is not None and ((in_channels_xyz + 7) // 8, (in_channels_dir + 7) // 8) != (25, 7):
            raise NotImplementedError("act_checkpoint: the forward that leaves the ReLU masks as bits serves the default feature row (198 + 54)")
        self.act_checkpoint = act_checkpoint
        if D != 8 or W != 256 or tuple(skips) != (4,):
            raise NotImplementedError("the MFMA kernel implements the reference's D=8, W=256, skips=[4] network")
        self.D, self.W, self.skips = D, W, list(skips)
        self.in_channels_xyz, self.in_channels_dir = in_channels_xyz, in_channels_dir
        for i in range(D):
            if i == 0:
                layer = nn.Linear(in_channels_xyz, W)
            elif i in self.skips:
                layer = nn.Linear(W + in_channels_xyz, W)
            else:
                layer = nn.Linear(W, W)
            setattr(self, f"xyz_encoding_{i + 1}", nn.Sequential(layer, nn.ReLU(True)))
        self.xyz_encoding_final = nn.Linear(W, W)
        self.dir_encoding = nn.Sequential(nn.Linear(W + in_channels_dir, W // 2), nn.ReLU(True))
        self.sigma = nn.Linear(W, 1)
        self.rgb = nn.Sequential(nn.Linear(W // 2, 3), nn.Sigmoid())

    def linear_layers(self):
        """The 12 Linear modules in the C-ABI order (nf_nerf_params_t)."""
        return [getattr(self, f"xyz_encoding_{i}")[0] for i in range(1, 9)] + [
            self.xyz_encoding_final, self.dir_encoding[0], self.sigma, self.rgb[0]]

    def forward(self, x, sigma_only=False):
        """x: (B, in_channels_xyz + in_channels_dir) -> (B, 4) = [rgb (after the sigmoid), sigma];
        sigma_only: x is (B, in_channels_xyz) -> sigma (B, 1)   (models/nerf.py:83-124)."""
        want = self.in_channels_xyz + (0 if sigma_only else self.in_channels_dir)
        if x.dim() != 2 or x.shape[1] != want:
            raise ValueError(f"NeRF.forward expects (B, {want}) features, got {tuple(x.shape)}")
        ops._require_cuda(x)
        layers = self.linear_layers()
        params = [l.weight for l in layers] + [l.bias for l in layers]
        return _NerfFn.apply(self, x, bool(sigma_only), *params)
