"""The 8-bit form of activations by its definition, in float64 on the CPU (exact halving and doubling)."""
import torch


def quantised(x):
    """The values that the codes of x (rows, K) stand for."""
    v = x.double()
    rows, K = v.shape
    out = torch.empty_like(v)
    for c in range(0, K, 32):
        b = v[:, c:c + 32]
        fin = torch.isfinite(b)
        top = torch.where(fin, b.abs(), torch.zeros_like(b)).amax(1, keepdim=True) if b.shape[1] else torch.zeros(rows, 1).double()
        k = torch.full((rows, 1), -110, dtype=torch.int64)
        for _ in range(240):
            k = torch.where(top > 448 * torch.exp2(k.double()), k + 1, k)
        s = torch.exp2(k.double())
        # (magnitudes above 1.875 2^127 would round to 2^128, which fp32 does not hold: they are taken as that)
        w = torch.where(fin, b.clamp(-1.875 * 2.0 ** 127, 1.875 * 2.0 ** 127), b) / s
        step = torch.full_like(w, 2.0 ** -9)                # spacing of e4m3 at |w|: subnormals below 2^-6
        for e in range(-6, 9):
            step = torch.where(w.abs() >= 2.0 ** e, torch.full_like(w, 2.0 ** (e - 3)), step)
        q = torch.round(torch.where(fin, w, torch.zeros_like(w)) / step) * step * s          # torch.round: half to even
        out[:, c:c + 32] = torch.where(fin, q, torch.full_like(q, float("nan")))
    return out
