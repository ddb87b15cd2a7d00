"""Layer normalisation, dropout and their residual step in float64 on the CPU, with error bounds for fp32 kernels.

Bounds.  u = 2^-24 is half a step of fp32.  A row's deviations from its mean are formed by a corrected two-pass sum, so
they carry the rounding of one subtraction plus the error of a mean of C small numbers: at most k(C) u (|h| + 1) of a
standard deviation, where k(C) counts the roundings on the longest chain of the sums (C / 64 serial additions of the
widest-striding kernel, the tree behind them, and the dozen operations of the formulas).  Every result is rounded once to
its type (half a step of the value)."""
import torch

U = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
IDS = ["fp32", "bf16", "fp16"]


def half(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """Half of the smallest step the type has (results that are subnormal in it)."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def depth(C):
    return 24 + C / 32


def rows_of(t):
    """(rows, C) float64 view of the elements in memory order: channels of a voxel, or the last axis."""
    t = t.detach().cpu().double()
    t = t.permute(0, 2, 3, 4, 1) if t.dim() == 5 else t
    return t.reshape(-1, t.shape[-1])


def norm(x, w, b, eps):
    mean = x.mean(1, keepdim=True)
    xc = x - mean
    r = 1 / torch.sqrt((xc * xc).mean(1, keepdim=True) + eps)
    h = xc * r
    y = h if w is None else h * w
    return (y if b is None else y + b), h, r


def norm_tol(h, w, b, y, dtype):
    C = h.shape[1]
    aw = 1.0 if w is None else w.abs()
    ab = 0.0 if b is None else b.abs()
    return half(dtype) * y.abs() + tiny(dtype) + U * depth(C) * (aw * (h.abs() + 1) + ab)


def norm_grad(dy, h, r, w):
    """(dx, dw, db) of one call."""
    g = dy if w is None else dy * w
    c1, c2 = g.mean(1, keepdim=True), (g * h).mean(1, keepdim=True)
    return r * (g - c1 - h * c2), (dy * h).sum(0), dy.sum(0)


def dx_tol(dy, h, r, w, dx, dtype):
    """dx = r (g - c1 - h c2): the roundings of the three terms, of the two means, and of h (absolute k u (|h| + 1))."""
    g = (dy if w is None else dy * w).abs()
    C = h.shape[1]
    k = U * depth(C)
    m1, m2 = g.mean(1, keepdim=True), (g * (h.abs() + 1)).mean(1, keepdim=True)
    return half(dtype) * dx.abs() + tiny(dtype) + 2 * k * r * (g + m1 + (h.abs() + 1) * m2)


def param_tol(dy, h, ref, dtype):
    """Column sums over the rows: a chain of at most rows / 128 + 64 additions (fewer rows: at most one each) of terms
    that carry h's own error."""
    R, C = h.shape
    k = U * (depth(C) + min(R, R / 128 + 64) + 16)
    return half(dtype) * ref.abs() + tiny(dtype) + k * (dy.abs() * (h.abs() + 1)).sum(0)


def close(got, ref, tol, what):
    got = got.detach().cpu().double().reshape(ref.shape)
    bad = ~((got - ref).abs() <= tol)
    assert not bool(bad.any()), (
        f"{what}: {int(bad.sum())} of {bad.numel()} outside the bound, worst "
        f"{float(((got - ref).abs() / tol)[bad].max()) if bool(bad.any()) else 0:.3g} x at "
        f"{torch.nonzero(bad)[0].tolist()}: {float(got[bad][0])} for {float(ref[bad][0])}")
