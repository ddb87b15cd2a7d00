"""Error bounds of the layer-norm kernels that do not grow with the length of a row, and the float64 values they hold for.

u = 2^-24 is half a step of fp32.  Chains of additions, from the kernels (csrc/layer_norm.hip): a lane adds at most two packs
of eight elements (16), the lanes of a wave are a tree (6), the waves of a block one after the other (15): D = 37 roundings at
most for a row in registers.  A long row's chunk has 16 + 6 + 3, its tiles are joined in doubles, its chunks by four additions
a lane and a tree of 6, with each chunk's numbers rounded to fp32 once: fewer.  With the deviations d = x - m0 formed by one
subtraction, sigma the row's standard deviation and |m0 - mean| below sigma / 8 (holds while mean |x| < 5e4 sigma), chunks'
means within sigma of each other:

  mean of d         (D + 3) u mean|d|                                                          <= 44 u sigma
  r                 ((D + 5) / 2 + 1/2 + 4) u r        (sum of d^2, eps, one step or two of rsqrt)  <= 27 u r
  h = d r + dr      u (1 + 27 + 2) |h| + 44 u                                                  <= u (32 |h| + 44)
  y = h w + b       |w| err(h) + 2 u (|h w| + |b|), rounded to its type once
  c1 = mean g       (D + 3) u mean|g|                                                          <= 42 u mean|g|
  c2 = mean(g h)    (D + 5) u mean(|g| (|h| + 1/8)) + 44 u mean|g| + 27 u |c2|
  dx = r (g - c1 - h c2)   r u (34 |g| + 80 mean|g| + 160 (|h| + 1) mean(|g| (|h| + 1))), rounded once

A parameter's gradient adds over the rows: `chain` follows the launch plan (rows a lane sees, the fold of a block, the join of
the blocks' partial sums)."""
import math

import torch

U = 2.0 ** -24


def half(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def rows64(t):
    """(rows, C) float64 of the elements in memory order."""
    t = t.detach().double()
    t = t.permute(0, 2, 3, 4, 1) if t.dim() == 5 else t
    return t.reshape(-1, t.shape[-1])


def cdiv(a, b):
    return -(-a // b)


def plan(R, C, dtype):
    """(rows of a step, steps, parts) of the backward pass over dense rows: how many partial sums, and for rows in registers
    how many steps the blocks walk.  A long row's `step` is one row."""
    size = dtype.itemsize
    packs = cdiv(C, 16 // size)
    if packs <= 64:
        per, threads = 256 >> math.ceil(math.log2(packs)) if packs > 1 else 256, 256
    elif packs <= 1024 or (packs <= 2048 and size == 4):
        nt = 128 if packs <= 128 else 256 if packs <= 256 else 512 if packs <= 512 else 1024
        per = {128: 4, 256: 2}.get(nt, 1)
        threads = nt * per
    else:
        tiles = cdiv(C, 512 * (16 // size))
        return 1, R, max(1, min(cdiv(1024, tiles), R // 8))
    steps = cdiv(R, per)
    cap = (768 if packs <= 64 else 1024) * 256 // threads
    return per, steps, 1 if steps <= 4 else min(max(steps // 4, 256), cap, steps)


def chain(R, C, dtype):
    """Roundings on the longest chain of additions of a parameter's gradient."""
    per, steps, parts = plan(R, C, dtype)
    down = 4 if parts <= 32 else 16 if parts <= 256 or C >= 4096 else 64
    return cdiv(steps, parts) + 6 + 4 + (cdiv(parts, down) + int(math.log2(down)) if parts > 1 else 0)


def norm(x, w, b, eps):
    """(y, h, r) of float64 rows."""
    var, mean = torch.var_mean(x, dim=1, keepdim=True, correction=0)
    r = 1 / torch.sqrt(var + eps)
    h = (x - mean) * r
    y = h if w is None else h * w
    return (y if b is None else y + b), h, r


def h_tol(h):
    return U * (32 * h.abs() + 44)


def y_tol(h, w, b, y, dtype):
    aw = 1.0 if w is None else w.abs()
    ab = 0.0 if b is None else b.abs()
    return half(dtype) * y.abs() + tiny(dtype) + aw * h_tol(h) + 2 * U * (h.abs() * aw + ab)


def grads(dy, h, r, w):
    """(dx, dw, db)."""
    g = dy if w is None else dy * w
    return r * (g - g.mean(1, keepdim=True) - h * (g * h).mean(1, keepdim=True)), (dy * h).sum(0), dy.sum(0)


def dx_tol(dy, h, r, w):
    """Before the rounding to the result's type."""
    g = (dy if w is None else dy * w).abs()
    m1, m2 = g.mean(1, keepdim=True), (g * (h.abs() + 1)).mean(1, keepdim=True)
    return U * r * (34 * g + 80 * m1 + 160 * (h.abs() + 1) * m2)


def dw_tol(dy, h, dw, R, C, dtype, wdtype):
    n = chain(R, C, dtype)
    return half(wdtype) * dw.abs() + tiny(wdtype) + U * (dy.abs() * ((n + 34) * h.abs() + 44)).sum(0)


def db_tol(dy, db, R, C, dtype, wdtype):
    return half(wdtype) * db.abs() + tiny(wdtype) + U * chain(R, C, dtype) * dy.abs().sum(0)


def within(got, ref, tol):
    """Whether every element is inside its bound (NaN is not)."""
    return bool(((got.double().reshape(ref.shape) - ref).abs() <= tol).all())


def check(got, ref, tol, what):
    err = (got.detach().double().reshape(ref.shape) - ref).abs()
    bad = ~(err <= tol)
    n = int(bad.sum())
    assert n == 0, f"{what}: {n} of {bad.numel()} outside the bound, worst {float((err / tol)[bad].max()):.3g} x"


def inputs(R, C, dtype, seed, device="cpu"):
    """(x, dy, w, b): rows off zero, and an upstream gradient with a mean and a part along h, so that both row terms of dx and
    the sums over the rows stand far above their rounding."""
    g = torch.Generator(device=device).manual_seed(seed)
    x = (torch.randn(R, C, generator=g, device=device) * 1.5 + 0.5).to(dtype)
    h = (x.float() - x.float().mean(1, keepdim=True)) / x.float().std(1, keepdim=True, correction=0).clamp_min(1e-3)
    dy = (0.1 * (torch.randn(R, C, generator=g, device=device) + 0.7 * h + 0.5)).to(dtype)
    w = 1 + 0.2 * torch.randn(C, generator=g, device=device)
    b = 0.1 * torch.randn(C, generator=g, device=device)
    return x, dy, w, b
