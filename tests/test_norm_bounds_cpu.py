"""The bounds of tests/norm_bounds.py let fp32 arithmetic pass and mistakes not: a missing term, a tile left out of the
statistics, a block's partial sums or a tail of rows left out of the parameters' gradients."""
import pytest
import torch

from tests import norm_bounds as B

EPS = 1e-5
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
IDS = ["fp32", "bf16", "fp16"]


def fp32(x, dy, w, b):
    """The operator in fp32 arithmetic: corrected two-pass statistics, rounded once."""
    xf, g = x.float(), dy.float() * w
    m0 = xf.mean(1, keepdim=True)
    d = xf - m0
    delta = d.mean(1, keepdim=True)
    r = torch.rsqrt((d * d).mean(1, keepdim=True) - delta * delta + EPS)
    h = d * r - delta * r
    dx = r * (g - g.mean(1, keepdim=True) - h * (g * h).mean(1, keepdim=True))
    return (h * w + b).to(x.dtype), dx.to(x.dtype), (dy.float() * h).sum(0), dy.float().sum(0)


def refs(x, dy, w, b):
    x, dy, w, b = (B.rows64(t) if t.dim() > 1 else t.double() for t in (x, dy, w, b))
    y, h, r = B.norm(x, w, b, EPS)
    return (y, h, r) + B.grads(dy, h, r, w)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("R,C", [(4, 8), (3, 600), (5, 1025), (2, 9001), (1, 614400)])
def test_bounds_reject_a_missing_term(R, C, dtype):
    x, dy, w, b = B.inputs(R, C, dtype, R + C)
    y, h, r, dx, dw, db = refs(x, dy, w, b)
    dy64, w64, b64 = dy.double(), w.double(), b.double()
    y_tol = B.y_tol(h, w64, b64, y, dtype)
    dx_tol = B.dx_tol(dy64, h, r, w64) + B.half(dtype) * dx.abs() + B.tiny(dtype)
    dw_tol = B.dw_tol(dy64, h, dw, R, C, dtype, torch.float32)
    db_tol = B.db_tol(dy64, db, R, C, dtype, torch.float32)
    got = fp32(x, dy, w, b)
    for a, ref, tol in zip(got, (y, dx, dw, db), (y_tol, dx_tol, dw_tol, db_tol)):
        assert B.within(a, ref, tol)
    g = dy64 * w64
    c1, c2 = g.mean(1, keepdim=True), (g * h).mean(1, keepdim=True)
    for wrong in (r * (g - h * c2), r * (g - c1), r * g):
        assert not B.within(wrong.to(dtype), dx, dx_tol)
    assert not B.within((h * w64).to(dtype), y, y_tol)
    assert not B.within(dw * (1 + 1e-4), dw, dw_tol) and not B.within(db * (1 + 1e-4), db, db_tol)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("C,tile", [(9001, 2048), (614400, 2048), (614400, 4096)])
def test_bounds_reject_statistics_without_a_tile(C, tile, dtype):
    x, dy, w, b = B.inputs(1, C, dtype, C)
    y, h, r, dx, dw, db = refs(x, dy, w, b)
    dy64, w64, b64 = dy.double(), w.double(), b.double()
    for at in (0, (C // tile - 1) * tile):
        seen = torch.ones(C, dtype=torch.bool)
        seen[at:at + tile] = False
        part = x.double()[:, seen]
        var, mean = torch.var_mean(part, dim=1, keepdim=True, correction=0)
        rw = 1 / torch.sqrt(var + EPS)
        hw = (x.double() - mean) * rw
        assert not B.within((hw * w64 + b64).to(dtype), y, B.y_tol(h, w64, b64, y, dtype))
        assert not B.within((dy64 * hw).sum(0), dw, B.dw_tol(dy64, h, dw, 1, C, dtype, torch.float32))
        g = dy64 * w64
        c1, c2 = g[:, seen].mean(1, keepdim=True), (g * h)[:, seen].mean(1, keepdim=True)
        tol = B.dx_tol(dy64, h, r, w64) + B.half(dtype) * dx.abs() + B.tiny(dtype)
        assert not B.within((r * (g - c1 - h * c2)).to(dtype), dx, tol)


@pytest.mark.parametrize("R,C,dtype", [(9603, 256, torch.bfloat16), (40001, 64, torch.float32), (20003, 33, torch.float32),
                                       (5003, 601, torch.bfloat16), (300, 9001, torch.float16)])
def test_bounds_reject_missing_partial_sums(R, C, dtype):
    """One block's share of the rows, or the last step's rows, left out of dw and db; both are well outside their bounds."""
    x, dy, w, b = B.inputs(R, C, dtype, R + C)
    y, h, r, dx, dw, db = refs(x, dy, w, b)
    dy64 = dy.double()
    per, steps, parts = B.plan(R, C, dtype)
    assert parts > 1 and steps > parts
    tw, tb = B.dw_tol(dy64, h, dw, R, C, dtype, torch.float32), B.db_tol(dy64, db, R, C, dtype, torch.float32)
    got = fp32(x, dy, w, b)
    assert B.within(got[2], dw, tw) and B.within(got[3], db, tb)
    block = torch.arange(R) // per % parts
    for seen in (block != parts - 1, torch.arange(R) < (steps - 1) * per):
        wrong = (dy64 * h)[seen].sum(0), dy64[seen].sum(0)
        assert not B.within(wrong[0], dw, tw) and not B.within(wrong[1], db, tb)


@pytest.mark.parametrize("C", [100, 1200, 614400])
def test_bounds_do_not_grow_with_the_row(C):
    """The bound of a result is the same multiple of |h| + 1 at every row length."""
    h = torch.ones(1, C, dtype=torch.float64)
    assert float(B.h_tol(h).max()) < 80 * B.U
