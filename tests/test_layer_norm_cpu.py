"""Layer norm and mask-free dropout without a GPU: refusals of the C entry points (checked before anything is
launched) and of the tensor-level calls, and the float64 oracle of the GPU tests against difference quotients."""
import ctypes

import pytest
import torch

from tests import norm_oracle as N

PTR = ctypes.c_void_p(4096)      # never dereferenced: every call below is refused first
NULL = None


@pytest.fixture(scope="module")
def lib():
    from siv import _lib
    return _lib.load()


def refused(lib, rc, word, code=-1):
    assert rc == code, (rc, lib.siv_last_error())
    assert word in lib.siv_last_error(), lib.siv_last_error()


def ln_fwd(lib, x=PTR, ldx=8, w=PTR, b=PTR, wt=0, eps=1e-5, y=PTR, t=0, rows=4, C=8, ws=NULL, wsb=0):
    return lib.siv_layer_norm_fwd(x, ldx, w, b, wt, eps, y, t, rows, C, ws, wsb, None)


def ln_bwd(lib, dy=PTR, lddy=8, x=PTR, ldx=8, w=PTR, wt=0, eps=1e-5, dx=PTR, dw=PTR, db=PTR, acc=0, t=0, rows=4, C=8,
           ws=PTR, wsb=1 << 20):
    return lib.siv_layer_norm_bwd(dy, lddy, x, ldx, w, wt, eps, dx, dw, db, acc, t, rows, C, ws, wsb, None)


@pytest.mark.parametrize("over,word", [
    ({"x": NULL}, b"null"), ({"y": NULL}, b"null"), ({"rows": 0}, b"positive"), ({"rows": -1}, b"positive"),
    ({"C": 0}, b"positive"), ({"C": -5, "ldx": 8}, b"positive"), ({"C": 1 << 31, "ldx": 1 << 31}, b"positive"),
    ({"ldx": 7}, b"stride"), ({"t": 3}, b"type"), ({"t": -1}, b"type"), ({"wt": 1}, b"weights"),
    ({"t": 1, "wt": 2}, b"weights"), ({"eps": -1e-5}, b"eps"), ({"eps": float("nan")}, b"eps")])
def test_forward_refuses(lib, over, word):
    refused(lib, ln_fwd(lib, **over), word)


@pytest.mark.parametrize("over,word", [
    ({"dy": NULL}, b"null"), ({"x": NULL}, b"null"), ({"dx": NULL, "dw": NULL, "db": NULL}, b"null"),
    ({"lddy": 3}, b"stride"), ({"ldx": 3}, b"stride"), ({"rows": 0}, b"positive"), ({"t": 9}, b"type"),
    ({"wt": 2}, b"weights")])
def test_backward_refuses(lib, over, word):
    refused(lib, ln_bwd(lib, **over), word)


def test_backward_refuses_a_short_workspace(lib):
    n = ctypes.c_size_t(0)
    assert lib.siv_layer_norm_workspace(5000, 640, 0, 1, ctypes.addressof(n)) == 0 and n.value > 0
    refused(lib, ln_bwd(lib, rows=5000, C=640, ldx=640, lddy=640, wsb=n.value - 1), b"workspace", -2)
    refused(lib, ln_bwd(lib, rows=5000, C=640, ldx=640, lddy=640, ws=NULL, wsb=n.value), b"workspace")
    refused(lib, lib.siv_layer_norm_workspace(0, 640, 0, 1, ctypes.addressof(n)), b"workspace")
    refused(lib, lib.siv_layer_norm_workspace(4, 640, 0, 1, None), b"workspace")
    refused(lib, lib.siv_layer_norm_workspace(4, 640, 7, 1, ctypes.addressof(n)), b"workspace")


@pytest.mark.parametrize("rows,C", [(1, 1), (3, 70000), (5_000_000, 64), (2, (1 << 31) - 1), ((1 << 40) - 1, 2)])
def test_workspace_is_bounded(lib, rows, C):
    """No more scratch than 8 tensors' worth of the parameters' gradients per compute unit and 64 bytes a row."""
    n = ctypes.c_size_t(0)
    for t in range(3):
        for bwd in (0, 1):
            assert lib.siv_layer_norm_workspace(rows, C, t, bwd, ctypes.addressof(n)) == 0
            assert n.value <= 8 * 256 * 8 * min(C, rows * C) + 64 * rows + (1 << 20)


@pytest.mark.parametrize("p", [-0.1, 1.0, 1.5, float("nan")])
def test_dropout_refuses_p(lib, p):
    refused(lib, lib.siv_dropout_fwd(PTR, NULL, NULL, 1, 2, NULL, p, 1.0, PTR, 0, 10, None), b"dropout p")
    refused(lib, lib.siv_dropout_bwd(PTR, NULL, NULL, 1, 2, NULL, p, 1.0, PTR, 0, 10, None), b"dropout p")
    refused(lib, lib.siv_add_layer_norm_fwd(PTR, PTR, NULL, 1, 2, NULL, p, PTR, PTR, 0, 1e-5, PTR, PTR, 0, 4, 8, NULL, 0,
                                            None), b"dropout p")
    refused(lib, lib.siv_add_layer_norm_bwd(PTR, NULL, PTR, NULL, 1, 2, NULL, p, PTR, 0, 1e-5, PTR, PTR, PTR, PTR, 0, 0, 4,
                                            8, PTR, 1 << 20, None), b"dropout p")


def test_dropout_refuses(lib):
    refused(lib, lib.siv_dropout_fwd(NULL, NULL, NULL, 1, 2, NULL, 0.5, 1.0, PTR, 0, 10, None), b"bad argument")
    refused(lib, lib.siv_dropout_fwd(PTR, NULL, NULL, 1, 2, NULL, 0.5, 1.0, NULL, 0, 10, None), b"bad argument")
    refused(lib, lib.siv_dropout_fwd(PTR, NULL, NULL, 1, 2, NULL, 0.5, 1.0, PTR, 0, 0, None), b"bad argument")
    refused(lib, lib.siv_dropout_fwd(PTR, NULL, NULL, 1, 2, NULL, 0.5, 1.0, PTR, 3, 10, None), b"type")
    refused(lib, lib.siv_dropout_bwd(PTR, NULL, NULL, 1, 2, NULL, 0.5, 0.2, PTR, 0, 10, None), b"needs x")
    refused(lib, lib.siv_add_layer_norm_fwd(PTR, NULL, NULL, 1, 2, NULL, 0.5, PTR, PTR, 0, 1e-5, PTR, PTR, 0, 4, 8, NULL,
                                            0, None), b"null")
    refused(lib, lib.siv_add_layer_norm_bwd(NULL, PTR, PTR, NULL, 1, 2, NULL, 0.5, PTR, 0, 1e-5, PTR, PTR, PTR, PTR, 0, 0,
                                            4, 8, PTR, 1 << 20, None), b"null")


def test_tensor_calls_refuse_cpu_tensors_and_types():
    import siv.backend as sb
    from siv import ops, rng
    sb.set_backend(None)
    assert ops.draws_masks()
    x = torch.zeros(2, 8)
    for call in (lambda t: ops.layer_norm(t), lambda t: ops.dropout(t, rng.PhiloxKeep(1, 2), 0.5),
                 lambda t: ops.add_layer_norm(t, t), lambda t: ops.act_dropout(t, 0.0, rng.PhiloxKeep(1, 2), 0.5)):
        with pytest.raises(Exception, match="no CPU fallback"):
            call(x)
        with pytest.raises(Exception, match="unsupported dtype"):
            call(x.double())
        with pytest.raises(Exception, match="unsupported dtype"):
            call(x.long())


@pytest.mark.parametrize("C", [1, 2, 3, 16])
def test_oracle_gradients_are_difference_quotients(C):
    """<dx, v>, <dw, v>, <db, v> of the float64 formulas against central differences of the float64 forward pass: step
    1e-5, so truncation ~1e-10 and rounding ~1e-11 of the values."""
    g = torch.Generator().manual_seed(C)
    rnd = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)
    x, w, b, dy = rnd(5, C), 1 + 0.2 * rnd(C), rnd(C), rnd(5, C)
    eps, e = 1e-2, 1e-5
    f = lambda x, w, b: float((N.norm(x, w, b, eps)[0] * dy).sum())
    _, h, r = N.norm(x, w, b, eps)
    dx, dw, db = N.norm_grad(dy, h, r, w)
    vx, vw, vb = rnd(5, C), rnd(C), rnd(C)
    assert abs((f(x + e * vx, w, b) - f(x - e * vx, w, b)) / (2 * e) - float((dx * vx).sum())) < 1e-6 * r.max() ** 3
    assert abs((f(x, w + e * vw, b) - f(x, w - e * vw, b)) / (2 * e) - float((dw * vw).sum())) < 1e-8
    assert abs((f(x, w, b + e * vb) - f(x, w, b - e * vb)) / (2 * e) - float((db * vb).sum())) < 1e-8
