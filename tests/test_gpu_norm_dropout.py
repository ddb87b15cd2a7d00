"""Layer norm, dropout that draws its mask, and their residual step on the device against float64 formulas
(tests/norm_oracle.py, where the bounds are derived)."""
import gc

import pytest
import torch

from tests import norm_oracle as N

pytestmark = pytest.mark.gpu
CL3D = torch.channels_last_3d


@pytest.fixture(autouse=True, params=["nodes", "python"])
def hip(request):
    """The backend, with its native autograd nodes and with the Python autograd functions only."""
    import siv.backend as sb
    sb.set_backend(None)
    b = sb.get_backend()
    nodes = b.nodes
    assert nodes is not None, "siv/_siv_torch.so is not built"
    if request.param == "python":
        b.nodes = None
    yield b
    b.nodes = nodes


def ops():
    from siv import ops as o
    return o


def key(seed=5, sid=11, epoch=None):
    from siv import rng
    return rng.PhiloxKeep(seed, sid, epoch)


def rnd(seed, *shape, scale=1.0, offset=0.0, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale + offset).to(dtype)


def mask_rows(B, shape, p, k):
    """The stored mask of a key, as (rows, C) float64 in memory order."""
    five = shape if len(shape) == 5 else (1, 1, 1, 1, int(torch.Size(shape).numel()))
    m = B.dropout_keep(five, torch.device("cuda"), p, k.seed, k.stream_id, k.epoch)
    m = m.permute(0, 2, 3, 4, 1).reshape(-1, shape[1]) if len(shape) == 5 else m.reshape(-1, shape[-1])
    return m.cpu().double()


def scale_of(p):
    one = torch.tensor(1.0)
    return float(one / (one - torch.tensor(p, dtype=torch.float32)))


# ---- layer norm -------------------------------------------------------------------------------------------------------
ROWS = [(1, 1), (3, 1), (5, 2), (7, 3), (1, 4), (9, 5), (4, 7), (33, 8), (65, 12), (17, 16), (300, 31), (129, 32),
        (70, 33), (257, 64), (31, 96), (64, 100), (1031, 128), (40, 150), (19, 255), (530, 256), (23, 257), (3, 500),
        (12, 512), (6, 513), (4, 600), (77, 601), (5, 1000), (37, 1024), (9, 1025), (1, 1200), (6, 2048), (3, 2049),
        (7, 4096), (3, 4097), (2, 5000), (3, 8192), (5, 8200), (2, 16384), (3, 19201), (8, 38400), (1, 65536),
        (2, 100003), (1, 614400), (20000, 8), (4097, 20)]


def check_norm(x, dy, w, b, eps, dtype, wdtype):
    o = ops()
    xd = x.detach().requires_grad_()
    wd, bd = (None if t is None else t.detach().requires_grad_() for t in (w, b))
    y = o.layer_norm(xd, wd, bd, eps)
    assert y.dtype == dtype and y.shape == x.shape
    leaves = [t for t in (xd, wd, bd) if t is not None]
    grads = dict(zip([n for n, t in (("x", xd), ("w", wd), ("b", bd)) if t is not None],
                     torch.autograd.grad(y, leaves, dy)))
    x64, dy64 = N.rows_of(x), N.rows_of(dy)
    w64, b64 = (None if t is None else t.detach().cpu().double() for t in (w, b))
    ref, h, r = N.norm(x64, w64, b64, eps)
    N.close(N.rows_of(y), ref, N.norm_tol(h, w64, b64, ref, dtype), "y")
    dx, dw, db = N.norm_grad(dy64, h, r, w64)
    N.close(N.rows_of(grads["x"]), dx, N.dx_tol(dy64, h, r, w64, dx, dtype), "dx")
    assert grads["x"].dtype == dtype
    for n, t, g in (("w", w, dw), ("b", b, db)):
        if t is not None:
            assert grads[n].dtype == wdtype
            N.close(grads[n], g, N.param_tol(dy64, h, g, wdtype), "d" + n)
    return y, grads


@pytest.mark.parametrize("dtype", N.DTYPES, ids=N.IDS)
@pytest.mark.parametrize("R,C", ROWS)
def test_layer_norm_rows(R, C, dtype):
    x = rnd(R + C, R, C, scale=1.5, offset=0.5, dtype=dtype).cuda()
    dy = rnd(2 * R + C, R, C, scale=0.1, dtype=dtype).cuda()
    w, b = (1 + 0.2 * rnd(3, C)).cuda(), rnd(4, C, scale=0.1).cuda()
    check_norm(x, dy, w, b, 1e-5, dtype, torch.float32)


@pytest.mark.parametrize("dtype", N.DTYPES, ids=N.IDS)
@pytest.mark.parametrize("what", ["none", "weight", "bias", "own_type"])
@pytest.mark.parametrize("R,C", [(5, 64), (9, 203), (3, 1200), (2, 9001)])
def test_layer_norm_parameters(R, C, what, dtype):
    x, dy = rnd(1, R, C, dtype=dtype).cuda(), rnd(2, R, C, dtype=dtype).cuda()
    wdt = dtype if what == "own_type" else torch.float32
    w = (1 + 0.2 * rnd(3, C)).to(wdt).cuda() if what in ("weight", "own_type") else None
    b = rnd(4, C).to(wdt).cuda() if what in ("bias", "own_type") else None
    check_norm(x, dy, w, b, 1e-5, dtype, wdt)


@pytest.mark.parametrize("dtype", N.DTYPES, ids=N.IDS)
@pytest.mark.parametrize("shape", [(2, 64, 3, 4, 5), (1, 7, 5, 6, 5), (3, 256, 2, 1, 2), (2, 1, 4, 4, 4), (1, 600, 1, 1, 1)])
def test_layer_norm_channels_of_volumes(shape, dtype):
    x = rnd(1, *shape, dtype=dtype).cuda()
    dy = rnd(2, *shape, dtype=dtype).cuda()
    w, b = (1 + 0.2 * rnd(3, shape[1])).cuda(), rnd(4, shape[1]).cuda()
    y1, g1 = check_norm(x.contiguous(memory_format=CL3D), dy.contiguous(memory_format=CL3D), w, b, 1e-5, dtype, torch.float32)
    y2, g2 = check_norm(x, dy, w, b, 1e-5, dtype, torch.float32)          # NCDHW memory is brought into order first
    assert torch.equal(y1, y2) and all(torch.equal(g1[n], g2[n]) for n in g1)
    assert y1.is_contiguous(memory_format=CL3D)
    # against the rows of the same memory
    y3 = ops().layer_norm(x.permute(0, 2, 3, 4, 1).reshape(-1, shape[1]), w, b)
    assert torch.equal(y1.permute(0, 2, 3, 4, 1).reshape(-1, shape[1]), y3)


@pytest.mark.parametrize("dtype", N.DTYPES, ids=N.IDS)
@pytest.mark.parametrize("C", [8, 65, 600, 5000])
def test_layer_norm_slices_of_wider_rows(C, dtype):
    wide, dwide = rnd(1, 6, 2 * C + 3, dtype=dtype).cuda(), rnd(2, 6, 2 * C + 3, dtype=dtype).cuda()
    w, b = (1 + 0.2 * rnd(3, C)).cuda(), rnd(4, C).cuda()
    keep = wide.clone()
    for lo in (0, 1, 3, C):
        y, g = check_norm(wide[:, lo:lo + C], dwide[:, lo + 1:lo + 1 + C], w, b, 1e-5, dtype, torch.float32)
    assert torch.equal(wide, keep)
    # every second row, a transposed tensor, a broadcast one, and channel slices of a volume
    check_norm(wide[::2, :C], dwide[1::2, :C], w, b, 1e-5, dtype, torch.float32)
    t = rnd(5, C, 9, dtype=dtype).cuda().t()
    check_norm(t, rnd(6, 9, C, dtype=dtype).cuda(), w, b, 1e-5, dtype, torch.float32)
    e = rnd(7, 1, C, dtype=dtype).cuda().expand(4, C)
    check_norm(e, rnd(8, 4, C, dtype=dtype).cuda(), w, b, 1e-5, dtype, torch.float32)
    v = rnd(9, 2, 2 * C, 2, 3, 2, dtype=dtype).cuda().contiguous(memory_format=CL3D)
    check_norm(v[:, C:], rnd(10, 2, C, 2, 3, 2, dtype=dtype).cuda(), w, b, 1e-5, dtype, torch.float32)


def test_row_views_take_no_copy(hip):
    x = torch.zeros(6, 20, device="cuda")
    for v, ld in ((x, 20), (x[:, 3:9], 20), (x[::2], 40), (x[2:3, 4:8], 4), (x.view(2, 3, 20)[..., :5], 20)):
        t, got = hip._row_view(v, v.shape[-1])
        assert t.data_ptr() == v.data_ptr() and got == ld, (v.shape, got, ld)
    vol = torch.zeros(2, 8, 3, 4, 5, device="cuda").contiguous(memory_format=CL3D)
    t, got = hip._row_view(vol[:, 2:5], 3)
    assert t.data_ptr() == vol[:, 2:5].data_ptr() and got == 8
    for v in (x.t(), x[:, ::2], x[:1].expand(6, 20), x.view(2, 3, 20)[:, :2]):
        t, got = hip._row_view(v, v.shape[-1])
        assert t.data_ptr() != v.data_ptr() and got == v.shape[-1] and torch.equal(t, v)


@pytest.mark.parametrize("dtype", N.DTYPES, ids=N.IDS)
@pytest.mark.parametrize("C", [1, 3, 8, 100, 700])
def test_layer_norm_rows_far_apart(C, dtype):
    """Rows 2^21 and more elements apart (a step of many rows no longer spans 31-bit offsets), and one pair 2^30 apart."""
    w, b = (1 + 0.2 * rnd(3, C)).cuda(), rnd(4, C).cuda()
    for R, ld in ((9, (1 << 21) + 8), (5, (1 << 21) - 3), (2, (1 << 30) + 1)):
        base, dbase = (torch.zeros((R - 1) * ld + C + 64, dtype=dtype, device="cuda") for _ in range(2))
        x, dy = (t[3:].as_strided((R, C), (ld, 1)) for t in (base, dbase))
        x.copy_(rnd(1, R, C, scale=1.5, offset=0.5, dtype=dtype))
        dy.copy_(rnd(2, R, C, dtype=dtype))
        check_norm(x, dy, w, b, 1e-5, dtype, torch.float32)
        del base, dbase, x, dy


@pytest.mark.parametrize("dtype", N.DTYPES, ids=N.IDS)
def test_layer_norm_stays_in_its_rows(dtype):
    """Results of short calls inside larger buffers: nothing before, behind or between is written."""
    from siv import backend as sb
    lib, st = sb.get_backend().lib, torch.cuda.current_stream().cuda_stream
    t = sb.HipBackend._TYPES[dtype]
    for R, C, off in ((3, 5, 1), (2, 64, 8), (5, 130, 3), (1, 4099, 1), (2, 9000, 5)):
        x, w = rnd(1, R * C + 64, dtype=dtype).cuda(), torch.ones(C, device="cuda")
        out = torch.full((R * C + 64,), 7.0, dtype=dtype, device="cuda")
        es = x.element_size()
        ws = torch.empty(1 << 22, dtype=torch.uint8, device="cuda")
        rc = lib.siv_layer_norm_fwd(x.data_ptr() + off * es, C, w.data_ptr(), None, 0, 1e-5, out.data_ptr() + off * es, t, R,
                                    C, ws.data_ptr(), ws.numel(), st)
        assert rc == 0
        assert bool((out[:off] == 7).all()) and bool((out[off + R * C:] == 7).all())
        x64 = N.rows_of(x[off:off + R * C].view(R, C))
        ref, h, r = N.norm(x64, None, None, 1e-5)
        N.close(out[off:off + R * C], ref, N.norm_tol(h, None, None, ref, dtype), "y")
        out.fill_(7.0)
        dy = rnd(2, R * C + 64, dtype=dtype).cuda()
        dw = torch.full((C + 2,), 7.0, device="cuda")
        rc = lib.siv_layer_norm_bwd(dy.data_ptr() + 2 * es, C, x.data_ptr() + off * es, C, w.data_ptr(), 0, 1e-5,
                                    out.data_ptr() + off * es, dw.data_ptr() + 4, None, 0, t, R, C, ws.data_ptr(), ws.numel(),
                                    st)
        assert rc == 0
        assert bool((out[:off] == 7).all()) and bool((out[off + R * C:] == 7).all())
        assert float(dw[0]) == 7 and float(dw[-1]) == 7
        dy64 = N.rows_of(dy[2:2 + R * C].view(R, C))
        dx, dwr, _ = N.norm_grad(dy64, h, r, None)
        N.close(out[off:off + R * C], dx, N.dx_tol(dy64, h, r, None, dx, dtype), "dx")
        N.close(dw[1:-1], dwr, N.param_tol(dy64, h, dwr, torch.float32), "dw")


def test_layer_norm_hard_rows():
    """Constant rows, rows far off zero, and rows with NaN / infinities, which keep to themselves."""
    o = ops()
    for C in (1, 4, 64, 100, 1200, 9000):
        x = rnd(C, 6, C)
        x[0] = 3.0
        x[1] = 0.0
        x[2] = x[2] * 0.5 + 1.0e4
        x[3] = x[3] * 1e-3 - 17.0
        w, b = 1 + 0.2 * rnd(1, C), rnd(2, C)
        check_norm(x.cuda(), rnd(3, 6, C).cuda(), w.cuda(), b.cuda(), 1e-5, torch.float32, torch.float32)
        clean = o.layer_norm(x.cuda(), w.cuda(), b.cuda())
        bad = x.clone()
        bad[4, C // 2] = float("nan")
        bad[5, 0] = float("inf")
        y = o.layer_norm(bad.cuda(), w.cuda(), b.cuda())
        assert torch.equal(y[:4], clean[:4]) and bool(torch.isnan(y[4:]).all())
        xd = bad.cuda().requires_grad_()
        dx, = torch.autograd.grad(o.layer_norm(xd, w.cuda(), b.cuda()), xd, torch.ones(6, C, device="cuda"))
        assert bool(torch.isfinite(dx[:4]).all()) and bool(torch.isnan(dx[4:]).all())


def test_layer_norm_empty_and_one_dimensional():
    o = ops()
    w, b = torch.ones(8, device="cuda", requires_grad=True), torch.zeros(8, device="cuda", requires_grad=True)
    x = torch.empty(0, 8, device="cuda", requires_grad=True)
    y = o.layer_norm(x, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.empty(0, 8, device="cuda"))
    assert y.shape == (0, 8) and dx.shape == (0, 8) and not dw.any() and not db.any()
    y, s = o.add_layer_norm(x, x.detach(), w, b, keep=key(), p=0.5)
    g = torch.autograd.grad((y, s), (x, w, b), (torch.empty(0, 8, device="cuda"),) * 2)
    assert not g[1].any() and not g[2].any()
    assert o.dropout(x, key(), 0.5).shape == (0, 8)
    v = rnd(1, 8).cuda()
    assert torch.equal(o.layer_norm(v, w, b), o.layer_norm(v[None], w, b)[0])


def test_refusals(hip):
    from siv._lib import SivError
    o = ops()
    x = torch.zeros(4, 8, device="cuda")
    for bad, word in ((lambda: o.layer_norm(x, torch.ones(7, device="cuda")), "shape"),
                      (lambda: o.layer_norm(x, torch.ones(8)), "on cuda"),
                      (lambda: o.layer_norm(x, torch.ones(8, device="cuda", dtype=torch.bfloat16)), "weight and bias"),
                      (lambda: o.layer_norm(x.bfloat16(), torch.ones(8, device="cuda"),
                                            torch.ones(8, device="cuda", dtype=torch.bfloat16)), "weight and bias"),
                      (lambda: o.layer_norm(torch.zeros(4, 0, device="cuda")), "length 0"),
                      (lambda: o.layer_norm(torch.zeros((), device="cuda")), "one axis"),
                      (lambda: o.layer_norm(x, eps=-1.0), "eps"),
                      (lambda: o.dropout(x, key(), 1.0), "dropout p"),
                      (lambda: o.dropout(x, key(), float("nan")), "dropout p"),
                      (lambda: o.dropout(x, torch.ones(4, 8, device="cuda"), 0.5), "uint8"),
                      (lambda: o.dropout(x, torch.ones(4, 7, device="cuda", dtype=torch.uint8), 0.5), "uint8"),
                      (lambda: o.dropout(x, key(epoch=torch.zeros(1, device="cuda")), 0.5), "epoch"),
                      (lambda: o.dropout(x, key(), 0.5, residual=torch.zeros(4, 7, device="cuda")), "shapes"),
                      (lambda: o.dropout(x, key(), 0.5, residual=x.bfloat16()), "beside"),
                      (lambda: o.add_layer_norm(x, x.half()), "beside"),
                      (lambda: o.add_layer_norm(x, x[:2]), "shapes")):
        with pytest.raises(SivError, match=word):
            bad()
    # no second derivative: an error, not a zero, also where another path leads to the same leaf
    xg = rnd(1, 4, 8).cuda().requires_grad_()
    for f in (lambda: o.layer_norm(xg), lambda: o.add_layer_norm(xg, xg, keep=key(), p=0.5)[0],
              lambda: o.dropout(xg, key(), 0.5).square()):
        first, = torch.autograd.grad(f().sum(), xg)
        dx, = torch.autograd.grad(f().sum(), xg, create_graph=True)
        assert torch.equal(dx, first)
        with pytest.raises(RuntimeError, match="differentia"):
            torch.autograd.grad((dx * xg.sin()).sum(), xg)
    # the residual's gradient is the upstream one, with its history
    a, res = rnd(2, 4, 8).cuda().requires_grad_(), rnd(3, 4, 8).cuda().requires_grad_()
    for f in (lambda: o.dropout(xg, key(), 0.5, residual=res), lambda: o.add_layer_norm(xg, res, keep=key(), p=0.5)[1],
              lambda: o.add_layer_norm(xg, res)[1]):
        dr, = torch.autograd.grad((f() * a).sum(), res, create_graph=True)
        assert torch.equal(torch.autograd.grad(dr.square().sum(), a)[0], 2 * a.detach())
    dx, = torch.autograd.grad(o.dropout(xg, key(), 0.5).sum(), xg, create_graph=True)      # does not depend on xg
    assert torch.equal(torch.autograd.grad((dx * xg.sin()).sum(), xg)[0], dx.detach() * xg.detach().cos())


def test_gradients_that_are_not_dense(hip):
    """Upstream gradients as autograd hands them on: expanded, transposed, strided."""
    o = ops()
    x, w, b = rnd(1, 12, 40).cuda().requires_grad_(), torch.ones(40, device="cuda", requires_grad=True), None
    ups = (torch.ones((), device="cuda").expand(12, 40), rnd(2, 40, 12).cuda().t(), rnd(3, 12, 90).cuda()[:, 5:45],
           rnd(4, 24, 80).cuda()[::2, ::2])
    for dy in ups:
        for f in (lambda: o.layer_norm(x, w), lambda: o.add_layer_norm(x, x.detach(), w, keep=key(), p=0.5)[0],
                  lambda: o.add_layer_norm(x, x.detach(), w, keep=key(), p=0.5)[1], lambda: o.dropout(x, key(), 0.5),
                  lambda: o.act_dropout(x, 0.2, key(), 0.5)):
            got = torch.autograd.grad(f(), (x, w), dy, allow_unused=True)
            want = torch.autograd.grad(f(), (x, w), dy.contiguous(), allow_unused=True)
            assert all(a is c or torch.equal(a, c) for a, c in zip(got, want))
    v = rnd(5, 2, 6, 3, 4, 5).cuda().contiguous(memory_format=CL3D).requires_grad_()
    dy = rnd(6, 2, 6, 3, 4, 5).cuda()                      # NCDHW memory
    for f in (lambda: o.layer_norm(v), lambda: o.dropout(v, key(), 0.5), lambda: o.add_layer_norm(v, v.detach())[0]):
        got, = torch.autograd.grad(f(), v, dy)
        want, = torch.autograd.grad(f(), v, dy.contiguous(memory_format=CL3D))
        assert torch.equal(got, want)


def test_a_changed_input_is_noticed(hip):
    """The kept input written between forward and backward: an error, as for torch's own operators."""
    o = ops()
    x = rnd(1, 4, 8).cuda().requires_grad_()
    for f in (lambda t: o.layer_norm(t), lambda t: o.act_dropout(t, 0.0, key(), 0.5)):
        t = x * 1.0
        y = f(t)
        t.add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace"):
            y.sum().backward()
    y, s = o.add_layer_norm(x, x.detach())
    s.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()


def test_leaf_gradients_are_separate(hip):
    """x and residual share one gradient where nothing is dropped; their .grad tensors do not share memory."""
    o = ops()
    for f in (lambda x, r: o.add_layer_norm(x, r)[0], lambda x, r: o.add_layer_norm(x, r)[1],
              lambda x, r: o.dropout(x, key(), 0.5, residual=r)):
        x, r = rnd(1, 6, 40).cuda().requires_grad_(), rnd(2, 6, 40).cuda().requires_grad_()
        up = rnd(3, 6, 40).cuda()
        keep = up.clone()
        f(x, r).backward(up)
        want = r.grad.clone()
        x.grad.zero_()
        assert torch.equal(r.grad, want) and torch.equal(up, keep)
        f(x, r).backward(up)
        assert torch.equal(r.grad, 2 * want)
        assert torch.equal(up, keep)


def test_frozen_parameters_and_inputs(hip):
    """Only what requires a gradient gets one; parameters that are frozen stay as they are."""
    o = ops()
    x, w, b = rnd(1, 12, 40).cuda(), torch.ones(40, device="cuda"), torch.zeros(40, device="cuda")
    full = [t.clone().requires_grad_() for t in (x, w, b)]
    want = torch.autograd.grad(o.layer_norm(*full), full, torch.ones(12, 40, device="cuda"))
    for mask in range(1, 8):
        ts = [t.clone().requires_grad_(bool(mask >> i & 1)) for i, t in enumerate((x, w, b))]
        y = o.layer_norm(*ts)
        y.backward(torch.ones(12, 40, device="cuda"))
        for i, t in enumerate(ts):
            assert (t.grad is None) == (not mask >> i & 1)
            assert t.grad is None or torch.equal(t.grad, want[i])
    assert not o.layer_norm(x, w, b).requires_grad and not o.dropout(x, key(), 0.5).requires_grad
    with torch.no_grad():
        assert not o.layer_norm(*full).requires_grad


# ---- dropout ----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", N.DTYPES, ids=N.IDS)
@pytest.mark.parametrize("p", [0.0, 0.1, 0.35, 0.999])
@pytest.mark.parametrize("shape", [(1,), (3,), (4,), (5,), (8, 1200), (13, 77), (1031, 33), (2, 3, 5, 7, 4), (70001,)])
def test_dropout(hip, shape, p, dtype):
    """Out, gradient and mask: the bits dropout_keep stores for the key; a product and (residual) one addition."""
    o, k = ops(), key(2 ** 63 + 9, (3 << 40) | 17)
    x = rnd(1, *shape, dtype=dtype).cuda()
    x = x.contiguous(memory_format=CL3D) if x.dim() == 5 else x
    res, dy = (rnd(s, *shape, dtype=dtype).cuda() for s in (2, 3))
    m = mask_rows(hip, shape, p, k)
    sc = scale_of(p)
    for r in (None, res):
        xd = x.detach().requires_grad_()
        rd = None if r is None else r.detach().requires_grad_()
        out = o.dropout(xd, k, p, residual=rd)
        prod = N.rows_of(x) * m * sc
        ref = prod if r is None else prod + N.rows_of(r)
        tol = N.half(dtype) * ref.abs() + N.tiny(dtype) + 2 * N.U * (prod.abs() + ref.abs())
        N.close(N.rows_of(out), ref, tol, "out")
        assert torch.equal((N.rows_of(o.dropout(torch.ones_like(x), k, p)) != 0).double(), m)
        g = torch.autograd.grad(out, (xd,) if r is None else (xd, rd), dy)
        gr = N.rows_of(dy) * m * sc
        N.close(N.rows_of(g[0]), gr, N.half(dtype) * gr.abs() + N.tiny(dtype) + 2 * N.U * gr.abs(), "dx")
        if r is not None:
            assert torch.equal(g[1], dy)
    mt = hip.dropout_keep(shape if len(shape) == 5 else (1, 1, 1, 1, x.numel()), x.device, p, k.seed, k.stream_id)
    mt = mt if len(shape) == 5 else mt.reshape(shape)
    assert torch.equal(o.dropout(x, mt, p), o.dropout(x, k, p))
    assert torch.equal(o.dropout(x, None, p), x)


@pytest.mark.parametrize("dtype", N.DTYPES, ids=N.IDS)
def test_dropout_drops_nan_and_infinity(hip, dtype):
    o, k, n = ops(), key(), 4096
    m = mask_rows(hip, (n,), 0.5, k)[0].bool().cuda()
    for bad in (float("nan"), float("inf"), torch.finfo(dtype).min):
        x = torch.where(m, torch.ones((), device="cuda", dtype=dtype), torch.full((), bad, device="cuda", dtype=dtype))
        out = o.dropout(x, k, 0.5)
        assert torch.equal(out, torch.where(m, 2.0, 0.0).to(dtype))
        xd = torch.ones(n, device="cuda", dtype=dtype, requires_grad=True)
        dx, = torch.autograd.grad(o.dropout(xd, k, 0.5), xd, x)
        assert torch.equal(dx, torch.where(m, 2.0, 0.0).to(dtype))
        y, s = o.add_layer_norm(x.view(64, 64), torch.zeros(64, 64, device="cuda", dtype=dtype), keep=k, p=0.5)
        assert torch.equal(s.view(-1), out) and bool(torch.isfinite(y).all())


@pytest.mark.parametrize("dtype", N.DTYPES, ids=N.IDS)
@pytest.mark.parametrize("off", [0, 1, 2, 3, 5])
def test_dropout_alignments(hip, off, dtype):
    """Tensors that start anywhere: same values, and nothing outside them is written."""
    o, k, n = ops(), key(), 1003
    base = rnd(1, n + 16, dtype=dtype).cuda()
    want = o.dropout(base[off:off + n].clone(), k, 0.25, residual=base[:n].clone())
    assert torch.equal(o.dropout(base[off:off + n], k, 0.25, residual=base[:n]), want)
    out = torch.full((n + 16,), 7.0, dtype=dtype, device="cuda")
    es, st = base.element_size(), torch.cuda.current_stream().cuda_stream
    rc = hip.lib.siv_dropout_fwd(base.data_ptr() + off * es, base.data_ptr(), None, k.seed, k.stream_id, None, 0.25, 1.0,
                                 out.data_ptr() + 3 * es, hip._TYPES[dtype], n, st)
    assert rc == 0 and torch.equal(out[3:3 + n], want) and bool((out[:3] == 7).all()) and bool((out[3 + n:] == 7).all())


def test_dropout_epoch_and_act_dropout(hip):
    """The device epoch moves the draw; act_dropout with a key gives what it gives with that key's stored mask."""
    o = ops()
    ep = torch.zeros(1, dtype=torch.int64, device="cuda")
    k = key(9, 4, ep)
    x = rnd(1, 2, 1, 6, 7, 5).cuda().contiguous(memory_format=CL3D)
    seen = []
    for _ in range(3):
        m = hip.dropout_keep(x.shape, x.device, 0.35, 9, 4, ep)
        for slope in (0.0, 0.2, 1.0):
            a, b = (x.detach().requires_grad_() for _ in range(2))
            ya, yb = o.act_dropout(a, slope, k, 0.35), o.act_dropout(b, slope, m, 0.35)
            assert torch.equal(ya, yb)
            assert torch.equal(*(torch.autograd.grad(y, t, x)[0] for y, t in ((ya, a), (yb, b))))
        seen.append(m.clone())
        hip.counter_add(ep, 1)
    assert not torch.equal(seen[0], seen[1]) and not torch.equal(seen[1], seen[2])


def test_decoder_output_layer_draws_its_mask():
    """The model's output dropout: same bits whether its mask is stored or drawn where it is used."""
    from siv import rng
    from siv.models import _core, models
    torch.manual_seed(0)
    net = models.SoftIntroVAE(8, [[8, 1, 2], [16, 1, 2]]).cuda().train()
    z = torch.randn(net.latent_shape(2, (8, 8, 8)), device="cuda")
    outs = []
    draws = _core.ops.draws_masks
    for stored in (False, True):
        state = {k: v.clone() for k, v in net.state_dict().items()}
        _core.ops.draws_masks = (lambda: False) if stored else draws
        try:
            with rng.use_rng(rng.DeviceRng(3)):
                y = net.decoder(z)
                net.zero_grad()
                y.square().sum().backward()
                outs.append([y.detach()] + [p.grad.clone() for p in net.decoder.parameters() if p.grad is not None])
        finally:
            _core.ops.draws_masks = draws
        net.load_state_dict(state)
    assert len(outs[0]) == len(outs[1]) > 4
    assert all(torch.equal(a, b) for a, b in zip(*outs))
    assert float((outs[0][0] == 0).float().mean()) > 0.3


# ---- residual + dropout + layer norm ------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", N.DTYPES, ids=N.IDS)
@pytest.mark.parametrize("source", ["key", "mask", "none"])
@pytest.mark.parametrize("shape", [(1, 1), (5, 3), (7, 8), (40, 30), (129, 64), (33, 129), (9, 601), (6, 1200), (3, 2050),
                                   (2, 4100), (3, 8193), (2, 38401), (2, 64, 3, 4, 5), (1, 6, 5, 6, 5)])
def test_add_layer_norm(hip, shape, source, dtype):
    o, k, p = ops(), key(77, 1 << 41), (0.35 if source != "none" else 0.0)
    mk = lambda s, **kw: rnd(s, *shape, dtype=dtype, **kw).cuda().contiguous(
        memory_format=CL3D if len(shape) == 5 else torch.contiguous_format)
    x, res, dy, ds = mk(1), mk(2, offset=0.3), mk(3, scale=0.1), mk(4, scale=0.1)
    C = shape[1] if len(shape) == 5 else shape[-1]
    w, b = (1 + 0.2 * rnd(5, C)).cuda().requires_grad_(), rnd(6, C, scale=0.1).cuda().requires_grad_()
    m = mask_rows(hip, shape, p, k) if p else torch.ones_like(N.rows_of(x))
    keep = None if source == "none" else k
    if source == "mask":
        keep = m.to(torch.uint8).cuda().view(shape) if len(shape) != 5 else \
            hip.dropout_keep(shape, x.device, p, k.seed, k.stream_id)
    sc = scale_of(p)
    xd, rd = x.detach().requires_grad_(), res.detach().requires_grad_()
    y, s = o.add_layer_norm(xd, rd, w, b, 1e-5, keep=keep, p=p)
    x64, r64 = N.rows_of(x), N.rows_of(res)
    sref = r64 + x64 * m * sc
    N.close(N.rows_of(s), sref, N.half(dtype) * sref.abs() + N.tiny(dtype) + 2 * N.U * ((x64 * sc).abs() + sref.abs()), "s")
    # the norm of the sum as it is held, and the separate operators' results bit for bit
    w64, b64 = w.detach().cpu().double(), b.detach().cpu().double()
    yref, h, r = N.norm(N.rows_of(s), w64, b64, 1e-5)
    N.close(N.rows_of(y), yref, N.norm_tol(h, w64, b64, yref, dtype), "y")
    assert torch.equal(s, o.dropout(x, keep, p, residual=res))
    dy64, ds64 = N.rows_of(dy), N.rows_of(ds)
    for with_ds in (True, False):
        outs, ups = ((y, s), (dy, ds)) if with_ds else ((y,), (dy,))
        gx, gr, gw, gb = torch.autograd.grad(outs, (xd, rd, w, b), ups, retain_graph=True)
        d, dw, db = N.norm_grad(dy64, h, r, w64)
        tol = N.dx_tol(dy64, h, r, w64, 0 * d, dtype)
        if with_ds:
            d = d + ds64
        N.close(N.rows_of(gr), d, tol + (N.half(dtype) + 2 * N.U) * d.abs(), "dresidual")
        N.close(N.rows_of(gx), d * m * sc, tol * sc + (N.half(dtype) + 3 * N.U) * (d * sc).abs(), "dx")
        N.close(gw, dw, N.param_tol(dy64, h, dw, torch.float32), "dw")
        N.close(gb, db, N.param_tol(dy64, h, db, torch.float32), "db")
    gx, gr = torch.autograd.grad(s, (xd, rd), ds, retain_graph=True)       # the norm's output unused
    assert torch.equal(gr, ds)
    ref = ds64 * m * sc
    N.close(N.rows_of(gx), ref, (N.half(dtype) + 2 * N.U) * ref.abs() + N.tiny(dtype), "dx of the sum alone")
    # one gradient at a time
    for i, leaf in enumerate((xd, rd, w, b)):
        one, = torch.autograd.grad((y, s), (leaf,), (dy, ds), retain_graph=True)
        full = torch.autograd.grad((y, s), (xd, rd, w, b), (dy, ds), retain_graph=True)[i]
        assert torch.equal(one, full)


# ---- in use -------------------------------------------------------------------------------------------------------------
def branch(o, x, w, b, cw, w2, b2, k1, k2, p):
    """A pre-norm residual branch over the channels of a volume, and a second dropout onto its stream."""
    u = o.conv1x1(o.layer_norm(x, w, b), cw)
    y, s = o.add_layer_norm(u, x, w2, b2, keep=k1, p=p)
    return o.dropout(y, k2, p, residual=s)


def branch_inputs(shape, seed=0):
    C = shape[1]
    x = rnd(seed + 1, *shape, offset=0.5).cuda().contiguous(memory_format=CL3D)
    ps = [1 + 0.2 * rnd(seed + 2, C), 0.1 * rnd(seed + 3, C), rnd(seed + 4, C, C, 1, 1, 1, scale=C ** -0.5),
          1 + 0.2 * rnd(seed + 5, C), 0.1 * rnd(seed + 6, C)]
    return x, [t.cuda() for t in ps], rnd(seed + 7, *shape).cuda().contiguous(memory_format=CL3D)


@pytest.mark.parametrize("shape", [(2, 16, 5, 6, 5), (3, 64, 4, 3, 7)])
def test_residual_branch_matches_float64(hip, shape):
    """Forward and every gradient of the run of them against autograd of the float64 formulas, 1e-4 of the maximum (the
    framework's tolerance for a kernel; here four in a row)."""
    o, p, k1, k2 = ops(), 0.25, key(1, 2), key(1, 3)
    x, ps, dy = branch_inputs(shape)
    leaves = [t.detach().requires_grad_() for t in (x, *ps)]
    out = branch(o, *leaves, k1, k2, p)
    got = [out.detach()] + list(torch.autograd.grad(out, leaves, dy))
    l64 = [t.detach().cpu().double().requires_grad_() for t in (x, *ps)]
    m1, m2 = (mask_rows(hip, shape, p, k) for k in (k1, k2))
    sc = scale_of(p)
    X, w, b, cw, w2, b2 = l64
    xr = X.permute(0, 2, 3, 4, 1).reshape(-1, shape[1])
    u = N.norm(xr, w, b, 1e-5)[0] @ cw.view(shape[1], shape[1]).t()
    s = xr + u * m1 * sc
    ref = s + N.norm(s, w2, b2, 1e-5)[0] * m2 * sc
    refs = [ref.detach()] + list(torch.autograd.grad(ref, l64, N.rows_of(dy)))
    for i, (a, r) in enumerate(zip(got, refs)):
        a = N.rows_of(a) if i < 2 else a.cpu().double()
        r = N.rows_of(r) if i == 1 else r
        assert float((a - r.reshape(a.shape)).abs().max()) <= 1e-4 * float(r.abs().max()), i


def test_flat_optimiser_buffers_collect_the_gradients():
    """Parameters of a FlatAdam: two backward passes add into its flat buffer what autograd.grad returns."""
    from siv.optim import FlatAdam
    o = ops()
    x, dy = rnd(1, 300, 96).cuda(), rnd(2, 300, 96).cuda()
    w, b = (torch.nn.Parameter(t.cuda()) for t in (1 + rnd(3, 96, scale=0.2), rnd(4, 96)))
    wr, br = w.detach().clone().requires_grad_(), b.detach().clone().requires_grad_()
    dw, db = torch.autograd.grad(o.layer_norm(x, wr, br), (wr, br), dy)
    opt = FlatAdam([w, b], lr=1e-3)
    opt.zero_grad()
    for _ in range(2):
        o.layer_norm(x, w, b).backward(dy)
    assert torch.equal(w.grad, dw + dw) and torch.equal(b.grad, db + db)
    dw2, db2 = torch.autograd.grad(o.add_layer_norm(x, dy, wr, br, keep=key(), p=0.5)[0], (wr, br), dy)
    opt.zero_grad()
    o.add_layer_norm(x, dy, w, b, keep=key(), p=0.5)[0].backward(dy)
    assert torch.equal(w.grad, dw2) and torch.equal(b.grad, db2)


@pytest.mark.parametrize("mode", ["fp32", "bf16"])
def test_saved_activations_follow_the_storage_mode(mode):
    """Under bf16 activation storage the norm's input is kept as bf16: the gradient is that of the rounded input."""
    from siv import activations
    o = ops()
    x0, dy = rnd(1, 600, 128).cuda(), rnd(2, 600, 128).cuda()
    w, b = torch.ones(128, device="cuda"), torch.zeros(128, device="cuda")

    @activations.scoped
    def run(t):
        return o.layer_norm(t * 1.0, w, b)
    xd = x0.clone().requires_grad_()
    with activations.storage(mode):
        y = run(xd)
    assert torch.equal(y, o.layer_norm(x0, w, b))
    dx, = torch.autograd.grad(y, xd, dy)
    seen = x0 if mode == "fp32" else x0.bfloat16().float()
    xr = seen.clone().requires_grad_()
    assert torch.equal(dx, torch.autograd.grad(o.layer_norm(xr, w, b), xr, dy)[0])


def test_another_stream_and_two_at_once():
    """Calls on two streams, each with its own workspace, give what they give alone."""
    o, p = ops(), 0.25
    shape = (2, 64, 10, 12, 10)
    x, ps, dy = branch_inputs(shape)
    leaves = [t.detach().requires_grad_() for t in (x, *ps)]

    def go(i):
        out = branch(o, *leaves, key(i, 2), key(i, 3), p)
        return [out.detach()] + list(torch.autograd.grad(out, leaves, dy))
    want = [go(i) for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        got = []
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got.append(go(i))
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert all(torch.equal(a, b) for a, b in zip(g, w))


def test_recomputed_branch_and_inference_mode():
    """Activation checkpointing (the branch runs again in backward, drawing the same masks), inference mode, and a second
    Python thread give what the plain call gives."""
    import threading
    from torch.utils.checkpoint import checkpoint
    o, p, shape = ops(), 0.25, (2, 64, 4, 5, 6)
    x, ps, dy = branch_inputs(shape)
    leaves = [t.detach().requires_grad_() for t in (x, *ps)]
    out = branch(o, *leaves, key(1, 2), key(1, 3), p)
    want = [out.detach()] + list(torch.autograd.grad(out, leaves, dy))
    out = checkpoint(lambda *a: branch(o, *a, key(1, 2), key(1, 3), p), *leaves, use_reentrant=False)
    got = [out.detach()] + list(torch.autograd.grad(out, leaves, dy))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    with torch.inference_mode():
        assert torch.equal(branch(o, x, *ps, key(1, 2), key(1, 3), p), want[0])
    res = []

    def work():
        ls = [t.detach().requires_grad_() for t in (x, *ps)]
        y = branch(o, *ls, key(1, 2), key(1, 3), p)
        res.append([y.detach()] + list(torch.autograd.grad(y, ls, dy)))
    threads = [threading.Thread(target=work) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(res) == 2 and all(torch.equal(a, b) for r in res for a, b in zip(r, want))


def test_forward_mode_derivatives_are_refused(hip):
    """A tensor with a tangent: there is no forward-mode rule, and none may be lost without a word."""
    import torch.autograd.forward_ad as fwd
    o, gen = ops(), torch.Generator(device="cuda").manual_seed(3)
    x, r, t = (torch.randn(6, 40, device="cuda", generator=gen) for _ in range(3))
    w, tw = (torch.randn(40, device="cuda", generator=gen) for _ in range(2))
    with fwd.dual_level():
        dx, dw = fwd.make_dual(x, t), fwd.make_dual(w, tw)
        for call in (lambda: o.layer_norm(dx, w), lambda: o.layer_norm(x, dw), lambda: o.layer_norm(x, w, dw),
                     lambda: o.dropout(dx, key(1, 2), 0.5), lambda: o.dropout(x, key(1, 2), 0.5, residual=dx),
                     lambda: o.add_layer_norm(dx, r, w), lambda: o.add_layer_norm(r, dx, w),
                     lambda: o.add_layer_norm(x, r, dw)):
            with pytest.raises(RuntimeError):
                call()
        assert torch.equal(o.layer_norm(x, w), o.layer_norm(x.clone(), w))        # without a tangent: as ever


def test_captured_branches_replay(hip):
    """Two captured graphs of forward + backward, replayed with eager work between, each replay with the next epoch's
    masks, against the eager result of the same epoch."""
    o, p, shape = ops(), 0.25, (2, 64, 4, 5, 6)
    ep = torch.zeros(1, dtype=torch.int64, device="cuda")
    x, ps, dy = branch_inputs(shape)

    def go(src, sid):
        leaves = [t.detach().requires_grad_() for t in (src, *ps)]
        out = branch(o, *leaves, key(4, sid, ep), key(4, sid + 1, ep), p)
        return [out.detach()] + list(torch.autograd.grad(out, leaves, dy))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        go(x, 2)
    torch.cuda.current_stream().wait_stream(side)
    gc.collect()
    graphs = []
    for sid in (2, 8):
        src = x.clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res = go(src, sid)
        graphs.append((g, src, res, sid))
    for step in range(4):
        for g, src, res, sid in graphs:
            src.copy_(rnd(step + sid, *shape))
            g.replay()
        eager = [go(src, sid) for _, src, _, sid in graphs]
        torch.cuda.synchronize()
        for (g, src, res, sid), e in zip(graphs, eager):
            assert all(torch.equal(a, b) for a, b in zip(res, e)), (step, sid)
        hip.counter_add(ep, 1)
        torch.zeros(1000, 1000, device="cuda").sum().item()


def test_results_repeat():
    """No result depends on the order blocks finish in."""
    o = ops()
    for R, C, dt in ((5000, 64, torch.float32), (333, 1000, torch.bfloat16), (64, 9000, torch.float16)):
        x, dy = rnd(1, R, C, dtype=dt).cuda(), rnd(2, R, C, dtype=dt).cuda()
        w, b = torch.ones(C, device="cuda", requires_grad=True), torch.zeros(C, device="cuda", requires_grad=True)
        xd = x.requires_grad_()
        first = None
        for _ in range(4):
            y = o.layer_norm(xd, w, b)
            now = [y.detach()] + list(torch.autograd.grad(y, (xd, w, b), dy))
            first = first or now
            assert all(torch.equal(a, c) for a, c in zip(first, now))


@pytest.mark.parametrize("C", [3, 64, 700, 9001])
def test_gradients_against_differences(C):
    """<dx, v> and <dw, v> of the kernels against difference quotients of the float64 forward pass (step 1e-4: truncation
    below 1e-6 of the third derivatives' size, r^3 |g| |v|^3)."""
    x, dy, v = rnd(1, 4, C), rnd(2, 4, C), rnd(3, 4, C)
    w, b, vw = 1 + 0.2 * rnd(4, C), rnd(5, C), rnd(6, C)
    xd, wd, bd = (t.cuda().requires_grad_() for t in (x, w, b))
    eps = 1e-2
    dx, dw, db = torch.autograd.grad(ops().layer_norm(xd, wd, bd, eps), (xd, wd, bd), dy.cuda())
    x64, dy64, w64, b64, v64, vw64 = (t.double() for t in (x, dy, w, b, v, vw))
    f = lambda a, c: float((N.norm(a, c, b64, eps)[0] * dy64).sum())
    e = 1e-4
    _, h, r = N.norm(x64, w64, b64, eps)
    size = float((dy64 * w64 * v64).abs().sum())
    want = (f(x64 + e * v64, w64) - f(x64 - e * v64, w64)) / (2 * e)
    tol = float((N.dx_tol(dy64, h, r, w64, dx.cpu().double(), torch.float32) * v64.abs()).sum())
    assert abs(float((dx.cpu().double() * v64).sum()) - want) <= tol + 1e-6 * float(r.max()) ** 3 * size
    want = (f(x64, w64 + e * vw64) - f(x64, w64 - e * vw64)) / (2 * e)
    tol = float((N.param_tol(dy64, h, dw.cpu().double(), torch.float32) * vw64.abs()).sum())
    assert abs(float((dw.cpu().double() * vw64).sum()) - want) <= tol + 1e-8 * float((dy64 * h * vw64).abs().sum())


# ---- beyond 32-bit offsets ------------------------------------------------------------------------------------------------
def test_offsets_beyond_32_bits(hip):
    """2^32 + 2^13 half-precision elements: the far end against the same values in a small tensor."""
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB of device memory")
    o, C = ops(), 4096
    R = (1 << 20) + 2
    x = torch.empty(R, C, dtype=torch.float16, device="cuda").fill_(1.0)
    tail = rnd(1, 3, C, dtype=torch.float16).cuda()
    x[-3:] = tail
    w, b = (1 + 0.2 * rnd(2, C)).cuda(), rnd(3, C).cuda()
    y = hip.layer_norm_fwd(x, w, b, 1e-5)
    assert torch.equal(y[-3:], o.layer_norm(tail, w, b))
    assert torch.equal(y[:2], o.layer_norm(torch.ones(2, C, dtype=torch.float16, device="cuda"), w, b))
    dx, dw, db = hip.layer_norm_bwd(x, x, w, 1e-5)
    sx, _, _ = hip.layer_norm_bwd(tail, tail, w, 1e-5)
    assert torch.equal(dx[-3:], sx)
    del y, dx
    k = key(3, 5)
    out = hip.dropout_fwd(x, k, 0.5)
    m = hip.dropout_keep((1, 1, 1, R, C), x.device, 0.5, 3, 5).view(R, C)
    assert torch.equal(out[-3:], torch.where(m[-3:] != 0, tail * 2, torch.zeros_like(tail)))
    assert torch.equal(out[:2] != 0, m[:2] != 0)
    s = hip.add_layer_norm_fwd(x, x, k, 0.5, w, b, 1e-5)[1]
    assert torch.equal(s[-3:], tail + out[-3:])
