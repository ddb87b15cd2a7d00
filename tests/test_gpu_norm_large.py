"""Layer norm and the residual step where many rows, long rows and many blocks meet, against float64 values on the device
with bounds that do not grow with a row's length (tests/norm_bounds.py); dropout where blocks walk over the tensor."""
import pytest
import torch

from tests import norm_bounds as B

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
EPS = 1e-5


@pytest.fixture
def hip():
    import siv.backend as sb
    sb.set_backend(None)
    b = sb.get_backend()
    assert b.nodes is not None, "siv/_siv_torch.so is not built"
    return b


def key(seed=5, sid=11):
    from siv import rng
    return rng.PhiloxKeep(seed, sid)


def check_norm(R, C, dtype, wdtype=F32):
    from siv import ops as o
    x, dy, w, b = B.inputs(R, C, dtype, R + C, "cuda")
    x, w, b = x.requires_grad_(), w.to(wdtype).requires_grad_(), b.to(wdtype).requires_grad_()
    y = o.layer_norm(x, w, b, EPS)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    x64, dy64, w64, b64 = (t.detach().double() for t in (x, dy, w, b))
    ry, h, r = B.norm(x64, w64, b64, EPS)
    B.check(y, ry, B.y_tol(h, w64, b64, ry, dtype), "y")
    rx, rw, rb = B.grads(dy64, h, r, w64)
    B.check(dx, rx, B.dx_tol(dy64, h, r, w64) + B.half(dtype) * rx.abs() + B.tiny(dtype), "dx")
    B.check(dw, rw, B.dw_tol(dy64, h, rw, R, C, dtype, wdtype), "dweight")
    B.check(db, rb, B.db_tol(dy64, rb, R, C, dtype, wdtype), "dbias")


def check_add(hip, R, C, dtype, p=0.25):
    from siv import ops as o
    x, dy, w, b = B.inputs(R, C, dtype, R + C, "cuda")
    res, ds, _, _ = B.inputs(R, C, dtype, R + C + 1, "cuda")
    x, res, w, b = (t.requires_grad_() for t in (x, res, w, b))
    k = key(77, 1 << 41)
    y, s = o.add_layer_norm(x, res, w, b, EPS, keep=k, p=p)
    dx, dr, dw, db = torch.autograd.grad((y, s), (x, res, w, b), (dy, ds))
    m = hip.dropout_keep((1, 1, 1, 1, R * C), x.device, p, k.seed, k.stream_id).view(R, C).double()
    sc = float(torch.tensor(1.0) / (torch.tensor(1.0) - torch.tensor(p)))
    x64, res64, dy64, ds64, w64, b64 = (t.detach().double() for t in (x, res, dy, ds, w, b))
    rs = res64 + x64 * m * sc
    B.check(s, rs, B.half(dtype) * rs.abs() + B.tiny(dtype) + 2 * B.U * ((x64 * sc).abs() + rs.abs()), "s")
    ry, h, r = B.norm(s.detach().double(), w64, b64, EPS)
    B.check(y, ry, B.y_tol(h, w64, b64, ry, dtype), "y")
    d, rw, rb = B.grads(dy64, h, r, w64)
    tol = B.dx_tol(dy64, h, r, w64) + 2 * B.U * (d.abs() + ds64.abs())
    d = d + ds64
    B.check(dr, d, tol + B.half(dtype) * d.abs() + B.tiny(dtype), "dresidual")
    B.check(dx, d * m * sc, tol * sc + (B.half(dtype) + 2 * B.U) * (d * sc).abs() + B.tiny(dtype), "dx")
    B.check(dw, rw, B.dw_tol(dy64, h, rw, R, C, dtype, F32), "dweight")
    B.check(db, rb, B.db_tol(dy64, rb, R, C, dtype, F32), "dbias")


# ---- row lengths of every form, few rows: the bounds at their tightest ---------------------------------------------------
LENGTHS = [(3, 4), (9, 7), (5, 33), (6, 64), (4, 100), (5, 256), (4, 500), (3, 601), (4, 1000), (3, 1200), (2, 2049),
           (3, 4096), (2, 4099), (2, 8190), (3, 8200), (2, 16384), (2, 38400), (2, 100003), (1, 614400), (2, 614401)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("R,C", LENGTHS)
def test_row_lengths(hip, R, C, dtype):
    check_norm(R, C, dtype)
    check_add(hip, R, C, dtype)


# ---- blocks that walk, and their partial sums joined ----------------------------------------------------------------------
# (rows, C, type, least number of partial sums, least steps a block walks): every form of the backward pass
WALKS = [(9603, 256, BF16, 257, 4), (40001, 64, F32, 257, 4), (20003, 33, F32, 257, 4), (20003, 33, F16, 256, 2),
         (614403, 8, F32, 768, 6), (100003, 3, F32, 2, 1), (5003, 601, BF16, 257, 4), (3001, 1000, F32, 257, 4),
         (1303, 1200, F32, 257, 4), (2003, 4099, F16, 256, 7), (1101, 4096, F32, 256, 4), (1101, 8190, F32, 256, 4)]


@pytest.mark.parametrize("R,C,dtype,parts,steps", WALKS)
def test_blocks_that_walk(hip, R, C, dtype, parts, steps):
    _, n, got = B.plan(R, C, dtype)
    assert got >= parts and n / got > steps - 1
    check_norm(R, C, dtype)
    check_add(hip, R, C, dtype)


@pytest.mark.parametrize("R,C,dtype", [(9603, 256, BF16), (40001, 64, F16), (300, 9001, BF16)])
def test_parameters_of_the_activations_type(hip, R, C, dtype):
    check_norm(R, C, dtype, dtype)


# ---- long rows in chunks: several parts of the rows, and more rows to a block than it keeps statistics of (16) -------------
@pytest.mark.parametrize("R,C,dtype,rows", [(40, 9001, F32, 8), (40, 9001, BF16, 8), (40, 16385, F16, 8), (300, 9001, F16, 8),
                                            (72, 614401, F32, 17), (130, 614400, F16, 17)])
def test_long_rows_in_several_parts(hip, R, C, dtype, rows):
    _, n, parts = B.plan(R, C, dtype)
    assert parts > 1 and n / parts > rows - 1
    check_norm(R, C, dtype)
    check_add(hip, R, C, dtype)


# ---- forward grids that walk ------------------------------------------------------------------------------------------------
def test_forward_of_two_packs_walks(hip):
    """33001 rows of 76 packs: more steps than the 8192 blocks of the two-pack wave form."""
    check_norm(33001, 601, BF16)
    check_add(hip, 33001, 601, BF16)


def test_forward_beyond_a_million_blocks(hip):
    """Rows behind the 2^20 blocks of the one-pack wave form, which load their next row after the present one: the rows on
    both sides of that border and the last ones against float64, and against the same rows in a small tensor."""
    from siv import ops as o
    C, border = 264, (1 << 20) * 4
    R = border + 7
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB of device memory")
    g = torch.Generator(device="cuda").manual_seed(1)
    x, res = (torch.randn(R, C, generator=g, device="cuda", dtype=BF16) for _ in range(2))
    w, b = 1 + 0.2 * torch.randn(C, generator=g, device="cuda"), torch.randn(C, generator=g, device="cuda")
    k = key(3, 5)
    torch.manual_seed(2)
    at = torch.cat((torch.arange(0, 9), torch.arange(border - 9, R), torch.randint(0, R, (999,)))).cuda()
    y = o.layer_norm(x, w, b, EPS)
    ref, h, _ = B.norm(x[at].double(), w.double(), b.double(), EPS)
    B.check(y[at], ref, B.y_tol(h, w.double(), b.double(), ref, BF16), "y")
    assert torch.equal(y[at], o.layer_norm(x[at], w, b, EPS))
    y, s = o.add_layer_norm(x, res, w, b, EPS, keep=k, p=0.5)
    m = hip.dropout_keep((1, 1, 1, R, C), x.device, 0.5, 3, 5).view(R, C)[at] != 0
    assert torch.equal(s[at], (res[at].float() + torch.where(m, x[at].float() * 2, 0.0)).to(BF16))
    ref, h, _ = B.norm(s[at].double(), w.double(), b.double(), EPS)
    B.check(y[at], ref, B.y_tol(h, w.double(), b.double(), ref, BF16), "y of the sum")


def test_parameter_gradients_beyond_32_bit_offsets(hip):
    """2^32 + 2^13 elements whose upstream gradient is zero but in the first and the last rows: dweight and dbias are those
    rows' sums."""
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB of device memory")
    C, n = 4096, 3
    R = (1 << 20) + 2
    x = torch.empty(R, C, dtype=F16, device="cuda").fill_(1.0)
    dy = torch.zeros(R, C, dtype=F16, device="cuda")
    few, up, w, _ = B.inputs(2 * n, C, F16, 9, "cuda")
    x[:n], x[-n:], dy[:n], dy[-n:] = few[:n], few[n:], up[:n], up[n:]
    dx, dw, db = hip.layer_norm_bwd(dy, x, w, EPS)
    _, h, r = B.norm(few.double(), w.double(), None, EPS)
    rx, rw, rb = B.grads(up.double(), h, r, w.double())
    B.check(dw, rw, B.dw_tol(up.double(), h, rw, R, C, F16, F32), "dweight")
    B.check(db, rb, B.db_tol(up.double(), rb, R, C, F16, F32), "dbias")
    tol = B.dx_tol(up.double(), h, r, w.double()) + B.half(F16) * rx.abs() + B.tiny(F16)
    B.check(torch.cat((dx[:n], dx[-n:])), rx, tol, "dx")
    assert not bool(dx[n:-n].any())


# ---- dropout: blocks that walk over the tensor ------------------------------------------------------------------------------
@pytest.mark.parametrize("n,dtype", [(9_000_003, BF16), (9_000_003, F16), (20_000_001, BF16), (44_739_243, F16),
                                     (50_000_001, BF16), ((1 << 26) + 4099, F16), ((1 << 27) + 4099, BF16),
                                     ((1 << 30) + 5003, F32)])
def test_dropout_walks(hip, n, dtype):
    """Two packs a thread over a grid of 2048, four and one over a grid of 2^20: every bit is the stored mask's, with and
    without a residual and an activation, forward and backward."""
    from siv import ops as o
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB of device memory")
    k, p = key(2 ** 63 + 9, (3 << 40) | 17), 0.5
    g = torch.Generator(device="cuda").manual_seed(n)
    x, res = (torch.randn(n, generator=g, device="cuda", dtype=dtype) for _ in range(2))
    m = hip.dropout_keep((1, 1, 1, 1, n), x.device, p, k.seed, k.stream_id).view(n) != 0
    twice = (2 * x).masked_fill_(~m, 0)                       # exact: 1 / (1 - p) is 2
    xg, rg = x.requires_grad_(), res.requires_grad_()
    out = o.dropout(xg, k, p)
    assert torch.equal(out, twice)
    dx, = torch.autograd.grad(out, xg, res.detach())
    assert torch.equal(dx, (2 * res.detach()).masked_fill_(~m, 0))
    del out, dx
    out = o.dropout(xg, k, p, residual=rg)
    assert torch.equal(out, (res.detach() + twice))           # (the product is exact; both add in fp32 and round once)
    del out
    out = o.act_dropout(xg, 0.0, k, p)
    assert torch.equal(out, twice.clamp_min(0))
    dx, = torch.autograd.grad(out, xg, res.detach())
    assert torch.equal(dx, (2 * res.detach()).masked_fill_(~m | (x.detach() <= 0), 0))


# ---- long rows beyond a grid's 65535 -----------------------------------------------------------------------------------------
@pytest.mark.parametrize("C", [8200, 16392])
def test_more_long_rows_than_a_grid_holds(hip, C):
    """65541 chunked rows: the blocks of the statistics, of the forward pass (16392) and of the backward pass walk."""
    if torch.cuda.mem_get_info()[0] < 200 << 30:
        pytest.skip("needs 200 GB of device memory")
    check_norm(65541, C, BF16)


# ---- parameters at odd addresses ----------------------------------------------------------------------------------------------
@pytest.mark.parametrize("wdtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("C", [5, 64, 601, 1200, 9001])
def test_parameters_at_odd_addresses(hip, C, wdtype):
    from siv import ops as o
    x, dy, w, b = B.inputs(7, C, BF16, C, "cuda")
    w, b = w.to(wdtype), b.to(wdtype)
    wide = torch.zeros(2 * C + 5, dtype=wdtype, device="cuda")
    wide[1:1 + C], wide[C + 4:2 * C + 4] = w, b
    x.requires_grad_()
    got = [o.layer_norm(x, wide[1:1 + C], wide[C + 4:2 * C + 4])]
    want = [o.layer_norm(x, w, b)]
    assert torch.equal(got[0], want[0])
    assert torch.equal(*(torch.autograd.grad(y[0], x, dy)[0] for y in (got, want)))
