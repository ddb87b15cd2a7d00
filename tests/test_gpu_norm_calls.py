"""Layer norm, dropout and the residual step called through what torch puts around an operator -- recorded traces, function
transforms, hooks on saved tensors, one parameter twice -- and dropout behind an activation in every type."""
import pytest
import torch

pytestmark = pytest.mark.gpu
CL3D = torch.channels_last_3d


@pytest.fixture(params=["nodes", "python"])
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


def key(seed=5, sid=11):
    from siv import rng
    return rng.PhiloxKeep(seed, sid)


def rnd(seed, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def operators(o):
    """(name, call on (x, residual, weight, bias)) of every entry point; one result each."""
    return [("layer_norm", lambda x, r, w, b: o.layer_norm(x, w, b)),
            ("layer_norm_plain", lambda x, r, w, b: o.layer_norm(x)),
            ("dropout", lambda x, r, w, b: o.dropout(x, key(), 0.5)),
            ("dropout_residual", lambda x, r, w, b: o.dropout(x, key(), 0.5, residual=r)),
            ("act_dropout", lambda x, r, w, b: o.act_dropout(x, 0.2, key(), 0.5)),
            ("add_layer_norm", lambda x, r, w, b: o.add_layer_norm(x, r, w, b, keep=key(), p=0.5)[0]),
            ("add_layer_norm_sum", lambda x, r, w, b: o.add_layer_norm(x, r, w, b, keep=key(), p=0.5)[1]),
            ("add_layer_norm_plain", lambda x, r, w, b: sum(o.add_layer_norm(x, r)))]


NAMES = [n for n, _ in operators(None)]


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("name", NAMES)
def test_traced_calls_compute(hip, name, grad):
    """A function recorded by torch.jit.trace computes the operator on the inputs of each later call (memory of other
    values handed back to the allocator in between)."""
    from siv import ops as o
    f = dict(operators(o))[name]
    args = [rnd(1, 6, 40), rnd(2, 6, 40), rnd(3, 40), rnd(4, 40)]
    if grad:
        args = [t.requires_grad_() for t in args]
    traced = torch.jit.trace(lambda x, r, w, b: f(x, r, w, b) * 1.0 + 0 * (x + r + w + b), args, check_trace=False)
    for seed in (10, 20, 30):
        args = [rnd(seed + i, 6, 40) for i in range(2)] + [rnd(seed + i, 40) for i in (2, 3)]
        want = f(*args)
        junk = [torch.full((6, 40), 1e3, device="cuda") for _ in range(16)]
        del junk
        assert torch.equal(traced(*args), want)


@pytest.mark.parametrize("mode", ["real", "fake", "symbolic"])
@pytest.mark.parametrize("name", NAMES)
def test_make_fx_is_refused(hip, name, mode):
    """make_fx has no way to record a kernel: an error, not a graph without it.  Modes that only watch change nothing."""
    from siv import ops as o
    from torch.fx.experimental.proxy_tensor import make_fx
    from torch.utils.flop_counter import FlopCounterMode
    f = dict(operators(o))[name]
    args = [rnd(1, 6, 40), rnd(2, 6, 40), rnd(3, 40), rnd(4, 40)]
    with pytest.raises(Exception, match="make_fx"):
        make_fx(f, tracing_mode=mode)(*args)
    want = f(*args)
    with FlopCounterMode(display=False):
        got = f(*args)
    assert torch.equal(got, want)


@pytest.mark.parametrize("name", NAMES)
def test_function_transforms_are_refused(hip, name):
    """vmap, grad, jvp, functionalize and batched gradients have no rule here: an error in words, not one about storage."""
    import torch.func as F
    from siv import ops as o
    f = dict(operators(o))[name]
    x, r, w, b = args = [rnd(1, 6, 40), rnd(2, 6, 40), rnd(3, 40), rnd(4, 40)]
    calls = [lambda: F.vmap(lambda t: f(t, r, w, b))(torch.stack((x, x))), lambda: F.grad(lambda t: f(t, r, w, b).sum())(x),
             lambda: F.grad(lambda t: (t * f(*args)).sum())(x), lambda: F.jvp(lambda t: f(t, r, w, b), (x,), (x,)),
             lambda: F.functionalize(lambda t: f(t, r, w, b))(x)]
    xg = x.clone().requires_grad_()
    y = f(xg, r, w, b)
    calls.append(lambda: torch.autograd.grad(y, xg, rnd(5, 3, 6, 40), is_grads_batched=True))
    for call in calls:
        with pytest.raises(RuntimeError, match="functorch transforms|torch.func"):
            call()
    assert torch.equal(f(*args), y)
    # what is handed on as it came may be anything
    rg, up = r.clone().requires_grad_(), rnd(5, 3, 6, 40)
    for out in (o.dropout(x, key(), 0.5, residual=rg), o.add_layer_norm(x, rg, keep=key(), p=0.5)[1]):
        assert torch.equal(torch.autograd.grad(out, rg, up, is_grads_batched=True)[0], up)


def volume(seed, dtype=torch.float32):
    return rnd(seed, 2, 6, 3, 4, 5, dtype=dtype).contiguous(memory_format=CL3D)


def masked_operators(o, m):
    """Every entry point on volumes with the stored mask ``m`` where it takes one."""
    return [lambda x, r, w, b: o.layer_norm(x, w, b), lambda x, r, w, b: o.dropout(x, m, 0.5),
            lambda x, r, w, b: o.dropout(x, m, 0.5, residual=r), lambda x, r, w, b: o.act_dropout(x, 0.2, m, 0.5),
            lambda x, r, w, b: o.act_dropout(x, 0.2, key(), 0.5),
            lambda x, r, w, b: sum(o.add_layer_norm(x, r, w, b, keep=m, p=0.5)),
            lambda x, r, w, b: o.add_layer_norm(x, r, w, b, keep=m, p=0.5)[1]]


@pytest.mark.parametrize("i", range(7))
def test_saved_tensors_come_back_in_other_memory(hip, i):
    """Hooks on saved tensors hand back the values in memory of another order (pinned host copies do): same gradients."""
    from siv import ops as o
    m = (volume(9) > 0).to(torch.uint8)
    f = masked_operators(o, m)[i]
    args = [t.requires_grad_() for t in (volume(1), volume(2), rnd(3, 6), rnd(4, 6))]
    dy = volume(5)

    def apart(t):
        if t.dim() == 5:
            return t.contiguous()                                   # NCDHW memory
        return torch.stack((t, t + 1), -1)[..., 0] if t.dim() == 1 else t
    want = torch.autograd.grad(f(*args), args, dy, allow_unused=True)
    for hooks in (torch.autograd.graph.saved_tensors_hooks(lambda t: t, apart),
                  torch.autograd.graph.save_on_cpu(pin_memory=True), torch.autograd.graph.save_on_cpu()):
        with hooks:
            y = f(*args)
        got = torch.autograd.grad(y, args, dy, allow_unused=True)
        assert all(a is b or torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("i", [0, 1, 2, 4, 5, 6])
def test_saved_tensors_that_come_back_changed_are_refused(hip, i):
    """Hooks that hand back another device, type or shape than was saved -- of everything, of the weights, of the mask --
    meet an error before anything is launched."""
    from siv import ops as o
    m = (volume(9) > 0).to(torch.uint8)
    f = masked_operators(o, m)[i]
    args = [t.requires_grad_() for t in (volume(1), volume(2), rnd(3, 6), rnd(4, 6))]
    which = {"all": lambda t: True, "weight": lambda t: t.dim() == 1, "mask": lambda t: t.dtype == torch.uint8}
    touched = {"weight": i in (0, 5, 6), "mask": i in (1, 2, 5, 6), "all": True}
    for name, mine in which.items():
        for change in (lambda t: t.cpu(), lambda t: t.to(torch.float16 if t.is_floating_point() else torch.int16),
                       lambda t: t[:1], lambda t: t.double()):
            if not touched[name]:
                continue
            with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: change(t) if mine(t) else t):
                y = f(*args)
            if name == "weight" and i == 6 and hip.nodes is None:
                continue                    # (the sum alone: the Python function does not look at the weights)
            with pytest.raises(RuntimeError):
                torch.autograd.grad(y, args, volume(5), allow_unused=True)


@pytest.mark.parametrize("held,back", [(torch.float32, torch.bfloat16), (torch.bfloat16, torch.float32)])
def test_weights_that_come_back_in_the_other_type_are_refused(hip, held, back):
    """Weights may be float32 or of x's type; their gradient has the type they had, not the one a hook made of it."""
    from siv import ops as o
    x = rnd(1, 4, 40, dtype=torch.bfloat16).requires_grad_()
    w = rnd(2, 40, dtype=held).requires_grad_()
    for f in (lambda: o.layer_norm(x, w), lambda: o.add_layer_norm(x, x.detach(), w)[0]):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t.to(back) if t.dim() == 1 else t):
            y = f()
        with pytest.raises(RuntimeError):
            torch.autograd.grad(y, (x, w), rnd(3, 4, 40, dtype=torch.bfloat16))


@pytest.mark.parametrize("R,C", [(5, 96), (9603, 256), (300, 9001)])
def test_one_parameter_as_weight_and_bias(hip, R, C):
    """Both gradients of a parameter that is weight and bias at once reach its flat optimiser buffer: the sum of the two."""
    from siv import ops as o
    from siv.optim import FlatAdam
    x, dy = rnd(1, R, C), rnd(2, R, C)
    w = torch.nn.Parameter(1 + 0.2 * rnd(3, C))
    a, b = w.detach().clone().requires_grad_(), w.detach().clone().requires_grad_()
    dw, db = torch.autograd.grad(o.layer_norm(x, a, b), (a, b), dy)
    opt = FlatAdam([w], lr=1e-3)
    opt.zero_grad()
    o.layer_norm(x, w, w).backward(dy)
    assert torch.equal(w.grad, dw + db)
    o.add_layer_norm(x, dy, w, w)[0].backward(dy)
    dw2, db2 = torch.autograd.grad(o.add_layer_norm(x, dy, a, b)[0], (a, b), dy)
    assert torch.equal(w.grad, (dw + db) + (dw2 + db2))       # the order of the additions: a pass's two, then into .grad


# ---- dropout behind an activation ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("slope", [0.0, 0.2, 1.0])
@pytest.mark.parametrize("shape", [(1,), (5,), (13, 77), (70001,), (2, 3, 5, 7, 4)])
def test_act_dropout_of_every_type(hip, shape, slope, dtype):
    """LeakyReLU, dropout from a key, and (backend and C entry point) a residual: float64 values within a product's, a scaling's
    and an addition's roundings in fp32 and one to the type; the gradient likewise."""
    from siv import ops as o
    u, half = 2.0 ** -24, torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).smallest_normal * half
    fmt = CL3D if len(shape) == 5 else torch.contiguous_format
    x, dy, res = (rnd(s, *shape, dtype=dtype).contiguous(memory_format=fmt) for s in (1, 2, 3))
    k, p = key(2 ** 63 + 9, (3 << 40) | 17), 0.35
    m = hip.dropout_keep(shape if len(shape) == 5 else (1, 1, 1, 1, x.numel()), x.device, p, k.seed, k.stream_id)
    m = (m if len(shape) == 5 else m.view(shape)).double()
    one = torch.tensor(1.0)
    sc, a = float(one / (one - torch.tensor(p))), float(torch.tensor(slope))
    xg = x.clone().requires_grad_()
    out = o.act_dropout(xg, slope, k, p)
    x64 = x.double()
    ref = torch.where(x64 > 0, x64, a * x64) * m * sc
    assert out.dtype == dtype and bool(((out.double() - ref).abs() <= (half + 2 * u) * ref.abs() + tiny).all())
    dx, = torch.autograd.grad(out, xg, dy)
    gref = dy.double() * m * sc * torch.where(x64 > 0, 1.0, a)
    assert bool(((dx.double() - gref).abs() <= (half + 2 * u) * gref.abs() + tiny).all())
    got = hip.dropout_fwd(x, k, p, slope, res)
    both = res.double() + ref
    assert bool(((got.double() - both).abs() <= (half + u) * both.abs() + 2 * u * ref.abs() + tiny).all())
    assert torch.equal(got, hip.dropout_fwd(x, m.to(torch.uint8), p, slope, res))
    raw = torch.empty_like(x)
    rc = hip.lib.siv_dropout_fwd(x.data_ptr(), res.data_ptr(), None, k.seed, k.stream_id, None, p, slope, raw.data_ptr(),
                                 hip._TYPES[dtype], x.numel(), torch.cuda.current_stream().cuda_stream)
    assert rc == 0 and torch.equal(raw, got)


@pytest.mark.parametrize("dynamic", [False, True])
@pytest.mark.parametrize("i", [0, 2, 4, 5])
def test_compiled_functions_compute(hip, i, dynamic):
    """torch.compile runs the operators between its graphs, for fixed and for changing shapes, volumes in either order."""
    from siv import ops as o
    torch._dynamo.reset()
    m = {n: (torch.rand(n, 6, 3, 4, 5, device="cuda") > 0.5).to(torch.uint8) for n in (2, 3)}

    def f(x, r, w, b):
        return masked_operators(o, m[x.shape[0]])[i](x * 2, r, w, b) + 1
    run = torch.compile(f, backend="eager", dynamic=dynamic)
    for n, fmt in ((2, CL3D), (3, CL3D), (3, torch.contiguous_format)):
        args = [t.contiguous(memory_format=fmt).requires_grad_() for t in (rnd(n, n, 6, 3, 4, 5), rnd(n + 5, n, 6, 3, 4, 5))]
        args += [rnd(3, 6).requires_grad_(), rnd(4, 6).requires_grad_()]
        dy = rnd(9, n, 6, 3, 4, 5)
        want, got = f(*args), run(*args)
        assert torch.equal(got, want)
        for a, c in zip(*(torch.autograd.grad(y, args, dy, allow_unused=True) for y in (got, want))):
            assert a is c or torch.equal(a, c)
    torch._dynamo.reset()
