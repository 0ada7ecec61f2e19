"""Calls of the expert block's operators that are not the ordinary ones: what reaches a kernel, and what must not."""

import threading

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import adambridge_amd as ab
from adambridge_amd import _hip, experts, norms

pytestmark = pytest.mark.gpu

NAMES = ("layer_norm", "route", "route_all", "dispatch", "combine", "expert_mm")


def _gen(seed):
    return torch.Generator("cuda").manual_seed(seed)


def _operator(name, dtype=torch.float32):
    """The operator as a function of its differentiable operands, and those."""
    gen = _gen(len(name))
    leaf = lambda *shape: torch.randn(*shape, generator=gen, device="cuda").to(dtype).requires_grad_()
    r = ab.route(torch.randn(24, 6, generator=gen, device="cuda"), 2)
    if name == "layer_norm":
        return ab.layer_norm, [leaf(24, 40), leaf(40), leaf(40)]
    if name.startswith("route"):
        return lambda x: ab.route(x, 3, normalize=name == "route").weights, [leaf(24, 16)]
    if name == "dispatch":
        return lambda x: ab.dispatch(x, r), [leaf(24, 40)]
    if name == "combine":
        return lambda y, w: ab.combine(y, r._replace(weights=w)), [leaf(48, 40), r.weights.detach().clone().requires_grad_()]
    return lambda x, w: ab.expert_mm(x, w, r.ends), [leaf(48, 40), leaf(6, 24, 40)]


def _gradients(name, dtype=torch.float32, seed=1):
    fn, leaves = _operator(name, dtype)
    out = fn(*leaves)
    g = torch.randn(out.shape, generator=_gen(seed), device="cuda").to(out.dtype)
    return torch.autograd.grad(out, leaves, g)


def _near(got, want):
    return torch.allclose(got, want, rtol=1e-4, atol=1e-5 * (1.0 + want.abs().max().item()))


# ------------------------------------------------------------------------------- tangents

@pytest.mark.parametrize("name", NAMES)
def test_a_gradient_s_tangent_is_carried_on(name):
    """Forward mode over a backward pass, the dual operand behind the operator: its gradient is linear in the one that
    arrives, so the tangent of its gradient is the gradient of the tangent."""
    fn, leaves = _operator(name)
    out = fn(*leaves)
    scale, tangent = (torch.randn(out.shape, generator=_gen(s), device="cuda") for s in (5, 6))
    with forward_ad.dual_level():
        grads = torch.autograd.grad((fn(*leaves) * forward_ad.make_dual(scale, tangent)).sum(), leaves)
        got = [forward_ad.unpack_dual(t) for t in grads]
        got = [(t.primal.clone(), None if t.tangent is None else t.tangent.clone()) for t in got]
    want = zip(torch.autograd.grad(out, leaves, scale, retain_graph=True), torch.autograd.grad(out, leaves, tangent))
    for (primal, moved), (want_primal, want_moved) in zip(got, want):
        assert moved is not None
        assert _near(primal, want_primal) and _near(moved, want_moved)


@pytest.mark.parametrize("name", NAMES)
def test_second_derivatives(name):
    """The kernels' gradients, differentiated in turn: as torch operations differentiate the definition in 64 bits."""
    _, leaves = _operator(name)
    r = ab.route(torch.randn(24, 6, generator=_gen(9), device="cuda"), 2)
    fns = {"layer_norm": lambda r: ab.layer_norm, "route": lambda r: lambda x: ab.route(x, 3).weights,
           "route_all": lambda r: lambda x: ab.route(x, 3, normalize=False).weights, "dispatch": lambda r: lambda x: ab.dispatch(x, r),
           "combine": lambda r: lambda y, w: ab.combine(y, r._replace(weights=w)), "expert_mm": lambda r: lambda x, w: ab.expert_mm(x, w, r.ends)}
    results = []
    for cast in (lambda t: t, lambda t: t.cpu().double() if t.is_floating_point() else t.cpu()):
        here = [cast(t.detach()).requires_grad_() for t in leaves]
        out = fns[name](ab.Routing(*map(cast, r)))(*here)
        g, *moves = [cast(torch.randn(t.shape, generator=_gen(20 + i), device="cuda")) for i, t in enumerate((out, *here))]
        g.requires_grad_()
        first = torch.autograd.grad((out * out).sum() if name == "dispatch" else (out * g).sum(), here, create_graph=True)
        second = torch.autograd.grad(sum((a * m).sum() for a, m in zip(first, moves)), [g, *here], allow_unused=True)
        results.append([t if t is None else t.cpu().float() for t in second])
    for got, want in zip(*results):
        assert (got is None) == (want is None) and (got is None or _near(got, want) or torch.allclose(got, want, rtol=1e-3, atol=1e-3))
    assert any(t is not None for t in results[0])


# ------------------------------------------------------------------------- saved tensors

def _strided(t):
    """The same values in memory of another order."""
    if t.dim() == 1:
        return torch.stack((t, t), 1)[:, 0]
    return t.transpose(-1, -2).contiguous().transpose(-1, -2)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("name", NAMES)
def test_saved_tensors_that_come_back_strided(name, dtype):
    want = _gradients(name, dtype)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, _strided):
        got = _gradients(name, dtype)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_saved_tensors_that_come_back_expanded():
    """Equal rows given back as one row of memory, expanded."""
    r = ab.route(torch.randn(24, 6, generator=_gen(0), device="cuda"), 2)

    def rows(*shape):
        return torch.randn(shape[1:], generator=_gen(1), device="cuda").expand(shape).contiguous().requires_grad_()

    cases = [(ab.layer_norm, [rows(24, 40), rows(1, 40)[0].detach().requires_grad_()]),
             (lambda y, w: ab.combine(y, r._replace(weights=w)), [rows(48, 40), rows(24, 2)]),
             (lambda x, w: ab.expert_mm(x, w, r.ends), [rows(48, 40), rows(6, 24, 40)])]
    for fn, leaves in cases:
        ordinary = fn(*leaves)
        g = torch.randn(ordinary.shape, generator=_gen(2), device="cuda")
        want = torch.autograd.grad(ordinary, leaves, g)
        equal_rows = lambda t: t.dim() > 1 and t.is_floating_point() and bool((t == t[:1]).all())
        with torch.autograd.graph.saved_tensors_hooks(lambda t: (t[:1].clone(), t.shape) if equal_rows(t) else t,
                                                      lambda p: p[0].expand(p[1]) if type(p) is tuple else p):
            out = fn(*leaves)
            got = torch.autograd.grad(out, leaves, g)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("name", ["layer_norm", "route_all", "combine"])
def test_saved_tensors_that_come_back_of_another_type(name):
    """Torch operations take them, in whatever type they are."""
    want = _gradients(name)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t.double() if t.is_floating_point() else t):
        got = _gradients(name)
    assert all(a.dtype == b.dtype and _near(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("back", [lambda t: t[:-1], lambda t: t[..., None], lambda t: t.cpu()],
                         ids=["fewer", "another dimension", "the host's"])
@pytest.mark.parametrize("name", NAMES)
def test_saved_tensors_that_cannot_be_the_operand_s_are_refused(name, back):
    """On the host, before any address of a smaller tensor reaches a kernel or an index a device."""
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, back), pytest.raises(RuntimeError, match="came back|same device"):
        _gradients(name)
    fn, leaves = _operator(name)   # nor where torch operations follow
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, back), pytest.raises(RuntimeError, match="came back|same device"):
        out = fn(*leaves)
        torch.autograd.grad(out, leaves, torch.ones_like(out), create_graph=True)


# ----------------------------------------------------------------------- default devices

def test_a_default_device_leaves_the_kernels_on(monkeypatch):
    """A default device says where factory calls put their tensors; it observes no operation."""
    want = [_gradients(name) for name in NAMES]
    for module, name in ((experts, "_torch_route"), (experts, "_torch_dispatch"), (experts, "_torch_gather_sum"),
                         (experts, "_torch_rows"), (norms, "_torch_layer_norm")):
        monkeypatch.setattr(module, name, None)
    for device in ("cuda", "cpu"):
        with torch.device(device):
            got = [_gradients(name) for name in NAMES]
        assert all(torch.equal(a, b) for one, two in zip(got, want) for a, b in zip(one, two))


def test_a_mode_that_observes_operations_sees_them():
    class Count(torch.overrides.TorchFunctionMode):
        def __init__(self):
            self.seen = 0

        def __torch_function__(self, func, types, args=(), kwargs=None):
            self.seen += 1
            return func(*args, **(kwargs or {}))

    for name in NAMES:
        fn, leaves = _operator(name)
        with torch.device("cuda"), Count() as count:
            fn(*leaves)
        assert count.seen > 4, name


# -------------------------------------------------------------------------- zero tensors

def test_tensors_without_memory_take_torch_operations():
    """A tensor of zeros that holds no memory has no address to give to a kernel."""
    zero = lambda *shape: torch._efficientzerotensor(shape, device="cuda")
    some = lambda *shape: torch.randn(*shape, generator=_gen(3), device="cuda")
    r = ab.route(some(12, 4), 2)
    bias = some(16)
    assert torch.equal(ab.layer_norm(zero(12, 16), some(16), bias), bias.expand(12, 16))
    assert torch.equal(ab.route(zero(12, 4), 2).experts, torch.tensor([0, 1], device="cuda").int().expand(12, 2))
    assert not ab.dispatch(zero(12, 16), r).any() and not ab.combine(zero(24, 16), r).any()
    assert not ab.expert_mm(zero(24, 16), some(4, 8, 16), r.ends).any()
    assert not ab.expert_mm(some(24, 16), zero(4, 8, 16), r.ends).any()


# ---------------------------------------------------------------------------- transforms

@pytest.mark.parametrize("name", NAMES)
def test_function_transforms(name):
    """torch.func's grad, jvp and vmap give the ordinary gradients, linear forms and rows."""
    fn, leaves = _operator(name)
    out = fn(*leaves)
    g = torch.randn(out.shape, generator=_gen(1), device="cuda")
    want = torch.autograd.grad(out, leaves, g)
    free = [t.detach() for t in leaves]
    got = torch.func.grad(lambda *ts: (fn(*ts) * g).sum(), argnums=tuple(range(len(free))))(*free)
    assert all(_near(a, b) for a, b in zip(got, want))
    moves = [torch.randn(t.shape, generator=_gen(8 + i), device="cuda") for i, t in enumerate(free)]
    primal, moved = torch.func.jvp(fn, tuple(free), tuple(moves))
    assert _near(primal, out.detach())
    assert torch.allclose((moved * g).sum(), sum((a * b).sum() for a, b in zip(want, moves)), rtol=1e-3, atol=1e-2)
    if name not in ("route", "route_all"):   # (theirs: test_routings_of_a_batch)
        twice = torch.func.vmap(fn, in_dims=(0,) + (None,) * (len(free) - 1))(torch.stack((free[0], 2 * free[0])), *free[1:])
        assert _near(twice[0], out.detach()) and _near(twice[1], fn(2 * free[0], *free[1:]))


def test_routings_of_a_batch():
    logits = torch.randn(3, 70, 12, generator=_gen(4), device="cuda")
    for normalize in (True, False):
        one_by_one = [ab.route(t, 2, normalize) for t in logits]
        at_once = torch.func.vmap(lambda t: tuple(ab.route(t, 2, normalize)))(logits)
        assert _near(at_once[0], torch.stack([r.weights for r in one_by_one]))
        for i in range(1, 5):
            assert torch.equal(at_once[i], torch.stack([r[i] for r in one_by_one]))


# ----------------------------------------------------------------- threads and refusals

def test_threads_have_a_stream_each():
    want = [_gradients(name) for name in NAMES]
    torch.cuda.synchronize()
    got, errors = {}, []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(5):
                    got[i] = [_gradients(name) for name in NAMES]
                torch.cuda.current_stream().synchronize()
        except Exception as error:   # reported by the thread that asserts
            errors.append(error)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(3)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not errors and len(got) == 3
    for one in got.values():
        assert all(torch.equal(a, b) for x, y in zip(one, want) for a, b in zip(x, y))


def test_calls_that_are_not_ordinary_ones_are_left_to_python():
    """The native calls answer None, before anything is done, to what their kernels do not take."""
    o = _hip.ops()
    x, w, b = (torch.randn(*s, device="cuda") for s in ((6, 16), (16,), (16,)))
    for args in ((x.half(), w, b, 1e-5), (x.t(), w[:6], None, 1e-5), (x[:, ::2], None, None, 1e-5), (x, w[:8], None, 1e-5),
                 (x, w, b.bfloat16(), 1e-5), (x, w.cpu(), None, 1e-5), (x.cpu(), None, None, 1e-5), (x, w.double(), None, 1e-5),
                 (x, w, b, 1), (x[:0], w, b, 1e-5), (x[0, 0], None, None, 1e-5), (x, w, 3.0, 1e-5), (x, w, None)):
        assert o.layer_norm(*args) is None
    for args in ((x.half(), 2, True), (x, 17, True), (x, 0, True), (x, True, True), (x, 2, 1), (x, 1 << 70, True), (x.t(), 2, True),
                 (x[0], 1, True), (x[:0], 2, True), (torch.randn(2, 1025, device="cuda"), 2, True),
                 (torch.randn(2, 100, device="cuda"), 65, True)):
        assert o.route(*args) is None
    r = ab.route(torch.randn(6, 4, device="cuda"), 2)
    y = torch.randn(12, 16, device="cuda")
    for args in ((x, r.position.long()), (x, r.position[:5]), (x, r.position.t()), (x, r.position.cpu()), (x.double(), r.position),
                 (x[0], r.position), (x, r.position[0]), (x, None)):
        assert o.dispatch(*args) is None
    for args in ((x, r.weights, r.position), (y, r.weights.double(), r.position), (y, r.weights[:, :1].contiguous(), r.position),
                 (y, r.weights, r.position.long()), (y, r.weights.cpu(), r.position), (y.t(), r.weights, r.position), (y, None, r.position)):
        assert o.combine(*args) is None
    w = torch.randn(4, 8, 16, device="cuda")
    for args in ((y, w.bfloat16(), r.ends), (y, w, r.ends.long()), (y, w, r.ends[:3]), (y, w[:, :, :8].contiguous(), r.ends),
                 (y, w.transpose(1, 2), r.ends), (y.half(), w.half(), r.ends), (y, w[0], r.ends), (y, w, r.ends.cpu()),
                 (y, w[:, :0], r.ends), (y[0], w, r.ends)):
        assert o.expert_mm(*args) is None
    with torch.autocast("cuda", dtype=torch.bfloat16):
        assert o.expert_mm(y, w, r.ends) is None
    with pytest.raises(ValueError, match="of one type"):
        ab.layer_norm(x, torch.ones(16, device="cuda"), b.bfloat16())
    with pytest.raises(ValueError, match="top_k must be an int"):
        ab.route(x, 17)
    with pytest.raises(ValueError, match="int32"):
        ab.dispatch(x, r._replace(position=r.position.long()))
    with pytest.raises(ValueError, match="weights must be float32"):
        ab.combine(y, r._replace(weights=r.weights.double()))
    with pytest.raises(ValueError, match="on one device"):
        ab.expert_mm(y, w, r.ends.cpu())
    assert ab.expert_mm(y.half(), w.half(), r.ends).dtype == torch.float16   # torch operations
