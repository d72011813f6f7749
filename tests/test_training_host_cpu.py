"""What the host side of the training operators hands to the library, on CPU tensors and with a library that records its
arguments in place of the kernels."""
import ctypes

import pytest
import torch

from conversenet_amd import functional

EPS = 1e-5


def _read(address, n):
    return torch.tensor((ctypes.c_float * n).from_address(address)[:])


class Library:
    """cvn_residual_norm_fwd leaves 1, 2, 3 .. in each output; cvn_residual_norm_bwd keeps what it was given to read;
    cvn_clip_grads halves."""

    def __init__(self):
        self.forwards = 0
        self.read = None

    def cvn_residual_norm_fwd(self, x, xt, h, ht, B, C, HW, s, gate, kind, pw, pb, peps, nw, nb, neps, r, y, stats, stream):
        self.forwards += 1
        for p, n in ((r, B * C * HW), (y, B * C * HW), (stats, (4 if pw else 2) * B * HW)):
            if p:
                (ctypes.c_float * n).from_address(p)[:] = [float(i + 1) for i in range(n)]
        return 0

    def cvn_residual_norm_bwd_workspace(self, B, C, HW, kind):
        return 64

    def cvn_residual_norm_bwd(self, gr, gy, base, xt, h, ht, B, C, HW, s, gate, kind, pw, pb, nw, stats, *rest):
        n = B * C * HW
        sizes = dict(gr=n, gy=n, base=n, h=n, s=C, gate=n if kind == 2 else B * C, pw=C, pb=C, nw=C,
                     stats=(4 if pw else 2) * B * HW)
        at = dict(gr=gr, gy=gy, base=base, h=h, s=s, gate=gate, pw=pw, pb=pb, nw=nw, stats=stats)
        self.read = {k: _read(at[k], sizes[k]) for k in at if at[k]}
        return 0

    def cvn_grad_norm_workspace(self, sizes, n):
        return 64

    def cvn_clip_grads(self, grads, out, sizes, types, n, *rest):
        """Every output half its float32 gradient."""
        table = lambda at, t: (t * n).from_address(at)[:]  # noqa: E731
        for g, o, k in zip(table(grads, ctypes.c_uint64), table(out, ctypes.c_uint64), table(sizes, ctypes.c_int64)):
            (ctypes.c_float * k).from_address(o)[:] = (_read(g, k) / 2).tolist()
        return 0


@pytest.fixture
def library(monkeypatch):
    lib = Library()
    monkeypatch.setattr(torch.Tensor, "get_device", lambda t: 0)
    monkeypatch.setattr(functional._lib, "load", lambda: lib)
    monkeypatch.setattr(functional, "_stream", lambda dev: 0)
    monkeypatch.setattr(functional, "_on", lambda dev: functional._NO_SWITCH)
    functional._norm_workspace.cache_clear()
    yield lib
    functional._norm_workspace.cache_clear()
    functional.release_workspace()


def _args(shape=(2, 3, 4, 5), seed=0):
    g = torch.Generator().manual_seed(seed)
    C = shape[1]
    d = {k: torch.randn(shape, generator=g) for k in ("x", "h", "gate")}
    d.update({k: torch.randn(C, generator=g) for k in ("s", "w", "b", "pw", "pb")})
    return {k: v.requires_grad_(True) for k, v in d.items()}


def _call(d):
    return functional.residual_norm_train(d["x"], d["h"], (d["w"], d["b"], EPS), d["s"], d["gate"], (d["pw"], d["pb"], EPS))


def _spread(t):
    """The same values, two addresses apart."""
    big = torch.full((*t.shape, 2), float("nan"))
    big[..., 0] = t
    return big[..., 0]


def _expanded(t):
    """A tensor of one value as a view of a single element; what lies behind it is something else."""
    big = torch.full((t.numel() + 1,), float("nan"))
    big[0] = t.flatten()[0]
    return big[:1].view((1,) * t.dim()).expand(t.shape)


@pytest.mark.parametrize("layout", ["channels last", "spread", "expanded"])
def test_saved_tensors_of_any_layout(library, layout):
    """A saved-tensor hook may give a tensor back with other strides: its values, size and type are what counts."""
    d = _args()
    if layout == "expanded":
        with torch.no_grad():
            for i, v in enumerate(d.values()):
                v.fill_(i + 0.5)

    def unpack(t):
        t = t.clone()
        if layout == "channels last":
            return t.to(memory_format=torch.channels_last) if t.dim() == 4 else t
        if layout == "expanded":
            return _expanded(t) if t.unique().numel() == 1 else t
        return _spread(t)

    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach(), unpack):
        r, y = _call(d)
    gr, gy = torch.randn(r.shape), torch.randn(y.shape)
    torch.autograd.grad((r, y), list(d.values()), (gr, gy))
    want = dict(gr=gr, gy=gy, base=r, h=d["h"], s=d["s"], gate=d["gate"], pw=d["pw"], pb=d["pb"], nw=d["w"],
                stats=torch.arange(1.0, 4 * 2 * 20 + 1))
    assert set(library.read) == set(want)
    for k, v in want.items():
        assert torch.equal(library.read[k], v.detach().flatten()), k


@pytest.fixture
def on_device(library, monkeypatch):
    monkeypatch.setattr(torch.Tensor, "is_cuda", True, raising=False)
    return library


def _norm_module(C=3):
    from conversenet_amd import util_converse as U

    m = U.LayerNorm(C, eps=EPS, data_format="channels_first")
    with torch.no_grad():
        m.weight.copy_(torch.arange(1.0, C + 1))
        m.bias.copy_(torch.arange(C) - 0.5)
    return m


def _block():
    """A block of three channels whose convolutions are torch's."""
    from conversenet_amd import util_converse as U

    blk = U.ConverseBlockAlphaVariant(3, 3, kernel_size=3, padding=1)
    for m in blk.modules():
        if isinstance(m, U.Converse2D):
            m.backend = "pytorch"
    return blk


def _definition(m, x):
    d = x - x.mean(1, keepdim=True)
    hat = d / torch.sqrt(d.pow(2).mean(1, keepdim=True) + EPS)
    return m.weight.view(-1, 1, 1) * hat + m.bias.view(-1, 1, 1)


@pytest.mark.parametrize("pre_dispatch", [False, True])
def test_a_traced_norm_is_its_operations(on_device, pre_dispatch):
    """A graph of torch operations cannot hold the library's calls: what traces a module's operations sees all of them."""
    from torch.fx.experimental.proxy_tensor import make_fx

    m = _norm_module()

    def step(x, go):
        y = m(x)
        # (torch traces sqrt's gradient before dispatch with the result of the tracing call as a constant)
        return (y,) if pre_dispatch else (y, *torch.autograd.grad(y, (x, m.weight), go))

    def inputs(seed):
        g = torch.Generator().manual_seed(seed)
        return torch.randn(2, 3, 4, 5, generator=g).requires_grad_(True), torch.randn(2, 3, 4, 5, generator=g)

    graph = make_fx(step, pre_dispatch=pre_dispatch)(*inputs(0))
    assert on_device.forwards == 0
    x, go = inputs(1)
    y = _definition(m, x)
    want = (y, *torch.autograd.grad(y, (x, m.weight), go))
    for a, b in zip(graph(x, go), want):
        assert torch.allclose(a, b, rtol=0, atol=1e-5)
    m(x)
    assert on_device.forwards == 1


def test_modes_see_a_norms_operations(on_device):
    from torch.overrides import TorchFunctionMode
    from torch.utils._python_dispatch import TorchDispatchMode

    seen = []

    class Dispatch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))

    class Function(TorchFunctionMode):
        def __torch_function__(self, func, types, args=(), kwargs=None):
            seen.append(getattr(func, "__name__", ""))
            return func(*args, **(kwargs or {}))

    m = _norm_module()
    x = torch.randn(1, 3, 2, 2, requires_grad=True)
    for mode in (Dispatch, Function):
        seen.clear()
        with mode():
            y = m(x)
        assert torch.allclose(y, _definition(m, x), rtol=0, atol=1e-5) and any("mean" in s for s in seen)
    assert on_device.forwards == 0
    with torch.device("cpu"):  # a default device is a mode too, and observes nothing
        m(x)
    assert on_device.forwards == 1


def test_a_traced_backward_is_its_operations(library):
    """A forward on the library, and its backward traced."""
    from torch.fx.experimental.proxy_tensor import make_fx

    d = _args()
    r, y = _call(d)
    keys = ("x", "h", "gate", "s", "w", "b", "pw", "pb")

    def back(gr, gy):
        return torch.autograd.grad((r, y), [d[k] for k in keys], (gr, gy), retain_graph=True)

    gr, gy = torch.randn(r.shape), torch.randn(y.shape)
    graph = make_fx(back)(torch.randn(r.shape), torch.randn(y.shape))
    assert library.read is None
    want = torch.autograd.grad((r, y), [d[k] for k in keys], (gr, gy), create_graph=True)
    for a, b in zip(graph(gr, gy), want):
        assert torch.allclose(a, b, rtol=1e-4, atol=1e-5)


def test_traced_calls_are_refused(library):
    """The library's calls leave nothing in a graph: tracing one raises, and does not give a graph of empty outputs."""
    from torch.fx.experimental.proxy_tensor import make_fx

    F = functional
    x, w = torch.randn(1, 3, 2, 2), torch.ones(3)
    norm = (w, w, EPS)
    stats = torch.ones(2, 4)
    calls = [lambda x: F.residual_norm(x, x, norm)[0], lambda x: F.residual_norm_stats(x, x, norm)[0],
             lambda x: F.residual_norm_train(x, x, norm)[0], lambda x: F.layernorm_cf_train(x, w, w, EPS),
             lambda x: F.residual_norm_backward(x, x, x, x, stats, w)[0], lambda x: F.grad_norm([x]),
             lambda x: F.clip_grads([x], 1.0)[1]]
    for f in calls:
        with pytest.raises(RuntimeError, match="traced"):
            make_fx(f)(x)
        with pytest.raises(RuntimeError, match="traced"):
            torch.jit.trace(f, (x,), check_trace=False)
    assert library.forwards == 0 and library.read is None


@pytest.mark.parametrize("change", ["forward", "compile"])
@pytest.mark.parametrize("path", ["", "conv1", "conv2", "conv1.0", "conv2.0"])
def test_modules_with_a_forward_of_their_own_are_called(on_device, monkeypatch, path, change):
    from conversenet_amd import util_converse as U

    blk = U.ConverseBlockAlphaVariant(4, 4, kernel_size=3, padding=1)
    x = torch.randn(1, 4, 5, 5)
    ran = []
    monkeypatch.setattr(U, "_block_train", lambda b, x, n=None, ln=None: (ran.append("fused"), (x, n))[1])
    assert U._trainable(blk, x) and U._plain(blk)
    U.run_blocks([blk], x)
    assert ran == ["fused"]
    m = blk.get_submodule(path)
    if change == "forward":
        m.forward = lambda x: x
    else:
        m.compile(backend="eager")
    assert not (U._trainable(blk, x) and U._plain(blk))
    if path == "" and change == "forward":  # a chain calls it
        assert U.run_blocks([blk], x) is x and ran == ["fused"]


def test_clipping_records_nothing(library):
    """Gradients that have a graph of their own (create_graph) are scaled outside of it, whatever their strides."""
    ps = [torch.nn.Parameter(torch.zeros(3, 4)) for _ in range(5)]
    leaf = torch.randn(3, 4, requires_grad=True)
    strided = torch.randn(4, 3).t().requires_grad_(True)
    base = torch.randn(4, 3, requires_grad=True)
    for p, g in zip(ps, (leaf, leaf * 2, strided, strided * 2, base.t())):
        p.grad = g
    keep = [p.grad.detach().clone() for p in ps]
    nodes = [p.grad.grad_fn for p in ps]
    assert [p.grad.is_contiguous() for p in ps] == [True, True, False, False, False]
    functional.clip_grad_norm_(ps, 1.0)
    for i, (p, k, f) in enumerate(zip(ps, keep, nodes)):
        assert torch.equal(p.grad.detach(), k / 2) and p.grad.requires_grad
        assert i == 4 or p.grad.grad_fn is f  # (autograd writes a view's own node anew, with no_grad too)
    out, _ = functional.clip_grads([p.grad for p in ps], 1.0)
    assert not any(o.requires_grad for o in out) and torch.equal(out[2], keep[2] / 4)


def test_a_gradient_that_is_a_negated_view(library):
    """The gradient of a scalar that was an imaginary part may be a view whose memory holds its negative."""
    ps = [torch.nn.Parameter(torch.tensor(v)) for v in (2.0, 3.0)]
    (torch.complex(*ps).conj() * torch.tensor(1 + 2j)).abs().backward()
    grads = [p.grad for p in ps] + [torch.ones(4), torch.ones(1)]
    keep = [g.clone() for g in grads]
    assert [g.is_neg() for g in grads] == [False, True, False, False]
    for out in (None, [torch.zeros_like(g) for g in keep]):
        got, _ = functional.clip_grads(grads, 1.0, out=out)
        assert all(torch.equal(a, b / 2) for a, b in zip(got, keep))
    turned = torch.tensor([3.0, 5.0], dtype=torch.complex64).conj().imag[:1]
    functional.clip_grads([torch.ones(1)], 1.0, out=[turned])
    assert turned.is_neg() and turned.item() == 0.5
    functional.clip_grads(grads, 1.0, out=grads)
    functional.clip_grad_norm_(ps, 1.0)
    assert all(torch.equal(p.grad, k / 4) for p, k in zip(ps, keep))


def test_a_map_changed_after_its_norm(on_device):
    """A module's input may be changed in place behind it, as the composition allows: its backward has the values that the
    norm had."""
    m = _norm_module()
    x = torch.randn(2, 3, 4, 5, requires_grad=True)
    z = x * 1.0
    y = m(z)
    z.add_(1.0)
    torch.autograd.grad(y, x, torch.randn(2, 3, 4, 5))
    assert torch.equal(on_device.read["base"], torch.arange(1.0, 121))  # the copy that the forward made
    blk = _block()
    z = x * 1.0
    out = blk(z)
    z.mul_(2.0)
    torch.autograd.grad(out, x, torch.ones_like(x))


def test_a_bias_changed_before_the_backward(library):
    """The gradients do not depend on the norm's bias, and do not keep it."""
    d = _args()
    r, y = _call(d)
    with torch.no_grad():
        d["b"].add_(1.0)
    g = torch.autograd.grad((r, y), list(d.values()), (torch.ones_like(r), torch.ones_like(y)))
    assert g[5].shape == d["b"].shape and library.read is not None


def test_strided_gradients_in_one_place_are_refused(library):
    """As contiguous ones are: each would be counted twice and scaled once."""
    p, q, r = (torch.nn.Parameter(torch.zeros(3, 4)) for _ in range(3))
    p.grad = torch.randn(4, 3).t()
    q.grad = p.grad.view_as(p.grad)
    r.grad = torch.randn(3, 4)
    for ps in ((p, p), (p, q), (r, p, q)):
        keep = [t.grad.clone() for t in ps]
        with pytest.raises(RuntimeError, match="share memory"):
            functional.clip_grad_norm_(ps, 1.0)
        assert all(torch.equal(t.grad, k) for t, k in zip(ps, keep))
    both = torch.randn(3, 8)  # columns of one matrix share none
    p.grad, q.grad = both[:, :4], both[:, 4:]
    keep = both.clone()
    functional.clip_grad_norm_((p, q, r), 1.0)
    assert torch.equal(both, keep / 2)
    empty = [torch.nn.Parameter(torch.zeros(0, 2)) for _ in range(2)]
    for e in empty:
        e.grad = torch.zeros(2, 0).t()
    functional.clip_grad_norm_((p, *empty), 1.0)
