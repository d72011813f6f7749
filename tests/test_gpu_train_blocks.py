"""Blocks under autograd on the library's norm and residual kernels, against the same modules in 64 bits on the CPU (the
composition), and what must go on seeing the composition: hooks, function transforms, other layouts.

Tolerances of whole blocks, relative to the norm of the reference: every layer of a block (8) is off by at most 1e-5 of
its values (a 1 x 1 convolution of 128 channels 128 * 2^-24; Converse2D 1e-5, which its own tests bound; a norm
(64 + 32) 2^-24 times the spread of its values), forward and backward, so a chain of n blocks stays below 16 n * 1e-5."""
import copy

import pytest
import torch
import torch.nn as nn

from conversenet_amd import functional as Fh
from conversenet_amd import util_converse as U

pytestmark = pytest.mark.gpu


def _fill(m, seed=0):
    g = torch.Generator().manual_seed(seed)
    with torch.no_grad():
        for name, p in m.named_parameters():
            r = torch.randn(p.shape, generator=g)
            if p.dim() == 4 and p.shape[0] == 1 and p.shape[-1] > 1:
                p.copy_(torch.softmax(r.flatten(2), -1).view(p.shape))
            elif "alpha" in name:
                p.copy_(0.3 * r)
            elif p.dim() == 4:
                p.copy_(r / p[0].numel() ** 0.5)
            elif name.endswith("weight"):
                p.copy_(1 + 0.1 * r)
            else:
                p.copy_(0.1 * r)
    return m


class Count:
    """Calls of the library's norm kernels, forward."""

    def __init__(self, monkeypatch):
        self.n = 0
        inner = Fh._residual_norm

        def counted(*a, **k):
            self.n += 1
            return inner(*a, **k)

        monkeypatch.setattr(Fh, "_residual_norm", counted)


def _run(m, x, go):
    x = x.clone().requires_grad_(True)
    y = m(x)
    grads = torch.autograd.grad(y, [x, *m.parameters()], go)
    return [y.detach(), *grads]


def _close(got, ref, tol, what=""):
    for i, (g, r) in enumerate(zip(got, ref)):
        g, r = g.detach(), r.detach().double().cpu()
        err = float((g.double().cpu() - r).norm())
        assert err <= tol * float(r.norm()) + 1e-12, (what, i, err, float(r.norm()))


def _inputs(shape, seed=1):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g), torch.randn(shape, generator=g)


@pytest.mark.parametrize("shape", [(2, 64, 24, 20), (1, 5, 9, 7), (2, 300, 8, 8), (1, 64, 1, 1)])
def test_layernorm_module(shape, monkeypatch):
    count = Count(monkeypatch)
    m = _fill(U.LayerNorm(shape[1], eps=1e-6, data_format="channels_first"))
    x, go = _inputs(shape)
    ref = _run(copy.deepcopy(m).double(), x.double(), go.double())
    got = _run(m.cuda(), x.cuda(), go.cuda())
    assert count.n == 1
    _close(got, ref, 1e-5)


@pytest.mark.parametrize("cls,C,hw", [(U.ConverseBlock, 64, (24, 24)), (U.ConverseBlockAlphaVariant, 64, (17, 21)),
                                      (U.ConverseBlockAlphaVariant, 32, (12, 40)), (U.ConverseBlock, 20, (11, 13))])
def test_block(cls, C, hw, monkeypatch):
    count = Count(monkeypatch)
    m = _fill(cls(C, C, kernel_size=5, padding=2, padding_mode="circular"))
    x, go = _inputs((2, C, *hw))
    ref = _run(copy.deepcopy(m).double(), x.double(), go.double())
    got = _run(m.cuda(), x.cuda(), go.cuda())
    assert count.n == (3 if cls is U.ConverseBlockAlphaVariant else 2)
    _close(got, ref, 1.6e-4, cls.__name__)


def test_chain_fuses_across_blocks(monkeypatch):
    from conversenet_amd.converse_usrnet import MultiConverseBlock, MultiConverseBlockAlphaVariant

    for cls, calls in ((MultiConverseBlock, 6), (MultiConverseBlockAlphaVariant, 7)):
        m = _fill(cls(32, num_blocks=3, kernel_size=3, padding=1))
        x, go = _inputs((2, 32, 18, 22))
        ref = _run(copy.deepcopy(m).double(), x.double(), go.double())
        m.cuda()
        with monkeypatch.context() as mp:
            count = Count(mp)
            got = _run(m, x.cuda(), go.cuda())
            assert count.n == calls  # the first norm, two residuals a block, the last without a norm only when scaled
        _close(got, ref, 4.8e-4, cls.__name__)


def test_denoiser_trains(monkeypatch):
    from conversenet_amd.converse_dncnn import ConverseDnCNN

    net = _fill(ConverseDnCNN()).cuda()
    x = torch.rand(1, 1, 20, 24, device="cuda")
    with torch.no_grad():
        want = net(x)
    count = Count(monkeypatch)
    y = net(x)
    assert count.n == 40
    assert float((y.detach() - want).abs().max()) <= 1e-3 * float(want.abs().max())  # 20 blocks, two sets of kernels
    y.sum().backward()
    assert all(torch.isfinite(p.grad).all() for p in net.parameters())


def test_training_steps_with_clipping():
    """Forward, backward, clipping and a step, three times, as the same in 64 bits."""
    from conversenet_amd.converse_usrnet import MultiConverseBlockAlphaVariant

    m = _fill(MultiConverseBlockAlphaVariant(32, num_blocks=2, kernel_size=3, padding=1))
    ref = copy.deepcopy(m).double()
    m.cuda()
    opts = [torch.optim.SGD(n.parameters(), lr=0.05) for n in (m, ref)]
    for step in range(3):
        x, t = _inputs((2, 32, 16, 16), seed=step)
        loss = ((m(x.cuda()) - t.cuda()) ** 2).mean()
        opts[0].zero_grad()
        loss.backward()
        norm = Fh.clip_grad_norm_(m.parameters(), 0.1)
        opts[0].step()
        loss64 = ((ref(x.double()) - t.double()) ** 2).mean()
        opts[1].zero_grad()
        loss64.backward()
        norm64 = torch.nn.utils.clip_grad_norm_(ref.parameters(), 0.1)
        opts[1].step()
        assert abs(float(norm) - float(norm64)) <= 1e-3 * float(norm64)
        assert float(norm64) > 0.1
    for p, q in zip(m.parameters(), ref.parameters()):
        # three steps of at most 0.05 * 0.1, each off by 3.2e-4 of itself
        assert float((p.detach().double().cpu() - q.detach()).norm()) <= 3 * 0.005 * 1e-3 + 1e-6 * float(q.detach().norm())


def test_hooks_see_their_modules(monkeypatch):
    m = _fill(U.ConverseBlockAlphaVariant(32, 32, kernel_size=3, padding=1, padding_mode="circular")).cuda()
    x, go = (t.cuda() for t in _inputs((1, 32, 12, 12)))
    want = _run(m, x, go)
    for mod in (m.conv1, m.conv2, m.conv1[0], m.conv2[0]):
        seen = []
        h = mod.register_forward_hook(lambda mod, i, o: seen.append(o.shape))
        got = _run(m, x, go)
        h.remove()
        assert len(seen) == 1
        _close(got, want, 1e-4)
    h = m.conv2[0].register_forward_hook(lambda mod, i, o: o * 0)  # a hook that changes the output
    changed = _run(m, x, go)
    h.remove()
    assert float((changed[0] - want[0]).abs().max()) > 1e-3
    count = Count(monkeypatch)
    seen = []
    h = nn.modules.module.register_module_forward_hook(lambda mod, i, o: seen.append(type(mod).__name__))
    _run(m, x, go)
    h.remove()
    assert seen.count("LayerNorm") == 2 and seen.count("Sequential") == 2


def test_chain_calls_hooked_blocks():
    from conversenet_amd.converse_usrnet import MultiConverseBlock

    m = _fill(MultiConverseBlock(32, num_blocks=2, kernel_size=3, padding=1)).cuda()
    x, go = (t.cuda() for t in _inputs((1, 32, 12, 12)))
    want = _run(m, x, go)
    seen = []
    m.m_body[1].register_forward_hook(lambda mod, i, o: seen.append(o.shape))
    _close(_run(m, x, go), want, 1e-4)
    assert len(seen) == 1


def test_function_transforms():
    m = _fill(U.LayerNorm(16, eps=1e-6, data_format="channels_first")).cuda()
    x, t = (v.cuda() for v in _inputs((3, 16, 6, 5)))
    params = {k: v.detach() for k, v in m.named_parameters()}

    def loss(p, x):
        return (torch.func.functional_call(m, p, (x,)) ** 3).sum()

    got = torch.func.grad(loss)(params, x)
    y = (m(x) ** 3).sum()
    want = torch.autograd.grad(y, list(m.parameters()))
    _close(list(got.values()), want, 1e-5)
    per = torch.func.vmap(torch.func.grad(loss), in_dims=(None, 0))(params, x[:, None])
    _close([per["weight"].sum(0)], [want[0]], 1e-5)
    _, tangent = torch.func.jvp(m, (x,), (t,))
    ref = torch.autograd.functional.jvp(copy.deepcopy(m).cpu().double(), x.cpu().double(), t.cpu().double())[1]
    _close([tangent], [ref], 1e-5)


def test_gradient_penalty():
    m = _fill(U.LayerNorm(24, eps=1e-6, data_format="channels_first"))
    x, go = _inputs((2, 24, 7, 5))

    def penalty(m, x, go):
        x = x.clone().requires_grad_(True)
        gx, = torch.autograd.grad(m(x), x, go, create_graph=True)
        return torch.autograd.grad((gx ** 2).sum(), [x, m.weight])

    ref = penalty(copy.deepcopy(m).double(), x.double(), go.double())
    _close(penalty(m.cuda(), x.cuda(), go.cuda()), ref, 1e-4)


def test_other_calls_keep_the_composition(monkeypatch):
    count = Count(monkeypatch)
    m = _fill(U.LayerNorm(16, eps=1e-6, data_format="channels_first")).cuda()
    x = torch.randn(2, 16, 6, 6, device="cuda")
    y = m(x.to(memory_format=torch.channels_last))
    assert y.is_contiguous(memory_format=torch.channels_last)
    m(x.double().float()[:, :, ::2])
    assert m(x.half()).dtype is torch.float32  # promoted by the float32 weight
    one = U.LayerNorm(1, data_format="channels_first").cuda()
    assert one(x).shape == x.shape  # one weight for all channels
    assert count.n == 0
    m(x)
    assert count.n == 1
    monkeypatch.setenv("CONVERSE2D_BACKEND", "pytorch")
    blk = _fill(U.ConverseBlock(16, 16, kernel_size=3, padding=1, padding_mode="circular")).cuda()
    assert not U._trainable(blk, x)
    monkeypatch.delenv("CONVERSE2D_BACKEND")
    assert U._trainable(blk, x)
    monkeypatch.setattr(torch.compiler, "is_compiling", lambda: True)
    assert not U._trainable(blk, x)


def test_checkpoint_and_inplace_after():
    from torch.utils.checkpoint import checkpoint

    m = _fill(U.ConverseBlockAlphaVariant(32, 32, kernel_size=3, padding=1, padding_mode="circular")).cuda()
    x, go = (t.cuda() for t in _inputs((1, 32, 12, 12)))
    want = _run(m, x, go)

    class Wrapped(nn.Module):
        def __init__(self):
            super().__init__()
            self.m = m

        def forward(self, x):
            return checkpoint(self.m, x, use_reentrant=False)

    _close(_run(Wrapped(), x, go), want, 1e-6)

    class Inplace(Wrapped):
        def forward(self, x):
            return self.m(x).mul_(2.0).add_(1.0)  # on the block's own output

    got = _run(Inplace(), x, go)
    _close(got[1:], [2 * w for w in want[1:]], 1e-6)


def test_a_norms_own_forward_is_called():
    m = _fill(U.ConverseBlockAlphaVariant(32, 32, kernel_size=3, padding=1, padding_mode="circular")).cuda()
    x, go = (t.cuda() for t in _inputs((1, 32, 12, 12)))
    want = _run(m, x, go)
    inner = m.conv2[0].forward
    m.conv2[0].forward = lambda v: inner(v)
    _close(_run(m, x, go), want, 1e-4)
    m.conv2[0].forward = lambda v: 2 * inner(v)
    twice = _run(m, x, go)
    del m.conv2[0].forward
    m.conv2[0].register_forward_hook(lambda mod, i, o: 2 * o)
    _close(twice, _run(m, x, go), 1e-4)
    assert float((twice[0] - want[0]).abs().max()) > 1e-3


@pytest.mark.parametrize("second", [False, True])
def test_input_changed_in_place_behind_a_module(second):
    """x += block(x), and the like: the backward has the values that the module had, as the composition's."""
    for m in (_fill(U.LayerNorm(24, eps=1e-6, data_format="channels_first")),
              _fill(U.ConverseBlockAlphaVariant(24, 24, kernel_size=3, padding=1, padding_mode="circular"))):
        x, go = _inputs((2, 24, 9, 11))

        def run(m, x, go, change):
            x = x.clone().requires_grad_(True)
            z = x * 1.5
            y = m(z)
            if change:
                z.add_(y)
            else:
                z = z + y
            if not second:
                return torch.autograd.grad(z, [x, *m.parameters()], go)
            gx, = torch.autograd.grad(z, x, go, create_graph=True)
            return torch.autograd.grad((gx ** 2).sum(), x)

        ref = run(copy.deepcopy(m).double(), x.double(), go.double(), False)
        if type(m) is U.LayerNorm or not second:  # (Converse2D's backward is not differentiable)
            _close(run(m.cuda(), x.cuda(), go.cuda(), True), ref, 1.6e-4, type(m).__name__)


@pytest.mark.parametrize("unpack", [lambda t: t.to(memory_format=torch.channels_last) if t.dim() == 4 else t,
                                    lambda t: torch.stack([t, t * 0], -1)[..., 0]])
def test_saved_tensors_with_other_strides(unpack):
    """Saved-tensor hooks that keep values, sizes and types, but not strides."""
    for m, tol in ((_fill(U.LayerNorm(24, eps=1e-6, data_format="channels_first")), 1e-5),
                   (_fill(U.ConverseBlockAlphaVariant(24, 24, kernel_size=3, padding=1, padding_mode="circular")), 1.6e-4)):
        x, go = _inputs((2, 24, 9, 11))
        ref = _run(copy.deepcopy(m).double(), x.double(), go.double())
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach(), unpack):
            got = _run(m.cuda(), x.cuda(), go.cuda())
        _close(got, ref, tol, type(m).__name__)
    with torch.autograd.graph.save_on_cpu():
        _close(_run(m, x.cuda(), go.cuda()), ref, tol)


def test_traced_on_the_device():
    from torch.fx.experimental.proxy_tensor import make_fx

    m = _fill(U.LayerNorm(16, eps=1e-6, data_format="channels_first")).cuda()

    def step(x, go):
        y = m(x)
        return (y, *torch.autograd.grad(y, (x, m.weight), go))

    x, go = (t.cuda() for t in _inputs((1, 16, 5, 6)))
    graph = make_fx(step)(x.clone().requires_grad_(True), go)
    x, go = (t.cuda() for t in _inputs((1, 16, 5, 6), seed=9))
    x.requires_grad_(True)
    _close(graph(x, go), [t.detach() for t in step(x, go)], 1e-5)
