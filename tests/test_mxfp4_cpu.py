"""The MXFP4 entry points' checks of arguments, without a device, the modules on the CPU, and the oracle's own figures."""
import copy

import numpy as np
import pytest
import torch

from conversenet_amd import _lib, composite
from conversenet_amd import functional as F
from conversenet_amd.util_converse import Conv1x1MXFP4, ConverseBlock, ConverseBlockAlphaVariant, use_mxfp4
from oracle import mxfp4_oracle as O

D = 256  # an address that is never used: the checks fail first


def test_oracle_rounds_to_the_nearest_and_even():
    """Against the nearest of all 16 values, found by distance; on a tie the code whose lowest bit is zero."""
    rng = np.random.default_rng(0)
    x = np.concatenate((rng.standard_normal((50, 32)) * 3, rng.choice(np.concatenate((O.MIDS, O.GRID)), (50, 32)) *
                        rng.choice((-1, 1), (50, 32)))).astype(np.float32).astype(np.float64)
    x = np.clip(x, -7.9, 7.9)
    x[:, 0] = 7.0  # the scale is 1
    codes, scales = O.quantize(x[:, :, None])
    assert (scales == 127).all()
    got = np.stack((codes & 15, codes >> 4), -1).reshape(100, 32)
    for v, c in zip(x.ravel(), got.ravel()):
        d = np.abs(O.GRID - abs(v))
        near = np.flatnonzero(d == d.min())
        assert (c & 7) in near and (len(near) == 1 or (c & 1) == 0), (v, c)
        assert (c >= 8) == np.signbit(v)


def test_oracle_scales():
    x = np.zeros((1, 64, 4))
    x[0, 0], x[0, 40] = [1.0, 0.99, 2.0 ** -149, 3.3e38], [0.0, np.inf, 2.0 ** -124, np.nan]
    _, s = O.quantize(x)
    assert s[0].tolist() == [[125, 0], [124, 255], [0, 1], [252, 255]]
    v = O.rounded(x)
    assert v[0, 0, 0] == 1.0 and np.isnan(v[0, 32:, 1]).all() and (v[0, :32, 1] < 1.01).all()


def test_arguments():
    lib = _lib.load()
    A, U, W = _lib.CVN_ERR_ARG, _lib.CVN_ERR_UNSUPPORTED, _lib.CVN_ERR_WORKSPACE
    q, d, f, g = lib.cvn_mxfp4_quantize, lib.cvn_mxfp4_dequantize, lib.cvn_conv1x1_mxfp4, lib.cvn_conv1x1_mxfp4_bwd
    assert q(None, 0, 1, 32, 4, None, None, None) == A and b"null" in lib.cvn_last_error()
    assert q(D, 3, 1, 32, 4, D, D, None) == A and q(D, 0, 1, 0, 4, D, D, None) == A and q(D, 0, -1, 32, 4, D, D, None) == A
    assert q(D, 0, 1, 32, 4, D + 8, D, None) == A and b"aligned" in lib.cvn_last_error()
    assert q(D, 0, 1, 65537, 4, D, D, None) == U and q(D, 0, 1 << 20, 32, 1 << 12, D, D, None) == U
    assert q(None, 0, 0, 32, 4, None, None, None) == d(None, None, 3, 32, 0, None, 0, None) == _lib.CVN_OK
    assert d(None, None, 1, 32, 4, None, 0, None) == A and d(D, D, 1, 32, 4, D, 7, None) == A

    def conv(x=D, xc=None, xs=None, B=1, C=64, HW=4, w=None, wt=0, wc=D << 20, ws=D << 24, N=8, act=0, res=None, y=D << 30, type=0,
             wsp=D << 10, wsb=1 << 20):
        return f(x, xc, xs, B, C, HW, w, wt, wc, ws, N, None, act, res, None, y, type, wsp, wsb, None)

    assert conv(B=0) == _lib.CVN_OK
    for bad in (dict(x=None), dict(wc=None), dict(ws=None), dict(y=None), dict(act=2), dict(type=3), dict(N=0), dict(C=0),
                dict(xc=D << 12), dict(x=None, xc=D << 12), dict(wc=(D << 20) + 4), dict(y=D), dict(y=D + 1020),
                dict(y=(D << 20) + 16),
                dict(res=(D << 30) + 4), dict(wc=None, ws=None), dict(w=D << 28, wt=3), dict(w=D << 28, wc=D << 28),
                dict(w=D << 28, wc=D, ws=D << 24), dict(xc=D << 12, xs=D << 12), dict(xc=D << 20, xs=D << 13)):
        assert conv(**bad) == A, bad
    assert conv(N=65537) == conv(C=65537) == conv(B=1 << 16, HW=1 << 16) == U
    need = lib.cvn_conv1x1_mxfp4_workspace(0, 1, 1, 64, 4, 8)
    assert need >= 4 * 2 * 17 and lib.cvn_conv1x1_mxfp4_workspace(0, 1, 1, 0, 4, 8) == 0
    assert lib.cvn_conv1x1_mxfp4_workspace(0, 0, 1, 64, 4, 8) >= need + 8 * 2 * 17
    assert conv(wsb=need - 1) == conv(wsp=None) == conv(wsp=(D << 10) + 8) == W
    assert conv(w=D << 28, wc=None, ws=None, wsb=need) == W

    def bwd(gy=D, xc=D << 20, xs=D << 21, wc=D << 22, ws=D << 23, B=1, C=64, HW=4, N=8, type=0, gx=D << 24, gw=D << 25, gb=None):
        return g(gy, type, xc, xs, wc, ws, B, C, HW, N, gx, gw, gb, D << 26, 1 << 24, None)

    assert bwd(gx=None, gw=None) == _lib.CVN_OK and bwd(B=-1) == A
    for bad in (dict(gy=None), dict(xc=None), dict(xs=None), dict(wc=None), dict(ws=None), dict(type=5), dict(C=0), dict(N=0),
                dict(HW=-1), dict(wc=(D << 22) + 8), dict(xc=(D << 20) + 1)):
        assert bwd(**bad) == A, bad
    assert bwd(C=65537) == bwd(N=65537) == bwd(B=1 << 16, HW=1 << 16) == U


def test_device_tensors_are_needed():
    x, w = torch.zeros(1, 32, 2, 2), torch.zeros(4, 32)
    q = F.MXFP4(torch.zeros(1, 2, 2, 16, dtype=torch.uint8), torch.zeros(1, 2, 2, 1, dtype=torch.uint8), 32)
    assert q.shape == (1, 32, 2, 2)
    for call in (lambda: F.quantize_mxfp4(x), lambda: F.dequantize_mxfp4(q), lambda: F.conv1x1_mxfp4(x, w),
                 lambda: F.conv1x1_mxfp4(q, w), lambda: F.conv1x1_mxfp4_train(x.requires_grad_(), w),
                 lambda: F.conv1x1_mxfp4_backward(x, q, None)):
        with pytest.raises(RuntimeError, match="HIP device"):
            call()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(2, 70, 3, 5), (4, 32), (1, 1, 1), (3, 100, 2)])
def test_composite_values(shape, dtype):
    g = torch.Generator().manual_seed(len(shape))
    x = (torch.randn(shape, generator=g) * 10 ** torch.randn(shape, generator=g)).to(dtype)
    flat = x.double().numpy().reshape(shape[0], shape[1], -1)
    got = composite.mxfp4_values(x)
    assert got.dtype is dtype and got.shape == x.shape
    # (rounded to x's type: fp16 keeps no value below half its smallest number)
    assert np.array_equal(got.double().numpy().reshape(flat.shape), torch.from_numpy(O.rounded(flat)).to(dtype).double().numpy())
    x[0, 0] = float("inf")
    assert torch.isnan(composite.mxfp4_values(x)[0, :min(32, shape[1])]).all()


def test_convolution_on_the_cpu():
    """Float64 as the oracle, with its gradients; parameters shared with the convolution it was made of."""
    conv = torch.nn.Conv2d(40, 9, 1).double()
    mx = Conv1x1MXFP4.of(conv)
    assert mx.weight is conv.weight and mx.bias is conv.bias and list(mx.state_dict()) == list(conv.state_dict())
    x = torch.randn(2, 40, 3, 4, dtype=torch.float64, requires_grad=True)
    gy = torch.randn(2, 9, 3, 4, dtype=torch.float64)
    y = mx(x)
    grads = torch.autograd.grad(y, (x, mx.weight, mx.bias), gy)
    n = lambda t: t.detach().numpy().reshape(t.shape[0], t.shape[1], -1)  # noqa: E731
    xq, wq = O.rounded(n(x)), O.rounded(n(conv.weight))[:, :, 0]
    want, mag = O.conv1x1(xq, wq, conv.bias.detach().numpy())
    assert (np.abs(n(y) - want) <= 42 * 2.0 ** -52 * mag).all()
    for g, (want, mag), terms in zip(grads, O.gradients(n(gy), xq, wq), (9, 24, 24)):
        assert (np.abs(g.numpy().reshape(want.shape) - want) <= (terms + 2) * 2.0 ** -52 * mag).all()
    assert torch.equal(mx(x[0]), mx(x[:1])[0])
    for bad in (torch.nn.Conv2d(4, 4, 3), torch.nn.Conv2d(4, 4, 1, stride=2), torch.nn.Conv2d(4, 4, 1, groups=2)):
        with pytest.raises(ValueError):
            Conv1x1MXFP4.of(bad)


@pytest.mark.parametrize("cls", [ConverseBlock, ConverseBlockAlphaVariant])
def test_block_on_the_cpu(cls):
    torch.manual_seed(0)
    blk = cls(8, 8, kernel_size=3, padding=2, padding_mode="circular")
    if cls is ConverseBlockAlphaVariant:
        torch.nn.init.normal_(blk.alpha1), torch.nn.init.normal_(blk.alpha2)
    keys, plain = list(blk.state_dict()), copy.deepcopy(blk)
    assert use_mxfp4(blk) is blk and list(blk.state_dict()) == keys
    kinds = [type(m) for m in (blk.conv1[1], blk.conv1[5], blk.conv2[1], blk.conv2[3])]
    assert kinds == [Conv1x1MXFP4] * 4
    x = torch.randn(2, 8, 6, 7)
    y = blk(x)
    t = x
    for seq, alpha in ((plain.conv1, getattr(plain, "alpha1", 1)), (plain.conv2, getattr(plain, "alpha2", 1))):
        v = t
        for m in seq:
            v = composite.conv1x1_mxfp4(v, m.weight, m.bias) if type(m) is torch.nn.Conv2d else m(v)
        t = alpha * v + t
    assert torch.equal(y, t)
    y.square().sum().backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in blk.parameters())
    blk.load_state_dict(plain.state_dict(), strict=True)


def test_evaluation_flag(tmp_path, capsys):
    from PIL import Image

    from conversenet_amd import evaluate as E
    rng = np.random.default_rng(0)
    Image.fromarray(rng.integers(0, 255, (16, 20), dtype=np.uint8)).save(tmp_path / "a.png")
    lines = []
    for flags in ([], ["--mxfp4"]):
        torch.manual_seed(0)
        E.main(["dncnn", "--testset", str(tmp_path), *flags])
        lines.append(capsys.readouterr().out)
    assert all("Average PSNR" in t for t in lines) and lines[0] != lines[1]


def test_leaves_of_other_graphs_are_found():
    x, w = torch.randn(3, requires_grad=True), torch.randn(3, requires_grad=True)
    F._own_leaves([x, w], 5)
    y = x * 2
    for _ in range(2):
        with pytest.raises(RuntimeError, match="holds one of its leaves"):
            F._own_leaves([w, x], 5)
    F._accumulator(x).metadata[F._RECORDING] = 5  # made in the recording on stream 5
    F._own_leaves([x, w], 5)
    with pytest.raises(RuntimeError, match="holds one of its leaves"):
        F._own_leaves([x], 6)
    del y
    F._own_leaves([x, w], 6)


def test_views_of_leaves_of_other_graphs_are_found():
    """An operand that is a view (or another result) of a leaf is refused as the leaf itself is."""
    w, x = torch.randn(6, 4, requires_grad=True), torch.randn(3, 4)
    F._own_operands([w], 5)
    alive = w * 2
    for v in (w.view(6, 4, 1, 1), w.flatten(), w.unsqueeze(0), w * 1.0, (w * 1.0).exp().view(4, 6)):
        with pytest.raises(RuntimeError, match="outside of the recording"):
            F._own_operands([v], 5)
    with pytest.raises(RuntimeError, match="holds one of its leaves"):
        F._own_operands([w], 5)
    del alive, v
    F._own_operands([w], 5)
    F._own_operands([t for t in (x, w) if t.requires_grad], 5)


def test_graphs_are_walked():
    """Every node behind a tensor is looked at, each once; a tensor without a graph has none."""
    from conversenet_amd import _lib
    w, x = torch.randn(4, requires_grad=True), torch.randn(4)
    assert _lib.graph_streams(w) == [] and _lib.graph_streams(x) == []
    y = w
    for _ in range(200):  # 2^200 paths, 200 nodes
        y = y + y
    assert _lib.graph_streams(y) == [(-1, 0)] == _lib.graph_streams(w)
    with torch.no_grad():
        assert _lib.graph_streams(y.detach()) == []
    del y
    assert _lib.graph_streams(w) == []
    with pytest.raises(RuntimeError, match="not a tensor"):
        _lib.graph_streams(None)


def test_use_mxfp4_keeps_what_convolutions_carry():
    """Hooks, weights made in hooks, shared convolutions and the state dict; all or nothing."""
    torch.manual_seed(0)
    blk = ConverseBlock(8, 8, kernel_size=3, padding=2, padding_mode="circular")
    x = torch.randn(2, 8, 6, 7)
    seen, conv = [], blk.conv2[3]
    handle = conv.register_forward_hook(lambda m, args, out: seen.append(out))
    with pytest.warns(FutureWarning):
        torch.nn.utils.weight_norm(blk.conv1[1])
    blk.conv2.append(conv), blk.conv2.insert(3, torch.nn.Conv2d(16, 16, 1, padding="same"))
    blk.conv2[5] = torch.nn.Conv2d(8, 8, 1, padding="valid")
    keys = list(blk.state_dict())
    assert use_mxfp4(blk) is blk and list(blk.state_dict()) == keys and blk.conv2[4] is conv
    assert all(type(blk.conv1[i]) is Conv1x1MXFP4 for i in (1, 5)) and all(type(blk.conv2[i]) is Conv1x1MXFP4 for i in (1, 3, 4, 5))
    with torch.no_grad():
        blk.conv1[1].weight_g.mul_(3.0)
        n = blk.conv1[0](x)
        w = torch._weight_norm(blk.conv1[1].weight_v, blk.conv1[1].weight_g, 0)
        assert torch.equal(blk.conv1[1](n), composite.conv1x1_mxfp4(n, w, blk.conv1[1].bias))
        blk(x)
    assert len(seen) == 1
    handle.remove()
    blk(x).sum().backward()
    assert len(seen) == 1 and blk.conv1[1].weight_g.grad is not None and blk.conv1[1].weight_v.grad is not None

    for spoil in (lambda c: setattr(c, "forward", c.forward), lambda c: setattr(c, "stride", (2, 2)), lambda c: c.compile()):
        blk = ConverseBlockAlphaVariant(8, 8, kernel_size=3, padding=2, padding_mode="circular")
        spoil(blk.conv2[3])
        with pytest.raises(ValueError):
            use_mxfp4(blk)
        assert all(type(m) is not Conv1x1MXFP4 for m in blk.modules())


def test_convolutions_that_would_lose_something_are_refused():
    c = lambda: torch.nn.Conv2d(4, 6, 1)  # noqa: E731
    hooked, pre, late = c(), c(), c()
    hooked.register_forward_hook(lambda *a: None), pre.register_forward_pre_hook(lambda *a: None)
    late.register_full_backward_hook(lambda *a: None)
    with pytest.warns(FutureWarning):
        normed = torch.nn.utils.weight_norm(c())
    bad = [hooked, pre, late, normed, torch.nn.utils.parametrizations.weight_norm(c()), torch.nn.utils.spectral_norm(c())]
    buffer, child = c(), c()
    buffer.register_buffer("mask", torch.ones(1)), child.add_module("extra", torch.nn.Identity())
    for conv in (*bad, buffer, child):
        with pytest.raises(ValueError):
            Conv1x1MXFP4.of(conv)
    assert Conv1x1MXFP4.of(torch.nn.Conv2d(4, 6, 1, padding="same", bias=False)).bias is None


def test_hooks_see_a_single_sample_once():
    conv = Conv1x1MXFP4(8, 4)
    seen = []
    conv.register_forward_pre_hook(lambda m, args: seen.append(args[0].shape))
    conv.register_forward_hook(lambda m, args, out: seen.append(out.shape))
    conv(torch.randn(8, 3, 5))
    assert seen == [(8, 3, 5), (4, 3, 5)]


def test_blocks_whose_modules_are_observed_run_them():
    """The joint forward of a block is for plain modules."""
    from conversenet_amd import util_converse as U
    make = lambda: use_mxfp4(ConverseBlock(8, 8, kernel_size=3, padding=2, padding_mode="circular"))  # noqa: E731
    assert U._all_mxfp4(make())
    for i in (0, 1, 2, 3, 4, 5):
        blk = make()
        handle = blk.conv1[i].register_forward_hook(lambda *a: None)
        assert not U._all_mxfp4(blk)
        handle.remove()
        assert U._all_mxfp4(blk)
    blk = make()
    blk.conv2[3].register_forward_pre_hook(lambda *a: None)
    assert not U._all_mxfp4(blk)
    for i, m in ((2, torch.nn.ReLU()), (4, torch.nn.GELU("tanh")), (1, torch.nn.Conv2d(8, 16, 1))):
        blk = make()
        blk.conv1[i] = m
        assert not U._all_mxfp4(blk)
    blk = make()
    with pytest.warns(FutureWarning):
        torch.nn.utils.weight_norm(blk.conv2[1])
    assert not U._all_mxfp4(blk)


@pytest.mark.parametrize("cast", [torch.bfloat16, torch.float16])
def test_autocast_changes_nothing_on_the_cpu(cast):
    conv = Conv1x1MXFP4(40, 8)
    x = torch.randn(2, 40, 5, 6)
    y = conv(x)
    with torch.autocast("cpu", dtype=cast):
        z = conv(x)
        assert torch.is_autocast_enabled("cpu")
    assert z.dtype is torch.float32 and torch.equal(y, z)


@pytest.mark.parametrize("tx", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tw", [torch.float32, torch.bfloat16, torch.float16])
def test_types_of_a_convolution_on_the_cpu(tx, tw):
    """Parameters of another type than the input: the result has the input's, and gradients are of the parameters'."""
    conv = Conv1x1MXFP4(40, 8).to(tw)
    x = torch.randn(2, 40, 5, 6).to(tx).requires_grad_()
    y = conv(x)
    n = lambda t: t.detach().double().numpy().reshape(t.shape[0], t.shape[1], -1)  # noqa: E731
    want, mag = O.conv1x1(O.rounded(n(x)), O.rounded(n(conv.weight))[:, :, 0], conv.bias.detach().double().numpy())
    # sums of 41 terms in float32, then the rounding of a result of x's type (fp16: also of numbers below its smallest normal one)
    lim = 43 * 2.0 ** -24 * mag + torch.finfo(tx).eps / 2 * np.abs(want) + 2.0 ** -25
    assert y.dtype is tx and (np.abs(n(y) - want) <= lim).all()
    y.float().sum().backward()
    assert x.grad.dtype is tx and conv.weight.grad.dtype is tw and conv.bias.grad.dtype is tw


def test_tensors_without_memory_are_no_operands():
    class Holder(torch.Tensor):
        @classmethod
        def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
            raise NotImplementedError

    held = torch.Tensor._make_wrapper_subclass(Holder, (3, 4))
    with pytest.raises(RuntimeError, match="no memory"):
        F._values(held)
    with pytest.raises(RuntimeError, match="no memory"):
        F._param32([], held, 12, -1, "bias")
    assert F._values(torch.empty(0, 4)).numel() == 0 and F._values(None) is None


def test_only_convolutions_become_mxfp4_ones():
    class Own(torch.nn.Conv2d):
        def forward(self, x):
            return 2 * super().forward(x)

    class Plain(torch.nn.Conv2d):
        pass

    for m in (torch.nn.ConvTranspose2d(4, 4, 1), Own(4, 6, 1), torch.nn.Linear(4, 6)):
        with pytest.raises(ValueError):
            Conv1x1MXFP4.of(m)
    assert Conv1x1MXFP4.of(Plain(4, 6, 1)).out_channels == Conv1x1MXFP4.of(Conv1x1MXFP4(4, 6)).out_channels == 6


def test_outputs_that_share_memory_are_refused():
    """By the C entry points, whose callers choose every address; a byte beside is another matter for the device to run."""
    lib = _lib.load()

    def refused(rc):
        return rc == _lib.CVN_ERR_ARG and b"shares memory" in lib.cvn_last_error()

    # 64 channels of 4 pixels: 1024 bytes of float32, 128 of codes, 8 of scales
    x, codes, scales = D << 20, D << 21, D << 22
    q, d, g = lib.cvn_mxfp4_quantize, lib.cvn_mxfp4_dequantize, lib.cvn_conv1x1_mxfp4_bwd
    for c, s in ((x, scales), (x + 1008, scales), (x - 112, scales), (codes, x + 1023), (codes, x - 7), (codes, codes + 127),
                 (codes, codes - 7)):
        assert refused(q(x, 0, 1, 64, 4, c, s, None)), (c, s)
    for y in (codes, codes + 112, codes - 1020, scales + 4, scales - 1020):
        assert refused(d(codes, scales, 1, 64, 4, y, 0, None)), y
    # and to 8 channels: grad_y 128 bytes, the matrix 256 of codes and 16 of scales, its gradient 2048, the bias' 32
    gy, wc, ws, gx, gw, gb = D << 23, D << 24, D << 25, D << 26, D << 27, D << 28

    def bwd(gx=gx, gw=gw, gb=gb):
        return g(gy, 0, codes, scales, wc, ws, 1, 64, 4, 8, gx, gw, gb, D << 29, 1 << 24, None)

    for bad in (dict(gx=gy), dict(gx=gy - 1020), dict(gx=wc + 240), dict(gx=ws), dict(gx=codes), dict(gx=scales), dict(gx=gw + 2044),
                dict(gx=gb), dict(gw=gy), dict(gw=codes), dict(gw=scales - 2044), dict(gw=wc), dict(gw=gb + 28), dict(gb=gy + 124),
                dict(gb=gw - 28), dict(gb=gx + 1020), dict(gx=gy, gw=None, gb=None), dict(gx=None, gb=None, gw=codes + 124)):
        assert refused(bwd(**bad)), bad
