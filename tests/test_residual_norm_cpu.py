"""Host checks of the residual-norm and gradient-norm entry points: what they refuse, before anything reaches a device."""
import ctypes
import math
from array import array

import pytest
import torch

from conversenet_amd import _lib, composite, functional

P = 4096  # an address that no refused call touches


def fwd(x=P, xt=0, h=P, ht=0, B=2, C=8, HW=4, s=None, gate=None, kind=0, pw=None, pb=None, nw=P, nb=P, r=P, y=P):
    return _lib.load().cvn_residual_norm_fwd(x, xt, h, ht, B, C, HW, s, gate, kind, pw, pb, 1e-5, nw, nb, 1e-5, r, y, None,
                                             None)


@pytest.mark.parametrize("kw", [dict(x=None), dict(y=None), dict(r=None), dict(nb=None), dict(h=None, nw=None, nb=None),
                                dict(h=None, s=P), dict(h=None, pw=P, pb=P), dict(gate=P), dict(kind=1), dict(kind=9, gate=P),
                                dict(pw=P), dict(xt=3), dict(ht=-1), dict(xt=1, ht=0), dict(xt=1, ht=2), dict(B=-1),
                                dict(C=0), dict(HW=-1)])
def test_forward_argument_errors(kw):
    assert fwd(**kw) == _lib.CVN_ERR_ARG and _lib.load().cvn_last_error()


def test_forward_limits_and_nothing_to_do():
    assert fwd(C=65537) == _lib.CVN_ERR_UNSUPPORTED
    assert fwd(B=1 << 20, HW=1 << 20) == _lib.CVN_ERR_UNSUPPORTED
    assert fwd(B=1, HW=(1 << 31) - 255) == _lib.CVN_ERR_UNSUPPORTED
    assert fwd(B=0, HW=(1 << 31) - 256) == _lib.CVN_OK
    assert fwd(B=0) == _lib.CVN_OK and fwd(HW=0) == _lib.CVN_OK


def bwd(gr=P, gy=P, base=P, xt=0, h=P, ht=0, B=2, C=8, HW=4, s=None, gate=None, kind=0, pw=None, pb=None, nw=P, stats=P,
        dx=P, dh=P, dg=None, ds=None, dnw=P, dnb=P, dpw=None, dpb=None, ws=P, n=1 << 30):
    return _lib.load().cvn_residual_norm_bwd(gr, gy, base, xt, h, ht, B, C, HW, s, gate, kind, pw, pb, nw, stats, dx, dh, dg,
                                             ds, dnw, dnb, dpw, dpb, ws, n, None)


@pytest.mark.parametrize("kw,rc", [(dict(gr=None, gy=None), -1), (dict(stats=None), -1), (dict(base=None), -1),
                                   (dict(nw=None), -1), (dict(ds=P), -1), (dict(dg=P), -1), (dict(dpw=P), -1),
                                   (dict(gate=P), -1), (dict(xt=2, ht=1), -1), (dict(ws=None), -3), (dict(n=64), -3),
                                   (dict(gy=None), -1), (dict(C=1 << 20), -2), (dict(h=None, s=P), -1),
                                   (dict(xt=5, h=None, dh=None), -1)])
def test_backward_argument_errors(kw, rc):
    assert bwd(**kw) == rc


@pytest.mark.parametrize("t", [1, 2])
def test_backward_of_a_16_bit_branch_needs_it(t):
    """Of 16-bit maps the residual is summed up again, so a gradient of r or of h, which only a branch has, needs h."""
    for kw in (dict(), dict(dh=None), dict(gr=None)):
        assert bwd(xt=t, ht=t, h=None, **kw) == _lib.CVN_ERR_ARG
    g = torch.zeros(2, 8, 4, dtype=(torch.bfloat16, torch.float16)[t - 1])
    w, stats = torch.ones(8), torch.ones(2, 8)
    for gr, gy, h_dtype in ((g, g, None), (g, g, g.dtype), (None, g, g.dtype)):
        with pytest.raises(RuntimeError, match="needs the branch"):
            functional.residual_norm_backward(gr, gy, g, None, stats, w, h_dtype=h_dtype)


def test_backward_workspace():
    q = _lib.load().cvn_residual_norm_bwd_workspace
    assert q(1, 64, 1, 0) > 0 and q(2, 64, 100, 1) > q(2, 64, 100, 0) and q(1, 0, 1, 0) == 0 and q(1, 1 << 20, 1, 0) == 0


def grads(sizes=(4, 8), types=(0, 1), src=(P, 2 * P), dst=None, kind=0, max_norm=1.0, norm=P, ws=P, nb=1 << 20, n=None):
    lib = _lib.load()
    n = len(sizes) if n is None else n
    a, b, t = array("Q", src), array("q", sizes), array("i", types)
    at = lambda v: v.buffer_info()[0]  # noqa: E731
    if dst is None:
        return lib.cvn_grad_norm(at(a), at(b), at(t), n, kind, norm, ws, nb, None)
    d = array("Q", dst)
    return lib.cvn_clip_grads(at(a), at(d), at(b), at(t), n, kind, max_norm, norm, ws, nb, None)


@pytest.mark.parametrize("kw,rc", [(dict(types=(0, 7)), -1), (dict(sizes=(-1, 8)), -1), (dict(src=(0, P)), -1),
                                   (dict(kind=2), -1), (dict(norm=None), -1), (dict(n=-1), -1), (dict(ws=None), -3),
                                   (dict(nb=8), -3), (dict(ws=P + 4), -3), (dict(sizes=(1 << 60, 8)), -1),
                                   (dict(dst=(0, P)), -1), (dict(dst=(P, 2 * P), max_norm=-1.0), -1),
                                   (dict(dst=(P, 2 * P), max_norm=math.nan), -1),
                                   (dict(dst=(3 * P, 3 * P)), -1),               # two outputs in one place
                                   (dict(dst=(2 * P, P)), -1),                   # an output on another's gradient
                                   (dict(dst=(P + 8, 3 * P)), -1),               # an output across its gradient
                                   (dict(src=(P, P), dst=(P, P), types=(1, 1), sizes=(8, 8)), -1),
                                   (dict(src=(P, P + 8), dst=(P, P + 8)), -1)])  # gradients that share memory, in place
def test_gradient_list_errors(kw, rc):
    assert grads(**kw) == rc


def test_gradient_workspace():
    q = _lib.load().cvn_grad_norm_workspace
    one = array("q", [10_000_000])
    assert q(one.buffer_info()[0], 1) >= 8 and q(None, 0) >= 8 and q(None, 3) == 0


def test_cpu_tensors_are_refused():
    x = torch.zeros(1, 8, 2, 2)
    w = torch.ones(8)
    for f in (functional.residual_norm, functional.residual_norm_train):
        with pytest.raises(RuntimeError):
            f(x, x, norm=(w, w, 1e-5))
    with pytest.raises(RuntimeError):
        functional.layernorm_cf_train(x, w, w, 1e-5)
    with pytest.raises(RuntimeError):
        functional.grad_norm([x])
    with pytest.raises(RuntimeError):
        functional.clip_grads([x], 1.0)
    assert float(functional.grad_norm([])) == 0.0


def test_composition_matches_the_definition():
    """composite.residual_branch, standardised and its gradient, which a differentiated backward runs, against the
    formulas."""
    g = torch.Generator().manual_seed(0)
    h, gate = (torch.randn(2, 5, 3, 4, generator=g, dtype=torch.float64) for _ in range(2))
    s, pw, pb = (torch.randn(5, generator=g, dtype=torch.float64) for _ in range(3))
    ref = torch.empty_like(h)
    for b in range(2):
        for i in range(3):
            for j in range(4):
                v = h[b, :, i, j]
                hat = (v - v.mean()) / math.sqrt(((v - v.mean()) ** 2).mean() + 1e-3)
                ref[b, :, i, j] = s * gate[b, :, i, j] * (hat * pw + pb)
    got = composite.residual_branch(h, s, gate, (pw, pb, 1e-3))
    assert torch.allclose(got, ref, rtol=0, atol=1e-13)
    v = h.clone().requires_grad_(True)
    hat, rho = composite.standardised(v, 1e-3)
    want, = torch.autograd.grad(hat, v, gate, create_graph=True)
    assert torch.allclose(composite.standardised_grad(gate, hat, rho), want, rtol=0, atol=1e-12)
    per_sample = torch.randn(2, 5, generator=g, dtype=torch.float64)
    assert torch.equal(composite.residual_branch(h, None, per_sample), h * per_sample[:, :, None, None])
    assert composite.residual_branch(h.float().half()).dtype == torch.float32


def test_tables_live_through_the_call(monkeypatch):
    """The host tables handed to the library are the lists' own while it reads them, whatever is allocated meanwhile."""
    ts = [torch.ones(n) for n in (3, 5, 7)]
    seen = {}

    class Lib:
        def cvn_grad_norm_workspace(self, sizes, n):
            seen["churn"] = [array("Q", [1] * 3) for _ in range(200)]
            return 64

        def _read(self, grads, out, sizes, types, n):
            seen["src"] = list((ctypes.c_uint64 * n).from_address(grads))
            seen["dst"] = list((ctypes.c_uint64 * n).from_address(out))
            seen["sizes"] = list((ctypes.c_int64 * n).from_address(sizes))
            seen["types"] = list((ctypes.c_int * n).from_address(types))
            return 0

        def cvn_grad_norm(self, grads, sizes, types, n, *rest):
            return self._read(grads, grads, sizes, types, n)

        def cvn_clip_grads(self, grads, out, sizes, types, n, *rest):
            return self._read(grads, out, sizes, types, n)

    index = functional._grad_list
    monkeypatch.setattr(torch.Tensor, "get_device", lambda t: 0)
    monkeypatch.setattr(functional._lib, "load", lambda: Lib())
    monkeypatch.setattr(functional, "_stream", lambda dev: 0)
    monkeypatch.setattr(functional, "_on", lambda dev: functional._NO_SWITCH)
    assert index(ts)[0] == 0
    functional.grad_norm(ts)
    want = {"src": [t.data_ptr() for t in ts], "sizes": [3, 5, 7], "types": [0, 0, 0]}
    assert {k: seen[k] for k in want} == want
    out, _ = functional.clip_grads(ts, 1.0)
    assert {k: seen[k] for k in want} == want and seen["dst"] == [t.data_ptr() for t in out]
    functional.release_workspace()
