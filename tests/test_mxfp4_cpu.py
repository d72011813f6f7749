"""The MXFP4 entry points' checks of arguments, without a device, and the oracle's own figures."""
import numpy as np

from conversenet_amd import _lib
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
                dict(xc=D << 12), dict(x=None, xc=D << 12), dict(wc=(D << 20) + 4), dict(y=D), dict(y=D + 1020), dict(y=(D << 20) + 16),
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
