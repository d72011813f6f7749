"""MXFP4 quantisation and the 1x1 convolution of MXFP4 operands with its gradients, in numpy and 64 bits.

A map is (B,C,P), a matrix (N,C) a map of one pixel.  Codes and scales are laid out by pixels: (B,P,16 blocks) and
(B,P,blocks) bytes, blocks of 32 channels."""
import math

import numpy as np

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
MIDS = (GRID[1:] + GRID[:-1]) / 2  # a magnitude on the i-th goes to the even one of codes i and i + 1


def quantize(x):
    """(codes, scales) of a float map whose values are exact in float32."""
    x = np.asarray(x, dtype=np.float64)
    B, C, P = x.shape
    nb = (C + 31) // 32
    v = np.zeros((B, P, nb * 32))
    v[:, :, :C] = x.transpose(0, 2, 1)
    v = v.reshape(B, P, nb, 32)
    bad = ~np.isfinite(v).all(-1)
    v = np.where(bad[..., None], 0.0, v)
    top = np.abs(v).max(-1)
    s = np.where(top > 0, np.maximum(np.frexp(top)[1] - 1 - 2, -127), -127)
    a = np.abs(v) / np.exp2(s.astype(np.float64))[..., None]
    low = np.searchsorted(MIDS, a.ravel(), side="left").reshape(a.shape)   # ties down
    high = np.searchsorted(MIDS, a.ravel(), side="right").reshape(a.shape)  # ties up
    code = np.where(low % 2 == 0, low, high)
    code = np.where(bad[..., None], 0, code + 8 * (np.signbit(v) & ~bad[..., None]))
    scales = np.where(bad, 255, s + 127).astype(np.uint8)
    code = code.reshape(B, P, nb * 32)
    return (code[..., 0::2] + 16 * code[..., 1::2]).astype(np.uint8), scales


def values(codes, scales, C):
    """The map (B,C,P) that codes and scales stand for."""
    B, P, nb = scales.shape
    code = np.stack((codes & 15, codes >> 4), -1).reshape(B, P, nb, 32)
    s = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127))
    v = np.where(code >= 8, -1.0, 1.0) * GRID[code & 7] * s[..., None]
    return v.reshape(B, P, nb * 32)[:, :, :C].transpose(0, 2, 1)


def rounded(x):
    return values(*quantize(x), np.asarray(x).shape[1])


def gelu(v):
    return 0.5 * v * np.vectorize(math.erfc, otypes=[np.float64])(-v / math.sqrt(2.0))


def conv1x1(xq, wq, bias=None, act=None, residual=None, res_scale=None):
    """xq (B,C,P), wq (N,C): values.  The result, and the sum of its terms' magnitudes before act."""
    y = np.einsum("nc,bcp->bnp", wq, xq)
    mag = np.einsum("nc,bcp->bnp", np.abs(wq), np.abs(xq))
    col = lambda t: np.asarray(t, dtype=np.float64).reshape(1, -1, 1)  # noqa: E731
    if bias is not None:
        y, mag = y + col(bias), mag + np.abs(col(bias))
    if act == "gelu":
        y = gelu(y)
    if res_scale is not None:
        y = y * col(res_scale)
    if residual is not None:
        y = y + residual
    return y, mag


def gradients(gy, xq, wq):
    """Gradients of x, weight and bias, straight through the quantisation, each with the sum of its terms' magnitudes."""
    a = np.abs
    return ((np.einsum("nc,bnp->bcp", wq, gy), np.einsum("nc,bnp->bcp", a(wq), a(gy))),
            (np.einsum("bnp,bcp->nc", gy, xq), np.einsum("bnp,bcp->nc", a(gy), a(xq))),
            (gy.sum((0, 2)), a(gy).sum((0, 2))))
