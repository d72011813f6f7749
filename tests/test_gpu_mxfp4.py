"""MXFP4 maps, their 1x1 convolution and its gradients (functional.quantize_mxfp4, dequantize_mxfp4, conv1x1_mxfp4,
conv1x1_mxfp4_train) against the same in 64 bits.

Quantisation is exact: codes and scales are equal.  A product of 4-bit values is exact in float32, and so is a block's sum
of 32 of them but for the scales; a sum over K blocks rounds once a block at most in whatever order, each time by 2^-24 of no
more than the sum M of the terms' magnitudes (the matrix units align 128 terms to the largest one and may drop bits below
2^-24 of it: twice that).  With the bias, |error| <= (K + 2) 2^-23 M.  GELU's slope is below 1.13 and its own error below 4e-7
max(1, |v|).  A gradient's sum of T terms rounds T times in the worst order, and where its float32 operand is taken in parts,
the smallest of them may lose 2^-24 of it: (T + 2) 2^-24 M.  Each result is rounded once more: eps / 2 of its type."""
import copy
import threading

import numpy as np
import pytest
import torch

from oracle import mxfp4_oracle as O

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [F32, BF16, F16]


def fh():
    from conversenet_amd import functional

    return functional


def gen(seed):
    return torch.Generator().manual_seed(seed)


def make(shape, dtype=F32, seed=0):
    """A feature map: channels of different size, some values far from the others."""
    g = gen(seed)
    x = torch.randn(shape, generator=g) * torch.exp(0.7 * torch.randn((1, shape[1]) + (1,) * (len(shape) - 2), generator=g))
    x = torch.where(torch.rand(shape, generator=g) < 0.01, 20 * x, x)
    return x.to(dtype)


def np64(t):
    return t.detach().cpu().double().numpy()


def flat(t):
    a = np64(t)
    return a.reshape(a.shape[0], a.shape[1], -1)


def half_step(dtype, v):
    """What a rounding to dtype may change v by."""
    f = torch.finfo(dtype)
    return np.abs(v) * f.eps / 2 + f.smallest_normal * f.eps


def check(got, want, lim):
    got, want = np64(got).reshape(want.shape), np.asarray(want)
    bad = ~(np.abs(got - want) <= lim)
    assert not bad.any(), (int(bad.sum()), bad.size, np.abs(got - want).max(), np.max(np.abs(got - want) / (lim + 1e-300)))


def check_quantized(q, x):
    codes, scales = O.quantize(flat(x))
    assert q.channels == x.shape[1] and q.shape == tuple(x.shape)
    assert np.array_equal(q.scales.cpu().numpy().reshape(scales.shape), scales)
    assert np.array_equal(q.codes.cpu().numpy().reshape(codes.shape), codes)


SHAPES = [(1, 1, 1, 1), (1, 64, 1, 1), (2, 31, 3, 5), (1, 32, 1, 7), (3, 33, 4, 4), (2, 64, 16, 16), (1, 100, 67, 45),
          (5, 7, 2, 1), (2, 128, 9, 9), (300, 65), (1, 4096), (3, 257, 5), (2, 48, 3, 4, 5), (1, 320, 32, 33), (4, 96, 8, 63)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_round_trip(shape, dtype):
    x = make(shape, dtype, sum(shape)).cuda()
    q = fh().quantize_mxfp4(x)
    check_quantized(q, x)
    want = O.rounded(flat(x))
    for t in TYPES:
        v = fh().dequantize_mxfp4(q, t)
        assert v.dtype is t and v.shape == x.shape
        assert np.array_equal(flat(v), torch.from_numpy(want).to(t).double().numpy())


def test_round_trip_of_every_tie_and_scale():
    """Every border between two codes and its float32 neighbours, at every scale a number can have."""
    rows = []
    for e in range(-149, 128):
        top = np.float32(2.0) ** np.float32(e) if e >= -126 else np.float32(np.ldexp(1.0, e))
        unit = 2.0 ** max(e - 2, -127)
        m = np.float32(np.concatenate(([0.0], O.MIDS, O.GRID)) * unit)
        with np.errstate(over="ignore"):
            v = np.concatenate((m, np.nextafter(m, np.float32(np.inf)), np.nextafter(m, np.float32(0))))
        v = v[np.abs(v) < 2 * np.float64(top)][:31]
        v = v * np.where(np.arange(v.size) % 2, -1, 1).astype(np.float32)
        rows.append(np.concatenate(([top], v, np.zeros(31 - v.size, np.float32))))
    x = torch.from_numpy(np.stack(rows).astype(np.float32)).cuda()
    check_quantized(fh().quantize_mxfp4(x), x)
    planes = x.t().reshape(1, 32, -1).contiguous()  # the same as the pixels of a map
    check_quantized(fh().quantize_mxfp4(planes), planes)
    assert np.array_equal(flat(fh().dequantize_mxfp4(fh().quantize_mxfp4(planes))), O.rounded(flat(planes)))


@pytest.mark.parametrize("dtype", TYPES)
def test_blocks_that_hold_no_number(dtype):
    x = make((2, 70, 3, 5), dtype, 1)
    x[0, 3, 1, 1], x[0, 40, 1, 2], x[1, 69, 0, 0], x[1, 0, 2, 4] = float("nan"), float("inf"), -float("inf"), float("nan")
    x[0, :, 2, 2] = 0
    x[0, :, 2, 3] = -0.0
    x = x.cuda()
    q = fh().quantize_mxfp4(x)
    check_quantized(q, x)
    v, want = flat(fh().dequantize_mxfp4(q)), O.rounded(flat(x))
    assert np.array_equal(np.isnan(v), np.isnan(want)) and np.array_equal(np.nan_to_num(v), np.nan_to_num(want))
    w = make((40, 70), F32, 2).cuda()
    y = flat(fh().conv1x1_mxfp4(x, w))
    bad = np.isnan(want).any(1)
    assert bad.sum() == 4 and np.array_equal(np.isnan(y), np.broadcast_to(bad[:, None], y.shape))


def limits(K, mag, y, act, res_scale, residual, dtype):
    lim = (K + 2) * 2.0 ** -23 * mag
    if act == "gelu":
        lim = 1.13 * lim + 4e-7 * np.maximum(1, mag)
    if res_scale is not None:
        s = np.abs(np64(res_scale).reshape(1, -1, 1))
        lim = lim * s + 2.0 ** -24 * np.abs(s) * (mag + 1)
    if residual is not None:
        lim = lim + 2.0 ** -23 * (np.abs(y) + np.abs(flat(residual)))
    return lim + half_step(dtype, np.abs(y) + lim)


CONVS = [  # B, N, C, pixels
    (1, 1, 1, (1, 1)), (1, 16, 64, (1, 1)), (3, 50, 100, (1, 1)), (16, 96, 320, (1, 1)), (17, 33, 65, (1, 1)), (70, 40, 129, ()),
    (1, 128, 64, (16, 16)), (2, 64, 128, (8, 33)), (1, 3, 7, (67, 45)), (2, 80, 48, (5, 7)), (1, 100, 31, (13,)),
    (2, 260, 257, (9, 9)), (1, 65, 1000, (12, 20)), (3, 17, 33, (2, 1)), (1, 300, 512, (32, 20)), (4, 130, 96, (20, 12)),
    (1, 40, 4100, (3, 3)), (2, 1, 300, (4, 65)), (1, 2048, 32, (4, 4)), (1, 70, 300, (2, 3, 7)), (5, 8210, 100, (1, 1)),
    (2, 8192, 33, (2, 3)),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", CONVS, ids=str)
def test_conv1x1(case, dtype):
    B, N, C, space = case
    x, w = make((B, C, *space), dtype, 3).cuda(), (make((N, C), F32, 4) / C ** 0.5).cuda()
    g = gen(5)
    bias, s = torch.randn(N, generator=g).cuda(), torch.randn(N, generator=g).cuda()
    residual = torch.randn((B, N, *space), generator=g).to(dtype).cuda()
    xq, wq = O.rounded(flat(x)), O.rounded(np64(w)[:, :, None])[:, :, 0]
    K = (C + 31) // 32
    for b, act, r, rs in ((None, None, None, None), (bias, "gelu", None, None), (bias, None, residual, s),
                          (bias, "gelu", residual, None)):
        want, mag = O.conv1x1(xq, wq, None if b is None else np64(b), act, None if r is None else flat(r),
                              None if rs is None else np64(rs))
        lim = limits(K, mag, want, act, rs, r, dtype)
        y = fh().conv1x1_mxfp4(x, w, b, act, r, rs)
        assert y.dtype is dtype and y.shape == (B, N, *space)
        check(y, want, lim)
    # the same operands quantised before
    q = fh().quantize_mxfp4(x)
    wm = fh().quantize_mxfp4(w.view(N, C, 1, 1))
    assert torch.equal(fh().conv1x1_mxfp4(x, wm, bias, "gelu", residual), y)
    check(fh().conv1x1_mxfp4(q, wm, bias, "gelu", residual), want, lim)
    want, mag = O.conv1x1(xq, wq)
    check(fh().conv1x1_mxfp4(q, wm, dtype=BF16), want, limits(K, mag, want, None, None, None, BF16))


def by_channels(t):
    """A map (B,C,*) as (C, pixels) in 64 bits, on the device."""
    return t.detach().double().flatten(2).transpose(0, 1).flatten(1) if t.dim() > 2 else t.detach().double().t()


def check64(got, want, lim):
    bad = ~((got.double() - want).abs() <= lim)
    assert not bad.any(), (int(bad.sum()), bad.numel(), float((got.double() - want).abs().max()))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("case", [((1, 290, 4100), 2100), ((3, 520, 37, 37), 2176), ((2, 300, 32, 64), 2210), ((4100, 290), 2100),
                                  ((4096, 544), 2176)], ids=str)
def test_conv1x1_of_many_tiles(case, dtype):
    """More tiles than blocks, whole and partial ones, rows of the result on lines and off them."""
    shape, N = case
    F = fh()
    x, w = make(shape, dtype, 46).cuda(), F.quantize_mxfp4((make((N, shape[1]), F32, 47) / shape[1] ** 0.5).cuda())
    bias = torch.randn(N, generator=gen(48)).cuda()
    res = torch.randn((shape[0], N) + shape[2:], generator=gen(49)).to(dtype).cuda()
    q = F.quantize_mxfp4(x)
    xv, wv = by_channels(F.dequantize_mxfp4(q)), F.dequantize_mxfp4(w).double()
    want, mag = wv @ xv + bias.double()[:, None], wv.abs() @ xv.abs() + bias.double().abs()[:, None]
    want = want * torch.special.erfc(-want / 2 ** 0.5) / 2 + by_channels(res)
    K = (shape[1] + 31) // 32
    lim = 1.13 * (K + 2) * 2.0 ** -23 * mag + 4e-7 * mag.clamp(min=1) + (2.0 ** -23 + torch.finfo(dtype).eps / 2) * (
        want.abs() + by_channels(res).abs() + 1)
    for v in (x, q):
        y = F.conv1x1_mxfp4(v, w, bias, "gelu", res)
        assert y.shape == res.shape and y.dtype is dtype
        check64(by_channels(y), want, lim)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", [((1, 200, 130, 131), 40), ((17000, 200), 33), ((3, 130, 80, 71), 130), ((2, 500, 32, 33), 600),
                                  ((2000, 500), 600), ((2, 96, 160, 128), 64)], ids=str)
def test_gradients_of_many_tiles(case, dtype):
    shape, N = case
    F = fh()
    x, w = F.quantize_mxfp4(make(shape, dtype, 50).cuda()), F.quantize_mxfp4(make((N, shape[1]), F32, 51).cuda())
    gy = torch.randn((shape[0], N) + shape[2:], generator=gen(52)).to(dtype).cuda()
    gx, gw, gb = F.conv1x1_mxfp4_backward(gy, x, w)
    xv, wv, g = by_channels(F.dequantize_mxfp4(x)), F.dequantize_mxfp4(w).double(), by_channels(gy)
    P = g.shape[1]
    for got, a, b, terms, t in ((by_channels(gx), wv.t().contiguous(), g, N, dtype), (gw, g, xv.t().contiguous(), P, F32),
                                (gb, g, torch.ones_like(g[:1]).t().contiguous(), P, F32)):
        want, mag = (a @ b).view(got.shape), (a.abs() @ b.abs()).view(got.shape)
        check64(got, want, (terms + 2) * 2.0 ** -24 * mag + torch.finfo(t).eps / 2 * want.abs() + torch.finfo(t).smallest_normal)


def test_conv1x1_layouts_and_outputs():
    F = fh()
    x = make((2, 70, 12, 10), F32, 6).cuda()
    w = make((50, 70), F32, 7).cuda()
    ref = F.conv1x1_mxfp4(x, w)
    base = torch.zeros(2 * 70 * 120 + 1, device="cuda")
    odd = base[1:].view(2, 70, 12, 10)  # not aligned to 16 bytes
    odd.copy_(x)
    strided = torch.zeros(2, 70, 12, 20, device="cuda")[..., ::2]
    strided.copy_(x)
    for t in (odd, strided, x.to(memory_format=torch.channels_last), x.transpose(2, 3).contiguous().transpose(2, 3)):
        assert torch.equal(F.conv1x1_mxfp4(t, w), ref)
        check_quantized(F.quantize_mxfp4(t), x)
    q = F.quantize_mxfp4(w)
    moved = torch.zeros(q.codes.numel() + 1, dtype=torch.uint8, device="cuda")[1:].view(q.codes.shape)
    moved.copy_(q.codes)
    assert torch.equal(F.conv1x1_mxfp4(x, F.MXFP4(moved, q.scales, 70)), ref)
    out = torch.full((2, 50, 12, 10), 7.0, device="cuda")
    assert F.conv1x1_mxfp4(x, w, out=out) is out and torch.equal(out, ref)
    res = torch.randn(2, 50, 12, 10, device="cuda")
    want = F.conv1x1_mxfp4(x, w, residual=res)
    version = res._version
    assert F.conv1x1_mxfp4(x, w, residual=res, out=res) is res and torch.equal(res, want) and res._version > version
    guard = torch.full((2 * 50 * 120 + 64,), 3.0, device="cuda")
    inner = guard[32:-32].view(2, 50, 12, 10)
    F.conv1x1_mxfp4(x, w, out=inner)
    assert torch.equal(inner, ref) and (guard[:32] == 3).all() and (guard[-32:] == 3).all()
    for t in (F16, BF16):  # parameters of other types
        assert torch.equal(F.conv1x1_mxfp4(x, w, torch.ones(50, dtype=t, device="cuda")),
                           F.conv1x1_mxfp4(x, w, torch.ones(50, device="cuda")))


@pytest.mark.parametrize("shape", [(2, 70, 3, 5), (1, 70), (40, 300)])
def test_infinite_sums(shape):
    """GELU of an infinity is that infinity or zero, of a NaN a NaN, beside numbers that stay as they are."""
    F = fh()
    x, w = make(shape, F32, 36).cuda(), make((9, shape[1]), F32, 37).cuda()
    bias = torch.zeros(9, device="cuda")
    ref = F.conv1x1_mxfp4(x, w, bias, act="gelu")
    bias[2], bias[5], bias[7] = float("inf"), -float("inf"), float("nan")
    y = F.conv1x1_mxfp4(x, w, bias, act="gelu")
    assert (y[:, 2] == float("inf")).all() and (y[:, 5] == 0).all() and torch.isnan(y[:, 7]).all()
    keep = [0, 1, 3, 4, 6, 8]
    assert torch.equal(y[:, keep], ref[:, keep])


def test_negated_views():
    F = fh()
    for shape in ((2, 40, 3, 3), (1, 1, 1, 1)):
        z = torch.randn(shape, dtype=torch.complex64, device="cuda")
        x = z.conj().imag
        assert x.is_neg()
        plain = x.resolve_neg().clone()
        w = torch.randn(6, shape[1], device="cuda")
        assert torch.equal(F.dequantize_mxfp4(F.quantize_mxfp4(x)), F.dequantize_mxfp4(F.quantize_mxfp4(plain)))
        res = torch.randn((shape[0], 6) + shape[2:], dtype=torch.complex64, device="cuda").conj().imag
        assert torch.equal(F.conv1x1_mxfp4(x, w, residual=res), F.conv1x1_mxfp4(plain, w, residual=res.resolve_neg().clone()))
        lx, lw = plain.requires_grad_(True), w.requires_grad_(True)
        gy = torch.randn((shape[0], 6) + shape[2:], dtype=torch.complex64, device="cuda").conj().imag
        y = F.conv1x1_mxfp4_train(lx, lw)
        got = torch.autograd.grad(y, (lx, lw), gy, retain_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(got, torch.autograd.grad(y, (lx, lw), gy.resolve_neg().clone())))


def test_nothing_to_do():
    F = fh()
    w = make((5, 40), F32, 8).cuda()
    for shape in ((0, 40, 3, 3), (2, 40, 0, 3), (0, 40)):
        x = torch.empty(shape, device="cuda")
        q = F.quantize_mxfp4(x)
        assert F.dequantize_mxfp4(q).shape == x.shape and q.shape == x.shape
        assert F.conv1x1_mxfp4(x, w).shape == F.conv1x1_mxfp4(q, w).shape == (shape[0], 5) + shape[2:]
        x.requires_grad_(True)
        wl, b = w.clone().requires_grad_(True), torch.zeros(5, device="cuda", requires_grad=True)
        y = F.conv1x1_mxfp4_train(x, wl, b)
        gx, gw, gb = torch.autograd.grad(y, (x, wl, b), torch.empty_like(y))
        assert gx.shape == x.shape and (gw == 0).all() and (gb == 0).all()


TRAINS = [(1, 1, 1, (1, 1)), (1, 16, 64, (1, 1)), (3, 50, 100, (1, 1)), (37, 33, 65, ()), (2, 128, 64, (16, 16)),
          (2, 64, 128, (8, 33)), (1, 3, 7, (67, 45)), (3, 80, 48, (13, 7)), (1, 100, 31, (13,)), (2, 260, 257, (9, 9)), (3, 17, 33, (2, 1)),
          (1, 300, 512, (32, 20)), (4, 130, 96, (20, 12)), (1, 64, 64, (129, 131)), (300, 5, 40, (1, 1)), (2, 257, 40, (3, 5, 2))]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", TRAINS, ids=str)
def test_gradients(case, dtype):
    B, N, C, space = case
    F = fh()
    x, w = make((B, C, *space), dtype, 9).cuda(), (make((N, C, 1, 1), F32, 10) / C ** 0.5).cuda()
    bias = torch.randn(N, generator=gen(11)).cuda()
    gy = torch.randn((B, N, *space), generator=gen(12)).to(dtype).cuda()
    for t in (x, w, bias):
        t.requires_grad_(True)
    y = F.conv1x1_mxfp4_train(x, w, bias)
    assert y.dtype is dtype
    grads = torch.autograd.grad(y, (x, w, bias), gy, retain_graph=True)
    again = torch.autograd.grad(y, (x, w, bias), gy)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))
    xq, wq = O.rounded(flat(x)), O.rounded(np64(w)[:, :, 0])[:, :, 0]
    want, mag = O.conv1x1(xq, wq, np64(bias))
    check(y, want, limits((C + 31) // 32, mag, want, None, None, None, dtype))
    P = flat(x).shape[0] * flat(x).shape[2]
    for g, leaf, (want, mag), terms in zip(grads, (x, w, bias), O.gradients(flat(gy), xq, wq), (N, P, P)):
        assert g.dtype is leaf.dtype and g.shape == leaf.shape
        check(g, want, (terms + 2) * 2.0 ** -24 * mag + half_step(g.dtype, want))


@pytest.mark.parametrize("shape", [(2, 70, 5, 6), (5, 70)])
@pytest.mark.parametrize("mag", [1e-37, 1e-30, 1e30, 1e37])
def test_gradients_of_far_sizes(shape, mag):
    """The matrix units take bfloat16 numbers below 2^-126 for zeros: of each term, three parts of less than that are lost.
    Where the terms' magnitudes add up to more than float32's largest number, so may a sum on its way."""
    F = fh()
    x, w = make(shape, F32, 38).cuda(), make((30, 70), F32, 39).cuda()
    gy = (mag * torch.randn((shape[0], 30) + shape[2:], generator=gen(40))).cuda()
    xq, wq = F.quantize_mxfp4(x), F.quantize_mxfp4(w)
    got = F.conv1x1_mxfp4_backward(gy, xq, wq)
    xv, wv = O.rounded(flat(x)), O.rounded(np64(w)[:, :, None])[:, :, 0]
    P = xv.shape[0] * xv.shape[2]
    lost = (3 * 2.0 ** -126 * np.abs(wv).sum(0).max(), 3 * 2.0 ** -126 * np.abs(xv).sum((0, 2)).max(), 0)
    for g, (want, m), terms, tiny in zip(got, O.gradients(flat(gy), xv, wv), (30, P, P), lost):
        keep = m <= torch.finfo(F32).max
        g = np64(g).reshape(want.shape)[keep]
        assert (np.abs(g - want[keep]) <= ((terms + 2) * 2.0 ** -24 * m + tiny + half_step(F32, want))[keep]).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_gradients_that_are_no_numbers(dtype):
    """An infinite or NaN gradient reaches what its terms reach, and nothing else."""
    F = fh()
    x, w = make((2, 70, 5, 6), dtype, 41).cuda(), make((30, 70), F32, 42).cuda()
    w[:, 3] = 0  # a channel with zeros only: infinity times zero
    gy = torch.randn((2, 30, 5, 6), generator=gen(43)).to(dtype).cuda()
    gy[0, 4, 1, 2], gy[1, 7, 0, 0], gy[1, 20, 4, 5] = float("inf"), -float("inf"), float("nan")
    xq, wq = F.quantize_mxfp4(x), F.quantize_mxfp4(w)
    xv, wv = O.rounded(flat(x)), O.rounded(np64(w)[:, :, None])[:, :, 0]
    with np.errstate(invalid="ignore"):
        wants = O.gradients(flat(gy), xv, wv)
    for g, (want, m), terms in zip(F.conv1x1_mxfp4_backward(gy, xq, wq), wants, (30, 60, 60)):
        g = np64(g).reshape(want.shape)
        fin = np.isfinite(want)
        assert np.array_equal(np.isnan(g), np.isnan(want)) and np.array_equal(np.isinf(g), np.isinf(want))
        assert np.array_equal(g[np.isinf(g)], want[np.isinf(want)])
        lim = (terms + 2) * 2.0 ** -24 * m[fin] + half_step(dtype, want[fin])
        assert (np.abs(g[fin] - want[fin]) <= lim).all()


def test_hooks_that_change_what_is_kept():
    F = fh()
    x, w = make((2, 40, 3, 3), F32, 44).cuda().requires_grad_(True), make((8, 40), F32, 45).cuda().requires_grad_(True)
    gy = torch.randn(2, 8, 3, 3, device="cuda")
    want = torch.autograd.grad(F.conv1x1_mxfp4_train(x, w), (x, w), gy)
    with torch.autograd.graph.save_on_cpu():
        y = F.conv1x1_mxfp4_train(x, w)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, (x, w), gy), want))
    for unpack in (lambda t: t.cpu(), lambda t: t[1:], lambda t: t.float()):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
            y = F.conv1x1_mxfp4_train(x, w)
        with pytest.raises(RuntimeError, match="hook"):
            torch.autograd.grad(y, (x, w), gy)


def test_gradients_against_differences():
    """Straight through the quantisation the loss is that of the rounded operands: its differences about them."""
    F = fh()
    x, w = make((2, 40, 3, 4), F32, 13).cuda(), make((9, 40), F32, 14).cuda()
    x.requires_grad_(True), w.requires_grad_(True)
    b = torch.zeros(9, device="cuda", requires_grad=True)
    gy = torch.randn(2, 9, 3, 4, generator=gen(15)).cuda()
    gx, gw, gb = torch.autograd.grad(F.conv1x1_mxfp4_train(x, w, b), (x, w, b), gy)
    xq, wq, g = O.rounded(flat(x)), O.rounded(np64(w)[:, :, None])[:, :, 0], flat(gy)
    loss = lambda xv, wv, bv: (O.conv1x1(xv, wv, bv)[0] * g).sum()  # noqa: E731
    rng = np.random.default_rng(16)
    for leaf, grad in enumerate((gx, gw, gb)):
        ops = [xq, wq, np.zeros(9)]
        d = rng.standard_normal(ops[leaf].shape)
        ends = []
        for h in (0.5, -0.5):  # linear in each operand: any step will do
            moved = list(ops)
            moved[leaf] = ops[leaf] + h * d
            ends.append(loss(*moved))
        terms = np64(grad).reshape(d.shape) * d
        assert abs((ends[0] - ends[1]) - terms.sum()) <= 60 * 2.0 ** -23 * np.abs(terms).sum() + 1e-12 * abs(ends[0])


def test_gradient_arguments():
    F = fh()
    x, w = make((2, 70, 5, 6), F32, 17).cuda().requires_grad_(True), make((30, 70), F16, 18).cuda().requires_grad_(True)
    b = torch.randn(30, device="cuda", dtype=BF16, requires_grad=True)
    y = F.conv1x1_mxfp4_train(x, w, b)
    gx, gw, gb = torch.autograd.grad(y.sum(), (x, w, b), retain_graph=True)  # an expanded gradient
    g1 = torch.autograd.grad(y, (x, w, b), torch.ones_like(y))
    assert all(torch.equal(p, q) and p.dtype is q.dtype for p, q in zip((gx, gw, gb), g1))
    assert gw.dtype is F16 and gb.dtype is BF16
    # each gradient by itself, and the function behind them
    for i, leaf in enumerate((x, w, b)):
        ls = [t.detach().clone().requires_grad_(j == i) for j, t in enumerate((x, w, b))]
        yi = F.conv1x1_mxfp4_train(*ls)
        assert torch.equal(torch.autograd.grad(yi, ls[i], torch.ones_like(yi))[0], g1[i])
    gy = torch.randn(2, 30, 5, 6, device="cuda")
    xq, wq = F.quantize_mxfp4(x.detach()), F.quantize_mxfp4(w.detach())
    full = F.conv1x1_mxfp4_backward(gy, xq, wq)
    strided = gy.to(memory_format=torch.channels_last)
    for need in ((True, False, False), (False, True, False), (False, False, True), (True, True, False)):
        got = F.conv1x1_mxfp4_backward(strided, xq if need[1] else None, wq if need[0] else None, need)
        assert all(g is None if not n else torch.equal(g, f) for g, f, n in zip(got, full, need))
    # no bias, no gradients wanted, and twice
    assert F.conv1x1_mxfp4_train(x.detach(), w.detach()).requires_grad is False
    yb = F.conv1x1_mxfp4_train(x, w)
    g2 = torch.autograd.grad(yb, (x, w), torch.ones_like(yb), create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g2[0].sum(), w)
    with pytest.raises(RuntimeError, match="plain tensors|vmap"):
        torch.autograd.grad(F.conv1x1_mxfp4_train(x, w), x, torch.ones((2,) + tuple(y.shape), device="cuda"), is_grads_batched=True)


def test_saved_operands_are_the_forward_s():
    """x and weight may change in place between forward and backward: the operands are kept in 4 bits."""
    F = fh()
    x, w = make((2, 64, 8, 8), F32, 19).cuda(), make((32, 64), F32, 20).cuda()
    gy = torch.randn(2, 32, 8, 8, device="cuda")
    lx, lw = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    want = torch.autograd.grad(F.conv1x1_mxfp4_train(lx, lw), (lx, lw), gy)
    lx, lw = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    y = F.conv1x1_mxfp4_train(lx, lw)
    with torch.no_grad():
        lx.zero_(), lw.zero_()
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, (lx, lw), gy), want))


@pytest.mark.parametrize("shape", [(4, 320, 1, 1), (1, 64, 16, 16), (1, 320, 16, 16)])
def test_graph_stream_and_threads(shape):
    F = fh()
    x, w = make(shape, F32, 21).cuda(), F.quantize_mxfp4(make((96, shape[1]), F32, 22).cuda())
    ref = F.conv1x1_mxfp4(x, w, act="gelu")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(F.conv1x1_mxfp4(x, w, act="gelu"), ref)
        g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
        xs = [x.clone(), x.clone()]
        with torch.cuda.graph(g1, stream=side):
            y1 = F.conv1x1_mxfp4(xs[0], w, act="gelu")
        with torch.cuda.graph(g2, stream=side):
            y2 = F.conv1x1_mxfp4(xs[1], w, act="gelu")
    torch.cuda.synchronize()
    for i in range(4):
        xs[0].copy_(make(shape, F32, 30 + i)), xs[1].copy_(make(shape, F32, 40 + i))
        g1.replay(), g2.replay()
        torch.cuda.synchronize()
        assert torch.equal(y1, F.conv1x1_mxfp4(xs[0], w, act="gelu")) and torch.equal(y2, F.conv1x1_mxfp4(xs[1], w, act="gelu"))
    bad = []

    def work(i):
        xi = make(shape, F32, 50 + i).cuda()
        want = F.conv1x1_mxfp4(xi, w)
        for _ in range(20):
            if not torch.equal(F.conv1x1_mxfp4(xi, w), want):
                bad.append(i)

    ts = [threading.Thread(target=work, args=(i,)) for i in range(3)]
    [t.start() for t in ts], [t.join() for t in ts]
    assert not bad


def test_recorded_training_pass():
    F = fh()
    x, w = make((2, 64, 12, 12), F32, 23).cuda().requires_grad_(True), make((128, 64), F32, 24).cuda().requires_grad_(True)
    b, gy = torch.zeros(128, device="cuda", requires_grad=True), torch.randn(2, 128, 12, 12, device="cuda")

    def step():
        y = F.conv1x1_mxfp4_train(x, w, b)
        return (y.detach(), *torch.autograd.grad(y, (x, w, b), gy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for i in range(4):
        with torch.no_grad():
            x.copy_(make((2, 64, 12, 12), F32, 60 + i)), w.copy_(make((128, 64), F32, 70 + i))
            gy.copy_(torch.randn(2, 128, 12, 12, generator=gen(80 + i)))
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(out, step()))


def test_offsets_past_32_bits():
    """A map of more than 2^32 bytes whose last pixels count."""
    F = fh()
    x = torch.zeros((1, 64, 4100, 4200), device="cuda")  # 4.4 GB
    x[..., -3:, -70:] = make((1, 64, 3, 70), F32, 25).cuda()
    w = make((16, 64), F32, 26).cuda()
    tail = x[..., -3:, -70:].contiguous()
    assert torch.equal(F.conv1x1_mxfp4(x, w)[..., -3:, -70:], F.conv1x1_mxfp4(tail, w))
    q = F.quantize_mxfp4(x)
    assert torch.equal(q.codes[:, -3:, -70:], F.quantize_mxfp4(tail).codes)
    assert torch.equal(F.dequantize_mxfp4(q)[..., -3:, -70:], F.dequantize_mxfp4(F.quantize_mxfp4(tail)))


def test_refusals():
    F = fh()
    x, w = make((2, 40, 3, 3), F32, 27).cuda(), make((6, 40), F32, 28).cuda()
    q, wm = F.quantize_mxfp4(x), F.quantize_mxfp4(w)
    y = torch.empty(2, 6, 3, 3, device="cuda")
    for call, what in (
            (lambda: F.quantize_mxfp4(x.double()), "float32, bfloat16 or float16"),
            (lambda: F.quantize_mxfp4(x.cpu()), "HIP device"),
            (lambda: F.quantize_mxfp4(x[0, 0, 0]), "channels"),
            (lambda: F.quantize_mxfp4(x[:, :0]), "channels"),
            (lambda: F.dequantize_mxfp4(q, torch.float64), "float32, bfloat16 or float16"),
            (lambda: F.dequantize_mxfp4(F.MXFP4(q.codes, q.scales, 65)), "blocks"),
            (lambda: F.dequantize_mxfp4(F.MXFP4(q.codes.float(), q.scales, 40)), "uint8"),
            (lambda: F.dequantize_mxfp4(F.MXFP4(q.codes.cpu(), q.scales.cpu(), 40)), "HIP device"),
            (lambda: F.conv1x1_mxfp4(x, w[:, :39]), "input channels"),
            (lambda: F.conv1x1_mxfp4(x, x), "matrix"),
            (lambda: F.conv1x1_mxfp4(x, q), "input channels"),
            (lambda: F.conv1x1_mxfp4(x, w.cpu()), "device"),
            (lambda: F.conv1x1_mxfp4(x, w, torch.zeros(5, device="cuda")), "bias"),
            (lambda: F.conv1x1_mxfp4(x, w, act="relu"), "activation"),
            (lambda: F.conv1x1_mxfp4(x, w, residual=y[:1]), "residual"),
            (lambda: F.conv1x1_mxfp4(x, w, residual=y.half()), "residual"),
            (lambda: F.conv1x1_mxfp4(x, w, out=y.permute(0, 1, 3, 2)), "contiguous"),
            (lambda: F.conv1x1_mxfp4(x, w, dtype=F16), "type of x"),
            (lambda: F.conv1x1_mxfp4(q, wm, dtype=torch.float64), "float32, bfloat16 or float16"),
            (lambda: F.conv1x1_mxfp4_train(q, w), "quantises"),
            (lambda: F.conv1x1_mxfp4_backward(y, None, wm), "operand"),
            (lambda: F.conv1x1_mxfp4_backward(y, q, F.quantize_mxfp4(w[:5])), "match"),
            (lambda: F.conv1x1_mxfp4_backward(y[:1], q, wm), "match")):
        with pytest.raises(RuntimeError, match=what):
            call()
    buf = torch.zeros(4 * 2 * 40 * 9, device="cuda")
    xb = buf[:720].view(2, 40, 3, 3)
    for lo in (0, 700):  # an output on top of x
        with pytest.raises(RuntimeError, match="shares memory"):
            F.conv1x1_mxfp4(xb, w, out=buf[lo:lo + 108].view(2, 6, 3, 3))
    with pytest.raises(RuntimeError, match="shares memory"):
        F.conv1x1_mxfp4(x, w, residual=buf[:108].view(2, 6, 3, 3), out=buf[8:116].view(2, 6, 3, 3))
    with pytest.raises(RuntimeError, match="shares memory"):
        F.conv1x1_mxfp4(x, w, buf[100:106], out=buf[:108].view(2, 6, 3, 3))
    with pytest.raises(RuntimeError, match="traced"):
        torch.jit.trace(lambda t: F.conv1x1_mxfp4(t, wm), x)


def block(cls, C=64, k=5, seed=0):
    from conversenet_amd import util_converse as U
    torch.manual_seed(seed)
    blk = getattr(U, cls)(C, C, kernel_size=k, padding=2, padding_mode="circular")
    if cls != "ConverseBlock":
        torch.nn.init.normal_(blk.alpha1), torch.nn.init.normal_(blk.alpha2)
    return U.use_mxfp4(blk).cuda()


@pytest.mark.parametrize("cls", ["ConverseBlock", "ConverseBlockAlphaVariant"])
@pytest.mark.parametrize("C,shape", [(64, (2, 64, 24, 20)), (24, (1, 24, 13, 9))])
def test_block_of_mxfp4_convolutions(cls, C, shape):
    """Quantisation, products with GELU and residuals, norms and the Converse2D of a block, as its forward runs them."""
    F = fh()
    blk = block(cls, C)
    x = make(shape, F32, 31).cuda()
    with torch.no_grad():
        y = blk(x)
        t = x
        for seq, alpha in ((blk.conv1, getattr(blk, "alpha1", None)), (blk.conv2, getattr(blk, "alpha2", None))):
            v = F.conv1x1_mxfp4(seq[0](t), F.quantize_mxfp4(seq[1].weight), seq[1].bias, act="gelu")
            if seq is blk.conv1:
                v = seq[3](v, act="gelu")
            t = F.conv1x1_mxfp4(v, F.quantize_mxfp4(seq[-1].weight), seq[-1].bias, residual=t, res_scale=alpha)
    assert torch.equal(y, t)
    from conversenet_amd.util_converse import run_blocks
    with torch.no_grad():
        assert torch.equal(run_blocks([blk, blk], x), blk(blk(x)))


def test_training_step_of_mxfp4_blocks():
    """Forward, gradients, clipping and an update of two blocks, each gradient against the chain of functions."""
    F = fh()
    blks = torch.nn.Sequential(block("ConverseBlockAlphaVariant", seed=1), block("ConverseBlockAlphaVariant", seed=2))
    x = make((2, 64, 16, 18), F32, 32).cuda()
    opt = torch.optim.SGD(blks.parameters(), lr=1e-3)

    def convs(h, seq):
        for m in list(seq)[1:]:
            h = F.conv1x1_mxfp4_train(h, m.weight, m.bias) if isinstance(m, torch.nn.Conv2d) else m(h)
        return h

    def chain(v):
        for b in blks:
            n1, n2 = b.conv1[0], b.conv2[0]
            h = convs(F.layernorm_cf_train(v, n1.weight, n1.bias, n1.eps, copy=True), b.conv1)
            v, h = F.residual_norm_train(v, h, (n2.weight, n2.bias, n2.eps), b.alpha1)
            v, _ = F.residual_norm_train(v, convs(h, b.conv2), None, b.alpha2)
        return v

    for _ in range(2):
        want = torch.autograd.grad(chain(x).square().mean(), list(blks.parameters()))
        opt.zero_grad()
        blks(x).square().mean().backward()
        assert all(torch.equal(p.grad, w) and torch.isfinite(w).all() for p, w in zip(blks.parameters(), want))
        F.clip_grad_norm_(blks.parameters(), 1.0)
        opt.step()
    assert torch.isfinite(blks(x)).all()


def test_recording_beside_an_eager_graph_is_refused():
    """A training pass is not recorded while an eager graph of the same leaves lives, and is once that is gone."""
    F = fh()
    x, w = make((2, 64, 12, 12), F32, 33).cuda().requires_grad_(True), make((32, 64), F32, 34).cuda().requires_grad_(True)
    gy = torch.randn(2, 32, 12, 12, device="cuda")
    alive = F.conv1x1_mxfp4_train(x, w)
    gx = torch.zeros_like(x)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        gx.add_(1)
        for leaf in (x, w):
            with pytest.raises(RuntimeError, match="holds one of its leaves"):
                F.conv1x1_mxfp4_train(x if leaf is x else x.detach(), w if leaf is w else w.detach())
        with torch.no_grad():
            F.conv1x1_mxfp4_train(x, w)
    want = torch.autograd.grad(alive, (x, w), gy)
    del alive, g
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = F.conv1x1_mxfp4_train(x, w)
        z = F.conv1x1_mxfp4_train(x, w)  # the same leaves twice in one recording
        got = torch.autograd.grad(y, (x, w), gy), torch.autograd.grad(z, (x, w), gy)
    for _ in range(3):
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for pair in got for a, c in zip(pair, want))


def test_modules_under_modes_and_transforms():
    """Tracers, transforms and observers see torch operations, hooks and other types what they asked for."""
    from conversenet_amd.util_converse import Conv1x1MXFP4
    conv = Conv1x1MXFP4(40, 8).cuda()
    x = make((2, 40, 5, 6), F32, 35).cuda()
    ref = conv(x)
    mag = O.conv1x1(O.rounded(flat(x)), O.rounded(flat(conv.weight))[:, :, 0], np64(conv.bias))[1]
    lim = 2 * 42 * 2.0 ** -23 * mag.max()  # both sides' sums of 41 terms
    traced = torch.jit.trace(conv, x)
    assert torch.allclose(traced(x), ref, rtol=0, atol=lim)
    from torch.fx.experimental.proxy_tensor import make_fx
    assert torch.allclose(make_fx(lambda t: conv(t))(x)(x), ref, rtol=0, atol=lim)
    assert torch.equal(conv(x[0]), conv(x[:1])[0])
    assert torch.equal(conv(x.half()), fh().conv1x1_mxfp4(x.half(), conv.weight, conv.bias))
    d = copy.deepcopy(conv).double()
    assert d(x.double()).dtype is torch.float64 and torch.allclose(d(x.double()).float(), ref, rtol=0, atol=lim)
    with torch.inference_mode():
        assert torch.equal(conv(x), ref)


def test_recording_with_views_of_held_leaves_is_refused():
    """Operands that are views of a leaf, or come from it, are refused where the leaf itself would be; views made in the recording of
    leaves that no other graph holds are recorded."""
    from conversenet_amd.util_converse import Conv1x1MXFP4
    F = fh()
    x, w = make((64, 12, 12), F32, 33).cuda().requires_grad_(True), make((32, 64), F32, 34).cuda().requires_grad_(True)
    gy = torch.randn(1, 32, 12, 12, device="cuda")
    plain_x, plain_w, conv = x.detach()[None], w.detach(), Conv1x1MXFP4(64, 32, bias=False).cuda()
    alive = [x * 2, w * 2]
    early = w.view(32, 64, 1, 1)
    fill = torch.zeros(4, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        fill.add_(1)
        for a, b in ((plain_x, w.view(32, 64, 1, 1)), (plain_x, w.flatten(1) * 1.0), (x.unsqueeze(0), plain_w), (plain_x, early)):
            with pytest.raises(RuntimeError, match="outside of the recording"):
                F.conv1x1_mxfp4_train(a, b)
        with pytest.raises(RuntimeError, match="outside of the recording"):
            conv(x)  # (a single sample)
    want = torch.autograd.grad(F.conv1x1_mxfp4_train(x[None], w), (x, w), gy)
    del alive, early, a, b, g
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = torch.autograd.grad(F.conv1x1_mxfp4_train(x.unsqueeze(0), w.view(32, 64, 1, 1)), (x, w), gy)
    for _ in range(3):
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_recordings_whose_leaves_have_nodes_of_their_own():
    """What a recording's leaves are used for before in the same recording, on the same stream before it, or on a stream that it forks
    onto does not keep a training pass from being recorded."""
    F = fh()
    x, w = make((2, 64, 12, 12), F32, 33).cuda().requires_grad_(True), make((32, 64), F32, 34).cuda().requires_grad_(True)
    gy = torch.randn(2, 32, 12, 12, device="cuda")
    side, fork = torch.cuda.Stream(), torch.cuda.Stream()

    def penalty():
        p = 0.5 * w.square().sum(1)
        y = F.conv1x1_mxfp4_train(x * 2.0, w.view(32, 64, 1, 1))
        return torch.autograd.grad((y, p), (x, w), (gy, torch.ones_like(p)))

    def forked():
        fork.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(fork):
            v = w * 2.0
        torch.cuda.current_stream().wait_stream(fork)
        grads = torch.autograd.grad(F.conv1x1_mxfp4_train(x, v), (x, w), gy)
        torch.cuda.current_stream().wait_stream(fork)
        return grads

    def again():
        return torch.autograd.grad(F.conv1x1_mxfp4_train(x, w), (x, w), gy)

    for step, held in ((penalty, False), (forked, False), (again, True)):
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            want = step()
            alive = [x * 2.0, w * 2.0] if held else None  # nodes on the recording's stream
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            got = step()
        for _ in range(3):
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, want))
        del alive


def test_evaluation_of_blocks_with_hooks():
    """Hooks of a block's convolutions run in evaluation, and a weight that a hook makes is the current one."""
    F = fh()
    blk = block("ConverseBlockAlphaVariant", seed=3)
    x = make((2, 64, 16, 18), F32, 36).cuda()
    with torch.no_grad():
        seen = []
        handle = blk.conv2[3].register_forward_hook(lambda m, args, out: seen.append(out))
        y = blk(x)
        assert len(seen) == 1
        handle.remove()
        t = blk.alpha1 * blk.conv1(x) + x
        assert torch.equal(y, blk.alpha2 * blk.conv2(t) + t)
        with pytest.warns(FutureWarning):
            conv = torch.nn.utils.weight_norm(blk.conv2[1])
        n = make((2, 64, 16, 18), F32, 37).cuda()
        args = {}
        conv.register_forward_hook(lambda m, a, out: args.update(x=a[0], y=out))
        conv.weight_g.mul_(3.0)
        blk(x)
        w = torch._weight_norm(conv.weight_v, conv.weight_g, 0)
        assert torch.equal(args["y"], F.conv1x1_mxfp4(args["x"], w, conv.bias))


def test_autocast_changes_nothing():
    """The kernels and the composition that stands in for them give the input's type under autocast, forward and backward."""
    from conversenet_amd import composite
    from conversenet_amd.util_converse import Conv1x1MXFP4
    conv = Conv1x1MXFP4(40, 8).cuda()
    x = make((2, 40, 5, 6), F32, 38).cuda()
    params = list(conv.parameters())
    y = conv(x)
    grads = torch.autograd.grad(y.square().sum(), params)
    mag = O.conv1x1(O.rounded(flat(x)), O.rounded(flat(conv.weight))[:, :, 0], np64(conv.bias))[1]
    for t in (torch.bfloat16, torch.float16):
        with torch.autocast("cuda", dtype=t):
            z = conv(x)
            assert z.dtype is F32 and torch.equal(z, y)
            assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(z.square().sum(), params), grads))
            with torch.no_grad():
                assert torch.equal(conv(x), y)
                c = composite.conv1x1_mxfp4(x, conv.weight, conv.bias)
                assert c.dtype is F32 and torch.allclose(c, y, rtol=0, atol=2 * 42 * 2.0 ** -23 * mag.max())
                h = conv(x.to(t))  # what a convolution under autocast hands on
                assert h.dtype is t and torch.equal(h, fh().conv1x1_mxfp4(x.to(t), conv.weight, conv.bias))


class Holder(torch.Tensor):
    """A tensor that stands for another one and has no memory of its own."""

    @staticmethod
    def __new__(cls, inner):
        return torch.Tensor._make_wrapper_subclass(cls, inner.shape, dtype=inner.dtype, device=inner.device,
                                                   requires_grad=inner.requires_grad)

    def __init__(self, inner):
        self.inner = inner

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        from torch.utils._pytree import tree_map
        return func(*tree_map(lambda t: t.inner if isinstance(t, cls) else t, args), **(kwargs or {}))


def test_parameters_that_stand_for_others():
    from conversenet_amd.util_converse import Conv1x1MXFP4
    conv = Conv1x1MXFP4(40, 8).cuda().requires_grad_(False)
    x = make((2, 40, 5, 6), F32, 39).cuda()
    y = conv(x)
    mag = O.conv1x1(O.rounded(flat(x)), O.rounded(flat(conv.weight))[:, :, 0], np64(conv.bias))[1]
    for name in ("weight", "bias"):
        other = copy.deepcopy(conv)
        delattr(other, name)
        setattr(other, name, Holder(getattr(conv, name).detach()))
        # (the composition: both sides' sums of 41 terms)
        assert torch.allclose(other(x), y, rtol=0, atol=2 * 42 * 2.0 ** -23 * mag.max())


def test_tensors_without_memory_are_refused():
    """An operand that stands for another tensor is not taken for one that is not there."""
    F = fh()
    x, w = make((2, 40, 3, 4), F32, 40).cuda(), make((8, 40), F32, 41).cuda()
    q, wm, v = F.quantize_mxfp4(x), F.quantize_mxfp4(w), torch.ones(8, device="cuda")
    r = torch.ones(2, 8, 3, 4, device="cuda")
    H = Holder
    for call in (lambda: F.quantize_mxfp4(H(x)), lambda: F.conv1x1_mxfp4(H(x), w), lambda: F.conv1x1_mxfp4(x, H(w)),
                 lambda: F.conv1x1_mxfp4(x, w, H(v)), lambda: F.conv1x1_mxfp4(x, w, res_scale=H(v)),
                 lambda: F.conv1x1_mxfp4(x, w, residual=H(r)), lambda: F.conv1x1_mxfp4(x, w, out=H(r)),
                 lambda: F.conv1x1_mxfp4(F.MXFP4(H(q.codes), q.scales, 40), w),
                 lambda: F.conv1x1_mxfp4(q, F.MXFP4(wm.codes, H(wm.scales), 40)),
                 lambda: F.dequantize_mxfp4(F.MXFP4(q.codes, H(q.scales), 40)),
                 lambda: F.conv1x1_mxfp4_backward(H(r), q, wm),
                 lambda: F.conv1x1_mxfp4_backward(r, F.MXFP4(H(q.codes), q.scales, 40), wm),
                 lambda: F.conv1x1_mxfp4_backward(r, q, F.MXFP4(wm.codes, H(wm.scales), 40)),
                 lambda: F.conv1x1_mxfp4_train(H(x), w.requires_grad_()), lambda: F.conv1x1_mxfp4_train(x.requires_grad_(), H(w)),
                 lambda: F.conv1x1_mxfp4_train(x, w, H(v))):
        with pytest.raises(RuntimeError, match="no memory|null pointer"):
            call()


EXACT = [((1, 64, 129, 131), 64), ((1, 200, 130, 131), 40), ((2, 40, 131, 65), 9), ((3, 300, 67, 71), 130), ((17003, 200), 33),
         ((5003, 64), 130), ((1, 64, 401, 503), 128), ((7, 33, 1, 3), 257), ((2, 130, 257), 1)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", EXACT, ids=str)
def test_sums_that_are_exact(case, dtype):
    """Whole numbers whose sums float32 holds: every term counts, to the last pixel of the last split, and none is counted twice.
    x and w are MXFP4 values in steps of 1/2 (each block's scale reaches them), grad_y whole numbers of up to 9 bits (8 in
    bfloat16): products in steps of 1/4 and 1/2, the sums of their magnitudes below 2^24 steps."""
    shape, N = case
    F = fh()
    g = gen(shape[0] + shape[1])
    values = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.5, -1, -1.5, -2, -3, -4, -6])
    pick = lambda *s: values[torch.randint(0, 15, s, generator=g)]  # noqa: E731
    P = shape[0] * int(np.prod(shape[2:]))
    most = min(200 if dtype is BF16 else 300, 5000000 // P)
    x, w, bias = pick(*shape), pick(N, shape[1]), torch.randint(-9, 10, (N,), generator=g).float()
    gy = torch.randint(-most, most + 1, (shape[0], N) + shape[2:], generator=g).float()
    gy.view(shape[0], N, -1)[-1, :, -1], x.view(*shape[:2], -1)[-1, :, -1] = most, 6.0  # a lost last pixel shows everywhere
    xs, ws, gs, bs = (t.to(d).cuda() for t, d in ((x, dtype), (w, F32), (gy, dtype), (bias, F32)))
    for t in (xs, ws, bs):
        t.requires_grad_(True)
    y = F.conv1x1_mxfp4_train(xs, ws, bs)
    gx, gw, gb = torch.autograd.grad(y, (xs, ws, bs), gs)
    xc, gc, wd = by_channels(x).double(), by_channels(gy).double(), w.double()
    for got, a, b, steps, t, extra in ((by_channels(y), wd, xc, 4, dtype, bias[:, None].double()), (by_channels(gx), wd.t(), gc, 2, dtype, 0),
                                       (gw, gc, xc.t(), 2, F32, 0), (gb[:, None], gc, torch.ones(P, 1, dtype=torch.float64), 1, F32, 0)):
        assert steps * ((a.abs() @ b.abs()).max() + 9) < 2 ** 24
        want = a @ b + extra
        assert t is not F16 or want.abs().max() < 65504
        assert torch.equal(got.detach().cpu().double().view(want.shape), want.to(t).double())
    q, m = F.quantize_mxfp4(xs.detach()), F.quantize_mxfp4(ws.detach())
    again = F.conv1x1_mxfp4_backward(gs, q, m)
    assert torch.equal(again[0], gx) and torch.equal(again[1], gw) and torch.equal(again[2], gb)
    assert torch.equal(F.conv1x1_mxfp4(q, m, bs.detach(), dtype=dtype), y)
    assert torch.equal(F.conv1x1_mxfp4_backward(gs, q, m, (True, False, True))[2], gb)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", [((1, 64, 129, 131), 64), ((1, 200, 130, 131), 40), ((17003, 70), 33), ((3, 40, 80, 71), 130)], ids=str)
def test_bias_gradients_are_sums_in_64_bits(case, dtype):
    """grad_bias is summed in float64 and rounded once, with the matrix' gradient and without it."""
    shape, N = case
    F = fh()
    x, w = F.quantize_mxfp4(make(shape, dtype, 53).cuda()), F.quantize_mxfp4(make((N, shape[1]), F32, 54).cuda())
    gy = torch.randn((shape[0], N) + shape[2:], generator=gen(55)).to(dtype)
    g = by_channels(gy).double()
    want, mag, P = g.sum(1), g.abs().sum(1), g.shape[1]
    assert (g[:, -1].abs() > 2.0 ** -23 * want.abs() + 2 * P * 2.0 ** -52 * mag).float().mean() > 0.9  # a lost pixel shows
    for need in ((True, True, True), (False, True, True), (True, False, True), (False, False, True)):
        gb = F.conv1x1_mxfp4_backward(gy.cuda(), x, w, need)[2].cpu().double()
        # both sides' sums of P terms in float64, one rounding to float32
        assert ((gb - want).abs() <= 2.0 ** -24 * want.abs() + 2 * P * 2.0 ** -53 * mag).all()
