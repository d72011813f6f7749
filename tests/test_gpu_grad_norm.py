"""The norm over many gradients and clipping (functional.grad_norm, clip_grads, clip_grad_norm_) against the same in 64
bits.  The norm is accumulated in 64 bits and rounded once: 2^-24 of itself and what a 64-bit sum of n squares loses,
n 2^-53.  A clipped value is the product with the factor, which is rounded to float32 once, rounded in float32 and then
to its type: 2^-23 and eps / 2 of the value."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def fh():
    from conversenet_amd import functional

    return functional


def make(sizes, types=(F32,), seed=0, mag=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(mag * torch.randn(n, generator=g)).to(types[i % len(types)]).cuda() for i, n in enumerate(sizes)]


def norm64(ts, p=2.0):
    if p == math.inf:
        return max((float(t.double().abs().max()) for t in ts if t.numel()), default=0.0)
    return math.sqrt(math.fsum(float((t.double() ** 2).sum()) for t in ts))


def check_norm(got, ts, p=2.0):
    assert got.dtype == F32 and got.shape == ()
    ref = norm64(ts, p)
    n = sum(t.numel() for t in ts)
    assert abs(float(got) - ref) <= ref * (2.0 ** -24 + n * 2.0 ** -53) + 1e-45, (float(got), ref)


def check_clipped(got, ts, ref_norm, max_norm):
    f = min(1.0, max_norm / (ref_norm + 1e-6))
    for o, t in zip(got, ts):
        assert o.dtype == t.dtype and o.shape == t.shape
        want = t.double() * f
        lim = want.abs() * (2.0 ** -22 + torch.finfo(t.dtype).eps / 2) + torch.finfo(t.dtype).smallest_normal * \
            torch.finfo(t.dtype).eps
        assert ((o.double() - want).abs() <= lim).all()


LISTS = {"one": [1], "odd": [1, 7, 64, 63, 1023, 0, 8191, 8192, 8193], "empty tensors": [0, 0, 5, 0],
         "many": [(37 * i) % 300 + 1 for i in range(700)], "exactly a launch": [10] * 128, "a launch and one": [10] * 129,
         "large": [5_000_003, 12, 17_000_001], "mixed": [3_000_000, 1, 100_000, 20_000, 9]}


@pytest.mark.parametrize("name", LISTS)
@pytest.mark.parametrize("types", [(F32,), (BF16,), (F16,), (F32, BF16, F16)])
@pytest.mark.parametrize("p", [2.0, math.inf])
def test_norm_and_clip(name, types, p):
    ts = make(LISTS[name], types, seed=len(name))
    keep = [t.clone() for t in ts]
    check_norm(fh().grad_norm(ts, p), ts, p)
    ref = norm64(ts, p)
    for max_norm in (0.25 * ref, 3 * ref + 1, 0.0):
        out, norm = fh().clip_grads(ts, max_norm, p)
        check_norm(norm, ts, p)
        check_clipped(out, ts, ref, max_norm)
        if max_norm > ref:
            assert all(torch.equal(a, b) for a, b in zip(out, ts))
    assert all(torch.equal(a, b) for a, b in zip(ts, keep))
    got, norm = fh().clip_grads(ts, 0.5 * ref, p, out=ts)
    check_norm(norm, keep, p)
    check_clipped(ts, keep, ref, 0.5 * ref)


def test_magnitudes_outside_float32_squares():
    for mag in (1e25, 1e-30):
        ts = make([1000, 77], mag=mag)
        check_norm(fh().grad_norm(ts), ts)
    out, norm = fh().clip_grads(make([1000, 77], mag=1e25), 1.0)
    assert abs(math.sqrt(sum(float((o.double() ** 2).sum()) for o in out)) - 1) < 1e-5


@pytest.mark.parametrize("p", [2.0, math.inf])
@pytest.mark.parametrize("at", [0, 4000, 8999])
def test_nan_and_inf(p, at):
    ts = make([9000, 50])
    ts[0][at] = math.nan
    assert math.isnan(float(fh().grad_norm(ts, p)))
    out, norm = fh().clip_grads(ts, 1.0, p)
    assert math.isnan(float(norm)) and all(torch.isnan(o).all() for o in out)
    ts[0][at] = -math.inf
    assert float(fh().grad_norm(ts, p)) == math.inf
    out, norm = fh().clip_grads(ts, 1.0, p)
    want = [t * 0.0 for t in ts]  # the factor is 0, and infinity times 0 is NaN
    for o, w in zip(out, want):
        assert torch.equal(torch.isnan(o), torch.isnan(w)) and not o[~torch.isnan(o)].any()


def _params(shapes, types=(F32,), seed=1):
    ps = []
    g = torch.Generator().manual_seed(seed)
    for i, s in enumerate(shapes):
        p = torch.nn.Parameter(torch.zeros(s, device="cuda", dtype=types[i % len(types)]))
        p.grad = torch.randn(s, generator=g).to(p)
        ps.append(p)
    return ps


@pytest.mark.parametrize("types", [(F32,), (BF16, F32)])
@pytest.mark.parametrize("p", [2.0, math.inf])
def test_in_place_as_torch_does(types, p):
    shapes = [(64,), (128, 64, 1, 1), (), (1, 128, 7, 7), (3, 5)]
    ps = _params(shapes, types) + [torch.nn.Parameter(torch.zeros(4, device="cuda"))]  # the last has no gradient
    keep = [q.grad.clone() for q in ps[:-1]]
    ref = norm64(keep, p)
    norm = fh().clip_grad_norm_(ps, 0.5, p)
    check_norm(norm, keep, p)
    check_clipped([q.grad for q in ps[:-1]], keep, ref, 0.5)
    assert ps[-1].grad is None
    one = _params([(300,)])[0]
    g = one.grad.clone()
    check_norm(fh().clip_grad_norm_(one, 1.0), [g])  # one tensor
    check_norm(fh().clip_grad_norm_((q for q in _params([(300,)])), 1.0), [g])  # a generator
    assert float(fh().clip_grad_norm_([], 1.0)) == 0.0
    assert float(fh().clip_grad_norm_([torch.nn.Parameter(torch.zeros(3, device="cuda"))], 1.0)) == 0.0


def test_strides():
    ps = _params([(6, 8, 3, 3), (40, 50), (16,)])
    ps[0].grad = ps[0].grad.to(memory_format=torch.channels_last)
    ps[1].grad = torch.randn(50, 40, device="cuda").t()
    base = torch.randn(33, device="cuda")
    ps[2].grad = base[1::2]
    rest = base[::2].clone()
    keep = [q.grad.clone() for q in ps]
    addr = [q.grad.data_ptr() for q in ps]
    norm = fh().clip_grad_norm_(ps, 0.5)
    check_norm(norm, keep)
    check_clipped([q.grad for q in ps], keep, norm64(keep), 0.5)
    assert addr == [q.grad.data_ptr() for q in ps] and torch.equal(base[::2], rest)
    flat = torch.randn(5000, device="cuda", dtype=BF16)
    parts = [flat[1:2000], flat[2003:4999]]  # addresses that are multiples of 2 bytes only
    keep = [t.clone() for t in parts]
    check_norm(fh().grad_norm(parts), keep)
    out, _ = fh().clip_grads(parts, 0.5)
    check_clipped(out, keep, norm64(keep), 0.5)
    check_norm(fh().grad_norm([torch.ones(1, device="cuda").expand(100)]), [torch.ones(100)])


def test_version_counters():
    ps = _params([(10,), (4, 4)])
    w = torch.randn(10, device="cuda", requires_grad=True)
    y = (w * ps[0].grad).sum()  # keeps the gradient for its own backward
    fh().clip_grad_norm_(ps, 1e-3)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    with torch.inference_mode():
        t = torch.randn(10, device="cuda")
        fh().clip_grads([t], 0.5, out=[t])


def test_error_if_nonfinite_leaves_the_gradients():
    ps = _params([(10,), (4, 4)])
    ps[0].grad[3] = math.nan
    keep = [q.grad.clone() for q in ps]
    with pytest.raises(RuntimeError, match="norm of the gradients"):
        fh().clip_grad_norm_(ps, 1.0, error_if_nonfinite=True)
    for q, k in zip(ps, keep):
        assert torch.equal(torch.nan_to_num(q.grad), torch.nan_to_num(k))
    ps[0].grad[3] = 1.0
    fh().clip_grad_norm_(ps, 1.0, error_if_nonfinite=True)


def test_refusals():
    a, b = torch.ones(8, device="cuda"), torch.ones(8, device="cuda")
    F = fh()
    p = torch.nn.Parameter(torch.ones(8, device="cuda"))
    p.grad = torch.ones(1, device="cuda").expand(8)
    q = torch.nn.Parameter(torch.ones(8, device="cuda"))
    q.grad = torch.ones(8, device="cuda")
    for call in (lambda: F.grad_norm([a.double()]), lambda: F.grad_norm([a, b.cpu()]), lambda: F.grad_norm([a.cpu()]),
                 lambda: F.grad_norm([a], 1.0), lambda: F.clip_grads([a], -1.0), lambda: F.clip_grads([a], math.nan),
                 lambda: F.clip_grads([a, b], 1.0, out=[a]), lambda: F.clip_grads([a], 1.0, out=[b.half()]),
                 lambda: F.clip_grads([a], 1.0, out=[torch.ones(16, device="cuda")[::2]]),
                 lambda: F.clip_grads([a, b], 1.0, out=[b, a]), lambda: F.clip_grads([a, a], 1.0, out=[a, a]),
                 lambda: F.clip_grads([a, b], 1.0, out=[a, a]), lambda: F.clip_grad_norm_([q, q], 1.0),
                 lambda: F.clip_grad_norm_([p], 1.0), lambda: F.grad_norm([torch.eye(4, device="cuda").to_sparse()])):
        with pytest.raises(RuntimeError):
            call()
    flat = torch.ones(20, device="cuda")
    with pytest.raises(RuntimeError):
        F.clip_grads([flat[:10]], 1.0, out=[flat[5:15]])
    assert torch.equal(a, torch.ones_like(a)) and torch.equal(flat, torch.ones_like(flat))
    F.grad_norm([a, a])  # reading a tensor twice is no harm


def test_other_stream_and_recorded_graph():
    F = fh()
    ts = make([100_000, 33, 8192 * 3], (F32, BF16))
    out = [torch.empty_like(t) for t in ts]
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        norm = F.clip_grads(ts, 0.5, out=out)[1]
    torch.cuda.current_stream().wait_stream(st)
    check_norm(norm, ts)
    check_clipped(out, ts, norm64(ts), 0.5)
    graphs = []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            o, n = F.clip_grads(ts, 0.5 + i)
        graphs.append((g, o, n, 0.5 + i))
    for rep in range(3):
        for t, v in zip(ts, make([100_000, 33, 8192 * 3], (F32, BF16), seed=50 + rep)):
            t.copy_(v)
        ref = norm64(ts)
        for g, o, n, m in graphs:
            g.replay()
        torch.cuda.synchronize()
        for g, o, n, m in graphs:
            check_norm(n, ts)
            check_clipped(o, ts, ref, m)
        F.grad_norm(make([5_000_000]))


def test_beyond_32_bit_offsets():
    t = torch.zeros(2_200_000_000, dtype=BF16, device="cuda")
    t[-3] = 3.0
    t[5] = 4.0
    assert float(fh().grad_norm([t])) == 5.0
    _, norm = fh().clip_grads([t], 2.5, out=[t])
    assert float(norm) == 5.0 and abs(float(t[-3]) - 1.5) < 1e-2 and abs(float(t[5]) - 2.0) < 1e-2
