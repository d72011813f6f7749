"""Scaled residual and channels-first LayerNorms of a block (functional.residual_norm and its gradients), through the C
ABI, against the same in 64 bits.

Tolerances.  An output of type t is off by its own rounding, eps_t / 2 of its value, and by what float32 arithmetic
loses before, which `oracle` follows through the formulas to first order beside each value: U = 2^-24 of the result for
each operation, an error of an argument times the derivative, and C U <|v|> for a mean over C channels added up in any
order.  A sum over P pixels adds up tiles of at most 256 pixels, then a block's tiles, then the blocks in 64 bits: at
most (256 + P / 64) U of the sum of magnitudes, and the terms' own errors."""
import itertools

import pytest
import torch

pytestmark = pytest.mark.gpu
EPS = 1e-5
U = 2.0 ** -24
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _cf(t, d):
    return t.reshape((-1,) + (1,) * (d - 2))


def make(shape, tx=F32, th=F32, scale=True, gate=None, post=False, norm=True, branch=True, seed=0, pt=F32, offset=0.5):
    """Inputs on the CPU, of their types."""
    g = torch.Generator().manual_seed(seed)
    B, C = shape[:2]
    rn = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    a = {"x": (rn(*shape) + offset).to(tx)}
    if branch:
        a["h"] = rn(*shape).to(th)
    if scale and branch:
        a["s"] = (0.3 * rn(1, C, 1, 1)).to(pt)
    if gate:
        gs = {"full": shape, "sample": (B, C) + (1,) * (len(shape) - 2), "sample2": (B, C)}[gate]
        a["gate"] = torch.sigmoid(rn(*gs)).to(th)
    if post:
        a["pw"], a["pb"] = (1 + 0.2 * rn(C)).to(pt), (0.2 * rn(C)).to(pt)
    if norm:
        a["w"], a["b"] = (1 + 0.2 * rn(C)).to(pt), (0.2 * rn(C)).to(pt)
    a["gr"] = rn(*shape).to(tx)
    a["gy"] = rn(*shape).to(tx)
    return a


def _mean(v):
    return v.mean(1, keepdim=True)


def _standard(v, e, eps):
    """rhat, rho, and the errors of both for an error e of v (rho's relative)."""
    C = v.shape[1]
    u = _mean(v)
    d = v - u
    ed = e + _mean(e) + C * U * _mean(v.abs()) + U * d.abs()
    var = _mean(d * d) + eps
    rho = 1 / torch.sqrt(var)
    rel = _mean(d.abs() * ed) / var + (C / 2 + 5) * U
    hat = d * rho
    return hat, rho, rho * ed + hat.abs() * (rel + U), rel


def _standard_grad(g, eg, hat, ehat, rho, rel):
    """rho (g - <g> - hat <g hat>) and its error."""
    C = g.shape[1]
    s1, s2 = _mean(g), _mean(g * hat)
    es1 = _mean(eg) + (C + 1) * U * _mean(g.abs())
    es2 = _mean(eg * hat.abs() + g.abs() * ehat) + (C + 2) * U * _mean((g * hat).abs())
    v = rho * (g - s1 - hat * s2)
    e = rho * (eg + es1 + hat.abs() * es2 + ehat * s2.abs() + 3 * U * (g.abs() + s1.abs() + (hat * s2).abs()))
    return v, e + v.abs() * (rel + U)


def oracle(a, use_r=True, use_y=True, eps=EPS):
    """Outputs and gradients in 64 bits, and their tolerances before the outputs' own rounding."""
    d = {k: v.double() for k, v in a.items()}
    x = d["x"]
    nd, C = x.dim(), x.shape[1]
    val, tol = {}, {}
    one = torch.ones((), dtype=torch.float64)
    s = _cf(d["s"], nd) if "s" in d else one
    gate = one
    r, er = x, torch.zeros_like(x)
    if "h" in d:
        n, en = d["h"], torch.zeros_like(x)
        if "pw" in d:
            phat, prho, ephat, prel = _standard(n, en, eps)
            pw = _cf(d["pw"], nd)
            n = phat * pw + _cf(d["pb"], nd)
            en = ephat * pw.abs() + 2 * U * ((phat * pw).abs() + n.abs())
        if "gate" in d:
            gate = d["gate"] if d["gate"].shape == x.shape else d["gate"].reshape(d["gate"].shape[:2] + (1,) * (nd - 2))
        r = x + s * gate * n
        er = (s * gate).abs() * (en + 2 * U * n.abs()) + U * r.abs()
        val["r"], tol["r"] = r, er
    if "w" in d:
        w, b = _cf(d["w"], nd), _cf(d["b"], nd)
        rhat, rho, ehat, rel = _standard(r, er, eps)
        val["y"] = rhat * w + b
        tol["y"] = ehat * w.abs() + 2 * U * ((rhat * w).abs() + val["y"].abs())
    gr = d["gr"] if use_r and "h" in d else torch.zeros_like(x)
    gy = d["gy"] if use_y and "w" in d else torch.zeros_like(x)
    dr, edr = gr, torch.zeros_like(x)
    sums = {}
    if "w" in d:
        if a["x"].dtype == F32 and "h" in d:
            ehat = ehat + rho * U * r.abs()  # the backward reads r as it was stored
        dr, edr = _standard_grad(gy * w, U * (gy * w).abs(), rhat, ehat, rho, rel)
        dr = dr + gr
        edr = edr + 2 * U * (gr.abs() + dr.abs())
        sums["w"] = (gy * rhat, gy.abs() * ehat + U * (gy * rhat).abs())
        sums["b"] = (gy, torch.zeros_like(gy))
    val["dx"], tol["dx"] = dr, edr
    pix = [0] + list(range(2, nd))
    hw = x[0, 0].numel() if x.shape[0] else 0
    P = x.shape[0] * hw
    if "h" in d:
        dn, edn = dr * s * gate, (s * gate).abs() * (edr + 2 * U * dr.abs())
        if "s" in d:
            sums["s"] = (dr * gate * n, (gate * n).abs() * (edr + 3 * U * dr.abs()) + (dr * gate).abs() * en)
        if "gate" in d:
            dg = dr * s * n
            edg = (s * n).abs() * (edr + 2 * U * dr.abs()) + (dr * s).abs() * en
            if d["gate"].shape == x.shape:
                val["dgate"], tol["dgate"] = dg, edg
            else:
                k = list(range(2, nd))
                edg = edg + U * min(256, hw) * dg.abs()  # a tile's pixels; the tiles in 64 bits
                val["dgate"] = (dg.sum(k) if k else dg).reshape(d["gate"].shape)
                tol["dgate"] = (edg.sum(k) if k else edg).reshape(d["gate"].shape)
        if "pw" in d:
            dh, edh = _standard_grad(dn * pw, edn * pw.abs() + U * (dn * pw).abs(), phat, ephat, prho, prel)
            sums["pw"] = (dn * phat, edn * phat.abs() + dn.abs() * ephat + U * (dn * phat).abs())
            sums["pb"] = (dn, edn)
        else:
            dh, edh = dn, edn
        val["dh"], tol["dh"] = dh, edh
    for k, (t, e) in sums.items():
        val["d" + k] = t.sum(pix)
        tol["d" + k] = (256 + P / 64) * U * t.abs().sum(pix) + e.sum(pix)
    return val, tol


def _dev(a, keys=("x", "h", "gate", "s", "pw", "pb", "w", "b")):
    return {k: v.cuda().requires_grad_(k in keys) for k, v in a.items()}


def call(d, train=True, eps=EPS):
    from conversenet_amd import functional as Fh

    norm = (d["w"], d["b"], eps) if "w" in d else None
    if "h" not in d:
        return {"y": Fh.layernorm_cf_train(d["x"], *norm)}
    post = (d["pw"], d["pb"], eps) if "pw" in d else None
    f = Fh.residual_norm_train if train else Fh.residual_norm
    r, y = f(d["x"], d["h"], norm=norm, res_scale=d.get("s"), gate=d.get("gate"), post=post)
    return {"r": r, "y": y} if y is not None else {"r": r}


def grads(d, out, use_r=True, use_y=True):
    pairs = [(out[k], d["g" + k]) for k, use in (("r", use_r), ("y", use_y)) if k in out and use]
    leaves = [k for k in ("x", "h", "gate", "s", "pw", "pb", "w", "b") if k in d and d[k].requires_grad]
    got = torch.autograd.grad([p[0] for p in pairs], [d[k] for k in leaves], [p[1] for p in pairs], allow_unused=True)
    return {"d" + k: g for k, g in zip(leaves, got)}


def compare(got, val, tol, what):
    for k, g in got.items():
        if g is None:
            assert not val[k].abs().any(), (what, k, "no gradient")
            continue
        ref = val[k].reshape(g.shape)
        err = (g.detach().double().cpu() - ref).abs()
        lim = ref.abs() * (torch.finfo(g.dtype).eps / 2) * 1.001 + tol[k].reshape(g.shape) + torch.finfo(g.dtype).tiny * \
            torch.finfo(g.dtype).eps
        assert torch.isfinite(g).all(), (what, k)
        assert (err <= lim).all(), (what, k, float(err.max()), float((err / lim).max()))


def check(a, use_r=True, use_y=True, what=""):
    val, tol = oracle(a, use_r, use_y)
    d = _dev(a)
    out = call(d)
    compare(out, val, tol, what)
    compare(grads(d, out, use_r, use_y), val, tol, what)
    return d, out


SHAPES = [(1, 64, 1, 1), (1, 1, 5, 7), (2, 3, 9, 11), (2, 64, 32, 40), (1, 64, 37, 53), (3, 48, 5, 5), (70, 8, 1, 1),
          (2, 128, 17, 16), (1, 100, 33, 32), (2, 200, 12, 13), (1, 256, 20, 20), (1, 257, 9, 9), (1, 600, 8, 33),
          (5, 16, 40, 30), (1, 65, 64, 64)]
WIDE = [(3, 512, 1, 1), (70, 300, 1, 1), (2, 1040, 3, 5), (1, 2000, 1, 2), (1, 272, 30, 40)]
TYPES = [(F32, F32), (BF16, BF16), (F16, F16), (F32, BF16), (F32, F16)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("gate,post", [(None, False), ("full", True), ("sample", True), ("sample", False)])
def test_shapes_f32(shape, gate, post):
    check(make(shape, gate=gate, post=post, seed=sum(shape)), what=str(shape))


@pytest.mark.parametrize("shape", WIDE)
@pytest.mark.parametrize("tx,th", TYPES)
@pytest.mark.parametrize("scale,gate,post", [(True, None, False), (False, "full", True), (True, "sample", True)])
def test_many_channels(shape, tx, th, scale, gate, post):
    check(make(shape, tx, th, scale, gate, post, seed=sum(shape)), what=str((shape, tx, th)))


@pytest.mark.parametrize("shape,gate", [((5, 128, 96, 96), "sample"), ((2, 200, 100, 100), None), ((2, 192, 101, 99), "full"),
                                        ((2, 100, 100, 100), "sample"), ((1, 300, 130, 130), "full")])
def test_several_tiles_a_block(shape, gate):
    """More tiles than blocks of the backward, of each kernel: the sums go on from tile to tile."""
    check(make(shape, gate=gate, post=True, seed=sum(shape)), what=str(shape))


@pytest.mark.parametrize("shape", [(1, 64, 1, 1), (2, 64, 33, 31), (2, 128, 16, 24), (1, 300, 7, 10), (3, 20, 64, 64)])
@pytest.mark.parametrize("tx,th", TYPES[1:])
@pytest.mark.parametrize("scale,gate,post", [(True, None, False), (False, None, False), (True, "full", True),
                                             (False, "sample", True), (True, "full", False)])
def test_types(shape, tx, th, scale, gate, post):
    check(make(shape, tx, th, scale, gate, post, seed=sum(shape)), what=str((shape, tx, th)))


@pytest.mark.parametrize("scale,gate,post,norm", [c for c in itertools.product((False, True), (None, "full", "sample2"),
                                                                               (False, True), (False, True))])
def test_every_combination(scale, gate, post, norm):
    check(make((2, 24, 13, 12), scale=scale, gate=gate, post=post, norm=norm, seed=3))


@pytest.mark.parametrize("tx", [F32, BF16, F16])
@pytest.mark.parametrize("shape", [(2, 64, 24, 20), (1, 3, 50, 50), (4, 130, 7, 7), (2, 8), (3, 16, 100)])
def test_layernorm_alone(tx, shape):
    check(make(shape, tx, tx, branch=False, seed=1))


@pytest.mark.parametrize("tx,th", TYPES)
@pytest.mark.parametrize("use_r,use_y", [(True, False), (False, True)])
@pytest.mark.parametrize("plain", [True, False])
def test_one_output_used(tx, th, use_r, use_y, plain):
    check(make((2, 32, 15, 18), tx, th, scale=not plain, gate=None if plain else "sample", post=not plain, seed=5), use_r,
          use_y)


@pytest.mark.parametrize("keys", [("x",), ("h",), ("s",), ("gate",), ("pw", "pb"), ("w",), ("b",), ("h", "b")])
def test_some_gradients_wanted(keys):
    a = make((2, 40, 18, 18), gate="full", post=True, seed=8)
    val, tol = oracle(a)
    d = _dev(a, keys)
    compare(grads(d, call(d)), val, tol, keys)


def test_parameters_of_16_bits():
    a = make((2, 64, 16, 18), BF16, BF16, gate="full", post=True, pt=BF16, seed=2)
    d, out = check(a)
    g = grads(d, call(d))
    assert g["dw"].dtype == BF16 and g["ds"].shape == (1, 64, 1, 1)


def test_parameters_of_other_shapes():
    a = make((2, 24, 9, 7), gate="sample", post=True, seed=21)
    shapes = {"w": (24, 1, 1), "b": (1, 24, 1, 1), "pw": (24,), "pb": (24, 1), "s": (24,)}
    val, tol = oracle(a)
    wide = torch.zeros(48, device="cuda")
    d = {k: v.cuda().reshape(shapes.get(k, v.shape)).clone() for k, v in a.items()}
    wide[::2] = d["pw"]
    d["pw"] = wide[::2]  # strided
    for k in ("x", "h", "gate", "s", "pw", "pb", "w", "b"):
        d[k].requires_grad_(True)
    out = call(d)
    compare(out, val, tol, "shapes")
    g = grads(d, out)
    compare(g, val, tol, "shapes")
    assert all(g["d" + k].shape == d[k].shape for k in shapes)
    g = grads(d, call(d), use_y=False)  # y unused: zeros of each parameter's shape, or none
    assert all(g["d" + k] is None or g["d" + k].shape == d[k].shape for k in shapes)


@pytest.mark.parametrize("tx,th", TYPES)
def test_forward_alone_is_the_same(tx, th):
    a = make((2, 64, 20, 22), tx, th, gate="full", post=True, seed=4)
    d = _dev(a)
    out = call(d)
    with torch.no_grad():
        alone = call(d, train=False)
    for k in out:
        assert torch.equal(out[k], alone[k])


def test_repeats_bit_for_bit():
    d = _dev(make((4, 64, 60, 61), gate="sample", post=True, seed=6))
    g0 = grads(d, call(d))
    for _ in range(3):
        g = grads(d, call(d))
        assert all(torch.equal(g[k], g0[k]) for k in g0)


def _expand(v):
    """The same values behind strides and an odd address."""
    big = torch.zeros(v.numel() + 3, dtype=v.dtype, device=v.device)
    flat = big[3:].view(v.shape[0], *v.shape[2:], v.shape[1])
    t = flat.movedim(-1, 1)  # channels last
    t.copy_(v)
    return t


def test_strides_and_alignment():
    a = make((2, 64, 13, 15), gate="full", post=True, seed=9)
    val, tol = oracle(a)
    d = {k: (_expand(v.cuda()) if v.dim() == 4 and k != "s" else v.cuda()).requires_grad_(k not in ("gr", "gy"))
         for k, v in a.items()}
    out = call(d)
    compare(out, val, tol, "strides")
    compare(grads(d, out), val, tol, "strides")
    # contiguous, at an address that is only a multiple of the type's size
    for shape, t in (((2, 64, 16, 16), F32), ((2, 64, 16, 16), BF16), ((1, 16, 64, 64), F16)):
        a = make(shape, t, t, gate="full", post=True, seed=9)
        val, tol = oracle(a)

        def odd(v):
            big = torch.zeros(v.numel() + 1, dtype=v.dtype, device="cuda")
            big[1:].copy_(v.flatten())
            return big[1:].view(v.shape)

        d = {k: odd(v.cuda()).requires_grad_(k not in ("gr", "gy")) for k, v in a.items()}
        out = call(d)
        compare(out, val, tol, "alignment")
        compare(grads(d, out), val, tol, "alignment")


@pytest.mark.parametrize("shape", [(3, 37, 40, 40), (3, 65, 7, 9), (5, 8, 33, 33), (2, 257, 6, 5), (3, 131, 33, 32)])
@pytest.mark.parametrize("tx,th", [(BF16, BF16), (F32, F16)])
def test_sample_gates_at_any_address(shape, tx, th):
    """16-bit gates of samples that start at multiples of 2 bytes only."""
    a = make(shape, tx, th, gate="sample", post=True, seed=sum(shape))
    val, tol = oracle(a)
    d = _dev(a)
    big = torch.zeros(a["gate"].numel() + 1, dtype=th, device="cuda")
    big[1:].copy_(a["gate"].flatten())
    d["gate"] = big[1:].view(a["gate"].shape).requires_grad_(True)
    out = call(d)
    compare(out, val, tol, "gates")
    compare(grads(d, out), val, tol, "gates")


def test_expanded_gradient_and_input():
    a = make((2, 32, 12, 12), seed=10)
    a["h"] = a["h"][:, :, :1, :1].expand(2, 32, 12, 12)
    a["gy"] = a["gy"][:1, :1, :1, :1].expand(2, 32, 12, 12)
    val, tol = oracle(a)
    d = {k: v.cuda() if k in ("gy",) else v.cuda().requires_grad_(k != "gr") for k, v in a.items()}
    d["gy"] = d["gy"][:1, :1, :1, :1].expand(2, 32, 12, 12)
    out = call(d)
    compare(out, val, tol, "expanded")
    compare(grads(d, out), val, tol, "expanded")


@pytest.mark.parametrize("shape", [(0, 64, 8, 8), (2, 64, 0, 8), (0, 8)])
def test_empty(shape):
    d = _dev(make(shape, gate="sample", post=True))
    out = call(d)
    assert out["r"].shape == shape and out["y"].shape == shape
    g = grads(d, out)
    assert g["dx"].shape == shape and g["dgate"].shape == d["gate"].shape
    for k in ("ds", "dw", "db", "dpw", "dpb", "dgate"):
        assert not g[k].any()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("shape", [(2, 64, 24, 24), (1, 300, 10, 10)])
def test_a_bad_pixel_stays_one(bad, shape):
    a = make(shape, gate="full", post=True, seed=11)
    a["x"][0, 5, 3, 4] = bad
    a["h"][0, 7, 6, 1] = bad
    clean = make(shape, gate="full", post=True, seed=11)
    d, c = _dev(a), _dev(clean)
    out, ref = call(d), call(c)
    g, gref = grads(d, out), grads(c, ref)
    ok = torch.ones(shape[0], 1, *shape[2:], dtype=torch.bool, device="cuda").expand(shape).clone()
    ok[0, :, 3, 4] = ok[0, :, 6, 1] = False
    for t, u in ((out["r"], ref["r"]), (out["y"], ref["y"]), (g["dx"], gref["dx"]), (g["dh"], gref["dh"]),
                 (g["dgate"], gref["dgate"])):
        assert torch.equal(t[ok], u[ok])
    assert not torch.isfinite(out["y"][0, :, 3, 4]).any() and not torch.isfinite(out["y"][0, :, 6, 1]).any()
    assert not torch.isfinite(g["dw"]).any()


def test_constant_pixels():
    """No spread over the channels: y is the bias, and rho is 1 / sqrt(eps)."""
    a = make((1, 64, 8, 8), scale=False, seed=12)
    a["x"][:] = 2.0
    a["h"][:] = 0.5
    val, tol = oracle(a)
    d = _dev(a)
    out = call(d)
    compare(out, val, tol, "constant")
    compare(grads(d, out), val, tol, "constant")
    assert torch.equal(out["y"], d["b"].detach().view(1, -1, 1, 1).expand_as(out["y"]))


def test_large_mean():
    """A mean of 1000 deviations: two-pass moments, within the bound that the values' size gives."""
    check(make((2, 64, 16, 16), offset=1000.0, seed=13))


def test_gradients_against_differences():
    """Central differences of the 64-bit forward along random directions, for every argument."""
    a = make((2, 16, 6, 7), gate="full", post=True, seed=14)
    d = _dev(a)
    g = grads(d, call(d))
    gen = torch.Generator().manual_seed(1)

    def loss(b):
        v, _ = oracle(b)
        return (v["r"] * a["gr"].double()).sum() + (v["y"] * a["gy"].double()).sum()

    for k in ("x", "h", "gate", "s", "pw", "pb", "w", "b"):
        e = torch.randn(a[k].shape, generator=gen).double()
        h = 1e-5
        diff = (loss({**a, k: a[k].double() + h * e}) - loss({**a, k: a[k].double() - h * e})) / (2 * h)
        got = (g["d" + k].double().cpu() * e).sum()
        # third derivatives times h^2, rounding of the loss (2^-53 of ~1e3) over h, float32 gradients
        assert abs(float(got - diff)) <= 1e-5 * float((g["d" + k].double().cpu() * e).abs().sum()) + 1e-6, k


@pytest.mark.parametrize("strided", [False, True])
@pytest.mark.parametrize("tx,th,plain", [(F32, F32, False), (F32, F32, True), (F32, BF16, False), (BF16, BF16, False)])
def test_backward_is_differentiable(tx, th, plain, strided):
    """A gradient penalty: gradients of gradients, against the same composition in 64 bits."""
    from conversenet_amd import composite

    a = make((2, 12, 5, 6), tx, th, scale=not plain, gate=None if plain else "full", post=not plain, seed=15)
    keys = [k for k in ("x", "h", "gate", "s", "pw", "pb", "w", "b") if k in a]

    def penalty(d, r, y):
        g = torch.autograd.grad((r, y), [d[k] for k in ("x", "h", "w")], (d["gr"], d["gy"]), create_graph=True)
        return sum((t.double() ** 2).sum() for t in g)

    d = {k: (_expand(v.cuda()) if strided and v.dim() == 4 and k != "s" else v.cuda()).requires_grad_(k in keys)
         for k, v in a.items()}
    out = call(d)
    got = torch.autograd.grad(penalty(d, out["r"], out["y"]), [d[k] for k in keys], allow_unused=True)
    c = {k: v.double().requires_grad_(k in keys) for k, v in a.items()}
    post = None if plain else (c["pw"], c["pb"], EPS)
    r = c["x"] + composite.residual_branch(c["h"], c.get("s"), c.get("gate"), post)
    y = composite.standardised(r, EPS)[0] * _cf(c["w"], 4) + _cf(c["b"], 4)
    ref = torch.autograd.grad(penalty(c, r, y), [c[k] for k in keys], allow_unused=True)
    # first gradients rounded to 16 bits enter the penalty's own gradient: a relative 2^-8 of its terms
    rel = 1e-4 if tx == th == F32 else 2.0 ** -5
    for k, g, w in zip(keys, got, ref):
        if w is None or not w.abs().any():
            assert g is None or float(g.abs().max()) <= rel
            continue
        assert float((g.double().cpu() - w).norm()) <= rel * float(w.norm()), (k, tx, th)


@pytest.mark.parametrize("tx,th,gate,plain", [(F32, F32, "full", False), (BF16, BF16, "sample", False), (F32, F32, None, True),
                                              (F32, F16, "sample2", False)])
def test_composed_backward_is_the_same(tx, th, gate, plain):
    """The composition a differentiated backward runs: within the kernels' bounds too."""
    a = make((2, 24, 9, 8), tx, th, not plain, gate, not plain, seed=17)
    val, tol = oracle(a)
    d = _dev(a)
    out = call(d)
    keys = [k for k in ("x", "h", "gate", "s", "pw", "pb", "w", "b") if k in d]
    g = torch.autograd.grad((out["r"], out["y"]), [d[k] for k in keys], (d["gr"], d["gy"]), create_graph=True)
    compare({"d" + k: v for k, v in zip(keys, g)}, val, tol, "composed")


def test_many_gradients_at_once():
    a = make((2, 12, 4, 5), gate="full", post=True, seed=18)
    d = _dev(a)
    out = call(d)
    keys = ("x", "h", "gate", "s", "pw", "pb", "w", "b")
    many = [torch.stack([t, 2 * t, -t]) for t in (d["gr"], d["gy"])]
    got = torch.autograd.grad((out["r"], out["y"]), [d[k] for k in keys], many, is_grads_batched=True)
    want = grads(d, call(d))
    for k, g in zip(keys, got):
        w = want["d" + k]
        for i, f in enumerate((1, 2, -1)):
            assert float((g[i] - f * w).norm()) <= 2e-6 * float(w.norm()) + 1e-12


@pytest.mark.parametrize("scale", [False, True])
def test_one_tensor_as_stream_and_branch(scale):
    a = make((2, 16, 9, 9), scale=scale, seed=19)
    a["h"] = a["x"]
    val, tol = oracle(a)
    d = _dev(a)
    d["h"] = d["x"]
    out = call(d)
    compare(out, val, tol, "shared")
    g, = torch.autograd.grad((out["r"], out["y"]), (d["x"],), (d["gr"], d["gy"]))
    compare({"dx": g}, {"dx": val["dx"] + val["dh"]}, {"dx": tol["dx"] + tol["dh"] + 2 * U * val["dx"].abs()}, "shared")


def test_threads_on_one_stream():
    """Passes of four threads at once, on the stream they share: each as alone."""
    import threading

    from conversenet_amd import functional as Fh

    sets = [_dev(make((2, 64, 40, 41 + i), gate="sample", post=True, seed=60 + i)) for i in range(4)]
    want = [grads(d, call(d)) for d in sets]
    norms = [float(Fh.grad_norm(list(w.values()))) for w in want]
    bad = []

    def work(i):
        for _ in range(8):
            g = grads(sets[i], call(sets[i]))
            n = float(Fh.grad_norm(list(g.values())))
            if n != norms[i] or not all(torch.equal(g[k], want[i][k]) for k in g):
                bad.append(i)

    ts = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    assert not bad


def test_other_stream():
    a = make((2, 64, 40, 40), gate="sample", post=True, seed=16)
    val, tol = oracle(a)
    d = _dev(a)
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        out = call(d)
        g = grads(d, out)
    torch.cuda.current_stream().wait_stream(st)
    compare(out, val, tol, "stream")
    compare(g, val, tol, "stream")


def test_recorded_graphs():
    """Two graphs with forward and backward, replayed in turn with eager work between: no workspace is shared."""
    from conversenet_amd import functional as Fh

    sets, graphs, outs = [], [], []
    st = torch.cuda.Stream()

    def step(d):
        r, y, stats = Fh.residual_norm_stats(d["x"], d["h"], (d["w"], d["b"], EPS), d["s"], d["gate"],
                                             (d["pw"], d["pb"], EPS))
        return (r, y) + Fh.residual_norm_backward(d["gr"], d["gy"], r, d["h"], stats, d["w"], d["s"], d["gate"],
                                                  (d["pw"], d["pb"], EPS))

    for i, shape in enumerate(((2, 64, 24, 24), (1, 64, 65, 40))):
        d = {k: v.cuda() for k, v in make(shape, gate="sample", post=True, seed=20 + i).items()}
        sets.append(d)
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            step(d)
        st.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            outs.append(step(d))
        graphs.append(g)
    for rep in range(3):
        for i, d in enumerate(sets):
            for k, v in make(tuple(d["x"].shape), gate="sample", post=True, seed=100 + 10 * rep + i).items():
                d[k].copy_(v)
            want = step(d)
            torch.cuda.synchronize()
            graphs[i].replay()
            graphs[1 - i].replay()
            torch.cuda.synchronize()
            for t, u in zip(outs[i], want):
                assert torch.equal(t, u)


def test_recorded_training_pass():
    """Forward and autograd's backward in one graph, replayed on new inputs against eager passes on leaves of their own."""
    shape = (2, 64, 20, 30)
    d = _dev(make(shape, gate="full", post=True, seed=30))
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        for _ in range(2):
            grads(d, call(d))  # nothing of these passes is kept
    torch.cuda.current_stream().wait_stream(st)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        out = call(d)
        got = grads(d, out)
    for rep in range(3):
        new = make(shape, gate="full", post=True, seed=40 + rep)
        with torch.no_grad():
            for k, v in new.items():
                d[k].copy_(v)
        e = _dev(new)
        eout = call(e)
        want = grads(e, eout)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        for k in out:
            assert torch.equal(out[k], eout[k])
        for k in want:
            assert torch.equal(got[k], want[k])


def test_offsets_beyond_32_bits():
    """2.3e9 elements: each sample's pixels are what a call on that part alone gives."""
    from conversenet_amd import functional as Fh

    B, C, H, W = 3, 48, 4000, 4000
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(B, C, H, W, device="cuda", dtype=BF16, generator=g)
    h = torch.randn(B, C, H, W, device="cuda", dtype=BF16, generator=g)
    w, b = torch.randn(2, C, device="cuda", generator=g)
    s = torch.randn(C, device="cuda", generator=g)
    args = dict(norm=(w, b, EPS), res_scale=s)
    r, y = Fh.residual_norm(x, h, **args)
    rows = slice(H - 40, H)
    for i in (0, B - 1):
        rr, yy = Fh.residual_norm(x[i:i + 1, :, rows].contiguous(), h[i:i + 1, :, rows].contiguous(), **args)
        assert torch.equal(r[i:i + 1, :, rows], rr) and torch.equal(y[i:i + 1, :, rows], yy)
    del r, y
    x.requires_grad_(True)
    h.requires_grad_(True)
    r, y = Fh.residual_norm_train(x, h, **args)
    gx, gh = torch.autograd.grad(y, (x, h), y.detach())
    xs, hs = (t.detach()[B - 1:, :, rows].contiguous().requires_grad_(True) for t in (x, h))
    rr, yy = Fh.residual_norm_train(xs, hs, **args)
    gxs, ghs = torch.autograd.grad(yy, (xs, hs), yy.detach())
    assert torch.equal(gx[B - 1:, :, rows], gxs) and torch.equal(gh[B - 1:, :, rows], ghs)


def test_refusals_on_the_device():
    from conversenet_amd import functional as Fh

    x = torch.zeros(2, 8, 4, 4, device="cuda")
    w = torch.ones(8, device="cuda")
    norm = (w, w, EPS)
    for kw in (dict(h=None), dict(h=x[:, :4]), dict(h=x.double()), dict(h=x, gate=x[:, :1]), dict(h=x, gate=x.half()),
               dict(h=x, res_scale=w[:4]), dict(h=x, post=(w[:4], w, EPS)), dict(h=x, res_scale=w.cpu()),
               dict(h=x.cpu())):
        with pytest.raises(RuntimeError):
            Fh.residual_norm(x, norm=norm, **kw)
    with pytest.raises(RuntimeError):
        Fh.residual_norm(x.half(), x)
    with pytest.raises(RuntimeError):
        Fh.residual_norm(x, x, norm=(w.double(), w, EPS))
    with pytest.raises(RuntimeError):
        Fh.layernorm_cf_train(torch.zeros(8, device="cuda"), w, w, EPS)


@pytest.mark.parametrize("shape", [(2, 64, 33, 32), (2, 64, 37, 53), (1, 128, 41, 43)])
@pytest.mark.parametrize("tx,th", TYPES)
@pytest.mark.parametrize("scale,gate,post", [(True, None, False), (True, "full", True), (False, "sample", True),
                                             (False, "full", False)])
def test_two_pixels_a_lane_with_a_rest(shape, tx, th, scale, gate, post):
    """1024 pixels and more of 8 n channels, the last tile not a whole one."""
    check(make(shape, tx, th, scale, gate, post, seed=sum(shape)), what=str((shape, tx, th)))


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("tx,th", [(F32, F32), (BF16, BF16), (F32, F16)])
@pytest.mark.parametrize("shape", [(2, 64, 33, 33), (2, 128, 45, 25), (2, 20, 33, 33), (2, 300, 33, 33)])
def test_bad_pixels_at_a_samples_end(bad, tx, th, shape):
    """The last pixels of a sample, which two lanes read where their number is odd."""
    H, W = shape[2:]
    for x_at, h_at in ((W - 1, W - 2), (W - 2, W - 1)):
        a, clean = (make(shape, tx, th, gate="full", post=True, seed=12) for _ in range(2))
        a["x"][0, 5, H - 1, x_at] = bad
        a["h"][0, 7, H - 1, h_at] = bad
        d, c = _dev(a), _dev(clean)
        out, ref = call(d), call(c)
        g, gref = grads(d, out), grads(c, ref)
        ok = torch.ones(shape[0], 1, *shape[2:], dtype=torch.bool, device="cuda").expand(shape).clone()
        ok[0, :, H - 1, W - 2:] = False
        for t, u in ((out["r"], ref["r"]), (out["y"], ref["y"]), (g["dx"], gref["dx"]), (g["dh"], gref["dh"]),
                     (g["dgate"], gref["dgate"])):
            assert torch.equal(t[ok], u[ok])
        assert not torch.isfinite(out["y"][0, :, H - 1, W - 2:]).any() and not torch.isfinite(g["dw"]).any()


@pytest.mark.parametrize("C", [64, 256, 272, 512, 1040])
@pytest.mark.parametrize("t", [F32, BF16])
def test_means_beyond_the_root_of_float32(C, t):
    """Values of 2^65, whose squares no float32 holds, without a spread and with one of 2^45 (2^58 in bfloat16: 1040
    squares are below 2^127) about them.  Their means are exact in any order: sums of up to 2^11 equal values or pairs."""
    from conversenet_amd import functional as Fh

    big, step = 2.0 ** 65, 2.0 ** (45 if t == F32 else 58)
    a = make((2, C, 5, 7), t, t, scale=False, seed=C)
    w, b = a["w"].cuda(), a["b"].cuda()
    cf = (1, -1, 1, 1)
    x = torch.full((2, C, 5, 7), big, dtype=t, device="cuda").requires_grad_(True)
    y = Fh.layernorm_cf_train(x, w, b, EPS)
    assert torch.equal(y.detach(), b.view(cf).to(t).expand_as(y))
    gx, = torch.autograd.grad(y, x, a["gy"].cuda())
    gw = a["gy"].double() * a["w"].double().view(cf)
    want = (gw - _mean(gw)) / EPS ** 0.5
    # a product, a mean over C channels, a difference, and the deviation: 1 / sqrt(eps) of a rounded eps
    lim = (gw.abs() + (C + 1) * _mean(gw.abs())) / EPS ** 0.5 * 8 * U + want.abs() * torch.finfo(t).eps / 2 * 1.001
    assert ((gx.double().cpu() - want).abs() <= lim).all()
    sign = (1 - 2 * (torch.arange(C) % 2)).double().view(cf)
    x = (big + sign * step).to(t).expand(2, C, 5, 7).cuda()
    assert torch.equal(x.double().cpu(), (big + sign * step).expand(2, C, 5, 7))
    want = sign * a["w"].double().view(cf) + a["b"].double().view(cf)
    y = Fh.residual_norm(torch.zeros_like(x), x, (w, b, EPS))[1]  # a branch on nothing
    post = Fh.residual_norm(torch.zeros_like(x), x, None, post=(w, b, EPS))[0]  # and its own norm
    lim = 4 * U * (a["w"].abs() + a["b"].abs()).double().view(cf) + want.abs() * torch.finfo(t).eps / 2 * 1.001
    for got in (y, post):
        assert ((got.double().cpu() - want).abs() <= lim).all()


@pytest.mark.parametrize("shape", [(1024, 65536, 1), (1 << 20, 64, 2)])
def test_many_gates_of_samples(shape):
    """2^26 gates and more: a wave for each is more threads than one launch holds."""
    from conversenet_amd import functional as Fh

    B, C, n = shape
    g = torch.Generator(device="cuda").manual_seed(4)
    x, h, gr = (torch.randn(shape, device="cuda", generator=g).requires_grad_(i < 2) for i in range(3))
    gate = torch.rand(B, C, device="cuda", generator=g).requires_grad_(True)
    s = torch.randn(C, device="cuda", generator=g).requires_grad_(True)
    r, _ = Fh.residual_norm_train(x, h, None, s, gate)
    gx, gh, gg, gs = torch.autograd.grad(r, (x, h, gate, s), gr)
    assert torch.equal(gx, gr)
    for part in (slice(0, 64), slice(B // 2, B // 2 + 64), slice(B - 64, B)):
        hp, dp, gp, sp = h[part].double(), gr[part].double(), gate[part].double()[..., None], s.double()[:, None]
        want = x[part].double() + sp * gp * hp
        assert ((r[part].double() - want).abs() <= 3 * U * ((sp * gp * hp).abs() + want.abs())).all()
        want = sp * gp * dp
        assert ((gh[part].double() - want).abs() <= 3 * U * want.abs()).all()
        terms = dp * hp * sp
        assert ((gg[part].double() - terms.sum(2)).abs() <= 4 * U * terms.abs().sum(2)).all()
    want, size = torch.zeros(2, C, dtype=torch.float64, device="cuda")
    for part in range(0, B, B // 8):
        terms = (gr[part:part + B // 8] * h[part:part + B // 8].double() * gate[part:part + B // 8, :, None]).detach()
        want += terms.sum((0, 2))
        size += terms.abs().sum((0, 2))
    P = B * n
    assert ((gs.double() - want).abs() <= (256 + P / 64) * U * size).all()


def test_more_tiles_than_one_launch_holds():
    """1.45e9 pixels of 33 channels, 3 waves a tile: as many launches as they take, on either side of whose border (and at
    both ends) pixels are what a call on them alone gives."""
    from conversenet_amd import _lib, functional as Fh

    C, n = 33, 1_450_000_000
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 2 * 2 * C * n + (8 << 30):
        pytest.skip("needs 200 GB of device memory")
    w, b = torch.randn(2, C, device="cuda")
    border = ((1 << 32) - 1) // 192 // 64 * 64 * 64
    assert 4096 < border < n - 4096
    try:
        x, y = (torch.empty(1, C, n, dtype=BF16, device="cuda") for _ in range(2))
        parts = [slice(0, 2048), slice(border - 2048, border + 2048), slice(n - 2048, n)]
        for p in parts:
            x[:, :, p] = torch.randn(1, C, p.stop - p.start, device="cuda")
            y[:, :, p] = 7.0
        rc = _lib.load().cvn_residual_norm_fwd(
            x.data_ptr(), _lib.TYPES[BF16], None, _lib.TYPES[BF16], 1, C, n, None, None, 0, None, None, 0.0, w.data_ptr(),
            b.data_ptr(), EPS, None, y.data_ptr(), None, torch.cuda.current_stream().cuda_stream)
        _lib.check(rc, "residual_norm")
        for p in parts:
            part = x[:, :, p].contiguous().requires_grad_(True)
            assert torch.equal(y[:, :, p], Fh.layernorm_cf_train(part, w, b, EPS))
    finally:
        x = y = part = None
        torch.cuda.empty_cache()


@pytest.mark.parametrize("C,H,W", [(64, 4096, 4096), (128, 2048, 4096), (200, 2048, 2048), (272, 2048, 2048)])
def test_sums_over_many_pixels(C, H, W):
    """The parameters' gradients of a map of equal pixels are those of 1024 of its pixels times a whole number: tiles of
    equal sums, which 64 bits add up exactly, so that either is off by at most two roundings, of a block's sum and of the
    gradient.  (In 32 bits a block's sum loses up to half a step a tile, always to one side.)"""
    from conversenet_amd import functional as Fh

    g = torch.Generator().manual_seed(C)
    row = {k: torch.randn(1, C, 1, 1, generator=g).cuda() for k in ("x", "h", "gate", "gr", "gy")}
    p = {k: torch.randn(C, generator=g).cuda().requires_grad_(True) for k in ("s", "w", "b", "pw", "pb")}

    def sums(H, W):
        d = {k: v.expand(1, C, H, W).contiguous() for k, v in row.items()}
        out = Fh.residual_norm_train(d["x"], d["h"], (p["w"], p["b"], EPS), p["s"], d["gate"], (p["pw"], p["pb"], EPS))
        return dict(zip(p, torch.autograd.grad(out, list(p.values()), (d["gr"], d["gy"]))))

    n = H * W // 1024
    big, small = sums(H, W), sums(32, 32)
    size = {k: v.double().abs() for k, v in small.items()}
    # the scale's gradient is a sum of two: the branch norm's, over the scale, times its parameters
    size["s"] = (size["pw"] * p["pw"].abs() + size["pb"] * p["pb"].abs()) / p["s"].abs()
    for k in p:
        assert ((big[k].double() - n * small[k].double()).abs() <= 4 * U * 1.001 * n * size[k]).all(), k


def test_recorded_training_pass_of_128_channels():
    """The widest tiles of two pixels a lane, whose backward takes more shared memory than a launch has by itself."""
    shape = (1, 128, 33, 32)
    d = _dev(make(shape, gate="sample", post=True, seed=31))
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        grads(d, call(d))
    torch.cuda.current_stream().wait_stream(st)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        out = call(d)
        got = grads(d, out)
    for rep in range(3):
        new = make(shape, gate="sample", post=True, seed=50 + rep)
        with torch.no_grad():
            for k, v in new.items():
                d[k].copy_(v)
        e = _dev(new)
        want = grads(e, call(e))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(got[k], want[k]) for k in want)


@pytest.mark.parametrize("shape", [(2, 64, 33, 33), (2, 24, 5, 7), (1, 20, 40, 30), (1, 128, 36, 36), (1, 300, 6, 5), (3, 16), (0, 8, 4, 4)])
@pytest.mark.parametrize("t", [F32, BF16, F16])
def test_layernorm_that_keeps_a_copy(shape, t):
    """The gradients of the values that the forward had, bit for bit, whatever becomes of x."""
    from conversenet_amd import functional as Fh

    a = make(shape, t, t, branch=False, seed=sum(shape))
    got = []
    for copy in (False, True):
        d = _dev(a)
        x = d["x"] * 1.0
        y = Fh.layernorm_cf_train(x, d["w"], d["b"], EPS, copy=copy)
        if copy:
            x.fill_(float("nan"))
        got.append([y, *torch.autograd.grad(y, (d["x"], d["w"], d["b"]), d["gy"])])
    assert all(torch.equal(u, v) for u, v in zip(*got))


@pytest.mark.parametrize("t", [F32, BF16])
def test_gradient_penalty_through_a_copy(t):
    """The gradient of the copy, which only a differentiated backward gives, beside that of the norm."""
    from conversenet_amd import functional as Fh

    a = make((2, 24, 7, 5), t, t, branch=False, seed=70)
    got = []
    for copy in (False, True):
        d = _dev(a)
        y = Fh.layernorm_cf_train(d["x"], d["w"], d["b"], EPS, copy=copy)
        gx, = torch.autograd.grad(y, d["x"], d["gy"], create_graph=True)
        loss = (gx.double() ** 2).sum() + (y.double() ** 3).sum()
        got.append(torch.autograd.grad(loss, (d["x"], d["w"], d["b"])))
    for u, v in zip(*got):  # the two gradients of x are added in one rounding there, in two here
        assert float((u.double() - v.double()).norm()) <= 4 * torch.finfo(t).eps * float(u.double().norm())
