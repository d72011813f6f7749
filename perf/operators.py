"""The operators of a training step around the convolutions of a block, and of its forward alone, as measurable cases.

Kinds of cases:
  serve  functional.residual_norm under no_grad: r = x + res_scale * gate * post(h), y = norm(r), channels first
  train  functional.residual_norm_train (without a branch: functional.layernorm_cf_train), and all its gradients
  gnorm  functional.grad_norm: the norm over all gradients of a model
  clip   functional.clip_grads into kept buffers: the gradients scaled to a largest norm, and the norm

`own` says whether run() makes those calls or computes the same from elementary torch operations.
"""
import math
import random

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
EPS = 1e-5  # the blocks' LayerNorms


def _norm(name, kind, B, C, H, W, x="f32", h="f32", branch=True, scale=True, gate="none", post=False):
    """x: type of x, r and y; h: type of the branch and its gate; gate: "none", "sample" (a factor per sample and
    channel) or "full" (a factor per element)."""
    c = {"kind": kind, "B": B, "C": C, "H": H, "W": W, "x": x, "h": h, "branch": branch, "scale": scale, "gate": gate,
         "post": post}
    return dict(c, name=name) if name else c


def _grads(name, kind, tensors, type, n=0, lo=0, hi=0, sizes=0, max_norm=1.0):
    """tensors: "denoiser" (the 284 parameters of ConverseDnCNN) or "any": n tensors of lo to hi elements, spread over
    their logarithm, drawn from the number `sizes`."""
    c = {"kind": kind, "tensors": tensors, "type": type, "n": n, "lo": lo, "hi": hi, "sizes": sizes, "max_norm": max_norm}
    return dict(c, name=name) if name else c


def listed():
    return [
        # one pixel of the blocks' 64 channels: latency and host work count
        _norm("serve_pixel", "serve", 1, 64, 1, 1),
        # the residual stream of one photo of odd size
        _norm("serve_photo", "serve", 1, 64, 321, 481),
        # a batch of half-precision feature maps with channel attention and a norm on both sides of the branch
        _norm("serve_gated_bf16", "serve", 8, 64, 256, 256, "bf16", "bf16", gate="sample", post=True),
        # training on 96 x 96 patches: a block's scaled residual and its next norm
        _norm("train_patch", "train", 8, 64, 96, 96),
        # the same at the headline layer's batch
        _norm("train_256", "train", 16, 64, 256, 256),
        # mixed precision: half-precision branch and gate on a float32 residual stream, 128 channels, both norms
        _norm("train_mixed", "train", 4, 128, 128, 128, "f32", "bf16", gate="full", post=True),
        # ragged half-precision maps with channel attention and no residual scale
        _norm("train_odd_f16", "train", 3, 48, 67, 45, "f16", "f16", scale=False, gate="sample"),
        # a LayerNorm by itself, the first layer of a block
        _norm("train_layernorm", "train", 8, 64, 128, 128, branch=False, scale=False),
        # the gradients of the denoiser, nearly all of them small
        _grads("gnorm_denoiser", "gnorm", "denoiser", "f32"),
        _grads("clip_denoiser", "clip", "denoiser", "f32"),
        # a model of large half-precision matrices
        _grads("gnorm_large_bf16", "gnorm", "any", "bf16", 40, 1_000_000, 16_000_000, 7),
        # large float32 gradients next to small ones, more than the card's last-level cache holds
        _grads("clip_large", "clip", "any", "f32", 96, 1_000, 30_000_000, 11),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("serve", "serve", "train", "train", "train", "gnorm", "clip"))
    if kind in ("gnorm", "clip"):
        if rng.random() < 0.25:
            return _grads(None, kind, "denoiser", rng.choice(("f32", "bf16")), max_norm=rng.choice((0.1, 1.0, 1e6)))
        lo = _log(rng, 1, 10_000)
        hi = _log(rng, lo, 8_000_000)
        n = _log(rng, 1, max(1, min(500, 200_000_000 // hi)))
        return _grads(None, kind, "any", rng.choice(("f32", "f32", "bf16", "f16")), n, lo, hi, rng.randrange(1 << 20),
                      rng.choice((0.1, 1.0, 1e6)))
    C = rng.choice((8, 16, 32, 48, 64, 64, 64, 96, 128, 128, 192, 256, rng.randint(8, 256)))
    H = _log(rng, 1, 384)
    W = max(1, min(512, int(round(H * math.exp(rng.uniform(-0.5, 0.5))))))
    B = _log(rng, 1, max(1, min(64, 30_000_000 // (C * H * W))))
    x, h = rng.choice((("f32", "f32"), ("f32", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("f32", "bf16"), ("f32", "f16")))
    if kind == "train" and rng.random() < 0.2:
        return _norm(None, kind, B, C, H, W, x, x, branch=False, scale=False)
    return _norm(None, kind, B, C, H, W, x, h, scale=rng.random() < 0.7, gate=rng.choice(("none", "none", "sample", "full")),
                 post=rng.random() < 0.4)


# --------------------------------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------------------------------
def _sizes(c):
    if c["tensors"] == "any":
        rng = random.Random(c["sizes"])
        return [_log(rng, c["lo"], c["hi"]) for _ in range(c["n"])]
    block = [64, 64, 128 * 64, 128, 128 * 49, 128, 64 * 128, 64, 64, 64, 128 * 64, 128, 64 * 128, 64]
    return [64, 64] + 20 * block + [64, 1]


def _buckets(sizes, dtype):
    """One buffer for all clipped gradients, as an optimizer or an all-reduce takes them, and its parts, each from a
    multiple of 64 elements on."""
    starts = [0]
    for n in sizes:
        starts.append(starts[-1] + (n + 63) // 64 * 64)
    flat = torch.zeros(starts[-1], dtype=dtype, device="cuda")
    return flat, [flat[i:i + n] for i, n in zip(starts, sizes)]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    c, kind = case, case["kind"]

    def randn(*shape):
        return torch.randn(shape, device="cuda", generator=g)

    if kind in ("gnorm", "clip"):
        t = TYPES[c["type"]]
        # gradients of layers of different depth differ by orders of magnitude
        mag = (10 ** (-3 * torch.rand(len(_sizes(c)), generator=g, device="cuda"))).tolist()
        grads = [(randn(n) * m).to(t) for n, m in zip(_sizes(c), mag)]
        st = {"case": c, "grads": grads}
        if kind == "clip":
            st["flat"], st["out"] = _buckets([v.numel() for v in grads], t)
        return st
    B, C, H, W = c["B"], c["C"], c["H"], c["W"]
    tx, th = TYPES[c["x"]], TYPES[c["h"]]
    st = {"case": c, "x": (randn(B, C, H, W) + 0.5).to(tx), "w": 1 + 0.1 * randn(C), "b": 0.1 * randn(C)}
    if c["branch"]:
        st["h"] = randn(B, C, H, W).to(th)
    if c["scale"]:
        st["s"] = 0.3 * randn(1, C, 1, 1)
    if c["gate"] != "none":
        st["gate"] = torch.sigmoid(randn(B, C, 1, 1) if c["gate"] == "sample" else randn(B, C, H, W)).to(th)
    if c["post"]:
        st["pw"], st["pb"] = 1 + 0.1 * randn(C), 0.1 * randn(C)
    if kind == "train":
        for k in [k for k in st if k != "case"]:
            st[k].requires_grad_(True)
        if c["branch"]:
            st["gr"] = randn(B, C, H, W).to(tx)
        st["gy"] = randn(B, C, H, W).to(tx)
    return st


# --------------------------------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------------------------------
LEAVES = ("x", "h", "gate", "s", "w", "b", "pw", "pb")


def _ln(v, w, b):
    d = v - v.mean(1, keepdim=True)
    return d / torch.sqrt((d * d).mean(1, keepdim=True) + EPS) * w.view(-1, 1, 1) + b.view(-1, 1, 1)


def _forward_plain(st):
    x = st["x"].float()
    if "h" not in st:
        return (_ln(x, st["w"], st["b"]).to(st["x"].dtype),)
    u = st["h"].float()
    if "pw" in st:
        u = _ln(u, st["pw"], st["pb"])
    if "gate" in st:
        u = st["gate"].float() * u
    if "s" in st:
        u = st["s"] * u
    r = x + u
    return r.to(st["x"].dtype), _ln(r, st["w"], st["b"]).to(st["x"].dtype)


def _forward_own(st, train):
    from conversenet_amd import functional as F

    norm = (st["w"], st["b"], EPS)
    if "h" not in st:
        return (F.layernorm_cf_train(st["x"], *norm),)
    post = (st["pw"], st["pb"], EPS) if "pw" in st else None
    f = F.residual_norm_train if train else F.residual_norm
    return f(st["x"], st["h"], norm=norm, res_scale=st.get("s"), gate=st.get("gate"), post=post)


def _clip_plain(grads, max_norm, out):
    norm = torch.stack([g.float().square().sum(dtype=torch.float64) for g in grads]).sum().sqrt()
    if max_norm is None:
        return norm.float()
    coef = (max_norm / (norm + 1e-6)).clamp(max=1.0).float()
    for g, o in zip(grads, out):
        o.copy_(g.float() * coef)
    return norm.float()


def run(state):
    c = state["case"]
    if c["kind"] in ("gnorm", "clip"):
        grads, m = state["grads"], c["max_norm"] if c["kind"] == "clip" else None
        if not own:
            norm = _clip_plain(grads, m, state.get("out"))
        else:
            from conversenet_amd import functional as F

            norm = F.grad_norm(grads) if m is None else F.clip_grads(grads, m, out=state["out"])[1]
        return norm if m is None else {"norm": norm, "grads": state["flat"]}
    if c["kind"] == "serve":
        with torch.no_grad():
            return _forward_own(state, False) if own else _forward_plain(state)
    out = _forward_own(state, True) if own else _forward_plain(state)
    leaves = [k for k in LEAVES if k in state]
    gos = [state[k] for k in ("gr", "gy") if k in state]
    grads = torch.autograd.grad(out, [state[k] for k in leaves], gos)
    return {"out": [v.detach() for v in out], "grads": dict(zip(leaves, grads))}


# --------------------------------------------------------------------------------------------------
# the work a pass cannot do without
# --------------------------------------------------------------------------------------------------
def work(case):
    c = case
    if c["kind"] in ("gnorm", "clip"):
        n = sum(_sizes(c))
        return {"bytes": n * BYTES[c["type"]] * (2 if c["kind"] == "clip" else 1), "flops": n * (3 if c["kind"] == "clip" else 2)}
    n = c["B"] * c["C"] * c["H"] * c["W"]
    bx, bh = BYTES[c["x"]], BYTES[c["h"]]
    bg = {"none": 0, "sample": c["B"] * c["C"] * bh, "full": n * bh}[c["gate"]]
    if not c["branch"]:  # x, y; grad_y, grad_x
        return {"bytes": 4 * n * bx, "flops": 18 * n}
    fwd = 3 * n * bx + n * bh + bg  # x, h, gate; r, y
    if c["kind"] == "serve":
        return {"bytes": fwd, "flops": (10 + 8 * c["post"]) * n}
    # grad_r, grad_y; the gradients of x, h and gate
    return {"bytes": fwd + 3 * n * bx + n * bh + bg, "flops": (25 + 20 * c["post"]) * n}


# --------------------------------------------------------------------------------------------------
# 64-bit results, with the gradients from their formulas
# --------------------------------------------------------------------------------------------------
def _standard(v):
    """The standardised values over the channels, and 1 / their deviation."""
    u = v.sum(1, keepdim=True) / v.shape[1]
    rho = 1 / torch.sqrt(((v - u) ** 2).sum(1, keepdim=True) / v.shape[1] + EPS)
    return (v - u) * rho, rho


def _standard_grad(g, hat, rho):
    """The gradient of standardised values with respect to the values."""
    C = g.shape[1]
    return rho * (g - g.sum(1, keepdim=True) / C - hat * ((g * hat).sum(1, keepdim=True) / C))


def exact(case, seed):
    c = case
    st = prepare(case, seed)
    if c["kind"] in ("gnorm", "clip"):
        grads = [g.double() for g in st["grads"]]
        norm = math.sqrt(math.fsum((g * g).sum().item() for g in grads))
        if c["kind"] == "gnorm":
            return torch.tensor(norm, dtype=torch.float64, device="cuda")
        f = min(1.0, c["max_norm"] / (norm + 1e-6))
        flat, parts = _buckets([g.numel() for g in grads], torch.float64)
        for g, p in zip(grads, parts):
            p.copy_(g * f)
        return {"norm": torch.tensor(norm, dtype=torch.float64, device="cuda"), "grads": flat}
    with torch.no_grad():
        d = {k: v.double() for k, v in st.items() if k != "case"}
        cf = (1, -1, 1, 1)
        w, b = d["w"].view(cf), d["b"].view(cf)
        if not c["branch"]:
            hat, rho = _standard(d["x"])
            gy = d["gy"]
            return {"out": [hat * w + b],
                    "grads": {"x": _standard_grad(gy * w, hat, rho), "w": (gy * hat).sum((0, 2, 3)), "b": gy.sum((0, 2, 3))}}
        s, gate = d.get("s", 1.0), d.get("gate", 1.0)
        n = d["h"]
        if c["post"]:
            phat, prho = _standard(n)
            n = phat * d["pw"].view(cf) + d["pb"].view(cf)
        r = d["x"] + s * gate * n
        hat, rho = _standard(r)
        out = [r, hat * w + b]
        if c["kind"] == "serve":
            return tuple(out)
        gy = d["gy"]
        dr = d["gr"] + _standard_grad(gy * w, hat, rho)
        grads = {"x": dr}
        dn = dr * s * gate
        if c["post"]:
            grads["h"] = _standard_grad(dn * d["pw"].view(cf), phat, prho)
        else:
            grads["h"] = dn
        if c["gate"] != "none":
            dg = dr * s * n
            grads["gate"] = dg.sum((2, 3), keepdim=True) if c["gate"] == "sample" else dg
        if c["scale"]:
            grads["s"] = (dr * gate * n).sum((0, 2, 3)).view(cf)
        grads["w"], grads["b"] = (gy * hat).sum((0, 2, 3)), gy.sum((0, 2, 3))
        if c["post"]:
            grads["pw"], grads["pb"] = (dn * phat).sum((0, 2, 3)), dn.sum((0, 2, 3))
        return {"out": out, "grads": grads}
