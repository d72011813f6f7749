"""1x1 convolutions of microscaled 4-bit maps and matrices (MXFP4), as measurable cases.

A matrix' columns or a map's channels come in blocks of 32 with a scale 2^s and values 0, 0.5, 1, 1.5, 2, 3, 4, 6 with a sign;
s is floor(log2) of the block's largest magnitude, less 2.

Kinds of cases:
  round  functional.quantize_mxfp4 of a map, and functional.dequantize_mxfp4 of that: the values the 4 bits stand for
  conv   functional.conv1x1_mxfp4: a map quantised on its way into the product with a matrix that was quantised before; bias,
         GELU, scaled residual
  train  functional.conv1x1_mxfp4_train: the product of both quantised, and the gradients straight through the quantisation

`own` says whether run() makes those calls or computes the same from elementary torch operations.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}


def _case(name, kind, type, B, C, H, W, N=0, act="none", residual=False):
    """type: of the map and the result; C: channels in, N: channels out."""
    c = {"kind": kind, "type": type, "B": B, "C": C, "H": H, "W": W, "N": N, "act": act, "residual": residual}
    return dict(c, name=name) if name else c


def listed():
    return [
        # one pixel of the blocks' 64 channels: latency and host work count
        _case("round_pixel", "round", "f32", 1, 64, 1, 1),
        # the feature maps of the headline layer, more than the card's last-level cache holds
        _case("round_map", "round", "f32", 16, 64, 256, 256),
        # half-precision maps of odd size, whose last block of channels is not full
        _case("round_odd_bf16", "round", "bf16", 3, 100, 67, 45),
        # a vector through a wide layer, one at a time: the matrix' bytes and latency count
        _case("conv_vector", "conv", "f32", 1, 4096, 1, 1, 4096),
        # a small batch of half-precision vectors through a wide layer
        _case("conv_vectors_f16", "conv", "f16", 16, 2048, 1, 1, 8192, act="gelu"),
        # a block's first layer on a batch of maps
        _case("conv_block_up", "conv", "f32", 8, 64, 256, 256, 128, act="gelu"),
        # a block's last layer with its scaled residual
        _case("conv_block_down", "conv", "f32", 8, 128, 256, 256, 64, residual=True),
        # a block's first layer on one photo of odd size, half precision
        _case("conv_photo_bf16", "conv", "bf16", 1, 64, 321, 481, 128, act="gelu"),
        # wide half-precision layers: the matrix units count
        _case("conv_wide_bf16", "conv", "bf16", 4, 2048, 64, 64, 4096),
        # training a block's layer on patches
        _case("train_block", "train", "f32", 8, 64, 96, 96, 128),
        # training a wide half-precision layer
        _case("train_wide_bf16", "train", "bf16", 8, 1024, 32, 32, 1024),
        # ragged maps with channels that fill no tile
        _case("train_odd_f16", "train", "f16", 3, 48, 67, 45, 80),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("round", "conv", "conv", "conv", "conv", "train", "train", "train"))
    type = rng.choice(("f32", "f32", "bf16", "f16"))

    def channels(hi):
        return rng.choice((rng.choice((16, 32, 64, 64, 128, 128, 256)), min(hi, 32 * _log(rng, 1, 128)), _log(rng, 1, hi)))

    shape = rng.choice(("vectors", "map", "map"))
    if kind == "round":
        C = channels(4096)
        N = 0
        limit = 60_000_000 // C  # pixels
    else:
        hi = 4096 if kind == "conv" else 2048
        C, N = channels(hi), channels(hi)
        limit = min(60_000_000 // (C + N), (100_000_000_000 if kind == "conv" else 16_000_000_000) // (C * N))
    if shape == "vectors":
        B, H, W = _log(rng, 1, max(1, min(256, limit))), 1, 1
    else:
        H = _log(rng, 1, max(1, min(384, math.isqrt(limit))))
        W = max(1, min(512, limit // H, int(round(H * math.exp(rng.uniform(-0.5, 0.5))))))
        B = _log(rng, 1, max(1, min(16, limit // (H * W))))
    conv = kind == "conv"
    return _case(None, kind, type, B, C, H, W, N, rng.choice(("none", "gelu")) if conv else "none",
                 conv and rng.random() < 0.4)


# --------------------------------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------------------------------
def _blocks(x):
    """(B,C,*) -> (B,blocks,32,*), float32, the last block filled up with zeros."""
    x = x.float()
    B, C = x.shape[:2]
    k = (C + 31) // 32
    if 32 * k != C:
        x = torch.cat((x, x.new_zeros((B, 32 * k - C) + x.shape[2:])), 1)
    return x.view((B, k, 32) + x.shape[2:])


def _pow2(e):
    """2^e in float32, from -127 to 127."""
    return torch.where(e > -127, (e + 127) << 23, 1 << 22).to(torch.int32).view(torch.float32)


def _scaled(x):
    """Blocks of x over their scales, and the scales' exponents."""
    v = _blocks(x)
    top = v.abs().amax(2, keepdim=True)
    e = (torch.frexp(top).exponent - 3).clamp(min=-127)
    e = torch.where(top > 0, e, torch.full_like(e, -127))
    return v * _pow2(-e), e


def _grid(v):
    """Number of the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 to each magnitude; ties to the even number."""
    a = v.abs()
    n = (a > 0.25).to(torch.int32)
    for t, above in ((0.75, False), (1.25, True), (1.75, False), (2.5, True), (3.5, False), (5.0, True)):
        n += (a > t) if above else (a >= t)
    return n


def _values(x):
    """What the 4 bits of x stand for, float32."""
    v, e = _scaled(x)
    n = _grid(v)
    mag = torch.where(n < 4, n * 0.5, torch.where(n < 6, n - 2.0, n * 2.0 - 8.0))
    q = torch.copysign(mag, v) * _pow2(e)
    return q.flatten(1, 2)[:, :x.shape[1]]


def _codes(w):
    """A matrix (N,C) as stored: (N,16 blocks) bytes, the lower half the value of lower number; (N,blocks) exponents + 127."""
    v, e = _scaled(w)
    c = (_grid(v) + 8 * torch.signbit(v)).flatten(1, 2)
    return (c[:, 0::2] + 16 * c[:, 1::2]).to(torch.uint8), (e + 127).flatten(1, 2).to(torch.uint8)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    c = case
    B, C, H, W, N = c["B"], c["C"], c["H"], c["W"], c["N"]
    t = TYPES[c["type"]]

    def randn(*shape):
        return torch.randn(shape, device="cuda", generator=g)

    # channels of a feature map differ in size
    st = {"case": c, "x": (randn(B, C, H, W) * torch.exp(0.7 * randn(1, C, 1, 1))).to(t)}
    if c["kind"] == "round":
        return st
    w = randn(N, C) / math.sqrt(C)
    st["b"] = 0.1 * randn(N)
    if c["kind"] == "conv":  # the matrix is kept in 4 bits
        st["w"] = _values(w)
        st["codes"], st["scales"] = _codes(w)
        if c["residual"]:
            st["residual"], st["s"] = randn(B, N, H, W).to(t), 0.3 * randn(N)
        return st
    st["w"] = w.view(N, C, 1, 1)
    for k in ("x", "w", "b"):
        st[k].requires_grad_(True)
    st["gy"] = randn(B, N, H, W).to(t)
    return st


# --------------------------------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------------------------------
def _product(w, x):
    """(N,C) times (B,C,H,W)."""
    B, C, H, W = x.shape
    if H * W == 1:
        return (x.view(B, C) @ w.t()).view(B, -1, 1, 1)
    return torch.matmul(w, x.reshape(B, C, H * W)).view(B, -1, H, W)


def _conv_plain(st):
    y = _product(st["w"], _values(st["x"])) + st["b"].view(-1, 1, 1)
    if st["case"]["act"] == "gelu":
        y = 0.5 * y * (1 + torch.erf(y * math.sqrt(0.5)))
    if "residual" in st:
        y = st["s"].view(-1, 1, 1) * y + st["residual"].float()
    return y.to(st["x"].dtype)


def _train_plain(st):
    x, w, gy = st["x"].detach(), st["w"].detach(), st["gy"].float()
    xq, wq = _values(x), _values(w.flatten(1))
    y = (_product(wq, xq) + st["b"].detach().view(-1, 1, 1)).to(x.dtype)
    gx = _product(wq.t().contiguous(), gy).to(x.dtype)
    n = max(1, gy.shape[2] * gy.shape[3])
    if n == 1:
        gw = gy.flatten(1).t().contiguous() @ xq.flatten(1)
    else:
        gw = sum((a.reshape(-1, n) @ b.reshape(-1, n).t().contiguous()).double() for a, b in zip(gy, xq)).float()
    return {"y": y, "x": gx, "w": gw.view(w.shape), "b": gy.sum((0, 2, 3), dtype=torch.float64).float()}


def run(state):
    c = state["case"]
    if not own:
        if c["kind"] == "round":
            return _values(state["x"]).to(state["x"].dtype)
        return _conv_plain(state) if c["kind"] == "conv" else _train_plain(state)
    from conversenet_amd import functional as F

    if c["kind"] == "round":
        return F.dequantize_mxfp4(F.quantize_mxfp4(state["x"]), state["x"].dtype)
    if c["kind"] == "conv":
        w = F.MXFP4(state["codes"], state["scales"], c["C"])
        return F.conv1x1_mxfp4(state["x"], w, state["b"], act="gelu" if c["act"] == "gelu" else None,
                               residual=state.get("residual"), res_scale=state.get("s"))
    y = F.conv1x1_mxfp4_train(state["x"], state["w"], state["b"])
    gx, gw, gb = torch.autograd.grad(y, (state["x"], state["w"], state["b"]), state["gy"])
    return {"y": y.detach(), "x": gx, "w": gw, "b": gb}


# --------------------------------------------------------------------------------------------------
# the work a pass cannot do without
# --------------------------------------------------------------------------------------------------
def work(case):
    c = case
    P, C, N, b = c["B"] * c["H"] * c["W"], c["C"], c["N"], BYTES[c["type"]]
    if c["kind"] == "round":  # the map, its 4 bits there and back, the values
        return {"bytes": P * C * 2 * b + 2 * P * ((C + 31) // 32) * 17, "flops": 4 * P * C}
    if c["kind"] == "conv":
        w = N * ((C + 31) // 32) * 17
        return {"bytes": P * b * (C + N * (2 if c["residual"] else 1)) + w, "flops": 2 * P * C * N}
    # x and its gradient, y and its gradient; the matrix and its gradient
    return {"bytes": 2 * P * b * (C + N) + 8 * C * N, "flops": 6 * P * C * N}


# --------------------------------------------------------------------------------------------------
# 64-bit results
# --------------------------------------------------------------------------------------------------
def _exact_values(x):
    """Rounds each block to multiples of the step its power of two has, in 64 bits."""
    x = x.detach().double()
    out = torch.empty_like(x)
    for i in range(0, x.shape[1], 32):
        v = x[:, i:i + 32]
        top = v.abs().amax(1, keepdim=True)
        unit = ((torch.frexp(top)[1].clamp(min=-124).long() + 1020) << 52).view(torch.float64)
        a = (v / unit).abs()
        step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0)).double()
        q = torch.clamp(torch.round(a / step) * step, max=6.0)  # torch.round: ties to even
        out[:, i:i + 32] = torch.where(top > 0, torch.sign(v) * q * unit, torch.zeros_like(v))
    return out


def exact(case, seed):
    c = case
    st = prepare(case, seed)
    with torch.no_grad():
        x = _exact_values(st["x"])
        if c["kind"] == "round":
            return x
        B, C, H, W = x.shape
        N = c["N"]
        px = x.permute(1, 0, 2, 3).reshape(C, -1)  # channels by pixels
        w = st["w"].double() if c["kind"] == "conv" else _exact_values(st["w"].flatten(1))
        y = w @ px + st["b"].detach().double()[:, None]
        if c["act"] == "gelu":
            y = y * torch.special.erfc(-y / math.sqrt(2.0)) / 2

        def maps(v):
            return v.view(-1, B, H, W).permute(1, 0, 2, 3).contiguous()

        if c["kind"] == "conv":
            y = maps(y)
            if c["residual"]:
                y = st["residual"].double() + st["s"].double()[None, :, None, None] * y
            return y
        g = st["gy"].double().permute(1, 0, 2, 3).reshape(N, -1)
        gw = torch.matmul(g, px.t().contiguous()).view(N, C, 1, 1)
        return {"y": maps(y), "x": maps(w.t().contiguous() @ g), "w": gw, "b": g.sum(1)}
