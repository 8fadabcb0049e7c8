"""What is measured of the layer norm and of the 8-bit activation checkpoints: cases, inputs, and both ways to compute them.

With ``own`` false a pass is computed from elementary torch operations in 32 bits; with ``own`` true it makes the calls a user of
``pivotcvae_amd.ops`` makes.  Kinds of cases:

    ln_fwd    y of a layer norm over the rows of x [M, D]                                  (an answer)
    ln_train  y, then dx, dweight, dbias for a given output gradient                        (a train step's norm)
    pack      x [M, D] kept in 8 bits, and the values that stands for
    wgrad     a linear layer [D -> N]: its input kept in 8 bits, then dW, db from the codes
    norm8     activation -> norm -> linear [D -> N] with the activation kept in 8 bits: the norm's y; then dW, db of the linear, and
              the gradient in front of the activation (LeakyReLU), dweight and dbias of the norm, all from the codes
"""
import math

import torch

own = False

EPS = 1e-5
SLOPE = 0.01
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
BLOCK = 32


def listed():
    def case(name, kind, M, D, t, N=0):
        return {"name": name, "kind": kind, "M": M, "D": D, "N": N, "type": t}

    return [
        # one slate is answered: the norm behind a hidden layer of width 256
        case("ln_fwd_1x256_f32", "ln_fwd", 1, 256, "f32"),
        # the norm of a hidden layer (width 256) of a stack in a train step over 8192 slates
        case("ln_train_8192x256_f32", "ln_train", 8192, 256, "f32"),
        # an odd width (the encoder's input row: 10 items and a user of 128, an 11-way condition), a batch that fills no grid
        case("ln_train_1000x1419_f16", "ln_train", 1000, 1419, "f16"),
        # a wide stack in half precision, many rows
        case("ln_train_32768x2048_bf16", "ln_train", 32768, 2048, "bf16"),
        # the encoder's input at 20 items of width 256: odd rows of 5397
        case("pack_8192x5397_f32", "pack", 8192, 5397, "f32"),
        # hidden activations of a long batch in half precision
        case("pack_65536x1024_bf16", "pack", 65536, 1024, "bf16"),
        # the smallest train step: 64 slates, the encoder's first layer at 5 items of width 16
        case("wgrad_64_256x102_f32", "wgrad", 64, 102, "f32", 256),
        # the encoder's first layer in a train step over 8192 slates
        case("wgrad_8192_256x1419_f32", "wgrad", 8192, 1419, "f32", 256),
        # a square layer in half precision
        case("wgrad_16384_2048x2048_bf16", "wgrad", 16384, 2048, "bf16", 2048),
        # the completion stack's last layer at 20 items of width 256, hidden width 1024, a long batch
        case("wgrad_32768_4864x1024_f32", "wgrad", 32768, 1024, "f32", 4864),
        # hidden layer -> norm -> hidden layer of a stack, 8192 slates
        case("norm8_8192_256x256_f32", "norm8", 8192, 256, "f32", 256),
        # the same of a wide stack
        case("norm8_16384_1024x2048_f32", "norm8", 16384, 2048, "f32", 1024),
    ]


def _between(rng, lo, hi):
    """a whole number, its logarithm spread evenly"""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["ln_fwd", "ln_train", "pack", "wgrad", "norm8"])
    t = rng.choice(["f32", "bf16", "f16"])
    D = _between(rng, 16, 8192)
    if rng.random() < 0.5:   # widths are multiples of 8 as often as not
        D = max(16, D // 8 * 8)
    room = (1 << 25) if t == "f32" else (1 << 26)   # values of the largest operand
    M = _between(rng, 1, 65536)
    M = max(1, min(M, room // D))
    N = 0
    if kind in ("wgrad", "norm8"):
        N = _between(rng, 8, 4096)
        D = min(D, 5397)
        M = max(1, min(M, int(1.5e11 / (2.0 * N * D)), room // max(D, N)))
    return {"kind": kind, "M": M, "D": D, "N": N, "type": t}


def _leaky(x):
    return torch.where(x > 0, x, SLOPE * x)


def _inputs(case, seed):
    dev = "cuda"
    gen = torch.Generator(device=dev).manual_seed(seed)
    t = TYPES[case["type"]]
    M, D, N = case["M"], case["D"], case["N"]

    def normal(*shape):
        return torch.randn(*shape, device=dev, generator=gen)

    st = {"case": dict(case)}
    row = torch.exp(0.25 * normal(M, 1))          # rows differ in scale as slates do
    st["x"] = _leaky((normal(M, D) + 0.1) * row).to(t)
    if case["kind"] != "pack":
        st["w"] = 1.0 + 0.1 * normal(D)
        st["b"] = 0.1 * normal(D)
    if case["kind"] in ("ln_train", "norm8"):
        st["g"] = (0.01 * normal(M, D)).to(t)
    if case["kind"] in ("wgrad", "norm8"):
        st["gz"] = (0.01 * normal(M, N)).to(t)
    return st


def prepare(case, seed):
    return _inputs(case, seed)


# ---- the plain form -------------------------------------------------------------------------------------------------------------
def _ln_plain(x, w, b):
    xf = x.float()
    mean = xf.mean(1, keepdim=True)
    c = xf - mean
    rstd = 1.0 / torch.sqrt((c * c).mean(1, keepdim=True) + EPS)
    return (c * rstd * w + b).to(x.dtype), mean, rstd


def _ln_plain_bwd(g, xf, w, mean, rstd, masked):
    gf = g.float()
    xh = (xf - mean) * rstd
    wg = gf * w
    dx = rstd * (wg - wg.mean(1, keepdim=True) - xh * (wg * xh).mean(1, keepdim=True))
    if masked:
        dx = torch.where(xf > 0, dx, SLOPE * dx)
    return dx.to(g.dtype), (gf * xh).sum(0), gf.sum(0)


def _pack_plain(x):
    """the values of the 8-bit checkpoint, fp32"""
    M, D = x.shape
    nb = (D + BLOCK - 1) // BLOCK
    xf = torch.zeros(M, nb * BLOCK, device=x.device)
    xf[:, :D] = x.float()
    xf = xf.view(M, nb, BLOCK)
    mag = torch.clamp(xf.abs(), max=2.0 ** 127 * 1.875)
    top = torch.where(torch.isfinite(xf), mag, torch.zeros_like(mag)).amax(2, keepdim=True)
    bits = top.view(torch.int32)
    field = (bits + 0x1FFFFF) >> 23                        # the exponent, one more where the significand is over 1.75
    field = torch.clamp(field - 8, min=10)
    scale = (field << 23).view(torch.float32)
    inv = ((254 - field) << 23).view(torch.float32)
    v = torch.copysign(mag, xf) * inv
    q = v.to(torch.float8_e4m3fn).float()
    q = torch.where((v > 0) & (q == 0), torch.full_like(q, 2.0 ** -9), q)
    q = torch.where(torch.isfinite(xf), q * scale, torch.full_like(q, float("nan")))
    return q.view(M, nb * BLOCK)[:, :D]


def _run_plain(st):
    case = st["case"]
    kind, x = case["kind"], st["x"]
    if kind == "ln_fwd":
        return _ln_plain(x, st["w"], st["b"])[0]
    if kind == "ln_train":
        y, mean, rstd = _ln_plain(x, st["w"], st["b"])
        return (y,) + _ln_plain_bwd(st["g"], x.float(), st["w"], mean, rstd, False)
    if kind == "pack":
        return _pack_plain(x).to(x.dtype)
    if kind == "wgrad":
        gz = st["gz"].float()
        return gz.t() @ _pack_plain(x), gz.sum(0)
    y, mean, rstd = _ln_plain(x, st["w"], st["b"])
    xq = _pack_plain(x)
    gz = st["gz"].float()
    n = (xq - mean) * rstd * st["w"] + st["b"]
    return (y, gz.t() @ n, gz.sum(0)) + _ln_plain_bwd(st["g"], xq, st["w"], mean, rstd, True)


def _run_own(st):
    from pivotcvae_amd import ops
    kind, x = st["case"]["kind"], st["x"]
    if kind == "ln_fwd":
        return ops.layer_norm_fwd_raw(x, st["w"], st["b"], EPS)[0]
    if kind == "ln_train":
        y, mean, rstd, _ = ops.layer_norm_fwd_raw(x, st["w"], st["b"], EPS)
        return (y,) + ops.layer_norm_bwd_raw(st["g"], x, st["w"], mean, rstd)
    if kind == "pack":
        return ops.act8_pack(x).unpack(x.dtype)
    if kind == "wgrad":
        return ops.act8_bwd_weight_raw(st["gz"], ops.act8_pack(x))
    y, mean, rstd, kept = ops.layer_norm_fwd_raw(x, st["w"], st["b"], EPS, checkpoint="e4m3")
    dW, db = ops.act8_bwd_weight_raw(st["gz"], kept, norm=(mean, rstd, st["w"], st["b"]))
    return (y, dW, db) + ops.layer_norm_bwd_raw(st["g"], kept, st["w"], mean, rstd, leaky=True)


def run(state):
    return _run_own(state) if own else _run_plain(state)


def work(case):
    M, D, N, s = case["M"], case["D"], case["N"], SIZE[case["type"]]
    kind = case["kind"]
    codes = M * D + M * ((D + BLOCK - 1) // BLOCK)
    if kind == "ln_fwd":
        return {"bytes": 2 * s * M * D + 8 * D, "flops": 8 * M * D}
    if kind == "ln_train":     # x and the gradient read, y and dx written; what the forward hands the backward is x itself
        return {"bytes": 4 * s * M * D + 16 * D, "flops": 24 * M * D}
    if kind == "pack":         # x read, the codes written, the values they stand for written
        return {"bytes": 2 * s * M * D + codes, "flops": 4 * M * D}
    if kind == "wgrad":        # x and the gradient read, the codes written, dW and db written
        return {"bytes": s * M * (D + N) + codes + 4 * N * (D + 1), "flops": 2 * M * N * D}
    return {"bytes": s * M * (4 * D + N) + codes + 4 * N * (D + 1) + 16 * D, "flops": 2 * M * N * D + 28 * M * D}


# ---- the definition in 64 bits ---------------------------------------------------------------------------------------------------
def _kept64(x):
    """what the checkpoint holds, from its definition: per block of 32 columns the smallest power of two p = 2^e with
    max|x| <= 448 p (e >= -117), every value rounded to the nearest e4m3 multiple of p, ties to even, positive ones at least p 2^-9"""
    M, D = x.shape
    pad = -D % BLOCK
    d = torch.nn.functional.pad(x.double(), (0, pad)).view(M, -1, BLOCK)
    top = d.abs().amax(2, keepdim=True)
    mant, ex = torch.frexp(top / 448.0)                    # top / 448 = mant 2^ex, mant in [1/2, 1)
    e = torch.where(mant == 0.5, ex - 1, ex)
    e = torch.where(top == 0, torch.full_like(e, -117), e).clamp(min=-117).double()
    v = d * torch.exp2(-e)
    _, vx = torch.frexp(v)
    step = torch.exp2((vx.double() - 4).clamp(min=-9.0))   # 4 significand bits; below 2^-6 the grid is 2^-9
    q = torch.round(v / step) * step                       # torch rounds halves to even
    q = torch.where((v > 0) & (q == 0), torch.full_like(q, 2.0 ** -9), q)
    return (q * torch.exp2(e)).view(M, D + pad)[:, :D]


def exact(case, seed):
    st = _inputs(case, seed)
    kind, x = case["kind"], st["x"]
    if kind == "pack":
        return _kept64(x)
    xd = x.double()
    if kind == "wgrad":
        gz = st["gz"].double()
        return gz.t() @ _kept64(x), gz.sum(0)
    w, b = st["w"].double(), st["b"].double()
    mu = xd.sum(1, keepdim=True) / xd.shape[1]
    var = ((xd - mu) ** 2).sum(1, keepdim=True) / xd.shape[1]
    sd = torch.sqrt(var + EPS)
    y = w * (xd - mu) / sd + b
    if kind == "ln_fwd":
        return y
    src = xd if kind == "ln_train" else _kept64(x)
    g = st["g"].double()
    xh = (src - mu) / sd
    u = g * w
    dx = (u - u.mean(1, keepdim=True) - xh * (u * xh).mean(1, keepdim=True)) / sd
    if kind == "ln_train":
        return y, dx, (g * xh).sum(0), g.sum(0)
    dx = dx * torch.where(xd > 0, 1.0, SLOPE)              # the mask of the activation itself: the codes keep its sign
    gz = st["gz"].double()
    return y, gz.t() @ (xh * w + b), gz.sum(0), dx, (g * xh).sum(0), g.sum(0)
