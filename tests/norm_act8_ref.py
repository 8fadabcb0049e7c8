"""64-bit restatements of the layer norm and of the 8-bit activation checkpoints, with bounds of what fp32 arithmetic may be off by.

Bounds count roundings: u = 2^-24 per fp32 operation, half a step of the output's type at the end.  A sum of n terms in fp32 in any
order of chains of length c is off by at most c u times the sum of the terms' magnitudes."""
import torch

U = 2.0 ** -24
SLOPE = float(torch.tensor(0.01, dtype=torch.float32))
TYPES = (torch.float32, torch.bfloat16, torch.float16)


def half_step(t):
    return torch.finfo(t).eps / 2


def tiny(t):   # half the smallest subnormal: what rounding near zero may be off by
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2


def kept64(x):
    """the values of the 8-bit form of x [M, D] (NaN where x is not finite), float64"""
    M, D = x.shape
    pad = -D % 32
    d = torch.nn.functional.pad(x.double().cpu(), (0, pad)).view(M, (D + pad) // 32, 32)
    finite = torch.isfinite(d)
    mag = torch.where(finite, d.abs().clamp(max=1.875 * 2.0 ** 127), torch.zeros_like(d))
    top = mag.amax(2, keepdim=True)
    mant, ex = torch.frexp(top / 448.0)
    e = torch.where(mant == 0.5, ex - 1, ex)   # smallest e with top <= 448 * 2^e
    e = torch.where(top == 0, torch.full_like(e, -117), e).clamp(min=-117).double()
    v = mag * torch.exp2(-e)
    _, vx = torch.frexp(v)
    step = torch.exp2((vx.double() - 4).clamp(min=-9.0))
    q = torch.round(v / step) * step
    q = torch.where((d > 0) & (q == 0) & finite, torch.full_like(q, 2.0 ** -9), q)
    q = torch.where(finite, torch.copysign(q, d) * torch.exp2(e), torch.full_like(q, float("nan")))
    return q.view(M, D + pad)[:, :D]


def _chain(D):
    """fp32 additions behind a row statistic, at most: 32 values per thread, 6 steps over a wave, 16 waves, and the scaling"""
    return 32 + 6 + 16 + 2


class Norm64:
    """y and its bound; then gradients and their bounds"""

    def __init__(self, x, w, b, eps):
        self.x = x.double().cpu()
        D = x.shape[1]
        self.w = torch.ones(D, dtype=torch.float64) if w is None else w.double().cpu()
        self.b = torch.zeros(D, dtype=torch.float64) if b is None else b.double().cpu()
        self.mean = self.x.mean(1, keepdim=True)
        c = self.x - self.mean
        var = (c * c).mean(1, keepdim=True)
        eps = float(torch.tensor(eps, dtype=torch.float32))
        self.rstd = 1.0 / torch.sqrt(var + eps)
        self.h = c * self.rstd
        n = _chain(D)
        self.d_mean = n * U * self.x.abs().mean(1, keepdim=True) + 2.0 ** -149
        # relative error of rstd: half that of var + eps, which is a mean of squares each off by its factors' errors, + root and division
        d_c = self.d_mean + U * c.abs()
        d_var = (2 * c.abs() * d_c + d_c * d_c).mean(1, keepdim=True) + (n + 1) * U * var
        self.d_rstd = 0.5 * d_var / (var + eps) * 1.01 + 4 * U
        self.n = n
        self.y = self.h * self.w + self.b
        self.d_h = self.rstd * d_c + self.h.abs() * (self.d_rstd + 2 * U)
        self.d_y = self.w.abs() * self.d_h + 2 * U * (self.w * self.h).abs() + U * self.y.abs()

    def y_bound(self, t):
        return self.d_y + half_step(t) * self.y.abs() * 1.01 + tiny(t)

    def backward(self, g, src=None, leaky=False, chain=None):
        """gradients at `src` (default x itself) with x's statistics; chain = additions behind a column sum, at most"""
        g = g.double().cpu()
        src = self.x if src is None else src
        h = (src - self.mean) * self.rstd
        d_c = self.d_mean + U * (src - self.mean).abs()
        d_h = self.rstd * d_c + h.abs() * (self.d_rstd + 2 * U)
        u = g * self.w
        c0, c1 = u.mean(1, keepdim=True), (u * h).mean(1, keepdim=True)
        dx = self.rstd * (u - c0 - h * c1)
        d_c0 = (self.n + 2) * U * u.abs().mean(1, keepdim=True)
        d_c1 = (self.n + 3) * U * (u * h).abs().mean(1, keepdim=True) + (u.abs() * d_h).mean(1, keepdim=True)
        terms = u.abs() + c0.abs() + (h * c1).abs()
        d_dx = self.rstd * (d_c0 + d_h * c1.abs() + h.abs() * d_c1 + d_h * d_c1 + 5 * U * terms) + dx.abs() * (self.d_rstd + 2 * U)
        if leaky:
            m = torch.where(src > 0, 1.0, SLOPE)
            dx, d_dx = dx * m, d_dx * m + U * (dx * m).abs()
        M = g.shape[0]
        chain = chain if chain is not None else M // 512 + 2 + 32 + 32 + 16
        dw, db = (g * h).sum(0), g.sum(0)
        d_dw = (g.abs() * d_h).sum(0) + chain * U * (g * h).abs().sum(0)
        d_db = chain * U * g.abs().sum(0)
        self.dx, self.d_dx, self.dw, self.d_dw, self.db, self.d_db = dx, d_dx, dw, d_dw, db, d_db
        return self

    def dx_bound(self, t):
        return self.d_dx + half_step(t) * self.dx.abs() * 1.01 + tiny(t)


def inside(got, want, bound, what):
    got = got.double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    err = (got - want).abs()
    bad = ~(err <= bound)
    bad &= ~(torch.isnan(got) & torch.isnan(want))
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} outside, first at {bad.nonzero()[0].tolist()}: " \
        f"{got[tuple(bad.nonzero()[0])].item()} for {want[tuple(bad.nonzero()[0])].item()}, allowed {torch.as_tensor(bound).expand_as(err)[tuple(bad.nonzero()[0])].item()}"


def weight_grad(g, q, norm=None):
    """dW, db in 64 bits and bounds.  Products of bf16 components are exact; the sum over m runs in chains whose rounding errors, each at
    most u of the running sum, are independent: 4 standard deviations of a random walk of n steps, 4 u sqrt(n) times the sum of
    magnitudes over sqrt(3) < 4 u sqrt(n) sum |g q|, + 8 u for the joins.  Behind a norm: both halves of w (S - c) + b db, each with
    roundings of g r (1 u)."""
    g = g.double().cpu()
    n = 3 * (g.shape[0] + 15) // 16 + 16
    k = U * (8 + 4 * n ** 0.5)
    db, d_db = g.sum(0), k * g.abs().sum(0)
    if norm is None:
        return g.t() @ q, k * (g.abs().t() @ q.abs()), db, d_db
    mean, rstd, w, b = (None if t is None else t.double().cpu() for t in norm)
    w = torch.ones(q.shape[1], dtype=torch.float64) if w is None else w
    b = torch.zeros(q.shape[1], dtype=torch.float64) if b is None else b
    mean, rstd = mean[:, None], rstd[:, None]
    dW = g.t() @ ((q - mean) * rstd * w + b)
    mag = (g.abs().t() @ ((q.abs() + mean.abs()) * rstd)) * w.abs() + b.abs() * g.abs().sum(0)[:, None]
    return dW, (k + 4 * U) * mag, db, d_db
