"""Loss and gradients of a linear layer under softmax cross-entropy in 64 bits, with bounds of the error that the kernels may make.

The bounds, eps = 2^-24 (fp32, to nearest), b = 2^-8 (bf16, to nearest: 8 significant bits), A = sum_c |x w| of a logit:
  * logits: fp32 sums of exact products, 16 at a time on the tensor cores, whose additions may truncate (2 eps each): dz = (C / 16 + 2) 4 eps A;
  * lse: dz, the relative errors of the exponentials (ex2.approx: 4 eps) and of the sums of 64 terms, of the tiles and of the logarithm (2^-17 together), and 4 eps
    of its own size for its rounding and that of the references;
  * g: rel = dz + d(lse) relative (the error of an exponent) and b for its rounding; products over K terms add (K / 16 + 2) 4 eps of the sum of magnitudes, each
    slice's or piece's sum an eps more; the results are rounded once, b of their size."""
import torch

EPS, B = 2.0 ** -24, 2.0 ** -8


def make(N, C, V, seed=0, rows=None, left_out=0.0, dtype=torch.bfloat16, scale=2.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(N, C, generator=g).to(dtype)
    w = (torch.randn(rows or V, C, generator=g) * scale / C ** 0.5).to(dtype)
    t = torch.randint(0, V, (N,), generator=g, dtype=torch.int32)
    t[torch.rand(N, generator=g) < left_out] = -1
    return x, w, t


def certain(N, V, dtype=torch.bfloat16):
    """Logits of 1024 for the target, 1 to 7 less for one other column, 0 for the rest, all exact.  The loss, log(1 + e^-k), has the errors of two exponentials (4 eps each),
    a handful of sums near 1 (an eps each; adding 0 is exact) and the logarithm, absolute, and the rounding of log2(e) relative.  Half an ulp of the logit would be 1024 eps."""
    C = 64
    g = torch.Generator().manual_seed(N)
    k = torch.randint(1, 8, (N,), generator=g)
    x, w = torch.zeros(N, C), torch.zeros(V, C)
    t, other = torch.randperm(V, generator=g)[:2 * min(N, 32)].int().chunk(2)
    i = torch.arange(len(t))
    rows = torch.arange(N) % len(t)
    w[t.long(), i] = 32.0
    x[torch.arange(N), rows] = 32.0
    w[other.long(), i], w[other.long(), 32 + i] = 31.75, 1.0   # 1016 from the target's channel
    x[torch.arange(N), 32 + rows] = (8 - k).float()
    want = torch.log1p(torch.exp(-k.double()))
    return x.to(dtype), w.to(dtype), t[rows].contiguous(), want, 16 * EPS * (1 + want)


def forward(x, w, t, V):
    """losses, lse and their bounds"""
    x, w, t = x.double().cpu(), w[:V].double().cpu(), t.long().cpu()
    z = x @ w.t()
    dz = (x.shape[1] / 16 + 2) * 4 * EPS * (x.abs() @ w.abs().t()).amax(1)
    lse = torch.logsumexp(z, 1)
    dl = dz + 2.0 ** -17 + 4 * EPS * lse.abs()
    keep = (t >= 0) & (t < V)
    loss = torch.where(keep, lse - z.gather(1, t.clamp(0, V - 1)[:, None])[:, 0], torch.zeros_like(lse))
    return loss, lse, torch.where(keep, dl + dz + EPS * loss.abs(), torch.zeros_like(dl)), dl


def gradient(x, w, t, V, lse, factor, old=None, pieces=1, b=B):
    """dinp, dweight and their bounds; ``factor`` (N) fp64.  ``b``: rounding of g and of the results"""
    x, w, t, lse = x.double().cpu(), w[:V].double().cpu(), t.long().cpu(), lse.double().cpu()
    N, C = x.shape
    keep = (t >= 0) & (t < V)
    f = torch.where(keep, factor.double().cpu(), torch.zeros(N, dtype=torch.float64))[:, None]
    z = x @ w.t()
    p = torch.exp(z - lse[:, None])
    one = torch.zeros_like(p)
    one[torch.arange(N)[keep], t[keep]] = 1.0
    g = (p - one) * f
    rel = (C / 16 + 2) * 4 * EPS * (x.abs() @ w.abs().t()) + 8 * EPS * (z.abs() + lse.abs()[:, None]) + 8 * EPS
    dg = (p * rel + 2 * EPS * one) * f.abs() + (b + 2 * EPS) * g.abs()
    dinp, dw = g @ w, g.t() @ x
    e_in = dg @ w.abs() + ((V / 16 + 2) * 4 + 16 + pieces) * EPS * (g.abs() @ w.abs()) + b * dinp.abs() * 1.01
    e_w = dg.t() @ x.abs() + ((N / 16 + 2) * 4 + 16) * EPS * (g.abs().t() @ x.abs())
    if old is not None:
        dw = dw + old[:V].double().cpu()
    return dinp, dw, e_in + 1e-30, e_w + b * dw.abs() * 1.01 + 1e-30


def within(got, want, bound):
    got = got.double().cpu()
    assert torch.isfinite(got).all()
    err = (got - want).abs()
    worst = (err / bound.clamp_min(1e-300)).max() if err.numel() else 0.0
    assert (err <= bound).all(), "error %.3g times its bound" % float(worst)
