"""64-bit statements of the row operators (scoring, block joint, 8-bit activations)
and the error bounds that their FP32 arithmetic allows, shared by the CPU and GPU tests."""
import torch

U = 2.0 ** -24   # half a step of FP32
GROUP = 128


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def smallest(dtype):
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps  # half a subnormal step and more


# -------------------------------------------------------------------- scoring
def scores(logits, targets, k):
    """(logprob, entropy, top logprobs, top ids, log-softmax) in FP64."""
    z = logits.double() + 0.0
    m = z.amax(1, keepdim=True)
    empty = (m == -torch.inf)[:, 0]
    base = torch.where(m == -torch.inf, torch.zeros_like(m), m)
    d = z - base
    s = d.exp().sum(1, keepdim=True)
    logp = d - s.log()
    p = logp.exp()
    entropy = -(p * torch.where(p > 0, logp, torch.zeros_like(p))).sum(1)
    bad = ~(m < torch.inf)[:, 0]
    entropy = torch.where(empty, torch.zeros_like(entropy), entropy)
    entropy = torch.where(bad, torch.full_like(entropy, torch.nan), entropy)
    logp = torch.where(empty[:, None], torch.full_like(logp, -torch.inf), logp)
    logp = torch.where(bad[:, None], torch.full_like(logp, torch.nan), logp)
    lp = logp.gather(1, targets.clamp(0, z.shape[1] - 1)[:, None])[:, 0]
    lp = torch.where(targets < 0, torch.zeros_like(lp), lp)
    lp = torch.where(targets >= z.shape[1], torch.full_like(lp, torch.nan), lp)
    ids = torch.sort(z, dim=1, descending=True, stable=True).indices[:, :k]
    return lp, entropy, logp.gather(1, ids), ids, logp


def score_bound(logits):
    """Absolute error of ln s and u/s per row: e^d has a few 2^-23 of relative error, a
    thread adds V/256 + 1 of them in order (a part at most), and 5 + 8 + 7 joins follow."""
    V = logits.shape[1]
    z = logits.double()
    finite = torch.where(z.isfinite(), z, torch.zeros_like(z))
    spread = (finite.amax(1) - finite.amin(1)).clamp(max=200.0)
    rel = (V / 256 + 24) * U + 2.0 ** -21
    return rel * (2 + spread) + 4 * U * spread


def check_scores(got, logits, targets, k):
    lp, ent, top, ids, _ = scores(logits, targets, k)
    bound = score_bound(logits)
    z = logits.double()
    wide = torch.where(z.isfinite(), z, torch.zeros_like(z))
    size = 4 * U * (wide.amax(1) - wide.amin(1))  # (z - m) - ln s in FP32
    close(got.logprob, lp, bound + size)
    close(got.entropy, ent, bound)
    assert torch.equal(got.top_ids, ids)
    close(got.top_logprobs, top, (bound + size)[:, None])
    assert got.top_ids.dtype == torch.int64 and got.logprob.dtype == torch.float32


def score_grad(logits, targets, dlogprob, dentropy):
    _, ent, _, _, logp = scores(logits, targets, 1)
    empty = torch.isneginf(logp).all(1)
    p = logp.exp()
    lp = torch.where(p > 0, logp, torch.zeros_like(p))
    a = torch.where(targets >= 0, dlogprob.double(), torch.zeros_like(ent))
    hot = torch.zeros_like(p)
    rows = torch.nonzero((targets >= 0) & (targets < p.shape[1]))[:, 0]
    hot[rows, targets[rows]] = 1.0
    b = torch.zeros_like(ent) if dentropy is None else dentropy.double()
    g = a[:, None] * (hot - p) - b[:, None] * p * (lp + ent[:, None])
    g = torch.where(targets[:, None] >= p.shape[1], torch.full_like(g, torch.nan), g)
    size = a.abs()[:, None] * (hot + p) + b.abs()[:, None] * p * (lp.abs() + ent[:, None].abs() + 1)
    return torch.where(empty[:, None], torch.zeros_like(g), g), size


def close(got, want, bound):
    """|got - want| <= bound where want is finite, the same infinities and NaN elsewhere."""
    got, want = got.double(), want.double()
    assert got.shape == want.shape
    fine = want.isfinite()
    assert torch.equal(fine, got.isfinite()), "other infinities or NaN"
    assert torch.equal(want.isnan(), got.isnan())
    over = torch.where(fine, (got - want).abs() - bound, torch.full_like(want, -1.0))
    over = torch.nan_to_num(over, nan=-1.0)  # bounds of rows without numbers
    assert bool((over <= 0).all()), f"worst excess {over.max().item():.3e} at {int(over.argmax())}"


def rounded(ref, dtype):
    return half_step(dtype) * ref.abs() + smallest(dtype)


# ------------------------------------------------------------------ block joint
def norm(v, eps):
    mean = v.mean(1)
    rstd = (v.var(1, unbiased=False) + eps) ** -0.5
    return (v - mean[:, None]) * rstd[:, None], mean, rstd


def join(x, y, pw, pb, gate, w, b, eps, alpha):
    x, y, pw, pb, gate, w, b = (t.double() for t in (x, y, pw, pb, gate, w, b))
    yhat, mean_y, rstd_y = norm(y, eps)
    u = alpha * x + gate * (yhat * pw + pb)
    uhat, mean_u, rstd_u = norm(u, eps)
    return u, uhat * w + b, torch.stack([mean_y, rstd_y, mean_u, rstd_u])


def norm_grad(g, hat, rstd):
    return rstd[:, None] * (g - g.mean(1, keepdim=True) - hat * (g * hat).mean(1, keepdim=True))


def join_grad(dh, du, u, y, stats, pw, pb, gate, w, alpha):
    """Gradients in the order of JoinGrads (without h), and the size of the terms behind each."""
    dh, u, y, pw, pb, gate, w, stats = (t.double() for t in (dh, u, y, pw, pb, gate, w, stats))
    uhat = (u - stats[2][:, None]) * stats[3][:, None]
    yhat = (y - stats[0][:, None]) * stats[1][:, None]
    a = dh * w
    dt = norm_grad(a, uhat, stats[3])
    big = stats[3][:, None] * _terms(a, uhat)
    if du is not None:
        dt = dt + du.double()
        big = big + du.double().abs()
    dn = dt * gate
    c = dn * pw
    dy = norm_grad(c, yhat, stats[1])
    big_c = big * (gate * pw).abs()
    # hat itself is off by a few half steps of |u| rstd
    off_u = (u.abs() + stats[2].abs()[:, None]) * stats[3][:, None]
    off_y = (y.abs() + stats[0].abs()[:, None]) * stats[1][:, None]
    big_dy = stats[1][:, None] * (big_c.amax(1, keepdim=True) * (2 + off_y + yhat.abs() * yhat.abs().amax(1, keepdim=True)))
    return ((alpha * dt, dy, (dn * yhat).sum(0), dn.sum(0), (dt * (yhat * pw + pb)).sum(0), (dh * uhat).sum(0),
             dh.sum(0)),
            (abs(alpha) * big, big_dy, (big * gate.abs() * (off_y + 1)).sum(0), (big * gate.abs()).sum(0),
             (big * ((off_y + 1) * pw.abs() + pb.abs())).sum(0), (dh.abs() * (off_u + 1)).sum(0), dh.abs().sum(0)))


def _terms(a, hat):
    """Magnitude of a - <a> - hat <a hat>, with every term positive and its row's largest factor."""
    return a.abs() + a.abs().mean(1, keepdim=True) + (hat.abs() + 1) * (a * hat).abs().mean(1, keepdim=True) \
        + (a.abs() * (hat.abs() + 1)).mean(1, keepdim=True) * hat.abs()


# ------------------------------------------------------------ 8-bit activations
def kept(x):
    """Nearest E4M3 value (ties to even) under the group's power of two, in FP64."""
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for lo in range(0, x.shape[1], GROUP):
        v = x[:, lo:lo + GROUP].double()
        a = torch.where(v.isfinite(), v.abs(), torch.zeros_like(v)).amax(1, keepdim=True)
        unit = torch.full_like(a, 2.0 ** -126)
        for _ in range(250):
            unit = torch.where(a > 448.0 * unit, unit * 2, unit)
        s = v / unit
        s = torch.where(unit >= 2.0 ** 120, s.clamp(-240, 240), s)  # the next code up is 2^128
        step = torch.exp2(torch.floor(torch.log2(s.abs().clamp(min=2.0 ** -6)))) / 8
        q = torch.round(s / step) * step * unit
        out[:, lo:lo + GROUP] = torch.where(v.isfinite(), q, torch.full_like(q, torch.nan))
    return out


def gelu(v):
    """v Phi(v) in FP64, by erfc: 1 + erf loses all digits of Phi below about -8."""
    phi = 0.5 * torch.special.erfc(-v * 0.5 ** 0.5)
    return torch.where(v.isinf(), v.clamp(min=0), v * torch.where(v.isinf(), torch.zeros_like(v), phi))


def gelu_bound(v, gelu, dtype):
    """v Phi(v) with Phi in FP32: e^x and erfcx are good to a few steps, 16 half steps in
    all; and a Phi below 2^-126 (|v| > 13) is itself off by up to half a subnormal step,
    2^-150, and two more from e^x and the product, all of it times |v|."""
    size = torch.where(v.isfinite(), v.abs(), torch.zeros_like(v))
    return rounded(gelu, dtype) + 16 * U * gelu.abs() + size * 3 * 2.0 ** -150
