"""Cases of the operators around GPT's matrix products: scoring of given tokens
(log probability, entropy, top alternatives, and the gradient), the joint of two
blocks (norm of the branch, gate, residual scale and the next norm in one pass,
and its gradient), and activations kept in 8 bits for the backward pass.

`run` computes them in plain torch operations, or calls the package where `own`
is true.  `exact` states the definitions in 64 bits.
"""
import math

import torch

own = False

BF16, FP16, FP32 = "bf16", "fp16", "fp32"
TYPES = {BF16: torch.bfloat16, FP16: torch.float16, FP32: torch.float32}
BYTES = {BF16: 2, FP16: 2, FP32: 4}
EPS = 1e-5
GROUP = 128          # values that share an exponent in the 8-bit form
MOST = 8192 * 50304  # logits of the largest listed case
LARGE = 8192 * 4096  # residual-stream values of one step of the benchmark


def listed():
    return [
        # one token's answer: a row of the benchmark's vocabulary, the calls that count in latency
        dict(name="score_1x50304_top20", op="score", rows=1, vocab=50304, top_k=20, dtype=BF16),
        # a whole benchmark batch scored in evaluation, prompt tokens ignored
        dict(name="score_8192x50304_top8", op="score", rows=8192, vocab=50304, top_k=8, dtype=BF16),
        # a policy step over one sequence of the benchmark: weighted log probabilities and entropy, with the gradient
        dict(name="score_grad_2048x50304", op="score_grad", rows=2048, vocab=50304, top_k=0, dtype=BF16),
        # an odd vocabulary and FP32 logits, no row on a 16-byte boundary but the first
        dict(name="score_grad_517x32003_fp32", op="score_grad", rows=517, vocab=32003, top_k=0, dtype=FP32),
        # the joint for a few rows (a short sequence, or one rank's share of it)
        dict(name="join_128x4096", op="join", rows=128, hidden=4096, scale=1.0, dtype=BF16),
        # the joint of the benchmark step
        dict(name="join_8192x4096", op="join", rows=8192, hidden=4096, scale=0.9, dtype=BF16),
        # an odd width in FP32
        dict(name="join_grad_1000x1001_fp32", op="join_grad", rows=1000, hidden=1001, scale=0.7, dtype=FP32),
        dict(name="join_grad_8192x4096", op="join_grad", rows=8192, hidden=4096, scale=0.9, dtype=BF16),
        # the MLP's pre-activation of the small test configuration's kind, ragged last group
        dict(name="mlp_kept_300x1100", op="mlp_kept", rows=300, hidden=1100, dtype=BF16),
        # the benchmark's pre-activation of one layer
        dict(name="mlp_kept_8192x16384", op="mlp_kept", rows=8192, hidden=16384, dtype=BF16),
        # LayerNorm's input kept in 8 bits, and its backward pass from there
        dict(name="norm_kept_777x2050", op="norm_kept", rows=777, hidden=2050, dtype=BF16),
        dict(name="norm_kept_8192x4096", op="norm_kept", rows=8192, hidden=4096, dtype=BF16),
    ]


def _log_uniform(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["score", "score_grad", "join", "join_grad", "mlp_kept", "norm_kept"])
    if op in ("score", "score_grad"):
        dtype = rng.choice([BF16, BF16, FP16, FP32])
        vocab = _log_uniform(rng, 1000, 50304)
        room = MOST // (vocab * (4 if op == "score_grad" else 1) * (2 if dtype == FP32 else 1))
        return dict(op=op, rows=_log_uniform(rng, 1, min(8192, room)), vocab=vocab,
                    top_k=rng.randint(1, 32) if op == "score" else 0, dtype=dtype)
    dtype = rng.choice([BF16, BF16, FP32])
    hidden = _log_uniform(rng, 64, 16384 if op == "mlp_kept" else 8192)
    room = LARGE // (hidden * (2 if dtype == FP32 else 1))
    case = dict(op=op, rows=_log_uniform(rng, 1, min(8192, room)), hidden=hidden, dtype=dtype)
    if op in ("join", "join_grad"):
        case["scale"] = round(rng.uniform(0.5, 1.5), 3)
    return case


def work(case):
    size, rows = BYTES[case["dtype"]], case["rows"]
    if case["op"] == "score":
        n = rows * case["vocab"]
        return {"bytes": n * size + rows * (8 + 8 + 12 * case["top_k"]), "flops": 5 * n}
    if case["op"] == "score_grad":
        n = rows * case["vocab"]
        return {"bytes": 2 * n * size + rows * 24, "flops": 11 * n}
    hidden = case["hidden"]
    n = rows * hidden
    kept = rows * (hidden + (hidden + GROUP - 1) // GROUP)
    if case["op"] == "join":
        return {"bytes": 4 * n * size + 5 * hidden * size + 16 * rows, "flops": 17 * n}
    if case["op"] == "join_grad":
        return {"bytes": 6 * n * size + 9 * hidden * size + 16 * rows, "flops": 34 * n}
    if case["op"] == "mlp_kept":  # written once and read once in 8 bits, between the two passes
        return {"bytes": 3 * n * size + 2 * kept, "flops": 12 * n}
    return {"bytes": 5 * n * size + 2 * kept + 4 * hidden * size + 8 * rows, "flops": 20 * n}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype, rows = TYPES[case["dtype"]], case["rows"]

    def normal(*shape, std=1.0, mean=0.0, to=dtype):
        return torch.randn(shape, generator=g, device="cuda").mul_(std).add_(mean).to(to)

    s = dict(case)
    if case["op"] in ("score", "score_grad"):
        vocab = case["vocab"]
        logits = torch.empty((rows, vocab), dtype=dtype, device="cuda")
        for part in logits.split(1024):
            part.copy_(torch.randn(part.shape, generator=g, device="cuda").mul_(2.5))
        targets = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
        # a trained model favours the given token in most rows, and prompt tokens are not scored
        lift = torch.rand(rows, generator=g, device="cuda") * 12
        at = torch.arange(rows, device="cuda")
        logits[at, targets] = (logits[at, targets].float() + lift).to(dtype)
        if rows > 8:
            targets[torch.rand(rows, generator=g, device="cuda") < 0.1] = -100
        s.update(logits=logits, targets=targets)
        if case["op"] == "score_grad":
            s["dlogprob"] = normal(rows, to=torch.float32) / rows
            s["dentropy"] = torch.full((rows,), 0.01 / rows, device="cuda")
        return s
    hidden = case["hidden"]
    if case["op"] == "mlp_kept":
        s["pre"] = normal(rows, hidden, std=1.3)
        return s
    # residual stream: a few channels an order of magnitude above the rest, and an offset
    spread = torch.exp(0.7 * torch.randn(hidden, generator=g, device="cuda"))
    x = (torch.randn((rows, hidden), generator=g, device="cuda") * spread + 0.2).to(dtype)
    s.update(x=x, pre_weight=normal(hidden, std=0.2, mean=1.0), pre_bias=normal(hidden, std=0.1))
    if case["op"] == "norm_kept":
        wide = x.double()
        s["mean"] = wide.mean(1).float()
        s["rstd"] = torch.rsqrt(wide.var(1, unbiased=False) + EPS).float()
        s.update(dy=normal(rows, hidden), dres=normal(rows, hidden))
        return s
    s.update(y=normal(rows, hidden, std=0.6, mean=0.1), post_weight=normal(hidden, std=0.2, mean=1.0),
             post_bias=normal(hidden, std=0.1), gate=normal(hidden, std=0.3, mean=0.5))
    if case["op"] == "join_grad":
        joined, _, stats = _join(s)
        s.update(x_out=joined.to(dtype), stats=stats, dh=normal(rows, hidden), dx_out=normal(rows, hidden))
        del s["x"]
    return s


# ------------------------------------------------------------- plain forms
def _score(s):
    z, targets, k = s["logits"].float(), s["targets"], s["top_k"]
    vocab = z.shape[1]
    top = z.max(1, keepdim=True).values
    shifted = z - top
    e = shifted.exp()
    total = e.sum(1)
    log_total = total.log()
    entropy = log_total - (e * shifted).sum(1) / total
    given = targets >= 0
    picked = shifted.gather(1, targets.clamp(min=0)[:, None])[:, 0]
    out = dict(logprob=torch.where(given, picked - log_total, torch.zeros_like(picked)), entropy=entropy)
    if k:
        # whole numbers in the order of the values, lower indices first among equal ones
        order = (s["logits"].float() + 0.0).view(torch.int32)
        order = torch.where(order < 0, order ^ 0x7FFFFFFF, order).to(torch.int64)
        order.mul_(1 << 20).sub_(torch.arange(vocab, device=z.device))
        keys = order.topk(k, dim=1).values
        out["top_ids"] = (-keys) & ((1 << 20) - 1)
        out["top_logprobs"] = shifted.gather(1, out["top_ids"]) - log_total[:, None]
    return out, shifted - log_total[:, None]


def _score_grad(s):
    out, logp = _score(s)
    p = logp.exp()
    up = torch.where(s["targets"] >= 0, s["dlogprob"], torch.zeros_like(s["dlogprob"]))
    dz = -p * (up[:, None] + s["dentropy"][:, None] * (logp + out["entropy"][:, None]))
    dz.scatter_add_(1, s["targets"].clamp(min=0)[:, None], up[:, None])
    return dict(logprob=out["logprob"], entropy=out["entropy"], dlogits=dz.to(s["logits"].dtype))


def _normed(v):
    mean = v.mean(1)
    centred = v - mean[:, None]
    rstd = torch.rsqrt((centred * centred).mean(1) + EPS)
    return centred * rstd[:, None], mean, rstd


def _join(s):
    branch, mean_y, rstd_y = _normed(s["y"].float())
    branch = branch * s["post_weight"].float() + s["post_bias"].float()
    joined = s["scale"] * s["x"].float() + s["gate"].float() * branch
    h, mean_x, rstd_x = _normed(joined)
    h = h * s["pre_weight"].float() + s["pre_bias"].float()
    return joined, h, torch.stack([mean_y, rstd_y, mean_x, rstd_x])


def _norm_grad(g, xhat, rstd):
    """The gradient of a norm's input from that of its normed values."""
    return rstd[:, None] * (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True))


def _join_grad(s):
    mean_y, rstd_y, mean_x, rstd_x = s["stats"]
    xhat = (s["x_out"].float() - mean_x[:, None]) * rstd_x[:, None]
    yhat = (s["y"].float() - mean_y[:, None]) * rstd_y[:, None]
    post_w, post_b, gate, pre_w = (s[n].float() for n in ("post_weight", "post_bias", "gate", "pre_weight"))
    dh = s["dh"].float()
    total = s["dx_out"].float() + _norm_grad(dh * pre_w, xhat, rstd_x)
    inner = total * gate
    to = s["y"].dtype
    return dict(dx=(s["scale"] * total).to(to), dy=_norm_grad(inner * post_w, yhat, rstd_y).to(to),
                dpost_weight=(inner * yhat).sum(0).to(to), dpost_bias=inner.sum(0).to(to),
                dgate=(total * (yhat * post_w + post_b)).sum(0).to(to),
                dpre_weight=(dh * xhat).sum(0).to(to), dpre_bias=dh.sum(0).to(to))


def _kept(x):
    """The values that the 8-bit form stands for: E4M3 with a power of two for each
    group of 128 along the row, the smallest that keeps the group within 448."""
    rows, cols = x.shape
    groups = torch.nn.functional.pad(x.float(), (0, -cols % GROUP)).view(rows, -1, GROUP)
    fraction, exponent = torch.frexp(groups.abs().amax(2, keepdim=True))
    exponent = torch.where(fraction > 0.875, exponent - 8, exponent - 9).clamp(min=-126)
    codes = torch.ldexp(groups, -exponent).to(torch.float8_e4m3fn)
    return torch.ldexp(codes.float(), exponent).reshape(rows, -1)[:, :cols]


def _mlp_kept(s):
    pre = _kept(s["pre"])
    act = 0.5 * pre * (1.0 + torch.erf(pre * math.sqrt(0.5)))
    return dict(pre=pre.to(s["pre"].dtype), act=act.to(s["pre"].dtype))


def _norm_kept(s):
    xhat = (_kept(s["x"]) - s["mean"][:, None]) * s["rstd"][:, None]
    w, dy, to = s["pre_weight"].float(), s["dy"].float(), s["x"].dtype
    dx = s["dres"].float() + _norm_grad(dy * w, xhat, s["rstd"])
    return dict(dx=dx.to(to), dweight=(dy * xhat).sum(0).to(to), dbias=dy.sum(0).to(to),
                y=(xhat * w + s["pre_bias"].float()).to(to))


# ------------------------------------------------------- the package's calls
def _own(s):
    from tempname_5090_b200.ops import actpack, loss, norm
    op = s["op"]
    if op == "score":
        scores, _ = loss.token_logprobs(s["logits"], s["targets"], top_k=s["top_k"])
        return dict(logprob=scores.logprob, entropy=scores.entropy, top_ids=scores.top_ids,
                    top_logprobs=scores.top_logprobs)
    if op == "score_grad":
        scores, state = loss.token_logprobs(s["logits"], s["targets"])
        dlogits = loss.token_logprobs_backward(s["logits"], s["targets"], state, s["dlogprob"], s["dentropy"])
        return dict(logprob=scores.logprob, entropy=scores.entropy, dlogits=dlogits)
    if op == "join":
        x_out, h, stats = norm.block_join_fwd(s["x"], s["y"], s["post_weight"], s["post_bias"], s["gate"],
                                              s["pre_weight"], s["pre_bias"], EPS, residual_scale=s["scale"])
        return dict(x_out=x_out, h=h, stats=stats)
    if op == "join_grad":
        grads = norm.block_join_bwd(s["dh"], s["dx_out"], s["x_out"], s["y"], s["stats"], s["post_weight"],
                                    s["post_bias"], s["gate"], s["pre_weight"], residual_scale=s["scale"])
        return dict(dx=grads.dx, dy=grads.dy, dpost_weight=grads.dpost_weight, dpost_bias=grads.dpost_bias,
                    dgate=grads.dgate, dpre_weight=grads.dpre_weight, dpre_bias=grads.dpre_bias)
    if op == "mlp_kept":
        pre, act = actpack.unpack_gelu(actpack.pack(s["pre"]))
        return dict(pre=pre, act=act)
    kept = actpack.pack(s["x"])
    dx, dw, db, y = norm.layer_norm_bwd_packed(s["dy"], kept, s["pre_weight"], s["mean"], s["rstd"],
                                               dres=s["dres"], bias=s["pre_bias"])
    return dict(dx=dx, dweight=dw, dbias=db, y=y)


def run(state):
    if own:
        return _own(state)
    op = state["op"]
    if op == "score":
        return _score(state)[0]
    if op == "score_grad":
        return _score_grad(state)
    if op == "join":
        joined, h, stats = _join(state)
        return dict(x_out=joined.to(state["x"].dtype), h=h.to(state["x"].dtype), stats=stats)
    if op == "join_grad":
        return _join_grad(state)
    return _mlp_kept(state) if op == "mlp_kept" else _norm_kept(state)


# ------------------------------------------------- the definitions in 64 bits
def _exact_score(s, grad):
    found = []
    for lo in range(0, s["logits"].shape[0], 256):
        z, t = s["logits"][lo:lo + 256].double(), s["targets"][lo:lo + 256]
        logp = z - torch.logsumexp(z, 1, keepdim=True)
        p = torch.exp(logp)
        entropy = -(p * logp).sum(1)
        hot = torch.zeros_like(z)
        rows = torch.nonzero(t >= 0)[:, 0]
        hot[rows, t[rows]] = 1.0
        part = dict(logprob=(hot * logp).sum(1), entropy=entropy)
        if s["top_k"]:
            ids = torch.sort(z, dim=1, descending=True, stable=True).indices[:, :s["top_k"]]
            part.update(top_ids=ids, top_logprobs=torch.take_along_dim(logp, ids, 1))
        if grad:
            # d logprob_t / dz = onehot - p;  d entropy / dz = -p (log p + entropy)
            a, b = s["dlogprob"][lo:lo + 256].double()[:, None], s["dentropy"][lo:lo + 256].double()[:, None]
            scored = (t >= 0).double()[:, None]
            part["dlogits"] = a * (hot - scored * p) - b * p * (logp + entropy[:, None])
        found.append(part)
    return {k: torch.cat([part[k] for part in found]) for k in found[0]}


def _exact_kept(x):
    """Nearest E4M3 value, ties to even: steps of an eighth of the power of two below, of 2^-9 under 2^-6."""
    wide = x.double()
    out = torch.empty_like(wide)
    for lo in range(0, x.shape[1], GROUP):
        v = wide[:, lo:lo + GROUP]
        most = v.abs().max(1, keepdim=True).values
        unit = torch.exp2(torch.ceil(torch.log2((most / 448.0).clamp(min=2.0 ** -126))))
        unit = torch.where(most > 448.0 * unit, unit * 2, unit)
        unit = torch.where((most <= 224.0 * unit) & (unit > 2.0 ** -126), unit / 2, unit)
        scaled = v / unit
        below = torch.exp2(torch.floor(torch.log2(scaled.abs().clamp(min=2.0 ** -6))))
        out[:, lo:lo + GROUP] = torch.round(scaled / (below / 8)) * (below / 8) * unit
    return out


def _layer_norm_and_grad(v, w, dout, mean, rstd):
    hat = (v - mean.double()[:, None]) * rstd.double()[:, None]
    a = dout * w
    n = v.shape[1]
    dv = (a - (a.sum(1) / n)[:, None] - hat * ((a * hat).sum(1) / n)[:, None]) * rstd.double()[:, None]
    return dv, torch.einsum("rc,rc->c", dout, hat), dout.sum(0), hat


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("score", "score_grad"):
        return _exact_score(s, case["op"] == "score_grad")
    d = {k: v.double() for k, v in s.items() if isinstance(v, torch.Tensor)}
    if case["op"] == "join":
        var_y, mean_y = torch.var_mean(d["y"], 1, unbiased=False)
        rstd_y = (var_y + EPS) ** -0.5
        normed = (d["y"] - mean_y[:, None]) * rstd_y[:, None] * d["post_weight"] + d["post_bias"]
        x_out = case["scale"] * d["x"] + d["gate"] * normed
        var_x, mean_x = torch.var_mean(x_out, 1, unbiased=False)
        rstd_x = (var_x + EPS) ** -0.5
        h = (x_out - mean_x[:, None]) * rstd_x[:, None] * d["pre_weight"] + d["pre_bias"]
        return dict(x_out=x_out, h=h, stats=torch.stack([mean_y, rstd_y, mean_x, rstd_x]))
    if case["op"] == "join_grad":
        mean_y, rstd_y, mean_x, rstd_x = s["stats"]
        dstream, dpre_w, dpre_b, _ = _layer_norm_and_grad(d["x_out"], d["pre_weight"], d["dh"], mean_x, rstd_x)
        dstream = dstream + d["dx_out"]
        dbranch = dstream * d["gate"]
        dy, dpost_w, dpost_b, yhat = _layer_norm_and_grad(d["y"], d["post_weight"], dbranch, mean_y, rstd_y)
        dgate = torch.einsum("rc,rc->c", dstream, yhat * d["post_weight"] + d["post_bias"])
        return dict(dx=case["scale"] * dstream, dy=dy, dpost_weight=dpost_w, dpost_bias=dpost_b, dgate=dgate,
                    dpre_weight=dpre_w, dpre_bias=dpre_b)
    if case["op"] == "mlp_kept":
        kept = _exact_kept(s["pre"])
        return dict(pre=kept, act=kept * torch.special.ndtr(kept))
    dx, dw, db, xhat = _layer_norm_and_grad(_exact_kept(s["x"]), d["pre_weight"], d["dy"], s["mean"], s["rstd"])
    return dict(dx=dx + d["dres"], dweight=dw, dbias=db, y=xhat * d["pre_weight"] + d["pre_bias"])
