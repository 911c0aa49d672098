"""Vocab-parallel cross-entropy (FP32 statistics over BF16 logits).

Forward per row: max over the local vocabulary shard -> all-reduce MAX;
sum exp(x - max) and the target logit (if local) -> one all-reduce SUM of both;
loss = log(sum) + max - target.  Backward writes dlogits = (softmax - onehot) *
scale in place over the logits (they are dead after the loss).
Semantics: VocabCrossEntropy, TempName-5090 python/flux_5090/model.py:143-176.

Scoring (`token_logprobs`): per row the log probability of a given token, the
entropy of the row and its most probable alternatives, from one pass over the
logits; `token_logprobs_backward` is the gradient of log probability and entropy
(weighted, policy and entropy-regularised losses).  Vocabulary-parallel ranks
exchange one small record a row.
"""
from __future__ import annotations

from typing import NamedTuple

import torch
import torch.distributed as dist

from .._native import count_launch, lib


class CEState:
    __slots__ = ("gmax", "sumexp", "start", "rows")

    def __init__(self, gmax, sumexp, start, rows):
        self.gmax, self.sumexp, self.start, self.rows = gmax, sumexp, start, rows


def forward(logits: torch.Tensor, targets: torch.Tensor, group=None, rank: int = 0, world: int = 1,
            scale: float | None = None):
    """Return (mean loss scalar tensor [fp32], state).  `scale` defaults to 1/rows."""
    M, V = logits.shape
    start = rank * V
    scale = 1.0 / M if scale is None else scale
    if logits.is_cuda:
        dev = logits.device
        stats = torch.empty((3, M), dtype=torch.float32, device=dev)
        rowmax, both = stats[0], stats[1:]
        lib().ce_stats(logits, targets, start, rowmax, both[1])
        count_launch()
        if world > 1:
            dist.all_reduce(rowmax, op=dist.ReduceOp.MAX, group=group)
        lib().ce_sumexp(logits, rowmax, both[0])
        count_launch()
        if world > 1:
            dist.all_reduce(both, group=group)
        loss = torch.empty(1, dtype=torch.float32, device=dev)
        lib().ce_loss(rowmax, both[0], both[1], None, loss, scale)
        count_launch()
        return loss, CEState(rowmax, both[0], start, M)
    work = logits.float()
    gmax = work.max(-1).values
    if world > 1:
        dist.all_reduce(gmax, op=dist.ReduceOp.MAX, group=group)
    exps = (work - gmax[:, None]).exp()
    denom = exps.sum(-1)
    local = targets - start
    mask = (local >= 0) & (local < V)
    picked = work.gather(1, local.clamp(0, V - 1)[:, None]).squeeze(1) * mask
    if world > 1:
        both = torch.stack([denom, picked])
        dist.all_reduce(both, group=group)
        denom, picked = both[0], both[1]
    loss = ((denom.log() + gmax - picked).sum() * scale).reshape(1)
    return loss, CEState(gmax, denom, start, M)


def backward(logits: torch.Tensor, targets: torch.Tensor, state: CEState, scale: float):
    """In place: logits <- (softmax - onehot) * scale (BF16)."""
    M, V = logits.shape
    if logits.is_cuda:
        lib().ce_bwd(logits, targets, state.start, state.gmax, state.sumexp, scale, None)
        count_launch()
        return logits
    p = (logits.float() - state.gmax[:, None]).exp() / state.sumexp[:, None]
    local = targets - state.start
    mask = (local >= 0) & (local < V)
    rows = torch.arange(M)
    p[rows[mask], local[mask]] -= 1.0
    logits.copy_((p * scale).to(logits.dtype))
    return logits


# ------------------------------------------------------------------- scoring
MAX_TOP = 32
SCORE_DTYPES = (torch.bfloat16, torch.float16, torch.float32)


class TokenScores(NamedTuple):
    """Per row, FP32: log probability of the given token, entropy (nats), and the
    `top_k` most probable tokens (descending, ties to the lowest id)."""
    logprob: torch.Tensor        # [M]
    entropy: torch.Tensor        # [M]
    top_logprobs: torch.Tensor   # [M, top_k]
    top_ids: torch.Tensor        # [M, top_k] int64, ids of the whole vocabulary


class ScoreState:
    """What the gradient needs beside the logits: max, log of the sum and entropy of
    each row over the whole vocabulary ([3, M]), and this rank's place in it."""
    __slots__ = ("stats", "start", "vocab")

    def __init__(self, stats, start, vocab):
        self.stats, self.start, self.vocab = stats, start, vocab


def _check_scoring(logits, targets, top_k=0, world=1):
    if logits.dim() != 2 or logits.dtype not in SCORE_DTYPES:
        raise ValueError("logits must be a BF16, FP16 or FP32 matrix [rows, vocabulary]")
    if logits.shape[1] == 0:
        raise ValueError("scoring needs a vocabulary")
    if logits.shape[1] > 1 and logits.stride(1) != 1:
        raise ValueError("logits need contiguous rows")
    if targets.dtype != torch.int64 or targets.shape != logits.shape[:1] or targets.device != logits.device:
        raise ValueError("targets must be int64 [rows] on the logits' device")
    most = min(MAX_TOP, logits.shape[1])
    if not 0 <= top_k <= most:
        raise ValueError(f"top_k must be between 0 and {most}")
    if logits.shape[1] * world > 2 ** 31 - 1:
        raise ValueError("the vocabulary must fit 32-bit ids")


def token_logprobs(logits: torch.Tensor, targets: torch.Tensor, top_k: int = 0, group=None, rank: int = 0,
                   world: int = 1):
    """Return (TokenScores, ScoreState) of logits [M, V/world] (this rank's shard).

    A negative target is not scored (log probability 0, which passes no gradient on
    whatever the row holds; the entropy is the row's all the same); one at or above
    the vocabulary's end gives NaN.  A logit of -inf is a token that cannot occur; a
    row of nothing else has log probability -inf, entropy 0 and no
    gradient.  A NaN or +inf makes its row's numbers NaN.  `top_k` is at most 32
    and at most the shard's vocabulary.
    """
    if logits.is_cuda and world == 1:
        try:
            logprob, entropy, top, ids, stats = lib().token_logprobs(logits, targets, top_k)
        except (RuntimeError, TypeError):
            _check_scoring(logits, targets, top_k)
            raise
        count_launch()
        return TokenScores(logprob, entropy, top, ids), ScoreState(stats, 0, logits.shape[1])
    _check_scoring(logits, targets, top_k, world)
    if not logits.is_cuda:
        return _token_logprobs_cpu(logits, targets, top_k, group, rank, world)
    M, V = logits.shape
    dev = logits.device
    targets = targets.contiguous()
    out = torch.empty(M * (5 + top_k), dtype=torch.float32, device=dev)
    ids = torch.empty((M, top_k), dtype=torch.int64, device=dev)
    if M:
        records = torch.empty((world, M, 4 + 2 * top_k), dtype=torch.float32, device=dev)
        mine = torch.empty((M, 4 + 2 * top_k), dtype=torch.float32, device=dev)
        lib().score_fwd(logits, targets, rank * V, V * world, top_k, None, None, mine)
        dist.all_gather_into_tensor(records, mine, group=group)
        lib().score_merge(records, targets, V, top_k, out, ids)
        count_launch(2)
    scores = TokenScores(out[:M], out[M:2 * M], out[5 * M:].view(M, top_k), ids)
    return scores, ScoreState(out[2 * M:5 * M].view(3, M), rank * V, V * world)


@torch.no_grad()
def _token_logprobs_cpu(logits, targets, top_k, group, rank, world):
    """The same numbers in torch, with the same records between ranks."""
    M, V = logits.shape
    z = logits.float() + 0.0
    m = z.amax(1)
    d = (z - torch.where(m == -torch.inf, torch.zeros(()), m)[:, None])
    e = d.exp()
    s, u = e.sum(1), torch.where(e > 0, e * d, torch.zeros(())).sum(1)
    local = targets - rank * V
    mine = (local >= 0) & (local < V)
    picked = torch.where(mine, z.gather(1, local.clamp(0, V - 1)[:, None])[:, 0], torch.zeros(()))
    values, ids = torch.sort(z, dim=1, descending=True, stable=True)
    values, ids = values[:, :top_k], ids[:, :top_k] + rank * V
    if world > 1:
        record = torch.cat([torch.stack([m, s, u, picked], 1), values], 1).contiguous()
        records = [torch.empty_like(record) for _ in range(world)]
        dist.all_gather(records, record, group=group)
        everyone = [torch.empty_like(ids) for _ in range(world)]
        dist.all_gather(everyone, ids.contiguous(), group=group)
        r = torch.stack(records)
        m = r[:, :, 0].amax(0)
        shift = (r[:, :, 0] - torch.where(m == -torch.inf, torch.zeros(()), m)).clamp(min=-200.0)
        f = shift.exp()
        s, u = (r[:, :, 1] * f).sum(0), ((r[:, :, 2] + shift * r[:, :, 1]) * f).sum(0)
        picked = r[:, :, 3].sum(0)
        values, order = torch.sort(torch.cat(list(r[:, :, 4:]), 1), dim=1, descending=True, stable=True)
        values, ids = values[:, :top_k], torch.cat(everyone, 1).gather(1, order[:, :top_k])
    nan = torch.full((), float("nan"))
    bad, empty = ~(m < torch.inf), m == -torch.inf
    log_s = torch.where(empty, torch.zeros(()), s.log())
    logprob = torch.where(empty, -torch.inf, (picked - m) - log_s)
    entropy = torch.where(empty, torch.zeros(()), log_s - u / s)
    top = torch.where(empty[:, None], -torch.inf, (values - m[:, None]) - log_s[:, None])
    logprob, entropy, m = (torch.where(bad, nan, t) for t in (logprob, entropy, m))
    top = torch.where(bad[:, None], nan, top)
    logprob = torch.where(targets < 0, torch.zeros(()), torch.where(targets >= V * world, nan, logprob))
    return (TokenScores(logprob, entropy, top, ids),
            ScoreState(torch.stack([m, log_s, entropy]), rank * V, V * world))


def token_logprobs_backward(logits: torch.Tensor, targets: torch.Tensor, state: ScoreState,
                            dlogprob: torch.Tensor, dentropy: torch.Tensor | None = None,
                            out: torch.Tensor | None = None) -> torch.Tensor:
    """Gradient of the logits [M, V/world] from that of the log probabilities and
    (optional) of the entropies, both FP32 [M].  `out` may be the logits themselves,
    which are dead after the loss; otherwise it must not overlap them."""
    if logits.is_cuda:
        try:
            out = lib().token_logprobs_backward(logits, targets, state.start, state.vocab, state.stats, dlogprob,
                                                dentropy, out)
        except (RuntimeError, TypeError):
            _check_score_gradient(logits, targets, state, dlogprob, dentropy, out)
            raise
        count_launch()
        return out
    _check_score_gradient(logits, targets, state, dlogprob, dentropy, out)
    return _score_gradient_cpu(logits, targets, state, dlogprob, dentropy, out)


def _check_score_gradient(logits, targets, state, dlogprob, dentropy, out):
    _check_scoring(logits, targets)
    M, V = logits.shape
    for name, t in (("dlogprob", dlogprob), ("dentropy", dentropy)):
        if t is not None and (t.dtype != torch.float32 or t.shape != (M,) or t.device != logits.device):
            raise ValueError(f"{name} must be FP32 [rows] on the logits' device")
    if state.stats.shape != (3, M) or state.stats.device != logits.device:
        raise ValueError("the state belongs to other logits")
    if out is not None and (out.shape != logits.shape or out.dtype != logits.dtype or out.device != logits.device
                            or (V > 1 and out.stride(1) != 1) or (M > 1 and out.stride(0) < V)):
        raise ValueError("out must be like the logits, with contiguous rows of its own")


@torch.no_grad()
def _score_gradient_cpu(logits, targets, state, dlogprob, dentropy, out):
    M, V = logits.shape
    out = torch.empty((M, V), dtype=logits.dtype) if out is None else out
    m, log_s, entropy = state.stats
    b = torch.zeros(M) if dentropy is None else dentropy
    empty = (m == -torch.inf) | ((targets < 0) & (b == 0))  # no gradient, whatever the logits hold
    a = torch.where(targets >= 0, dlogprob, torch.zeros(()))
    a = torch.where((targets >= state.vocab) | m.isnan(), torch.full((), float("nan")), a)
    logp = ((logits.float() - torch.where(empty, torch.zeros(()), m)[:, None]) - log_s[:, None]).clamp(min=-200.0)
    g = -logp.exp() * (a[:, None] + b[:, None] * (logp + entropy[:, None]))
    local = targets - state.start
    rows = torch.nonzero((local >= 0) & (local < V))[:, 0]
    g[rows, local[rows]] += a[rows]
    out.copy_(torch.where(empty[:, None], torch.zeros(()), g))
    return out
