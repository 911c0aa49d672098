"""Scores of finite logits of any magnitude against 64 bits."""
import pytest
import torch

import operators_reference as ref

pytestmark = pytest.mark.gpu
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(seed, *shape, std=1.0, to=BF16):
    return (torch.randn(shape, generator=gen(seed), device="cuda") * std).to(to)


def ops():
    from tempname_5090_b200.ops import actpack, loss, norm
    return actpack, loss, norm


FILLS = {BF16: [-1e5, -4e6, -5e6, -1e7, -1.5e7, -2e7, -5e7, -1e8, -1e9, -3e9, -1e10, -1e15, -1e20, -1e28, -2e29,
                1e5, 4e6, 5e6, 1e7, 1e9, 3e9, 1e10, 1e20, 1e28],
         FP16: [-1e4, -5.9e4, -6.1e4, -65504.0, 1e4, 6e4, 65504.0]}
FILLS[FP32] = FILLS[BF16]


def filled(fill, V, dtype, seed):
    """Rows in which a large value is all there is, masks all but a few tokens, a third of
    them or one, stands once among ordinary ones, or is what the row's values lie around."""
    z = randn(seed, 6, V, std=3.0, to=FP32)
    z[0] = fill
    z[1, 4:] = fill
    z[2, :V - V // 3] = fill
    z[3, :V // 2], z[3, V // 2 + 1:] = fill, fill
    z[4, V // 3] = fill
    z[5] = fill + z[5] * max(1.0, abs(fill) * 2.0 ** -22)
    return z.clamp(torch.finfo(dtype).min, torch.finfo(dtype).max).to(dtype)


def rows_of(V, dtype):
    z = torch.cat([filled(f, V, dtype, 30 + n) for n, f in enumerate(FILLS[dtype])])
    t = torch.randint(0, V, (len(z),), generator=gen(29), device="cuda")
    return z, torch.where(torch.arange(len(z), device="cuda") % 2 == 0, t, z.float().argmax(1))


def check_gradient(g, z, t, a, b, dtype):
    want, size = ref.score_grad(z, t, a, b)
    # A probability below 2^-126 (ln p < -87.3) is taken as zero.  What that leaves out of
    # a p + b p (ln p + H) is less than 2^-126 (|a| + |b| (88 + H)): p |ln p| falls with p there.
    entropy = ref.scores(z, t, 1)[1]
    flushed = 2.0 ** -126 * (a.double().abs() + b.double().abs() * (88 + entropy))
    ref.close(g, want, ref.rounded(want, dtype) + (ref.score_bound(z)[:, None] + 64 * ref.U) * 2 * size
              + flushed[:, None])


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("V", [100, 9001])
@pytest.mark.parametrize("k", [0, 1, 20])
def test_scores_of_large_logits(V, k, dtype):
    """Any finite logits: whole rows and masks of any magnitude."""
    _, loss, _ = ops()
    z, t = rows_of(V, dtype)
    a, b = randn(27, len(z), to=FP32), randn(28, len(z), to=FP32)
    # all rows at once (a CTA a row), then as many as are split over a cluster's CTAs
    for part in [slice(0, len(z))] + [slice(n, n + 36) for n in range(0, len(z), 36)]:
        zp, tp = z[part], t[part]
        got, state = loss.token_logprobs(zp, tp, top_k=k)
        ref.check_scores(got, zp, tp, k)
        check_gradient(loss.token_logprobs_backward(zp, tp, state, a[part], b[part]), zp, tp, a[part], b[part], dtype)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("world", [2, 8])
def test_merged_records_of_large_logits(world, dtype):
    _, loss, _ = ops()
    from tempname_5090_b200._native import lib
    V, k = 8 * 512, 9
    z, t = rows_of(V, dtype)
    rows, Vl = len(z), V // world
    records = torch.empty((world, rows, 4 + 2 * k), device="cuda")
    for r in range(world):
        lib().score_fwd(z[:, r * Vl:(r + 1) * Vl], t, r * Vl, V, k, None, None, records[r])
    out = torch.empty(rows * (5 + k), device="cuda")
    ids = torch.empty((rows, k), dtype=torch.int64, device="cuda")
    lib().score_merge(records, t, Vl, k, out, ids)
    ref.check_scores(loss.TokenScores(out[:rows], out[rows:2 * rows], out[5 * rows:].view(rows, k), ids), z, t, k)
    a, b = randn(27, rows, to=FP32), randn(28, rows, to=FP32)
    parts = [loss.token_logprobs_backward(z[:, r * Vl:(r + 1) * Vl], t,
                                          loss.ScoreState(out[2 * rows:5 * rows].view(3, rows), r * Vl, V), a, b)
             for r in range(world)]
    check_gradient(torch.cat(parts, 1), z, t, a, b, dtype)
