"""Scoring, block joint and 8-bit activations on CPU: the torch statements against
64 bits and against differences, two Gloo ranks against one, and every refusal."""
import math
import os
import socket
import tempfile

import pytest
import torch

import operators_reference as ref
from tempname_5090_b200.ops import actpack, loss, norm

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def gen(seed):
    return torch.Generator().manual_seed(seed)


def randn(seed, *shape, std=1.0, mean=0.0, to=BF16):
    return (torch.randn(shape, generator=gen(seed)) * std + mean).to(to)


# -------------------------------------------------------------------- scoring
def special_logits(dtype=FP32, V=100):
    z = randn(1, 9, V, std=3.0, to=dtype)
    z[1] = -torch.inf                       # nothing left
    z[2, 7:] = -torch.inf                   # a few tokens left
    z[3] = torch.finfo(dtype).min           # the type's lowest value everywhere
    z[4, 5] = torch.nan
    z[5, 6] = torch.inf
    z[6] = 0.25                             # all equal
    z[7, 10:20] = z[7].max() + 1            # ties at the top
    z[8, :50] = torch.finfo(dtype).min
    return z


def test_scores_of_special_rows():
    z = special_logits()
    t = torch.tensor([3, 4, 2, 0, 1, 1, 99, 12, -100])
    got, _ = loss.token_logprobs(z, t, top_k=20)
    fine = torch.tensor([0, 1, 2, 3, 6, 7, 8])  # ids of rows with NaN are checked apart
    ref.check_scores(loss.TokenScores(*(a[fine] for a in got)), z[fine], t[fine], 20)
    assert got.logprob[1] == -math.inf and got.entropy[1] == 0
    assert torch.equal(got.top_ids[1], torch.arange(20))
    assert got.logprob[4].isnan() and got.logprob[5].isnan() and got.entropy[5].isnan()
    assert got.logprob[8] == 0


def test_score_gradient_against_differences():
    z = randn(2, 4, 9, std=2.0, to=FP32)
    t = torch.tensor([0, 8, -1, 4])
    a, b = randn(3, 4, to=FP32), randn(4, 4, to=FP32)
    _, state = loss.token_logprobs(z, t)
    g = loss.token_logprobs_backward(z, t, state, a, b)
    want, size = ref.score_grad(z, t, a, b)
    ref.close(g, want, ref.rounded(want, FP32) + 64 * ref.U * size)

    def value(zz):
        lp, ent, *_ = ref.scores(zz, t, 1)
        return (a.double() * lp + b.double() * ent).sum().item()

    for i, j in ((0, 0), (1, 3), (2, 2), (3, 4), (3, 8)):
        step = torch.zeros(4, 9, dtype=torch.float64)
        step[i, j] = 1e-5
        slope = (value(z.double() + step) - value(z.double() - step)) / 2e-5
        assert abs(slope - g[i, j].item()) < 1e-6 * (1 + abs(slope)) + 64 * ref.U * size[i, j].item()


def _port():
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        return s.getsockname()[1]


def _rank(rank, world, port, out_dir):
    import torch.distributed as dist
    dist.init_process_group("gloo", init_method=f"tcp://127.0.0.1:{port}", rank=rank, world_size=world)
    try:
        z, t, a, b = _parallel_data()
        V = z.shape[1] // world
        shard = z[:, rank * V:(rank + 1) * V].clone()
        got, state = loss.token_logprobs(shard, t, top_k=5, rank=rank, world=world)
        g = loss.token_logprobs_backward(shard, t, state, a, b, out=shard)
        torch.save((tuple(got), g), os.path.join(out_dir, f"{rank}.pt"))
    finally:
        dist.destroy_process_group()


def _parallel_data():
    z = randn(5, 12, 64, std=3.0, to=FP32)
    z[1, :32] = -torch.inf   # a rank with nothing
    z[2] = -torch.inf
    z[3] = 1.0               # ties over both ranks
    t = torch.randint(0, 64, (12,), generator=gen(6))
    t[4], t[5] = -100, 64
    return z, t, randn(7, 12, to=FP32), randn(8, 12, to=FP32)


def test_two_ranks_score_like_one():
    import torch.multiprocessing as mp
    with tempfile.TemporaryDirectory() as d:
        mp.spawn(_rank, args=(2, _port(), d), nprocs=2, join=True)
        res = [torch.load(os.path.join(d, f"{r}.pt")) for r in range(2)]
    z, t, a, b = _parallel_data()
    for got, _ in res:
        ref.check_scores(loss.TokenScores(*got), z, t, 5)
    want, size = ref.score_grad(z, t, a, b)
    ref.close(torch.cat([g for _, g in res], 1), want, ref.rounded(want, FP32) + 64 * ref.U * size)


def test_scoring_refusals():
    z, t = randn(9, 4, 40), torch.zeros(4, dtype=torch.int64)
    _, state = loss.token_logprobs(z, t)
    up = torch.ones(4)
    bad = [lambda: loss.token_logprobs(z[0], t), lambda: loss.token_logprobs(z.long(), t),
           lambda: loss.token_logprobs(z.double(), t),
           lambda: loss.token_logprobs(z.t().contiguous().t(), t), lambda: loss.token_logprobs(z, t[:3]),
           lambda: loss.token_logprobs(z, t.int()), lambda: loss.token_logprobs(z, t, top_k=33),
           lambda: loss.token_logprobs(z, t, top_k=-1), lambda: loss.token_logprobs(z[:, :5], t, top_k=6),
           lambda: loss.token_logprobs(z[:, :0], t),
           lambda: loss.token_logprobs_backward(z, t, state, up.double()),
           lambda: loss.token_logprobs_backward(z, t, state, up[:3]),
           lambda: loss.token_logprobs_backward(z, t, state, up, up[:2]),
           lambda: loss.token_logprobs_backward(z[:3], t[:3], state, up[:3]),
           lambda: loss.token_logprobs_backward(z, t, state, up, out=z.float()),
           lambda: loss.token_logprobs_backward(z, t, state, up, out=z[:1].expand(4, 40))]
    for call in bad:
        with pytest.raises(ValueError):
            call()


# ------------------------------------------------------------------ block joint
def joint(seed, rows, H, dtype):
    return dict(x=randn(seed, rows, H, std=2.0, mean=0.3, to=dtype), y=randn(seed + 1, rows, H, std=0.7, to=dtype),
                pw=randn(seed + 2, H, std=0.2, mean=1.0, to=dtype), pb=randn(seed + 3, H, std=0.1, to=dtype),
                gate=randn(seed + 4, H, std=0.4, mean=0.5, to=dtype),
                w=randn(seed + 5, H, std=0.2, mean=1.0, to=dtype), b=randn(seed + 6, H, std=0.1, to=dtype))


def test_joint_against_64_bits_and_differences():
    j = joint(10, 3, 11, FP32)
    x_out, h, stats = norm.block_join_fwd(*j.values(), 1e-5, residual_scale=0.8)
    u64, h64, stats64 = ref.join(*j.values(), 1e-5, 0.8)
    assert (x_out.double() - u64).abs().max() < 1e-6 and (h.double() - h64).abs().max() < 1e-5
    assert (stats.double() - stats64).abs().max() < 1e-5
    dh, du = randn(20, 3, 11, to=FP32), randn(21, 3, 11, to=FP32)
    g = norm.block_join_bwd(dh, du, x_out, j["y"], stats, j["pw"], j["pb"], j["gate"], j["w"], residual_scale=0.8,
                            pre_bias=j["b"])
    assert (g.h - h).abs().max() < 1e-5

    def value(**moved):
        v = {k: t.double() for k, t in j.items()} | moved
        u, hh, _ = ref.join(*v.values(), 1e-5, 0.8)
        return ((u * du.double()).sum() + (hh * dh.double()).sum()).item()

    names = dict(x="dx", y="dy", pw="dpost_weight", pb="dpost_bias", gate="dgate", w="dpre_weight", b="dpre_bias")
    for name, of in names.items():
        grad = getattr(g, of)
        flat = j[name].numel()
        for at in (0, flat // 2, flat - 1):
            step = torch.zeros(flat, dtype=torch.float64)
            step[at] = 1e-5
            step = step.view(j[name].shape)
            base = j[name].double()
            slope = (value(**{name: base + step}) - value(**{name: base - step})) / 2e-5
            assert abs(slope - grad.reshape(-1)[at].item()) < 2e-5 * (1 + abs(slope)), (name, at)


def test_joint_refusals():
    j = joint(30, 4, 16, BF16)
    args = list(j.values())
    x_out, h, stats = norm.block_join_fwd(*args, 1e-5)

    def with_(i, t):
        return lambda: norm.block_join_fwd(*[t if k == i else a for k, a in enumerate(args)], 1e-5)

    back = dict(dh=h, dx_out=None, x_out=x_out, y=j["y"], stats=stats, post_weight=j["pw"], post_bias=j["pb"],
                gate=j["gate"], pre_weight=j["w"])

    def but(**other):
        return lambda: norm.block_join_bwd(**(back | other))

    wide = torch.zeros(2, 8193, dtype=BF16)
    p = actpack.pack(h)
    bad = [with_(0, j["x"].half()), with_(1, j["y"].float()), with_(1, j["y"][:3]),
           with_(0, j["x"].t().contiguous().t()), with_(4, j["gate"][:15]), with_(2, j["pw"].float()),
           lambda: norm.block_join_fwd(wide, wide, *[wide[0]] * 5, 1e-5),
           lambda: norm.block_join_fwd(*args, 1e-5, out=torch.zeros(1, 16, dtype=BF16).expand(4, 16)),
           but(dx_out=h[:2]), but(x_out=p), but(stats=stats[:2]), but(stats=stats.double()),
           but(x_out=actpack.pack(h[:2]), y=actpack.pack(h[:2])), but(pre_bias=j["b"][:3]),
           but(out=torch.zeros(4, 16)), but(gate=j["gate"].expand(2, 16)),
           lambda: norm.layer_norm_bwd_packed(h, h, j["w"], stats[0], stats[1]),
           lambda: norm.layer_norm_bwd_packed(h, p, j["w"], stats[0][:2], stats[1]),
           lambda: norm.layer_norm_bwd_packed(h.half(), p, j["w"], stats[0], stats[1]),
           lambda: norm.layer_norm_bwd_packed(h, p, j["w"], stats[0], stats[1], dres=h.float())]
    for n, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            print("accepted", n)


def test_norm_gradient_from_packed_input():
    x, w, b = randn(40, 6, 200, std=2.0, mean=0.2, to=FP32), randn(41, 200, mean=1.0, to=FP32), randn(42, 200, to=FP32)
    dy, dres = randn(43, 6, 200, to=FP32), randn(44, 6, 200, to=FP32)
    p = actpack.pack(x)
    xk = actpack.unpack(p)
    _, mean, rstd = norm.layer_norm_fwd(x, w, b, 1e-5)
    dx, dw, db, y = norm.layer_norm_bwd_packed(dy, p, w, mean, rstd, dres=dres, bias=b)
    dx0, dw0, db0 = norm.layer_norm_bwd(dy, xk, w, mean, rstd)
    assert (dx - (dx0 + dres)).abs().max() < 1e-5 and (dw - dw0).abs().max() < 1e-4
    assert torch.equal(db, db0)
    assert (y - ((xk - mean[:, None]) * rstd[:, None] * w + b)).abs().max() < 1e-5


# ------------------------------------------------------------ 8-bit activations
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 128), (4, 129), (2, 300), (5, 16)])
def test_pack_is_the_nearest_code(rows, cols):
    x = randn(50 + cols, rows, cols, std=5.0, to=FP32)
    got = actpack.unpack(actpack.pack(x))
    assert torch.equal(got.double(), ref.kept(x))
    # half a code's step: 2^-4 relative, or 2^-10 units where the unit leaves amax in (224, 448]
    amax = torch.nn.functional.pad(x.abs(), (0, -cols % 128)).view(rows, -1, 128).amax(2)
    unit = (amax / 224).repeat_interleave(128, 1)[:, :cols]
    assert bool(((got - x).abs() <= torch.maximum(x.abs() * 2.0 ** -4, unit * 2.0 ** -10)).all())


def test_pack_special_values_and_refusals():
    x = randn(60, 5, 256, to=FP32)
    x[0, 3], x[0, 4], x[0, 5] = torch.inf, -torch.inf, torch.nan
    x[1] = 0.0
    x[2, :128] = 3.4e38
    x[3] = 1e-38
    x[4, 128:] = 1e-30
    p = actpack.pack(x)
    assert p.nbytes() == 5 * actpack.row_bytes(256) == 5 * 272
    got = actpack.unpack(p).double()
    ref.close(got, ref.kept(x), torch.zeros(()))
    assert got[0].isnan().sum() == 3
    v, act = actpack.unpack_gelu(p)
    assert torch.equal(v.nan_to_num(7.0).double(), got.nan_to_num(7.0)) and act[0, 3].isnan()
    empty = actpack.pack(x[:0])
    assert actpack.unpack(empty).shape == (0, 256)
    for call in (lambda: actpack.pack(x[0]), lambda: actpack.pack(x.half()), lambda: actpack.pack(x[:, :0]),
                 lambda: actpack.pack(x.t().contiguous().t()), lambda: actpack.unpack(x),
                 lambda: actpack.Packed8(p.data[:, :-1], 256), lambda: actpack.Packed8(p.data, 256, FP16),
                 lambda: actpack.Packed8(p.data.float(), 256), lambda: actpack.unpack_gelu(p.data)):
        with pytest.raises(ValueError):
            call()
