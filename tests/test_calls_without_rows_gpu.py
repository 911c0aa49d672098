"""Row operators called without rows: the same outputs' shapes and the same refusals as with rows."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(seed, *shape, std=1.0, to=BF16):
    return (torch.randn(shape, generator=gen(seed), device="cuda") * std).to(to)


def ops():
    from tempname_5090_b200.ops import actpack, loss, norm
    return actpack, loss, norm


def no_rows(H=64):
    vec = randn(1, H)
    e = torch.empty((0, H), dtype=BF16, device="cuda")
    return e, vec, torch.empty((0,), dtype=torch.int64, device="cuda"), torch.empty((0,), device="cuda")


def test_scoring_refusals_without_rows():
    _, loss, _ = ops()
    z, _, t, up = no_rows()
    got, state = loss.token_logprobs(z, t, top_k=32)
    assert got.top_ids.shape == (0, 32)
    assert loss.token_logprobs_backward(z, t, state, up, up).shape == (0, 64)
    bad = [lambda: loss.token_logprobs(z, t.cpu()), lambda: loss.token_logprobs(z, t.int()),
           lambda: loss.token_logprobs(z, torch.zeros(2, dtype=torch.int64, device="cuda")),
           lambda: loss.token_logprobs(z, t, top_k=33), lambda: loss.token_logprobs(z[:, :5], t, top_k=6),
           lambda: loss.token_logprobs(z[:, :0], t), lambda: loss.token_logprobs(z.double(), t),
           lambda: loss.token_logprobs_backward(z, t.cpu(), state, up),
           lambda: loss.token_logprobs_backward(z, t, state, up.double()),
           lambda: loss.token_logprobs_backward(z, t, state, up.cpu()),
           lambda: loss.token_logprobs_backward(z, t, state, up, up.half()),
           lambda: loss.token_logprobs_backward(z, t, state, up, out=z.float()),
           lambda: loss.token_logprobs_backward(z, t, state, up, out=z[:, :5])]
    for n, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            print("accepted", n)


def test_packing_refusals_without_rows():
    actpack, _, _ = ops()
    x = no_rows()[0]
    assert actpack.unpack(actpack.pack(x)).shape == (0, 64)
    for n, call in enumerate((lambda: actpack.pack(x.half()), lambda: actpack.pack(x[:, :0]))):
        with pytest.raises(ValueError):
            call()
            print("accepted", n)


def test_joint_refusals_without_rows():
    actpack, _, norm = ops()
    e, vec, _, _ = no_rows()
    args = [e, e] + [vec] * 5
    x_out, h, stats = norm.block_join_fwd(*args, 1e-5)
    back = dict(dh=h, dx_out=None, x_out=x_out, y=e, stats=stats, post_weight=vec, post_bias=vec, gate=vec,
                pre_weight=vec, pre_bias=vec)
    g = norm.block_join_bwd(**back)
    assert g.dx.shape == g.h.shape == (0, 64) and not any(bool(t.any()) for t in g[2:7])
    p = actpack.pack(e)
    one = stats[0]
    dx, dw, db, y = norm.layer_norm_bwd_packed(h, p, vec, one, one, bias=vec)
    assert dx.shape == y.shape == (0, 64) and not bool(dw.any()) and not bool(db.any())

    def with_(i, t):
        return lambda: norm.block_join_fwd(*[t if k == i else a for k, a in enumerate(args)], 1e-5)

    def but(**other):
        return lambda: norm.block_join_bwd(**(back | other))

    wide = torch.empty((0, 8193), dtype=BF16, device="cuda")
    big = torch.zeros(8193, dtype=BF16, device="cuda")
    bad = [with_(1, e[:, :7]), with_(1, e.float()), with_(1, e.cpu()),
           with_(1, torch.empty((2, 64), dtype=BF16, device="cuda")), with_(2, vec[:63]),
           with_(4, vec.float()), with_(0, e.half()),
           lambda: norm.block_join_fwd(wide, wide, *[big] * 5, 1e-5),
           lambda: norm.block_join_fwd(e[:, :0], e[:, :0], *[vec[:0]] * 5, 1e-5),
           lambda: norm.block_join_fwd(*args, 1e-5, out=e[:, :9]),
           but(y=e[:, :9]), but(x_out=e.float()), but(dx_out=e.float()), but(gate=vec[:9]), but(pre_weight=vec.cpu()),
           but(pre_bias=vec[:9]), but(out=e.float()), but(stats=stats.double()),
           but(x_out=actpack.pack(e[:, :9]), y=actpack.pack(e[:, :9])),
           lambda: norm.layer_norm_bwd_packed(h, actpack.pack(e[:, :9]), vec, one, one),
           lambda: norm.layer_norm_bwd_packed(h, p, vec[:9], one, one),
           lambda: norm.layer_norm_bwd_packed(h, p, vec, one, one, dres=e[:, :9]),
           lambda: norm.layer_norm_bwd_packed(h, p, vec, one.double(), one)]
    for n, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            print("accepted", n)
