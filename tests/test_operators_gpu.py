"""Scoring, block joint and 8-bit activation kernels against 64 bits."""
import math

import pytest
import torch

import operators_reference as ref

pytestmark = pytest.mark.gpu
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(seed, *shape, std=1.0, mean=0.0, to=BF16):
    return (torch.randn(shape, generator=gen(seed), device="cuda") * std + mean).to(to)


def ops():
    from tempname_5090_b200.ops import actpack, loss, norm
    return actpack, loss, norm


# ------------------------------------------------------------ 8-bit activations
SHAPES = [(1, 1), (1, 7), (3, 16), (2, 128), (5, 129), (4, 1000), (300, 1100), (33, 2050), (7, 8200), (130, 4096)]


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_pack_and_unpack(rows, cols, dtype):
    actpack, _, _ = ops()
    x = randn(rows + cols, rows, cols, std=4.0, to=dtype)
    p = actpack.pack(x)
    assert torch.equal(p.data.cpu(), actpack.pack(x.cpu()).data)  # to the bit, padding too
    want = ref.kept(x)
    assert torch.equal(actpack.unpack(p).double(), want.to(dtype).double())
    v, act = actpack.unpack_gelu(p)
    assert torch.equal(v, actpack.unpack(p))
    gelu = ref.gelu(want)
    # e^x and erfcx are good to a few steps of FP32
    ref.close(act, gelu, ref.gelu_bound(want, gelu, dtype))


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_pack_special_values(dtype):
    actpack, _, _ = ops()
    x = randn(1, 8, 384, to=dtype)
    x[0, 3], x[0, 4], x[0, 5] = torch.inf, -torch.inf, torch.nan
    x[1] = 0.0
    x[2, :128] = torch.finfo(dtype).max
    x[2, 128:] = torch.finfo(dtype).min
    x[3] = 1e-38
    x[4, 128:] = 1e-30
    x[5] = torch.nan
    x[6] = -torch.inf
    x[7] = x[7] * 1e4
    p = actpack.pack(x)
    ref.close(actpack.unpack(p), ref.kept(x).to(dtype), torch.zeros((), device="cuda"))
    assert torch.equal(actpack.unpack(p).cpu().nan_to_num(9.0), actpack.unpack(actpack.pack(x.cpu())).nan_to_num(9.0))
    v, act = actpack.unpack_gelu(p)
    assert torch.equal(v.nan_to_num(9.0), actpack.unpack(p).nan_to_num(9.0))
    want = ref.kept(x)
    gelu = ref.gelu(want)
    ref.close(act, gelu, ref.gelu_bound(want, gelu, dtype))


def test_every_code_under_every_unit():
    """All 254 numbers that a code can be, under every power of two, and their GeLU."""
    actpack, _, _ = ops()
    codes = torch.arange(256, device="cuda").to(torch.uint8)
    rows = 247
    data = torch.zeros((rows, actpack.row_bytes(256)), dtype=torch.uint8, device="cuda")
    data[:, :256] = codes
    units = torch.arange(1, rows + 1, device="cuda").to(torch.uint8)
    data[:, 256] = units
    data[:, 257] = units
    p = actpack.Packed8(data, 256, FP32)
    want = codes.view(torch.float8_e4m3fn).double() * torch.exp2(units.double() - 127)[:, None]
    want = want.float().double()  # the largest leave FP32's range
    v, act = actpack.unpack_gelu(p)
    ref.close(v, want, torch.zeros((), device="cuda"))
    gelu = ref.gelu(want)
    ref.close(act, gelu, ref.gelu_bound(want, gelu, FP32))


def test_pack_of_strided_and_unaligned_rows():
    actpack, _, _ = ops()
    base = randn(2, 20, 520)
    for x in (base[:, :512], base[:, 1:513], base[::3, 8:264], base[4:5].expand(6, 520), base[:, 3:4]):
        assert torch.equal(actpack.unpack(actpack.pack(x)).double(), ref.kept(x).to(BF16).double())
    assert actpack.unpack(actpack.pack(base[:0])).shape == (0, 520)
    assert actpack.unpack_gelu(actpack.pack(base[:0]))[1].shape == (0, 520)


# ------------------------------------------------------------------ block joint
def joint(seed, rows, H, dtype):
    spread = torch.exp(0.5 * torch.randn(H, generator=gen(seed + 9), device="cuda"))
    return dict(x=(randn(seed, rows, H, std=2.0, mean=0.3, to=FP32) * spread).to(dtype),
                y=randn(seed + 1, rows, H, std=0.7, mean=0.1, to=dtype),
                pw=randn(seed + 2, H, std=0.2, mean=1.0, to=dtype), pb=randn(seed + 3, H, std=0.1, to=dtype),
                gate=randn(seed + 4, H, std=0.4, mean=0.5, to=dtype),
                w=randn(seed + 5, H, std=0.2, mean=1.0, to=dtype), b=randn(seed + 6, H, std=0.1, to=dtype))


def check_joint(got, j, eps, alpha, dtype):
    x_out, h, stats = got
    u64, h64, s64 = ref.join(*j.values(), eps, alpha)
    x, y, pw, pb, gate, w, b = (t.double().abs() for t in j.values())
    # sums over a row: 16 values a thread, 5 + 16 joins; every further step is a rounding of a term
    n = 64 * ref.U
    size_y = (y + s64[0].abs()[:, None]) * s64[1][:, None]
    size_u = abs(alpha) * x + gate * ((size_y + size_y.amax(1, keepdim=True)) * pw + pb)
    ref.close(x_out, u64, ref.rounded(u64, dtype) + n * size_u)
    size_h = (size_u.amax(1, keepdim=True) * s64[3][:, None] * (1 + h64.abs())) * w + b
    ref.close(h, h64, ref.rounded(h64, dtype) + n * size_h)
    ref.close(stats[0], s64[0], n * y.amax(1))
    ref.close(stats[1], s64[1], n * s64[1] * (1 + size_y.amax(1)))
    ref.close(stats[2], s64[2], n * size_u.amax(1))
    ref.close(stats[3], s64[3], n * s64[3] * (1 + size_u.amax(1) * s64[3]) ** 2)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("rows,H", [(1, 8), (1, 1), (3, 33), (2, 256), (17, 1001), (130, 1024), (64, 2050), (40, 4096),
                                    (9, 4104), (5, 8192), (6, 8191)])
def test_joint(rows, H, dtype):
    _, _, norm = ops()
    j = joint(100 + H, rows, H, dtype)
    eps, alpha = 1e-5, 0.8
    got = norm.block_join_fwd(*j.values(), eps, residual_scale=alpha)
    check_joint(got, j, eps, alpha, dtype)
    x_out, h, stats = got
    dh, du = randn(200, rows, H, to=dtype), randn(201, rows, H, to=dtype)
    args = (x_out, j["y"], stats, j["pw"], j["pb"], j["gate"], j["w"])
    for with_du in (True, False):
        d = du if with_du else None
        g = norm.block_join_bwd(dh, d, *args, residual_scale=alpha)
        assert g.h is None
        want, size = ref.join_grad(dh, d, x_out, j["y"], stats, j["pw"], j["pb"], j["gate"], j["w"], alpha)
        check_grads(g, want, size, rows, dtype)
        again = norm.block_join_bwd(dh, d, *args, residual_scale=alpha)
        assert all(torch.equal(a, b) for a, b in zip(g[:7], again[:7]))  # a fixed order


def check_grads(got, want, size, rows, dtype):
    for k, (a, r, s) in enumerate(zip(got, want, size)):
        # a row: 64 roundings of its terms; a column: a CTA's rows in order, then the CTAs
        n = 64 * ref.U if k < 2 else (64 + rows / 148 + 148 / 8 + 8) * ref.U
        ref.close(a, r, ref.rounded(r, dtype) + n * s)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("rows,H", [(1, 1), (3, 130), (17, 1001), (300, 256), (50, 4096), (5, 8192), (700, 2056)])
def test_gradients_from_packed_inputs(rows, H, dtype):
    actpack, _, norm = ops()
    j = joint(300 + H, rows, H, dtype)
    x_out, h, stats = norm.block_join_fwd(*j.values(), 1e-5, residual_scale=0.9)
    pu, py = actpack.pack(x_out), actpack.pack(j["y"])
    dh, du = randn(301, rows, H, to=dtype), randn(302, rows, H, to=dtype)
    g = norm.block_join_bwd(dh, du, pu, py, stats, j["pw"], j["pb"], j["gate"], j["w"], residual_scale=0.9,
                            pre_bias=j["b"])
    u8, y8 = ref.kept(x_out), ref.kept(j["y"])
    want, size = ref.join_grad(dh, du, u8, y8, stats, j["pw"], j["pb"], j["gate"], j["w"], 0.9)
    check_grads(g, want, size, rows, dtype)
    hat = (u8 - stats[2].double()[:, None]) * stats[3].double()[:, None]
    again = hat * j["w"].double() + j["b"].double()
    off = (u8.abs() + stats[2].double().abs()[:, None]) * stats[3].double()[:, None] * j["w"].double().abs()
    ref.close(g.h, again, ref.rounded(again, dtype) + 4 * ref.U * (off + again.abs() + j["b"].double().abs()))
    # LayerNorm alone
    for dres in (du, None):
        dx, dw, db, y = norm.layer_norm_bwd_packed(dh, pu, j["w"], stats[2], stats[3], dres=dres, bias=j["b"])
        one = torch.ones(H, device="cuda")
        lw, ls = ref.join_grad(dh, dres, u8, y8, stats, one, one, one, j["w"], 1.0)
        check_grads((dx, dx), (lw[0], lw[0]), (ls[0], ls[0]), rows, dtype)
        for a, k in ((dw, 5), (db, 6)):
            ref.close(a, lw[k], ref.rounded(lw[k], dtype) + (64 + rows / 148 + 148 / 8 + 8) * ref.U * ls[k])
        assert torch.equal(y, g.h)
    assert norm.layer_norm_bwd_packed(dh, pu, j["w"], stats[2], stats[3])[3] is None


def test_joint_strides_alignment_and_outputs():
    _, _, norm = ops()
    rows, H, eps, alpha = 13, 512, 1e-5, 1.1
    j = joint(400, rows, H, BF16)
    plain = norm.block_join_fwd(*j.values(), eps, residual_scale=alpha)
    dh, du = randn(401, rows, H), randn(402, rows, H)
    rest = (plain[2], j["pw"], j["pb"], j["gate"], j["w"])
    back = norm.block_join_bwd(dh, du, plain[0], j["y"], *rest, residual_scale=alpha)
    for pad, off in ((24, 8), (7, 3)):
        def spaced(t):
            wide = torch.full((rows, H + pad), torch.nan, dtype=BF16, device="cuda")
            wide[:, off:off + H] = t
            return wide[:, off:off + H]
        hole = torch.full((rows, H + pad), 5.0, dtype=BF16, device="cuda")
        got = norm.block_join_fwd(spaced(j["x"]), spaced(j["y"]), *list(j.values())[2:], eps, residual_scale=alpha,
                                  out=hole[:, off:off + H])
        check_joint(got, j, eps, alpha, BF16)
        assert bool((hole[:, :off] == 5).all()) and bool((hole[:, off + H:] == 5).all())
        hole.fill_(5.0)
        g = norm.block_join_bwd(spaced(dh), spaced(du), spaced(plain[0]), spaced(j["y"]), *rest, residual_scale=alpha,
                                out=hole[:, off:off + H])
        want, size = ref.join_grad(dh, du, plain[0], j["y"], *rest[:2], *rest[2:], alpha)
        check_grads(g, want, size, rows, BF16)
        assert bool((hole[:, :off] == 5).all()) and bool((hole[:, off + H:] == 5).all())
    # a broadcast gradient, and no rows at all
    g = norm.block_join_bwd(dh[:1].expand(rows, H), du, plain[0], j["y"], *rest, residual_scale=alpha)
    want, size = ref.join_grad(dh[:1].expand(rows, H), du, plain[0], j["y"], *rest[:2], *rest[2:], alpha)
    check_grads(g, want, size, rows, BF16)
    x_out, h, stats = norm.block_join_fwd(j["x"][:0], j["y"][:0], *list(j.values())[2:], eps)
    g = norm.block_join_bwd(h, None, x_out, x_out, stats, *rest[1:])
    assert g.dx.shape == (0, H) and bool((g.dgate == 0).all()) and bool((g.dpre_weight == 0).all())


def test_many_rows_per_cta():
    actpack, _, norm = ops()
    rows, H = 5003, 264
    j = joint(500, rows, H, FP32)
    x_out, _, stats = norm.block_join_fwd(*j.values(), 1e-5)
    dh = randn(501, rows, H, to=FP32)
    g = norm.block_join_bwd(dh, None, x_out, j["y"], stats, j["pw"], j["pb"], j["gate"], j["w"])
    want, size = ref.join_grad(dh, None, x_out, j["y"], stats, j["pw"], j["pb"], j["gate"], j["w"], 1.0)
    check_grads(g, want, size, rows, FP32)


# -------------------------------------------------------------------- scoring
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("rows,V,k", [(1, 1, 1), (1, 7, 7), (3, 33, 32), (1, 50304, 20), (2, 32003, 32), (5, 1000, 0),
                                      (40, 2049, 5), (300, 4097, 8), (700, 513, 3), (37, 33792, 10)])
def test_scores(rows, V, k, dtype):
    _, loss, _ = ops()
    z = randn(600 + V, rows, V, std=3.0, to=dtype)
    t = torch.randint(0, V, (rows,), generator=gen(601), device="cuda")
    if rows > 2:
        t[1], t[2] = -100, V
    got, state = loss.token_logprobs(z, t, top_k=k)
    ref.check_scores(got, z, t, k)
    a, b = randn(602, rows, to=FP32), randn(603, rows, to=FP32)
    for up in (None, b):
        g = loss.token_logprobs_backward(z, t, state, a, up)
        want, size = ref.score_grad(z, t, a, up)
        # e^l is off by |l| half steps and a few 2^-23, the statistics by their own bound
        ref.close(g, want, ref.rounded(want, dtype) + (ref.score_bound(z)[:, None] + 64 * ref.U) * 2 * size)
    work = z.clone()
    assert loss.token_logprobs_backward(work, t, state, a, b, out=work) is work
    assert torch.equal(work.nan_to_num(3.0), g.nan_to_num(3.0))


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("V", [100, 9001])
def test_scores_of_special_rows(V, dtype):
    _, loss, _ = ops()
    z = randn(1, 9, V, std=3.0, to=dtype)
    z[1] = -torch.inf                       # nothing left
    z[2, 7:] = -torch.inf                   # a few tokens left
    z[3] = torch.finfo(dtype).min           # the type's lowest value everywhere
    z[4, 5] = torch.nan
    z[5, 6] = torch.inf
    z[6] = 0.25                             # all equal
    z[7, 10:20] = z[7].max() + 1            # ties at the top
    z[8, :50] = torch.finfo(dtype).min
    t = torch.tensor([3, 4, 2, 0, 1, 1, 99, 12, -100], device="cuda")
    got, state = loss.token_logprobs(z, t, top_k=20)
    fine = torch.tensor([0, 1, 2, 3, 6, 7, 8], device="cuda")
    ref.check_scores(loss.TokenScores(*(a[fine] for a in got)), z[fine], t[fine], 20)
    cpu, _ = loss.token_logprobs(z.cpu(), t.cpu(), top_k=20)
    assert torch.equal(got.top_ids.cpu(), cpu.top_ids)
    assert got.logprob[1] == -math.inf and got.entropy[1] == 0
    assert torch.equal(got.top_ids[1].cpu(), torch.arange(20))
    assert got.logprob[4].isnan() and got.logprob[5].isnan() and got.entropy[5].isnan()
    a, b = randn(2, 9, to=FP32), randn(3, 9, to=FP32)
    g = loss.token_logprobs_backward(z, t, state, a, b)
    want, size = ref.score_grad(z[fine], t[fine], a[fine], b[fine])
    bound = ref.score_bound(z[fine])[:, None] + 64 * ref.U
    ref.close(g[fine], want, ref.rounded(want, dtype) + bound * 2 * size)
    assert bool(g[4:6].isnan().all()) and bool((g[1] == 0).all())


@pytest.mark.parametrize("rows", [1, 70])
def test_alternatives_in_few_threads_vectors(rows):
    """The largest values where one thread's vectors lie (more candidates than are
    collected), in one contiguous run, in falling order, and all equal."""
    _, loss, _ = ops()
    V, k = 32768, 32
    for dtype in (BF16, FP32):
        per = 8 if dtype == BF16 else 4
        z = randn(4, rows, V, std=1.0, to=dtype)
        for first in range(40):  # 40 threads' vectors hold all large values
            block = z.view(rows, -1, 256 * per)[:, :, first * per:(first + 1) * per]
            block.add_(20.0)
        flat = torch.zeros(rows, V, dtype=dtype, device="cuda")
        fall = (-torch.arange(V, device="cuda").float() / 64).to(dtype).expand(rows, V).contiguous()
        run = randn(5, rows, V, to=dtype)
        run[:, 12345:12445] += 30.0
        rise = fall.flip(1).contiguous()
        for t in (z, flat, fall, run, rise):
            got, _ = loss.token_logprobs(t, torch.zeros(rows, dtype=torch.int64, device="cuda"), top_k=k)
            want = torch.sort(t.float(), dim=1, descending=True, stable=True).indices[:, :k]
            assert torch.equal(got.top_ids, want)


def test_scores_of_strided_unaligned_and_far_rows():
    _, loss, _ = ops()
    base = randn(6, 24, 4100, std=3.0)
    t = torch.randint(0, 4000, (24,), generator=gen(7), device="cuda")
    a = randn(8, 24, to=FP32)
    for x in (base[:, :4000], base[:, 3:4003], base[:, 8:4008], base[:1].expand(24, 4100)[:, :4000]):
        got, state = loss.token_logprobs(x, t, top_k=6)
        ref.check_scores(got, x, t, 6)
        want, size = ref.score_grad(x, t, a, None)
        bound = ref.rounded(want, BF16) + (ref.score_bound(x)[:, None] + 64 * ref.U) * 2 * size
        ref.close(loss.token_logprobs_backward(x, t, state, a), want, bound)
        hole = torch.full((24, 4100), 5.0, dtype=BF16, device="cuda")
        ref.close(loss.token_logprobs_backward(x, t, state, a, out=hole[:, 5:4005]), want, bound)
        assert bool((hole[:, :5] == 5).all()) and bool((hole[:, 4005:] == 5).all())
    none, state = loss.token_logprobs(base[:0], t[:0], top_k=3)
    assert none.top_ids.shape == (0, 3) and none.logprob.shape == (0,)
    assert loss.token_logprobs_backward(base[:0], t[:0], state, a[:0]).shape == (0, 4100)


def test_offsets_beyond_32_bits():
    """Rows whose element offsets pass 2^31 (a wide row stride over a small matrix)."""
    actpack, loss, norm = ops()
    rows, V, ld = 3, 1024, 1_200_000_000
    flat = torch.empty((rows - 1) * ld + V, dtype=BF16, device="cuda")
    x = flat.as_strided((rows, V), (ld, 1))
    small = randn(9, rows, V, std=3.0)
    x.copy_(small)
    t = torch.tensor([5, 1023, 0], device="cuda")
    got, state = loss.token_logprobs(x, t, top_k=4)
    want, ws = loss.token_logprobs(small, t, top_k=4)
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    assert torch.equal(actpack.pack(x).data, actpack.pack(small).data)
    vec = randn(10, V)
    a = norm.block_join_fwd(x, small, vec, vec, vec, vec, vec, 1e-5)
    b = norm.block_join_fwd(small, small, vec, vec, vec, vec, vec, 1e-5)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    up = torch.ones(rows, device="cuda")
    g = loss.token_logprobs_backward(small, t, ws, up)
    assert torch.equal(loss.token_logprobs_backward(x, t, state, up, out=x), g)


@pytest.mark.parametrize("world", [2, 4, 8])
def test_records_of_emulated_ranks(world):
    """The partial results of a vocabulary's shards, merged as the group's ranks do."""
    _, loss, _ = ops()
    from tempname_5090_b200._native import lib
    rows, V, k = 50, 8 * 1001, 12
    z = randn(11, rows, V, std=3.0)
    z[3, :V // 2] = -torch.inf
    z[4] = 0.5
    z[5] = -torch.inf
    t = torch.randint(0, V, (rows,), generator=gen(12), device="cuda")
    t[0], t[1] = -1, V
    Vl = V // world
    records = torch.empty((world, rows, 4 + 2 * k), device="cuda")
    for r in range(world):
        lib().score_fwd(z[:, r * Vl:(r + 1) * Vl], t, r * Vl, V, k, None, None, records[r])
    out = torch.empty(rows * (5 + k), device="cuda")
    ids = torch.empty((rows, k), dtype=torch.int64, device="cuda")
    lib().score_merge(records, t, Vl, k, out, ids)
    got = loss.TokenScores(out[:rows], out[rows:2 * rows], out[5 * rows:].view(rows, k), ids)
    ref.check_scores(got, z, t, k)
    a, b = randn(13, rows, to=FP32), randn(14, rows, to=FP32)
    want, size = ref.score_grad(z, t, a, b)
    parts = [loss.token_logprobs_backward(z[:, r * Vl:(r + 1) * Vl], t,
                                          loss.ScoreState(out[2 * rows:5 * rows].view(3, rows), r * Vl, V), a, b)
             for r in range(world)]
    ref.close(torch.cat(parts, 1), want, ref.rounded(want, BF16) + (ref.score_bound(z)[:, None] + 64 * ref.U) * 2 * size)


# ------------------------------------------------- streams, graphs, the whole run
def step(j, z, t, a, b):
    """The operators as a training step calls them, one after another."""
    actpack, loss, norm = ops()
    x_out, h, stats = norm.block_join_fwd(*j.values(), 1e-5, residual_scale=0.9)
    kept = actpack.pack(x_out), actpack.pack(j["y"])
    pre, act = actpack.unpack_gelu(actpack.pack(h))
    scores, state = loss.token_logprobs(z, t, top_k=4)
    dz = loss.token_logprobs_backward(z, t, state, a, b)
    g = norm.block_join_bwd(act, pre, *kept, stats, j["pw"], j["pb"], j["gate"], j["w"], residual_scale=0.9,
                            pre_bias=j["b"])
    dx, dw, db, y = norm.layer_norm_bwd_packed(g.dx, kept[0], j["w"], stats[2], stats[3], dres=g.dy, bias=j["b"])
    return [x_out, h, stats, pre, act, *scores, dz, *g, dx, dw, db, y]


def test_run_on_another_stream_and_in_a_captured_graph():
    rows, H, V = 200, 1024, 5001
    j = joint(700, rows, H, BF16)
    z = randn(701, rows, V, std=3.0)
    t = torch.randint(0, V, (rows,), generator=gen(702), device="cuda")
    a, b = randn(703, rows, to=FP32), randn(704, rows, to=FP32)
    want = [v.clone() for v in step(j, z, t, a, b)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(j, z, t, a, b)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    graphs = []
    for _ in range(2):  # two graphs at once, replayed in turn: no workspace is shared
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(j, z, t, a, b)
        graphs.append((graph, out))
    fresh = joint(800, rows, H, BF16)
    other = [v.clone() for v in step(fresh, z, t, b, a)]
    keep = {k: v.clone() for k, v in j.items()}, a.clone(), b.clone()
    for k in j:
        j[k].copy_(fresh[k])
    a.copy_(keep[2]), b.copy_(keep[1])
    graphs[0][0].replay()
    for k in j:
        j[k].copy_(keep[0][k])
    a.copy_(keep[1]), b.copy_(keep[2])
    graphs[1][0].replay()
    assert all(torch.equal(p, q) for p, q in zip(graphs[0][1], other))
    assert all(torch.equal(p, q) for p, q in zip(graphs[1][1], want))


def test_two_streams_at_once():
    rows, H, V = 300, 512, 3001
    j, k = joint(900, rows, H, BF16), joint(950, rows, H, BF16)
    z = randn(901, rows, V, std=3.0)
    t = torch.randint(0, V, (rows,), generator=gen(902), device="cuda")
    a, b = randn(903, rows, to=FP32), randn(904, rows, to=FP32)
    want = [[v.clone() for v in step(q, z, t, a, b)] for q in (j, k)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for _ in range(3):
        got = []
        for s, q in zip(streams, (j, k)):
            with torch.cuda.stream(s):
                got.append(step(q, z, t, a, b))
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(p, q) for p, q in zip(g, w))


def test_refusals_of_the_native_entries():
    actpack, loss, norm = ops()
    from tempname_5090_b200._native import lib
    x = randn(15, 4, 64)
    p = actpack.pack(x)
    with pytest.raises(ValueError):
        loss.token_logprobs(x, torch.zeros(4, dtype=torch.int64))  # targets on the CPU
    with pytest.raises(ValueError):
        norm.block_join_fwd(x, x.cpu(), *[x[0]] * 5, 1e-5)
    with pytest.raises(RuntimeError):
        lib().act_pack(x, p.data[:3])
    with pytest.raises(RuntimeError):
        lib().act_unpack(p.data, x.half(), None)
    with pytest.raises(RuntimeError):
        lib().score_fwd(x, torch.zeros(3, dtype=torch.int64, device="cuda"), 0, 64, 0, torch.empty(20, device="cuda"),
                        None, None)
    with pytest.raises(RuntimeError):
        lib().join_bwd(x, None, p.data, None, x.new_zeros(4, dtype=FP32), x.new_zeros(4, dtype=FP32), None, None, None,
                       None, None, x[0], None, torch.empty_like(x), None, None, x.new_zeros(2, 64),
                       torch.empty(3, device="cuda"), 1.0)


@pytest.mark.parametrize("rows,V", [(1, 50304), (3, 20001), (900, 4001)])
def test_scores_in_a_captured_graph(rows, V):
    """Rows split over a cluster, and rows of their own, replayed on new logits."""
    _, loss, _ = ops()
    z = randn(16, rows, V, std=3.0)
    t = torch.randint(0, V, (rows,), generator=gen(17), device="cuda")
    a = randn(18, rows, to=FP32)
    loss.token_logprobs(z, t, top_k=20)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, state = loss.token_logprobs(z, t, top_k=20)
        g = loss.token_logprobs_backward(z, t, state, a)
    for seed in (19, 20):
        z.copy_(randn(seed, rows, V, std=3.0))
        graph.replay()
        want, ws = loss.token_logprobs(z, t, top_k=20)
        assert all(torch.equal(p, q) for p, q in zip(got, want))
        assert torch.equal(g, loss.token_logprobs_backward(z, t, ws, a))
        ref.check_scores(got, z, t, 20)


def test_outputs_may_take_the_place_of_inputs():
    """dy over dh, and LayerNorm's dx over the gradient it joins: a row is written after it is read."""
    actpack, _, norm = ops()
    for rows, H in ((700, 512), (333, 1001)):
        j = joint(20, rows, H, BF16)
        x_out, h, stats = norm.block_join_fwd(*j.values(), 1e-5)
        dh, du = randn(21, rows, H), randn(22, rows, H)
        args = (x_out, j["y"], stats, j["pw"], j["pb"], j["gate"], j["w"])
        want = norm.block_join_bwd(dh, du, *args)
        work = dh.clone()
        got = norm.block_join_bwd(work, du, *args, out=work)
        assert all(torch.equal(p, q) for p, q in zip(got[:7], want[:7]))
        p = actpack.pack(x_out)
        want = norm.layer_norm_bwd_packed(dh, p, j["w"], stats[2], stats[3], dres=du)
        work = du.clone()
        got = norm.layer_norm_bwd_packed(dh, p, j["w"], stats[2], stats[3], dres=work, out=work)
        assert all(torch.equal(p, q) for p, q in zip(got[:3], want[:3]))


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("H", [256, 512, 1024, 2048, 4096, 8192])
def test_widths_that_fill_the_threads_over_many_rows(H, dtype):
    """Several rows per CTA, one after another through the same shared memory."""
    actpack, _, norm = ops()
    rows = 1501
    j = joint(60 + H, rows, H, dtype)
    got = norm.block_join_fwd(*j.values(), 1e-5, residual_scale=0.9)
    check_joint(got, j, 1e-5, 0.9, dtype)
    x_out, _, stats = got
    dh, du = randn(61, rows, H, to=dtype), randn(62, rows, H, to=dtype)
    rest = (stats, j["pw"], j["pb"], j["gate"], j["w"])
    want, size = ref.join_grad(dh, du, x_out, j["y"], *rest, 0.9)
    check_grads(norm.block_join_bwd(dh, du, x_out, j["y"], *rest, residual_scale=0.9), want, size, rows, dtype)
    del want, size
    pu, py = actpack.pack(x_out), actpack.pack(j["y"])
    u8, y8 = ref.kept(x_out), ref.kept(j["y"])
    want, size = ref.join_grad(dh, du, u8, y8, *rest, 0.9)
    g = norm.block_join_bwd(dh, du, pu, py, *rest, residual_scale=0.9, pre_bias=j["b"])
    check_grads(g, want, size, rows, dtype)
    dx, dw, db, y = norm.layer_norm_bwd_packed(dh, pu, j["w"], stats[2], stats[3], dres=du, bias=j["b"])
    assert torch.equal(y, g.h)
    one = torch.ones(H, device="cuda")
    lw, ls = ref.join_grad(dh, du, u8, y8, stats, one, one, one, j["w"], 1.0)
    check_grads((dx, dx), (lw[0], lw[0]), (ls[0], ls[0]), rows, dtype)
    for a, k in ((dw, 5), (db, 6)):
        ref.close(a, lw[k], ref.rounded(lw[k], dtype) + (64 + rows / 148 + 148 / 8 + 8) * ref.U * ls[k])


def test_refusals_of_other_packed_rows():
    """Packed rows of another width (250 and 256 columns take as many bytes), raw bytes in
    their place, and bytes off the 16-byte boundary that the native entries are given."""
    actpack, _, norm = ops()
    rows, H = 4, 256
    j = joint(80, rows, H, BF16)
    x_out, _, stats = norm.block_join_fwd(*j.values(), 1e-5)
    dh = randn(81, rows, H)
    narrow, wide = actpack.pack(x_out[:, :250]), actpack.pack(x_out)
    rest = (stats, j["pw"], j["pb"], j["gate"], j["w"])
    for u, y in ((narrow, wide), (wide, narrow), (wide.data, wide.data)):
        with pytest.raises(ValueError):
            norm.block_join_bwd(dh, None, u, y, *rest)
    with pytest.raises(ValueError):
        norm.layer_norm_bwd_packed(dh, narrow, j["w"], stats[2], stats[3])
    from tempname_5090_b200._native import lib
    off = torch.empty(wide.data.numel() + 8, dtype=torch.uint8, device="cuda")[8:].view(wide.data.shape)
    for call in (lambda: lib().act_pack(x_out, off), lambda: lib().unpack(off, H, False, False),
                 lambda: lib().layer_norm_bwd_packed(dh, None, off, stats[2], stats[3], j["w"], None, None, None)):
        with pytest.raises(RuntimeError):
            call()
