"""Tensor/sequence-parallel GPT (pre-LN, exact GeLU, tied embedding) for B200.

Parameter names, per-rank shapes, sharding and initialisation reproduce
TempName-5090 python/flux_5090/model.py:178-229 (state_dict layout):

    embedding [V/W, h] (tied LM head)        position [S, h] (replicated)
    layers.i.{ln1,ln2}_{weight,bias} [h]     layers.i.qkv_weight [3h/W, h], qkv_bias [3h/W]
    layers.i.attn_weight [h, h/W]            layers.i.attn_bias [h] (replicated)
    layers.i.fc1_weight [f/W, h], fc1_bias [f/W]
    layers.i.fc2_weight [h, f/W]             layers.i.fc2_bias [h] (replicated)
    final_weight / final_bias [h]

Seeds are name-derived (seed + sha256(tag)[:8] + 1000003*rank for sharded
tensors), std 0.02 (0.02/sqrt(2L) for attn/fc2 weights), LN weights 1, biases 0.

Unlike the reference (torch autograd over custom Functions), the training
program here is explicit: `forward_backward` runs the forward with the fused
AG->GEMM / GEMM->RS operators, saves exactly the activations the backward
needs, and writes every gradient straight into one flat BF16 gradient buffer
(weight gradients are tcgen05 GEMM outputs, no extra copies).  Forward
arithmetic order matches the reference: value = (value + RowLinear(...)) + bias.
Two choices beside the reference's: `block_norm="sandwich"` in the configuration
gives every branch a norm and a gate after it as well (layers.i.{attn,mlp}_post_
{weight,bias} and {attn,mlp}_gate, replicated), with the joint of two branches as
one kernel; `kept="e4m3"` keeps the tape in 8 bits (ops/actpack.py): residual
stream, branch outputs, QKV and the MLP's pre-activation, from which the backward
pass computes the norms' and the activation's outputs and the attention again.
All parameters live in one flat BF16 buffer ordered [sharded matrices |
sharded vectors | replicated matrices | replicated vectors] so the optimizer
is two fused launches.
"""
from __future__ import annotations

import hashlib
import math
from dataclasses import dataclass

import torch

from ..config import parameter_counts, validate_config
from ..ops import actpack as K
from ..ops import attention as A
from ..ops import embedding as E
from ..ops import gemm as G
from ..ops import loss as CE
from ..ops import norm as N
from ..parallel.tp import TensorParallel
from ..utils import tracing

ALIGN = 64  # elements; keeps every parameter view 128-byte aligned


@dataclass
class ParamSpec:
    name: str
    shape: tuple
    replicated: bool
    init: str          # "normal" | "one" | "zero"
    std: float
    tag: str

    @property
    def numel(self) -> int:
        n = 1
        for s in self.shape:
            n *= s
        return n

    @property
    def matrix(self) -> bool:
        return len(self.shape) >= 2


def param_specs(c: dict, world: int) -> list:
    h, f, V, S, L = c["hidden"], c["ffn"], c["vocab"], c["sequence"], c["layers"]
    specs = [ParamSpec("embedding", (V // world, h), False, "normal", 0.02, "embedding"),
             ParamSpec("position", (S, h), True, "normal", 0.02, "position")]
    small = 0.02 / math.sqrt(2 * L)
    for i in range(L):
        p = f"layers.{i}"
        for norm in ("ln1", "ln2"):
            specs.append(ParamSpec(f"{p}.{norm}_weight", (h,), True, "one", 0.0, f"{p}{norm}w"))
            specs.append(ParamSpec(f"{p}.{norm}_bias", (h,), True, "zero", 0.0, f"{p}{norm}b"))
        specs += [
            ParamSpec(f"{p}.qkv_weight", (3 * h // world, h), False, "normal", 0.02, f"{p}qkvw"),
            ParamSpec(f"{p}.qkv_bias", (3 * h // world,), False, "zero", 0.0, f"{p}qkvb"),
            ParamSpec(f"{p}.attn_weight", (h, h // world), False, "normal", small, f"{p}attnw"),
            ParamSpec(f"{p}.attn_bias", (h,), True, "zero", 0.0, f"{p}attnb"),
            ParamSpec(f"{p}.fc1_weight", (f // world, h), False, "normal", 0.02, f"{p}fc1w"),
            ParamSpec(f"{p}.fc1_bias", (f // world,), False, "zero", 0.0, f"{p}fc1b"),
            ParamSpec(f"{p}.fc2_weight", (h, f // world), False, "normal", small, f"{p}fc2w"),
            ParamSpec(f"{p}.fc2_bias", (h,), True, "zero", 0.0, f"{p}fc2b"),
        ]
        if c.get("block_norm") == "sandwich":
            for branch in ("attn", "mlp"):
                for name, init in (("post_weight", "one"), ("post_bias", "zero"), ("gate", "one")):
                    specs.append(ParamSpec(f"{p}.{branch}_{name}", (h,), True, init, 0.0, f"{p}{branch}{name}"))
    specs.append(ParamSpec("final_weight", (h,), True, "one", 0.0, "final_ln_w"))
    specs.append(ParamSpec("final_bias", (h,), True, "zero", 0.0, "final_ln_b"))
    return specs


def _round_up(x: int) -> int:
    return (x + ALIGN - 1) // ALIGN * ALIGN


class ParamStore:
    """Flat BF16 parameters and gradients with named views and optimizer regions."""

    def __init__(self, specs, device, rank: int, seed: int, dtype=torch.bfloat16, init: bool = True):
        self.specs = specs
        self.device = torch.device(device)
        groups = [[s for s in specs if not s.replicated and s.matrix],
                  [s for s in specs if not s.replicated and not s.matrix],
                  [s for s in specs if s.replicated and s.matrix],
                  [s for s in specs if s.replicated and not s.matrix]]
        self.offsets = {}
        off = 0
        bounds = []
        for g in groups:
            for s in g:
                self.offsets[s.name] = off
                off += _round_up(s.numel)
            bounds.append(off)
        self.total = off
        self.sharded_end = bounds[1]
        self.sharded_decay_end = bounds[0]
        self.replicated_decay_end = bounds[2]
        self.flat = torch.zeros(self.total, dtype=dtype, device=self.device)
        self.grad = torch.zeros(self.total, dtype=dtype, device=self.device)
        self.params = {}
        self.grads = {}
        for s in specs:
            o = self.offsets[s.name]
            self.params[s.name] = self.flat[o:o + s.numel].view(s.shape)
            self.grads[s.name] = self.grad[o:o + s.numel].view(s.shape)
        self.replicated = {s.name for s in specs if s.replicated}
        if init:
            self.initialize(rank, seed)

    def initialize(self, rank: int, seed: int) -> None:
        for s in self.specs:
            t = self.params[s.name]
            if s.init == "one":
                t.fill_(1)
            elif s.init == "zero":
                t.zero_()
            else:
                salt = int.from_bytes(hashlib.sha256(s.tag.encode()).digest()[:8], "little")
                g = torch.Generator(device=self.device)
                g.manual_seed((seed + salt + (0 if s.replicated else 1000003 * rank)) % (2 ** 63 - 1))
                t.normal_(0, s.std, generator=g)

    def named_parameters(self):
        return [(s.name, self.params[s.name]) for s in self.specs]

    def numel(self) -> int:
        return sum(s.numel for s in self.specs)


class GPT:
    """TP/SP GPT over `TensorParallel`; one instance per rank."""

    def __init__(self, config: dict, arm: str = "flux", group=None, device="cuda", seed: int = 1234,
                 transport: str = "nvlink", execution_plan: dict | None = None, init: bool = True,
                 timeout_ns: int = 10_000_000_000, kept: str = "bf16"):
        if kept not in ("bf16", "e4m3"):
            raise ValueError("kept must be 'bf16' or 'e4m3'")
        plans = None
        if execution_plan is not None:
            plans = execution_plan.get("roles", execution_plan)
        self.tp = TensorParallel(group, arm=arm, transport=transport, chunk_rows=int(config.get("chunk_rows", 128)),
                                 plans=plans, timeout_ns=timeout_ns)
        self.world, self.rank = self.tp.world, self.tp.rank
        self.config = validate_config(config, self.world)
        self.arm = arm
        self.kept = kept
        self.sandwich = self.config.get("block_norm") == "sandwich"
        self.residual_scale = self.config.get("residual_scale", 1.0)
        self.device = torch.device(device)
        self.seed = seed
        self.specs = param_specs(self.config, self.world)
        self.store = ParamStore(self.specs, self.device, self.rank, seed, init=init)
        self.p = self.store.params
        self.g = self.store.grads
        self.forward_calls = 0
        c = self.config
        self.M = c["sequence"] * c["micro_batch"]
        self.Ml = self.M // self.world
        self.h, self.f = c["hidden"], c["ffn"]
        self.lh = c["heads"] // self.world
        self.Vl = c["vocab"] // self.world
        self.eps = c["layer_norm_epsilon"]
        counts = parameter_counts(c, self.world)
        if self.store.numel() != counts["parameters_per_rank"]:
            raise RuntimeError("parameter count differs from the configuration")
        self._ws = {}

    # --------------------------------------------------------------- state
    def named_parameters(self):
        return self.store.named_parameters()

    def parameters(self):
        return [t for _, t in self.named_parameters()]

    def state_dict(self) -> dict:
        return {name: t for name, t in self.named_parameters()}

    def load_state_dict(self, state: dict) -> None:
        names = [n for n, _ in self.named_parameters()]
        if set(state) != set(names):
            raise ValueError("state_dict keys differ from the model's parameters")
        for name in names:
            src = state[name]
            if tuple(src.shape) != tuple(self.p[name].shape):
                raise ValueError(f"shape mismatch for {name}")
            self.p[name].copy_(src)

    def _workspace(self, name, numel, dtype):
        t = self._ws.get(name)
        if t is None or t.numel() < numel or t.dtype != dtype:
            t = torch.empty(numel, dtype=dtype, device=self.device)
            self._ws[name] = t
        return t

    # ------------------------------------------------------------- forward
    def _forward(self, tokens, targets, keep: bool, loss_scale: float):
        logits, trunk = self._logits(tokens, targets, keep)
        loss, ce_state = CE.forward(logits, targets, self.tp.group, self.rank, self.world, scale=loss_scale / self.M)
        return loss, (tokens, targets, trunk, logits, ce_state) if keep else None

    def _logits(self, tokens, targets, keep: bool):
        """This rank's logits [M, V/W] and the tape of the layers (when `keep`)."""
        c, tp = self.config, self.tp
        M, Ml, h, lh = self.M, self.Ml, self.h, self.lh
        if tokens.shape != (M,) or targets.shape != (M,):
            raise ValueError("tokens/targets must hold the full flattened micro-batch")
        start = self.rank * self.Vl
        row0 = self.rank * Ml
        contrib = E.lookup(tokens, self.p["embedding"], start)
        x = tp.scatter_sum(contrib)
        E.add_position(x, self.p["position"], row0)
        saved = []
        if self.sandwich:
            lnf, first = self._sandwich_forward(x, saved, keep)
            logits, lnf_full = tp.ag_linear(("head", 0), lnf, self.p["embedding"])
            self.forward_calls += 1
            return logits, (saved, first, None, None, lnf_full)
        for i in range(c["layers"]):
            with tracing.scope(f"gpt.layer{i}.forward"):
                x = self._layer_forward(i, x, saved, keep)
        x_final = x
        buf = tp.ag_input(("head", 0), M, self.h, self.Vl, x.is_cuda)
        lnf, meanf, rstdf = N.layer_norm_fwd(x_final, self.p["final_weight"], self.p["final_bias"], self.eps, out=buf)
        logits, lnf_full = tp.ag_linear(("head", 0), lnf, self.p["embedding"])
        self.forward_calls += 1
        return logits, (saved, x_final, meanf, rstdf, lnf_full)

    # ------------------------------------------------------ the tape in 8 bits
    def _keep(self, t):
        return K.pack(t) if self.kept == "e4m3" else t

    def _keep_normed(self, full):
        """A norm's gathered output: the backward pass computes it again on one rank;
        with TP it lies in the fused operator's gather buffer anyway."""
        return None if self.kept == "e4m3" and self.world == 1 else full

    def _attention_again(self, qkv, attn, lse):
        """(qkv, attn, lse) for the attention's backward pass.  From a kept QKV the
        forward is run again, so that output, LSE and gradient belong together."""
        if not isinstance(qkv, K.Packed8):
            return qkv, attn, lse
        qkv = K.unpack(qkv)
        attn, lse = A.forward(qkv, self.config["micro_batch"], self.config["sequence"], self.lh)
        return qkv, attn, lse

    def _mlp_again(self, pre, act):
        return K.unpack_gelu(pre) if isinstance(pre, K.Packed8) else (pre, act)

    def _layer_forward(self, i, x, saved, keep):
        """One transformer block forward (pre-LN); appends its tape when `keep`."""
        c, tp, M = self.config, self.tp, self.M
        lh = self.lh
        p = f"layers.{i}."
        x_in = x
        # LayerNorm outputs are written straight into the fused AG->GEMM's gather
        # buffer (published to the peers without a copy) when TP > 1.
        h, W = self.h, self.world
        buf = tp.ag_input(("qkv", i), M, h, 3 * h // W, x.is_cuda)
        ln1, mean1, rstd1 = N.layer_norm_fwd(x_in, self.p[p + "ln1_weight"], self.p[p + "ln1_bias"], self.eps,
                                             out=buf)
        qkv, ln1_full = tp.ag_linear(("qkv", i), ln1, self.p[p + "qkv_weight"], bias=self.p[p + "qkv_bias"])
        attn, lse = A.forward(qkv, c["micro_batch"], c["sequence"], lh)
        x2 = tp.linear_rs(attn, self.p[p + "attn_weight"], residual=x_in, bias=self.p[p + "attn_bias"],
                          role="attn")
        buf = tp.ag_input(("fc1", i), M, h, self.f // W, x.is_cuda)
        ln2, mean2, rstd2 = N.layer_norm_fwd(x2, self.p[p + "ln2_weight"], self.p[p + "ln2_bias"], self.eps,
                                             out=buf)
        pre = torch.empty((M, self.f // self.world), dtype=torch.bfloat16, device=self.device)
        act, ln2_full = tp.ag_linear(("fc1", i), ln2, self.p[p + "fc1_weight"], bias=self.p[p + "fc1_bias"],
                                     gelu_aux=pre)
        x = tp.linear_rs(act, self.p[p + "fc2_weight"], residual=x2, bias=self.p[p + "fc2_bias"], role="mlp")
        if keep and self.kept == "e4m3":
            saved.append((K.pack(x_in), mean1, rstd1, self._keep_normed(ln1_full), K.pack(qkv), None, None,
                          K.pack(x2), mean2, rstd2, self._keep_normed(ln2_full), K.pack(pre), None))
        elif keep:
            saved.append((x_in, mean1, rstd1, ln1_full, qkv, attn, lse, x2, mean2, rstd2, ln2_full, pre, act))
        return x

    def _norm_backward(self, name, dy, x, mean, rstd, dres, ln_ws, normed, out):
        """Norm `name`: writes its parameter gradients; returns (dx, its gathered output
        for the following product's weight gradient)."""
        g, w = self.g, self.p[name + "_weight"]
        if isinstance(x, K.Packed8):
            again = self.p[name + "_bias"] if normed is None else None
            dx, dw, db, y = N.layer_norm_bwd_packed(dy, x, w, mean, rstd, dres=dres, bias=again, out=out)
            normed = y if normed is None else normed
        else:
            dx, dw, db = N.layer_norm_bwd(dy, x, w, mean, rstd, dres=dres, workspace=ln_ws, out=out)
        g[name + "_weight"].copy_(dw)
        g[name + "_bias"].copy_(db)
        return dx, normed

    def _layer_backward(self, i, tape, dx, ln_ws, col_ws):
        """One transformer block backward: writes its parameter gradients and
        returns the gradient of its input."""
        c, tp, g = self.config, self.tp, self.g
        p = f"layers.{i}."
        (x_in, mean1, rstd1, ln1_full, qkv, attn, lse, x2, mean2, rstd2, ln2_full, pre, act) = tape
        pre, act = self._mlp_again(pre, act)
        # fc2 (row-parallel): x = x2 + RS(act @ Wfc2^T) + b
        N.column_sum(dx, out=g[p + "fc2_bias"], workspace=col_ws)
        dpre, dfull = tp.ag_linear(("fc2_bwd", i % 2), dx, self.p[p + "fc2_weight"], b_mn=True,
                                   gelu_grad_of=pre)
        G.matmul(dfull, act, a_t=True, b_t=True, out=g[p + "fc2_weight"])
        # fc1 (column-parallel): pre = gather(ln2) @ Wfc1^T + b
        N.column_sum(dpre, out=g[p + "fc1_bias"], workspace=col_ws)
        dln2 = tp.linear_rs(dpre, self.p[p + "fc1_weight"], b_mn=True, role="mlp_bwd")
        M, h, W = self.M, self.h, self.world
        dx2, ln2_full = self._norm_backward(p + "ln2", dln2, x2, mean2, rstd2, dx, ln_ws, ln2_full,
                                            tp.ag_input(("attn_bwd", i % 2), M, h, h // W, dx.is_cuda))
        G.matmul(dpre, ln2_full, a_t=True, b_t=True, out=g[p + "fc1_weight"])
        # attention out-projection (row-parallel): x2 = x_in + RS(attn @ Wattn^T) + b
        qkv, attn, lse = self._attention_again(qkv, attn, lse)
        N.column_sum(dx2, out=g[p + "attn_bias"], workspace=col_ws)
        dattn, dfull2 = tp.ag_linear(("attn_bwd", i % 2), dx2, self.p[p + "attn_weight"], b_mn=True)
        G.matmul(dfull2, attn, a_t=True, b_t=True, out=g[p + "attn_weight"])
        dqkv = A.backward(qkv, attn, dattn, lse, c["micro_batch"], c["sequence"], self.lh)
        # QKV (column-parallel)
        N.column_sum(dqkv, out=g[p + "qkv_bias"], workspace=col_ws)
        dln1 = tp.linear_rs(dqkv, self.p[p + "qkv_weight"], b_mn=True, role="attn_bwd")
        # The input gradient feeds the previous layer's FC2-backward AG->GEMM.
        nxt = tp.ag_input(("fc2_bwd", (i - 1) % 2), M, h, self.f // W, dx2.is_cuda) if i > 0 else None
        dx, ln1_full = self._norm_backward(p + "ln1", dln1, x_in, mean1, rstd1, dx2, ln_ws, ln1_full, nxt)
        G.matmul(dqkv, ln1_full, a_t=True, b_t=True, out=g[p + "qkv_weight"])
        return dx

    # ---------------------------------------------------------- sandwich blocks
    def _join(self, i: int, branch: str):
        """Parameters of the joint after layer i's branch: its norm and gate, and the
        norm before the next branch."""
        after = f"layers.{i}.ln2" if branch == "attn" else \
            f"layers.{i + 1}.ln1" if i + 1 < self.config["layers"] else "final"
        p = f"layers.{i}.{branch}_"
        return p, after

    def _join_forward(self, i, branch, x, y, site, n):
        p, after = self._join(i, branch)
        P = self.p
        return N.block_join_fwd(x, y, P[p + "post_weight"], P[p + "post_bias"], P[p + "gate"],
                                P[after + "_weight"], P[after + "_bias"], self.eps, residual_scale=self.residual_scale,
                                out=self.tp.ag_input(site, self.M, self.h, n, x.is_cuda))

    def _join_backward(self, i, branch, dh, dx, tape, normed, site, n):
        """Gradient of a joint from that of its norm's output and of the stream; returns
        (gradient of the stream before it, of the branch's output, the norm's output)."""
        p, after = self._join(i, branch)
        P, g = self.p, self.g
        x_out, y, stats = tape
        again = P[after + "_bias"] if normed is None else None
        r = N.block_join_bwd(dh, dx, x_out, y, stats, P[p + "post_weight"], P[p + "post_bias"], P[p + "gate"],
                             P[after + "_weight"], residual_scale=self.residual_scale, pre_bias=again,
                             out=self.tp.ag_input(site, self.M, self.h, n, dh.is_cuda))
        for name, value in ((p + "post_weight", r.dpost_weight), (p + "post_bias", r.dpost_bias),
                            (p + "gate", r.dgate), (after + "_weight", r.dpre_weight), (after + "_bias", r.dpre_bias)):
            g[name].copy_(value)
        return r.dx, r.dy, r.h if normed is None else normed

    def _sandwich_forward(self, x, saved, keep):
        """All blocks; returns (the final norm's output, (x, mean, rstd, output) of the first norm)."""
        c, tp, M, h, W = self.config, self.tp, self.M, self.h, self.world
        ln, mean, rstd = N.layer_norm_fwd(x, self.p["layers.0.ln1_weight"], self.p["layers.0.ln1_bias"], self.eps,
                                          out=tp.ag_input(("qkv", 0), M, h, 3 * h // W, x.is_cuda))
        first = [self._keep(x), mean, rstd] if keep else None
        for i in range(c["layers"]):
            p = f"layers.{i}."
            with tracing.scope(f"gpt.layer{i}.forward"):
                qkv, ln1_full = tp.ag_linear(("qkv", i), ln, self.p[p + "qkv_weight"], bias=self.p[p + "qkv_bias"])
                attn, lse = A.forward(qkv, c["micro_batch"], c["sequence"], self.lh)
                y1 = tp.linear_rs(attn, self.p[p + "attn_weight"], bias=self.p[p + "attn_bias"], role="attn")
                x2, ln, st1 = self._join_forward(i, "attn", x, y1, ("fc1", i), self.f // W)
                pre = torch.empty((M, self.f // W), dtype=torch.bfloat16, device=self.device)
                act, ln2_full = tp.ag_linear(("fc1", i), ln, self.p[p + "fc1_weight"], bias=self.p[p + "fc1_bias"],
                                             gelu_aux=pre)
                y2 = tp.linear_rs(act, self.p[p + "fc2_weight"], bias=self.p[p + "fc2_bias"], role="mlp")
                last = i + 1 == c["layers"]
                x, ln, st2 = self._join_forward(i, "mlp", x2, y2, ("head", 0) if last else ("qkv", i + 1),
                                                self.Vl if last else 3 * h // W)
                if keep:
                    packed = self.kept == "e4m3"
                    saved.append((self._keep_normed(ln1_full), self._keep(qkv), None if packed else attn,
                                  None if packed else lse, (self._keep(x2), self._keep(y1), st1),
                                  self._keep_normed(ln2_full), self._keep(pre), None if packed else act,
                                  (self._keep(x), self._keep(y2), st2)))
        return ln, first

    def _sandwich_backward(self, dlnf, saved, first, lnf_full, ln_ws, col_ws):
        c, tp, g = self.config, self.tp, self.g
        M, h, W, L = self.M, self.h, self.world, self.config["layers"]
        dx, dy, _ = self._join_backward(L - 1, "mlp", dlnf, None, saved[L - 1][8], lnf_full,
                                        ("fc2_bwd", (L - 1) % 2), self.f // W)
        for i in reversed(range(L)):
            p = f"layers.{i}."
            with tracing.scope(f"gpt.layer{i}.backward"):
                ln1_full, qkv, attn, lse, join1, ln2_full, pre, act, _ = saved[i]
                pre, act = self._mlp_again(pre, act)
                N.column_sum(dy, out=g[p + "fc2_bias"], workspace=col_ws)
                dpre, dfull = tp.ag_linear(("fc2_bwd", i % 2), dy, self.p[p + "fc2_weight"], b_mn=True,
                                           gelu_grad_of=pre)
                G.matmul(dfull, act, a_t=True, b_t=True, out=g[p + "fc2_weight"])
                N.column_sum(dpre, out=g[p + "fc1_bias"], workspace=col_ws)
                dln = tp.linear_rs(dpre, self.p[p + "fc1_weight"], b_mn=True, role="mlp_bwd")
                dx, dy, ln2_full = self._join_backward(i, "attn", dln, dx, join1, ln2_full, ("attn_bwd", i % 2), h // W)
                G.matmul(dpre, ln2_full, a_t=True, b_t=True, out=g[p + "fc1_weight"])
                qkv, attn, lse = self._attention_again(qkv, attn, lse)
                N.column_sum(dy, out=g[p + "attn_bias"], workspace=col_ws)
                dattn, dfull = tp.ag_linear(("attn_bwd", i % 2), dy, self.p[p + "attn_weight"], b_mn=True)
                G.matmul(dfull, attn, a_t=True, b_t=True, out=g[p + "attn_weight"])
                dqkv = A.backward(qkv, attn, dattn, lse, c["micro_batch"], c["sequence"], self.lh)
                N.column_sum(dqkv, out=g[p + "qkv_bias"], workspace=col_ws)
                dln = tp.linear_rs(dqkv, self.p[p + "qkv_weight"], b_mn=True, role="attn_bwd")
                if i:
                    dx, dy, ln1_full = self._join_backward(i - 1, "mlp", dln, dx, saved[i - 1][8], ln1_full,
                                                           ("fc2_bwd", (i - 1) % 2), self.f // W)
                else:
                    dx, ln1_full = self._norm_backward("layers.0.ln1", dln, *first, dx, ln_ws, ln1_full, None)
                G.matmul(dqkv, ln1_full, a_t=True, b_t=True, out=g[p + "qkv_weight"])
        return dx

    # ------------------------------------------------------------------ scoring
    @torch.no_grad()
    def score(self, tokens, targets, top_k: int = 0) -> CE.TokenScores:
        """Log probability of each target, entropy and the `top_k` most probable tokens
        of every position of one micro-batch (forward only; a negative target is not
        scored).  The same on every rank."""
        logits, _ = self._logits(tokens, targets, keep=False)
        scores, _ = CE.token_logprobs(logits, targets, top_k, self.tp.group, self.rank, self.world)
        return scores

    @torch.no_grad()
    def loss(self, tokens, targets) -> torch.Tensor:
        """Mean cross-entropy of one micro-batch (forward only)."""
        loss, _ = self._forward(tokens, targets, keep=False, loss_scale=1.0)
        return loss

    # ------------------------------------------------------------ backward
    @torch.no_grad()
    def forward_backward(self, tokens, targets, loss_scale: float = 1.0, weights: torch.Tensor | None = None,
                         entropy_bonus: float = 0.0) -> torch.Tensor:
        """Forward + backward of one micro-batch; gradients of `loss * loss_scale`
        are written into `self.store.grad`.  Returns the (unscaled) mean loss.

        The loss is the mean cross-entropy, whose targets all lie in the vocabulary; with
        `weights` (FP32, one a position) or an `entropy_bonus` it is
        -mean(weight * log p(target) + entropy_bonus * entropy) over the positions, of
        which those with a negative target count as zero whatever their weight."""
        if weights is None and entropy_bonus == 0.0:
            loss, tape = self._forward(tokens, targets, keep=True, loss_scale=1.0)
            self._backward(tape, loss_scale)
            return loss
        if weights is not None and (weights.shape != targets.shape or weights.dtype != torch.float32):
            raise ValueError("weights must be FP32, one for each target")
        logits, trunk = self._logits(tokens, targets, keep=True)
        scores, state = CE.token_logprobs(logits, targets, 0, self.tp.group, self.rank, self.world)
        scored = targets >= 0  # chosen, not multiplied: an ignored position may hold anything
        w = scored.float() if weights is None else torch.where(scored, weights, 0.0)
        bonus = scored.float() * entropy_bonus
        loss = -((w * scores.logprob).sum()
                 + torch.where(scored, bonus * scores.entropy, 0.0).sum()).reshape(1) / self.M
        scale = -loss_scale / self.M
        CE.token_logprobs_backward(logits, targets, state, w * scale, bonus * scale, out=logits)
        self._backward((tokens, targets, trunk, logits, None), loss_scale)
        return loss

    def _backward(self, tape, loss_scale: float):
        """Gradients of every parameter.  Without a cross-entropy state in the tape, the
        logits hold their own gradient already."""
        c, tp = self.config, self.tp
        tokens, targets, trunk, logits, ce_state = tape
        saved, x_final, meanf, rstdf, lnf_full = trunk
        M = self.M
        start = self.rank * self.Vl
        g = self.g
        ln_ws = self._workspace("ln", 2 * 64 * self.h, torch.float32)
        col_ws = self._workspace("col", 64 * max(self.f // self.world, 3 * self.h // self.world, self.h),
                                 torch.float32)
        # Cross-entropy -> dlogits (in place), LM head (tied embedding)
        if ce_state is not None:
            CE.backward(logits, targets, ce_state, loss_scale / M)
        dlnf = tp.linear_rs(logits, self.p["embedding"], b_mn=True, role="head")
        G.matmul(logits, lnf_full, a_t=True, b_t=True, out=g["embedding"])
        if self.sandwich:
            dx = self._sandwich_backward(dlnf, saved, x_final, lnf_full, ln_ws, col_ws)
            self._embedding_backward(tokens, dx, start)
            return
        L = c["layers"]
        dx, dwf, dbf = N.layer_norm_bwd(dlnf, x_final, self.p["final_weight"], meanf, rstdf, workspace=ln_ws,
                                        out=tp.ag_input(("fc2_bwd", (L - 1) % 2), M, self.h, self.f // self.world,
                                                        dlnf.is_cuda))
        g["final_weight"].copy_(dwf)
        g["final_bias"].copy_(dbf)
        for i in reversed(range(c["layers"])):
            with tracing.scope(f"gpt.layer{i}.backward"):
                dx = self._layer_backward(i, saved[i], dx, ln_ws, col_ws)
        self._embedding_backward(tokens, dx, start)

    def _embedding_backward(self, tokens, dx, start):
        # value = scatter_sum(embedding contributions) + position
        E.position_grad(dx, self.config["sequence"], self.rank * self.Ml, out=self.g["position"])
        dcontrib = self.tp.gather_rows(dx)
        E.lookup_grad(tokens, dcontrib, self.g["embedding"], start, accumulate=True)

    def close(self):
        self.tp.close()
