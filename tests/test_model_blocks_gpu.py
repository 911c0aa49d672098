"""Sandwich blocks, the 8-bit tape, scoring and weighted losses of GPT on the GPU
against the CPU oracle run of the same parameters."""
import pytest
import torch

pytestmark = pytest.mark.gpu

CFG = dict(layers=2, hidden=256, ffn=1024, heads=2, sequence=512, micro_batch=2,
           accumulation_steps=1, vocab=2048, chunk_rows=128)
SANDWICH = dict(CFG, block_norm="sandwich", residual_scale=0.9)


def rel(a, b):
    return ((a.float() - b.float()).norm() / b.float().norm().clamp_min(1e-12)).item()


def batch(seed=1):
    g = torch.Generator().manual_seed(seed)
    M = CFG["sequence"] * CFG["micro_batch"]
    tokens = torch.randint(0, CFG["vocab"], (M,), generator=g)
    targets = torch.randint(0, CFG["vocab"], (M,), generator=g)
    targets[::5] = -100
    return tokens, targets, torch.rand(M, generator=g)


def pair(cfg, kept):
    from tempname_5090_b200.models.gpt import GPT
    gpu = GPT(cfg, device="cuda", seed=3, kept=kept)
    g = torch.Generator(device="cuda").manual_seed(8)
    for _, t in gpu.named_parameters():
        if t.dim() == 1:
            t.add_((0.2 * torch.randn(t.shape, generator=g, device="cuda")).to(t.dtype))
    cpu = GPT(cfg, device="cpu", seed=3, init=False, kept=kept)
    cpu.load_state_dict({k: v.cpu() for k, v in gpu.state_dict().items()})
    return gpu, cpu


@pytest.mark.parametrize("kept", ["bf16", "e4m3"])
@pytest.mark.parametrize("cfg", [CFG, SANDWICH], ids=["pre", "sandwich"])
def test_gpu_matches_the_cpu_oracle(cfg, kept):
    from tempname_5090_b200._native import check_status
    gpu, cpu = pair(cfg, kept)
    tokens, targets, weights = batch()
    got = gpu.score(tokens.cuda(), targets.cuda(), top_k=5)
    want = cpu.score(tokens, targets, top_k=5)
    assert rel(got.logprob.cpu(), want.logprob) < 1e-2 and rel(got.entropy.cpu(), want.entropy) < 1e-2
    assert rel(got.top_logprobs.cpu(), want.top_logprobs) < 1e-2
    for wts, bonus in ((None, 0.0), (weights, 0.02)):
        t = targets if wts is not None else targets.clamp(min=0)
        lg = gpu.forward_backward(tokens.cuda(), t.cuda(), 1.0, None if wts is None else wts.cuda(), bonus)
        lc = cpu.forward_backward(tokens, t, 1.0, wts, bonus)
        torch.cuda.synchronize()
        check_status()
        assert abs(lg.item() - lc.item()) < 1e-2 * abs(lc.item())
        first = {k: v.clone() for k, v in gpu.g.items()}
        for name in gpu.state_dict():
            # a rounding that falls the other way moves a kept value by a code's step
            assert rel(gpu.g[name].cpu(), cpu.g[name]) < (5e-2 if kept == "bf16" else 1e-1), name
        gpu.forward_backward(tokens.cuda(), t.cuda(), 1.0, None if wts is None else wts.cuda(), bonus)
        assert all(torch.equal(gpu.g[k], first[k]) for k in first)


def test_weighted_training_steps_are_deterministic():
    from tempname_5090_b200.models.gpt import GPT
    from tempname_5090_b200.models.train import Trainer
    tokens, targets, weights = batch(2)
    ends = []
    for _ in range(2):
        model = GPT(SANDWICH, device="cuda", seed=5, kept="e4m3")
        trainer = Trainer(model, entropy_bonus=0.01)
        run = [trainer.train_step([(tokens.pin_memory(), targets.pin_memory(), weights.pin_memory())])
               for _ in range(3)]
        ends.append((run, model.store.flat.clone()))
    assert ends[0][0] == ends[1][0] and torch.equal(ends[0][1], ends[1][1])


def test_the_tape_in_8_bits_takes_less_memory():
    from tempname_5090_b200.models.gpt import GPT
    cfg = dict(CFG, layers=4, hidden=1024, ffn=4096, heads=8)
    tokens, targets, _ = batch()
    tokens, targets = tokens.cuda(), targets.clamp(min=0).cuda()
    sizes = {}
    for kept in ("bf16", "e4m3"):
        model = GPT(cfg, device="cuda", seed=1, kept=kept)
        before = torch.cuda.memory_allocated()
        _, tape = model._forward(tokens, targets, True, 1.0)
        logits = tape[3].numel() * 2
        sizes[kept] = torch.cuda.memory_allocated() - before - logits
        del tape, model
    assert sizes["e4m3"] < 0.4 * sizes["bf16"]
