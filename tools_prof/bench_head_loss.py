"""The vocabulary head's loss with and without logits where the package uses it: forward and backward of the operator with a
bf16 and an fp32 head, and whole training steps (packed rows, dropout 0.1, AdamW + clip) of the small denoiser with
``fused_head_loss`` off and on, with softmax and with differential attention and rotary positions."""
import os, sys, time
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "discrete-diffusion-model-for-inverse-polymer-design_amd")); sys.path.insert(0, ROOT)
import torch
import bench
from bidiff import ops
from bidiff.model.backbone import DiffusionBackbone
from bidiff.model.diffusion import DiscreteMaskingDiffusion
from bidiff.training.optimizer import FlatAdamW

dev = torch.device("cuda:0")


def micros(f, n=30):
    times = []
    for _ in range(5):
        for _ in range(3):
            f()
        torch.cuda.synchronize(); t0 = time.perf_counter()
        for _ in range(n):
            f()
        torch.cuda.synchronize()
        times.append((time.perf_counter() - t0) / n * 1e6)
    return sorted(times)[2]


for M, d, V in ((32768, 384, 39), (32768, 384, 803), (3001, 768, 32003), (8192, 2048, 65536)):
    h = torch.randn(M, d, device=dev).bfloat16().requires_grad_(True)
    t, ind = torch.randint(0, V, (M,), device=dev), torch.rand(M, device=dev) < 0.5
    line = []
    for dt in (torch.bfloat16, torch.float32):
        w = (torch.randn(V, d, device=dev) / d ** 0.5).to(dt).requires_grad_(True)
        line.append(micros(lambda: torch.autograd.grad(ops.linear_cross_entropy(h, w, t, ind), (h, w)), 10 if V > 40000 else 30))
    print(f"{M} x {d} -> {V}, half of the rows weighted, forward and backward: bf16 head {line[0]:.0f} us, fp32 head {line[1]:.0f} us", flush=True)

for V, B in ((39, 256), (803, 256)):
    ids, attn = bench.bpe_batch(B, 128, V, 1)
    tokens, lens = int(attn.sum()), attn.sum(1).tolist()
    ids, attn = torch.from_numpy(ids).to(dev), torch.from_numpy(attn).to(dev)
    for kind in ({}, {"attention": "differential", "rotary_base": 10000.0}):
        line = []
        for fused in (False, True):
            torch.manual_seed(0)
            bb = DiffusionBackbone(V, 384, 6, 6, 1536, 256, 50, 0.1, 0, **kind)
            model = DiscreteMaskingDiffusion(bb, num_steps=50, mask_token_id=1, pad_token_id=0, bos_token_id=2, eos_token_id=3).to(dev).train()
            model.corruption_rng, model.fused_head_loss = "philox", fused
            opt = FlatAdamW(model.parameters(), lr=3e-4, weight_decay=0.01)

            def step():
                model(ids, attn, lengths=lens)["loss"].backward()
                opt.step(max_norm=1.0)
                opt.zero_grad()
            torch.cuda.reset_peak_memory_stats()
            us = micros(step, 20)
            line.append(f"{us / 1e3:.2f} ms, {torch.cuda.max_memory_allocated() / 2**20:.0f} MB")
            del model, bb, opt
            torch.cuda.empty_cache()
        print(f"training step, V {V}, {B} x 128 ({tokens} tokens), d 384, 6 layers, 6 heads, {kind.get('attention', 'softmax')}"
              f"{' + rotary' if kind else ''}: logits {line[0]}; fused {line[1]}", flush=True)
