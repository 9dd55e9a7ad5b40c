"""Fine-tunes a DiT block's MLP sub-layer whose weights come from GGUF blocks, with the training-step operators together:

    x + gate * down(gelu(up(LayerNorm(x) * (1 + scale) + shift)))

``fused_norm.layer_norm`` (modulation), ``fused_dense.dense`` (GELU in the first product's epilogue, the gated residual in
the second's) and ``fused_adamw.AdamW`` (moments in 8 bits). The student starts from the Q4_K dequantisation of a teacher's
weights (``gguf_dequant.dequantize``) and learns to undo the quantisation on synthetic tokens.

    python -m comfyui-weightferry_amd.examples.finetune_mlp [--width 2048 --hidden 8192 --tokens 1024 --steps 200]

run from the directory that holds the package; needs an MI355X. Prints the loss before and after, and the time of a step."""
import argparse
import time

import torch

from .. import gguf_encode
from ..enhancers import fused_adamw, fused_dense, fused_norm, gguf_dequant

Q4_K = 12


class ModulatedMLP(torch.nn.Module):
    """The sub-layer on bfloat16 weights; ``modulation`` is (shift, scale, gate), each [batch, width]."""

    def __init__(self, up, down):
        super().__init__()
        self.up, self.down = torch.nn.Parameter(up), torch.nn.Parameter(down)
        self.up_bias = torch.nn.Parameter(up.new_zeros(up.shape[0]))
        self.down_bias = torch.nn.Parameter(down.new_zeros(down.shape[0]))

    def forward(self, x, modulation):
        shift, scale, gate = modulation
        h = fused_norm.layer_norm(x, scale, shift, eps=1e-6, modulation=True)
        h = fused_dense.dense(h, self.up, self.up_bias, act="gelu_tanh")
        return fused_dense.dense(h, self.down, self.down_bias, residual=x, gate=gate)


def quantised(shape, seed):
    """(a weight, its Q4_K dequantisation), both bfloat16 on the GPU."""
    w = gguf_encode.weights(shape, seed=seed)
    raw = torch.from_numpy(gguf_encode.encode(w, Q4_K)).cuda()
    back = gguf_dequant.dequantize(raw, Q4_K, shape, None, torch.bfloat16)
    return torch.from_numpy(w).to("cuda", torch.bfloat16), back.clone()


def run(width=2048, hidden=8192, tokens=1024, batch=2, steps=60, lr=1e-4, bits=8, seed=0):
    """{"before", "after": the loss, "ms": a step's time}"""
    g = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")                               # noqa: E731
    (up, up_q), (down, down_q) = quantised((hidden, width), seed), quantised((width, hidden), seed + 1)
    teacher, student = ModulatedMLP(up, down), ModulatedMLP(up_q, down_q)
    teacher.requires_grad_(False)
    optimizer = fused_adamw.AdamW(student.parameters(), lr=lr, weight_decay=0.0, bits=bits)
    losses, began = [], 0.0
    for step in range(steps + 1):
        if step == 1:                                    # (the first step loads the kernels)
            torch.cuda.synchronize()
            began = time.perf_counter()
        x = rnd(batch, tokens, width).to(torch.bfloat16)
        modulation = [(0.3 * rnd(batch, width)).to(torch.bfloat16) for _ in range(3)]
        with torch.no_grad():
            want = teacher(x, modulation)
        loss = (student(x, modulation) - want).float().square().mean()
        loss.backward()
        optimizer.step()
        optimizer.zero_grad()
        losses.append(loss.detach())
    torch.cuda.synchronize()
    ms = (time.perf_counter() - began) / max(1, steps) * 1e3
    ends = max(1, min(5, steps // 4))
    return {"before": float(torch.stack(losses[:ends]).mean()), "after": float(torch.stack(losses[-ends:]).mean()), "ms": ms}


def main():
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    for name, value in (("width", 2048), ("hidden", 8192), ("tokens", 1024), ("steps", 200), ("bits", 8)):
        ap.add_argument(f"--{name}", type=int, default=value)
    ap.add_argument("--lr", type=float, default=1e-4)
    a = ap.parse_args()
    r = run(a.width, a.hidden, a.tokens, steps=a.steps, lr=a.lr, bits=a.bits)
    print(f"loss {r['before']:.3e} -> {r['after']:.3e}, {r['ms']:.2f} ms a step")


if __name__ == "__main__":
    main()
