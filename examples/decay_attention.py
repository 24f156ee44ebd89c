"""A linear-attention block built from the package's operators: a prompt, the
tokens after it one by one, and a training step.

    python examples/decay_attention.py            # needs a ROCm GPU

Layer norm before the projections, linear attention with a learned decay per
token and head (or a fixed slope per head), a norm of every head's output with
parameters of its own, the output projection.  A prompt goes through the
chunked form and leaves the state; decode carries it from token to token.
"""
import math
import os
import sys

import torch
import torch.nn.functional as F

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import avelang_amd as ave  # noqa: E402


class DecayAttention(torch.nn.Module):
    def __init__(self, width, qk_heads, v_heads, k_size=128, v_size=128, slopes=False,
                 device="cuda"):
        super().__init__()
        self.sizes = qk_heads, v_heads, k_size, v_size
        self.widths = [qk_heads * k_size, qk_heads * k_size, v_heads * v_size]
        bf = dict(dtype=torch.bfloat16, device=device)
        f32 = dict(dtype=torch.float32, device=device)
        w = lambda *s: torch.nn.Parameter(torch.randn(*s, **bf) / math.sqrt(s[1]))  # noqa: E731
        self.norm_w = torch.nn.Parameter(torch.ones(width, **f32))
        self.norm_b = torch.nn.Parameter(torch.zeros(width, **f32))
        self.qkv = w(sum(self.widths), width)
        self.head_w = torch.nn.Parameter(torch.ones(v_heads, v_size, **f32))
        self.head_b = torch.nn.Parameter(torch.zeros(v_heads, v_size, **f32))
        self.out = w(width, v_heads * v_size)
        if slopes:
            s = -torch.exp2(-8.0 * torch.arange(1, v_heads + 1, **f32) / v_heads)
            self.register_buffer("slope", s)
        else:
            self.slope = None
            self.decay = w(v_heads, width)

    def forward(self, x, state=None, cu_seqlens=None, decode=False):
        """x [B, T, width] bf16 -> (y, state)."""
        hqk, hv, K, V = self.sizes
        B, T, _ = x.shape
        y = ave.layer_norm(x, self.norm_w, self.norm_b)
        q, k, v = F.linear(y, self.qkv).split(self.widths, -1)   # read in place
        q, k, v = q.view(B, T, hqk, K), k.view(B, T, hqk, K), v.view(B, T, hv, V)
        g = self.slope
        if g is None:
            g = F.logsigmoid(F.linear(y, self.decay).float() + 3.0)
        if decode:
            o, state = ave.fused_recurrent_linear_attn(q, k, v, g, initial_state=state,
                                                       output_final_state=True)
        else:
            o, state = ave.chunk_linear_attn(q, k, v, g, initial_state=state,
                                             output_final_state=True, cu_seqlens=cu_seqlens)
        o = ave.layer_norm(o, self.head_w, self.head_b)   # every head's row by itself
        return x + F.linear(o.reshape(B, T, hv * V), self.out), state


def main():
    torch.manual_seed(0)
    block = DecayAttention(1024, 4, 8)
    x = torch.randn(2, 300, 1024, device="cuda").bfloat16()
    with torch.no_grad():
        whole, end = block(x)
        y, state = block(x[:, :296])
        steps = [y]
        for t in range(296, 300):
            y, state = block(x[:, t:t + 1], state, decode=True)
            steps.append(y)
        far = (torch.cat(steps, 1) - whole).float().norm() / whole.float().norm()
        print(f"prompt of 296 and 4 tokens against a prompt of 300: {far:.1e} apart, "
              f"states {(state - end).norm() / end.norm():.1e}")
    opt = torch.optim.SGD(block.parameters(), lr=1.0)
    for step in range(3):
        y, _ = block(x)
        loss = (y.float() - 1).square().mean()
        opt.zero_grad()
        loss.backward()
        opt.step()
        print(f"step {step}: loss {loss.item():.4f}")


if __name__ == "__main__":
    main()
