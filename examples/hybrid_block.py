"""A hybrid block built from the package's operators: linear attention with a decay per head, then attention over a
paged cache, with the residual stream through RMS norms between them.

    python examples/hybrid_block.py            # needs a ROCm GPU

A prompt goes through in pieces, the tokens after it one by one: the linear layer carries its state, the attention
layer writes its keys and values into pages (in 8 bits) and reads them through a block table, and the last norm
leaves what a projection in 8 bits takes.  The linear layer's half also trains.
"""
import math
import os
import sys

import torch
import torch.nn.functional as F

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import avelang_amd as ave  # noqa: E402


class Pages:
    """A cache's pages, handed out to sequences as they grow."""

    def __init__(self, sequences, most, page, kv_heads, size, dtype, device="cuda"):
        width = -(-most // page)
        self.cache = ave.PagedKVCache.zeros(sequences * width, page, kv_heads, size, dtype, device)
        order = torch.randperm(sequences * width, device=device).int()
        self.table = order.view(sequences, width)
        self.lengths = torch.zeros(sequences, dtype=torch.int32, device=device)
        self.page = page

    def grow(self, tokens):
        """Positions and slots [N, tokens] of the next tokens of every sequence."""
        at = self.lengths[:, None].long() + torch.arange(tokens, device=self.lengths.device)
        self.lengths += tokens
        return at, self.table.gather(1, at // self.page).long() * self.page + at % self.page


class HybridBlock(torch.nn.Module):
    def __init__(self, width, linear_heads=(2, 4), heads=(8, 2), size=128, rotated=None, device="cuda"):
        super().__init__()
        self.linear, self.heads, self.size = linear_heads, heads, size
        bf = dict(dtype=torch.bfloat16, device=device)
        w = lambda *s: torch.nn.Parameter(torch.randn(*s, **bf) / math.sqrt(s[1]))  # noqa: E731
        self.norms = torch.nn.ParameterList(torch.nn.Parameter(0.1 * torch.randn(width, **bf)) for _ in range(3))
        hqk, hv = linear_heads
        self.lin_widths = [hqk * size, hqk * size, hv * size]
        self.lin_in, self.decay, self.lin_out = w(sum(self.lin_widths), width), w(hv, width), w(width, hv * size)
        hq, hkv = heads
        self.att_widths = [hq * size, hkv * size, hkv * size]
        self.att_in, self.att_out = w(sum(self.att_widths), width), w(width, hq * size)
        freq, self.magnitude = ave.rotary_frequencies(size if rotated is None else rotated, factor=8.0, original=4096)
        self.register_buffer("freq", freq.to(device))

    def rotate(self, q, k, positions):
        return ave.rotary_embedding(q, k, positions, self.freq, magnitude=self.magnitude)

    def linear_layer(self, x, positions, state=None, decode=False):
        """x [B, T, width] -> (its output, the state)."""
        B, T, _ = x.shape
        y = ave.rms_norm(x, self.norms[0], offset=1.0)
        q, k, v = F.linear(y, self.lin_in).split(self.lin_widths, -1)   # read in place
        q, k, v = (t.view(B, T, -1, self.size) for t in (q, k, v))
        q, k = self.rotate(q, k, positions)
        g = F.logsigmoid(F.linear(y, self.decay).float() + 3.0)
        if decode:
            o, state = ave.fused_recurrent_linear_attn(q, k, v, g, initial_state=state, output_final_state=True)
        else:
            o, state = ave.chunk_linear_attn(q, k, v, g, initial_state=state, output_final_state=True)
        return F.linear(o.flatten(2), self.lin_out), state

    def attention_layer(self, y, positions, slots, pages):
        """y [N, T, width] of new tokens, any T (every 64 rows of T tokens and a kv-head's q-heads read the whole
        cache: pieces of some dozens of tokens are what the operator is made for)."""
        N, T, _ = y.shape
        q, k, v = F.linear(y, self.att_in).split(self.att_widths, -1)
        q, k, v = (t.view(N, T, -1, self.size) for t in (q, k, v))
        q, k = self.rotate(q, k, positions)
        ave.paged_cache_write(pages.cache, k, v, slots)
        o = ave.paged_attention(q, pages.cache, pages.table, pages.lengths)
        return F.linear(o.flatten(2), self.att_out)

    def train_half(self, x, positions):
        """The linear layer and the norm behind it: (the next layer's input, the residual stream)."""
        a, _ = self.linear_layer(x, positions)
        return ave.rms_norm(a, self.norms[1], residual=x, offset=1.0)

    @torch.no_grad()
    def serve(self, x, state, pages, decode=False):
        """The next tokens x [N, T, width] of every sequence: (codes, scale, residual stream, state)."""
        positions, slots = pages.grow(x.shape[1])
        a, state = self.linear_layer(x, positions, state, decode)
        y, h = ave.rms_norm(a, self.norms[1], residual=x, offset=1.0)
        a = self.attention_layer(y, positions, slots, pages)
        codes, scale, h = ave.rms_norm_quant(a, self.norms[2], residual=h, offset=1.0)
        return codes, scale, h, state


def main():
    torch.manual_seed(0)
    block = HybridBlock(512)
    x = torch.randn(3, 200, 512, device="cuda").bfloat16()
    outs = {}
    for dtype in (torch.bfloat16, torch.float8_e4m3fn, torch.int8):
        pages, state, parts = Pages(3, 256, 16, 2, 128, dtype), None, []
        for t in range(0, 192, 64):   # the prompt in pieces
            *_, h, state = block.serve(x[:, t:t + 64], state, pages)
            parts.append(h)
        for t in range(192, 200):     # and token by token
            codes, scale, h, state = block.serve(x[:, t:t + 1], state, pages, decode=True)
            parts.append(h)
        outs[dtype] = torch.cat(parts, 1).float()
        base = outs[torch.bfloat16]
        far = (outs[dtype] - base).norm() / base.norm()
        print(f"cache in {dtype}: {far:.1e} from bf16's, the next projection's input {codes.dtype} "
              f"{tuple(codes.shape)}")
    opt = torch.optim.SGD(block.parameters(), lr=0.5)
    positions = torch.arange(200, device="cuda")
    for step in range(3):
        y, h = block.train_half(x, positions)
        loss = (y.float() - 1).square().mean() + 0.1 * h.float().square().mean()
        opt.zero_grad()
        loss.backward()
        opt.step()
        print(f"step {step}: loss {loss.item():.4f}")


if __name__ == "__main__":
    main()
