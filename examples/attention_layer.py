"""An attention layer that serves a model: prompts, then one token at a time, over a paged cache.

    python examples/attention_layer.py [--dtype bf16] [--cache fp8] [--steps 16]

One layer with random weights: its projections are `cmpext3.linear`, the rest is the attention
operators (`qk_norm_rope`, `kv_cache_write`, `attention`, `paged_attention`).  The script packs a few
prompts of different lengths, takes them through the layer in one pass, generates tokens for all of
them, and prints the times and how far the last step is from taking each whole sequence in one pass.
"""
import argparse
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import cmpext3  # noqa: E402


class PagedCache:
    """Pages of keys and values for several sequences, in 16 bits or as 8-bit codes with scales."""

    def __init__(self, pages, page_size, kv_heads, dim, dtype, batch, device):
        self.page_size = page_size
        self.k, self.v = (torch.zeros(pages, page_size, kv_heads, dim, dtype=dtype, device=device) for _ in range(2))
        self.k_scale = self.v_scale = None
        if dtype == torch.float8_e4m3fn:
            self.k_scale, self.v_scale = (torch.zeros(pages, page_size, kv_heads, device=device) for _ in range(2))
        self.free = list(range(pages))
        self.table = torch.zeros(batch, 0, dtype=torch.int32, device=device)
        self.lens = [0] * batch
        self.seq_lens = torch.zeros(batch, dtype=torch.int32, device=device)

    def grow(self, new):
        """Room for `new` more tokens of each sequence: (slots, positions) of the tokens, in order."""
        rows, slots, positions = self.table.tolist(), [], []
        for i, n in enumerate(new):
            have = -(-self.lens[i] // self.page_size)
            need = -(-(self.lens[i] + n) // self.page_size)
            rows[i] = rows[i][:have] + [self.free.pop() for _ in range(need - have)]
            places = range(self.lens[i], self.lens[i] + n)
            positions += places
            slots += [rows[i][p // self.page_size] * self.page_size + p % self.page_size for p in places]
            self.lens[i] += n
        width = max(map(len, rows))
        device = self.table.device
        self.table = torch.tensor([r + [-1] * (width - len(r)) for r in rows], dtype=torch.int32, device=device)
        self.seq_lens = torch.tensor(self.lens, dtype=torch.int32, device=device)
        return torch.tensor(slots, device=device), torch.tensor(positions, device=device)


class AttentionLayer:
    def __init__(self, width, heads, kv_heads, dim, dtype, device, max_positions=8192, seed=0):
        g = torch.Generator(device=device).manual_seed(seed)
        rand = lambda *s: torch.randn(*s, generator=g, device=device)  # noqa: E731
        self.heads, self.kv_heads, self.dim = heads, kv_heads, dim
        self.w_qkv = (rand((heads + 2 * kv_heads) * dim, width) * width**-0.5).to(dtype)
        self.w_out = (rand(width, heads * dim) * (heads * dim) ** -0.5).to(dtype)
        self.q_norm, self.k_norm = ((1 + 0.1 * rand(dim)).to(dtype) for _ in range(2))
        self.cos, self.sin = cmpext3.rope_table(max_positions, dim, device=device)

    def forward(self, x, new, cache):
        """x [tokens, width]: `new` tokens of each sequence, packed; the cache grows by them."""
        first = all(n == 0 for n in cache.lens)
        slots, positions = cache.grow(new)
        h, hk, d = self.heads, self.kv_heads, self.dim
        qkv = cmpext3.linear(x, self.w_qkv).unflatten(-1, (h + 2 * hk, d))
        q, k = cmpext3.qk_norm_rope(qkv[:, :h], qkv[:, h : h + hk], self.cos, self.sin, positions, self.q_norm, self.k_norm)
        v = qkv[:, h + hk :]
        cmpext3.kv_cache_write(k, v, cache.k, cache.v, slots, cache.k_scale, cache.v_scale)
        starts = torch.tensor([0] + new, device=x.device).cumsum(0).to(torch.int32)
        if first:  # whole prompts: the keys and values at hand, in 16 bits
            o = cmpext3.attention(q, k, v, starts, starts)
        else:
            one = all(n == 1 for n in new)
            o = cmpext3.paged_attention(q, cache.k, cache.v, cache.table, cache.seq_lens, cu_seqlens_q=None if one else starts,
                                        k_scale=cache.k_scale, v_scale=cache.v_scale)
        return cmpext3.linear(o.flatten(1), self.w_out)


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--dtype", choices=["fp16", "bf16"], default="bf16")
    ap.add_argument("--cache", choices=["same", "fp8"], default="same")
    ap.add_argument("--prompts", type=int, nargs="+", default=[700, 31, 256, 1])
    ap.add_argument("--steps", type=int, default=16)
    ap.add_argument("--width", type=int, default=1024)
    a = ap.parse_args()
    dtype = {"fp16": torch.float16, "bf16": torch.bfloat16}[a.dtype]
    held = torch.float8_e4m3fn if a.cache == "fp8" else dtype
    heads, kv_heads, dim, page = 16, 4, 64, 32
    layer = AttentionLayer(a.width, heads, kv_heads, dim, dtype, "cuda")
    batch = len(a.prompts)
    pages = sum(-(-(n + a.steps) // page) for n in a.prompts)
    cache = PagedCache(pages, page, kv_heads, dim, held, batch, "cuda")
    xs = [torch.randn(n + a.steps, a.width, device="cuda").to(dtype) for n in a.prompts]

    torch.cuda.synchronize()
    t = time.perf_counter()
    layer.forward(torch.cat([x[:n] for x, n in zip(xs, a.prompts)]), list(a.prompts), cache)
    torch.cuda.synchronize()
    print(f"prompts of {a.prompts} tokens: {1e3 * (time.perf_counter() - t):.2f} ms")
    t = time.perf_counter()
    for i in range(a.steps):
        y = layer.forward(torch.stack([x[n + i] for x, n in zip(xs, a.prompts)]), [1] * batch, cache)
    torch.cuda.synchronize()
    if a.steps:
        print(f"{a.steps} tokens for each: {1e3 * (time.perf_counter() - t) / a.steps:.3f} ms a step")
        again = PagedCache(pages, page, kv_heads, dim, held, batch, "cuda")
        whole = layer.forward(torch.cat(xs), [len(x) for x in xs], again)
        last = whole[torch.tensor([len(x) for x in xs]).cumsum(0) - 1]
        off = (y.float() - last.float()).norm() / last.float().norm()
        print(f"the last step against whole sequences: relative difference {off:.2e}")
    return 0


if __name__ == "__main__":
    sys.exit(main())
