"""An attention layer over the 4-bit cache, as a serving loop runs it:

    x -> MXFP8 GEMM (q, k, v) -> append -> attention -> MXFP8 GEMM -> y

and, every few steps, the cache thinned out to a budget by the attention weight its tokens have
gathered.  ``python -m gcnasm_b200.kv4_demo`` runs a prompt and some decode steps with random
weights on the current GPU and prints what they take.
"""
from __future__ import annotations

import torch

from . import kv4, ops


class KV4Attention:
    """One layer's weights (quantised once) and cache.  ``pages`` pages of ``page_size`` tokens are
    shared by the sequences; ``table`` [seqs, pages a sequence] names each one's."""

    def __init__(self, w_qkv: torch.Tensor, w_out: torch.Tensor, heads: int, kv_heads: int, head_dim: int, pages: int,
                 page_size: int = 64):
        self.heads, self.kv_heads, self.head_dim = heads, kv_heads, head_dim
        self.qkv, self.out = ops.quant_mxfp8(w_qkv), ops.quant_mxfp8(w_out)
        self.cache = kv4.alloc(pages, kv_heads, head_dim, page_size, device=w_qkv.device)
        self.gathered = kv4.alloc_weights(self.cache)

    def __call__(self, x: torch.Tensor, table: torch.Tensor, lens: torch.Tensor, cu: torch.Tensor | None = None,
                 max_new: int = 1, gather: bool = True) -> torch.Tensor:
        """bf16 rows [rows, dim] of the sequences' new tokens, which ``lens`` counts already -> [rows, dim]."""
        q8, sf = ops.quant_mxfp8(x)
        qkv = ops.mxfp8_gemm(q8, self.qkv[0], sf, self.qkv[1]).view(x.shape[0], -1, self.head_dim)
        q, k, v = qkv.split([self.heads, self.kv_heads, self.kv_heads], dim=1)
        kv4.append(self.cache, k, v, table, lens, cu, max_new=max_new, weights=self.gathered)
        o, lse = kv4.attention(q, self.cache, table, lens, cu, max_q=max_new)
        if gather:
            kv4.weights(q, lse, self.cache, table, lens, self.gathered, cu, max_q=max_new)
        o8, sf = ops.quant_mxfp8(o.view(x.shape[0], -1))
        return ops.mxfp8_gemm(o8, self.out[0], sf, self.out[1])

    def thin_out(self, table: torch.Tensor, lens: torch.Tensor, budget: int, sink: int = 4, recent: int = 64) -> torch.Tensor:
        """Thins the sequences out in place; ``lens`` is updated.  The numbers that the kept tokens had."""
        kept, _ = kv4.evict(self.cache, self.gathered, table, lens, budget, sink=sink, recent=recent, out_lens=lens)
        return kept


def generate(layer: KV4Attention, prompts: list[int], steps: int, dim: int, budget: int, every: int = 16, seed: int = 0):
    """Prompts of the given lengths at once, then ``steps`` decode steps; yields each call's output."""
    dev, page = layer.gathered.device, layer.cache.page_size
    gen = torch.Generator(device=dev).manual_seed(seed)
    seqs = len(prompts)
    width = -(-(max(max(prompts), budget + every) + steps + 1) // page)
    table = torch.randperm(layer.cache.pages, generator=gen, device=dev)[:seqs * width].to(torch.int32).view(seqs, width)
    lens = torch.tensor(prompts, dtype=torch.int32, device=dev)
    cu = torch.tensor([0, *prompts], dtype=torch.int32, device=dev).cumsum(0, dtype=torch.int32)

    def rows(n):
        return torch.randn((n, dim), generator=gen, device=dev).to(torch.bfloat16)

    yield layer(rows(sum(prompts)), table, lens, cu, max(prompts)), lens
    for step in range(steps):
        if step % every == 0:
            layer.thin_out(table, lens, budget, recent=min(64, budget // 2))
        lens += 1
        yield layer(rows(seqs), table, lens), lens


def main() -> None:
    torch.manual_seed(0)
    dim, heads, kv_heads, head_dim, prompts, steps, budget = 4096, 32, 8, 128, [1500, 700, 2048, 64], 64, 1024
    dev = torch.device("cuda")
    w_qkv = torch.randn(((heads + 2 * kv_heads) * head_dim, dim), device=dev) * dim ** -0.5
    w_out = torch.randn((dim, heads * head_dim), device=dev) * (heads * head_dim) ** -0.5
    layer = KV4Attention(w_qkv, w_out, heads, kv_heads, head_dim, pages=256)
    for what in ("first run", "second run"):
        events = [torch.cuda.Event(enable_timing=True) for _ in range(3)]
        events[0].record()
        for i, (y, lens) in enumerate(generate(layer, prompts, steps, dim, budget)):
            if i == 0:
                events[1].record()
        events[2].record()
        torch.cuda.synchronize()
        print(f"{what}: {sum(prompts)} prompt tokens {events[0].elapsed_time(events[1]):.2f} ms, {steps} steps of "
              f"{len(prompts)} tokens {events[1].elapsed_time(events[2]) / steps * 1e3:.0f} us each; lengths {lens.tolist()}, "
              f"cache {layer.cache.k.numel() * 2 * 17 / 16 / 1e6:.0f} MB, device status {ops.device_status()}")


if __name__ == "__main__":
    main()
