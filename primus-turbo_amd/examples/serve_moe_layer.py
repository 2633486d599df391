"""One transformer layer with a mixture of experts, served from a paged FP8 cache.

Every step takes the new tokens of some sequences, a prompt's chunk or one token
each, in any mixture: their keys and values are quantized into the cache
(``kv_cache_write``), they attend to their sequences' pages
(``paged_attention``), and the experts that they are routed to run on weights
quantized once: ``moe_decode`` for few tokens, for many the grouped GEMMs behind
``moe_permute``.  The projections are ``Float8Linear``.

    python serve_moe_layer.py        # prompts of several lengths, then single tokens
"""

from __future__ import annotations

import argparse
import os
import sys
from typing import List, Sequence

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))

import primus_turbo.pytorch as turbo  # noqa: E402
from primus_turbo.pytorch.core.low_precision import Float8QuantConfig, Format, ScalingGranularity  # noqa: E402
from primus_turbo.pytorch.core.quantized_tensor import create_quantized_weight  # noqa: E402
from primus_turbo.pytorch.modules import Float8Linear  # noqa: E402

#: tokens up to which moe_decode runs the experts; each 64 read the weights once more
FEW_TOKENS = 64


class PagedCache:
    """Pools of pages on the device and who owns which page, on the host."""

    def __init__(self, pages: int, heads: int, page: int, D: int, dtype=torch.float8_e4m3fn, device="cuda"):
        self.page, self.free = page, list(range(pages))[::-1]
        self.k, self.v = (torch.zeros(pages, heads, page, D, dtype=torch.uint8, device=device).view(dtype) for _ in range(2))
        self.ks, self.vs = (torch.zeros(pages, heads, page, device=device) for _ in range(2))
        self.pages: List[List[int]] = []
        self.lens: List[int] = []

    def add_sequence(self) -> int:
        self.pages.append([])
        self.lens.append(0)
        return len(self.lens) - 1

    def drop_sequence(self, s: int) -> None:
        self.free += self.pages[s]
        self.pages[s], self.lens[s] = [], 0

    def append(self, seqs: Sequence[int], new: Sequence[int]):
        """Room for ``new[i]`` tokens of sequence ``seqs[i]``: (slots of the new tokens, page table, cu_seqlens, lengths)."""
        slots = []
        for s, n in zip(seqs, new):
            while len(self.pages[s]) * self.page < self.lens[s] + n:
                self.pages[s].append(self.free.pop())
            slots += [self.pages[s][j // self.page] * self.page + j % self.page for j in range(self.lens[s], self.lens[s] + n)]
            self.lens[s] += n
        width = max(len(self.pages[s]) for s in seqs)
        table = [self.pages[s] + [-1] * (width - len(self.pages[s])) for s in seqs]
        cu = [0]
        for n in new:
            cu.append(cu[-1] + n)
        dev = self.k.device
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
        return torch.tensor(slots, dtype=torch.int64, device=dev), i32(table), i32(cu), i32([self.lens[s] for s in seqs])


class ServedLayer(torch.nn.Module):
    """x + attention(norm(x)), then + experts(norm(.)); weights random."""

    def __init__(self, hidden: int, heads: int, kv_heads: int, D: int, experts: int, topk: int, inner: int, ops=turbo.ops,
                 device="cuda", dtype=torch.bfloat16):
        super().__init__()
        self.heads, self.kv_heads, self.D, self.topk, self.ops = heads, kv_heads, D, topk, ops
        self.config = Float8QuantConfig(granularity=ScalingGranularity.ROWWISE, format=Format.E4M3)
        make = dict(bias=False, config=self.config, device=device, dtype=dtype)
        self.qkv = Float8Linear(hidden, (heads + 2 * kv_heads) * D, **make)
        self.proj = Float8Linear(heads * D, hidden, **make)
        self.router = torch.nn.Linear(hidden, experts, bias=False, device=device, dtype=torch.float32)
        self.norm1, self.norm2 = (torch.nn.RMSNorm(hidden, device=device, dtype=dtype) for _ in range(2))
        w1 = torch.randn(experts, 2 * inner, hidden, device=device, dtype=dtype) * hidden ** -0.5
        w2 = torch.randn(experts, hidden, inner, device=device, dtype=dtype) * inner ** -0.5
        self.w1, self.w2 = (create_quantized_weight(w, torch.float8_e4m3fn, self.config)[0] for w in (w1, w2))

    def experts(self, x: torch.Tensor) -> torch.Tensor:
        probs, idx = torch.topk(torch.softmax(self.router(x.float()), dim=1), self.topk, dim=1)
        if x.shape[0] <= FEW_TOKENS:
            return self.ops.moe_decode(x, self.w1, self.w2, idx, probs)
        E = self.w1.shape[0]
        rows, row_id_map, lens, _, total, _, p = self.ops.moe_permute(x, idx, num_local_experts=E, num_topk=self.topk, probs=probs)
        gate, up = self.ops.grouped_gemm_fp8(rows, self.w1, lens, trans_b=True, config=self.config).chunk(2, dim=1)
        act = (torch.nn.functional.silu(gate) * up * p.view(-1, 1)).to(x.dtype)
        y = self.ops.grouped_gemm_fp8(act, self.w2, lens, trans_b=True, config=self.config)
        return self.ops.moe_unpermute(y, row_id_map, total, restore_shape=x.shape, num_local_experts=E)[0]

    @torch.no_grad()
    def forward(self, x: torch.Tensor, cache: PagedCache, seqs: Sequence[int], new: Sequence[int]) -> torch.Tensor:
        """x: [sum(new), hidden], the new tokens of ``seqs`` one sequence after the other."""
        slots, table, cu, lens = cache.append(seqs, new)
        qkv = self.qkv(self.norm1(x)).view(x.shape[0], -1, self.D)
        q, k, v = qkv.split([self.heads, self.kv_heads, self.kv_heads], dim=1)
        self.ops.kv_cache_write(k, v, cache.k, cache.v, slots, cache.ks, cache.vs)
        a = self.ops.paged_attention(q, cache.k, cache.v, table, cu, lens, cache.ks, cache.vs)
        x = x + self.proj(a.reshape(x.shape[0], -1))
        return x + self.experts(self.norm2(x))


def main() -> None:
    p = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    p.add_argument("--hidden", type=int, default=2048)
    p.add_argument("--heads", type=int, default=16)
    p.add_argument("--kv-heads", type=int, default=4)
    p.add_argument("--experts", type=int, default=16)
    p.add_argument("--steps", type=int, default=32)
    args = p.parse_args()
    torch.manual_seed(0)
    layer = ServedLayer(args.hidden, args.heads, args.kv_heads, 128, args.experts, 2, 1024)
    prompts = [700, 33, 1500, 1]
    cache = PagedCache(256, args.kv_heads, 32, 128)
    seqs = [cache.add_sequence() for _ in prompts]
    layer(torch.randn(sum(prompts), args.hidden, device="cuda", dtype=torch.bfloat16), cache, seqs, prompts)
    x = torch.randn(len(seqs), args.hidden, device="cuda", dtype=torch.bfloat16)
    begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    for step in range(args.steps + 4):
        if step == 4:
            begin.record()
        x = layer(x, cache, seqs, [1] * len(seqs))
    end.record()
    torch.cuda.synchronize()
    print(f"{len(seqs)} sequences of {cache.lens} tokens: {begin.elapsed_time(end) / args.steps * 1e3:.0f} us a step and layer")


if __name__ == "__main__":
    main()
