"""Decode steps of one transformer layer, every product and the cache quantized.

A batch of sequences shares a prompt prefix, which is quantized into the cache
once.  Each step then runs, for one new token of every sequence,

    norm, int8 query/key/value product              mm
    the token's key and value into the cache        kv_cache_write
    attention over the prefix and the own tokens    kv_cache_attention
    int8 output product, residual, norm             mm
    router, then the int4 experts, residual         moe_swiglu_int4

Weights are random.  ``python examples/decode_step.py`` runs 64 steps of 16
sequences after a prefix of 1000 tokens and prints the time of a step, called
one by one and replayed from a HIP graph.
"""

from __future__ import annotations

import sys
import time
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "strix-halo-int4-gemms_amd"))

import amd_strix_halo_kernels as shk  # noqa: E402

CODE = 4.0 / 127  # int8 step of normalised activations; four standard deviations fit


def _norm(x):
    x = x.float()
    return x * torch.rsqrt(x.square().mean(dim=-1, keepdim=True) + 1e-6)


class Int8Linear:
    """y = x W for normalised x, with int8 codes of both."""

    def __init__(self, k, n, g, device):
        self.codes = torch.randint(-127, 128, (k, n), generator=g, dtype=torch.int8).to(device)
        self.scale = torch.full((n,), 1.7 / 127 / k**0.5, dtype=torch.bfloat16, device=device)

    def __call__(self, x):
        codes = shk.fake_quant_int(x, bits=8, scale=CODE)
        steps = torch.full((x.shape[0],), CODE, dtype=torch.bfloat16, device=x.device)
        return shk.mm(codes, self.codes, a_scale=steps, b_scale=self.scale, dtype=shk.OperandDType.INT8)


class DecoderLayer:
    def __init__(self, *, hidden=1024, heads=16, kv_heads=4, head_dim=64, experts=16, inner=704, top=2, batch=16,
                 prefix=1000, most=256, page=64, bits=4, seed=0, device="cuda"):
        g = torch.Generator().manual_seed(seed)
        self.heads, self.kv_heads, self.head_dim, self.top, self.page = heads, kv_heads, head_dim, top, page
        self.qkv = Int8Linear(hidden, (heads + 2 * kv_heads) * head_dim, g, device)
        self.project = Int8Linear(heads * head_dim, hidden, g, device)
        self.router = (torch.randn((hidden, experts), generator=g) / hidden**0.5).to(device)

        def expert(k, n):
            codes = torch.randint(-7, 8, (experts, n, k), generator=g, dtype=torch.int8)
            packed = shk.pack_int4_k_major(codes).transpose(1, 2).contiguous().to(device)
            return packed, torch.full((experts, n), 0.25 / k**0.5, dtype=torch.bfloat16, device=device)

        self.up_gate, self.up_gate_scale = expert(hidden, 2 * inner)
        self.down, self.down_scale = expert(inner, hidden)

        # pages: the prefix's first, then each sequence's in turn
        shared, own = -(-prefix // page), -(-most // page)
        self.cache = shk.new_kv_cache(shared + batch * own, page, kv_heads, head_dim, bits=bits, device=device)
        self.prefix, self.most = prefix, most
        self.prefix_pages = torch.arange(shared, dtype=torch.int32, device=device)
        self.table = shared + torch.arange(batch * own, dtype=torch.int32, device=device).view(batch, own)
        self.lengths = torch.zeros(batch, dtype=torch.int32, device=device)
        if prefix:
            kv = torch.randn((2, prefix, kv_heads, head_dim), generator=g).to(device, torch.bfloat16)
            shk.kv_cache_write(self.cache, kv[0], kv[1], torch.arange(prefix, device=device))

    def step(self, x):
        """The layer's output for one new token of each sequence, bf16 [batch,
        hidden], and what went into and came out of its operators.  Every
        sequence must hold fewer than `most` tokens."""
        batch = x.shape[0]
        n = self.lengths.long()
        page = self.table.gather(1, (n // self.page)[:, None])[:, 0].long()
        qkv = self.qkv(_norm(x)).view(batch, -1, self.head_dim)
        q, k, v = qkv.split([self.heads, self.kv_heads, self.kv_heads], dim=1)
        shk.kv_cache_write(self.cache, k, v, page * self.page + n % self.page)
        self.lengths += 1
        seen = shk.kv_cache_attention(q, self.cache, self.table, self.lengths, prefix_pages=self.prefix_pages,
                                      prefix_length=self.prefix)
        x = x + self.project(_norm(seen.reshape(batch, -1)))
        y = _norm(x)
        share, ids = torch.softmax(y @ self.router, dim=-1).topk(self.top, dim=-1)
        y = y.to(torch.bfloat16)
        out = shk.moe_swiglu_int4(y, self.up_gate, self.down, ids, share, up_gate_scale=self.up_gate_scale,
                                  down_scale=self.down_scale)
        return x + out, {"q": q, "seen": seen, "y": y, "ids": ids, "share": share, "out": out}


def main(steps=64, batch=16):
    layer = DecoderLayer(batch=batch)
    x = torch.randn((batch, 1024), device="cuda").to(torch.bfloat16)

    def run(call):
        layer.lengths.zero_()
        torch.cuda.synchronize()
        start = time.perf_counter()
        for _ in range(steps):
            call()
        torch.cuda.synchronize()
        return (time.perf_counter() - start) / steps * 1e6

    run(lambda: layer.step(x))
    eager = run(lambda: layer.step(x))
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        layer.step(x)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        layer.step(x)
    run(graph.replay)
    print(f"{steps} steps of {batch} sequences after a prefix of {layer.prefix}: {eager:.0f} us a step, "
          f"{run(graph.replay):.0f} us replayed")


if __name__ == "__main__":
    main()
