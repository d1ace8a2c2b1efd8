"""Steps of one decoder layer that verify drafted tokens, with fp8 projections.

Each sequence brings its last token and the tokens that were drafted after it.
A step runs, for all of them at once,

    pages and slots of the new tokens                kv_pages_step
    norm, fp8 query/key/value product                quantize_fp8, mm_fp8
    head norms and rotation, keys and values into
    the quantized cache                              rotate_qk
    attention over each sequence's cached tokens     kv_cache_attention
    fp8 output product, residual, norm               quantize_fp8, mm_fp8
    fp8 product with the vocabulary, softmax         quantize_fp8, mm_fp8
    which drafts stay, the token behind them, and
    the lengths without the others                   verify_draft

Weights are random, and the drafts are the layer's own likeliest tokens with
some noise.  Nothing of a step is read back to the host.  A sequence that gets no
places (the pool or its row of the table is full) sits the step out.  ``python
examples/draft_step.py`` runs steps of 16 sequences with five drafts each and
prints the time of a step, called one by one and replayed from a HIP graph, and
how many drafts were kept.
"""

from __future__ import annotations

import sys
import time
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "strix-halo-int4-gemms_amd"))

import amd_strix_halo_kernels as shk  # noqa: E402


def _norm(x):
    x = x.float()
    return (x * torch.rsqrt(x.square().mean(dim=-1, keepdim=True) + 1e-6)).to(torch.bfloat16)


class Fp8Linear:
    """y = x w^T with fp8 codes of both, one scale for 128 x 128 of w and for 1 x 128 of x."""

    def __init__(self, inputs, outputs, g, device, gain=1.0):
        w = torch.randn((outputs, inputs), generator=g) * gain / inputs**0.5
        self.codes, self.scales = shk.quantize_fp8(w.to(device), block_rows=128)

    def __call__(self, x, dtype=torch.bfloat16):
        codes, scales = shk.quantize_fp8(x)
        return shk.mm_fp8(codes, self.codes, a_scale=scales, b_scale=self.scales, out_dtype=dtype)


class DraftLayer:
    def __init__(self, *, hidden=1024, heads=16, kv_heads=4, head_dim=64, vocab=8192, batch=16, drafts=5, most=1024,
                 page=64, bits=8, rotated=None, seed=0, device="cuda"):
        g = torch.Generator().manual_seed(seed)
        self.batch, self.drafts, self.heads, self.kv_heads, self.head_dim = batch, drafts, heads, kv_heads, head_dim
        self.qkv = Fp8Linear(hidden, (heads + 2 * kv_heads) * head_dim, g, device)
        self.project = Fp8Linear(heads * head_dim, hidden, g, device)
        self.embedding = torch.randn((vocab, hidden), generator=g).to(device, torch.bfloat16)
        self.head = Fp8Linear(hidden, vocab, g, device, gain=3.0)
        self.norms = [(0.5 + torch.rand(head_dim, generator=g)).to(device) for _ in range(2)]
        frequencies, amplitude = shk.rotary_frequencies(rotated or head_dim, scaling="yarn", factor=4.0, trained=2048)
        self.rotary = shk.new_rotary(frequencies, amplitude=amplitude, device=device)
        width = -(-most // page)
        self.pages = shk.new_kv_pages(batch, width, batch * width, page, device=device)
        self.cache = shk.new_kv_cache(batch * width, page, kv_heads, head_dim, bits=bits, device=device)
        self.new = torch.full((batch,), 1 + drafts, dtype=torch.int32, device=device)

    def step(self, tokens, draft, uniforms):
        """tokens [batch, 1 + drafts]: each sequence's last token and its drafts, which draft [batch, drafts,
        vocab] gave; returns verify_draft's result, and what went into and came out of the operators.  A sequence
        that got no places keeps its length and has no token: its row is -1 and none of its drafts is kept."""
        count = self.batch * (1 + self.drafts)
        at = shk.kv_pages_step(self.pages, self.new, count)
        x = self.embedding[tokens.flatten()]
        qkv = self.qkv(_norm(x)).view(count, -1, self.head_dim)
        q, k, v = qkv.split([self.heads, self.kv_heads, self.kv_heads], dim=1)
        q = shk.rotate_qk(q, k, at.positions, self.rotary, q_weight=self.norms[0], k_weight=self.norms[1],
                          cache=self.cache, values=v, slots=at.slots)
        q = q.view(self.batch, 1 + self.drafts, self.heads, self.head_dim)
        lengths = self.pages.lengths.clone()
        seen = shk.kv_cache_attention(q, self.cache, self.pages.page_table, lengths)
        y = x + self.project(seen.reshape(count, -1))
        logits = self.head(_norm(y), torch.float32)
        target = torch.softmax(logits, dim=-1).view(self.batch, 1 + self.drafts, -1)
        # only drafts that got places are in the cache, and counted in the lengths
        out, kept = shk.verify_draft(target, draft, tokens[:, 1:].contiguous(), uniforms,
                                     counts=(at.taken - 1).clamp(min=0), lengths=self.pages.lengths)
        out = torch.where(at.taken[:, None] > 0, out, -1)
        return out, kept, {"step": at, "q": q, "qkv": qkv, "lengths": lengths, "seen": seen, "y": y, "logits": logits,
                           "target": target}


def propose(layer, tokens, g, noise=1.0):
    """Drafts behind each sequence's token: a random draft model that knows nothing but the vocabulary's head."""
    drafts = []
    probabilities = []
    for _ in range(layer.drafts):
        logits = layer.head(_norm(layer.embedding[tokens]), torch.float32)
        p = torch.softmax(logits + noise * torch.randn(logits.shape, device=logits.device, generator=g), dim=-1)
        tokens = torch.multinomial(p, 1, generator=g)[:, 0]
        drafts.append(tokens)
        probabilities.append(p)
    return torch.stack(drafts, dim=1), torch.stack(probabilities, dim=1)


def main(steps=24, batch=16):
    layer = DraftLayer(batch=batch)
    g = torch.Generator(device="cuda").manual_seed(1)
    last = torch.randint(0, 8192, (batch,), device="cuda", generator=g)
    drafted, draft = propose(layer, last, g)
    tokens = torch.cat((last[:, None], drafted), dim=1)
    uniforms = torch.rand((batch, 1 + layer.drafts), device="cuda", generator=g)

    def run(call):
        for t in (layer.pages.lengths, layer.pages.owned):
            t.zero_()
        fresh = shk.new_kv_pages(batch, layer.pages.page_table.shape[1], layer.cache.pages, layer.cache.page_size)
        layer.pages.free_pages.copy_(fresh.free_pages)
        layer.pages.free_count.copy_(fresh.free_count)
        torch.cuda.synchronize()
        start = time.perf_counter()
        for _ in range(steps):
            call()
        torch.cuda.synchronize()
        return (time.perf_counter() - start) / steps * 1e6

    kept = []
    run(lambda: kept.append(layer.step(tokens, draft, uniforms)[1]))
    eager = run(lambda: layer.step(tokens, draft, uniforms))
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        layer.step(tokens, draft, uniforms)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        layer.step(tokens, draft, uniforms)
    run(graph.replay)
    share = torch.stack(kept).float().mean().item()
    print(f"{steps} steps of {batch} sequences with {layer.drafts} drafts: {eager:.0f} us a step, "
          f"{run(graph.replay):.0f} us replayed, {share:.2f} drafts kept of each {layer.drafts}")


if __name__ == "__main__":
    main()
