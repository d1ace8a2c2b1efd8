"""Plain definitions of what a step needs around its cached attention: head
norms and rotation in float64, the pages of a step and the verification of drafts
in whole and exact numbers."""

from __future__ import annotations

from fractions import Fraction

import torch


def rotated(x, weight, eps, positions, frequencies, amplitude, interleaved, dtype):
    """(out, bound) for x [tokens, heads, dim], CPU.

    What the bound counts, in units of 2^-24 of each value: the sum of squares
    (eight fused adds, five across lanes, halved by the root), its division, the
    root and the reciprocal make at most 12; the two products with scale and
    weight 2; cosine and sine 6 (the angle's rounding, a series of five terms,
    the amplitude) and what 64 bits lose of the angle; the product and the sum of
    the rotation 3.  The result is rounded once, f16 also below its normal range.
    """
    x = x.double()
    dim, n = x.shape[-1], 2 * len(frequencies)
    if weight is not None:
        x = x / torch.sqrt(x.square().mean(dim=-1, keepdim=True) + eps) * weight.double()
    angle = positions.double()[:, None, None] * torch.tensor(frequencies, dtype=torch.float64)
    cos, sin = amplitude * torch.cos(angle), amplitude * torch.sin(angle)
    first, second = (slice(0, n, 2), slice(1, n, 2)) if interleaved else (slice(0, n // 2), slice(n // 2, n))
    a, b = x[..., first], x[..., second]
    out, off = x.clone(), 14 * 2.0**-24 * x.abs()
    out[..., first], out[..., second] = a * cos - b * sin, b * cos + a * sin
    if n:
        size = (a.abs() + b.abs()) * abs(amplitude) * (23 * 2.0**-24 + angle.abs() * 2.0**-51)
        off[..., first], off[..., second] = size, size
    bound = off + torch.finfo(dtype).eps / 2 * out.abs() + (2.0**-25 if dtype == torch.float16 else 2.0**-126)
    return out, bound


def step(state, new, capacity, page):
    """One step of the pages on Python lists.  state: page_table, lengths, owned,
    free (a list, the top last).  Returns slots, positions, sequences, starts, taken."""
    table, lengths, owned, free = state["page_table"], state["lengths"], state["owned"], state["free"]
    batch, width = len(lengths), len(table[0])
    for b in range(batch):
        if new[b] < 0:
            free.extend(table[b][:owned[b]])
            lengths[b] = owned[b] = 0
    starts, slots, positions, sequences, taken = [0], [], [], [], []
    asked, there = 0, len(free)
    for b in range(batch):
        count = max(0, new[b])
        starts.append(starts[-1] + count)
        total = -(-(lengths[b] + count) // page)
        fits = new[b] >= 0 and total <= width and starts[-1] <= capacity
        need = max(0, total - owned[b]) if fits else 0
        asked += need
        fits = fits and (need == 0 or asked <= there)
        if fits:
            for _ in range(need):
                table[b][owned[b]] = free.pop()
                owned[b] += 1
        for i in range(count):
            at = lengths[b] + i
            slots.append(table[b][at // page] * page + at % page if fits else -1)
            positions.append(at)
            sequences.append(b)
        taken.append(count if fits else 0)
        if fits:
            lengths[b] += count
    pad = max(0, capacity - len(slots))
    return ((slots + [-1] * pad)[:capacity], (positions + [0] * pad)[:capacity], (sequences + [-1] * pad)[:capacity],
            starts, taken)


def verified(target, draft, tokens, uniforms, count):
    """(out, kept) of one sequence in exact fractions; lists, draft None or [drafts][vocab]."""
    drafts = len(tokens)
    kept = 0
    exact = [Fraction(u) for u in uniforms]
    good = lambda v: Fraction(v) if v == v and v > 0 else Fraction(0)  # noqa: E731
    while kept < count:
        t = tokens[kept]
        if not 0 <= t < len(target[0]):
            break
        p, q = target[kept][t], 1.0 if draft is None else draft[kept][t]
        if not (p == p and q == q and exact[kept] * Fraction(q) < Fraction(p)):
            break
        kept += 1
    row = [good(v) for v in target[kept]]
    weights = row
    if kept < count:
        if draft is None:
            weights = [Fraction(0) if t == tokens[kept] else w for t, w in enumerate(row)]
        else:
            weights = [max(w - Fraction(q), Fraction(0)) if q == q else Fraction(0) for w, q in zip(row, draft[kept])]
        if not sum(weights):
            weights = row
    share, run, token = exact[-1] * sum(weights), Fraction(0), -1
    for t, w in enumerate(weights):
        run += w
        if run > share:
            token = t
            break
    return tokens[:kept] + [token] + [-1] * (drafts - kept), kept


def half_turns(n):
    """Frequencies of n pairs from fast to slow."""
    return [10000.0 ** (-i / max(1, n)) for i in range(n)]
