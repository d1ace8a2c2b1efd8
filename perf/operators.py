"""The decode step's operators beside the quantized GEMMs, as cases that can be timed.

Four operators, which a server of a quantized model calls in turn for every
new token:

* ``write``: new tokens' keys and values are quantized into the paged int4 or
  int8 cache (``kv_cache_write``), and read back (``kv_cache_read``), as a
  chunked prompt does with the chunk that it just wrote;
* ``read``: a sequence's cached tokens are dequantized in order;
* ``attend``: each sequence's newest token or tokens attend over its cached
  tokens (``kv_cache_attention``), optionally after a prefix which the whole
  batch shares and which is stored once;
* ``moe``: the gated mixture-of-experts layer on int4 weights for a few tokens
  (``moe_swiglu_int4``).

A case is a dict of plain values:

* cache operators: ``kv_heads``, ``head_dim``, ``bits`` (4 or 8), ``page``
  (tokens a page holds), ``dtype`` (of what goes in and comes out), and
  ``tokens`` (write, read);
* attend: ``batch``, ``queries`` (newest tokens of each sequence), ``ratio``
  (query heads a key head serves), ``length`` (cached tokens of the longest
  sequence), ``prefix`` (shared tokens), ``empty`` (one sequence has no token
  of its own);
* moe: ``tokens``, ``experts``, ``top`` (experts a token is routed to),
  ``hidden``, ``inner``, ``group`` (0: per-channel scales, else the scale
  group along K), ``layout`` (nn, nt), ``dtype``.
"""

import math
import os
import random
import sys

import torch

sys.path.insert(0, os.path.abspath("strix-halo-int4-gemms_amd"))

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# ---------------------------------------------------------------------------
# Cases


def _write(name, tokens, *, kv_heads=8, head_dim=128, bits=4, page=64, dtype="bf16", op="write"):
    case = {"op": op, "tokens": tokens, "kv_heads": kv_heads, "head_dim": head_dim, "bits": bits, "page": page,
            "dtype": dtype}
    return {"name": name, **case} if name else case


def _attend(name, batch, length, *, queries=1, ratio=4, kv_heads=8, head_dim=128, bits=4, page=64, prefix=0,
            empty=False, dtype="bf16"):
    case = {"op": "attend", "batch": batch, "length": length, "queries": queries, "ratio": ratio,
            "kv_heads": kv_heads, "head_dim": head_dim, "bits": bits, "page": page, "prefix": prefix, "empty": empty,
            "dtype": dtype}
    return {"name": name, **case} if name else case


def _moe(name, tokens, experts, top, hidden, inner, *, group=0, layout="nn", dtype="bf16"):
    case = {"op": "moe", "tokens": tokens, "experts": experts, "top": top, "hidden": hidden, "inner": inner,
            "group": group, "layout": layout, "dtype": dtype}
    return {"name": name, **case} if name else case


def listed():
    return [
        # One decode step of a batch of 16: a token of each sequence goes into
        # the int4 cache.  All launch and host time.
        _write("write_step", 16),
        # A long prompt's keys and values into the int8 cache.
        _write("write_prompt", 8191, bits=8),
        # The cached prefix of a continued conversation, dequantized for a
        # chunk of prefill.
        _write("read_long", 65536, op="read"),
        # One user, one new token, a short conversation of an odd length.
        _attend("step_one", 1, 1001),
        # A busy server's step: 32 sequences of uneven length over the int8
        # cache, one slot of the batch empty.
        _attend("step_batch", 32, 4096, bits=8, empty=True),
        # Long documents: the cache is streamed once.
        _attend("step_long", 4, 131072),
        # Five drafted tokens of each sequence are verified at once; wide
        # heads, few key heads, float16.
        _attend("step_draft", 8, 6000, queries=5, ratio=8, kv_heads=2, head_dim=256, bits=8, dtype="f16"),
        # A system prompt shared by a batch of 16, short own turns.
        _attend("prefix_short", 16, 90, prefix=2000, page=16),
        # A long document shared by 64 requests.
        _attend("prefix_long", 64, 300, prefix=65536),
        # Mixture of experts, one token through two of eight experts.
        _moe("moe_token", 1, 8, 2, 2048, 1408),
        # A batch of 16 tokens over 64 experts, group-quantized weights stored
        # output-major: most experts that are hit see one or two tokens.
        _moe("moe_batch", 16, 64, 6, 2048, 1408, group=128, layout="nt"),
        # 61 tokens over 16 large experts: all weights are streamed.
        _moe("moe_large", 61, 16, 2, 4096, 11008),
    ]


def _log(rng, lo, hi, step=1):
    """A multiple of `step` in [lo, hi], spread over the logarithm."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return min(hi // step, max(-(-lo // step), round(v / step))) * step


def draw(rng):
    op = rng.choices(["write", "read", "attend", "prefix", "moe"], [18, 10, 30, 20, 22])[0]
    head_dim, kv_heads = rng.choice([64, 128, 128, 256]), rng.choice([1, 2, 4, 8, 8, 16])
    common = {"head_dim": head_dim, "kv_heads": kv_heads, "bits": rng.choice([4, 4, 8]),
              "page": rng.choice([16, 32, 64, 64, 128]), "dtype": rng.choice(["bf16", "bf16", "f16"])}
    if op in ("write", "read"):
        most = 65536 * 8 * 128 // (kv_heads * head_dim)
        common["dtype"] = rng.choice(["bf16", "bf16", "f16", "f32"])
        return _write("", _log(rng, 1, min(65536, most)), op=op, **common)
    if op == "attend":
        # The cached values stay within the largest listed case's.
        batch, most = _log(rng, 1, 128), 4 * 131072 * 8 * 128 // (kv_heads * head_dim)
        length = _log(rng, 1, max(1, min(131072, most // batch)))
        queries = min(length, rng.choice([1, 1, 1, 1, 2, 3, 4, 8]))
        return _attend("", batch, length, queries=queries, ratio=rng.choice([1, 2, 4, 7, 8, 16]),
                       empty=batch > 1 and rng.random() < 0.3, **common)
    if op == "prefix":
        batch, ratio = _log(rng, 2, 128), rng.choice([1, 2, 4, 4, 8])
        most = 64 * 4 * 65536 * 8 * 128 // (batch * ratio * kv_heads * head_dim)
        prefix = _log(rng, 64, max(64, min(65536, most)))
        return _attend("", batch, _log(rng, 1, 2048), ratio=ratio, prefix=prefix, empty=rng.random() < 0.3, **common)
    experts = rng.choice([4, 8, 16, 32, 64])
    hidden, inner = _log(rng, 256, 4096, rng.choice([2, 32, 64])), _log(rng, 256, 11008, rng.choice([2, 32, 64]))
    while experts * hidden * inner > 16 * 4096 * 11008:
        inner = max(256, inner // 2 // 64 * 64)
    return _moe("", _log(rng, 1, 64), experts, min(experts, rng.choice([1, 2, 2, 4, 6, 8])), hidden, inner,
                group=rng.choice([0, 0, 32, 64, 128, 256]), layout=rng.choice(["nn", "nt"]),
                dtype=rng.choice(["bf16", "bf16", "f16"]))


def _lengths(case):
    """Own tokens of each sequence: the longest first, the others spread
    evenly over one to the longest, the last one empty where asked."""
    got = [case["queries"] + int((case["length"] - case["queries"]) * (1 - (i * 0.6180339887) % 1.0))
           for i in range(case["batch"])]
    if case["empty"]:
        got[-1] = 0
    return got


def _routes(case):
    """Experts of each token: `top` different ones, some asked for far more
    often than others, as a trained router leaves them."""
    rng = random.Random("%(tokens)d tokens over %(experts)d experts" % case)
    popular = [rng.expovariate(1.0) + 0.05 for _ in range(case["experts"])]
    return [sorted(range(case["experts"]), key=lambda e: rng.random() ** (1 / popular[e]), reverse=True)[:case["top"]]
            for _ in range(case["tokens"])]


# ---------------------------------------------------------------------------
# Inputs


def _codes(gen, bits, *shape):
    """Random codes as the cache and the weights hold them; int4 pairs along
    the last axis share a byte."""
    if bits == 8:
        return torch.randint(-127, 128, shape, dtype=torch.int8, device="cuda", generator=gen)
    return torch.randint(0, 256, (*shape[:-1], shape[-1] // 2), dtype=torch.uint8, device="cuda", generator=gen)


def _scales(gen, mean, *shape):
    x = torch.rand(shape, device="cuda", generator=gen)
    return ((0.5 + x) * mean).to(torch.bfloat16)


def _pool(gen, case, pages):
    """A cache of that many pages, filled: codes [pages, kv_heads, page,
    head_dim (packed)] and one scale for each row of head_dim codes."""
    bits = case["bits"]
    shape = (pages, case["kv_heads"], case["page"])
    step = 0.2 if bits == 4 else 0.013
    return {"key_codes": _codes(gen, bits, *shape, case["head_dim"]), "key_scales": _scales(gen, step, *shape),
            "value_codes": _codes(gen, bits, *shape, case["head_dim"]), "value_scales": _scales(gen, step, *shape)}


def _cache(pool):
    """The handle that a program keeps for its pool."""
    import amd_strix_halo_kernels as shk

    return shk.KVCache(**pool)


def _pages_of(tokens, page):
    return -(-tokens // page)


def _prepare_tokens(case, gen):
    tokens, page = case["tokens"], case["page"]
    pages = _pages_of(tokens, page) + 3
    order = torch.randperm(pages, device="cuda", generator=gen)
    at = torch.arange(tokens, device="cuda")
    state = {"bits": case["bits"], "dtype": DTYPES[case["dtype"]], "slots": order[at // page] * page + at % page}
    if case["op"] == "read":
        state["pool"] = _pool(gen, case, pages)
        return state
    # keys and values as the fused projection leaves them: slices of one
    # [tokens, 2 * kv_heads * head_dim] result
    both = torch.randn((tokens, 2, case["kv_heads"], case["head_dim"]), device="cuda", generator=gen)
    both[:, 0, :, : case["head_dim"] // 16] *= 6.0  # the few large channels that keys have
    both = both.to(DTYPES[case["dtype"]])
    pool = _pool(gen, case, pages)
    state.update(keys=both[:, 0], values=both[:, 1], pool={part: torch.zeros_like(v) for part, v in pool.items()})
    return state


def _prepare_attend(case, gen):
    page, lengths, batch = case["page"], _lengths(case), case["batch"]
    owned, shared = max(1, _pages_of(case["length"], page)), _pages_of(case["prefix"], page)
    pages = [_pages_of(n, page) for n in lengths]
    total = sum(pages) + shared + 1
    order = torch.randperm(total, device="cuda", generator=gen).to(torch.int32)
    pool = _pool(gen, case, total)
    table = torch.zeros((batch, owned), dtype=torch.int32, device="cuda")
    at = shared
    for i, n in enumerate(pages):
        table[i, :n] = order[at:at + n]
        if lengths[i] % page:  # what no token has been written to yet may hold anything
            for part in ("key_scales", "value_scales"):
                pool[part][order[at + n - 1].long(), :, lengths[i] % page:] = math.nan
        at += n
    heads = case["kv_heads"] * case["ratio"]
    q = 2.5 * torch.randn((batch, case["queries"], heads, case["head_dim"]), device="cuda", generator=gen)
    return {"pool": pool, "bits": case["bits"], "table": table, "prefix": case["prefix"],
            "lengths": torch.tensor(lengths, dtype=torch.int32, device="cuda"), "prefix_pages": order[:shared].clone(),
            "q": q.to(DTYPES[case["dtype"]])}


def _prepare_moe(case, gen):
    hidden, inner, experts, group = case["hidden"], case["inner"], case["experts"], case["group"]

    def weight(k, n):
        rows = (n, k) if case["layout"] == "nt" else (k // 2, 2 * n)
        codes = _codes(gen, 4, experts, *rows)
        scale = (experts, n) if not group else (experts, -(-k // group), n)
        return codes, _scales(gen, 0.2 / math.sqrt(k), *scale)

    up_gate, up_gate_scale = weight(hidden, 2 * inner)
    down, down_scale = weight(inner, hidden)
    x = torch.randn((case["tokens"], hidden), device="cuda", generator=gen)
    share = torch.rand((case["tokens"], case["top"]), device="cuda", generator=gen) + 0.1
    return {"x": x.to(DTYPES[case["dtype"]]), "up_gate": up_gate, "up_gate_scale": up_gate_scale, "down": down,
            "down_scale": down_scale, "group": group, "layout": case["layout"],
            "ids": torch.tensor(_routes(case), dtype=torch.int64, device="cuda"),
            "share": share / share.sum(dim=1, keepdim=True)}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    how = {"attend": _prepare_attend, "moe": _prepare_moe}.get(case["op"], _prepare_tokens)
    state = {"op": case["op"], **how(case, gen)}
    if own and "pool" in state:
        state["cache"] = _cache(state["pool"])  # over the same tensors
    return state


# ---------------------------------------------------------------------------
# One pass


def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(state):
    import amd_strix_halo_kernels as shk

    op = state["op"]
    if op == "write":
        shk.kv_cache_write(state["cache"], state["keys"], state["values"], state["slots"])
    if op in ("write", "read"):
        return shk.kv_cache_read(state["cache"], state["slots"], dtype=state["dtype"])
    if op == "attend":
        return shk.kv_cache_attention(state["q"], state["cache"], state["table"], state["lengths"],
                                      prefix_pages=state["prefix_pages"] if state["prefix"] else None,
                                      prefix_length=state["prefix"], return_lse=True)
    group = state["group"]
    scale = shk.ScaleSpec(shk.ScaleMode.SUBCHANNEL, group) if group else shk.ScaleSpec(shk.ScaleMode.PER_CHANNEL)
    return shk.moe_swiglu_int4(state["x"], state["up_gate"], state["down"], state["ids"], state["share"],
                               up_gate_scale=state["up_gate_scale"], down_scale=state["down_scale"], scale=scale,
                               layout=shk.GemmLayout(state["layout"]))


def _run_plain(state):
    return {"write": _plain_write, "read": _plain_read, "attend": _plain_attend, "moe": _plain_moe}[state["op"]](state)


def _pack(codes):
    codes = codes.to(torch.uint8) & 15
    return codes[..., 0::2] | (codes[..., 1::2] << 4)


def _unpack(packed):
    """int4 pairs of the last axis, as int8 in order."""
    return torch.stack(((packed << 4).view(torch.int8) >> 4, packed.view(torch.int8) >> 4), dim=-1).flatten(-2)


def _values(codes, scales, bits):
    return (_unpack(codes) if bits == 4 else codes).float() * scales.float()[..., None]


def _rows(pool, slots):
    """Pages and offsets of the slots."""
    page = pool["key_scales"].shape[2]
    return slots // page, slots % page


def _plain_write(state):
    pool, bits = state["pool"], state["bits"]
    at, offset = _rows(pool, state["slots"])
    most = 7 if bits == 4 else 127
    x = torch.stack((state["keys"], state["values"])).float()
    largest = x.abs().amax(dim=-1)
    scales = (largest / torch.full_like(largest, most)).to(torch.bfloat16)
    wide = scales.float()[..., None]
    codes = torch.where(wide > 0, torch.round(x / wide), 0.0).clamp(-most, most).nan_to_num(0.0).to(torch.int8)
    codes = _pack(codes) if bits == 4 else codes
    pool["key_codes"][at, :, offset] = codes[0]
    pool["value_codes"][at, :, offset] = codes[1]
    pool["key_scales"][at, :, offset] = scales[0]
    pool["value_scales"][at, :, offset] = scales[1]
    return _plain_read(state)


def _plain_read(state):
    pool, bits, dtype = state["pool"], state["bits"], state["dtype"]
    at, offset = _rows(pool, state["slots"])
    keys = _values(pool["key_codes"][at, :, offset], pool["key_scales"][at, :, offset], bits)
    values = _values(pool["value_codes"][at, :, offset], pool["value_scales"][at, :, offset], bits)
    return keys.to(dtype), values.to(dtype)


def _plain_tokens(codes, scales, table, bits):
    """[..., kv_heads, tokens, head_dim] of the pages of a table."""
    return _values(codes[table], scales[table], bits).transpose(-4, -3).flatten(-3, -2)


def _plain_attend(state):
    pool, bits, table, lengths = state["pool"], state["bits"], state["table"].long(), state["lengths"].long()
    batch, queries, heads, dim = state["q"].shape
    kv_heads = pool["key_scales"].shape[1]
    ratio = heads // kv_heads
    # [batch, kv_heads, queries * ratio, head_dim]
    q = state["q"].float().reshape(batch, queries, kv_heads, ratio, dim).transpose(1, 2).flatten(2, 3) / math.sqrt(dim)
    keys = _plain_tokens(pool["key_codes"], pool["key_scales"], table, bits)
    values = _plain_tokens(pool["value_codes"], pool["value_scales"], table, bits)
    at = torch.arange(keys.shape[2], device=q.device)
    held = (at < lengths[:, None])[:, None, :, None]
    keys, values = torch.where(held, keys, 0.0), torch.where(held, values, 0.0)
    # query t of the newest `queries` tokens sees what was written up to itself
    sees = lengths[:, None] - queries + 1 + torch.arange(queries, device=q.device)
    seen = (at < sees[..., None]).repeat_interleave(ratio, dim=1)[:, None]
    scores = torch.where(seen, q @ keys.transpose(-1, -2), -math.inf)
    prefix = state["prefix"]
    if prefix:
        # the shared tokens once: all sequences' rows of a head against them
        shared = state["prefix_pages"].long()
        first = _plain_tokens(pool["key_codes"], pool["key_scales"], shared, bits)[:, :prefix]
        rows = q.transpose(0, 1).flatten(1, 2)
        head = (rows @ first.transpose(-1, -2)).unflatten(1, (batch, queries * ratio)).transpose(0, 1)
        scores = torch.cat((head, scores), dim=-1)
    most = scores.amax(dim=-1, keepdim=True)
    most = torch.where(most == -math.inf, 0.0, most)
    p = torch.exp(scores - most)
    total = p.sum(dim=-1, keepdim=True)
    out = p[..., prefix:] @ values
    if prefix:
        first = _plain_tokens(pool["value_codes"], pool["value_scales"], shared, bits)[:, :prefix]
        rows = p[..., :prefix].transpose(0, 1).flatten(1, 2)
        out = out + (rows @ first).unflatten(1, (batch, queries * ratio)).transpose(0, 1)
    out = torch.where(total > 0, out / total, 0.0)
    lse = (most + torch.log(total))[..., 0]
    out = out.unflatten(2, (queries, ratio)).transpose(1, 2).flatten(2, 3)
    lse = lse.unflatten(2, (queries, ratio)).transpose(1, 2).flatten(2, 3)
    return out.to(state["q"].dtype), lse


def _plain_weight(codes, scales, k, group, layout):
    """[experts, K, N] of an int4 weight."""
    w = (_unpack(codes) if layout == "nt" else _unpack(codes.transpose(1, 2).contiguous())).transpose(1, 2).float()
    wide = scales.float()[:, None] if not group else scales.float().repeat_interleave(group, dim=1)[:, :k]
    return w * wide


def _plain_moe(state):
    x, group, layout = state["x"].float(), state["group"], state["layout"]
    experts, inner = state["up_gate"].shape[0], state["up_gate_scale"].shape[-1] // 2
    up_gate = x @ _plain_weight(state["up_gate"], state["up_gate_scale"], x.shape[1], group, layout)
    up, gate = up_gate.split(inner, dim=-1)
    h = up * (gate / (1.0 + torch.exp(-gate)))
    y = h @ _plain_weight(state["down"], state["down_scale"], inner, group, layout)
    chosen = state["ids"][..., None] == torch.arange(experts, device=x.device)
    share = (state["share"][..., None] * chosen).sum(dim=1)  # [tokens, experts]
    return (y * share.t()[..., None]).sum(dim=0).to(state["x"].dtype)


# ---------------------------------------------------------------------------
# The work of a pass, and its values in 64 bits


def work(case):
    op = case["op"]
    if op == "moe":
        tokens, hidden, inner, group = case["tokens"], case["hidden"], case["inner"], case["group"]
        used = len({e for token in _routes(case) for e in token})
        scales = 2 * (2 * inner * (-(-hidden // group) if group else 1) + hidden * (-(-inner // group) if group else 1))
        pairs = tokens * case["top"]
        return {"bytes": used * (3 * hidden * inner // 2 + scales) + 4 * tokens * hidden + 12 * pairs,
                "flops": 6 * pairs * hidden * inner}
    row = case["head_dim"] * case["bits"] // 8 + 2  # a head's codes of one token and their scale
    heads, dim = case["kv_heads"], case["head_dim"]
    if op in ("write", "read"):
        values = 2 * case["tokens"] * heads * (4 if case["dtype"] == "f32" else 2) * dim
        stored = 2 * case["tokens"] * heads * row
        # written: the values in, the rows out, and the same back again
        return {"bytes": (2 if op == "write" else 1) * (values + stored) + 8 * case["tokens"], "flops": 0}
    lengths, queries = _lengths(case), case["queries"]
    q_rows = case["batch"] * queries * case["ratio"] * heads
    cached = (sum(lengths) + case["prefix"]) * 2 * heads * row
    pairs = sum(queries * n - queries * (queries - 1) // 2 for n in lengths if n)
    pairs += case["batch"] * queries * case["prefix"]
    return {"bytes": cached + q_rows * (4 * dim + 4), "flops": 4 * pairs * heads * case["ratio"] * dim}


def exact(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    if op == "moe":
        return _exact_moe(case, _prepare_moe(case, gen))
    if op == "attend":
        return _exact_attend(case, _prepare_attend(case, gen))
    state = _prepare_tokens(case, gen)
    bits, slots, pool, page = case["bits"], state["slots"], state["pool"], case["page"]
    if op == "read":
        return tuple(_exact_rows(pool, part, slots // page, slots % page, bits) for part in ("key", "value"))

    def stored(x):
        # A row's scale is its largest magnitude over the largest code,
        # rounded to 32 bits and from there to bfloat16; a code is the value
        # over its scale, rounded to 32 bits and from there to a whole number
        # (ties to even).
        most = 7 if bits == 4 else 127
        x = x.double()
        scale = (x.abs().amax(dim=-1, keepdim=True) / most).float().bfloat16().double()
        code = (x / scale).float().double().round().clamp(-most, most)
        return torch.where(scale > 0, code, 0.0) * scale

    return stored(state["keys"]), stored(state["values"])


def _exact_rows(pool, part, at, offset, bits):
    codes, scales = pool[part + "_codes"][at, :, offset], pool[part + "_scales"][at, :, offset].double()
    if bits == 4:
        whole = codes.new_empty((*codes.shape[:-1], 2 * codes.shape[-1]), dtype=torch.float64)
        for i in range(2):
            nibble = (codes >> (4 * i)) & 15
            whole[..., i::2] = nibble.double() - 16.0 * (nibble > 7)
    else:
        whole = codes.double()
    return whole * scales[..., None]


def _exact_attend(case, state):
    """Sequence by sequence: its prefix and own tokens in a row, one softmax."""
    page, prefix, queries, bits = case["page"], case["prefix"], case["queries"], case["bits"]
    q = state["q"].double()
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    lse = torch.full(q.shape[:3], -math.inf, dtype=torch.float64, device="cuda")

    def rows(part, pages, count):
        at = torch.arange(count, device="cuda")
        return _exact_rows(state["pool"], part, pages.long()[at // page], at % page, bits)  # [count, kv_heads, dim]

    first = [rows(part, state["prefix_pages"], prefix) for part in ("key", "value")] if prefix else None
    for b, length in enumerate(_lengths(case)):
        keys, values = (rows(part, state["table"][b], length) for part in ("key", "value"))
        if prefix:
            keys, values = torch.cat((first[0], keys)), torch.cat((first[1], values))
        for t in range(queries):
            n = prefix + max(0, length - queries + t + 1)
            if n == 0:
                continue
            heads = q[b, t].view(case["kv_heads"], case["ratio"], -1)
            s = heads @ keys[:n].permute(1, 2, 0) / math.sqrt(case["head_dim"])
            lse[b, t] = torch.logsumexp(s, dim=-1).flatten()
            out[b, t] = (torch.softmax(s, dim=-1) @ values[:n].transpose(0, 1)).flatten(0, 1)
    return out, lse


def _exact_moe(case, state):
    """Expert by expert, for the tokens that ask for it."""
    group, inner = case["group"], case["inner"]
    x = state["x"].double()
    out = torch.zeros_like(x)

    def weight(name, e, k):
        packed = state[name][e] if case["layout"] == "nt" else state[name][e].t()
        nibbles = torch.stack((packed & 15, packed >> 4), dim=-1).flatten(1).double()
        w = torch.where(nibbles > 7, nibbles - 16, nibbles).t()  # [K, N]
        scale = state[name + "_scale"][e].double()
        return w * (scale.repeat_interleave(group, dim=0)[:k] if group else scale)

    ids = state["ids"]
    for e in sorted({e for token in _routes(case) for e in token}):
        share = (state["share"].double() * (ids == e)).sum(dim=1)
        rows = share.nonzero()[:, 0]
        up, gate = (x[rows] @ weight("up_gate", e, case["hidden"])).split(inner, dim=-1)
        out[rows] += share[rows, None] * ((up * gate * torch.sigmoid(gate)) @ weight("down", e, inner))
    return out
