"""The operators around a served decode step whose speed is measured here: new keys and values
rotated on their way into a paged cache of 16 bits or of 4 (MX blocks: 32 four-bit floats under a
shared power of two), attention over the 4-bit cache, and beam search's selection with the
reordering of the beams' states.

Head counts and sizes are those of the Llama-3-8B shaped layers of the benchmark (32 query heads
and 8 key-value heads of 128) and generic odd ones.  `run` calls the package's public operators
where `own` is true, and elementary torch operations where it is false.

A 4-bit page holds, for each key-value head, the codes of its tokens (head_dim / 2 bytes each, element
2 i in the low half of byte i), and behind all heads' codes the blocks' exponents (head_dim / 32 bytes
a token, heads and tokens in the same order).  A code is a sign and the magnitudes 0, 1/2, 1, 3/2, 2, 3,
4, 6; an exponent byte b stands for 2^(b - 127), 255 for NaN.  A block's exponent brings its largest
magnitude into [3.5, 7).
"""

from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda:0"
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


# ---- cases ----------------------------------------------------------------------------------


def _attention(batch: int, new: int, length: int, spread: float = 1.0, mixed: bool = False, kv_heads: int = 8,
               group: int = 4, dim: int = 128, page: int = 16, dtype: str = "bf16", window: int = 0,
               cap: float = 0.0) -> dict:
    """`batch` sequences of `length` tokens in the 4-bit cache down to `length / spread`, the last
    `new` of each (every second one a seventh of that where `mixed`) the queries."""
    return {"kind": "attention", "batch": batch, "new": new, "length": length, "spread": spread, "mixed": mixed,
            "kv_heads": kv_heads, "group": group, "dim": dim, "page": page, "dtype": dtype, "window": window,
            "cap": cap}


def _append(bits: int, batch: int, new: int, length: int, mixed: bool = False, kv_heads: int = 8, group: int = 4,
            dim: int = 128, rot: int = 128, interleaved: bool = False, page: int = 16, dtype: str = "bf16") -> dict:
    """`new` tokens (every second sequence a seventh of that where `mixed`) of sequences of up to
    `length`, the first `rot` elements of their heads rotated."""
    return {"kind": "append", "bits": bits, "batch": batch, "new": new, "length": length, "mixed": mixed,
            "kv_heads": kv_heads, "group": group, "dim": dim, "rot": rot, "interleaved": interleaved, "page": page,
            "dtype": dtype}


def _beams(batch: int, beams: int, vocab: int, history: int, ended: float = 0.0, dtype: str = "bf16") -> dict:
    """`batch` searches of `beams` beams, a share `ended` of them at their end."""
    return {"kind": "beams", "batch": batch, "beams": beams, "vocab": vocab, "history": history, "ended": ended,
            "dtype": dtype}


def listed() -> list[dict]:
    named = {
        # one sequence's next token on a short context: launch and host latency
        "fp4_attn_token": _attention(1, 1, 777),
        # a serving batch's next tokens, contexts of 2 to 32 thousand: the cache's bandwidth
        "fp4_attn_batch_long": _attention(16, 1, 32768, spread=16.0),
        # chunks of odd sizes over contexts of some thousand, a window and a cap, pages of 24 tokens,
        # 14 query heads on 2 key-value heads of 64
        "fp4_attn_chunk_window": _attention(6, 707, 5003, spread=5.0, mixed=True, kv_heads=2, group=7, dim=64,
                                            page=24, dtype="f16", window=1024, cap=30.0),
        # a whole prompt: the matrix cores
        "fp4_attn_prompt": _attention(1, 8192, 8192, page=64),
        # the next token of each sequence of a serving batch: rotated, and into one layer's cache
        "rope_append_tokens": _append(16, 64, 1, 4096),
        # chunks of prompts, a part of each head rotated in neighbouring pairs
        "rope_append_chunks": _append(16, 8, 2048, 8192, mixed=True, rot=64, interleaved=True, dtype="f16"),
        # the same into the 4-bit cache, and read back as the values that it holds
        "fp4_append_tokens": _append(4, 64, 1, 4096),
        # a whole prompt into the 4-bit cache, heads of 96, and read back
        "fp4_append_prompt": _append(4, 1, 16384, 16384, dim=96, rot=96, page=32),
        # one request's four beams
        "beams_request": _beams(1, 4, 128000, 300),
        # a batch of searches, an odd vocabulary, some beams at their end
        "beams_batch": _beams(32, 8, 100003, 500, ended=0.2),
        # wide beams, logits in 32 bits
        "beams_wide": _beams(6, 32, 32003, 200, dtype="f32"),
    }
    return [dict(c, name=name) for name, c in named.items()]


def _log(rng, lo: float, hi: float) -> int:
    return max(int(lo), min(int(hi), round(2 ** rng.uniform(math.log2(lo), math.log2(hi)))))


def draw(rng) -> dict:
    kind = rng.choices(("attention", "append", "beams"), (10, 8, 6))[0]
    if kind == "beams":
        beams, vocab = _log(rng, 1, 32), _log(rng, 1000, 160000)
        batch = max(1, min(_log(rng, 1, 64), int(2.5e7 // (beams * vocab))))
        return _beams(batch, beams, vocab, _log(rng, 1, 4096), rng.choice((0.0, 0.0, 0.3)),
                      rng.choice(("f16", "bf16", "bf16", "f32")))
    dtype = rng.choice(("f16", "bf16"))
    page = rng.choice((8, 16, 16, 24, 32, 64, 128))
    heads = rng.choice((1, 2, 4, 8))
    group = rng.choice((1, 2, 4, 4, 5, 7, 8, 16))
    dim = rng.choice((32, 64, 96, 128, 128, 128, 160, 192, 256))
    if kind == "attention":
        length = _log(rng, 1, 131072)
        new = rng.choice((1, 1, _log(rng, 1, 16), _log(rng, 1, 8192)))
        new = min(new, length)
        batch = _log(rng, 1, 64)
        # the plain form holds every score, and every key in 32 bits
        batch = max(1, min(batch, int(1e9 // (heads * group * new * length)), int(2.5e8 // (heads * dim * length))))
        new = max(1, min(new, int(1.5e9 // (batch * heads * group * length)),
                         int(0.5e12 // (4 * dim * batch * heads * group * length))))
        return _attention(batch, new, length, rng.choice((1.0, 4.0, 16.0)), rng.random() < 0.5, heads, group, dim,
                          page, dtype, rng.choice((0, 0, _log(rng, 16, 8192))), rng.choice((0.0, 0.0, 30.0)))
    bits = rng.choice((4, 16))
    if bits == 16:
        dim = rng.choice((64, 80, 96, 128, 128, 192, 256))
    rot = rng.choice((dim, dim, dim // 2, dim // 32 * 16))
    new = rng.choice((1, _log(rng, 1, 8192)))
    # as many elements as the prompt's at most
    batch = max(1, min(_log(rng, 1, 128), int(6e7 // ((group + 2) * heads * dim * new))))
    return _append(bits, batch, new, _log(rng, new, 32768), rng.random() < 0.5, heads, group, dim, max(2, rot),
                   rng.random() < 0.3, page, dtype)


# ---- inputs ---------------------------------------------------------------------------------


def _gen(seed: int) -> torch.Generator:
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    return g


def _lengths(case: dict) -> tuple[list[int], list[int]]:
    """Each sequence's tokens and, of them, its new ones."""
    n = case["batch"]
    order = [(b * 7919 + 3) % n if math.gcd(7919, n) == 1 else b for b in range(n)]
    lens = [max(1, round(case["length"] * case.get("spread", 4.0) ** (-o / max(1, n - 1)))) for o in order]
    new = [case["new"] // 7 if case["mixed"] and b % 2 else case["new"] for b in range(n)]
    return lens, [min(max(1, q), l) for q, l in zip(new, lens)]


def _ints(values, dtype=torch.int32) -> torch.Tensor:
    return torch.tensor(values, dtype=dtype, device=DEVICE)


def _offsets(counts: list[int]) -> torch.Tensor:
    total = [0]
    for c in counts:
        total.append(total[-1] + c)
    return _ints(total)


def _tables(lens: list[int], page: int, width: int, order: torch.Tensor) -> torch.Tensor:
    """Block tables [len(lens), width]: each sequence's pages out of `order`, -1 past its last."""
    held = [-(-l // page) for l in lens]
    held_t, first = _ints(held), _offsets(held)
    col = torch.arange(width, device=DEVICE)
    at = (first[:-1, None] + col).clamp(max=max(0, order.numel() - 1)).long()
    return torch.where(col < held_t[:, None], order[at].int(), -1).int()


def _randn(shape, case: dict, gen) -> torch.Tensor:
    return torch.randn(shape, device=DEVICE, generator=gen).to(DTYPES[case["dtype"]])


def _fp4_pool(planes: int, pages: int, page: int, heads: int, dim: int) -> torch.Tensor:
    """[planes, pages, page, heads, dim / 2 + dim / 32] bytes, pages 16 bytes apart or a multiple."""
    row = dim // 2 + dim // 32
    size = page * heads * row
    flat = torch.empty((planes, pages, -(-size // 16) * 16), dtype=torch.uint8, device=DEVICE)
    return flat[:, :, :size].unflatten(2, (page, heads, row))


def _prepare_attention(case: dict, gen) -> dict:
    lens, new = _lengths(case)
    page, heads, dim = case["page"], case["kv_heads"], case["dim"]
    held = [-(-l // page) for l in lens]
    pages = sum(held) + sum(held) // 8 + 1
    pool = _fp4_pool(2, pages, page, heads, dim)
    tables = _tables(lens, page, max(held), torch.randperm(pages, device=DEVICE, generator=gen))
    slot = torch.arange(max(held) * page, device=DEVICE)
    seen = torch.zeros(pages * page, dtype=torch.bool, device=DEVICE)
    at = tables.long().clamp(min=0).repeat_interleave(page, dim=1) * page + slot % page
    seen[at[slot < _ints(lens)[:, None]]] = True
    limit = 140 if case["dtype"] == "f16" else 254
    for plane in pool:
        for p0 in range(0, pages, 4096):  # keys and values are N(0, 1), rounded to blocks
            n = min(4096, pages - p0)
            x = torch.randn((n, page, heads, dim), device=DEVICE, generator=gen)
            codes, exps = _fp4_encode(x, limit)
            # what nothing has written may be anything, NaN included
            exps = torch.where(seen[p0 * page:(p0 + n) * page].view(n, page, 1, 1), exps, 255)
            flat = plane[p0:p0 + n].flatten(1)
            flat[:, :page * heads * dim // 2] = _fp4_pack(codes).transpose(1, 2).flatten(1)
            flat[:, page * heads * dim // 2:] = exps.transpose(1, 2).flatten(1).to(torch.uint8)
            plane[p0:p0 + n] = flat.view(n, page, heads, -1)
    return {"q": _randn((sum(new), heads * case["group"], dim), case, gen), "k_cache": pool[0], "v_cache": pool[1],
            "tables": tables, "lens": _ints(lens), "cu_q": _offsets(new), "max_new": max(new), "max_len": max(lens),
            "window": case["window"], "cap": case["cap"]}


def _prepare_append(case: dict, gen) -> dict:
    lens, new = _lengths(case)
    page, heads, dim, hq = case["page"], case["kv_heads"], case["dim"], case["kv_heads"] * case["group"]
    held = [-(-l // page) for l in lens]
    pages = sum(held) + 16
    tables = _tables(lens, page, max(held), torch.randperm(pages, device=DEVICE, generator=gen))
    t, n, cu = sum(new), _ints(new), _offsets(new)
    row = torch.repeat_interleave(torch.arange(len(lens), device=DEVICE), n, output_size=t)
    positions = (_ints(lens) - n)[row].long() + torch.arange(t, device=DEVICE) - cu[row]
    slots = tables[row, positions // page].long() * page + positions % page
    # queries, keys and values as they leave a fused q|k|v projection: slices of its rows
    qkv = _randn((t, (hq + 2 * heads) * dim), case, gen)
    q, k, v = (x.unflatten(1, (-1, dim)) for x in qkv.split((hq * dim, heads * dim, heads * dim), 1))
    half = case["rot"] // 2
    angle = torch.arange(max(lens), device=DEVICE, dtype=torch.float64)[:, None] * 500000.0 ** (
        -torch.arange(half, device=DEVICE, dtype=torch.float64) / half)
    rope = torch.cat([angle.cos(), angle.sin()], 1).float()
    if case["bits"] == 4:
        pool = _fp4_pool(2, pages, page, heads, dim).zero_()
    else:
        pool = torch.zeros((2, pages, page, heads, dim), dtype=DTYPES[case["dtype"]], device=DEVICE)
    return {"bits": case["bits"], "q": q, "k": k, "v": v, "pool": pool, "slots": slots, "rope": rope,
            "positions": positions, "interleaved": case["interleaved"]}


def _prepare_beams(case: dict, gen) -> dict:
    b, k, v = case["batch"], case["beams"], case["vocab"]
    x = torch.randn((b * k, v), device=DEVICE, generator=gen).mul_(2.5)
    # a model favours a few next tokens
    likely = torch.randint(0, v, (b * k, 8), device=DEVICE, generator=gen)
    x.scatter_add_(1, likely, torch.rand((b * k, 8), device=DEVICE, generator=gen) * 10)
    scores = -40 * torch.rand((b, 1), device=DEVICE, generator=gen) - 6 * torch.rand((b, k), device=DEVICE, generator=gen)
    state = {"logits": x.to(DTYPES[case["dtype"]]), "scores": scores.sort(dim=1, descending=True).values, "ended": None,
             "end_token": min(2, v - 1),
             "history": torch.randint(0, v, (b * k, case["history"]), device=DEVICE, generator=gen)}
    if case["ended"]:
        state["ended"] = torch.rand((b, k), device=DEVICE, generator=gen) < case["ended"]
    return state


def prepare(case: dict, seed: int) -> dict:
    make = {"attention": _prepare_attention, "append": _prepare_append, "beams": _prepare_beams}[case["kind"]]
    return {"kind": case["kind"], **make(case, _gen(seed))}


# ---- plain forms ----------------------------------------------------------------------------


def _fp4_encode(x: torch.Tensor, limit: int):
    """Codes 0 to 15 like x, and exponent bytes of its blocks of 32, [..., dim / 32]."""
    blocks = x.unflatten(-1, (-1, 32))
    top = blocks.abs().amax(-1)
    exps = (((top.float().view(torch.int32) + 0x200000) >> 23) - 2).clamp(0, limit)
    exps = torch.where(top.isfinite(), exps, 255)
    m = torch.ldexp(blocks, 127 - exps[..., None])
    sign, m = torch.signbit(m), m.abs()
    # halves of a step go to the even code
    code = ((m > 0.25).int() + (m >= 0.75).int() + (m > 1.25).int() + (m >= 1.75).int() + (m > 2.5).int()
            + (m >= 3.5).int() + (m > 5.0).int())
    return (code + 8 * sign.int()).flatten(-2), exps


def _fp4_pack(codes: torch.Tensor) -> torch.Tensor:
    return (codes[..., 0::2] + 16 * codes[..., 1::2]).to(torch.uint8)


def _fp4_values(packed: torch.Tensor, exps: torch.Tensor, dtype=torch.float32) -> torch.Tensor:
    steps = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=dtype, device=packed.device)
    steps = torch.cat([steps, -steps])
    codes = torch.stack([packed & 15, packed >> 4], -1).flatten(-2).int()
    scale = torch.where(exps == 255, float("nan"), torch.ldexp(torch.ones_like(exps, dtype=dtype), exps.int() - 127))
    return (steps[codes].unflatten(-1, (-1, 32)) * scale[..., None]).flatten(-2)


def _fp4_planes(cache: torch.Tensor):
    """Codes [pages, heads, page, dim / 2] and exponents [pages, heads, page, dim / 32] of a cache, as
    views where its pages lie as they do in a pool."""
    pages, page, heads, row = cache.shape
    dim = row * 32 // 17
    flat = cache.as_strided((pages, page * heads * row), (cache.stride(0), 1))
    cut = page * heads * dim // 2
    return flat[:, :cut].view(pages, heads, page, dim // 2), flat[:, cut:].view(pages, heads, page, dim // 32)


def _fp4_rows(cache: torch.Tensor, pages: torch.Tensor, rows: torch.Tensor, dtype=torch.float32) -> torch.Tensor:
    """Tokens [..., heads, dim] at rows of pages."""
    codes, exps = _fp4_planes(cache)
    return _fp4_values(codes[pages, :, rows], exps[pages, :, rows], dtype)


def _plain_attention(s: dict):
    q, k_cache, v_cache, tables, lens, cu = (s[n] for n in ("q", "k_cache", "v_cache", "tables", "lens", "cu_q"))
    t, hq, d = q.shape
    page, hkv = k_cache.shape[1], k_cache.shape[2]
    b, g, nmax, lmax = lens.numel(), hq // hkv, s["max_new"], s["max_len"]
    n = cu[1:] - cu[:-1]
    row = torch.repeat_interleave(torch.arange(b, device=q.device), n, output_size=t)
    i = torch.arange(t, device=q.device) - cu[row]
    qp = torch.zeros((b, nmax, hq, d), device=q.device)
    qp[row, i] = q.float()
    qp = qp.view(b, nmax, hkv, g, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, g * nmax, d)
    j = torch.arange(lmax, device=q.device)
    at = tables[:, j // page].long().clamp(min=0)
    there = j < lens[:, None]
    k = torch.where(there[:, :, None, None], _fp4_rows(k_cache, at, j % page), 0.0).permute(0, 2, 3, 1).contiguous()
    x = torch.matmul(qp, k).view(b, hkv, g, nmax, lmax) * (1.0 / math.sqrt(d))
    del k
    if s["cap"]:
        x = s["cap"] * torch.tanh(x / s["cap"])
    p = (lens - n)[:, None] + torch.arange(nmax, device=q.device)
    seen = there[:, None, :] & (j <= p[:, :, None])
    if s["window"]:
        seen = seen & (j > p[:, :, None] - s["window"])
    x = torch.where(seen[:, None, None], x, float("-inf"))
    m = x.amax(-1, keepdim=True).clamp(min=-3.0e38)
    x = torch.exp(x - m)
    z = x.sum(-1, keepdim=True)
    v = torch.where(there[:, :, None, None], _fp4_rows(v_cache, at, j % page), 0.0).permute(0, 2, 1, 3).contiguous()
    o = torch.matmul(x.view(b, hkv, g * nmax, lmax), v).view(b, hkv, g, nmax, d)
    o = torch.where(z > 0, o / z, 0.0)
    lse = (m + torch.log(z)).squeeze(-1)
    o = o.permute(0, 3, 1, 2, 4).reshape(b, nmax, hq, d)[row, i]
    return o.to(q.dtype), lse.permute(0, 3, 1, 2).reshape(b, nmax, hq)[row, i]


def _rotate(x: torch.Tensor, rope: torch.Tensor, positions: torch.Tensor, interleaved: bool) -> torch.Tensor:
    """In 64 bits: a block's exponent and codes are next to borders."""
    half = rope.shape[1] // 2
    c, s = rope.double()[positions][:, None].split(half, -1)
    y = x.double()
    if interleaved:
        a, b = y[..., 0:2 * half:2], y[..., 1:2 * half:2]
        turned = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    else:
        a, b = y[..., :half], y[..., half:2 * half]
        turned = torch.cat([a * c - b * s, b * c + a * s], -1)
    return torch.cat([turned, y[..., 2 * half:]], -1)


def _plain_append(s: dict):
    q, k, v, pool, slots = (s[n] for n in ("q", "k", "v", "pool", "slots"))
    q_out = _rotate(q, s["rope"], s["positions"], s["interleaved"]).float().to(q.dtype)
    k = _rotate(k, s["rope"], s["positions"], s["interleaved"]).float()
    page = pool.shape[2]
    if s["bits"] == 16:
        pool[0, slots // page, slots % page] = k.to(q.dtype)
        pool[1, slots // page, slots % page] = v
        return q_out, pool
    held = []
    for plane, x in zip(pool, (k, v)):
        codes, exps = _fp4_planes(plane)
        c, e = _fp4_encode(x.float(), 140 if q.dtype == torch.float16 else 254)
        codes[slots // page, :, slots % page] = _fp4_pack(c)
        exps[slots // page, :, slots % page] = e.to(torch.uint8)
        held.append(_fp4_rows(plane, slots // page, slots % page).to(q.dtype))
    return q_out, *held


def _plain_beams(s: dict):
    logits, scores, ended = s["logits"], s["scores"], s["ended"]
    (b, k), v = scores.shape, logits.shape[1]
    x = logits.float()
    m = x.amax(1, keepdim=True).double()
    lse = m + torch.log(torch.exp(x.double() - m).sum(1, keepdim=True))
    # each beam's k best: one whole number for each token, its logit in an order of whole numbers, then
    # the lower index
    index = torch.arange(v, device=x.device)
    bits = (x + 0.0).view(torch.int32)
    best = torch.topk((bits ^ ((bits >> 31) & 0x7FFFFFFF)).long() * (1 << 32) + (v - 1 - index), min(k, v), dim=1).values
    ids = v - 1 - (best & 0xFFFFFFFF)
    total = scores.double().view(-1, 1) + (x.gather(1, ids).double() - lse)
    order = total  # between the beams: the greater total, then the lower beam
    if ended is not None:
        done, first = ended.view(-1, 1), torch.arange(ids.shape[1], device=x.device) == 0
        total = torch.where(done & first, scores.double().view(-1, 1), total)
        ids = torch.where(done, s["end_token"], ids)
        order = torch.where(done & ~first, float("-inf"), total)
    pick = torch.sort(order.view(b, -1), dim=1, descending=True, stable=True).indices[:, :k]
    rows = torch.arange(b, device=x.device)[:, None] * k + pick // ids.shape[1]
    tokens = ids.view(b, -1).gather(1, pick)
    out = [total.view(b, -1).gather(1, pick).float(), rows.int(), tokens]
    if ended is not None:
        out.append(ended.view(-1)[rows] | (tokens == s["end_token"]))
    return [*out, s["history"][rows.view(-1)]]


# ---- one pass -------------------------------------------------------------------------------


def run(state: dict):
    kind, s = state["kind"], state
    if not own:
        return {"attention": _plain_attention, "append": _plain_append, "beams": _plain_beams}[kind](s)
    from pulsar_amd import ops

    if kind == "attention":
        return ops.paged_attention_fp4(s["q"], s["k_cache"], s["v_cache"], s["tables"], s["lens"], s["cu_q"],
                                       s["max_new"], s["max_len"], window=s["window"], softcap=s["cap"],
                                       return_lse=True)
    if kind == "append":
        pool, how = s["pool"], {"rope": s["rope"], "positions": s["positions"], "interleaved": s["interleaved"]}
        if s["bits"] == 16:
            return ops.paged_cache_append(s["q"], s["k"], s["v"], pool[0], pool[1], s["slots"], **how), pool
        q = ops.paged_cache_append_fp4(s["q"], s["k"], s["v"], pool[0], pool[1], s["slots"], **how)
        return q, *ops.paged_cache_read_fp4(pool[0], pool[1], s["slots"], s["q"].dtype)
    picked = ops.beam_select(s["logits"], s["scores"], ended=s["ended"], end_token=s["end_token"])
    return [*picked, *ops.beam_reorder([s["history"]], picked[1])]


# ---- what a pass cannot do without ------------------------------------------------------------


def _visible(length: int, new: int, window: int) -> int:
    """(query, key) pairs of one head."""
    if not window or window >= length:
        return new * length - new * (new - 1) // 2
    short = max(0, min(new, window - 1 - (length - new)))  # queries that see fewer than `window` keys
    first = length - new + 1
    return short * first + short * (short - 1) // 2 + (new - short) * window


def work(case: dict) -> dict:
    kind = case["kind"]
    if kind == "beams":
        rows, v = case["batch"] * case["beams"], case["vocab"]
        live = rows * (1.0 - case["ended"])
        size = 4 if case["dtype"] == "f32" else 2
        return {"bytes": int(live * v * size) + rows * (4 + 4 + 4 + 8 + 16 * case["history"]), "flops": int(4 * live * v)}
    heads, dim, page = case["kv_heads"], case["dim"], case["page"]
    lens, new = _lengths(case)
    hq, t = heads * case["group"], sum(new)
    token = heads * (dim // 2 + dim // 32)  # bytes of a 4-bit key, or value, of every head
    if kind == "attention":
        keys = sum(min(l, case["window"] + q - 1) if case["window"] else l for l, q in zip(lens, new))
        return {"bytes": t * hq * (4 * dim + 4) + 2 * keys * token + 4 * -(-keys // page),
                "flops": 4 * dim * hq * sum(_visible(l, q, case["window"]) for l, q in zip(lens, new))}
    moved = 4 * hq * dim + 4 * heads * dim + 4 * case["rot"] + 16  # q in and out, k and v in, angles
    # stored and, of 4 bits, read back
    moved += 4 * heads * dim if case["bits"] == 16 else 4 * token + 4 * heads * dim + 8
    return {"bytes": t * moved, "flops": 3 * t * (hq + heads) * case["rot"]}


# ---- the definitions, in 64 bits ----------------------------------------------------------------


def _turn(x: torch.Tensor, s: dict) -> torch.Tensor:
    """Each pair as a complex number, times e^(i angle)."""
    rot = s["rope"].shape[1]
    angle = s["rope"].double()[s["positions"]]
    e = torch.complex(angle[:, :rot // 2], angle[:, rot // 2:])[:, None]
    pairs = x[..., :rot].double()
    pairs = pairs.unflatten(-1, (rot // 2, 2)) if s["interleaved"] else pairs.unflatten(-1, (2, rot // 2)).transpose(-1, -2)
    turned = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * e)
    turned = turned if s["interleaved"] else turned.transpose(-1, -2)
    return torch.cat([turned.flatten(-2), x[..., rot:].double()], -1)


def _nearest(x: torch.Tensor, limit: int) -> torch.Tensor:
    """The values that blocks of 32 round to: the grid's nearest, of two the one of an even code."""
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device=x.device)
    blocks = x.unflatten(-1, (-1, 32))
    mant, exp = torch.frexp(blocks.abs().amax(-1, keepdim=True))  # in [1/2, 1)
    unit = torch.ldexp(torch.ones_like(mant), (exp - 3 + (mant >= 0.875).int()).clamp(-127, limit))
    m = (blocks / unit).abs()
    below = (torch.bucketize(m, grid, right=True) - 1).clamp(0, 6)
    lo, hi = grid[below], grid[below + 1]
    up = (m - lo > hi - m) | ((m - lo == hi - m) & (below % 2 == 1))
    return (torch.where(up, hi, lo) * unit * torch.sign(blocks)).flatten(-2)


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    if case["kind"] == "append":
        q, k, v = _turn(s["q"], s), _turn(s["k"], s), s["v"].double()
        if case["bits"] == 4:
            limit = 13 if case["dtype"] == "f16" else 127
            return q, _nearest(k, limit), _nearest(v, limit)
        pool, page = s["pool"].double(), case["page"]
        pool[0, s["slots"] // page, s["slots"] % page] = k
        pool[1, s["slots"] // page, s["slots"] % page] = v
        return q, pool
    if case["kind"] == "beams":
        b, k, v = case["batch"], case["beams"], case["vocab"]
        found = []
        for i in range(b):
            x = torch.log_softmax(s["logits"][i * k:(i + 1) * k].double(), 1) + s["scores"][i].double()[:, None]
            if s["ended"] is not None:
                x[s["ended"][i]] = float("-inf")
                x[s["ended"][i], s["end_token"]] = s["scores"][i][s["ended"][i]].double()
            found.append(x.view(-1).topk(k).values)
        return [torch.stack(found), None, None, *([] if s["ended"] is None else [None]), None]
    lens, new = _lengths(case)
    g, dim, page = case["group"], case["dim"], case["page"]
    outs, lses, at = [], [], 0
    for b, (length, n) in enumerate(zip(lens, new)):
        pos = torch.arange(length, device=DEVICE)
        pages = s["tables"][b].long()[pos // page]
        p = torch.arange(length - n, length, device=DEVICE)
        seen = pos[None, :] <= p[:, None]
        if case["window"]:
            seen &= pos[None, :] > p[:, None] - case["window"]
        out = torch.empty((n, case["kv_heads"] * g, dim), dtype=torch.float64, device=DEVICE)
        lse = torch.empty((n, case["kv_heads"] * g), dtype=torch.float64, device=DEVICE)
        keys, values = (_fp4_rows(s[c], pages, pos % page, torch.float64) for c in ("k_cache", "v_cache"))
        for h in range(case["kv_heads"] * g):
            k, v = keys[:, h // g], values[:, h // g]
            for r in range(0, n, 2048):
                x = s["q"][at + r:at + min(n, r + 2048), h].double() @ k.t().contiguous() / math.sqrt(dim)
                if case["cap"]:
                    x = case["cap"] * torch.tanh(x / case["cap"])
                x.masked_fill_(~seen[r:r + 2048], float("-inf"))
                lse[r:r + 2048, h] = torch.logsumexp(x, 1)
                out[r:r + 2048, h] = torch.softmax(x, 1) @ v
        outs.append(out)
        lses.append(lse)
        at += n
    return torch.cat(outs), torch.cat(lses)
