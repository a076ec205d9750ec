"""The paged-cache and log-probability operators whose speed is measured: attention of new tokens
over a paged cache, the cache's book-keeping (taking pages, storing tokens, forking, freeing,
compacting and copying), and log probabilities of given tokens.

Head counts and sizes are those of the Llama-3-8B shaped layers of the benchmark (32 query heads
and 8 key-value heads of 128) and generic odd ones.  `run` calls the package's public operators
where `own` is true, and elementary torch operations in 32 bits where it is false.  Keys and values
are N(0, 1); the cache's unused slots hold NaN for the attention, as memory that nothing has
written may.
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
    """`batch` sequences of `length` tokens in the cache down to `length / spread`, the last `new`
    of each (every second one a seventh of that where `mixed`) the queries."""
    return {"kind": "attention", "batch": batch, "new": new, "length": length, "spread": spread, "mixed": mixed,
            "kv_heads": kv_heads, "group": group, "dim": dim, "page": page, "dtype": dtype, "window": window,
            "cap": cap}


def _append(batch: int, new: int, length: int, spread: float = 1.0, mixed: bool = False, kv_heads: int = 8,
            dim: int = 128, page: int = 16, dtype: str = "bf16") -> dict:
    return {"kind": "append", "batch": batch, "new": new, "length": length, "spread": spread, "mixed": mixed,
            "kv_heads": kv_heads, "dim": dim, "page": page, "dtype": dtype}


def _branch(batch: int, length: int, spread: float = 4.0, layers: int = 8, kv_heads: int = 8, dim: int = 128,
            page: int = 16, dtype: str = "bf16") -> dict:
    return {"kind": "branch", "batch": batch, "length": length, "spread": spread, "layers": layers,
            "kv_heads": kv_heads, "dim": dim, "page": page, "dtype": dtype}


def _compact(pages: int, used: int, copied: int, batch: int, layers: int = 8, kv_heads: int = 8, dim: int = 128,
             page: int = 16, dtype: str = "bf16") -> dict:
    return {"kind": "compact", "pages": pages, "used": used, "copied": copied, "batch": batch, "layers": layers,
            "kv_heads": kv_heads, "dim": dim, "page": page, "dtype": dtype}


def _logprobs(tokens: int, vocab: int, top: int, dtype: str = "bf16") -> dict:
    return {"kind": "logprobs", "tokens": tokens, "vocab": vocab, "top": top, "dtype": dtype}


def listed() -> list[dict]:
    named = {
        # one sequence's next token on a short context: launch and host latency
        "attn_token": _attention(1, 1, 777),
        # a serving batch's next tokens, contexts of 2 to 32 thousand: the cache's bandwidth
        "attn_batch_long": _attention(16, 1, 32768, spread=16.0),
        # chunks of odd sizes over contexts of some thousand, a window and a cap, pages of 24 tokens,
        # 14 query heads on 2 key-value heads of 64
        "attn_chunk_window": _attention(6, 707, 5003, spread=5.0, mixed=True, kv_heads=2, group=7, dim=64, page=24,
                                        dtype="f16", window=1024, cap=30.0),
        # a whole prompt: the matrix cores
        "attn_prompt": _attention(1, 8192, 8192, page=64),
        # the next token of each sequence of a serving batch enters the cache of one layer
        "append_tokens": _append(64, 1, 4096, spread=16.0),
        # chunks of prompts enter the cache
        "append_chunks": _append(8, 2048, 8192, spread=3.0, mixed=True, dtype="f16"),
        # two beams branch: their sequences fork, the old ones go
        "branch_beams": _branch(2, 500),
        # every sequence of a batch branches, 16 layers
        "branch_batch": _branch(48, 2000, layers=16, page=64),
        # a small pool's holes are closed, and a prefix of eight pages is copied
        "compact_small": _compact(512, 300, 8, 5, layers=2),
        # a half-used pool's holes are closed, and a prefix of some pages is copied
        "compact_pool": _compact(4096, 2050, 64, 33, layers=4, page=32),
        # the next tokens of a few sequences, with five alternatives
        "logprobs_step": _logprobs(8, 128000, 5),
        # a prompt's tokens, odd vocabulary, twenty alternatives
        "logprobs_prompt": _logprobs(2048, 100003, 20),
    }
    return [dict(c, name=name) for name, c in named.items()]


def _log(rng, lo: float, hi: float) -> int:
    return max(int(lo), min(int(hi), round(2 ** rng.uniform(math.log2(lo), math.log2(hi)))))


def draw(rng) -> dict:
    kind = rng.choices(("attention", "append", "branch", "compact", "logprobs"), (10, 3, 3, 3, 4))[0]
    dtype = rng.choice(("f16", "bf16"))
    page = rng.choice((8, 16, 16, 24, 32, 64, 128))
    heads = rng.choice((1, 2, 4, 8))
    dim = rng.choice((64, 80, 96, 128, 128, 128, 192, 256))
    if kind == "attention":
        group = rng.choice((1, 2, 4, 4, 5, 7, 8, 16))
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
    if kind == "append":
        new = rng.choice((1, _log(rng, 1, 8192)))
        batch = max(1, min(_log(rng, 1, 128), 16384 // new))
        return _append(batch, new, _log(rng, new, 32768), rng.choice((1.0, 4.0)), rng.random() < 0.5, heads, dim,
                       page, dtype)
    if kind == "branch":
        length, layers = _log(rng, 1, 4096), _log(rng, 1, 16)
        token = 2 * layers * heads * dim * 2
        batch = max(1, min(_log(rng, 1, 64), int(1.5e9 // (token * (length + page)))))
        return _branch(batch, length, rng.choice((1.0, 4.0)), layers, heads, dim, page, dtype)
    if kind == "compact":
        layers = _log(rng, 1, 8)
        most = int(1e9 // (2 * layers * heads * dim * page * 2))
        pages = min(_log(rng, 64, 8192), max(64, most))
        used = max(1, min(pages // 2, round(pages * rng.uniform(0.05, 0.5))))
        return _compact(pages, used, rng.randint(1, min(used, pages // 8)), _log(rng, 1, min(64, used)), layers,
                        heads, dim, page, dtype)
    vocab = _log(rng, 1000, 160000)
    tokens = max(1, min(_log(rng, 1, 4096), int(2e8 // vocab)))
    return _logprobs(tokens, vocab, rng.choice((0, 1, 5, 20, 32)), rng.choice(("f16", "bf16", "bf16", "f32")))


# ---- inputs ---------------------------------------------------------------------------------


def _gen(seed: int) -> torch.Generator:
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    return g


def _lengths(case: dict) -> tuple[list[int], list[int]]:
    """Each sequence's tokens in the cache and, of them, its new ones."""
    n = case["batch"]
    order = [(b * 7919 + 3) % n if math.gcd(7919, n) == 1 else b for b in range(n)]
    lens = [max(1, round(case["length"] * case["spread"] ** (-o / max(1, n - 1)))) for o in order]
    new = [case.get("new", 0) // 7 if case.get("mixed") and b % 2 else case.get("new", 0) for b in range(n)]
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


def _prepare_attention(case: dict, gen) -> dict:
    lens, new = _lengths(case)
    page, heads, dim = case["page"], case["kv_heads"], case["dim"]
    held = [-(-l // page) for l in lens]
    pages = sum(held) + sum(held) // 8 + 1
    pool = torch.empty((2, pages, page, heads, dim), dtype=DTYPES[case["dtype"]], device=DEVICE)
    pool.normal_(generator=gen)
    tables = _tables(lens, page, max(held), torch.randperm(pages, device=DEVICE, generator=gen))
    slot = torch.arange(max(held) * page, device=DEVICE)
    seen = torch.zeros(pages * page, dtype=torch.bool, device=DEVICE)
    at = tables.long().clamp(min=0).repeat_interleave(page, dim=1) * page + slot % page
    seen[at[slot < _ints(lens)[:, None]]] = True
    pool.view(2, pages * page, heads, dim)[:, ~seen] = float("nan")
    return {"q": _randn((sum(new), heads * case["group"], dim), case, gen), "k_cache": pool[0], "v_cache": pool[1],
            "tables": tables, "lens": _ints(lens), "cu_q": _offsets(new), "max_new": max(new), "max_len": max(lens),
            "window": case["window"], "cap": case["cap"]}


def _meta(refs: torch.Tensor, tables: torch.Tensor, lens: torch.Tensor) -> dict:
    """The book-keeping of a pool in one buffer, and a second one that each pass works on."""
    flat = torch.cat([refs.reshape(-1), tables.reshape(-1), lens.reshape(-1)]).int()
    work = torch.empty_like(flat)
    r, t = refs.numel(), tables.numel()
    return {"given": flat, "work": work, "refs": work[:r], "tables": work[r:r + t].view(tables.shape),
            "lens": work[r + t:]}


def _refs_of(tables: torch.Tensor, pages: int) -> torch.Tensor:
    refs = torch.zeros(pages + 1, dtype=torch.int32, device=DEVICE)
    at = torch.where(tables >= 0, tables, pages).long().reshape(-1)
    refs.scatter_add_(0, at, torch.ones_like(at, dtype=torch.int32))
    return refs[:pages]


def _prepare_append(case: dict, gen) -> dict:
    lens, new = _lengths(case)
    before = [l - q for l, q in zip(lens, new)]
    page, heads, dim = case["page"], case["kv_heads"], case["dim"]
    held = [-(-l // page) for l in lens]
    pages = sum(held) + 16
    tables = _tables(before, page, max(held), torch.randperm(pages, device=DEVICE, generator=gen))
    pool = torch.zeros((2, pages, page, heads, dim), dtype=DTYPES[case["dtype"]], device=DEVICE)
    # keys and values as they leave a fused q|k|v projection: slices of its rows
    kv = _randn((sum(new), 2 * heads * dim), case, gen)
    return {"k": kv[:, :heads * dim].view(-1, heads, dim), "v": kv[:, heads * dim:].view(-1, heads, dim),
            "pool": pool, "meta": _meta(_refs_of(tables, pages), tables, _ints(before)), "cu_q": _offsets(new),
            "tokens": sum(new), "page": page}


def _prepare_branch(case: dict, gen) -> dict:
    lens, _ = _lengths(case)
    page, n = case["page"], case["batch"]
    held = [-(-l // page) for l in lens]
    pages = sum(held) + n + 16
    tables = _tables(lens, page, max(held), torch.randperm(pages, device=DEVICE, generator=gen))
    refs = _refs_of(tables, pages)
    tables = torch.cat([tables, torch.full_like(tables, -1)])
    pool = _randn((2 * case["layers"], pages, page, case["kv_heads"], case["dim"]), case, gen)
    # beams: each new one continues one of the old ones, the better half of them twice as often
    pick = torch.randint(0, max(1, n), (n,), device=DEVICE, generator=gen) // 2 if n > 2 else torch.zeros(n, device=DEVICE)
    return {"pool": pool, "meta": _meta(refs, tables, _ints(lens + [0] * n)), "src": pick.int(),
            "dst": torch.arange(n, 2 * n, dtype=torch.int32, device=DEVICE),
            "old": torch.arange(n, dtype=torch.int32, device=DEVICE), "page": page}


def _prepare_compact(case: dict, gen) -> dict:
    page, used, n = case["page"], case["used"], case["batch"]
    spare = case["copied"]
    each = [used // n + (b < used % n) for b in range(n)]
    order = torch.randperm(case["pages"] - spare, device=DEVICE, generator=gen)[:used]
    tables = _tables([e * page for e in each], page, max(each), order)
    pool = _randn((2 * case["layers"], case["pages"], page, case["kv_heads"], case["dim"]), case, gen)
    # a prefix is copied into pages that the pool keeps back
    return {"pool": pool, "meta": _meta(_refs_of(tables, case["pages"]), tables, _ints([e * page for e in each])),
            "src": torch.arange(spare, dtype=torch.int32, device=DEVICE),
            "dst": torch.arange(case["pages"] - spare, case["pages"], dtype=torch.int32, device=DEVICE)}


def _prepare_logprobs(case: dict, gen) -> dict:
    t, v = case["tokens"], case["vocab"]
    x = torch.randn((t, v), device=DEVICE, generator=gen).mul_(2.5)
    given = torch.randint(0, v, (t,), device=DEVICE, generator=gen)
    # a token that was sampled or read in a prompt mostly is a likely one
    likely = torch.rand((t, 1), device=DEVICE, generator=gen) * 14
    x.scatter_add_(1, given[:, None], likely)
    return {"logits": x.to(DTYPES[case["dtype"]]), "targets": given, "top": case["top"]}


def prepare(case: dict, seed: int) -> dict:
    make = {"attention": _prepare_attention, "append": _prepare_append, "branch": _prepare_branch,
            "compact": _prepare_compact, "logprobs": _prepare_logprobs}[case["kind"]]
    return {"kind": case["kind"], **make(case, _gen(seed))}


# ---- plain forms ----------------------------------------------------------------------------


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
    k = torch.where(there[:, :, None, None], k_cache[at, j % page].float(), 0.0).permute(0, 2, 3, 1).contiguous()
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
    v = torch.where(there[:, :, None, None], v_cache[at, j % page].float(), 0.0).permute(0, 2, 1, 3).contiguous()
    o = torch.matmul(x.view(b, hkv, g * nmax, lmax), v).view(b, hkv, g, nmax, d)
    o = torch.where(z > 0, o / z, 0.0)
    lse = (m + torch.log(z)).squeeze(-1)
    o = o.permute(0, 3, 1, 2, 4).reshape(b, nmax, hq, d)[row, i]
    return o.to(q.dtype), lse.permute(0, 3, 1, 2).reshape(b, nmax, hq)[row, i]


def _plain_extend(refs, tables, lens, cu, tokens: int, page: int):
    """Pages for the new tokens, in place, and the tokens' slots."""
    b, width = tables.shape
    n = cu[1:] - cu[:-1]
    have = (lens + page - 1) // page
    want = (lens + n + page - 1) // page
    need = want - have
    free = torch.sort(refs != 0, stable=True)  # the free pages first, lowest ahead
    missing = torch.clamp(need.sum() - (refs == 0).sum(), min=0) + torch.clamp(want - width, min=0).sum()
    ok = missing == 0
    col = torch.arange(width, device=refs.device)
    new = ok & (col >= have[:, None]) & (col < want[:, None])
    number = (torch.cumsum(need, 0) - need - have)[:, None] + col
    tables.copy_(torch.where(new, free.indices[number.clamp(0, refs.numel() - 1)], tables))
    count = torch.where(new, 1, 0).int()
    refs.scatter_add_(0, torch.where(new, tables, 0).long().reshape(-1), count.reshape(-1))
    row = torch.repeat_interleave(torch.arange(b, device=refs.device), n, output_size=tokens)
    at = lens[row] + torch.arange(tokens, device=refs.device) - cu[row]
    slots = tables[row, (at // page).clamp(max=width - 1).long()].long() * page + at % page
    lens.add_(torch.where(ok, n, 0))
    return torch.where(ok, slots, -1), missing.reshape(1).int()


def _plain_fork(pool, refs, tables, lens, src, dst):
    page = pool.shape[2]
    length = lens[src.long()]
    full, part = length // page, length % page != 0
    free = torch.sort(refs != 0, stable=True)
    missing = torch.clamp(part.sum() - (refs == 0).sum(), min=0)
    ok = missing == 0
    fresh = free.indices[(torch.cumsum(part, 0) - 1).clamp(0, refs.numel() - 1)]
    part = part & ok
    col = torch.arange(tables.shape[1], device=refs.device)
    old = tables[src.long()]
    shared, split = col < full[:, None], (col == full[:, None]) & part[:, None]
    tables[dst.long()] = torch.where(ok, torch.where(shared, old, torch.where(split, fresh[:, None].int(), -1)),
                                     tables[dst.long()])
    lens[dst.long()] = torch.where(ok, length, lens[dst.long()])
    refs.scatter_add_(0, torch.where(shared, old, 0).long().reshape(-1), (shared & ok).int().reshape(-1))
    refs.scatter_add_(0, torch.where(part, fresh, 0), part.int())
    last = old.gather(1, full[:, None].clamp(max=tables.shape[1] - 1).long())[:, 0].long()
    pool[:, fresh[part]] = pool[:, last[part]]
    return missing.reshape(1).int()


def _plain_free(refs, tables, lens, rows):
    old = tables[rows.long()]
    refs.scatter_add_(0, old.clamp(min=0).long().reshape(-1), -(old >= 0).int().reshape(-1))
    tables[rows.long()] = -1
    lens[rows.long()] = 0


def _plain_compact(pool, refs, tables):
    index = torch.arange(refs.numel(), device=refs.device)
    count = (refs > 0).sum()
    hole = index[(refs == 0) & (index < count)]
    high = index[(refs > 0) & (index >= count)]
    pool[:, hole] = pool[:, high]
    refs[hole] = refs[high]
    refs[high] = 0
    index[high] = hole
    tables.copy_(torch.where(tables >= 0, index[tables.clamp(min=0).long()], tables))
    return count.reshape(1).int()


def _plain_logprobs(logits, targets, top: int):
    x = logits.float()
    v = x.shape[1]
    m = x.amax(1, keepdim=True)
    e = torch.exp(x - m)
    z = e.sum(1)
    given = x.gather(1, targets[:, None])
    lse = m[:, 0] + torch.log(z)
    entropy = torch.log(z) - (e * (x - m)).sum(1) / z
    index = torch.arange(v, device=x.device)
    rank = ((x > given) | ((x == given) & (index < targets[:, None]))).sum(1)
    # one whole number for each token: its logit in an order of whole numbers, then the lower index
    bits = (x + 0.0).view(torch.int32)
    key = (bits ^ ((bits >> 31) & 0x7FFFFFFF)).long() * (1 << 32) + (v - 1 - index)
    best = torch.topk(key, top, dim=1).values if top else key[:, :0]
    ids = v - 1 - (best & 0xFFFFFFFF)
    return given[:, 0] - lse, rank, entropy, x.gather(1, ids) - lse[:, None], ids


# ---- one pass -------------------------------------------------------------------------------


def run(state: dict):
    kind, s = state["kind"], state
    if own:
        from pulsar_amd import ops
    if kind == "attention":
        if not own:
            return _plain_attention(s)
        return ops.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["tables"], s["lens"], s["cu_q"], s["max_new"],
                                   s["max_len"], window=s["window"], softcap=s["cap"], return_lse=True)
    if kind == "logprobs":
        if not own:
            return _plain_logprobs(s["logits"], s["targets"], s["top"])
        return ops.token_logprobs(s["logits"], s["targets"], s["top"])
    meta, pool = s["meta"], s["pool"]
    meta["work"].copy_(meta["given"])  # the pass starts from the pool's given book-keeping
    refs, tables, lens = meta["refs"], meta["tables"], meta["lens"]
    if kind == "append":
        if own:
            slots, short = ops.paged_cache_extend(refs, tables, lens, s["cu_q"], s["tokens"], s["page"])
            ops.paged_cache_write(s["k"], s["v"], pool[0], pool[1], slots)
        else:
            slots, short = _plain_extend(refs, tables, lens, s["cu_q"], s["tokens"], s["page"])
            flat = pool.view(2, -1, *pool.shape[3:])
            flat[0, slots] = s["k"]
            flat[1, slots] = s["v"]
        return [pool, meta["work"], slots, short]
    if kind == "branch":
        if own:
            short = ops.paged_cache_fork(pool, refs, tables, lens, s["src"], s["dst"])
            ops.paged_cache_free(refs, tables, lens, s["old"])
        else:
            short = _plain_fork(pool, refs, tables, lens, s["src"], s["dst"])
            _plain_free(refs, tables, lens, s["old"])
        return [pool, meta["work"], short]
    if own:
        used = ops.paged_cache_compact(pool, refs, tables)
        ops.paged_cache_copy(pool, s["src"], s["dst"])
    else:
        used = _plain_compact(pool, refs, tables)
        pool[:, s["dst"].long()] = pool[:, s["src"].long()]
    return [pool, meta["work"], used]


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
    if kind == "logprobs":
        t, v = case["tokens"], case["vocab"]
        size = 4 if case["dtype"] == "f32" else 2
        return {"bytes": t * v * size + t * (8 + 4 + 8 + 4 + 12 * case["top"]), "flops": 5 * t * v}
    heads, dim, page = case["kv_heads"], case["dim"], case["page"]
    if kind == "attention":
        lens, new = _lengths(case)
        keys = sum(min(l, case["window"] + q - 1) if case["window"] else l for l, q in zip(lens, new))
        hq = heads * case["group"]
        return {"bytes": sum(new) * hq * (4 * dim + 4) + keys * heads * dim * 4 + 4 * -(-keys // page),
                "flops": 4 * dim * hq * sum(_visible(l, q, case["window"]) for l, q in zip(lens, new))}
    if kind == "append":
        lens, new = _lengths(case)
        pages = sum(-(-l // page) for l in lens)
        return {"bytes": sum(new) * (heads * dim * 8 + 8) + 8 * pages, "flops": 0}
    held = 2 * case["layers"] * page * heads * dim * 2  # one page of every plane
    if kind == "branch":
        lens, _ = _lengths(case)
        parts = sum(l % page != 0 for l in lens)
        return {"bytes": 2 * held * parts + 4 * sum(4 * -(-l // page) for l in lens), "flops": 0}
    moved = case["used"] * (case["pages"] - case["used"]) // case["pages"] + case["copied"]
    return {"bytes": 2 * held * moved + 8 * case["pages"] + 8 * case["used"], "flops": 0}


# ---- the definitions, in 64 bits ----------------------------------------------------------------


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    if case["kind"] == "logprobs":
        lp, ent, top = [], [], []
        for rows, given in zip(s["logits"].split(64), s["targets"].split(64)):
            x = rows.double()
            logp = x - torch.logsumexp(x, 1, keepdim=True)
            lp.append(logp.gather(1, given[:, None])[:, 0])
            ent.append(-(logp.exp() * logp).sum(1))
            top.append(logp.topk(case["top"], dim=1).values if case["top"] else logp[:, :0])
        return torch.cat(lp), None, torch.cat(ent), torch.cat(top), None
    if case["kind"] != "attention":
        return None  # whole numbers, and values moved as they are
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
        for h in range(case["kv_heads"] * g):
            k = s["k_cache"][pages, pos % page, h // g].double()
            v = s["v_cache"][pages, pos % page, h // g].double()
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
