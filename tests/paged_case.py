"""Inputs and 64-bit references of the paged-cache and log-probability tests."""

from __future__ import annotations

import math

import torch

DEV = "cuda:0"


def gen(seed: int) -> torch.Generator:
    return torch.Generator().manual_seed(seed)


def paged_kv(lens, page, heads, dim, dtype, seed, layout="nhd", slack=3, junk=float("nan")):
    """(k_cache, v_cache, tables, k rows, v rows) on the device: each sequence's keys and values
    scattered over a shuffled pool whose other slots hold `junk`; rows are [len, heads, dim] on the
    host.  `layout` "hnd" keeps a page's tokens of one head together."""
    g = gen(seed)
    held = [-(-l // page) for l in lens]
    pages, width = sum(held) + slack, max(held + [1])
    order = torch.randperm(pages, generator=g)
    shape = (2, pages, page, heads, dim) if layout == "nhd" else (2, pages, heads, page, dim)
    pool = torch.full(shape, junk, dtype=dtype)
    if layout == "hnd":
        pool = pool.transpose(2, 3)
    tables = torch.full((len(lens), width), -1, dtype=torch.int32)
    ks, vs, at = [], [], 0
    for b, l in enumerate(lens):
        mine = order[at:at + held[b]]
        at += held[b]
        tables[b, :held[b]] = mine.int()
        k, v = (torch.randn(l, heads, dim, generator=g).to(dtype) for _ in range(2))
        j = torch.arange(l)
        pool[0, mine[j // page], j % page] = k
        pool[1, mine[j // page], j % page] = v
        ks.append(k)
        vs.append(v)
    dev = pool.to(DEV)  # keeps the strides
    assert dev.stride() == pool.stride()
    return dev[0], dev[1], tables.to(DEV), ks, vs


def offsets(counts) -> torch.Tensor:
    return torch.tensor([0, *torch.tensor(counts, dtype=torch.int64).cumsum(0).tolist()], dtype=torch.int32)


def attention_ref(q, k, v, length, n, scale, window, cap):
    """(out, lse, weight, reach) in 64 bits for one sequence: q [n, Hq, D], k and v [length, Hkv, D].
    `weight` is sum p |v|, `reach` the largest scale * sum |q| |k| of a visible key: what rounding
    errors are measured by."""
    q, k, v = q.double(), k.double(), v.double()
    hq, hkv, d = q.shape[1], k.shape[1], q.shape[2]
    k, v = (t.repeat_interleave(hq // hkv, dim=1).permute(1, 0, 2) for t in (k, v))
    q = q.permute(1, 0, 2)
    s = q @ k.transpose(1, 2) * scale
    reach = q.abs() @ k.abs().transpose(1, 2) * abs(scale)
    if cap:
        s = cap * torch.tanh(s / cap)
    pos = torch.arange(length)[None, :]
    p = torch.arange(length - n, length)[:, None]
    seen = (pos <= p) & ((pos > p - window) if window else True)
    # what a query does not see takes no part in any sum, whatever it holds
    s = torch.where(seen, s, -math.inf)
    reach = torch.where(seen, reach, 0.0)
    top = s.amax(-1, keepdim=True).clamp(min=-1e300) if length else torch.zeros(hq, n, 1, dtype=torch.float64)
    e = torch.exp(s - top)
    z = e.sum(-1, keepdim=True)
    pr = torch.where(z > 0, e / z, 0.0)
    finite = torch.where(v.isfinite(), v, 0.0)
    out = pr @ finite
    for h, j in {(int(h), int(j)) for h, j in torch.nonzero((~v.isfinite()).any(-1))}:  # hq, key
        out[h] = torch.where(seen[:, j, None], out[h] + torch.where(v[h, j].isfinite(), 0.0, v[h, j]), out[h])
    lse = (top + torch.log(z))[..., 0]
    most = reach.amax(-1) if length else torch.zeros(hq, n, dtype=torch.float64)
    return (out.permute(1, 0, 2), lse.t(), (pr @ finite.abs()).permute(1, 0, 2), most.t())


def check_attention(out, lse, ref, dim, keys, dtype):
    """Elementwise bounds: the scores' fp32 error d (a sum of dim + 8 roundings of the terms' absolute
    sum) changes each e^s by a factor of 1 +- d, hence the output by 2 d of sum p |v|; the probabilities
    are rounded to the cache's type (u of sum p |v|), the sums of `keys` terms and the hardware's exp2
    add (keys + 64) roundings, the output is rounded once (u of itself)."""
    want, want_lse, weight, reach = ref
    u = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -11
    eps = 2.0 ** -24
    d = ((dim + 8) * eps * reach + (keys + 64) * eps)[..., None]
    bound = u * want.abs() + 1.01 * (u + 2 * d) * weight + 2.0 ** -24
    got = out.cpu().double()
    finite = want.isfinite()
    assert torch.equal(got.isfinite(), finite)
    err = torch.where(finite, (got - want).abs(), 0.0)
    bound = torch.where(finite, bound, 1.0)
    assert bool((err <= bound).all()), f"worst {float((err / bound).max()):.2f} of the bound"
    if lse is not None:
        got_lse = lse.cpu().double()
        fine = want_lse > -math.inf
        assert torch.equal(got_lse > -math.inf, fine)
        lb = d[..., 0] + 4 * eps * want_lse.abs() + 4 * eps * reach
        assert bool(((got_lse - want_lse).abs()[fine] <= lb[fine]).all())


class Pages:
    """The book-keeping of a pool on the host, by its definition."""

    def __init__(self, refs, tables, lens, page):
        self.refs, self.tables, self.lens, self.page = refs.clone(), tables.clone(), lens.clone(), page

    def _free(self):
        return [p for p, r in enumerate(self.refs.tolist()) if r == 0]

    def extend(self, counts):
        b = len(counts)
        have = [-(-int(self.lens[i]) // self.page) for i in range(b)]
        want = [-(-(int(self.lens[i]) + counts[i]) // self.page) for i in range(b)]
        need = sum(w - h for w, h in zip(want, have))
        free = self._free()
        missing = max(need - len(free), 0) + sum(max(w - self.tables.shape[1], 0) for w in want)
        if missing:
            return [-1] * sum(counts), missing
        slots = []
        for i in range(b):
            for c in range(have[i], want[i]):
                p = free.pop(0)
                self.tables[i, c] = p
                self.refs[p] = 1
            for t in range(int(self.lens[i]), int(self.lens[i]) + counts[i]):
                slots.append(int(self.tables[i, t // self.page]) * self.page + t % self.page)
            self.lens[i] += counts[i]
        return slots, 0

    def fork(self, src, dst, pool):
        parts = [s for s in src if int(self.lens[s]) % self.page]
        free = self._free()
        if len(parts) > len(free):
            return len(parts) - len(free)
        for s, d in zip(src, dst):
            n = int(self.lens[s])
            self.tables[d] = -1
            for c in range(n // self.page):
                p = int(self.tables[s, c])
                self.tables[d, c] = p
                self.refs[p] += 1
            if n % self.page:
                c, p = n // self.page, free.pop(0)
                self.tables[d, c] = p
                self.refs[p] = 1
                pool[:, p] = pool[:, int(self.tables[s, c])]
            self.lens[d] = n
        return 0

    def free(self, rows):
        for r in sorted(set(rows)):
            for p in self.tables[r].tolist():
                if p >= 0:
                    self.refs[p] -= 1
            self.tables[r] = -1
            self.lens[r] = 0

    def compact(self, pool):
        used = [p for p, r in enumerate(self.refs.tolist()) if r > 0]
        n = len(used)
        holes = [p for p in range(n) if self.refs[p] == 0]
        name = {}
        for h, s in zip(holes, [p for p in used if p >= n]):
            pool[:, h] = pool[:, s]
            self.refs[h], self.refs[s] = self.refs[s].clone(), 0
            name[s] = h
        self.tables.apply_(lambda p: name.get(p, p))
        return n


def logprobs_ref(x, targets, top):
    """(logprobs, ranks, entropy, top logprobs, top ids) in 64 bits; ties by index."""
    x = x.double()
    t, v = x.shape
    lse = torch.logsumexp(x, 1)
    lp, rank = torch.zeros(t, dtype=torch.float64), torch.full((t,), -1)
    idx = torch.arange(v)
    for i, g in enumerate(targets.tolist()):
        if 0 <= g < v:
            lp[i] = x[i, g] - lse[i]
            rank[i] = int(((x[i] > x[i, g]) | ((x[i] == x[i, g]) & (idx < g))).sum())
    p = torch.exp(x - lse[:, None])
    ent = -torch.where(p > 0, p * (x - lse[:, None]), 0.0).sum(1)
    order = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :top]
    return lp, rank, ent, x.gather(1, order) - lse[:, None], order
