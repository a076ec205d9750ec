"""token_logprobs against its definition in 64 bits: whole numbers equal, computed ones within bounds
that follow from fp32 sums (below)."""

import ctypes
import math

import pytest
import torch

import pulsar_amd
from paged_case import DEV, gen, logprobs_ref
from pulsar_amd import ops

F, H, B = torch.float32, torch.float16, torch.bfloat16


def _check(x, targets, top, got):
    lp, rank, ent, tlp, ids = (g.cpu() for g in got)
    want = logprobs_ref(x.cpu(), targets.cpu(), top)
    assert torch.equal(rank, want[1]) and torch.equal(ids, want[4])
    # e^(x - m): its argument is rounded (eps of |x - m| <= range), the hardware's exp2 adds 2 eps, and a
    # sum of 64 terms a thread, 8 steps of a tree and the join adds 100 eps.  lse takes that, and its
    # own rounding; the entropy is a sum of p |x - m|, each with the same relative error.
    eps = 2.0 ** -24
    xd = x.cpu().double()
    m = xd.amax(1)
    low = torch.where(xd > -math.inf, xd, m[:, None]).amin(1)
    lse = torch.logsumexp(xd, 1)
    p = torch.exp(xd - lse[:, None])
    spread = torch.where(p > 0, p * (xd - m[:, None]).abs(), 0.0).sum(1)
    rel = eps * (160 + 2 * (torch.where(p > 0, p * p.log().abs(), 0.0).sum(1) + spread))
    rel = torch.minimum(rel, eps * (160 + 2 * (m - low)))
    b_lse = rel + 2 * eps * lse.abs()
    fine = want[0].isfinite()
    assert torch.equal(lp.isfinite(), fine)
    assert bool(((lp.double() - want[0]).abs() <= b_lse + 4 * eps * want[0].abs())[fine].all())
    assert bool(((ent.double() - want[2]).abs() <= 2 * rel * (1 + spread) + 4 * eps * (lse - m).abs() + 1e-7).all())
    fine = want[3].isfinite()
    assert torch.equal(tlp.isfinite(), fine)
    assert bool(((tlp.double() - want[3]).abs() <= b_lse[:, None] + 4 * eps * want[3].abs())[fine].all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F, H, B])
@pytest.mark.parametrize("vocab", [1, 2, 7, 31, 33, 255, 1000, 16375, 16376, 16377, 32768, 50001, 131073])
@pytest.mark.parametrize("tokens", [1, 5])
def test_sizes(vocab, tokens, dtype):
    g = gen(vocab + tokens)
    x = (torch.randn(tokens, vocab, generator=g) * 3).to(dtype).to(DEV)
    t = torch.randint(0, vocab, (tokens,), generator=g).to(DEV)
    for top in sorted({0, 1, min(5, vocab), min(32, vocab)}):
        _check(x, t, top, ops.token_logprobs(x, t, top))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F, H, B])
def test_many_tokens(dtype):
    g = gen(1)
    x = (torch.randn(700, 3001, generator=g) * 4).to(dtype).to(DEV)
    t = torch.randint(0, 3001, (700,), generator=g).to(DEV)
    _check(x, t, 20, ops.token_logprobs(x, t, 20))


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [40, 5000, 40000])
@pytest.mark.parametrize("levels", [1, 2, 3])
def test_ties_go_to_the_lower_index(vocab, levels):
    """Few different logits: every list of candidates is longer than it holds."""
    g = gen(vocab)
    x = torch.randint(0, levels, (4, vocab), generator=g).float().to(DEV)
    x[3] = 0.0
    x[3, ::2] = -0.0  # equal to 0
    t = torch.tensor([0, vocab - 1, vocab // 2, 5], device=DEV)
    for dtype in (F, B):
        for top in (1, 5, 32):
            _check(x.to(dtype), t, top, ops.token_logprobs(x.to(dtype), t, top))


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [50, 40000])
@pytest.mark.parametrize("left", [1, 3, 40])
def test_masked_logits(vocab, left):
    """All but a few logits -inf, or the type's lowest value: they hold no probability."""
    g = gen(left)
    for dtype in (F, H, B):
        for low in (-math.inf, torch.finfo(dtype).min):
            x = torch.full((3, vocab), low)
            keep = torch.randperm(vocab, generator=g)[:left]
            x[:, keep] = torch.randn(3, left, generator=g)
            x = x.to(dtype).to(DEV)
            t = torch.tensor([int(keep[0]), (int(keep[0]) + 1) % vocab, 0], device=DEV)
            _check(x, t, min(8, left), ops.token_logprobs(x, t, min(8, left)))
            # past the tokens left: -inf (or the lowest), by index
            _, _, _, tlp, ids = ops.token_logprobs(x, t, 32)
            assert torch.equal(ids.cpu(), logprobs_ref(x.cpu(), t.cpu(), 32)[4])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F, H, B])
@pytest.mark.parametrize("vocab", [9, 33000])
def test_a_row_of_nothing(vocab, dtype):
    x = torch.full((2, vocab), -math.inf, dtype=dtype, device=DEV)
    x[1, 3] = 1.0
    lp, rank, ent, tlp, ids = ops.token_logprobs(x, torch.tensor([2, 3], device=DEV), 4)
    assert lp.tolist() == [-math.inf, 0.0] and ent.tolist() == [0.0, 0.0] and rank.tolist() == [2, 0]
    assert tlp.tolist() == [[-math.inf] * 4, [0.0] + [-math.inf] * 3]
    assert ids.tolist() == [[0, 1, 2, 3], [3, 0, 1, 2]]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F, H, B])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_nan_and_infinity_stay_in_their_row(bad, dtype):
    vocab = 20000
    x = torch.randn(3, vocab, generator=gen(1)).to(dtype).to(DEV)
    t = torch.tensor([1, 2, 3], device=DEV)
    want = ops.token_logprobs(x, t, 5)
    x[1, 17000] = bad
    lp, rank, ent, tlp, ids = got = ops.token_logprobs(x, t, 5)
    for a, b in zip(got, want):
        assert torch.equal(a[::2], b[::2])
    assert bool(lp[1].isnan()) and bool(ent[1].isnan()) and bool(tlp[1].isnan().all())
    if bad == math.inf:
        assert ids[1].tolist() == [17000] + want[4][1, :4].tolist() and int(rank[1]) == int(want[1][1]) + 1
    else:
        assert torch.equal(ids[1], want[4][1]) and int(rank[1]) == int(want[1][1])


@pytest.mark.gpu
def test_no_token_given():
    x = torch.randn(4, 100, generator=gen(1)).to(DEV)
    t = torch.tensor([-1, 5, 100, 2 ** 40], device=DEV)
    lp, rank, ent, _, _ = ops.token_logprobs(x, t, 0)
    assert lp[[0, 2, 3]].tolist() == [0.0] * 3 and rank[[0, 2, 3]].tolist() == [-1] * 3
    want = logprobs_ref(x.cpu(), t.cpu(), 0)
    assert int(rank[1]) == int(want[1][1]) and abs(float(lp[1]) - float(want[0][1])) < 1e-5


@pytest.mark.gpu
def test_extreme_logits():
    x = torch.tensor([[3e38, -3e38, 0.0, 3e38], [-3e38, -3e38, -3e38, -2.9e38], [60000.0, -60000.0, 1.0, 2.0]], device=DEV)
    t = torch.tensor([0, 3, 1], device=DEV)
    lp, rank, ent, _, ids = ops.token_logprobs(x, t, 4)
    assert lp.tolist() == [pytest.approx(-math.log(2)), 0.0, -120000.0]
    assert ent.tolist() == [pytest.approx(math.log(2)), 0.0, 0.0]
    assert rank.tolist() == [0, 0, 3] and ids.tolist() == [[0, 3, 2, 1], [3, 0, 1, 2], [0, 3, 2, 1]]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F, H, B])
def test_strides(dtype):
    """Rows apart, rows at odd addresses, columns first."""
    g = gen(2)
    raw = (torch.randn(6, 20011, generator=g) * 2).to(dtype).to(DEV)
    t = torch.randint(0, 17000, (6,), generator=g).to(DEV)
    for x in (raw[:, :17000], raw[:, 3:17003], raw[1:, 1:17002]):
        tt = t[:x.shape[0]]
        _check(x, tt, 7, ops.token_logprobs(x, tt, 7))
    x = raw[:, :17000].t().contiguous().t()
    _check(x, t, 7, ops.token_logprobs(x, t, 7))
    x = raw[:1, :17000].expand(6, 17000)  # one row for all: laid out for the call
    _check(x, t, 7, ops.token_logprobs(x, t, 7))


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """Logits of more than 2^32 bytes."""
    vocab = 1 << 17
    x = torch.zeros(16400, vocab, dtype=H, device=DEV)
    x[-1, 7] = 3.0
    t = torch.full((16400,), 7, device=DEV)
    lp, rank, ent, tlp, ids = ops.token_logprobs(x, t, 1)
    _check(x[-2:], t[-2:], 1, [g[-2:] for g in (lp, rank, ent, tlp, ids)])


@pytest.mark.gpu
def test_repeats_streams_and_graphs():
    x = torch.randn(9, 40000, generator=gen(1)).to(B).to(DEV)
    t = torch.arange(9, device=DEV)
    first = ops.token_logprobs(x, t, 6)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        captured = ops.token_logprobs(x, t, 6)
    for _ in range(3):
        for c in captured:
            c.fill_(3)
        graph.replay()
        eager = ops.token_logprobs(x, t, 6)
        torch.cuda.synchronize()
        for a, b, c in zip(first, captured, eager):
            assert torch.equal(a, b) and torch.equal(a, c)


@pytest.mark.gpu
def test_refusals():
    x, t = torch.zeros(2, 40, device=DEV), torch.zeros(2, dtype=torch.int64, device=DEV)
    for call, message in ((lambda: ops.token_logprobs(x.double(), t, 1), "fp32, fp16 or bf16"),
                          (lambda: ops.token_logprobs(x[0], t, 1), "2-D"),
                          (lambda: ops.token_logprobs(x[:, :0], t, 0), "2-D"),
                          (lambda: ops.token_logprobs(x, t.int(), 1), "int64"),
                          (lambda: ops.token_logprobs(x, t[:1], 1), "targets"),
                          (lambda: ops.token_logprobs(x, t, 33), "top_k"),
                          (lambda: ops.token_logprobs(x, t, -1), "top_k"),
                          (lambda: ops.token_logprobs(x[:, :3], t, 4), "top_k"),
                          (lambda: ops.token_logprobs(x, t.cpu(), 1), "one CUDA device")):
        with pytest.raises(RuntimeError, match=message):
            call()
    empty = ops.token_logprobs(x[:0], t[:0], 3)
    assert [tuple(e.shape) for e in empty] == [(0,), (0,), (0,), (0, 3), (0, 3)]


def test_c_entry_refuses_before_any_launch():
    lib = pulsar_amd.capi()
    P, I, SZ = ctypes.c_void_p, ctypes.c_int64, ctypes.c_size_t
    lib.pw4_token_logprobs.argtypes = [P, ctypes.c_int, I, I, I, P, I, P, P, P, P, P, P, SZ, P]
    lib.pw4_token_logprobs_workspace_size.argtypes, lib.pw4_token_logprobs_workspace_size.restype = [I] * 3, SZ
    need = lib.pw4_token_logprobs_workspace_size(4, 50000, 5)
    assert need > 0 and lib.pw4_token_logprobs_workspace_size(0, 50000, 5) == 0
    x = P(4096)

    def call(dtype=1, n=4, v=50000, stride=50000, k=5, logits=x, top=x, ws=x, size=need):
        return lib.pw4_token_logprobs(logits, dtype, n, v, stride, x, k, x, x, x, top, x, ws, size, None)

    assert call(dtype=3) == -1 and call(v=0) == -1 and call(n=-1) == -1 and call(logits=None) == -1
    assert call(k=33) == -2 and call(v=3, k=4) == -2 and call(stride=49999) == -2 and call(v=2 ** 31) == -2
    assert call(top=None) == -1 and call(logits=P(4097)) == -1
    assert call(ws=None) == -3 and call(size=need - 1) == -3
    assert call(n=0, logits=None) == 0


def test_fake_kernel():
    x = torch.empty(3, 50, dtype=H, device="meta")
    got = ops.token_logprobs(x, torch.empty(3, dtype=torch.int64, device="meta"), 4)
    assert [tuple(g.shape) for g in got] == [(3,), (3,), (3,), (3, 4), (3, 4)]
    assert [g.dtype for g in got] == [F, torch.int64, F, F, torch.int64]


@pytest.mark.gpu
def test_opcheck():
    x = torch.randn(2, 50, generator=gen(1)).to(DEV)
    torch.library.opcheck(torch.ops.pulsar.token_logprobs.default, (x, torch.zeros(2, dtype=torch.int64, device=DEV), 3),
                          test_utils=("test_schema", "test_faketensor", "test_aot_dispatch_dynamic"))


@pytest.mark.gpu
def test_a_target_of_one_token_may_be_any_view():
    x = torch.randn(1, 100, generator=gen(1)).to(DEV)
    t = torch.tensor([5, 6, 7], device=DEV)
    for a, b in zip(ops.token_logprobs(x, t[::3], 2), ops.token_logprobs(x, t[:1], 2)):
        assert torch.equal(a, b)


def _spread_over_few_groups(vocab, dtype, seed):
    """A row whose larger logits, some thousand of a slice, all different, lie in the vectors that 124 of
    a workgroup's 256 threads take (31 groups of four), and whose others are equal."""
    vec = 128 // torch.finfo(dtype).bits
    x = torch.zeros(vocab)
    there = torch.nonzero((torch.arange(vocab) // (4 * vec)) % 64 < 31)[:, 0]
    x[there] = 1 + torch.rand(len(there), generator=gen(seed)) * 6
    return x.to(dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F, H, B])
@pytest.mark.parametrize("tokens,vocab", [(1, 4096), (2, 30000), (300, 8192), (64, 30000)])
def test_more_large_logits_than_a_list_holds(tokens, vocab, dtype):
    x = torch.stack([_spread_over_few_groups(vocab, dtype, i) for i in range(tokens)]).to(DEV)
    t = torch.randint(0, vocab, (tokens,), generator=gen(5)).to(DEV)
    for top in (31, 32):
        _check(x, t, top, ops.token_logprobs(x, t, top))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F, B])
@pytest.mark.parametrize("tokens,vocab,top", [(2, 100003, 32), (2, 100003, 26), (64, 150001, 32), (64, 150001, 20),
                                              (1, 600011, 32), (3, 600011, 5)])
def test_rows_of_many_slices(tokens, vocab, top, dtype):
    """More slices than top tokens and fewer, up to more slices than a wave has lanes; and the same rows
    of a few different logits, and of almost nothing."""
    g = gen(vocab + top)
    t = torch.randint(0, vocab, (tokens,), generator=g).to(DEV)
    x = (torch.randn(tokens, vocab, generator=g) * 3).to(dtype).to(DEV)
    _check(x, t, top, ops.token_logprobs(x, t, top))
    x = torch.randint(0, 3, (tokens, vocab), generator=g).to(dtype).to(DEV)
    _check(x, t, top, ops.token_logprobs(x, t, top))
    x = torch.full((tokens, vocab), -math.inf, dtype=dtype)
    x[:, vocab // 2] = 1.0
    x, t = x.to(DEV), torch.full_like(t, vocab // 2)
    assert torch.equal(ops.token_logprobs(x, t, top)[4].cpu(), logprobs_ref(x.cpu(), t.cpu(), top)[4])


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,vocab,top", [(1, 1, 1), (3, 9000, 32), (7, 50001, 5), (300, 8193, 20), (65, 20000, 0)])
def test_writes_stay_in_the_outputs_and_the_workspace(tokens, vocab, top):
    """The C entry on buffers with a margin behind each."""
    lib = pulsar_amd.capi()
    P, I, SZ = ctypes.c_void_p, ctypes.c_int64, ctypes.c_size_t
    lib.pw4_token_logprobs.argtypes = [P, ctypes.c_int, I, I, I, P, I, P, P, P, P, P, P, SZ, P]
    lib.pw4_token_logprobs_workspace_size.argtypes, lib.pw4_token_logprobs_workspace_size.restype = [I] * 3, SZ
    x = torch.randn(tokens, vocab, generator=gen(tokens)).to(B).to(DEV)
    t = torch.randint(0, vocab, (tokens,), generator=gen(vocab)).to(DEV)
    want = ops.token_logprobs(x, t, top)
    got = [torch.full((w.numel() + 16,), 77, dtype=w.dtype, device=DEV) for w in want]
    size = lib.pw4_token_logprobs_workspace_size(tokens, vocab, top)
    ws = torch.full((size + 256,), 0x5a, dtype=torch.uint8, device=DEV)
    torch.cuda.synchronize()
    assert lib.pw4_token_logprobs(x.data_ptr(), 1, tokens, vocab, vocab, t.data_ptr(), top, *(g.data_ptr() for g in got),
                                  ws.data_ptr(), size, None) == 0
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        assert torch.equal(g[:w.numel()].view(w.shape), w) and bool((g[w.numel():] == 77).all())
    assert bool((ws[size:] == 0x5a).all())
