"""beam_select and beam_reorder against their definitions: rows and tokens equal to a selection over the
totals in 64 bits, scores within what fp32 sums of a row leave.

A row's sum of e^(x - m) is fp32: the bound is token_logprobs' (an argument's rounding, exp2's two and
100 sums' roundings), relative to the sum and so absolute in its logarithm; a total's own rounding to
fp32 is half a step.  Where two beams' totals that the choice or the order depends on are as near as that, and
do not tie exactly, either is right: then the totals in 64 bits of what was chosen have to be as good."""

import ctypes
import math

import pytest
import torch

import pulsar_amd
from paged_case import DEV, gen
from pulsar_amd import ops

F, H, B = torch.float32, torch.float16, torch.bfloat16


def select_ref(logits, scores, width, ended=None, end_token=-1):
    """(totals in 64 bits, rows, tokens, ended) [batch, width], and the least gap between totals in the order."""
    (b, k), v = scores.shape, logits.shape[1]
    x = logits.double()
    lse = torch.logsumexp(x, 1, keepdim=True)
    total = scores.double().view(-1, 1) + (x - lse)
    total = torch.where(total.isnan(), -math.inf, total)
    logit = torch.where(x.isnan(), -math.inf, x) + 0.0
    out = []
    gap = math.inf
    for i in range(b):
        cands = []
        for j in range(k):
            row = i * k + j
            if ended is not None and ended[i, j]:
                s = float(scores[i, j])
                cands.append((-(s if s == s else -math.inf), j, 0.0, end_token))
                continue
            # the row's best by logit, then token
            order = torch.sort(logit[row], descending=True, stable=True).indices[:width + 1].tolist()
            cands += [(-float(total[row, t]), j, -float(logit[row, t]), t) for t in order]
        cands.sort()
        best = cands[:width]
        for a, c in zip(cands[:width], cands[1:width + 1]):
            if a[1] != c[1] and a[0] != c[0] and math.isfinite(a[0]) and math.isfinite(c[0]):
                gap = min(gap, c[0] - a[0])
        out.append([(-t, i * k + j, tok, bool(ended[i, j]) or tok == end_token if ended is not None else False)
                    for t, j, _, tok in best])
    cols = list(zip(*[list(zip(*o)) for o in out]))
    return (torch.tensor(cols[0], dtype=torch.float64), torch.tensor(cols[1]), torch.tensor(cols[2]),
            torch.tensor(cols[3]), gap)


EPS = 2.0 ** -24


def _sum_error(x):
    """Of a row's logarithm of its sum."""
    x = x.double()
    m = x.amax(1, keepdim=True)
    p = torch.softmax(x, 1)
    spread = torch.where(p > 0, p * (x - m).abs(), 0.0).sum(1)
    return EPS * (160 + 2 * spread)


def _check(logits, scores, width=None, ended=None, end_token=-1):
    args = (logits.to(DEV), scores.to(DEV), width, None if ended is None else ended.to(DEV), end_token)
    got = [g.cpu() for g in ops.beam_select(*args)]
    w = scores.shape[1] if width is None else width
    want = select_ref(logits, scores, w, ended, end_token)
    err = _sum_error(logits)
    fine = want[0].isfinite()
    finite = err[err.isfinite()]
    most = 2 * float(finite.max() if finite.numel() else 0.0)
    if want[4] > most:
        assert torch.equal(got[1].long(), want[1]) and torch.equal(got[2], want[2])
    else:
        row, token = got[1].long(), got[2]
        total = scores.double().view(-1)[row] + torch.log_softmax(logits.double(), 1)[row, token.clamp(min=0)]
        if ended is not None:
            total = torch.where(ended.view(-1)[row], scores.double().view(-1)[row], total)
        assert bool(((total - want[0]).abs() <= most)[fine].all())
        assert len(set(zip(row.view(-1).tolist(), token.view(-1).tolist()))) == row.numel()
    assert torch.equal(got[0][~fine].double(), want[0][~fine])
    bound = err[want[1]] + EPS * want[0].abs() + 1e-12
    assert bool(((got[0].double() - want[0]).abs() <= bound)[fine].all())
    if ended is None:
        assert len(got) == 3
    else:
        assert torch.equal(got[3], want[3])
    return got


def _logits(rows, vocab, dtype, seed, scale=3.0):
    return (torch.randn(rows, vocab, generator=gen(seed)) * scale).to(dtype)


def _scores(batch, beams, seed):
    return -torch.rand(batch, beams, generator=gen(seed)) * 5 - 20


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F, H, B])
@pytest.mark.parametrize("vocab", [1, 2, 7, 33, 1000, 16376, 16377, 50001])
@pytest.mark.parametrize("batch,beams", [(1, 1), (1, 4), (3, 5), (2, 32)])
def test_sizes(batch, beams, vocab, dtype):
    _check(_logits(batch * beams, vocab, dtype, vocab + beams), _scores(batch, beams, vocab))


@pytest.mark.gpu
@pytest.mark.parametrize("beams,width", [(1, 1), (1, 8), (1, 32), (4, 1), (4, 8), (8, 3), (32, 32), (3, 32)])
def test_widths(beams, width):
    """From one beam to many, from many to few."""
    _check(_logits(2 * beams, 3001, B, width), _scores(2, beams, width), width)
    if beams * 12 >= width:
        _check(_logits(2 * beams, 12, F, width), _scores(2, beams, width), width)


@pytest.mark.gpu
def test_many_searches():
    _check(_logits(500 * 3, 700, H, 1), _scores(500, 3, 2))


@pytest.mark.gpu
@pytest.mark.parametrize("beams", [1, 4, 9])
def test_ended_beams(beams):
    batch, vocab = 5, 2000
    ended = torch.rand(batch, beams, generator=gen(1)) < 0.5
    ended[0], ended[1] = True, False
    scores = _scores(batch, beams, 3) + torch.where(ended, 0.0, 4.0)
    logits = _logits(batch * beams, vocab, B, 4)
    logits[:, 7] = 12.0  # the end is likely: new beams end as well
    logits.view(batch, beams, vocab)[ended] = math.nan  # logits that are not read
    finite = torch.where(ended.view(-1, 1), 0.0, logits.float()).to(B)
    args = (scores, None, ended, 7)
    want = select_ref(finite, scores, beams, ended, 7)
    got = [g.cpu() for g in ops.beam_select(logits.to(DEV), scores.to(DEV), None, ended.to(DEV), 7)]
    assert want[4] > 4 * EPS * 200
    assert torch.equal(got[1].long(), want[1]) and torch.equal(got[2], want[2]) and torch.equal(got[3], want[3])
    assert bool(want[3].any()) and (beams == 1 or not bool(want[3].all()))
    for i in range(beams):  # a search at its end stays as it is, in the order of its scores
        assert sorted(got[0][0].tolist(), reverse=True) == got[0][0].tolist()
    assert torch.equal(got[0][0].sort().values, scores[0].sort().values)
    _check(finite, *args)
    _check(finite, scores, max(1, beams // 2), ended, 7)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F, B])
@pytest.mark.parametrize("vocab", [5, 40, 9000])
def test_ties(vocab, dtype):
    """Equal rows and equal logits: the lower beam, then the lower token."""
    beams = 4
    x = torch.randint(0, 3, (1, vocab), generator=gen(vocab)).to(dtype).repeat(2 * beams, 1)
    x[:, 1] = -0.0
    got = _check(x, torch.full((2, beams), -3.0))
    assert bool((got[0][:, 1:] <= got[0][:, :-1]).all())
    _check(x, torch.full((2, beams), -3.0), min(32, beams * vocab))
    _check(torch.zeros_like(x), torch.full((2, beams), -3.0), min(32, beams * vocab))


@pytest.mark.gpu
def test_unused_beams():
    """A search that begins: one beam counts, the others have scores of -inf."""
    scores = torch.full((2, 6), -math.inf)
    scores[:, 0] = 0.0
    x = _logits(12, 4000, B, 2)
    got = _check(x, scores)
    assert bool((got[1] == torch.tensor([[0], [6]])).all())
    # fewer tokens than beams: the rest comes from beams of no score
    got = _check(x[:, :4].contiguous(), scores)
    assert bool((got[0][:, 4:] == -math.inf).all()) and bool((got[0][:, :4] > -math.inf).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F, H, B])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_rows_that_are_not_finite(bad, dtype):
    """Their continuations count as -inf; the others are chosen as ever.  Masked tokens have no probability."""
    x = _logits(8, 20000, dtype, 3)
    x[1, 17000] = bad
    x[2] = -math.inf
    x[5, 100:] = -math.inf
    x[6, :-3] = torch.finfo(dtype).min
    scores = _scores(2, 4, 1)
    args = (x.to(DEV), scores.to(DEV))
    got = [g.cpu() for g in ops.beam_select(*args)]
    clean = x.clone()
    clean[1] = -math.inf  # no candidate of these is above -inf either way
    want = select_ref(clean, scores, 4)
    assert torch.equal(got[1].long(), want[1]) and torch.equal(got[2], want[2])
    assert bool(got[0].isfinite().all()) and not bool(torch.isin(got[1], torch.tensor([1, 2])).any())
    nothing = torch.full((4, 50), math.nan, dtype=dtype)
    got = [g.cpu() for g in ops.beam_select(nothing.to(DEV), torch.zeros(1, 4, device=DEV))]
    assert bool((got[0] == -math.inf).all()) and got[1].tolist() == [[0] * 4] and got[2].tolist() == [[0, 1, 2, 3]]
    got = [g.cpu() for g in ops.beam_select(x[:4].to(DEV), torch.tensor([[-1.0, -1.0, -1.0, math.nan]], device=DEV))]
    assert got[1].tolist() == [[0] * 4] and bool(got[0].isfinite().all())


@pytest.mark.gpu
def test_far_scores():
    """Scores of some thousand, where fp32 totals of two beams would tie."""
    scores = torch.tensor([[-5000.0, -5000.25, -5000.5, -4999.75]])
    x = _logits(4, 3000, F, 9, 0.01)
    _check(x, scores, 32)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F, H, B])
def test_strides(dtype):
    x = _logits(6, 1003, dtype, 1)
    s = _scores(2, 3, 1)
    want = ops.beam_select(x.to(DEV), s.to(DEV))
    wide = torch.zeros(6, 1100, dtype=dtype, device=DEV)
    for shift in (0, 1, 5):
        view = wide[:, shift:shift + 1003]
        view.copy_(x)
        for a, b in zip(want, ops.beam_select(view, s.to(DEV))):
            assert torch.equal(a, b)
    for view, scores in ((x.t().contiguous().to(DEV).t(), s.to(DEV)), (x.to(DEV), s.t().contiguous().to(DEV).t())):
        for a, b in zip(want, ops.beam_select(view, scores)):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_offsets_past_32_bits():
    x = torch.full((4, 2 ** 29), -40.0, dtype=B, device=DEV)
    x[3, 2 ** 29 - 1] = 5.0
    x[2, 2 ** 29 - 7] = 4.0
    got = ops.beam_select(x, torch.zeros(1, 4, device=DEV), 2)
    assert got[1].tolist() == [[2, 3]] or got[1].tolist() == [[3, 2]]
    assert sorted(got[2].tolist()[0]) == [2 ** 29 - 7, 2 ** 29 - 1]


@pytest.mark.gpu
def test_repeats_streams_and_graphs():
    x, s = _logits(24, 30011, B, 1).to(DEV), _scores(3, 8, 1).to(DEV)
    ended = (torch.rand(3, 8, generator=gen(5)) < 0.3).to(DEV)
    history = torch.arange(24 * 77, device=DEV).view(24, 77)

    def call():
        picked = ops.beam_select(x, s, None, ended, 2)
        return [*picked, *ops.beam_reorder([history, s.view(24, 1)], picked[1])]

    first = call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = call()
        graph = torch.cuda.CUDAGraph()
    side.synchronize()
    with torch.cuda.graph(graph, stream=side):
        captured = call()
    for i in range(3):
        for t in captured:
            t.zero_()
        graph.replay()
        eager = call()
        torch.cuda.synchronize()
        for a, b, c in zip(captured, eager, first):
            assert torch.equal(a, b) and (i > 0 or torch.equal(a, c))
        x.copy_(x.flip(0).clone())
        ended.copy_(ended.flip(0).clone())
    for a, b in zip(first, other):
        assert torch.equal(a, b)


# ---- reordering --------------------------------------------------------------------------------


@pytest.mark.gpu
def test_reorder():
    """States of any type and width, whole and empty, more than a launch takes; rows outside become zeros."""
    g = gen(1)
    rows = torch.tensor([3, 3, 0, -1, 6, 7, 2 ** 31 - 1], dtype=torch.int32)
    states = [torch.randint(-9, 9, (7, *shape), generator=g).to(dtype) for shape, dtype in (
        ((1,), torch.int64), ((300,), torch.int64), ((), torch.float32), ((3,), torch.uint8), ((5, 7), torch.bfloat16),
        ((2, 3, 4000), torch.float32), ((0,), torch.int32), ((17,), torch.float16), ((1,), torch.bool), ((16385,), torch.uint8),
        ((8,), torch.complex64))]
    there = (rows >= 0) & (rows < 7)
    got = ops.beam_reorder([s.to(DEV) for s in states], rows.to(DEV))
    assert len(got) == len(states)
    for s, o in zip(states, got):
        want = torch.where(there.view(-1, *[1] * (s.dim() - 1)), s[rows.clamp(0, 6).long()], torch.zeros((), dtype=s.dtype))
        assert o.dtype == s.dtype and torch.equal(o.cpu(), want)
    # more rows than states have, rows of two dimensions, states that are views
    many = torch.randint(0, 7, (5, 40), generator=g).int()
    view = states[1].to(DEV)[:, 1::2]
    assert torch.equal(ops.beam_reorder([view], many.to(DEV))[0].cpu(), states[1][:, 1::2][many.view(-1).long()])
    assert ops.beam_reorder([], rows.to(DEV)) == []
    assert ops.beam_reorder([view], rows[:0].to(DEV))[0].shape == (0, view.shape[1])
    assert not bool(ops.beam_reorder([view[:0]], rows.to(DEV))[0].any())
    # addresses that only single bytes reach
    odd = torch.arange(100, dtype=torch.uint8, device=DEV)[1:].view(9, 11)
    assert torch.equal(ops.beam_reorder([odd], rows[:2].to(DEV))[0], odd[rows[:2].long()])


@pytest.mark.gpu
def test_reorder_past_32_bits():
    x = torch.zeros(3, 2 ** 31 + 64, dtype=torch.uint8, device=DEV)
    x[2, -70:] = torch.arange(70, dtype=torch.uint8, device=DEV)
    x[1, 5] = 9
    out = ops.beam_reorder([x], torch.tensor([2, 1, 2], dtype=torch.int32, device=DEV))[0]
    assert torch.equal(out[0], x[2]) and torch.equal(out[1], x[1]) and torch.equal(out[2], x[2])


# ---- refusals ------------------------------------------------------------------------------------


def _good():
    return dict(logits=torch.zeros(6, 50, device=DEV), scores=torch.zeros(2, 3, device=DEV), width=None,
                ended=torch.zeros(2, 3, dtype=torch.bool, device=DEV), end_token=1)


@pytest.mark.gpu
@pytest.mark.parametrize("change,message", [
    (lambda a: dict(logits=a["logits"].double()), "fp32, fp16 or bf16"),
    (lambda a: dict(logits=a["logits"][0]), "2-D"),
    (lambda a: dict(logits=a["logits"][:5]), "batch"),
    (lambda a: dict(logits=a["logits"].cpu()), "CUDA"),
    (lambda a: dict(scores=a["scores"].half()), "scores"),
    (lambda a: dict(scores=a["scores"].view(-1)), "scores"),
    (lambda a: dict(scores=a["scores"].cpu()), "CUDA"),
    (lambda a: dict(logits=torch.zeros(66, 50, device=DEV), scores=torch.zeros(2, 33, device=DEV), ended=None), "beams"),
    (lambda a: dict(width=0), "width"),
    (lambda a: dict(width=33, ended=None), "width"),
    (lambda a: dict(width=4), "width"),
    (lambda a: dict(logits=a["logits"][:, :1], width=4, ended=None), "width"),
    (lambda a: dict(ended=a["ended"].int()), "ended"),
    (lambda a: dict(ended=a["ended"][:1]), "ended"),
])
def test_refusals(change, message):
    args = _good()
    ops.beam_select(**args)
    args.update(change(args))
    with pytest.raises(RuntimeError, match=message):
        ops.beam_select(**args)


@pytest.mark.gpu
def test_reorder_refusals():
    x = torch.zeros(3, 4, device=DEV)
    rows = torch.zeros(2, dtype=torch.int32, device=DEV)
    for states, r, message in (([x], rows.long(), "int32"), ([x.cpu()], rows, "CUDA"), ([x[0, 0]], rows, "1-D"),
                               ([x], rows.cpu(), "CUDA")):
        with pytest.raises((RuntimeError, NotImplementedError), match=message):
            ops.beam_reorder(states, r)


class _State(ctypes.Structure):
    _fields_ = [("src", ctypes.c_void_p), ("dst", ctypes.c_void_p), ("row_bytes", ctypes.c_int64), ("num_rows", ctypes.c_int64)]


def test_c_entries_refuse_before_any_launch():
    lib = pulsar_amd.capi()
    size = lib.pw4_beam_select_workspace_size
    size.argtypes, size.restype = [ctypes.c_int64] * 4, ctypes.c_size_t
    f = lib.pw4_beam_select
    f.argtypes = ([ctypes.c_void_p, ctypes.c_int] + [ctypes.c_int64] * 4 + [ctypes.c_void_p] * 2 + [ctypes.c_int64] * 2
                  + [ctypes.c_void_p] * 5 + [ctypes.c_size_t, ctypes.c_void_p])

    def call(logits=4096, dtype=1, batch=2, beams=3, vocab=50, stride=50, scores=4096, ended=None, end=0, width=3, out=4096,
             rows=4096, tokens=4096, out_ended=None, ws=4096, nbytes=0):
        return f(logits, dtype, batch, beams, vocab, stride, scores, ended, end, width, out, rows, tokens, out_ended, ws,
                 nbytes, None)

    assert size(2, 3, 50, 3) > 0 and size(0, 3, 50, 3) == size(2, 33, 50, 3) == size(2, 3, 0, 3) == size(2, 3, 50, 33) == 0
    assert call() == -3 and call(ws=None, nbytes=1 << 30) == -3 and call(ws=4104, nbytes=1 << 30) == -3
    assert call(dtype=3) == -1 and call(batch=-1) == -1 and call(beams=0) == -1 and call(vocab=0) == -1 and call(width=0) == -1
    assert call(beams=33) == -2 and call(width=33) == -2 and call(vocab=2 ** 31) == -2 and call(stride=49) == -2
    assert call(batch=30000) == -2 and call(batch=2 ** 62) == -2
    assert call(ended=4096, width=4) == -2 and call(vocab=1, stride=1, width=4) == -2
    assert call(logits=None) == -1 and call(scores=None) == -1 and call(tokens=None) == -1 and call(logits=4097) == -1
    assert call(out_ended=4096) == -1 and call(dtype=2, logits=4098) == -1
    assert call(batch=0, logits=None) == 0
    r = lib.pw4_beam_reorder
    r.argtypes = [ctypes.POINTER(_State), ctypes.c_int64, ctypes.c_void_p, ctypes.c_int64, ctypes.c_void_p]

    def move(n=2, rows=4096, count=1, **change):
        st = _State(**dict(dict(src=4096, dst=4096, row_bytes=16, num_rows=3), **change))
        return r(ctypes.byref(st), count, rows, n, None)

    assert r(None, 1, 4096, 1, None) == -1 and move(n=-1) == -1 and move(rows=None) == -1 and move(src=None) == -1
    assert move(dst=None) == -1 and move(row_bytes=-1) == -1 and move(num_rows=-1) == -1 and move(num_rows=2 ** 31) == -2
    assert move(n=2 ** 31) == -2 and move(n=2 ** 20, row_bytes=2 ** 30) == -2 and move(n=0, rows=None) == 0
    assert move(row_bytes=0, src=None, dst=None) == 0 and r(None, 0, None, 0, None) == 0


def test_fake_kernels():
    x, s = torch.empty(6, 50, device="meta"), torch.empty(2, 3, device="meta")
    e = torch.empty(2, 3, dtype=torch.bool, device="meta")
    out = ops.beam_select(x, s, 5)
    assert [o.shape for o in out] == [(2, 5)] * 3 and [o.dtype for o in out] == [F, torch.int32, torch.int64]
    assert ops.beam_select(x, s, None, e)[3].shape == (2, 3)
    assert ops.beam_reorder([x], torch.empty(2, 4, dtype=torch.int32, device="meta"))[0].shape == (8, 50)


@pytest.mark.gpu
def test_opcheck():
    utils = ("test_schema", "test_faketensor", "test_aot_dispatch_dynamic")
    torch.library.opcheck(torch.ops.pulsar.beam_select.default, tuple(_good().values()), test_utils=utils)
    torch.library.opcheck(torch.ops.pulsar.beam_reorder.default,
                          ([torch.zeros(3, 4, device=DEV)], torch.zeros(2, dtype=torch.int32, device=DEV)), test_utils=utils)


@pytest.mark.gpu
@pytest.mark.parametrize("batch,beams,vocab,width", [(1, 1, 40000, 32), (3, 7, 5000, 5), (1, 32, 9, 32)])
def test_writes_stay_in_the_outputs_and_the_workspace(batch, beams, vocab, width):
    x, s = _logits(batch * beams, vocab, B, 1).to(DEV), _scores(batch, beams, 1).to(DEV)
    want = ops.beam_select(x, s, width)
    lib = pulsar_amd.capi()
    lib.pw4_beam_select_workspace_size.argtypes = [ctypes.c_int64] * 4
    lib.pw4_beam_select_workspace_size.restype = ctypes.c_size_t
    n = lib.pw4_beam_select_workspace_size(batch, beams, vocab, width)
    ws = torch.full((n + 256,), 0x5a, dtype=torch.uint8, device=DEV)
    out = torch.full((batch * width + 16,), 7.0, device=DEV)
    rows = torch.full((batch * width + 16,), 7, dtype=torch.int32, device=DEV)
    tokens = torch.full((batch * width + 16,), 7, dtype=torch.int64, device=DEV)
    f = lib.pw4_beam_select
    f.argtypes = ([ctypes.c_void_p, ctypes.c_int] + [ctypes.c_int64] * 4 + [ctypes.c_void_p] * 2 + [ctypes.c_int64] * 2
                  + [ctypes.c_void_p] * 5 + [ctypes.c_size_t, ctypes.c_void_p])
    torch.cuda.synchronize()
    assert f(x.data_ptr(), 1, batch, beams, vocab, vocab, s.data_ptr(), None, 0, width, out.data_ptr(), rows.data_ptr(),
             tokens.data_ptr(), None, ws.data_ptr(), n, None) == 0
    torch.cuda.synchronize()
    for a, b in zip((out, rows, tokens), want):
        assert torch.equal(a[:-16].view(b.shape), b) and bool((a[-16:] == 7).all())
    assert bool((ws[n:] == 0x5a).all())


@pytest.mark.gpu
def test_reorder_of_more_rows_than_a_launch_has_workgroups():
    n = (1 << 24) + 3
    rows = torch.arange(n, dtype=torch.int32, device=DEV).remainder(7) - 1
    state = torch.arange(5, dtype=torch.int16, device=DEV) + 100
    out, = ops.beam_reorder([state], rows)
    assert torch.equal(out, torch.where((rows >= 0) & (rows < 5), state[rows.clamp(0, 4).long()], 0))


@pytest.mark.gpu
def test_reorder_of_views_that_stand_for_other_values():
    """Conjugate and negative views hold other numbers than their memory does."""
    x = torch.randn(5, 3, dtype=torch.complex64, generator=gen(1)).to(DEV)
    rows = torch.tensor([4, 0, 0], dtype=torch.int32, device=DEV)
    got = ops.beam_reorder([x.conj(), x.conj().imag, x], rows)
    for g, w in zip(got, (x.conj(), x.conj().imag, x)):
        assert torch.equal(g, w[rows.long()])
