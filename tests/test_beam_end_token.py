"""beam_select's end_token: a token of the vocabulary, or -1 for none."""

import ctypes

import pytest
import torch

import pulsar_amd
from paged_case import DEV, gen
from pulsar_amd import ops


def _inputs():
    logits = torch.randn(6, 50, generator=gen(1)).to(DEV)
    scores = -torch.rand(2, 3, generator=gen(2)).to(DEV)
    ended = torch.tensor([[True, False, True], [False, False, True]], device=DEV)
    return logits, scores, ended


@pytest.mark.gpu
@pytest.mark.parametrize("end", [-2, 50, 51, 2 ** 31, -2 ** 40, 2 ** 62])
def test_tokens_outside_the_vocabulary_are_refused(end):
    logits, scores, ended = _inputs()
    for e in (ended, torch.zeros_like(ended)):
        with pytest.raises(RuntimeError, match="end_token"):
            ops.beam_select(logits, scores, None, e, end)
    # without `ended` it is not used
    want = ops.beam_select(logits, scores)
    for a, b in zip(want, ops.beam_select(logits, scores, None, None, end)):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_no_end_token():
    """-1: beams that have ended go on with it, for the caller to replace, and no beam ends by its token."""
    logits, scores, ended = _inputs()
    out = ops.beam_select(logits, scores, None, ended)
    was = ended.view(-1)[out[1].long()]
    assert torch.equal(out[3], was) and bool(was.any()) and not bool(was.all())
    assert bool((out[2][was] == -1).all()) and bool((out[2][~was] >= 0).all())
    for end in (0, 49):
        got = ops.beam_select(logits, scores, None, ended, end)
        assert torch.equal(got[0], out[0]) and torch.equal(got[1], out[1])
        assert torch.equal(got[2], torch.where(was, end, out[2])) and torch.equal(got[3], was | (got[2] == end))


def test_the_c_entry_refuses_before_any_launch():
    f = pulsar_amd.capi().pw4_beam_select
    f.argtypes = ([ctypes.c_void_p, ctypes.c_int] + [ctypes.c_int64] * 4 + [ctypes.c_void_p] * 2 + [ctypes.c_int64] * 2
                  + [ctypes.c_void_p] * 5 + [ctypes.c_size_t, ctypes.c_void_p])

    def call(end, ended):  # a workspace of no bytes: -3 where all else is right
        return f(4096, 1, 2, 3, 50, 50, 4096, ended, end, 3, 4096, 4096, 4096, None, 4096, 0, None)

    for end in (-2, 50, 2 ** 31, -2 ** 40):
        assert call(end, 4096) == -1 and call(end, None) == -3
    for end in (-1, 0, 49):
        assert call(end, 4096) == -3 and call(end, None) == -3
