"""How far the inputs of test_paged_append.py's 4-bit cases stand from the borders between codes."""

import pytest
import torch

from test_paged_append import H, B, SHAPES, _case, rotate_ref

BORDERS = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], dtype=torch.float64)


def _clear_of_borders(x, rot, fp16):
    """The least distance, relative, of a rotated element from the borders of its block's codes, and of a block's
    largest magnitude, where that is a rotated element, from the borders of its exponent."""
    b = x.unflatten(-1, (-1, 32)).abs()
    mant, exp = torch.frexp(b.amax(-1))
    e = (exp - 3 + (mant >= 0.875).int()).clamp(-127, 13 if fp16 else 125)
    m = b / torch.ldexp(torch.ones_like(mant), e)[..., None]
    codes = ((m[..., None] - BORDERS).abs() / BORDERS).amin(-1).flatten(-2)[..., :rot]
    first = 32 * torch.arange(b.shape[-2])
    top = torch.where(b.argmax(-1) + first < rot, (mant - 0.875).abs() / 0.875, 1.0)
    return min(float(codes.amin()), float(top.amin()))


@pytest.mark.parametrize("dtype", [H, B])
@pytest.mark.parametrize("t,hq,hkv,dim,rot", SHAPES)
def test_rotated_inputs_stand_clear_of_borders(t, hq, hkv, dim, rot, dtype):
    """The inputs of test_append_4_bits: further than 2^-22 from any border, so their codes do not hang on how an
    element's sum is rounded to fp32."""
    _, k, _, positions, rope = _case(t, hq, hkv, dim, rot, dtype, t + dim)
    for interleaved in (False, True):
        assert _clear_of_borders(rotate_ref(k, rope, positions, interleaved)[0], rot, dtype == H) > 2.0 ** -22
