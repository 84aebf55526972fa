"""Borders of what the clear decoder's attention takes, on the host alone."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from clear_model import _native  # noqa: E402
from clear_model.attention import _checked  # noqa: E402
from test_clear_model import _attention_args, _Fake  # noqa: E402


@pytest.mark.parametrize("scale", [1e-46, 1e-39])
def test_scales_below_fp32(scale):
    """In fp32 such a scale is 0 or loses its bits, and a hidden key's -inf times 0
    is NaN."""
    with pytest.raises(ValueError, match="scale"):
        _native.check(_native.lib.clear_attention_forward(_attention_args(scale=scale), None))
    x = _Fake(torch.zeros(1, 2, 4, 64, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="scale"):
        _checked(x, x, x, None, None, scale)


def test_the_smallest_scale():
    n = _native.query(_native.lib.clear_attention_workspace, _attention_args(scale=1.2e-38), False)
    assert n == 0
    x = _Fake(torch.zeros(1, 2, 4, 64, dtype=torch.bfloat16))
    assert _checked(x, x, x, None, None, 1.2e-38)[2] == 1.2e-38


@pytest.mark.parametrize("n,m,fits", [(1 << 30, 1 << 30, False), (1 << 30, (1 << 30) - 256, True)])
def test_places_of_queries_have_31_bits(n, m, fits):
    """A query's last visible key, its place plus the start (at most the keys), is
    computed in 32 bits, up to a whole tile beyond the last query."""
    args = _attention_args(n=n, m=m, h=1, kv=1, d=8, causal=1)
    if fits:
        assert _native.query(_native.lib.clear_attention_workspace, args, True) > 0
        return
    for backward in (False, True):
        with pytest.raises(ValueError, match="large"):
            _native.query(_native.lib.clear_attention_workspace, args, backward)
