"""The clear decoder's vocabulary loss against 64-bit plain forms on every kind of
tile that its plan has, on both sides of each of the plan's borders."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from test_gpu_clear_loss import _check, _inputs  # noqa: E402

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


@pytest.mark.parametrize("t", [BF16, FP16])
@pytest.mark.parametrize("n,v,d,ignored", [
    # up to 128 tokens: 255 tiles of 128 classes (taken in halves) and 256
    (128, 32640, 72, 0.0), (128, 32641, 72, 0.2), (5, 40001, 264, 0.2), (1, 32769, 520, 0.0),
    # one token more: a second column of tiles, and the backward pass's list
    (129, 33000, 72, 0.2), (128, 33000, 72, 0.2),
    # without a list: fewer than 256 tiles, more, and the last count of them that
    # may hold 2^33 products
    (600, 3001, 264, 0.3), (600, 9001, 264, 0.3), (256, 32768, 520, 0.1),
    # from there on with a list, 128 classes a tile
    (256, 32769, 520, 0.1), (500, 20000, 512, 0.3), (400, 30001, 264, 0.3),
    # 255 tiles of 256 x 256 are too few, 256 are enough
    (200, 65280, 264, 0.3), (200, 65281, 264, 0.3),
    # no list, and a vocabulary of more than one piece in the backward pass
    (128, 1060001, 8, 0.2),
])
def test_every_kind_of_tile(n, v, d, ignored, t):
    x, w, y, dl = _inputs(n, v, d, t, ignored, seed=30, scale=1024.0 if t == FP16 else 1.0)
    _check(x, w, y, dl)


@pytest.mark.parametrize("t", [BF16, FP16])
@pytest.mark.parametrize("n,v,d,ignored", [(1 << 14, 300, 64, 0.4), (40001, 300, 64, 0.4),
                                           (70000, 129, 72, 0.9), (131072, 130, 8, 0.0)])
def test_lists_of_many_tokens(n, v, d, ignored, t):
    """Blocks of 16, 39, 68 and 128 tokens, taken 64 at a time."""
    x, w, y, dl = _inputs(n, v, d, t, ignored, seed=31, scale=1024.0 if t == FP16 else 1.0)
    _check(x, w, y, dl)
