"""The clear decoder's plain entry points on tensors that require gradients: no
result without a graph passes for one with it."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

import clear_model as cm  # noqa: E402


def _leaf(*shape):
    return torch.zeros(*shape, dtype=torch.bfloat16, requires_grad=True)


def _calls():
    q, k, h, w = _leaf(1, 2, 4, 64), _leaf(1, 2, 2, 64), _leaf(3, 8), _leaf(5, 8)
    plain, table = torch.zeros(1, 2, 2, 64).bfloat16(), cm.RopeTable(64)
    places, y = torch.zeros(2, dtype=torch.int32), torch.zeros(3, dtype=torch.int64)
    return [
        ("apply_rope", lambda: cm.rope(table, q, positions=places)),
        ("apply_rope", lambda: cm.rope(table, plain, k, positions=places)),
        ("attention", lambda: cm.attention_forward(q, plain, plain, causal=True)),
        ("attention", lambda: cm.attention_forward(plain, k, plain, causal=True)),
        ("attention", lambda: cm.attention_forward(plain, plain, k, causal=True)),
        ("linear_cross_entropy", lambda: cm.linear_cross_entropy_forward(h, w.detach(), y)),
        ("linear_cross_entropy", lambda: cm.linear_cross_entropy_forward(h.detach(), w, y)),
    ]


@pytest.mark.parametrize("i", range(7))
def test_gradients_are_refused_not_left_out(i):
    name, call = _calls()[i]
    with pytest.raises(ValueError, match=rf"use {name} "):
        call()
    # without a graph to be left out of, the next check is the device's
    with torch.no_grad(), pytest.raises(ValueError, match="GPU"):
        call()


def test_scores_of_a_head_that_is_being_adapted(monkeypatch):
    from clear_model import decoder as dec

    seen = []
    monkeypatch.setattr(dec, "linear_cross_entropy_forward",
                        lambda x, w, t, **kw: seen.append(torch.is_grad_enabled()) or (x.sum(), None))
    z = lambda *s: torch.zeros(*s).bfloat16()  # noqa: E731
    layer = dict(q=z(8, 8), k=z(8, 8), v=z(8, 8), o=z(8, 8), gate=z(8, 8), up=z(8, 8), down=z(8, 8))
    model = cm.ClearDecoder([layer], z(5, 8), _leaf(5, 8), heads=1, kv_heads=1, head_dim=8)
    model.score(torch.zeros(3, 8), torch.zeros(3, dtype=torch.int64))
    assert seen == [False]
