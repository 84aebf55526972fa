"""The clear decoder's host logic on the CPU, with plain stand-ins for its operators:
what a cache holds and refuses, and what `score` hands to the loss."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

import clear_model as cm  # noqa: E402
from clear_model import decoder as dec  # noqa: E402

H, KV, HD, D, V, L = 4, 2, 8, 32, 23, 2


@pytest.fixture
def model(monkeypatch):
    """A decoder whose operators run on the CPU: no turn, and the mean of the
    values that a sequence's length leaves visible."""
    def attend(q, k, v, *, causal, kv_lens=None):
        assert int(kv_lens.max()) <= k.shape[1]
        out = [v[b, :max(int(n), 1)].mean(0) for b, n in enumerate(kv_lens)]
        out = torch.stack(out).repeat_interleave(H // KV, 1)
        return out[:, None].expand(q.shape).contiguous(), None

    monkeypatch.setattr(dec, "rope", lambda table, q, k, positions: (q, k))
    monkeypatch.setattr(dec, "attention_forward", attend)
    g = torch.Generator().manual_seed(0)
    draw = lambda *s: torch.randn(*s, generator=g).mul_(0.2).bfloat16()  # noqa: E731
    layers = [dict(q=draw(H * HD, D), k=draw(KV * HD, D), v=draw(KV * HD, D), o=draw(D, H * HD),
                   gate=draw(D, D), up=draw(D, D), down=draw(D, D)) for _ in range(L)]
    return cm.ClearDecoder(layers, draw(V, D), draw(V, D), heads=H, kv_heads=KV, head_dim=HD)


def _ids(b, t):
    return torch.arange(b * t).reshape(b, t) % V


def _lens(*x):
    return torch.tensor(x, dtype=torch.int32)


def test_a_full_cache_takes_no_more_tokens(model):
    cache = model.cache(2, 4)
    model.prefill(_ids(2, 3), cache)
    model.decode(_ids(2, 1)[:, 0], cache)
    held = [x.clone() for x in cache.keys + cache.values]
    with pytest.raises(ValueError, match="room"):
        model.decode(_ids(2, 1)[:, 0], cache)
    assert cache.lens.tolist() == [4, 4]
    assert all(torch.equal(x, y) for x, y in zip(held, cache.keys + cache.values))


def test_short_prompts_leave_their_room(model):
    """The padded length is not what counts: every place of the longest can be used."""
    cache = model.cache(2, 6)
    model.prefill(_ids(2, 5), cache, _lens(2, 3))
    for _ in range(3):
        model.decode(_ids(2, 1)[:, 0], cache)
    assert cache.lens.tolist() == [5, 6]
    with pytest.raises(ValueError, match="room"):
        model.decode(_ids(2, 1)[:, 0], cache)
    # an emptied cache is as good as new
    model.prefill(_ids(2, 2), cache)
    model.decode(_ids(2, 1)[:, 0], cache)
    assert cache.lens.tolist() == [3, 3]


def test_a_cache_that_the_caller_filled(model):
    new = model.cache(2, 4)
    cache = cm.ClearCache(new.keys, new.values, _lens(1, 3))
    model.decode(_ids(2, 1)[:, 0], cache)
    assert cache.lens.tolist() == [2, 4]
    with pytest.raises(ValueError, match="room"):
        model.decode(_ids(2, 1)[:, 0], cache)


@pytest.mark.parametrize("lens", [(9, 1), (-3, 4), (4, 2 ** 31 - 1)])
def test_lengths_that_the_host_does_not_see_stay_inside(model, lens):
    """As in a replayed graph: whatever the lengths say, places are in the cache."""
    cache = model.cache(2, 4)
    cache.lens.copy_(_lens(*lens))
    cache.bound = 0
    model.decode(_ids(2, 1)[:, 0], cache)
    assert all(1 <= n <= 4 for n in cache.lens.tolist())


@pytest.mark.parametrize("lens", [(9, 1), (-1, 2)])
def test_prompt_lengths_are_within_the_prompts(model, lens):
    cache = model.cache(2, 16)
    model.prefill(_ids(2, 3), cache, _lens(*lens))
    assert cache.lens.tolist() == [min(max(n, 0), 3) for n in lens]


def test_prefill_refusals(model):
    with pytest.raises(ValueError, match="lens"):
        model.prefill(_ids(2, 3), model.cache(2, 8), _lens(1, 2, 3))
    with pytest.raises(ValueError, match="lens"):
        model.prefill(_ids(2, 3), model.cache(2, 8), _lens(1, 2).long())
    with pytest.raises(ValueError, match="sequences"):
        model.prefill(_ids(1, 3), model.cache(2, 8))
    with pytest.raises(ValueError, match="sequences"):
        model.decode(_ids(1, 1)[:, 0], model.cache(2, 8))
    with pytest.raises(ValueError, match="ids"):
        model.prefill(_ids(2, 3)[0], model.cache(2, 8))


@pytest.mark.parametrize("t", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("norm", [False, True])
def test_scored_states_are_rounded_once(model, monkeypatch, t, norm):
    """Decrypted states come in fp64, some far beyond fp16: what the loss gets is
    the normed state in 64 bits, off by half a step of the type and fp32's share."""
    got = []
    monkeypatch.setattr(dec, "linear_cross_entropy_forward",
                        lambda x, *a, **kw: got.append(x) or (None, None))
    model.lm_head = model.lm_head.to(t)
    g = torch.Generator().manual_seed(1)
    h = torch.randn(50, D, generator=g, dtype=torch.float64)
    h[:, 3] *= 3e5
    w = torch.rand(D, generator=g) + 0.5 if norm else None
    model.final_norm = w
    model.score(h, torch.zeros(50, dtype=torch.int64))
    model.score(h.numpy(), torch.zeros(50, dtype=torch.int64))
    want = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + 1e-5)
    if norm:
        want = want * w.double()
    u, tiny = torch.finfo(t).eps / 2, torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2
    # the state to fp32, the mean of D squares and its root, two products
    bound = want.abs() * (u + (D / 2 + 8) * 2.0 ** -24) + tiny
    for x in got:
        assert x.dtype is t and bool(((x.double() - want).abs() <= bound).all())
    assert len(got) == 2
