"""The clear decoder's cache on the device: tokens up to the last place, and a
captured step that is replayed beyond it."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from test_gpu_clear_decoder import BOUND, HD, KV, L, V, _decoder, _rel  # noqa: E402

pytestmark = pytest.mark.gpu


def _guarded(model, batch, capacity):
    """A cache in the middle of larger buffers."""
    import clear_model as cm

    whole = [torch.full((batch + 2, capacity, KV, HD), 7.0, dtype=torch.bfloat16, device="cuda")
             for _ in range(2 * L)]
    parts = [x[1:-1] for x in whole]
    lens = torch.zeros(batch, dtype=torch.int32, device="cuda")
    return whole, cm.ClearCache(parts[:L], parts[L:], lens, 0)


def _untouched(whole):
    return all(bool((x[0] == 7.0).all()) and bool((x[-1] == 7.0).all()) for x in whole)


def test_every_place_of_a_cache():
    """Generating up to the last place matches the whole sequence; then it ends."""
    model = _decoder(5)
    ids = torch.randint(0, V, (2, 12), device="cuda")
    whole, cache = _guarded(model, 2, 12)
    lens = torch.tensor([8, 3], dtype=torch.int32, device="cuda")
    model.prefill(ids[:, :9], cache, lens)
    rows = torch.arange(2, device="cuda")
    for step in range(4):
        y = model.decode(ids[rows, lens.long() + step], cache)
    assert cache.lens.tolist() == [12, 7]
    with torch.no_grad():
        want = model.logits(model.hidden(ids))
    for b, n in enumerate((12, 7)):
        assert _rel(y[b].double().cpu().numpy(), want[b, n - 1].double().cpu().numpy()) <= 2 * BOUND
    with pytest.raises(ValueError, match="room"):
        model.decode(ids[:, 0], cache)
    assert _untouched(whole)


def test_prompt_lengths_beyond_the_prompts():
    model = _decoder(6)
    ids = torch.randint(0, V, (3, 5), device="cuda")
    whole, cache = _guarded(model, 3, 9)
    y = model.prefill(ids, cache, torch.tensor([2 ** 31 - 1, -4, 5], dtype=torch.int32, device="cuda"))
    assert cache.lens.tolist() == [5, 0, 5] and bool(torch.isfinite(y).all())
    assert _untouched(whole)


def test_replays_stay_inside_the_cache():
    model = _decoder(7)
    ids = torch.randint(0, V, (2, 3), device="cuda")
    whole, cache = _guarded(model, 2, 6)
    token = ids[:, 0].contiguous()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        model.prefill(ids, cache)
        model.decode(token, cache)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        logits = model.decode(token, cache)
    model.prefill(ids, cache)
    for step in range(3):
        graph.replay()
        got = logits.clone()
        torch.cuda.synchronize()
        assert cache.lens.tolist() == [4 + step, 4 + step]
        with torch.no_grad():
            seen = torch.cat([ids] + [token[:, None]] * (step + 1), 1)
            want = model.logits(model.hidden(seen)[:, -1])
        for b in range(2):
            assert _rel(got[b].double().cpu().numpy(), want[b].double().cpu().numpy()) <= 2 * BOUND
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert cache.lens.tolist() == [6, 6] and _untouched(whole)
