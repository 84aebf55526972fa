"""Grouped attention of the clear decoder on values at the types' borders: NaN and
infinities that a query sees, long tails of small probabilities, and score
gradients beyond fp16's largest number."""

from __future__ import annotations

import math

import pytest

torch = pytest.importorskip("torch")

import clear_plain as plain  # noqa: E402

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


def _inputs(b, n, m, h, kv, d, t, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randn(b, x, y, d, generator=g, device="cuda").to(t)
            for x, y in ((n, h), (m, kv), (m, kv), (n, h))]


# one block and several for packed queries, then for whole tiles of them; the
# keys [a, b) are all that one wave, or one block, takes
SEEN = [(1, 100, 4, 2, 32, 64), (1, 3000, 4, 2, 256, 512), (200, 300, 4, 2, 64, 128),
        (1100, 1600, 1, 1, 320, 640), (3, 64, 4, 2, 0, 64), (200, 64, 4, 2, 0, 64)]


@pytest.mark.parametrize("t", [BF16, FP16])
@pytest.mark.parametrize("n,m,h,kv,a,b", SEEN)
def test_nan_that_a_query_sees_is_in_its_lse(n, m, h, kv, a, b, t):
    """-inf is for queries that see nothing."""
    import clear_model as cm

    q, k, v, _ = _inputs(2, n, m, h, kv, 64, t, 1)
    val, err = plain.attention(q, k, v, False)
    k[1, a:b] = float("nan")
    q[0, n // 2, h - 1] = float("nan")
    out, lse = cm.attention_forward(q, k, v, causal=False)
    assert bool(torch.isnan(lse[1]).all()) and bool(torch.isnan(out[1]).all())
    assert bool(torch.isnan(lse[0, h - 1, n // 2])) and bool(torch.isnan(out[0, n // 2, h - 1]).all())
    keep = torch.ones(n, h, dtype=torch.bool, device="cuda")
    keep[n // 2, h - 1] = False
    plain.assert_within(out[0][keep], val[0][0][keep], err[0][0][keep], "out")
    plain.assert_within(lse[0].t()[keep], val[1][0].t()[keep], err[1][0].t()[keep], "lse")


@pytest.mark.parametrize("t", [BF16, FP16])
@pytest.mark.parametrize("n,m,h,kv,a,b", SEEN[:4])
def test_a_score_of_minus_infinity_takes_its_key_out(n, m, h, kv, a, b, t):
    import clear_model as cm

    q, k, v, _ = _inputs(1, n, m, h, kv, 64, t, 2)
    q[..., 0] = 1.0
    keep = torch.ones(m, dtype=torch.bool, device="cuda")
    keep[a:b], keep[-1] = False, False
    val, err = plain.attention(q, k[:, keep], v[:, keep], False)
    k[:, ~keep, :, 0] = float("-inf")
    out, lse = cm.attention_forward(q, k, v, causal=False)
    plain.assert_within(out, val[0], err[0], "out")
    plain.assert_within(lse, val[1], err[1], "lse")


@pytest.mark.parametrize("n,m", [(5, 100), (200, 300), (200, 100)])
def test_nothing_but_scores_of_minus_infinity(n, m):
    """Finite operands whose products leave fp32: an output of 0, lse = -inf, and no
    part in any gradient."""
    import clear_model as cm

    q, k, v, do = _inputs(1, n, m, 2, 1, 64, BF16, 5)
    q.zero_(), k.fill_(1e20)
    q[0, 2, 1] = -1e20
    out, lse = cm.attention_forward(q, k, v, causal=False)
    dq, dk, dv = cm.attention_backward(do, q, k, v, out, lse, causal=False)
    assert float(out[0, 2, 1].abs().max()) == 0.0 and float(lse[0, 1, 2]) == float("-inf")
    assert float(dq[0, 2, 1].abs().max()) == 0.0 and bool(torch.isfinite(dq).all())
    assert float(dk.abs().max()) == 0.0  # the others' queries are 0
    rest = do.clone()
    rest[0, 2, 1] = 0.0
    val, err = plain.attention(torch.zeros_like(q), k, v, False, dout=rest)
    plain.assert_within(dv, val[4], err[4], "dv")


@pytest.mark.parametrize("t", [BF16, FP16])
@pytest.mark.parametrize("n,h,m,first", [(1, 4, 200000, True), (1, 4, 200000, False),
                                         (200, 1, 40000, True), (200, 1, 40000, False),
                                         (4096, 8, 40000, True), (4096, 8, 40000, False)])
def test_a_long_tail_of_small_probabilities(n, h, m, first, t):
    """One key with nearly all of the mass in front of or behind many with 2^-26 of
    it each: the values of the many are all that the output holds.

    Each probability is rounded once to the type, which keeps 2^-26 of a row's
    largest within half a step u; sums are fp32."""
    import clear_model as cm

    d = 64
    q = torch.ones(1, n, h, d, dtype=t, device="cuda")
    k, v = torch.zeros(1, m, 1, d, dtype=t, device="cuda"), torch.ones(1, m, 1, d, dtype=t, device="cuda")
    at = 0 if first else m - 1
    k[:, at], v[:, at] = 2.25, 0.0  # a score of 18
    out, lse = cm.attention_forward(q, k, v, causal=False)
    tail = (m - 1) * math.exp(-18.0)
    want, u = tail / (1.0 + tail), plain.half_step(t)
    # a probability's rounding and the result's; the power's argument, and a sum
    # of m equal numbers in fp32
    bound = want * (2 * u + (64 + m) * plain.F32)
    assert float((out.double() - want).abs().max()) <= bound
    assert float((lse.double() - math.log(1.0 + tail) - 18.0).abs().max()) <= (80 + m) * plain.F32


@pytest.mark.parametrize("b,n,m,h,kv,d,causal", [
    (1, 90, 100, 4, 2, 64, False), (1, 70, 128, 4, 2, 128, False), (1, 90, 300, 4, 2, 64, True),
    (2, 300, 633, 4, 2, 80, True), (1, 1031, 2400, 4, 1, 128, True), (1, 203, 403, 4, 4, 40, False),
])
def test_score_gradients_beyond_fp16(b, n, m, h, kv, d, causal):
    """Scores' gradients above 65504 whose sums, times the scale, are within it: in
    some rows and keys, beside others of every smaller size."""
    import clear_model as cm

    q, k, v, do = _inputs(b, n, m, h, kv, d, FP16, 3)
    scale = 0.004
    v = (v.float() * (4e4 * m / (1000.0 * math.sqrt(d)))).to(FP16)
    do = (do.float() * torch.logspace(-1, 3, n, device="cuda")[None, :, None, None]).to(FP16)
    val, err = plain.attention(q, k, v, causal, scale=scale, dout=do)
    # the largest score gradient of the first sequence's first head
    s = (q[0, :, 0].double() @ k[0, :, 0].double().t()) * scale
    s = s.masked_fill(~plain.visible(1, n, m, causal, None, None, "cuda")[0], float("-inf"))
    ds = torch.softmax(s, 1) * (do[0, :, 0].double() @ v[0, :, 0].double().t()
                                - (do[0, :, 0].double() * val[0][0, :, 0]).sum(1, keepdim=True))
    assert float(ds.abs().max()) > 65504.0
    assert all(float(x.abs().max()) < 65504.0 for x in val[2:])
    out, lse = cm.attention_forward(q, k, v, causal=causal, scale=scale)
    grads = cm.attention_backward(do, q, k, v, out, lse, causal=causal, scale=scale)
    for name, got, y, e in zip(("out", "lse", "dq", "dk", "dv"), (out, lse) + grads, val, err):
        plain.assert_within(got, y, e, name)


@pytest.mark.parametrize("n,m,h,kv,d", [(30, 40, 4, 2, 64), (130, 200, 2, 2, 128)])
def test_the_largest_score_gradients_of_fp16(n, m, h, kv, d):
    """Operands at the end of fp16, and a scale that brings the results back."""
    import clear_model as cm

    q, k, v, do = _inputs(1, n, m, h, kv, d, FP16, 4)
    v, do = (torch.sign(x) * 6e4 for x in (v, do))
    do = do * torch.logspace(-4, 0, n, device="cuda")[None, :, None, None]
    v, do, scale = v.to(FP16), do.to(FP16), 1e-6
    val, err = plain.attention(q, k, v, False, scale=scale, dout=do)
    # v - out at the flat probabilities, of the last and largest row
    far = do[0, -1, 0].double() @ (v[0, :, 0].double() - val[0][0, -1, 0]).t() / m
    assert float(far.abs().max()) > 65504.0 * 2 ** 13
    assert all(float(x.abs().max()) < 65504.0 for x in val[2:])
    out, lse = cm.attention_forward(q, k, v, causal=False, scale=scale)
    grads = cm.attention_backward(do, q, k, v, out, lse, causal=False, scale=scale)
    for name, got, y, e in zip(("dq", "dk", "dv"), grads, val[2:], err[2:]):
        plain.assert_within(got, y, e, name)
