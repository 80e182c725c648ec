"""Linear attention where numbers come to the ends of their ranges: decays that leave next to nothing, large values beside small ones, and what is not
finite behind them (linear_half_oracle.py has half precision's bounds)."""
import pytest
import torch

from tests.linear_half_oracle import linear_backward, linear_forward
from tests.linear_oracle import check
from tests.test_gpu_linear_attention import CASES, GRADS, IDS, backward, case, forward, inputs
from tests.util import DTYPE_IDS, DTYPES, randn

pytestmark = pytest.mark.gpu
STRONG = [-40.0, -70.0, -75.0, -78.0, -80.0, -82.0, -83.0, -84.0, -85.0, -86.0, -87.0]


@pytest.mark.parametrize("dtype", DTYPES, ids=DTYPE_IDS)
@pytest.mark.parametrize("decay", STRONG, ids=str)
def test_scores_that_have_all_but_decayed(device, decay, dtype):
    """Tokens 32 to 63 of a chunk see those before them with a weight of 2^-58 to 2^-126, beside values and gradients of thousands."""
    c = case(2, 130, 4, 2, 64, decay=[decay])
    q, k, v, dout, log_decay, before, d_after = inputs(c, dtype, device)
    v, dout = v * 1000, dout * 100
    want = {**linear_forward(q, k, v, log_decay, before, 0.0), **linear_backward(q, k, v, log_decay, before, dout, d_after, 0.0)}
    check(forward(c, q, k, v, log_decay, before)[0], want["out"], "out")
    for name, got in zip(GRADS[:3], backward(c, q, k, v, dout, log_decay, before, d_after)):
        check(got, want[name], name)
    there = tuple((randn(t.shape, dtype, 50 + i) * 1000).to(device) for i, t in enumerate((q, k, v)))
    grads = backward(c, q, k, v, dout, log_decay, before, d_after, tuple(t.clone() for t in there) + (torch.zeros_like(before),), True)
    step = max(torch.finfo(dtype).eps / 2, 2.0 ** -24)
    for name, got, was in zip(GRADS[:3], grads, there):
        want[name].value += was.double()
        want[name].error += step * (was.double().abs() + want[name].value.abs())
        check(got, want[name], name)


@pytest.mark.parametrize("decay", [-60.0, -80.0, -82.0, -84.0, -86.0])
def test_equal_values_under_strong_decays(device, decay):
    """Keys and queries of ones, values of 512 in half precision: every output is 8 x 512, to a half step of the score, the values' parts and the result."""
    c = case(1, 200, 2, 1, 64, decay=[decay])
    q, k, v = (torch.full((1, 200, heads, 64), value, dtype=torch.float16, device=device) for heads, value in ((2, 1.0), (1, 1.0), (1, 512.0)))
    out, after = forward(c, q, k, v, torch.tensor([decay], device=device), None)
    assert (out == 4096).all() and (after == 512).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=DTYPE_IDS)
@pytest.mark.parametrize("b,t", [(2, 60), (1, 700)], ids=str)
@pytest.mark.parametrize("decay", [-15.0, -30.0, -50.0], ids=str)
def test_stored_matrices_of_small_weights(device, decay, b, t, dtype):
    """The first state's gradient, of which g to the first power is the largest weight."""
    c = case(b, t, 4, 2, 64, decay=[decay])
    q, k, v, dout, log_decay, before, _ = inputs(c, dtype, device)
    check(backward(c, q, k, v, dout, log_decay, before, None)[3], linear_backward(q, k, v, log_decay, before, dout, None, 0.0)["d_before"], "d_before")


@pytest.mark.parametrize("dtype", DTYPES, ids=DTYPE_IDS)
@pytest.mark.parametrize("b,t", [(2, 60), (1, 700)], ids=str)
@pytest.mark.parametrize("decay", [-0.5, -1.0], ids=str)
def test_stored_matrices_behind_zeros(device, decay, b, t, dtype):
    """A sequence whose last values are zeros, as a padded one's are: what its tokens leave has decayed over all of them."""
    c = case(b, t, 4, 2, 64, states=False, decay=[decay])
    q, k, v, _, log_decay, _, _ = inputs(c, dtype, device)
    v[:, -50:] = 0
    check(forward(c, q, k, v, log_decay, None)[1], linear_forward(q, k, v, log_decay, None, 0.0)["after"], "after")


@pytest.mark.parametrize("t", [60, 700])
def test_stored_matrices_of_uneven_heads(device, t):
    """Heads of a group whose largest weighted gradients lie 2^130 apart: the larger ones keep their range where the small ones are enlarged."""
    c = case(1, t, 2, 1, 64, states=False, scale=64.0, decay=[-1.1])
    q, k, v, dout, log_decay, _, _ = inputs(c, torch.float16, device)
    q, dout = q * 4000, dout * 4000
    dout[:, :, 1] = 0
    dout[:, 58:60, 1] = 2.0 ** -24
    before = torch.zeros((1, 1, 64, 64), device=device)
    check(backward(c, q, k, v, dout, log_decay, before, None)[3], linear_backward(q, k, v, log_decay, before, dout, None, 64.0)["d_before"], "d_before")


@pytest.mark.parametrize("dtype", DTYPES, ids=DTYPE_IDS)
@pytest.mark.parametrize("bad", [float("nan"), float("inf")], ids=str)
@pytest.mark.parametrize("decay", [-3.0, -30.0, -87.5, -float("inf")], ids=str)
@pytest.mark.parametrize("t", [150, 700])
def test_what_is_not_finite_and_has_decayed(device, t, decay, bad, dtype):
    """It reaches every token behind it (backward: in front of it) and the state, also those whose weight for it rounds to nothing, and no other token."""
    c = case(1, t, 2, 1, 64, decay=[decay])
    q, k, v, dout, log_decay, before, d_after = inputs(c, dtype, device)
    want = {**linear_forward(q, k, v, log_decay, before, 0.0), **linear_backward(q, k, v, log_decay, before, dout, d_after, 0.0)}

    def spoilt(got, name, at):
        m = torch.zeros_like(got, dtype=torch.bool)
        m[at] = True
        assert not torch.isfinite(got[m]).any(), name
        assert bool(((got.double() - want[name].value).abs() <= want[name].error)[~m].all()), name

    for t0 in (3, 40, 70):
        for at, of_out, of_state in (((0, t0, 0, 5), (0, slice(t0, None)), (0, 0, 5)), ((0, t0, 0, 5), (0, slice(t0, None), slice(None), 5), (0, 0, slice(None), 5))):
            key = of_state == (0, 0, 5)
            broken = (k if key else v).clone()
            broken[at] = bad
            out, after = forward(c, q, broken if key else k, v if key else broken, log_decay, before)
            spoilt(out, "out", of_out)
            spoilt(after, "after", of_state)
        broken = q.clone()
        broken[0, t0, 1, 5] = bad
        dq, dk, dv, d_before = backward(c, broken, k, v, dout, log_decay, before, d_after)
        spoilt(dq, "dq", (0, slice(0, 0)))
        spoilt(dk, "dk", (0, slice(0, t0 + 1), 0, 5))
        spoilt(dv, "dv", (0, slice(0, t0 + 1), 0))
        spoilt(d_before, "d_before", (0, 0, 5))
        broken = dout.clone()
        broken[0, t0, 1, 5] = bad
        dq, dk, dv, d_before = backward(c, q, k, v, broken, log_decay, before, d_after)
        spoilt(dq, "dq", (0, t0, 1))
        spoilt(dk, "dk", (0, slice(0, t0 + 1), 0))
        spoilt(dv, "dv", (0, slice(0, t0 + 1), 0, 5))
        spoilt(d_before, "d_before", (0, 0, slice(None), 5))


@pytest.mark.parametrize("dtype", DTYPES, ids=DTYPE_IDS)
def test_states_at_the_end_of_the_range(device, dtype):
    """A first state (and a last one's gradient) of 2^120, which 0.4 a token brings back to outputs that half precision holds behind 270 tokens of 400.
    More sequences than compute units, so that none is cut."""
    c = case(130, 400, 2, 2, 32, decay=[-0.4 * 0.6931471805599453])
    q, k, v, dout, log_decay, before, d_after = inputs(c, dtype, device)
    before, d_after = before.sign() * 2.0 ** 120, d_after.sign() * 2.0 ** 120
    want = {**linear_forward(q, k, v, log_decay, before, 0.0), **linear_backward(q, k, v, log_decay, before, dout, d_after, 0.0)}
    for name, got in zip(("out", "after", *GRADS), (*forward(c, q, k, v, log_decay, before), *backward(c, q, k, v, dout, log_decay, before, d_after))):
        check(got, want[name], name)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
@pytest.mark.parametrize("t,hq,hkv,d,decay", [(4097, 2, 1, 64, -0.01), (1025, 4, 2, 128, -1e-3), (8000, 3, 1, 40, -0.1)], ids=str)
def test_long_sequences_in_the_2_norm(device, t, hq, hkv, d, decay, dtype):
    """Scores, the matrix and the result are rounded once, each by at most a half step u of terms whose signs are random, so that their sum's 2-norm is the
    terms': 3 u, and the decayed values' 2^-16. What a chunk, a segment or a join adds wrongly would show at several per cent of an output."""
    c = case(1, t, hq, hkv, d, decay=[decay])
    q, k, v, dout, log_decay, before, d_after = inputs(c, dtype, device)
    want = {**linear_forward(q, k, v, log_decay, before, 0.0), **linear_backward(q, k, v, log_decay, before, dout, d_after, 0.0)}
    tolerance = 3 * torch.finfo(dtype).eps / 2 + 2.0 ** -16
    for name, got in zip(("out", "after", *GRADS), (*forward(c, q, k, v, log_decay, before), *backward(c, q, k, v, dout, log_decay, before, d_after))):
        check(got, want[name], name)
        for rows in (slice(0, 64), slice(64, t // 2), slice(t // 2, None)) if got.shape[1] == t else (slice(None),):
            off = (got[:, rows].double() - want[name].value[:, rows]).norm() / want[name].value[:, rows].norm()
            assert off <= tolerance, f"{name}, {rows}: {off:.3g} of its norm, allowed {tolerance:.3g}"


@pytest.mark.parametrize("c", CASES, ids=IDS)
def test_half_precision_to_what_the_decays_leave(device, c):
    q, k, v, dout, log_decay, before, d_after = inputs(c, torch.float16, device)
    want = {**linear_forward(q, k, v, log_decay, before, c["scale"]), **linear_backward(q, k, v, log_decay, before, dout, d_after, c["scale"])}
    for name, got in zip(("out", "after", *GRADS), (*forward(c, q, k, v, log_decay, before), *backward(c, q, k, v, dout, log_decay, before, d_after))):
        check(got, want[name], name)
