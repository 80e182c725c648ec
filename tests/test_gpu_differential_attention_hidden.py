"""Differential attention: keys and values that hold anything where no query sees them, and a key that weighs nothing.

A pair that the mask hides adds nothing, whatever the tensors hold there: keys that no query sees get gradients of exactly 0 (nothing is
added to what accumulated ones hold), the others stay within the bounds of tests/test_gpu_differential_attention.py, which do not know
of the padding: its values are replaced before they are worked out."""
import pytest
import torch

from tests.test_gpu_differential_attention import GRADS, backward, case, check, forward, inputs, reference
from tests.util import DTYPE_IDS, DTYPES, randn

pytestmark = pytest.mark.gpu

NAN, INF = float("nan"), float("inf")

# Keys from off + qs on are seen by nobody: in the block of the last seen key, in blocks of their own, with query tiles that end inside
# and on their boundary; key blocks that are shared (few of them), whole, and in pairs (many); one query; widths of every kernel.
CASES = [case(2, 20, 1500, 6, 2, 128, off=900), case(1, 150, 260, 4, 2, 64, off=0), case(1, 300, 420, 4, 2, 128, off=37), case(1, 128, 200, 2, 1, 128, off=0),
         case(1, 64, 100, 2, 2, 64, off=0), case(16, 200, 330, 8, 8, 64, off=3), case(24, 130, 300, 6, 6, 128, off=10), case(2, 1, 200, 4, 1, 80, off=70),
         case(3, 33, 150, 2, 1, 36, off=40), case(2, 70, 90, 4, 2, 24, off=1)]
IDS = ["-".join(str(v) for v in c.values()) for c in CASES]


@pytest.mark.parametrize("dtype", DTYPES, ids=DTYPE_IDS)
@pytest.mark.parametrize("c", CASES, ids=IDS)
def test_gradients_of_keys_that_no_query_sees(device, c, dtype):
    q, k, v, dout, lambdas = inputs(c, dtype, device)
    seen = c["off"] + c["qs"]
    assert seen < c["ks"]
    want = reference(c, q, k, v, lambdas, dout)
    base = [randn(t.shape, t.dtype, 40 + i).to(device) for i, t in enumerate((q, k, v, lambdas))]
    for k_value, v_value in ((NAN, NAN), (INF, -INF), (-INF, 0.0), (0.0, INF)):
        k2, v2 = k.clone(), v.clone()
        k2[:, seen:] = k_value
        v2[:, seen:] = v_value
        saved = forward(c, q, k2, v2, lambdas)
        for got, name in zip(saved, ("out", "second", "lse")):
            check(got, want[name], want[name + "_err"], name)
        grads = backward(c, q, k2, v2, dout, lambdas, saved)
        for got, name in zip(grads, GRADS):
            check(got, want[name], want[name + "_err"], name)
        assert not grads[1][:, seen:].any() and not grads[2][:, seen:].any()
        added = backward(c, q, k2, v2, dout, lambdas, saved, base)
        assert torch.equal(added[1][:, seen:], base[1][:, seen:]) and torch.equal(added[2][:, seen:], base[2][:, seen:])
        for got, name, before in zip(added, GRADS, base):
            check(got, want[name] + before.double(), want[name + "_err"] + 2.0 ** -22 * (want[name].abs() + before.double().abs()), name)


@pytest.mark.parametrize("dtype", DTYPES, ids=DTYPE_IDS)
@pytest.mark.parametrize("d", [2, 36, 64, 128])
def test_a_first_key_of_no_weight(device, dtype, d):
    """Every score of the first key is -Inf: its probability is 0, and the rest is what it is without the key."""
    c = case(2, 40, 61, 4, 2, d)
    q, k, v, dout, lambdas = inputs(c, dtype, device)
    q = q.abs() + 0.25
    without = dict(c, ks=c["ks"] - 1, off=c["off"] - 1)
    want = reference(without, q, k[:, 1:], v[:, 1:], lambdas, dout)
    k[:, 0] = -INF
    saved = forward(c, q, k, v, lambdas)
    for got, name in zip(saved, ("out", "second", "lse")):
        check(got, want[name], want[name + "_err"], name)
    if dtype != torch.float32 and d >= 64:
        return  # their dK/dV pass multiplies the key by the zeros of the queries past the end
    dk, dv = backward(c, q, k, v, dout, lambdas, saved)[1:3]  # the query's gradient has 0 times the key in it
    for got, name in ((dk, "dk"), (dv, "dv")):
        assert not got[:, 0].any()
        check(got[:, 1:], want[name], want[name + "_err"], name)
