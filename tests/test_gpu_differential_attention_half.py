"""Differential attention's gradients where 16 bits have few digits: of small output gradients in half precision, of rows that see few keys.

Gradients are linear in dO: with dO times 2^-s, a product that is exact here, the results are those of dO times 2^-s, within as much less. What is
left beside that is half a step among the smallest numbers that the results themselves are stored in (check allows 2^-24)."""
import pytest
import torch

from tests.test_gpu_differential_attention import GRADS, backward, case, check, forward, inputs, options, reference
from tests.util import randn

pytestmark = pytest.mark.gpu

CASES = [case(1, 1001, 1001, 3, 1, 64), case(2, 333, 333, 8, 2, 128), case(1, 700, 900, 2, 1, 128, causal=False), case(1, 64, 3000, 2, 2, 64),
         case(1, 1, 4000, 8, 2, 128), case(9, 300, 300, 8, 8, 64), case(2, 20, 50, 4, 2, 96)]
IDS = ["-".join(str(v) for v in c.values()) for c in CASES]


def few_bits(shape, seed, device):
    """Normal numbers rounded to multiples of 2^-6: times 2^-18 they are still half-precision numbers."""
    return ((randn(shape, torch.float32, seed) * 64).round() / 64).to(torch.float16).to(device)


def scaled(want, shift):
    """The reference's values and bounds times 2^-shift, but for those of the forward pass."""
    return {n: v * 2.0 ** -shift for n, v in want.items() if n.removesuffix("_err") in GRADS}


@pytest.mark.parametrize("shift", [4, 8, 12, 18])
@pytest.mark.parametrize("c", CASES, ids=IDS)
def test_small_output_gradients(device, c, shift):
    q, k, v, _, lambdas = inputs(c, torch.float16, device)
    dout = few_bits(q.shape, 5, device)
    saved = forward(c, q, k, v, lambdas)
    want = scaled(reference(c, q, k, v, lambdas, dout), shift)
    for got, name in zip(backward(c, q, k, v, (dout.float() * 2.0 ** -shift).half(), lambdas, saved), GRADS):
        check(got, want[name], want[name + "_err"], name)


def test_large_and_small_ones_beside_each_other(device):
    """Batch entries and heads of their own sizes; in one head, dq goes by its row's and dk by the largest."""
    c = case(3, 500, 500, 4, 2, 128)
    q, k, v, _, lambdas = inputs(c, torch.float16, device)
    dout, saved = few_bits(q.shape, 6, device), forward(c, q, k, v, lambdas)
    want = reference(c, q, k, v, lambdas, dout)
    size = torch.ones(3, 1, 4, 1, device=device)  # by batch entry and pair of heads that share a kv head
    size[1], size[2] = 2.0 ** -9, 2.0 ** -16
    size[0, :, 2:] = 2.0 ** -13
    grads = backward(c, q, k, v, (dout.float() * size).half(), lambdas, saved)
    for got, name, by in zip(grads[:3], GRADS, (size, size[:, :, ::2], size[:, :, ::2])):
        check(got, want[name] * by, want[name + "_err"] * by, name)
    row = torch.ones(1, 500, 1, 1, device=device)
    row[:, 1::2] = 2.0 ** -12
    dq = backward(c, q, k, v, (dout.float() * row).half(), lambdas, saved)[0]
    check(dq, want["dq"] * row, want["dq_err"] * row, "dq")


@pytest.mark.parametrize("c", [case(1, 300, 300, 2, 1, 128), case(2, 140, 140, 4, 2, 64), case(16, 200, 200, 8, 4, 128)], ids=["shared", "64", "whole"])
def test_large_values_beside_small_output_gradients(device, c):
    """Score gradients that would not be half-precision numbers any more if they were enlarged as the output gradients allow."""
    q, k, v, _, lambdas = inputs(c, torch.float16, device)
    sign = torch.where(torch.arange(c["d"], device=device) % 3 == 0, -1.0, 1.0)
    v = (sign * torch.where(torch.arange(c["ks"], device=device) % 2 == 0, 24000.0, -24000.0)[None, :, None, None]).expand_as(v).half().contiguous()
    dout = (few_bits(q.shape, 5, device).abs() * sign).half()
    shift = 14
    saved = forward(c, q, k, v, lambdas)
    want = scaled(reference(c, q, k, v, lambdas, dout), shift)
    for got, name in zip(backward(c, q, k, v, (dout.float() * 2.0 ** -shift).half(), lambdas, saved), GRADS):
        # Not enlarged, what is below 2^-14 is rounded by up to 2^-25: of the score gradients and the maps, times the other factor's sum.
        lost = 2.0 ** -25 * {"dq": k, "dk": q, "dv": dout * 2.0 ** -shift, "dlam": lambdas * 0}[name].double().abs().sum().item()
        check(got, want[name], want[name + "_err"] + lost, name)


def test_output_gradients_that_are_no_numbers_stay_in_their_rows(device):
    """Whatever a row's dO is, the other rows' dq are what they are without it."""
    c = case(2, 200, 200, 4, 2, 64)
    q, k, v, _, lambdas = inputs(c, torch.float16, device)
    dout, saved = few_bits(q.shape, 7, device) * 2.0 ** -4, forward(c, q, k, v, lambdas)
    want = reference(c, q, k, v, lambdas, dout)
    for value in (float("nan"), float("inf")):
        bad = dout.clone()
        bad[:, 70] = value
        dq = backward(c, q, k, v, bad, lambdas, saved)[0]
        assert not torch.isfinite(dq[:, 70]).any()
        rest = [i for i in range(200) if i != 70]
        check(dq[:, rest], want["dq"][:, rest], want["dq_err"][:, rest], "dq")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
@pytest.mark.parametrize("c", [case(5, 1001, 1001, 12, 4, 64), case(16, 300, 300, 8, 2, 128), case(3, 100, 100, 4, 2, 64), case(24, 130, 140, 8, 8, 96)],
                         ids=["64", "128", "few-blocks", "offset"])
def test_rows_that_see_few_keys(device, c, dtype):
    """The first rows of a longer sequence, which most of dq's norm is in: rowsum(P (G - delta)) is taken off there, whatever O was rounded to.

    Bound: `reference` with deltas that are summed, for rows whose block of 32 sees one tile of 64 keys; for every row its usual bounds. In
    the 2-norm: dq's rounding is one error of half a step at most, evenly spread, and that of the score gradients another that is as
    large beside the result: sqrt(2) of the exact dq's rounding error, and 1.5 with what the deltas of the other rows add."""
    q, k, v, dout, lambdas = inputs(c, dtype, device)
    dq = backward(c, q, k, v, dout, lambdas, forward(c, q, k, v, lambdas))[0]
    want, summed = reference(c, q, k, v, lambdas, dout), reference(c, q, k, v, lambdas, dout, summed=True)
    few = (64 - c["off"]) // 32 * 32
    check(dq[:, :few], want["dq"][:, :few], summed["dq_err"][:, :few], "dq of few keys")
    check(dq, want["dq"], want["dq_err"], "dq")
    rounding = (want["dq"].to(dtype).double() - want["dq"]).norm().item()
    off = (dq.double() - want["dq"]).norm().item()
    print(f"[parity] dq: {off / rounding:.3f} of the exact dq's rounding")
    assert off <= 1.5 * rounding


@pytest.mark.parametrize("what", ["q", "k", "v"])
def test_tensors_with_an_infinity_beside_small_output_gradients(device, what):
    """Keys and heads that the infinity does not reach are what they are without it."""
    c = case(2, 260, 260, 4, 2, 64)
    q, k, v, _, lambdas = inputs(c, torch.float16, device)
    dout = few_bits(q.shape, 8, device) * 2.0 ** -6
    want = reference(c, q, k, v, lambdas, dout)
    {"q": q, "k": k, "v": v}[what][0, 130, :2 if what == "q" else 1] = float("inf")
    dq, dk, dv, _ = backward(c, q, k, v, dout, lambdas, forward(c, q, k, v, lambdas))
    for got, name in ((dq, "dq"), (dk, "dk"), (dv, "dv")):
        heads = 2 if name == "dq" else 1
        check(got[1], want[name][1], want[name + "_err"][1], name)
        check(got[0, :, heads:], want[name][0, :, heads:], want[name + "_err"][0, :, heads:], name)
    check(dq[0, :130], want["dq"][0, :130], want["dq_err"][0, :130], "dq")
