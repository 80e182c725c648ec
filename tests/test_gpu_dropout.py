"""Dropout through the operator interface: its masks against the generator written in numpy, its values against 64 bits.

Values: input * scale + residual in one fp32 rounding, then one of the storage type: half a step of each, relative to the value.
The scale, 65536 / (65536 - threshold), is itself rounded to fp32: the product is off by 2^-24 of itself, which a residual of the
other sign leaves while it takes the value away. Hence a term of 2^-24 of the product."""
import numpy as np
import pytest
import torch

from cgpt_amd import ops
from tests.util import DTYPE_IDS, DTYPES, randn

pytestmark = pytest.mark.gpu


def philox(counter, key, rounds=10):
    """Philox 4x32 over arrays of counters: four words in, four out."""
    c = [np.asarray(w, dtype=np.uint64) for w in counter]
    k = [np.uint64(key[0]), np.uint64(key[1])]
    low = np.uint64(0xFFFFFFFF)
    for _ in range(rounds):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ k[0], b & low, (a >> np.uint64(32)) ^ c[3] ^ k[1], a & low]
        k = [(k[0] + np.uint64(0x9E3779B9)) & low, (k[1] + np.uint64(0xBB67AE85)) & low]
    return c


def numbers(count, seed, offset):
    """Sixteen bits per element, as include/cgptx.h defines them; the counter wraps at 2^64."""
    n = np.array([(offset + j) % 2**64 for j in range((count + 7) // 8)], dtype=np.uint64)
    words = philox([n & np.uint64(0xFFFFFFFF), n >> np.uint64(32), np.zeros_like(n), np.zeros_like(n)], (seed & 0xFFFFFFFF, seed >> 32))
    return np.stack([w.astype("<u4") for w in words], axis=1).copy().view("<u2").reshape(-1)[:count]


def test_the_generator_of_this_file():
    """Known answers that were published with the generator."""
    def words(counter, key):
        return [int(w) for w in philox(counter, key)]

    assert words([0, 0, 0, 0], (0, 0)) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    ones = 0xFFFFFFFF
    assert words([ones] * 4, (ones, ones)) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
    assert words([0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344], (0xA4093822, 0x299F31D0)) == \
        [0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1]


def keep_mask(count, probability, seed, offset, device):
    threshold = int(np.float64(np.float32(probability)) * 65536 + 0.5)
    return torch.from_numpy(numbers(count, seed, offset) >= threshold).to(device), threshold


def expected(x, residual, keep, threshold):
    scale = 65536 / (65536 - threshold) if threshold < 65536 else 0.0
    out = torch.where(keep.view(x.shape), x.double() * scale, torch.zeros((), dtype=torch.float64, device=x.device))
    return out if residual is None else out + residual.double()


def check(got, want, residual=None):
    dtype = got.dtype
    product = want if residual is None else want - residual.double()
    bound = want.abs() * (torch.finfo(dtype).eps / 2 + 2.0 ** -22) + (2.0 ** -25 if dtype == torch.float16 else 1e-37)
    worst = ((got.double() - want).abs() / (bound + 1.0001 * 2.0 ** -24 * product.abs())).max().item()
    assert worst <= 1, f"{worst:.3f} times the bound"


CASES = [(1, 0.5, 0, 0), (7, 0.1, 1, 5), (8, 0.9, 2, 2**32 - 1), (9, 0.2, 2**63 + 12345, 2**40), (1000, 0.3, 7, 2**64 - 3),
         (4097, 0.05, 2**64 - 1, 1), (76799, 0.25, 99, 10**12), (100003, 0.1, 123456789, 0)]


@pytest.mark.parametrize("dtype", DTYPES, ids=DTYPE_IDS)
@pytest.mark.parametrize("count,probability,seed,offset", CASES)
def test_forward_and_backward(device, count, probability, seed, offset, dtype):
    options = ops.DropoutOptions(probability, seed, offset)
    x, residual, dy = (randn((count,), dtype, s).to(device) for s in (1, 2, 3))
    keep, threshold = keep_mask(count, probability, seed, offset, device)
    for res in (None, residual):
        out = torch.full_like(x, 9.0)
        ops.dropout_forward(out, x, res, None, options)
        check(out, expected(x, res, keep, threshold), res)
    dx = torch.full_like(x, 9.0)
    ops.dropout_backward(dx, dy, None, options)
    check(dx, expected(dy, None, keep, threshold))
    before = dx.clone()
    ops.dropout_backward(dx, dy, None, options, True)
    check(dx, expected(dy, before, keep, threshold), before)


@pytest.mark.parametrize("dtype", DTYPES, ids=DTYPE_IDS)
def test_never_always_and_the_steps_between(device, dtype):
    x = randn((5000,), dtype, 4).to(device)
    out = torch.empty_like(x)
    for probability in (0.0, 2.0 ** -18):  # both round to nothing dropped
        ops.dropout_forward(out, x, None, None, ops.DropoutOptions(probability, 3, 4))
        assert torch.equal(out, x)
    for probability in (1.0, 1.0 - 2.0 ** -20):
        ops.dropout_forward(out, x, x, None, ops.DropoutOptions(probability, 3, 4))
        assert torch.equal(out, x)
        ops.dropout_forward(out, x, None, None, ops.DropoutOptions(probability, 3, 4))
        assert (out == 0).all()
    last = numbers(5000, 3, 4) == 65535  # the only numbers that a probability of 1 - 2^-16 keeps
    ops.dropout_forward(out, torch.ones_like(x), None, None, ops.DropoutOptions(1 - 2.0 ** -16, 3, 4))
    assert ((out != 0).cpu().numpy() == last).all()


def test_what_is_dropped_is_zero_whatever_it_was(device):
    for dtype in DTYPES:
        x = torch.full((4099,), float("nan"), dtype=dtype, device=device)
        x[1::3] = float("inf")
        out = torch.empty_like(x)
        ops.dropout_forward(out, x, None, None, ops.DropoutOptions(0.5, 8, 9))
        keep, _ = keep_mask(4099, 0.5, 8, 9, device)
        assert (out[~keep] == 0).all() and not torch.isfinite(out[keep]).any()


@pytest.mark.parametrize("dtype", DTYPES, ids=DTYPE_IDS)
def test_a_mask_goes_by_nothing_but_its_options(device, dtype):
    """The same mask off the alignment, in place, on another stream, of a prefix, and cut at a counter value."""
    count, options = 4096 + 5, ops.DropoutOptions(0.4, 77, 1000)
    x, residual = randn((count,), dtype, 5).to(device), randn((count,), dtype, 6).to(device)
    want = torch.empty_like(x)
    ops.dropout_forward(want, x, residual, None, options)
    base = torch.empty(3, count + 1, dtype=dtype, device=device)
    moved = [base[i].view(-1)[1:] for i in range(3)]
    moved[1].copy_(x)
    moved[2].copy_(residual)
    ops.dropout_forward(moved[0], moved[1], moved[2], None, options)
    assert torch.equal(moved[0], want)
    for alias in (0, 1):
        pair = [x.clone(), residual.clone()]
        ops.dropout_forward(pair[alias], pair[0], pair[1], None, options)
        assert torch.equal(pair[alias], want)
    torch.cuda.synchronize()
    side, out = torch.cuda.Stream(), torch.empty_like(x)
    ops.dropout_forward(out, x, residual, side, options)
    side.synchronize()
    assert torch.equal(out, want)
    parts = torch.empty_like(x)
    ops.dropout_forward(parts[:1600], x[:1600], residual[:1600], None, options)
    ops.dropout_forward(parts[1600:], x[1600:], residual[1600:], None, ops.DropoutOptions(0.4, 77, 1200))
    assert torch.equal(parts, want)


def test_a_large_tensor(device):
    """More elements than 32 bits of bytes: the last ones have their own numbers."""
    count = (1 << 31) + 1003
    x = torch.ones(count, dtype=torch.bfloat16, device=device)
    ops.dropout_forward(x, x, None, None, ops.DropoutOptions(0.25, 5, 6))
    at = count - 2003 - (count - 2003) % 8
    keep, threshold = keep_mask(count - at, 0.25, 5, 6 + at // 8, device)
    check(x[at:], expected(torch.ones_like(x[at:]), None, keep, threshold))
    share = (x[: 1 << 26] != 0).double().mean().item()
    assert abs(share - 0.75) <= 6 * (0.75 * 0.25 / (1 << 26)) ** 0.5  # six deviations of the share


def test_no_elements(device):
    x = torch.empty(0, dtype=torch.bfloat16, device=device)
    ops.dropout_forward(x, x)
    ops.dropout_backward(x, x)


def test_neighbouring_seeds_and_calls_are_unrelated(device):
    """Agreement of two masks of 2^20 elements: binomial, six deviations."""
    count, p = 1 << 20, 0.3
    x, masks = torch.ones(count, device=device), []
    for options in (ops.DropoutOptions(p, 1, 0), ops.DropoutOptions(p, 2, 0), ops.DropoutOptions(p, 1, count // 8)):
        out = torch.empty_like(x)
        ops.dropout_forward(out, x, None, None, options)
        masks.append(out != 0)
    both = (p * p + (1 - p) * (1 - p))
    for a, c in ((0, 1), (0, 2), (1, 2)):
        agree = (masks[a] == masks[c]).double().mean().item()
        assert abs(agree - both) <= 6 * (both * (1 - both) / count) ** 0.5


def test_a_replayed_graph_draws_new_masks(device):
    """The counter on the device moves on between replays; the backward call of a replay has its forward call's mask."""
    count = 5001
    x, dy = randn((count,), torch.float32, 7).to(device), randn((count,), torch.float32, 8).to(device)
    out, dx = torch.empty_like(x), torch.empty_like(x)
    counter = torch.zeros(1, dtype=torch.int64, device=device)
    options = ops.DropoutOptions(0.5, 11, 100, counter)
    stream = torch.cuda.Stream()

    def step():
        ops.dropout_forward(out, x, None, None, options)
        ops.dropout_backward(dx, dy, None, options)
        counter.add_((count + 7) // 8)

    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        step()
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream, capture_error_mode="thread_local"):
        step()
    for replay in range(1, 5):
        graph.replay()
        torch.cuda.synchronize()
        keep, threshold = keep_mask(count, 0.5, 11, 100 + replay * ((count + 7) // 8), device)
        check(out, expected(x, None, keep, threshold))
        check(dx, expected(dy, None, keep, threshold))


def test_gradient_against_differences(device):
    """Dropout is linear in its input: the difference along a direction is the gradient's product with it, to rounding."""
    count, options = 999, ops.DropoutOptions(0.35, 21, 22)
    x, v, dy = (randn((count,), torch.float32, s).to(device) for s in (9, 10, 11))
    ahead, back, dx = torch.empty_like(x), torch.empty_like(x), torch.empty_like(x)
    ops.dropout_forward(ahead, x + 0.5 * v, None, None, options)
    ops.dropout_forward(back, x - 0.5 * v, None, None, options)
    ops.dropout_backward(dx, dy, None, options)
    terms = dy.double() * (ahead.double() - back.double())
    size = (dy.double().abs() * (x.abs() + v.abs()).double()).sum().item() / 0.65
    assert abs(terms.sum().item() - (dx.double() * v.double()).sum().item()) <= 8 * 2.0 ** -24 * size
