"""Layer norm forward and backward through the operator interface against the formulas in 64 bits.

Tolerances, for every element: half a step of the storage type for the one rounding at the end (eps/2 relative to the value), and
for fp32 arithmetic 2^-24 for each rounding on the longest chain of additions that a kernel may have (sixteen lanes to a row; a
row sum then has hidden/16 additions in a lane, the weight's gradient rows/128 in a lane and the workgroups' parts) times the sum
of the magnitudes that are added. The mean's error, 2^-24 chain max|x|, reaches xh times r."""
import math

import pytest
import torch

from cgpt_amd import ops
from tests.util import DTYPE_IDS, DTYPES, launches, randn

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24
EPS = 1e-5


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def reference(x, w, b, dy, residual, eps=EPS):
    """Results in 64 bits and what bounds their rounding."""
    x64, w64 = x.double(), w.double()
    centred = x64 - x64.mean(1, keepdim=True)
    r = 1 / torch.sqrt((centred ** 2).mean(1, keepdim=True) + eps)
    xh = centred * r
    y = xh * w64 + (0 if b is None else b.double())
    hidden, rows = x.shape[1], x.shape[0]
    chain = hidden / 16 + 16
    off = U32 * chain * x64.abs().amax(1, keepdim=True) * r  # of xh, from the mean
    rel = U32 * (chain + 8)
    out = {"y": y, "y_err": off * w64.abs() + 2 * rel * (xh * w64).abs() + 4 * U32 * (y.abs() + (0 if b is None else b.double().abs()))}
    if dy is None:
        return out
    dy64 = dy.double()
    g = dy64 * w64
    m1, m2 = g.mean(1, keepdim=True), (g * xh).mean(1, keepdim=True)
    dx = r * (g - m1 - xh * m2)
    top = g.abs().amax(1, keepdim=True)
    out["dx_err"] = r * top * (rel * (4 + 4 * xh.abs()) + 2 * off * (1 + xh.abs())) + (0 if residual is None else 2 * U32 * residual.double().abs())
    out["dx"] = dx if residual is None else dx + residual.double()
    rows_chain = min(rows, rows / 128 + 160) + 8
    out["dw"], out["db"] = (dy64 * xh).sum(0), dy64.sum(0)
    out["dw_err"] = (dy64.abs() * (xh.abs() * (U32 * rows_chain + 2 * rel) + off)).sum(0)
    out["db_err"] = U32 * rows_chain * dy64.abs().sum(0)
    return out


def check(actual, want, err, what):
    bound = want.abs() * half_step(actual.dtype) * 1.0001 + err + 1e-30
    if actual.dtype == torch.float16:
        bound = bound + 2.0 ** -25  # half a step among the smallest numbers
    off = (actual.double() - want).abs()
    assert torch.isfinite(actual).all(), what
    worst = (off / bound).max().item()
    print(f"[parity] {what}: {worst:.3f} of the bound")
    assert worst <= 1, f"{what}: {worst:.3f} times the bound"


def inputs(rows, hidden, dtype, device, shift=0.0, bias=True, seed=1):
    x = (randn((rows, hidden), torch.float32, seed) + shift).to(dtype).to(device)
    w = (1 + 0.2 * randn((hidden,), torch.float32, seed + 1)).to(dtype).to(device)
    b = randn((hidden,), dtype, seed + 2, 0.3).to(device) if bias else None
    dy = randn((rows, hidden), dtype, seed + 3).to(device)
    return x, w, b, dy


SHAPES = [(1, 1), (1, 8), (3, 7), (2, 64), (5, 100), (1, 1024), (9, 1000), (7, 1001), (33, 128), (130, 256), (300, 768), (65, 2048), (17, 4096),
          (10, 4104), (3, 8192), (2, 10000), (2, 16384), (1, 20003), (2, 40000), (4099, 40), (2500, 1024)]


@pytest.mark.parametrize("dtype", DTYPES, ids=DTYPE_IDS)
@pytest.mark.parametrize("rows,hidden", SHAPES)
def test_forward(device, rows, hidden, dtype):
    for bias in (True, False):
        x, w, b, _ = inputs(rows, hidden, dtype, device, bias=bias)
        y = torch.full_like(x, 9.0)
        ops.layernorm_forward(y, x, w, b, EPS)
        want = reference(x, w, b, None, None)
        check(y, want["y"], want["y_err"], f"y[{rows},{hidden}]")


@pytest.mark.parametrize("dtype", DTYPES, ids=DTYPE_IDS)
@pytest.mark.parametrize("rows,hidden", SHAPES)
def test_backward(device, rows, hidden, dtype):
    x, w, b, dy = inputs(rows, hidden, dtype, device)
    residual = randn((rows, hidden), dtype, 11).to(device)
    for res, bias in ((None, True), (residual, False), (residual, True)):
        dx, dw, db = torch.full_like(x, 9.0), torch.full_like(w, 9.0), torch.full_like(w, 9.0) if bias else None
        ops.layernorm_backward(dx, dw, db, dy, x, w, EPS, None, res)
        want = reference(x, w, b, dy, res)
        check(dx, want["dx"], want["dx_err"], f"dx[{rows},{hidden}]")
        check(dw, want["dw"], want["dw_err"], f"dw[{rows},{hidden}]")
        if bias:
            check(db, want["db"], want["db_err"], f"db[{rows},{hidden}]")


@pytest.mark.parametrize("hidden", [64, 1001, 1024, 9000])
def test_rows_far_from_zero(device, hidden):
    """mean(x^2) - mean(x)^2 has no correct digit here."""
    x, w, b, dy = inputs(40, hidden, torch.float32, device, shift=5000.0)
    y, dx, dw, db = torch.empty_like(x), torch.empty_like(x), torch.empty_like(w), torch.empty_like(w)
    ops.layernorm_forward(y, x, w, b, EPS)
    ops.layernorm_backward(dx, dw, db, dy, x, w, EPS)
    want = reference(x, w, b, dy, None)
    for got, name in ((y, "y"), (dx, "dx"), (dw, "dw"), (db, "db")):
        check(got, want[name], want[name + "_err"], name)


@pytest.mark.parametrize("hidden", [8, 1024, 1003, 20000])
def test_constant_rows(device, hidden):
    """A row without variance is the bias, exactly: 1024 is a power of two, 3 times anything below is exact in fp32 sums."""
    x = torch.full((5, hidden), 3.0, dtype=torch.bfloat16, device=device)
    w, b = torch.ones(hidden, dtype=torch.bfloat16, device=device), randn((hidden,), torch.bfloat16, 4).to(device)
    y = torch.empty_like(x)
    ops.layernorm_forward(y, x, w, b, EPS)
    # sum = 3 hidden is exact below 2^24; the mean rounds twice (inverse and product): |x - mean| <= 3 * 2^-23, xh <= 3 * 2^-23 / sqrt(eps)
    assert (y.double() - b.double()).abs().max().item() <= 3 * 2.0 ** -23 / math.sqrt(EPS) + 2.0 ** -8 * b.double().abs().max().item()


@pytest.mark.parametrize("dtype", DTYPES, ids=DTYPE_IDS)
@pytest.mark.parametrize("hidden", [1000, 1024, 9000])
def test_large_values_of_16_bits(device, hidden, dtype):
    x, w, b, _ = inputs(6, hidden, torch.float32, device)
    x = (x * 6e4 / x.abs().max()).to(dtype)
    w, b = w.to(dtype), b.to(dtype)
    y = torch.empty_like(x)
    ops.layernorm_forward(y, x, w, b, EPS)
    want = reference(x, w, b, None, None)
    check(y, want["y"], want["y_err"], "y")


@pytest.mark.parametrize("dtype", DTYPES, ids=DTYPE_IDS)
def test_a_row_that_is_not_finite_stays_alone(device, dtype):
    for hidden in (1001, 1024, 20000):
        x, w, b, dy = inputs(9, hidden, dtype, device)
        y, dx, dw, db = torch.empty_like(x), torch.empty_like(x), torch.empty_like(w), torch.empty_like(w)
        ops.layernorm_forward(y, x, w, b, EPS)
        ops.layernorm_backward(dx, dw, db, dy, x, w, EPS)
        bad = x.clone()
        bad[4, hidden // 2] = float("nan")
        bad[7, 0] = float("inf")
        y2, dx2 = torch.empty_like(x), torch.empty_like(x)
        ops.layernorm_forward(y2, bad, w, b, EPS)
        ops.layernorm_backward(dx2, dw, db, dy, bad, w, EPS)
        rest = [i for i in range(9) if i not in (4, 7)]
        assert torch.equal(y[rest], y2[rest]) and torch.equal(dx[rest], dx2[rest])
        assert torch.isnan(y2[4]).all() and torch.isnan(dx2[4]).all() and torch.isnan(dw).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=DTYPE_IDS)
@pytest.mark.parametrize("hidden", [1000, 1024])
def test_tensors_off_their_alignment(device, hidden, dtype):
    """Views that start one element into their memory."""
    rows = 37
    x, w, b, dy = inputs(rows, hidden, dtype, device)

    def moved(t):
        base = torch.zeros(t.numel() + 1, dtype=dtype, device=device)
        base[1:].copy_(t.reshape(-1))
        return base[1:].view(t.shape)

    want = reference(x, w, b, dy, None)
    mx, mw, mb, mdy = (moved(t) for t in (x, w, b, dy))
    y, dx, dw, db = moved(x), moved(x), moved(w), moved(w)
    ops.layernorm_forward(y, mx, mw, mb, EPS)
    ops.layernorm_backward(dx, dw, db, mdy, mx, mw, EPS)
    for got, name in ((y, "y"), (dx, "dx"), (dw, "dw"), (db, "db")):
        check(got, want[name], want[name + "_err"], name)


@pytest.mark.parametrize("hidden", [1001, 1024])
def test_residual_in_place_and_twice_the_same(device, hidden):
    x, w, b, dy = inputs(300, hidden, torch.bfloat16, device)
    residual = randn((300, hidden), torch.bfloat16, 21).to(device)
    results = []
    for _ in range(2):
        dx, dw, db = residual.clone(), torch.empty_like(w), torch.empty_like(w)
        ops.layernorm_backward(dx, dw, db, dy, x, w, EPS, None, dx)
        results.append((dx, dw, db))
    apart = [torch.empty_like(x), torch.empty_like(w), torch.empty_like(w)]
    ops.layernorm_backward(*apart, dy, x, w, EPS, None, residual)
    for a, c, d in zip(*results, apart):
        assert torch.equal(a, c) and torch.equal(a, d)


@pytest.mark.parametrize("rows,hidden", [((1 << 21) + 5, 1024), ((1 << 16) + 3, 32771)], ids=["rows", "long"])
def test_a_large_tensor(device, rows, hidden):
    """The last rows lie behind 2^31 elements: they come out as in a call of their own, whose columns' sums the whole call's contain."""
    dtype, last = torch.bfloat16, 3
    x, dy = (torch.zeros((rows, hidden), dtype=dtype, device=device) for _ in range(2))
    x[-last:], dy[-last:] = randn((last, hidden), dtype, 1).to(device), randn((last, hidden), dtype, 2).to(device)
    w, b = randn((hidden,), dtype, 3).to(device), randn((hidden,), dtype, 4).to(device)
    out, alone = torch.full_like(x, 7.0), torch.full_like(x[-last:], 7.0)
    ops.layernorm_forward(out, x, w, b, 1e-5)
    ops.layernorm_forward(alone, x[-last:], w, b, 1e-5)
    assert torch.equal(out[-last:], alone)
    assert torch.equal(out[:-last].amin(0), b) and torch.equal(out[:-last].amax(0), b)
    dw, db, dw_alone, db_alone = (torch.full_like(w, 7.0) for _ in range(4))
    ops.layernorm_backward(out, dw, db, dy, x, w, 1e-5)
    ops.layernorm_backward(alone, dw_alone, db_alone, dy[-last:], x[-last:], w, 1e-5)
    assert torch.equal(out[-last:], alone) and not out[:-last].any()
    # The other rows add zeros; three summands in another order, rounded to storage: a step of the sum and what fp32 loses of the terms.
    terms = dy[-last:].double().abs().sum(0)
    for got, want, size in ((db, db_alone, terms), (dw, dw_alone, terms * hidden ** 0.5)):
        assert ((got.double() - want.double()).abs() <= want.double().abs() * torch.finfo(dtype).eps + 2.0 ** -21 * size).all()


def test_gradient_against_differences(device):
    """Along a direction in x, w and b: central differences of the formula in 64 bits. Their error is h^2/6 of the third derivative
    (below 1e3 here, h = 1e-4) and 2^-53/h of the loss's terms."""
    rows, hidden = 6, 48
    x, w, b, dy = inputs(rows, hidden, torch.float32, device)
    dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty_like(w)
    ops.layernorm_backward(dx, dw, db, dy, x, w, EPS)
    directions = [randn(t.shape, torch.float32, 31 + i).double().to(device) for i, t in enumerate((x, w, b))]

    def loss(step):
        a, c, d = (t.double() + step * v for t, v in zip((x, w, b), directions))
        return (reference(a, c, d, None, None)["y"] * dy.double()).sum().item()

    h = 1e-4
    slope = (loss(h) - loss(-h)) / (2 * h)
    got = sum((g.double() * v).sum().item() for g, v in zip((dx, dw, db), directions))
    magnitude = sum((g.double() * v).abs().sum().item() for g, v in zip((dx, dw, db), directions))
    assert abs(slope - got) <= 2e-5 + U32 * 64 * magnitude


def test_captured_calls(device):
    """Recorded behind an eager run, replayed with other inputs and eager work between."""
    x, w, b, dy = inputs(200, 1024, torch.bfloat16, device)
    y, dx, dw, db = torch.empty_like(x), torch.empty_like(x), torch.empty_like(w), torch.empty_like(w)
    stream = torch.cuda.Stream()

    def both():
        ops.layernorm_forward(y, x, w, b, EPS)
        ops.layernorm_backward(dx, dw, db, dy, x, w, EPS)

    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        both()
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream, capture_error_mode="thread_local"):
        both()
    for seed in range(4):
        x.copy_(randn(x.shape, x.dtype, 50 + seed))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (y, dx, dw, db)]
        for t in (y, dx, dw, db):
            t.zero_()
        both()
        torch.cuda.synchronize()
        for a, c in zip(got, (y, dx, dw, db)):
            assert torch.equal(a, c)


def test_on_another_stream(device):
    x, w, b, dy = inputs(500, 1024, torch.float16, device)
    want = [torch.empty_like(t) for t in (x, w, w)]
    ops.layernorm_backward(*want, dy, x, w, EPS)
    torch.cuda.synchronize()
    got = [torch.empty_like(t) for t in (x, w, w)]
    side = torch.cuda.Stream()
    ops.layernorm_backward(*got, dy, x, w, EPS, side)
    side.synchronize()
    for a, c in zip(want, got):
        assert torch.equal(a, c)


def test_launches(device):
    """What a call enqueues: forward one kernel."""
    x, w, b, _ = inputs(64, 1024, torch.bfloat16, device)
    y = torch.empty_like(x)
    assert launches(lambda: ops.layernorm_forward(y, x, w, b, EPS)) == 1
