"""The norms between two branches through the operator interface, against the formulas in 64 bits (linear_oracle.py has the bounds)."""
import pytest
import torch

from cgpt_amd import capi, ops
from tests.linear_oracle import check, sandwich_backward, sandwich_forward
from tests.util import DTYPE_IDS, DTYPES, randn

pytestmark = pytest.mark.gpu
EPS = 1e-5

# Rows and widths around what lanes, wavefronts and workgroups hold; rows that are longer; one gate, some, one for each row, none.
CASES = [(1, 1, 0), (1, 1, 1), (3, 7, 3), (5, 8, 0), (64, 63, 4), (12, 128, 2), (33, 129, 33), (100, 255, 1), (9, 256, 3), (50, 511, 10), (40, 512, 0),
         (16, 768, 16), (7, 1000, 7), (30, 1001, 5), (6000, 64, 3000), (2500, 64, 1), (24, 1024, 3), (9, 2048, 9), (10, 2050, 2), (4, 4096, 4), (5, 5000, 0),
         (6, 8192, 3), (3, 16384, 3), (2, 16385, 0), (70, 20001, 70), (8, 33000, 2), (700, 1024, 700)]
IDS = ["-".join(map(str, c)) for c in CASES]


def inputs(rows, hidden, gates, dtype, device, seed=1):
    x, f, d_stream, dy = (randn((rows, hidden), dtype, seed + i).to(device) for i in range(4))
    u, w = (randn((hidden,), dtype, seed + 4 + i).to(device) for i in range(2))
    gate = randn((gates, hidden), dtype, seed + 6).to(device) if gates else None
    return x, f, u, gate, w, d_stream, dy


def fresh(*like):
    return [None if t is None else torch.full_like(t, float("nan")) for t in like]


def run(x, f, u, gate, w, d_stream, dy, scale=0.7, stream=None):
    s, y, dx, df, du, dgate, dw = fresh(x, x, x, x, u, gate, w)
    ops.sandwich_norm_forward(s, y, x, f, u, gate, w, scale, EPS, stream)
    ops.sandwich_norm_backward(dx, df, du, dgate, dw, d_stream, dy, s, f, u, gate, w, scale, EPS, stream)
    return {"stream": s, "y": y, "dx": dx, "df": df, "du": du, "d_gate": dgate, "dw": dw}


def check_all(got, x, f, u, gate, w, d_stream, dy, scale=0.7):
    want = {**sandwich_forward(x, f, u, gate, w, scale, EPS, got["stream"]), **sandwich_backward(got["stream"], f, u, gate, w, scale, EPS, d_stream, dy)}
    for name, bound in want.items():
        check(got[name], bound, name)


@pytest.mark.parametrize("dtype", DTYPES, ids=DTYPE_IDS)
@pytest.mark.parametrize("c", CASES, ids=IDS)
def test_against_the_formula(device, c, dtype):
    given = inputs(*c, dtype, device)
    check_all(run(*given), *given)


@pytest.mark.parametrize("dtype", DTYPES, ids=DTYPE_IDS)
@pytest.mark.parametrize("c", [(20, 200, 5), (8, 1000, 0), (4, 20000, 4)], ids=str)
def test_without_what_is_optional_and_in_place(device, c, dtype):
    x, f, u, gate, w, d_stream, dy = given = inputs(*c, dtype, device)
    want = run(*given)
    # The stream in place, its gradient in place: the same bits.
    s, y = x.clone(), torch.empty_like(x)
    ops.sandwich_norm_forward(s, y, s, f, u, gate, w, 0.7, EPS)
    assert torch.equal(s, want["stream"]) and torch.equal(y, want["y"])
    dx = d_stream.clone()
    df, du, dw = fresh(x, u, w)
    ops.sandwich_norm_backward(dx, df, du, None, dw, dx, dy, s, f, u, gate, w, 0.7, EPS)
    for got, name in ((dx, "dx"), (df, "df"), (du, "du"), (dw, "dw")):
        assert torch.equal(got, want[name]), name
    # No gradient but the norm's own.
    dx, df, du, dgate, dw = fresh(x, x, u, gate, w)
    ops.sandwich_norm_backward(dx, df, du, dgate, dw, None, dy, s, f, u, gate, w, 0.7, EPS)
    bounds = sandwich_backward(s, f, u, gate, w, 0.7, EPS, None, dy)
    for got, name in ((dx, "dx"), (df, "df"), (du, "du"), (dgate, "d_gate"), (dw, "dw")):
        if got is not None:
            check(got, bounds[name], name)


@pytest.mark.parametrize("dtype", DTYPES, ids=DTYPE_IDS)
@pytest.mark.parametrize("c", [(6, 64, 3), (10, 1000, 0), (3, 20000, 3)], ids=str)
def test_off_the_boundaries_and_between_guards(device, c, dtype):
    given = inputs(*c, dtype, device)

    def shifted(t, fill=None):
        if t is None:
            return None, None
        whole = torch.full((t.numel() + 17,), 7.0, dtype=t.dtype, device=device)
        view = whole[1:1 + t.numel()].view(t.shape)
        view.copy_(t) if fill is None else view.fill_(fill)
        return whole, view

    x, f, u, gate, w, d_stream, dy = (shifted(t)[1] for t in given)
    held = {name: shifted(t, float("nan")) for name, t in zip(("stream", "y", "dx", "df", "du", "d_gate", "dw"), (x, x, x, x, u, gate, w))}
    got = {name: view for name, (_, view) in held.items()}
    ops.sandwich_norm_forward(got["stream"], got["y"], x, f, u, gate, w, 0.7, EPS)
    ops.sandwich_norm_backward(got["dx"], got["df"], got["du"], got["d_gate"], got["dw"], d_stream, dy, got["stream"], f, u, gate, w, 0.7, EPS)
    check_all(got, *given)
    for whole, view in held.values():
        assert whole is None or (whole[0] == 7 and (whole[1 + view.numel():] == 7).all())


@pytest.mark.parametrize("dtype", DTYPES, ids=DTYPE_IDS)
def test_rows_of_nothing_and_rows_that_are_not_finite(device, dtype):
    """A row of zeros is normed by epsilon alone; a row that is not finite spoils itself, and of the gradients its columns' sums."""
    x, f, u, gate, w, d_stream, dy = inputs(9, 300, 3, dtype, device)
    x[4], f[4] = 0, 0
    given = (x, f, u, gate, w, d_stream, dy)
    got = run(*given)
    check_all(got, *given)
    assert (got["y"][4] == 0).all()
    spoilt = f.clone()
    spoilt[7, 11] = float("nan")
    others = torch.arange(9, device=device) != 7
    again = run(x, spoilt, u, gate, w, d_stream, dy)
    for name in ("stream", "y", "dx", "df"):
        assert torch.equal(again[name][others], got[name][others]) and again[name][7].isnan().any(), name
    assert torch.equal(again["d_gate"][:2], got["d_gate"][:2]) and again["d_gate"][2].isnan().all()


def test_differences(device):
    """fp32: the outputs' change along a direction against the gradients' product with it. A step of 2^-7 along a unit direction leaves
    cubic terms of a central difference (2^-14 of a value of a few) and the outputs' rounding, 2^-24 rows hidden / 2^-7."""
    given = list(inputs(6, 50, 3, torch.float32, device))
    d_stream, dy = given[5:]
    got = run(*given, scale=0.7)
    for at, name in ((0, "dx"), (1, "df"), (2, "du"), (3, "d_gate"), (4, "dw")):
        direction = randn(given[at].shape, torch.float32, 40 + at).to(device)
        direction /= direction.norm()
        ends = []
        for sign in (1, -1):
            moved = list(given)
            moved[at] = given[at] + sign * 2.0 ** -7 * direction
            r = run(*moved)
            ends.append(((r["stream"].double() * d_stream.double()).sum() + (r["y"].double() * dy.double()).sum()).item())
        slope = (ends[0] - ends[1]) * 2.0 ** 6
        assert abs(slope - (got[name].double() * direction.double()).sum().item()) <= 2.0 ** -14 * 100 + 2.0 ** -24 * 300 * 4 * 2 ** 6, name


@pytest.mark.parametrize("dtype", DTYPES, ids=DTYPE_IDS)
@pytest.mark.parametrize("c", [(600, 512, 4), (50, 20000, 5)], ids=str)
def test_recorded(device, c, dtype):
    x, f, u, gate, w, d_stream, dy = given = inputs(*c, dtype, device)
    capi.call("cgptx_release_scratch")
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        eager = run(*given)
    stream.synchronize()
    held = {name: torch.zeros_like(t) for name, t in eager.items()}
    with torch.cuda.graph(graph, stream=stream, capture_error_mode="thread_local"):
        ops.sandwich_norm_forward(held["stream"], held["y"], x, f, u, gate, w, 0.7, EPS)
        ops.sandwich_norm_backward(held["dx"], held["df"], held["du"], held["d_gate"], held["dw"], d_stream, dy, held["stream"], f, u, gate, w, 0.7, EPS)
    for _ in range(3):
        for t in held.values():
            t.fill_(5.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(held[name], eager[name]) for name in eager)
        run(*inputs(40, 300, 4, dtype, device, 30))  # other work between replays
    check_all(held, *given)


def test_refusals_by_shape(device):
    x, f, u, gate, w, _, dy = inputs(6, 32, 3, torch.bfloat16, device)
    s, y = torch.empty_like(x), torch.empty_like(x)
    for args in ((s[:5], y, x, f, u, gate, w), (s, y, x, f[:, :16].contiguous(), u, gate, w), (s, y, x, f, u[:16], gate, w), (s, y, x, f, u, torch.cat([gate, gate[:1]]), w),
                 (s, y, x, f, u, gate[:, :16].contiguous(), w), (s, y, x, f, u, gate.t().contiguous(), w), (s, y, x, f.float(), u, gate, w),
                 (s, y, x, f, u, gate, w.float()), (s, y, x, f.t().contiguous().t(), u, gate, w), (s, y, x.cpu(), f, u, gate, w),
                 (s, y, x, f, u, gate.float(), w)):
        with pytest.raises(ValueError):
            ops.sandwich_norm_forward(*args, 1.0, EPS)
    for scale, eps in ((float("nan"), EPS), (float("inf"), EPS), (1.0, 0.0), (1.0, -1.0), (1.0, float("nan"))):
        with pytest.raises(ValueError):
            ops.sandwich_norm_forward(s, y, x, f, u, gate, w, scale, eps)
    dx, df, du, dgate, dw = fresh(x, x, u, gate, w)
    for args in ((dx, df, du, dgate, dw, None, dy[:5], x, f, u, gate, w), (dx, df, du[:16], dgate, dw, None, dy, x, f, u, gate, w),
                 (dx, df, du, dgate[:1], dw, None, dy, x, f, u, gate, w), (dx, df, du, dgate, dw, None, dy, x, f, u, None, w),
                 (dx, df, du, dgate, dw, dy.float(), dy, x, f, u, gate, w)):
        with pytest.raises(ValueError):
            ops.sandwich_norm_backward(*args, 1.0, EPS)
