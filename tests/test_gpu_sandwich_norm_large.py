"""The norms between two branches over 2^31 elements and more: rows in registers and rows of any length, looked at where offsets pass 31 bits, and the sums
over all rows."""
import pytest
import torch

from cgpt_amd import ops
from tests.linear_oracle import check, sandwich_backward, sandwich_forward

pytestmark = pytest.mark.gpu
EPS = 1e-5


@pytest.mark.parametrize("rows,hidden,gates", [(3 * 700001, 1024, 3), (2 * 55001, 20001, 0)], ids=str)
def test_offsets_past_31_bits(device, rows, hidden, gates):
    g = torch.Generator(device=device).manual_seed(5)
    x, f, d_stream, dy = (torch.randn((rows, hidden), dtype=torch.bfloat16, device=device, generator=g) for _ in range(4))
    u, w = (torch.randn(hidden, dtype=torch.bfloat16, device=device, generator=g) for _ in range(2))
    gate = torch.randn((gates, hidden), dtype=torch.bfloat16, device=device, generator=g) if gates else None
    s, y, dx, df = (torch.full_like(x, float("nan")) for _ in range(4))
    du, dw, dgate = torch.empty_like(u), torch.empty_like(w), None if gate is None else torch.empty_like(gate)
    ops.sandwich_norm_forward(s, y, x, f, u, gate, w, 0.7, EPS)
    ops.sandwich_norm_backward(dx, df, du, dgate, dw, d_stream, dy, s, f, u, gate, w, 0.7, EPS)
    some = slice(rows - 300, None)
    last = None if gate is None else gate[-1:]
    part = [t[some] for t in (x, f, d_stream, dy, s)]
    want = {**sandwich_forward(part[0], part[1], u, last, w, 0.7, EPS, part[4]), **sandwich_backward(part[4], part[1], u, last, w, 0.7, EPS, part[2], part[3])}
    for name, got in (("stream", s), ("y", y), ("dx", dx), ("df", df)):
        check(got[some], want[name], name)
    # The sums: each row's terms in 64 bits, a few thousand rows at a time.
    sums, per_gate, step = {}, rows // max(gates, 1), 5000
    for first in range(0, rows, per_gate):
        for at in range(first, first + per_gate, step):
            r = slice(at, min(at + step, first + per_gate))
            b = sandwich_backward(s[r], f[r], u, None if gate is None else gate[first // per_gate:first // per_gate + 1], w, 0.7, EPS, d_stream[r], dy[r])
            for name in ("du", "dw", "d_gate"):
                if name in b:
                    key = (name, first // per_gate if name == "d_gate" else 0)
                    sums[key] = sums.get(key, 0.0) + b[name].value.view(-1)
    # Terms of random signs: the sum's size is sqrt(rows) of a term's. Each is off by some hundred fp32 steps at most, a workgroup's sum of n rows in
    # turn by 2^-24 n of its terms' sum: 2^-24 rows of a term for all, 2^-24 sqrt(rows) of the result's 2-norm, and the result by a half step.
    tolerance = 2.0 ** -24 * (rows ** 0.5 + 100) + 2.0 ** -8
    results = [("du", 0, du), ("dw", 0, dw)] + [("d_gate", i, dgate[i]) for i in range(gates)]
    for name, i, got in results:
        off = ((got.double() - sums[name, i]).norm() / sums[name, i].norm()).item()
        assert off <= tolerance, f"{name} {i}: {off:.3g} of its norm, allowed {tolerance:.3g}"
