"""Linear attention with a decay through the operator interface, against the formulas in 64 bits (linear_oracle.py has the bounds)."""
import pytest
import torch

from cgpt_amd import capi, ops
from tests.linear_oracle import check, linear_backward, linear_forward, linear_step
from tests.util import DTYPE_IDS, DTYPES, randn

pytestmark = pytest.mark.gpu
GRADS = ("dq", "dk", "dv", "d_before")


def case(b, t, hq, hkv, d, states=True, scale=0.0, decay=None):
    return dict(b=b, t=t, hq=hq, hkv=hkv, d=d, states=states, scale=scale, decay=decay)


# One token; lengths around chunks and around what is cut into segments; every way a head can be wide; groups of one to eight.
CASES = [case(1, 1, 1, 1, 1), case(1, 1, 2, 1, 128), case(3, 2, 4, 2, 64, False), case(1, 63, 2, 1, 8), case(2, 64, 3, 3, 64), case(1, 65, 8, 1, 128),
         case(2, 66, 2, 2, 24, False), case(1, 127, 6, 2, 33), case(1, 128, 5, 1, 40), case(2, 129, 4, 1, 96, False), case(1, 191, 2, 1, 100),
         case(1, 257, 7, 7, 72), case(2, 500, 4, 2, 128), case(1, 1000, 6, 2, 64, False), case(1, 1025, 2, 1, 127), case(40, 70, 8, 4, 64),
         case(1, 4097, 2, 1, 64), case(100, 130, 4, 2, 128), case(2, 333, 4, 2, 16, scale=0.3), case(1, 300, 2, 1, 65, scale=2.0)]
IDS = ["-".join(str(v) for v in c.values()) for c in CASES]


def options(c):
    return ops.FlashAttentionOptions(num_query_heads=c["hq"], num_kv_heads=c["hkv"], head_dim=c["d"], attention_scale=c["scale"])


def inputs(c, dtype, device, seed=1, size=1.0):
    q_shape, kv_shape, s_shape = (c["b"], c["t"], c["hq"], c["d"]), (c["b"], c["t"], c["hkv"], c["d"]), (c["b"], c["hkv"], c["d"], c["d"])
    q, k, v, dout = (randn(s, dtype, seed + i, size).to(device) for i, s in enumerate((q_shape, kv_shape, kv_shape, q_shape)))
    before, d_after = (randn(s_shape, torch.float32, seed + 5 + i).to(device) if c["states"] else None for i in range(2))
    decays = c["decay"] or [-0.02, -1e-4, -0.5, 0.0, -3.0, -0.1, -0.003]
    log_decay = torch.tensor([decays[i % len(decays)] for i in range(c["hkv"])], device=device)
    return q, k, v, dout, log_decay, before, d_after


def forward(c, q, k, v, log_decay, before, out=None, after=None, stream=None):
    out = torch.full_like(q, float("nan")) if out is None else out
    if after is None:
        after = torch.full((c["b"], c["hkv"], c["d"], c["d"]), float("nan"), device=q.device)
    ops.linear_attention_forward(out, after, q, k, v, log_decay, before, stream, options(c))
    return out, after


def backward(c, q, k, v, dout, log_decay, before, d_after, grads=None, accumulate=False, stream=None):
    if grads is None:
        grads = tuple(torch.full_like(t, float("nan")) for t in (q, k, v))
        grads += (torch.full((c["b"], c["hkv"], c["d"], c["d"]), float("nan"), device=q.device),)
    ops.linear_attention_backward(*grads, dout, d_after, q, k, v, log_decay, before, stream, options(c), accumulate)
    return grads


def run_and_check(c, dtype, device, size=1.0, seed=1):
    q, k, v, dout, log_decay, before, d_after = inputs(c, dtype, device, seed, size)
    want = {**linear_forward(q, k, v, log_decay, before, c["scale"]), **linear_backward(q, k, v, log_decay, before, dout, d_after, c["scale"])}
    for name, got in zip(("out", "after"), forward(c, q, k, v, log_decay, before)):
        check(got, want[name], name)
    for name, got in zip(GRADS, backward(c, q, k, v, dout, log_decay, before, d_after)):
        check(got, want[name], name)


@pytest.mark.parametrize("dtype", DTYPES, ids=DTYPE_IDS)
@pytest.mark.parametrize("c", CASES, ids=IDS)
def test_against_the_formula(device, c, dtype):
    run_and_check(c, dtype, device)


@pytest.mark.parametrize("dtype", DTYPES, ids=DTYPE_IDS)
@pytest.mark.parametrize("decay", [[0.0], [-float("inf")], [-1e-7], [-88.0], [-2000.0]], ids=str)
def test_decays(device, decay, dtype):
    run_and_check(case(2, 200, 4, 2, 64, decay=decay), dtype, device)
    run_and_check(case(1, 700, 2, 1, 33, decay=decay), dtype, device)


def test_growth_counts_as_none(device):
    c = case(1, 150, 4, 2, 64)
    q, k, v, _, _, before, _ = inputs(c, torch.bfloat16, device)
    none, growing = torch.zeros(2, device=device), torch.tensor([0.5, float("inf")], device=device)
    assert all(torch.equal(a, b) for a, b in zip(forward(c, q, k, v, none, before), forward(c, q, k, v, growing, before)))


@pytest.mark.parametrize("size", [1e-3, 8.0], ids=["small", "large"])
def test_half_precision_range(device, size):
    """Scores and matrices that leave the range of half precision on the way, results that do not."""
    c = case(1, 300, 2, 1, 64, scale=1e-3 if size > 1 else 2.0, decay=[-0.01])
    run_and_check(c, torch.float16, device, size)


@pytest.mark.parametrize("dtype", DTYPES, ids=DTYPE_IDS)
def test_accumulated(device, dtype):
    for c in (case(2, 130, 4, 2, 64), case(1, 90, 3, 1, 35)):
        q, k, v, dout, log_decay, before, d_after = inputs(c, dtype, device)
        want = linear_backward(q, k, v, log_decay, before, dout, d_after, c["scale"])
        there = tuple(randn(t.shape, dtype, 50 + i).to(device) for i, t in enumerate((q, k, v)))
        state = torch.zeros_like(before)
        grads = backward(c, q, k, v, dout, log_decay, before, d_after, tuple(t.clone() for t in there) + (state,), True)
        step = max(torch.finfo(dtype).eps / 2, 2.0 ** -24)
        for name, got, was in zip(GRADS, grads, there):
            want[name].value += was.double()
            want[name].error += step * (was.double().abs() + want[name].value.abs())
            check(got, want[name], name)


@pytest.mark.parametrize("dtype", DTYPES, ids=DTYPE_IDS)
def test_without_what_is_optional(device, dtype):
    c = case(2, 140, 4, 2, 64)
    q, k, v, dout, log_decay, before, d_after = inputs(c, dtype, device)
    out = torch.full_like(q, float("nan"))
    ops.linear_attention_forward(out, None, q, k, v, log_decay, before, None, options(c))
    check(out, linear_forward(q, k, v, log_decay, before, 0.0)["out"], "out")
    for first, last in ((before, None), (None, d_after)):
        grads = tuple(torch.full_like(t, float("nan")) for t in (q, k, v))
        ops.linear_attention_backward(*grads, None, dout, last, q, k, v, log_decay, first, None, options(c))
        want = linear_backward(q, k, v, log_decay, first, dout, last, 0.0)
        for name, got in zip(GRADS, grads):
            check(got, want[name], name)


@pytest.mark.parametrize("dtype", DTYPES, ids=DTYPE_IDS)
@pytest.mark.parametrize("c", [case(2, 70, 4, 2, 64), case(1, 333, 2, 1, 128)], ids=["short", "long"])
def test_off_the_boundaries_and_between_guards(device, c, dtype):
    """Tensors one element behind a boundary of 16 bytes, in buffers whose other elements stay."""
    q, k, v, dout, log_decay, before, d_after = inputs(c, dtype, device)

    def shifted(t, fill=None):
        whole = torch.full((t.numel() + 17,), 7.0, dtype=t.dtype, device=device)
        view = whole[1:1 + t.numel()].view(t.shape)
        view.copy_(t) if fill is None else view.fill_(fill)
        return whole, view

    held = [shifted(t) for t in (q, k, v, dout, before, d_after)]
    q1, k1, v1, do1, before1, d_after1 = (view for _, view in held)
    outs = [shifted(t, float("nan")) for t in (q, before, q, k, v, before)]
    o, after, dq, dk, dv, d_before = (view for _, view in outs)
    forward(c, q1, k1, v1, log_decay, before1, o, after)
    backward(c, q1, k1, v1, do1, log_decay, before1, d_after1, (dq, dk, dv, d_before))
    want = {**linear_forward(q, k, v, log_decay, before, 0.0), **linear_backward(q, k, v, log_decay, before, dout, d_after, 0.0)}
    for name, got in zip(("out", "after", *GRADS), (o, after, dq, dk, dv, d_before)):
        check(got, want[name], name)
    for whole, view in outs:
        assert whole[0] == 7 and (whole[1 + view.numel():] == 7).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=DTYPE_IDS)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")], ids=str)
@pytest.mark.parametrize("t0", [0, 40, 130])
def test_what_is_not_finite_stays_where_it_is_seen(device, t0, bad, dtype):
    c = case(1, 200, 4, 2, 64, decay=[-0.02])
    q, k, v, dout, log_decay, before, d_after = inputs(c, dtype, device)
    want = {**linear_forward(q, k, v, log_decay, before, 0.0), **linear_backward(q, k, v, log_decay, before, dout, d_after, 0.0)}

    def finite_part(got, name, hidden):
        w = want[name]
        assert not torch.isfinite(got[hidden]).any(), name
        error = (got.double() - w.value).abs()
        assert bool((error <= w.error)[~hidden].all()), name

    def mask(t, at):
        m = torch.zeros_like(t, dtype=torch.bool)
        m[at] = True
        return m

    broken = v.clone()  # one value: its own column of its group's heads from there on
    broken[0, t0, 1, 5] = bad
    out, after = forward(c, q, k, broken, log_decay, before)
    finite_part(out, "out", mask(out, (0, slice(t0, None), slice(2, 4), 5)))
    finite_part(after, "after", mask(after, (0, 1, slice(None), 5)))
    broken = q.clone()  # a query: its own token
    broken[0, t0, 1, 5] = bad
    out, after = forward(c, broken, k, v, log_decay, before)
    finite_part(out, "out", mask(out, (0, t0, 1)))
    finite_part(after, "after", mask(after, (0, 0, 0, 0)) & False)
    broken = k.clone()
    broken[0, t0, 1, 5] = bad
    out, after = forward(c, q, broken, v, log_decay, before)
    finite_part(out, "out", mask(out, (0, slice(t0, None), slice(2, 4))))
    finite_part(after, "after", mask(after, (0, 1, 5)))
    broken = dout.clone()  # a gradient: its own query, and keys and values up to it
    broken[0, t0, 1, 5] = bad
    dq, dk, dv, d_before = backward(c, q, k, v, broken, log_decay, before, d_after)
    finite_part(dq, "dq", mask(dq, (0, t0, 1)))
    finite_part(dk, "dk", mask(dk, (0, slice(0, t0 + 1), 0)))
    finite_part(dv, "dv", mask(dv, (0, slice(0, t0 + 1), 0, 5)))
    finite_part(d_before, "d_before", mask(d_before, (0, 0, slice(None), 5)))


@pytest.mark.parametrize("dtype", DTYPES, ids=DTYPE_IDS)
def test_differences(device, dtype):
    """Every result is linear in q, in k and v apart and in the state: a difference of two outputs is the gradient's product with the step, but for the
    bounds of both."""
    c = case(1, 150, 4, 2, 48)
    q, k, v, dout, log_decay, before, d_after = inputs(c, dtype, device)
    grads = backward(c, q, k, v, dout, log_decay, before, d_after)
    want = linear_backward(q, k, v, log_decay, before, dout, d_after, 0.0)
    given = [q, k, v, before]
    for i, name in enumerate(GRADS):
        step = randn(given[i].shape, dtype, 70 + i).to(device).to(given[i].dtype)
        moved = list(given)
        moved[i] = given[i] + step
        step = moved[i].double() - given[i].double()  # what is left of it after rounding
        slope, slack = 0.0, (want[name].error * step.abs()).sum().item()
        for sign, (q1, k1, v1, s1) in ((1, moved), (-1, given)):
            out, after = forward(c, q1, k1, v1, log_decay, s1)
            there = linear_forward(q1, k1, v1, log_decay, s1, 0.0)
            slope += sign * ((out.double() * dout.double()).sum() + (after.double() * d_after.double()).sum()).item()
            slack += ((there["out"].error * dout.double().abs()).sum() + (there["after"].error * d_after.double().abs()).sum()).item()
        assert abs(slope - (grads[i].double() * step).sum().item()) <= slack, name


@pytest.mark.parametrize("dtype", DTYPES, ids=DTYPE_IDS)
@pytest.mark.parametrize("b,hq,hkv,d", [(1, 1, 1, 1), (1, 8, 2, 128), (3, 6, 2, 33), (7, 9, 1, 64), (300, 4, 4, 40), (2, 5, 5, 127), (2, 12, 2, 96)])
def test_step(device, b, hq, hkv, d, dtype):
    c = case(b, 1, hq, hkv, d)
    q, k, v, _, log_decay, state, _ = inputs(c, dtype, device)
    want = linear_step(q, k, v, log_decay, state, 0.0)
    out, after = torch.full_like(q, float("nan")), torch.full_like(state, float("nan"))
    ops.linear_attention_step(out, after, state, q, k, v, log_decay, None, options(c))
    check(out, want["out"], "out")
    check(after, want["after"], "after")
    again = torch.full_like(q, float("nan"))
    ops.linear_attention_step(again, state, state, q, k, v, log_decay, None, options(c))  # in place
    assert torch.equal(again, out) and torch.equal(state, after)


@pytest.mark.parametrize("dtype", DTYPES, ids=DTYPE_IDS)
def test_step_off_the_boundaries(device, dtype):
    c = case(3, 1, 4, 2, 64)
    q, k, v, _, log_decay, state, _ = inputs(c, dtype, device)
    whole = torch.full((state.numel() + 9,), 7.0, device=device)
    view = whole[1:1 + state.numel()].view(state.shape)
    out = torch.empty_like(q)
    ops.linear_attention_step(out, view, state, q, k, v, log_decay, None, options(c))
    want = linear_step(q, k, v, log_decay, state, 0.0)
    check(out, want["out"], "out")
    check(view, want["after"], "after")
    assert whole[0] == 7 and (whole[1 + state.numel():] == 7).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=DTYPE_IDS)
def test_pieces_and_single_tokens(device, dtype):
    """A prompt in pieces, whose state the next one starts from, then token by token: the outputs of one call. A state that came through m calls
    carries their bounds, decayed."""
    c = case(2, 181, 6, 2, 64, decay=[-0.01, -0.2])
    q, k, v, _, log_decay, before, _ = inputs(c, dtype, device)
    whole = linear_forward(q, k, v, log_decay, before, 0.0)
    state, at, outs, lost = before, 0, [], torch.zeros_like(before, dtype=torch.float64)
    for length in (1, 64, 7, 100):
        piece = dict(c, t=length)
        part = [t[:, at:at + length].contiguous() for t in (q, k, v)]
        lost = linear_forward(*part, log_decay, state, 0.0)["after"].error + lost
        out, state = forward(piece, *part, log_decay, state)
        outs.append(out)
        at += length
    for t in range(at, c["t"]):
        one = [x[:, t:t + 1].contiguous() for x in (q, k, v)]
        out = torch.empty_like(one[0])
        lost = linear_step(*one, log_decay, state, 0.0)["after"].error + lost
        ops.linear_attention_step(out, state, state, *one, log_decay, None, options(c))
        outs.append(out)
    size = q.double().abs().sum(-1, keepdim=True) / 8 * lost.max()
    whole["out"].error += size
    whole["after"].error += lost
    check(torch.cat(outs, 1), whole["out"], "out")
    check(state, whole["after"], "after")


@pytest.mark.parametrize("dtype", DTYPES, ids=DTYPE_IDS)
@pytest.mark.parametrize("c", [case(1, 2000, 4, 2, 64), case(2, 60, 2, 1, 128)], ids=["cut", "whole"])
def test_recorded(device, c, dtype):
    """Recorded behind an eager call of its sizes a call has its bits; where the scratch arena has no room it stays within the bounds."""
    q, k, v, dout, log_decay, before, d_after = inputs(c, dtype, device)
    want = {**linear_forward(q, k, v, log_decay, before, 0.0), **linear_backward(q, k, v, log_decay, before, dout, d_after, 0.0)}
    results = [torch.zeros_like(t) for t in (q, before, q, k, v, before)]
    names = ("out", "after", *GRADS)

    def both():
        forward(c, q, k, v, log_decay, before, results[0], results[1])
        backward(c, q, k, v, dout, log_decay, before, d_after, results[2:])

    capi.call("cgptx_release_scratch")
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    graphs = []
    for eager_before in (False, True):
        if eager_before:
            with torch.cuda.stream(stream):
                both()
            stream.synchronize()
            eager = [t.clone() for t in results]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream, capture_error_mode="thread_local"):
            both()
        graphs.append(graph)
        for _ in range(3):
            for t in results:
                t.fill_(5.0)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            for got, name in zip(results, names):
                check(got, want[name], name)
            assert not eager_before or all(torch.equal(a, b) for a, b in zip(results, eager))
    graphs[0].replay()
    torch.cuda.synchronize()
    for got, name in zip(results, names):
        check(got, want[name], name)


def test_two_streams(device):
    """Calls side by side, each on its own stream with its own scratch, repeat their bits."""
    cs = [case(1, 3001, 4, 2, 64), case(1, 2500, 6, 2, 128)]
    given = [inputs(c, torch.bfloat16, device, seed=1 + 20 * i) for i, c in enumerate(cs)]
    alone = [(*forward(c, *g[:3], g[4], g[5]), *backward(c, *g)) for c, g in zip(cs, given)]
    streams = [torch.cuda.Stream() for _ in cs]
    torch.cuda.synchronize()
    for _ in range(5):
        together = []
        for c, g, stream in zip(cs, given, streams):
            with torch.cuda.stream(stream):
                together.append((*forward(c, *g[:3], g[4], g[5]), *backward(c, *g)))
        torch.cuda.synchronize()
        for one, other in zip(alone, together):
            assert all(torch.equal(a, b) for a, b in zip(one, other))


def test_offsets_past_32_bits(device):
    """2^31 elements and more in the queries, the outputs and their gradients. What is further than 300 tokens away has decayed to nothing (e^-150)."""
    c = case(1, (1 << 20) + 71, 16, 1, 128, states=False, decay=[-0.5])
    shape, kv = (1, c["t"], 16, 128), (1, c["t"], 1, 128)
    g = torch.Generator(device=device).manual_seed(3)
    q, dout = (torch.randn(shape, dtype=torch.bfloat16, device=device, generator=g) for _ in range(2))
    k, v = (torch.randn(kv, dtype=torch.bfloat16, device=device, generator=g) for _ in range(2))
    log_decay = torch.tensor([-0.5], device=device)
    out = torch.full_like(q, float("nan"))
    ops.linear_attention_forward(out, None, q, k, v, log_decay, None, None, options(c))
    end = slice(c["t"] - 500, None)
    part = [t[:, end].contiguous() for t in (q, k, v, dout)]
    want = linear_forward(*part[:3], log_decay, None, 0.0)["out"]
    check(out[:, end][:, 300:], type(want)(want.value[:, 300:], want.error[:, 300:]), "out")
    grads = [torch.full_like(t, float("nan")) for t in (out, k, v)]
    del out
    ops.linear_attention_backward(*grads, None, dout, None, q, k, v, log_decay, None, None, options(c))
    want = linear_backward(*part[:3], log_decay, None, part[3], None, 0.0)
    for name, got in zip(GRADS, grads):
        check(got[:, end][:, 300:], type(want[name])(want[name].value[:, 300:], want[name].error[:, 300:]), name)


def test_refusals_by_shape(device):
    c = case(2, 8, 4, 2, 16)
    q, k, v, dout, log_decay, before, _ = inputs(c, torch.bfloat16, device)
    out, after = torch.empty_like(q), torch.empty_like(before)
    o = options(c)

    def refused(*args, **more):
        with pytest.raises(ValueError):
            ops.linear_attention_forward(*args, **more)

    refused(out, after, q, k, v, log_decay.double(), before, None, o)
    refused(out, after, q, k, v, torch.zeros(3, device=device), before, None, o)
    refused(out, after, q, k, v, torch.zeros(4, device=device)[::2], before, None, o)
    refused(out, after.half(), q, k, v, log_decay, before, None, o)
    refused(out, after[:, :1], q, k, v, log_decay, before, None, o)
    refused(out, after.transpose(2, 3), q, k, v, log_decay, before, None, o)
    refused(out, before, q, k, v, log_decay, before, None, o)
    refused(out, after, q, k[:, :4].contiguous(), v[:, :4].contiguous(), log_decay, before, None, o)
    refused(out, after, q, k, v.float(), log_decay, before, None, o)
    refused(out[:1], after, q, k, v, log_decay, before, None, o)
    refused(out.transpose(1, 2), after, q, k, v, log_decay, before, None, o)
    refused(out, after, q, k, v, log_decay, before, None, ops.FlashAttentionOptions(num_query_heads=4, num_kv_heads=2, head_dim=16, causal=False))
    refused(out, after, q, k, v, log_decay, before, None,
            ops.FlashAttentionOptions(num_query_heads=4, num_kv_heads=2, head_dim=16, query_position_offset=1))
    refused(out, after, q, k, v, log_decay.cpu(), before, None, o)
    grads = (torch.empty_like(q), torch.empty_like(k), torch.empty_like(v))
    for bad in ((grads[1], *grads[1:], None), (*grads[:2], grads[2].float(), None), (*grads, before)):
        with pytest.raises(ValueError):
            ops.linear_attention_backward(*bad, dout, None, q, k, v, log_decay, before, None, o)
    q1, k1, v1 = (t[:, :1].contiguous() for t in (q, k, v))
    for args in ((q1.clone(), after, before, q1, k1, v1[..., :1, :].contiguous()), (q.clone(), after, before, q, k, v), (q1[:1], after, before, q1, k1, v1), (q1.clone(), after.half(), before, q1, k1, v1),
                 (q1.clone(), after, before[:1], q1, k1, v1)):
        with pytest.raises(ValueError):
            ops.linear_attention_step(*args, log_decay, None, o)
