"""Differential attention and the weights of its second maps through the operator interface against the formulas in 64 bits.

Tolerances, for every element. u = eps/2 of the storage type; the kernels round each probability and each score gradient to it
once before a product (relative to the value), and each result once. The backward pass is given the forward pass's rounded
outputs: delta2 = dO.O2 is then off by u sum|dO O2|, delta1 = dO.O + lambda delta2 by u sum|dO|(|O| + 2 lambda |O2|). What fp32
does to scores and exponentials is within C = 2^-24 (64 products + 32) (1 + max|score|) relative to a probability, and a sum of
n terms in fp32 within 2^-24 n of their magnitudes; 16-bit storage has both far below u.

Half precision rounds what is below 2^-14 by up to 2^-25 whatever its size, and the probabilities of a row of thousands of keys (5000
keys: 2e-4 on average, their difference less) and their score gradients get there. A factor that is off by 2^-25 adds 2^-25 of the
other factor: hence terms of 2^-25 sum|dO| for dv and 2^-25 s sum|k|, sum|q| for dq and dk. In the forward pass the factors
stand to the row's largest one, which is P's maximum times as much when all is done."""
import math

import pytest
import torch

from cgpt_amd import capi, ops
from tests.util import DTYPE_IDS, DTYPES, launches, randn

pytestmark = pytest.mark.gpu


def case(b, qs, ks, hq, hkv, d, causal=True, off=None, scale=0.0, **more):
    off = (ks - qs if causal else 0) if off is None else off
    return dict(b=b, qs=qs, ks=ks, hq=hq, hkv=hkv, d=d, causal=causal, off=off, scale=scale, **more)


# One token, one key; lengths around the tiles of 16, 32, 64 and 128; grouped and single heads; every way a head can be wide.
CASES = [case(1, 1, 1, 1, 1, 2), case(1, 1, 1, 2, 1, 128), case(2, 1, 77, 4, 2, 64), case(1, 5, 5, 3, 3, 20), case(2, 16, 16, 2, 2, 32),
         case(1, 31, 33, 2, 1, 48), case(2, 64, 64, 4, 2, 128), case(1, 65, 65, 4, 1, 96), case(3, 100, 100, 4, 2, 64),
         case(1, 127, 130, 2, 2, 112), case(1, 129, 129, 6, 2, 80), case(2, 200, 200, 3, 1, 36), case(1, 257, 300, 2, 1, 128),
         case(2, 70, 200, 4, 2, 128, off=13), case(1, 40, 100, 2, 2, 16), case(1, 90, 90, 2, 2, 6),
         case(2, 33, 150, 4, 2, 64, causal=False), case(1, 150, 33, 4, 4, 128, causal=False), case(1, 128, 256, 8, 2, 128, causal=False),
         case(1, 130, 130, 2, 1, 64, scale=0.4), case(1, 512, 512, 8, 8, 64), case(2, 333, 333, 8, 2, 128)]
IDS = ["-".join(str(v) for v in c.values()) for c in CASES]


def options(c):
    return ops.FlashAttentionOptions(num_query_heads=c["hq"], num_kv_heads=c["hkv"], head_dim=c["d"], attention_scale=c["scale"],
                                     causal=c["causal"], query_position_offset=c["off"])


def inputs(c, dtype, device, seed=1, size=1.0):
    q_shape, kv_shape = (c["b"], c["qs"], c["hq"], c["d"]), (c["b"], c["ks"], c["hkv"], c["d"])
    q, k, v, dout = (randn(s, dtype, seed + i, size).to(device) for i, s in enumerate((q_shape, kv_shape, kv_shape, q_shape)))
    lambdas = (0.2 + 0.6 * torch.rand(c["hq"], generator=torch.Generator().manual_seed(seed + 9))).to(device)
    return q, k, v, dout, lambdas


def heads_first(t, group=1):
    t = t.double().permute(0, 2, 1, 3)
    return t.repeat_interleave(group, dim=1) if group > 1 else t


def product(a, b):
    return torch.matmul(a.contiguous(), b.contiguous())


def reference(c, q, k, v, lambdas, dout=None, dtype=None, summed=False):
    """Results in 64 bits, [batch, sequence, heads, width], and their bounds; `summed`: for deltas that are rowsum(P G) in fp32, whatever
    the outputs were rounded to."""
    dtype = dtype or q.dtype
    u, f = torch.finfo(dtype).eps / 2, 2.0 ** -24
    if dtype == torch.float32:
        u = 0.0  # nothing is rounded on the way; the bounds' own terms stay
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    half, group = c["d"] // 2, c["hq"] // c["hkv"]
    scale = c["scale"] or 1 / math.sqrt(half)
    qh, kh, vh = heads_first(q), heads_first(k, group), heads_first(v, group)
    lam = lambdas.double().view(1, -1, 1, 1)
    position = torch.arange(c["qs"], device=q.device).view(-1, 1) + c["off"]
    hidden = (torch.arange(c["ks"], device=q.device).view(1, -1) > position) if c["causal"] else None
    maps, lses, top = [], [], 0.0
    for columns in (slice(0, half), slice(half, 2 * half)):
        s = product(qh[..., columns], kh[..., columns].transpose(2, 3)) * scale
        top = max(top, s.abs().max().item())
        if hidden is not None:
            s = s.masked_fill(hidden, -math.inf)
        lses.append(torch.logsumexp(s, -1))
        maps.append(torch.exp(s - lses[-1][..., None]))
    p1, p2 = maps
    soft = f * (64 + 32) * (1 + top)  # C
    o2 = product(p2, vh)
    out = product(p1, vh) - lam * o2
    n = c["ks"] + 8

    def back(t):
        return t.permute(0, 2, 1, 3)

    av1, av2 = product(p1, vh.abs()), product(p2, vh.abs())
    r = {"out": back(out), "second": back(o2), "lse": torch.stack([l.permute(0, 2, 1) for l in lses])}
    seen = torch.ones_like(p1) if hidden is None else (~hidden).double().expand_as(p1)
    small = tiny * product(seen, vh.abs())
    small1, small2 = (small * p.amax(-1, keepdim=True) for p in (p1, p2))
    r["out_err"] = back((u + 2 * soft + n * f) * (av1 + lam.abs() * av2) + small1 + lam.abs() * small2)
    r["second_err"] = back((u + 2 * soft + n * f) * av2 + small2)
    r["lse_err"] = 2 * soft + n * f + 4 * f * r["lse"].abs()
    if dout is None:
        return r
    do = heads_first(dout)
    g = product(do, vh.transpose(2, 3))
    g_err = f * (c["d"] + 8) * product(do.abs(), vh.abs().transpose(2, 3))
    d2 = (p2 * g).sum(-1, keepdim=True)
    d1 = (p1 * g).sum(-1, keepdim=True)
    # What delta is computed from are the forward pass's outputs, rounded to storage (fp32: half a step too) and within their bounds.
    step = torch.finfo(dtype).eps / 2
    o2_err = heads_first(r["second_err"]) + step * o2.abs()
    o_err = heads_first(r["out_err"]) + step * out.abs()
    d2_err = (do.abs() * o2_err).sum(-1, keepdim=True) + f * (c["d"] + 8) * (do * o2).abs().sum(-1, keepdim=True)
    d1_err = (do.abs() * o_err).sum(-1, keepdim=True) + lam.abs() * d2_err + 2 * f * (c["d"] + 8) * (do * out).abs().sum(-1, keepdim=True)
    # rowsum(P G) in fp32: the rounded delta comes back in with the sum of P's row, which is one to n f + 2 C.
    d1_sum, d2_sum = ((p * (g_err + (2 * soft + (n + 8) * f) * g.abs())).sum(-1, keepdim=True) + (2 * soft + (n + 8) * f) * (d.abs() + d_err) * 2
                      for p, d, d_err in ((p1, d1, d1_err), (p2, d2, d2_err)))
    if summed:
        d1_err, d2_err = d1_sum, d2_sum
    ds1, ds2 = p1 * (g - d1), -lam * p2 * (g - d2)
    spread1, spread2 = p1 * (g.abs() + d1.abs()), lam.abs() * p2 * (g.abs() + d2.abs())
    e1 = tiny * seen + u * ds1.abs() + p1 * (d1_err + g_err) * (1 + u) + (2 * soft + 4 * f) * spread1
    e2 = tiny * seen * torch.clamp(lam.abs(), min=1.0) + u * ds2.abs() + lam.abs() * p2 * (d2_err + g_err) * (1 + u) + (2 * soft + 4 * f) * spread2
    k1, k2, q1, q2 = kh[..., :half], kh[..., half:], qh[..., :half], qh[..., half:]
    dq = torch.cat([product(ds1, k1), product(ds2, k2)], -1) * scale
    dq_err = torch.cat([product(e1 + n * f * spread1, k1.abs()), product(e2 + n * f * spread2, k2.abs())], -1) * scale
    m = c["qs"] * group + 24
    pd = p1 - lam * p2
    pd_err = tiny * seen + u * pd.abs() + (2 * soft + (m + 4) * f) * (p1 + lam.abs() * p2)

    def grouped(t):
        return t.view(c["b"], c["hkv"], group, *t.shape[2:]).sum(2)

    t12 = lambda t: t.transpose(2, 3)  # noqa: E731
    dv, dv_err = grouped(product(t12(pd), do)), grouped(product(t12(pd_err), do.abs()))
    dk = grouped(torch.cat([product(t12(ds1), q1), product(t12(ds2), q2)], -1)) * scale
    dk_err = grouped(torch.cat([product(t12(e1 + m * f * spread1), q1.abs()), product(t12(e2 + m * f * spread2), q2.abs())], -1)) * scale
    for name, value in (("dq", dq), ("dq_err", dq_err), ("dk", dk), ("dk_err", dk_err), ("dv", dv), ("dv_err", dv_err)):
        r[name] = back(value)
    r["dlam"] = -d2.sum((0, 2, 3))
    r["dlam_err"] = d2_sum.sum((0, 2, 3)) + f * 64 * d2.abs().sum((0, 2, 3))
    return r


def check(got, want, err, what):
    bound = want.abs() * (torch.finfo(got.dtype).eps / 2) * 1.0001 + err * 1.0001 + (2.0 ** -24 if got.dtype == torch.float16 else 1e-30)
    assert torch.isfinite(got).all(), f"{what}: not finite"
    worst = ((got.double() - want).abs() / bound).max().item()
    print(f"[parity] {what}: {worst:.3f} of the bound")
    assert worst <= 1, f"{what}: {worst:.3f} times the bound"


def forward(c, q, k, v, lambdas, stream=None):
    out, second = torch.full_like(q, 7.0), torch.full_like(q, 7.0)
    lse = torch.full((2, *q.shape[:3]), 7.0, device=q.device)
    ops.differential_attention_forward(out, second, lse, q, k, v, lambdas, stream, options(c))
    return out, second, lse


def backward(c, q, k, v, dout, lambdas, saved, base=None, stream=None):
    grads = [torch.full_like(t, 3.0) for t in (q, k, v, lambdas)] if base is None else [t.clone() for t in base]
    ops.differential_attention_backward(*grads, dout, *saved, q, k, v, lambdas, stream, options(c), base is not None)
    return grads


GRADS = ("dq", "dk", "dv", "dlam")


@pytest.mark.parametrize("dtype", DTYPES, ids=DTYPE_IDS)
@pytest.mark.parametrize("c", CASES, ids=IDS)
def test_forward_and_backward(device, c, dtype):
    q, k, v, dout, lambdas = inputs(c, dtype, device)
    saved = forward(c, q, k, v, lambdas)
    want = reference(c, q, k, v, lambdas, dout)
    for got, name in zip(saved, ("out", "second", "lse")):
        check(got, want[name], want[name + "_err"], name)
    for got, name in zip(backward(c, q, k, v, dout, lambdas, saved), GRADS):
        check(got, want[name], want[name + "_err"], name)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_a_long_cache(device, dtype):
    """More than 2^31 elements of keys and values. The last key has scores of more than 32, the others 0: they share 2^21 e^-32 < 2^-25 of
    either map."""
    c = case(1, 1, (1 << 21) + 77, 8, 8, 128)
    q, _, _, dout, lambdas = inputs(dict(c, ks=1), dtype, device)
    k, v, dk, dv = (torch.zeros((1, c["ks"], 8, 128), dtype=dtype, device=device) for _ in range(4))
    v[:, :-1] = 1.0
    k[:, -1:], v[:, -1:] = q * 8.0, randn((1, 1, 8, 128), dtype, 40).to(device)
    scores = q.view(8, 2, 64).double().square().sum(-1)  # 8 times that / sqrt(64)
    assert scores.min() > 32
    lam, last, u = lambdas.double().view(1, 1, 8, 1), v[:, -1:].double(), torch.finfo(dtype).eps / 2
    # C of either map and what the other keys share, of values that are 1 or the last key's.
    rest = 2 * 2.0 ** -24 * (64 + 32) * (1 + scores.max().item()) + 2.0 ** -24
    out, second, lse = forward(c, q, k, v, lambdas)
    for got, want in ((second, last), (out, (1 - lam) * last)):
        assert ((got.double() - want).abs() <= want.abs() * u * 1.01 + 2 * rest * (1 + last.abs())).all()
    dq, dlambdas = torch.full_like(q, 7.0), torch.full_like(lambdas, 7.0)
    ops.differential_attention_backward(dq, dk, dv, dlambdas, dout, out, second, lse, q, k, v, lambdas, None, options(c))
    want = (1 - lam) * dout.double()  # the maps' difference is rounded to storage once, the result once more
    assert ((dv[:, -1:].double() - want).abs() <= want.abs() * 2.01 * u + 2 * rest * dout.double().abs()).all()
    assert dv[:, :-1].abs().max().item() <= 2 * rest * dout.abs().max().item()
    assert torch.isfinite(dq).all() and torch.isfinite(dk[:, -1:]).all()
    terms = dout.double() * last
    bound = (rest + 2.0 ** -24 * (128 + 8)) * (terms.abs() + dout.double().abs()).sum(-1).flatten()
    assert ((dlambdas.double() + terms.sum(-1).flatten()).abs() <= bound).all()


# Sequences of few tokens: a row's score gradients are differences of what its keys give, near nothing for the first rows.
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
@pytest.mark.parametrize("c", [case(3, 2, 2, 4, 2, 64), case(7, 4, 4, 4, 2, 128), case(1, 13, 13, 2, 1, 80), case(2, 64, 64, 2, 2, 32),
                               case(2, 100, 5, 2, 1, 128, causal=False), case(1, 300, 40, 2, 2, 64, causal=False)],
                         ids=["2", "4", "13", "64", "5-keys", "40-keys"])
def test_few_keys(device, c, dtype):
    q, k, v, dout, lambdas = inputs(c, dtype, device)
    want = reference(c, q, k, v, lambdas, dout, summed=True)
    for got, name in zip(backward(c, q, k, v, dout, lambdas, forward(c, q, k, v, lambdas)), GRADS):
        check(got, want[name], want[name + "_err"], name)


@pytest.mark.parametrize("dtype", DTYPES, ids=DTYPE_IDS)
@pytest.mark.parametrize("c", [case(2, 1, 1, 4, 2, 128), case(1, 150, 1, 4, 1, 64, causal=False), case(3, 7, 1, 2, 2, 36, causal=False)],
                         ids=["token", "queries", "narrow"])
def test_one_key_has_no_score_gradient(device, c, dtype):
    q, k, v, dout, lambdas = inputs(c, dtype, device)
    saved = forward(c, q, k, v, lambdas)
    dq, dk, _, _ = backward(c, q, k, v, dout, lambdas, saved)
    assert not dq.any() and not dk.any()
    base = [randn(t.shape, t.dtype, 50 + i).to(device) for i, t in enumerate((q, k, v, lambdas))]
    dq, dk, _, _ = backward(c, q, k, v, dout, lambdas, saved, base)
    assert torch.equal(dq, base[0]) and torch.equal(dk, base[1])


# A token or a few against many keys: the keys of a block of queries are shared by several workgroups, a group's heads share a block.
LONG = [case(1, 1, 3000, 8, 2, 128), case(2, 1, 700, 4, 1, 64), case(1, 1, 5000, 2, 2, 32), case(1, 7, 2000, 6, 2, 96), case(3, 21, 1100, 3, 1, 112),
        case(1, 22, 1100, 3, 1, 128), case(1, 30, 1500, 4, 4, 64, causal=False), case(1, 64, 2100, 2, 1, 128), case(1, 200, 2500, 1, 1, 128),
        case(1, 1000, 1000, 1, 1, 64), case(1, 2048, 2048, 10, 2, 128), case(2, 1600, 1700, 5, 5, 112, off=100), case(1, 1990, 1600, 20, 4, 64, causal=False),
        case(1, 3, 1300, 16, 1, 80, causal=False), case(1, 5, 900, 4, 2, 64, off=400)]


@pytest.mark.parametrize("dtype", DTYPES, ids=DTYPE_IDS)
@pytest.mark.parametrize("c", LONG, ids=["-".join(str(v) for v in c.values()) for c in LONG])
def test_few_queries_of_many_keys(device, c, dtype):
    q, k, v, dout, lambdas = inputs(c, dtype, device)
    saved = forward(c, q, k, v, lambdas)
    want = reference(c, q, k, v, lambdas, dout)
    for got, name in zip(saved, ("out", "second", "lse")):
        check(got, want[name], want[name + "_err"], name)
    for got, name in zip(backward(c, q, k, v, dout, lambdas, saved), GRADS):
        check(got, want[name], want[name + "_err"], name)
    again = forward(c, q, k, v, lambdas)
    assert all(torch.equal(a, b) for a, b in zip(saved, again))
    alone = torch.full_like(q, 7.0)
    ops.differential_attention_forward(alone, None, None, q, k, v, lambdas, None, options(c))
    assert torch.equal(alone, saved[0])


@pytest.mark.parametrize("dtype", DTYPES, ids=DTYPE_IDS)
def test_recorded_without_a_call_before(device, dtype):
    """A forward call asks for scratch only where it is faster with it: recorded first, it does without. A backward call says that it
    cannot."""
    c = case(1, 3, 2000, 4, 2, 64)
    q, k, v, dout, lambdas = inputs(c, dtype, device)
    want = reference(c, q, k, v, lambdas)
    out, second, lse = torch.zeros_like(q), torch.zeros_like(q), torch.zeros((2, *q.shape[:3]), device=device)
    grads = [torch.zeros_like(t) for t in (q, k, v, lambdas)]
    torch.cuda.synchronize()
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream, capture_error_mode="thread_local"):
        ops.differential_attention_forward(out, second, lse, q, k, v, lambdas, None, options(c))
        with pytest.raises(capi.CgptxCaptureError):
            ops.differential_attention_backward(*grads, dout, out, second, lse, q, k, v, lambdas, None, options(c))
    for _ in range(3):
        out.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for got, name in zip((out, second, lse), ("out", "second", "lse")):
            check(got, want[name], want[name + "_err"], name)


@pytest.mark.parametrize("dtype", DTYPES, ids=DTYPE_IDS)
@pytest.mark.parametrize("c", [case(2, 100, 100, 4, 2, 128), case(1, 70, 90, 2, 2, 36)], ids=["wide", "narrow"])
def test_gradients_are_added(device, c, dtype):
    q, k, v, dout, lambdas = inputs(c, dtype, device)
    saved = forward(c, q, k, v, lambdas)
    want = reference(c, q, k, v, lambdas, dout)
    base = [randn(t.shape, t.dtype, 40 + i).to(device) for i, t in enumerate((q, k, v, lambdas))]
    for got, name, before in zip(backward(c, q, k, v, dout, lambdas, saved, base), GRADS, base):
        check(got, want[name] + before.double(), want[name + "_err"] + 2.0 ** -22 * (want[name].abs() + before.double().abs()), name)


@pytest.mark.parametrize("dtype", DTYPES, ids=DTYPE_IDS)
def test_without_what_the_backward_pass_needs(device, dtype):
    for c in (case(2, 100, 100, 4, 2, 64), case(1, 20, 20, 2, 1, 10)):
        q, k, v, _, lambdas = inputs(c, dtype, device)
        out, second, lse = forward(c, q, k, v, lambdas)
        alone = torch.full_like(q, 7.0)
        ops.differential_attention_forward(alone, None, None, q, k, v, lambdas, None, options(c))
        assert torch.equal(alone, out)
        one = torch.full_like(q, 7.0)
        ops.differential_attention_forward(alone, one, None, q, k, v, lambdas, None, options(c))
        assert torch.equal(one, second)


@pytest.mark.parametrize("dtype", DTYPES, ids=DTYPE_IDS)
def test_equal_maps_cancel(device, dtype):
    """q1 = q2, k1 = k2, lambda = 1: both maps have the same bits, and nothing is left of the output or of the gradients of v. dk's halves
    are sums of terms of opposite signs, which the matrix unit does not round alike: they are held to the bounds of the formula, whose
    halves add up to zero."""
    c = case(2, 90, 90, 4, 2, 64)
    q, k, v, dout, lambdas = inputs(c, dtype, device)
    q[..., 32:] = q[..., :32]
    k[..., 32:] = k[..., :32]
    lambdas.fill_(1.0)
    saved = forward(c, q, k, v, lambdas)
    assert (saved[0] == 0).all() and torch.equal(saved[2][0], saved[2][1])
    dq, dk, dv, _ = backward(c, q, k, v, dout, lambdas, saved)
    assert (dv == 0).all() and torch.equal(dq[..., :32], -dq[..., 32:])
    want = reference(c, q, k, v, lambdas, dout)
    assert (want["dk"][..., :32] + want["dk"][..., 32:]).abs().max().item() <= 1e-12
    check(dk, want["dk"], want["dk_err"], "dk")


@pytest.mark.parametrize("dtype", DTYPES, ids=DTYPE_IDS)
@pytest.mark.parametrize("value", [0.0, -0.5, 3.0])
def test_any_weight(device, dtype, value):
    c = case(1, 65, 65, 2, 1, 64)
    q, k, v, dout, lambdas = inputs(c, dtype, device)
    lambdas.fill_(value)
    saved = forward(c, q, k, v, lambdas)
    want = reference(c, q, k, v, lambdas, dout)
    check(saved[0], want["out"], want["out_err"], "out")
    for got, name in zip(backward(c, q, k, v, dout, lambdas, saved), GRADS):
        check(got, want[name], want[name + "_err"], name)


@pytest.mark.parametrize("dtype", DTYPES, ids=DTYPE_IDS)
def test_large_scores(device, dtype):
    """Scores of some hundreds: the running maximum moves by more than exponentials can take."""
    c = case(1, 200, 200, 2, 1, 128)
    q, k, v, _, lambdas = inputs(c, dtype, device)
    q, k = (q * 6).contiguous(), (k * 6).contiguous()
    want = reference(c, q, k, v, lambdas)
    for got, name in zip(forward(c, q, k, v, lambdas), ("out", "second", "lse")):
        check(got, want[name], want[name + "_err"], name)


@pytest.mark.parametrize("dtype", DTYPES, ids=DTYPE_IDS)
@pytest.mark.parametrize("d", [64, 128, 36])
def test_what_stands_behind_the_mask_does_not_matter(device, dtype, d):
    """Padding behind a sequence: keys and values that the causal mask hides are NaN and infinite, and the rows before them do not see
    it, forward and in the gradient of q."""
    c = case(2, 150, 150, 4, 2, d)
    q, k, v, dout, lambdas = inputs(c, dtype, device)
    want = reference(c, q, k, v, lambdas, dout)
    for live in (1, 33, 64, 101, 149):
        k2, v2 = k.clone(), v.clone()
        k2[:, live:] = float("nan")
        v2[:, live:] = float("inf")
        v2[:, live::3] = float("nan")
        out, second, lse = forward(c, q, k2, v2, lambdas)
        dq = backward(c, q, k2, v2, dout, lambdas, (out, second, lse))[0]
        for got, name in ((out, "out"), (second, "second"), (dq, "dq")):
            check(got[:, :live], want[name][:, :live], want[name + "_err"][:, :live], name)
        check(lse[:, :, :live], want["lse"][:, :, :live], want["lse_err"][:, :, :live], "lse")


@pytest.mark.parametrize("dtype", DTYPES, ids=DTYPE_IDS)
def test_what_stands_behind_the_mask_of_few_queries(device, dtype):
    c = case(2, 20, 1500, 6, 2, 128, off=900)
    q, k, v, dout, lambdas = inputs(c, dtype, device)
    want = reference(c, q, k, v, lambdas)
    k[:, 920:] = float("nan")
    v[:, 920:] = float("inf")
    for got, name in zip(forward(c, q, k, v, lambdas), ("out", "second", "lse")):
        check(got, want[name], want[name + "_err"], name)
    k[:, 910:] = float("nan")
    v[:, 910:] = float("nan")
    out, second, lse = forward(c, q, k, v, lambdas)
    for got, name in ((out, "out"), (second, "second")):
        check(got[:, :10], want[name][:, :10], want[name + "_err"][:, :10], name)
        assert torch.isnan(got[:, 10:]).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=DTYPE_IDS)
def test_tensors_off_their_alignment(device, dtype):
    c = case(2, 50, 60, 4, 2, 64)
    q, k, v, dout, lambdas = inputs(c, dtype, device)
    want = reference(c, q, k, v, lambdas, dout)

    def moved(t):
        base = torch.zeros(t.numel() + 1, dtype=t.dtype, device=device)
        base[1:].copy_(t.reshape(-1))
        return base[1:].view(t.shape)

    q, k, v, dout = (moved(t) for t in (q, k, v, dout))
    out, second, lse = moved(q), moved(q), moved(torch.zeros(2, *q.shape[:3], device=device))
    ops.differential_attention_forward(out, second, lse, q, k, v, lambdas, None, options(c))
    grads = [moved(t) for t in (q, k, v, lambdas)]
    ops.differential_attention_backward(*grads, dout, out, second, lse, q, k, v, lambdas, None, options(c))
    for got, name in zip((out, second, lse, *grads), ("out", "second", "lse", *GRADS)):
        check(got, want[name], want[name + "_err"], name)


@pytest.mark.parametrize("dtype", DTYPES, ids=DTYPE_IDS)
@pytest.mark.parametrize("c", [case(2, 300, 300, 4, 2, 128), case(1, 600, 600, 2, 1, 64)], ids=["wide", "narrow"])
def test_twice_the_same_bits(device, c, dtype):
    q, k, v, dout, lambdas = inputs(c, dtype, device)
    saved = forward(c, q, k, v, lambdas)
    first = backward(c, q, k, v, dout, lambdas, saved)
    for _ in range(3):
        again = forward(c, q, k, v, lambdas)
        assert all(torch.equal(a, b) for a, b in zip(saved, again))
        assert all(torch.equal(a, b) for a, b in zip(first, backward(c, q, k, v, dout, lambdas, again)))


def test_gradient_against_differences(device):
    """Along a direction in q, k, v and the weights: central differences of the formula in 64 bits (their own error: h^2 times a third
    derivative below 1e4)."""
    c = case(1, 20, 24, 4, 2, 32)
    q, k, v, dout, lambdas = inputs(c, torch.float32, device)
    grads = backward(c, q, k, v, dout, lambdas, forward(c, q, k, v, lambdas))
    directions = [randn(t.shape, torch.float32, 60 + i).double().to(device) for i, t in enumerate((q, k, v, lambdas))]

    def loss(step):
        moved = [t.double() + step * d for t, d in zip((q, k, v, lambdas), directions)]
        return (reference(c, *moved, dtype=torch.float32)["out"] * dout.double()).sum().item()

    h = 1e-4
    slope = (loss(h) - loss(-h)) / (2 * h)
    terms = [(g.double() * d) for g, d in zip(grads, directions)]
    bounds = reference(c, q, k, v, lambdas, dout)
    off = sum((bounds[n + "_err"] * d.abs()).sum().item() for n, d in zip(GRADS, directions))
    assert abs(slope - sum(t.sum().item() for t in terms)) <= 1e-4 + off + 2.0 ** -24 * sum(t.abs().sum().item() for t in terms)


def test_captured_calls(device):
    c = case(2, 200, 200, 4, 2, 128)
    q, k, v, dout, lambdas = inputs(c, torch.bfloat16, device)
    out, second, lse = torch.empty_like(q), torch.empty_like(q), torch.empty((2, *q.shape[:3]), device=device)
    grads = [torch.empty_like(t) for t in (q, k, v, lambdas)]

    def both():
        ops.differential_attention_forward(out, second, lse, q, k, v, lambdas, None, options(c))
        ops.differential_attention_backward(*grads, dout, out, second, lse, q, k, v, lambdas, None, options(c))

    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        both()
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream, capture_error_mode="thread_local"):
        both()
    for seed in range(4):
        q.copy_(randn(q.shape, q.dtype, 70 + seed))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (out, second, lse, *grads)]
        for t in (out, second, lse, *grads):
            t.fill_(5.0)
        both()
        torch.cuda.synchronize()
        for a, b in zip(got, (out, second, lse, *grads)):
            assert torch.equal(a, b)


def test_on_another_stream(device):
    c = case(2, 130, 130, 4, 2, 64)
    q, k, v, dout, lambdas = inputs(c, torch.float16, device)
    saved = forward(c, q, k, v, lambdas)
    grads = backward(c, q, k, v, dout, lambdas, saved)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    saved2 = forward(c, q, k, v, lambdas)
    torch.cuda.synchronize()
    grads2 = backward(c, q, k, v, dout, lambdas, saved2, stream=side)
    side.synchronize()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip((*saved, *grads), (*saved2, *grads2)))


@pytest.mark.parametrize("dtype", DTYPES, ids=DTYPE_IDS)
def test_two_streams_at_once(device, dtype):
    """Calls on two streams have working memory of their own: the same bits as one after the other."""
    cases = [case(1, 1, 3000, 8, 2, 128), case(2, 300, 300, 4, 2, 128)]
    given = [inputs(c, dtype, device, seed=3 + i) for i, c in enumerate(cases)]

    def both(c, t, stream):
        saved = forward(c, *t[:3], t[4], stream)
        return [*saved, *backward(c, *t, saved, stream=stream)]

    want = [both(c, t, None) for c, t in zip(cases, given)]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(4):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(both(cases[i], given[i], stream))
    torch.cuda.synchronize()
    for expected, runs in zip(want, got):
        for run in runs:
            assert all(torch.equal(a, b) for a, b in zip(expected, run))


def test_launches(device):
    c = case(2, 300, 300, 4, 2, 128)
    q, k, v, _, lambdas = inputs(c, torch.bfloat16, device)
    out, second, lse = forward(c, q, k, v, lambdas)
    assert launches(lambda: ops.differential_attention_forward(out, second, lse, q, k, v, lambdas, None, options(c))) == 1


# ------------------------------------------------------------------------------------------------ the weights
@pytest.mark.parametrize("dtype", DTYPES, ids=DTYPE_IDS)
@pytest.mark.parametrize("sets,heads,width", [(1, 1, 1), (8, 8, 64), (1, 12, 32), (1, 100, 63), (3, 3, 130), (64, 64, 16)])
def test_weights(device, sets, heads, width, dtype):
    """Products of fp32 numbers: a chain of width/64 + 7 roundings, then the exponential's two steps; the gradients are rounded to
    storage once."""
    vectors = [randn((sets, width), dtype, 80 + i, 0.3).to(device) for i in range(4)]
    dlam = randn((heads,), torch.float32, 90).to(device)
    lambdas, grads = torch.full((heads,), 9.0, device=device), [torch.full_like(v, 9.0) for v in vectors]
    ops.differential_lambda_forward(lambdas, *vectors, 0.35)
    ops.differential_lambda_backward(*grads, dlam, *vectors)
    q1, k1, q2, k2 = (v.double() for v in vectors)
    e1, e2 = torch.exp((q1 * k1).sum(1)), torch.exp((q2 * k2).sum(1))
    f = 2.0 ** -24 * (width / 64 + 16)
    rel = f * (1 + torch.maximum((q1 * k1).abs().sum(1), (q2 * k2).abs().sum(1)))
    want = (e1 - e2 + 0.35).expand(heads)
    check(lambdas, want, (rel * (e1 + e2) + 4 * f).expand(heads), "lambda")
    of_set = dlam.double() if sets > 1 else dlam.double().sum().view(1)
    size = dlam.double().abs() if sets > 1 else dlam.double().abs().sum().view(1)
    for got, e, other, sign in zip(grads, (e1, e1, e2, e2), (k1, q1, k2, q2), (1, 1, -1, -1)):
        exact = (sign * of_set * e)[:, None] * other
        check(got, exact, ((size * e) * (rel + 2.0 ** -24 * (heads / 64 + 10)))[:, None] * other.abs(), "gradient")


# ------------------------------------------------------------------------------------------------ a branch
@pytest.mark.parametrize("dtype", DTYPES, ids=DTYPE_IDS)
def test_a_branch_around_the_stream(device, dtype):
    """Layer norm, projections, differential attention with learned weights, per-head norm, projection, dropout onto the stream, forward
    and backward by the operators, against autograd of the same branch in 64 bits.

    Bound: a chain of eight operators, each of which rounds its results to storage and its products once, leaves at most 2 x 8 half
    steps of the largest magnitudes that meet in a result, times the condition of the attention's differences and norms (under 8 here)."""
    b, t, hq, hkv, d, hidden = 2, 50, 4, 2, 32, 96
    eps, p = 1e-5, 0.2
    width = hq * d
    names = dict(ln_w=(hidden,), ln_b=(hidden,), wq=(width, hidden), wk=(hkv * d, hidden), wv=(hkv * d, hidden), wo=(hidden, width), hn=(d,),
                 l0=(1, d // 2), l1=(1, d // 2), l2=(1, d // 2), l3=(1, d // 2))
    weights = {}
    for i, (name, shape) in enumerate(names.items()):
        base = randn(shape, torch.float32, 100 + i, 0.1)
        weights[name] = (base + (1.0 if name in ("ln_w", "hn") else 0.0)).to(dtype).to(device)
    x, dout = randn((b * t, hidden), dtype, 120).to(device), randn((b * t, hidden), dtype, 121).to(device)
    drop = ops.DropoutOptions(p, 5, 6)
    att = ops.FlashAttentionOptions(num_query_heads=hq, num_kv_heads=hkv, head_dim=d)
    w = weights

    def empty(*shape):
        return torch.empty(shape, dtype=dtype, device=device)

    # forward
    normed, q, k, v = empty(b * t, hidden), empty(b, t, hq, d), empty(b, t, hkv, d), empty(b, t, hkv, d)
    ops.layernorm_forward(normed, x, w["ln_w"], w["ln_b"], eps)
    for out, weight in ((q, "wq"), (k, "wk"), (v, "wv")):
        ops.linear_forward(out.view(b * t, -1), normed, w[weight])
    lambdas = torch.empty(hq, device=device)
    ops.differential_lambda_forward(lambdas, w["l0"], w["l1"], w["l2"], w["l3"], 0.4)
    att_out, second, lse = empty(b, t, hq, d), empty(b, t, hq, d), torch.empty(2, b, t, hq, device=device)
    ops.differential_attention_forward(att_out, second, lse, q, k, v, lambdas, None, att)
    head_normed, projected, out = empty(b * t * hq, d), empty(b * t, hidden), empty(b * t, hidden)
    ops.rmsnorm_forward(head_normed, att_out.view(-1, d), w["hn"], eps)
    ops.linear_forward(projected, head_normed.view(b * t, width), w["wo"])
    ops.dropout_forward(out, projected, x, None, drop)

    # backward
    grads = {name: torch.empty_like(value) for name, value in weights.items()}
    d_projected, d_heads, d_att = empty(b * t, hidden), empty(b * t, width), empty(b, t, hq, d)
    ops.dropout_backward(d_projected, dout, None, drop)
    ops.linear_backward(d_heads, grads["wo"], None, d_projected, head_normed.view(b * t, width), w["wo"])
    ops.rmsnorm_backward(d_att.view(-1, d), grads["hn"], d_heads.view(-1, d), att_out.view(-1, d), w["hn"], eps)
    dq, dk, dv, dlam = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v), torch.empty_like(lambdas)
    ops.differential_attention_backward(dq, dk, dv, dlam, d_att, att_out, second, lse, q, k, v, lambdas, None, att)
    ops.differential_lambda_backward(grads["l0"], grads["l1"], grads["l2"], grads["l3"], dlam, w["l0"], w["l1"], w["l2"], w["l3"])
    d_normed = empty(b * t, hidden)
    for i, (grad, weight) in enumerate(((dq, "wq"), (dk, "wk"), (dv, "wv"))):
        ops.linear_backward(d_normed, grads[weight], None, grad.view(b * t, -1), normed, w[weight],
                            options=ops.LinearBackwardOptions(accumulate_input=i > 0))
    dx = empty(b * t, hidden)
    ops.layernorm_backward(dx, grads["ln_w"], grads["ln_b"], d_normed, x, w["ln_w"], eps, None, dout)

    # the same in 64 bits
    leaf = {name: value.double().cpu().requires_grad_() for name, value in weights.items()}
    x64 = x.double().cpu().requires_grad_()
    mask = torch.zeros(b * t, hidden, dtype=dtype, device=device)
    ops.dropout_forward(mask, torch.ones_like(mask), None, None, drop)
    keep = (mask != 0).cpu()
    n = torch.nn.functional.layer_norm(x64, (hidden,), leaf["ln_w"], leaf["ln_b"], eps)
    q64, k64, v64 = ((n @ leaf[name].T).view(b, t, -1, d).transpose(1, 2) for name in ("wq", "wk", "wv"))
    k64, v64 = k64.repeat_interleave(hq // hkv, 1), v64.repeat_interleave(hq // hkv, 1)
    lam = torch.exp((leaf["l0"] * leaf["l1"]).sum()) - torch.exp((leaf["l2"] * leaf["l3"]).sum()) + 0.4
    bias = torch.full((t, t), -math.inf, dtype=torch.float64).triu(1)
    m1, m2 = (torch.softmax(q64[..., s] @ k64[..., s].transpose(2, 3) / math.sqrt(d // 2) + bias, -1)
              for s in (slice(0, d // 2), slice(d // 2, d)))
    a = ((m1 - lam * m2) @ v64).transpose(1, 2)
    a = a * torch.rsqrt((a ** 2).mean(-1, keepdim=True) + eps) * leaf["hn"]
    threshold = int(p * 65536 + 0.5)
    y = x64 + torch.where(keep, a.reshape(b * t, width) @ leaf["wo"].T * (65536 / (65536 - threshold)), 0.0)
    wanted = torch.autograd.grad(y, [x64, *leaf.values()], dout.double().cpu())
    half = torch.finfo(dtype).eps / 2
    for name, got, want in zip(["y", "x", *leaf], [out, dx, *grads.values()], [y.detach(), *wanted]):
        off, size = (got.double().cpu() - want).abs().max().item(), want.abs().max().item()
        print(f"[parity] branch {name}: {off / size:.2e} of the largest")
        assert off <= 16 * 8 * half * max(size, 1e-3), name
