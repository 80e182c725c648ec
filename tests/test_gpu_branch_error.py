"""A branch around the residual stream (layer norm, projections, differential attention with learned weights, per-head norm, projection, dropout
onto the stream) in 16-bit storage: how far its results are from the same branch in 64 bits, in the 2-norm.

The yardstick is the branch in 64 bits with the results of every operator rounded to storage once. The operators round no result more
often; attention rounds its probabilities and score gradients and takes its row sums from rounded outputs beside that, roundings of the
same size: at most three for one in its part of the chain, and sqrt(3) times the error; 2.5 leaves room for chance. A missing factor
or term is some ten times that. The weights' vectors have one common number each, the gradient of lambda, a sum over all rows whose terms are
off by what three operators rounded: they are held to four half steps of the terms' magnitudes."""
import math

import pytest
import torch

from cgpt_amd import ops
from tests.util import randn

pytestmark = pytest.mark.gpu

B, T, HQ, HKV, D, HIDDEN, EPS, DROP = 2, 90, 4, 2, 32, 96, 1e-5, 0.2
WIDTH = HQ * D
SHAPES = dict(ln_w=(HIDDEN,), ln_b=(HIDDEN,), wq=(WIDTH, HIDDEN), wk=(HKV * D, HIDDEN), wv=(HKV * D, HIDDEN), wo=(HIDDEN, WIDTH), hn=(D,),
              l0=(1, D // 2), l1=(1, D // 2), l2=(1, D // 2), l3=(1, D // 2))


def run(w, x, dout, drop):
    """The branch by the operators: out, dx and the gradients by name."""
    def empty(*shape):
        return torch.empty(shape, dtype=x.dtype, device=x.device)

    n = B * T
    att = ops.FlashAttentionOptions(num_query_heads=HQ, num_kv_heads=HKV, head_dim=D)
    normed, q, k, v = empty(n, HIDDEN), empty(B, T, HQ, D), empty(B, T, HKV, D), empty(B, T, HKV, D)
    ops.layernorm_forward(normed, x, w["ln_w"], w["ln_b"], EPS)
    for to, weight in ((q, "wq"), (k, "wk"), (v, "wv")):
        ops.linear_forward(to.view(n, -1), normed, w[weight])
    lambdas = torch.empty(HQ, device=x.device)
    ops.differential_lambda_forward(lambdas, w["l0"], w["l1"], w["l2"], w["l3"], 0.4)
    mixed, second, lse = empty(B, T, HQ, D), empty(B, T, HQ, D), torch.empty(2, B, T, HQ, device=x.device)
    ops.differential_attention_forward(mixed, second, lse, q, k, v, lambdas, None, att)
    heads, projected, out = empty(n * HQ, D), empty(n, HIDDEN), empty(n, HIDDEN)
    ops.rmsnorm_forward(heads, mixed.view(-1, D), w["hn"], EPS)
    ops.linear_forward(projected, heads.view(n, WIDTH), w["wo"])
    ops.dropout_forward(out, projected, x, None, drop)

    g = {name: torch.empty_like(value) for name, value in w.items()}
    d_projected, d_heads, d_mixed = empty(n, HIDDEN), empty(n, WIDTH), empty(B, T, HQ, D)
    ops.dropout_backward(d_projected, dout, None, drop)
    ops.linear_backward(d_heads, g["wo"], None, d_projected, heads.view(n, WIDTH), w["wo"])
    ops.rmsnorm_backward(d_mixed.view(-1, D), g["hn"], d_heads.view(-1, D), mixed.view(-1, D), w["hn"], EPS)
    dq, dk, dv, dlam = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v), torch.empty_like(lambdas)
    ops.differential_attention_backward(dq, dk, dv, dlam, d_mixed, mixed, second, lse, q, k, v, lambdas, None, att)
    ops.differential_lambda_backward(g["l0"], g["l1"], g["l2"], g["l3"], dlam, w["l0"], w["l1"], w["l2"], w["l3"])
    d_normed, dx = empty(n, HIDDEN), empty(n, HIDDEN)
    for i, (grad, weight) in enumerate(((dq, "wq"), (dk, "wk"), (dv, "wv"))):
        ops.linear_backward(d_normed, g[weight], None, grad.view(n, -1), normed, w[weight], options=ops.LinearBackwardOptions(accumulate_input=i > 0))
    ops.layernorm_backward(dx, g["ln_w"], g["ln_b"], d_normed, x, w["ln_w"], EPS, None, dout)
    return {"out": out, "x": dx, **g}


def layernorm(x, w, b):
    return torch.nn.functional.layer_norm(x, (HIDDEN,), w, b, EPS)


def rmsnorm(x, w):
    return x * torch.rsqrt((x ** 2).mean(-1, keepdim=True) + EPS) * w


def weight_of(l0, l1, l2, l3):
    return torch.exp((l0 * l1).sum()) - torch.exp((l2 * l3).sum()) + 0.4


def maps(q, k):
    q, k = q.transpose(1, 2), k.transpose(1, 2).repeat_interleave(HQ // HKV, 1)
    hidden = torch.full((T, T), -math.inf, dtype=torch.float64).triu(1)
    return [torch.softmax(q[..., s] @ k[..., s].transpose(2, 3) / math.sqrt(D // 2) + hidden, -1) for s in (slice(0, D // 2), slice(D // 2, D))]


def attention(q, k, v, lam):
    p1, p2 = maps(q, k)
    return ((p1 - lam * p2) @ v.transpose(1, 2).repeat_interleave(HQ // HKV, 1)).transpose(1, 2)


def pull(f, inputs, gradient):
    """The gradients of f's inputs."""
    leaves = [t.detach().requires_grad_() for t in inputs]
    return torch.autograd.grad(f(*leaves), leaves, gradient.detach())


def reference(w, x, dout, factor, rounded):
    """The branch in 64 bits, operator by operator, with each result through `rounded`; and the magnitude of dlambda's terms."""
    n = B * T
    normed = rounded(layernorm(x, w["ln_w"], w["ln_b"]))
    q, k, v = (rounded(normed @ w[name].T).view(B, T, -1, D) for name in ("wq", "wk", "wv"))
    vectors = [w[f"l{i}"] for i in range(4)]
    lam = weight_of(*vectors)
    mixed = rounded(attention(q, k, v, lam))
    heads = rounded(rmsnorm(mixed, w["hn"]))
    projected = rounded(heads.reshape(n, WIDTH) @ w["wo"].T)
    result = {"out": rounded(x + factor * projected)}

    d_projected = rounded(dout * factor)
    result["wo"] = rounded(d_projected.T @ heads.reshape(n, WIDTH))
    d_heads = rounded(d_projected @ w["wo"]).view(B, T, HQ, D)
    d_mixed, d_hn = pull(rmsnorm, (mixed, w["hn"]), d_heads)
    d_mixed, result["hn"] = rounded(d_mixed), rounded(d_hn)
    dq, dk, dv, dlam = pull(attention, (q, k, v, lam), d_mixed)
    for name, grad in zip(("l0", "l1", "l2", "l3"), pull(weight_of, vectors, dlam)):
        result[name] = rounded(grad)
    d_normed = 0.0
    for name, grad in (("wq", dq), ("wk", dk), ("wv", dv)):
        grad = rounded(grad).reshape(n, -1)
        result[name] = rounded(grad.T @ normed)
        d_normed = rounded(d_normed + grad @ w[name])
    dx, d_w, d_b = pull(layernorm, (x, w["ln_w"], w["ln_b"]), d_normed)
    result["x"], result["ln_w"], result["ln_b"] = rounded(dx + dout), rounded(d_w), rounded(d_b)
    second = (maps(q, k)[1] @ v.transpose(1, 2).repeat_interleave(HQ // HKV, 1)).transpose(1, 2)
    return result, (d_mixed * second).abs().sum()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
@pytest.mark.parametrize("seed", [1, 2])
def test_a_branch_is_off_by_what_storage_rounds(device, dtype, seed):
    weights = {name: (randn(shape, torch.float32, 100 * seed + i, 0.1) + (1.0 if name in ("ln_w", "hn") else 0.0)).to(dtype)
               for i, (name, shape) in enumerate(SHAPES.items())}
    x, dout = randn((B * T, HIDDEN), dtype, 100 * seed + 50), randn((B * T, HIDDEN), dtype, 100 * seed + 51)
    drop = ops.DropoutOptions(DROP, seed, 6)
    got = run({name: value.to(device) for name, value in weights.items()}, x.to(device), dout.to(device), drop)
    mask = torch.zeros_like(x, device=device)
    ops.dropout_forward(mask, torch.ones_like(mask), None, None, drop)
    threshold = int(DROP * 65536 + 0.5)
    factor = (mask.cpu() != 0).double() * (65536 / (65536 - threshold))
    given = ({name: value.double() for name, value in weights.items()}, x.double(), dout.double(), factor)
    exact, terms = reference(*given, lambda t: t)
    yardstick, _ = reference(*given, lambda t: t.detach().to(dtype).double())
    half = torch.finfo(dtype).eps / 2
    for name, want in exact.items():
        want = want.detach()
        off, by = (got[name].double().cpu() - want).norm().item(), (yardstick[name] - want).norm().item()
        print(f"[parity] branch {name}: off by {off / want.norm().item():.2e}, rounded results by {by / want.norm().item():.2e}")
        if name in ("l0", "l1", "l2", "l3"):
            first = {"l0": "l1", "l1": "l0", "l2": "l3", "l3": "l2"}[name]
            pair = given[0][name], given[0][first]
            most = 4 * half * terms.item() * math.exp((pair[0] * pair[1]).sum().item()) * pair[1].norm().item() + half * want.norm().item()
        else:
            most = 2.5 * by
        assert off <= most, (name, off, most)
