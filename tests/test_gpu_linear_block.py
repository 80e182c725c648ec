"""A block whose mixer is linear attention, of the framework's operators as a model would run it: sandwich norm, projections, linear attention, output
projection, sandwich norm. Its gradients against automatic ones in 64 bits, a prompt continued token by token, and a step recorded into a graph.

fp32 tolerance, of a tensor's norm: seven operators one after the other, each off by at most 2^-24 (longest sum + 300) of its terms' magnitudes, which
are some 4 times a result's where terms cancel at random over a head's 32 products and the tokens' sums."""
import pytest
import torch

from cgpt_amd import ops
from tests.util import randn

pytestmark = pytest.mark.gpu
B, T, H, HQ, HKV, D, EPS, SCALE = 3, 90, 96, 4, 2, 32, 1e-5, 0.8
TOL = 2.0 ** -24 * (B * T + 300) * 7 * 4


def parameters(dtype, device):
    shapes = dict(u1=(H,), w1=(H,), g1=(B, H), wq=(HQ * D, H), wk=(HKV * D, H), wv=(HKV * D, H), wo=(H, HQ * D), u2=(H,), w2=(H,), g2=(B, H))
    p = {name: randn(s, dtype, 10 + i, 1.0 if len(s) < 2 or name[0] == "g" else s[1] ** -0.5).to(device) for i, (name, s) in enumerate(shapes.items())}
    p["log_decay"] = torch.tensor([-0.05, -0.3], device=device)
    return p


def options():
    return ops.FlashAttentionOptions(num_query_heads=HQ, num_kv_heads=HKV, head_dim=D)


def empty(like, *shape):
    return torch.full(shape, float("nan"), dtype=like.dtype, device=like.device)


def forward(p, x, f, before, tokens=T, after=None):
    """Streams and what the backward pass needs; x and f [B tokens, H]."""
    r, n = {}, B * tokens
    r["s1"], r["y1"] = empty(x, n, H), empty(x, n, H)
    ops.sandwich_norm_forward(r["s1"], r["y1"], x, f, p["u1"], p["g1"], p["w1"], SCALE, EPS)
    for name, heads in (("q", HQ), ("k", HKV), ("v", HKV)):
        r[name] = empty(x, n, heads * D)
        ops.linear_forward(r[name], r["y1"], p["w" + name])
    shaped = [r[name].view(B, tokens, heads, D) for name, heads in (("q", HQ), ("k", HKV), ("v", HKV))]
    r["o"] = empty(x, n, HQ * D)
    r["after"] = empty(p["log_decay"], B, HKV, D, D) if after is None else after
    if tokens == 1:
        ops.linear_attention_step(r["o"].view(B, 1, HQ, D), r["after"], before, *shaped, p["log_decay"], None, options())
    else:
        ops.linear_attention_forward(r["o"].view(B, tokens, HQ, D), r["after"], *shaped, p["log_decay"], before, None, options())
    r["f2"], r["s2"], r["y2"] = empty(x, n, H), empty(x, n, H), empty(x, n, H)
    ops.linear_forward(r["f2"], r["o"], p["wo"])
    ops.sandwich_norm_forward(r["s2"], r["y2"], r["s1"], r["f2"], p["u2"], p["g2"], p["w2"], SCALE, EPS)
    return r


def backward(p, x, f, before, r, d_stream, dy, d_after):
    n = B * T
    g = {name: torch.full_like(p[name], float("nan")) for name in p if name != "log_decay"}
    ds1, df2, do, dy1 = empty(x, n, H), empty(x, n, H), empty(x, n, HQ * D), empty(x, n, H)
    ops.sandwich_norm_backward(ds1, df2, g["u2"], g["g2"], g["w2"], d_stream, dy, r["s2"], r["f2"], p["u2"], p["g2"], p["w2"], SCALE, EPS)
    ops.linear_backward(do, g["wo"], None, df2, r["o"], p["wo"])
    d = {name: torch.full_like(r[name], float("nan")) for name in "qkv"}
    shape = dict(q=(B, T, HQ, D), k=(B, T, HKV, D), v=(B, T, HKV, D))
    g["before"] = torch.full_like(before, float("nan"))
    ops.linear_attention_backward(*(d[name].view(shape[name]) for name in "qkv"), g["before"], do.view(shape["q"]), d_after,
                                  *(r[name].view(shape[name]) for name in "qkv"), p["log_decay"], before, None, options())
    for name in "qkv":
        ops.linear_backward(dy1, g["w" + name], None, d[name], r["y1"], p["w" + name], options=ops.LinearBackwardOptions(accumulate_input=name != "q"))
    g["x"], g["f"] = empty(x, n, H), empty(x, n, H)
    ops.sandwich_norm_backward(g["x"], g["f"], g["u1"], g["g1"], g["w1"], ds1, dy1, r["s1"], f, p["u1"], p["g1"], p["w1"], SCALE, EPS)
    return g


def plain(p, x, f, before):
    def norm(t, w):
        return t / torch.sqrt((t * t).mean(1, keepdim=True) + EPS) * w

    s1 = SCALE * x + p["g1"].repeat_interleave(T, 0) * norm(f, p["u1"])
    y1 = norm(s1, p["w1"])
    q, k, v = ((y1 @ p["w" + name].t()).view(B, T, -1, D) for name in "qkv")
    decay, state, outs = torch.exp(p["log_decay"]).view(1, -1, 1, 1), before, []
    for t in range(T):
        state = decay * state + k[:, t, :, :, None] * v[:, t, :, None, :]
        outs.append((q[:, t, :, None] @ state.repeat_interleave(HQ // HKV, 1)).squeeze(2) * D ** -0.5)
    f2 = torch.stack(outs, 1).reshape(B * T, HQ * D) @ p["wo"].t()
    s2 = SCALE * s1 + p["g2"].repeat_interleave(T, 0) * norm(f2, p["u2"])
    return s2, norm(s2, p["w2"]), state


def given(dtype, device):
    x, f, d_stream, dy = (randn((B * T, H), dtype, 40 + i).to(device) for i in range(4))
    before, d_after = (randn((B, HKV, D, D), torch.float32, 50 + i).to(device) for i in range(2))
    return x, f, d_stream, dy, before, d_after


def near(got, want, name):
    off = ((got.double().cpu() - want).norm() / want.norm()).item()
    assert off <= TOL, f"{name}: {off:.3g} of its norm, allowed {TOL:.3g}"


def test_block_and_its_gradients(device):
    p = parameters(torch.float32, device)
    x, f, d_stream, dy, before, d_after = given(torch.float32, device)
    r = forward(p, x, f, before)
    g = backward(p, x, f, before, r, d_stream, dy, d_after)
    leaves = {name: t.double().cpu().requires_grad_() for name, t in (*p.items(), ("x", x), ("f", f), ("before", before))}
    s2, y2, after = plain(leaves, leaves["x"], leaves["f"], leaves["before"])
    total = sum((a * b.double().cpu()).sum() for a, b in ((s2, d_stream), (y2, dy), (after, d_after)))
    total.backward()
    for name, got, want in (("s2", r["s2"], s2), ("y2", r["y2"], y2), ("after", r["after"], after)):
        near(got, want.detach(), name)
    for name, got in g.items():
        near(got, leaves[name].grad, name)


def test_prompt_then_single_tokens(device):
    """The rows of a prompt of 70 and 20 tokens one by one are those of 90 tokens at once."""
    p = parameters(torch.float32, device)
    x, f, _, _, before, _ = given(torch.float32, device)
    whole = forward(p, x, f, before)

    def rows(t, first, last):
        return t.view(B, T, -1)[:, first:last].reshape(B * (last - first), -1).contiguous()

    r = forward(p, rows(x, 0, 70), rows(f, 0, 70), before, 70)
    for name in ("s2", "y2"):
        near(r[name], rows(whole[name], 0, 70).double().cpu(), name)
    state = r["after"]
    for t in range(70, T):
        r = forward(p, rows(x, t, t + 1), rows(f, t, t + 1), state, 1, state)
        for name in ("s2", "y2"):
            near(r[name], rows(whole[name], t, t + 1).double().cpu(), name)
    near(state, whole["after"].double().cpu(), "after")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
def test_recorded_block(device, dtype):
    """Forward and backward recorded: every replay has the eager pass's bits, with other eager work between them."""
    p = parameters(dtype, device)
    x, f, d_stream, dy, before, d_after = given(dtype, device)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        for _ in range(2):
            r = forward(p, x, f, before)
            eager = {**r, **{"g_" + k: v for k, v in backward(p, x, f, before, r, d_stream, dy, d_after).items()}}
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream, capture_error_mode="thread_local"):
        r = forward(p, x, f, before)
        held = {**r, **{"g_" + k: v for k, v in backward(p, x, f, before, r, d_stream, dy, d_after).items()}}
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        for name, t in eager.items():
            assert torch.isfinite(t).all() and torch.equal(held[name], t), name
        forward(p, f, x, before)  # other work between replays
        torch.cuda.synchronize()
