"""Arguments that linear attention and the sandwich norm refuse, through the C entries and the Python mirror, before anything is launched (so these run
without a GPU); and the formulas that the GPU tests compare with, against a recurrence and its automatic gradients."""
import ctypes

import pytest
import torch

from cgpt_amd import capi, ops
from tests.linear_oracle import linear_backward, linear_forward, linear_step, sandwich_backward, sandwich_forward

N = ctypes.c_void_p(0)
P = ctypes.c_void_p(0x1000)  # never dereferenced: validation fails first
Q = ctypes.c_void_p(0x2000)
NAN, INF = float("nan"), float("inf")
F, B, H = capi.F32, capi.BF16, capi.F16


def sizes(batch=1, tokens=8, hq=2, hkv=1, d=32, scale=0.0, dtype=B):
    return batch, tokens, hq, hkv, d, scale, dtype, N


def forward(*null, same=False, **shape):
    p = [N if i in null else P for i in range(7)]  # output, final, query, key, value, decay, initial
    if not same:
        p[1] = N if 1 in null else Q
    return (*p, *sizes(**shape))


def backward(*null, d_before=Q, **shape):
    p = [N if i in null else P for i in range(11)]
    p[3] = d_before
    s = sizes(**shape)
    return (*p, *s[:6], 0, *s[6:])


def step(*null, **shape):
    s = sizes(**shape)
    return (*(N if i in null else P for i in range(7)), s[0], *s[2:])


def norm(*null, rows=4, hidden=8, gates=2, scale=1.0, eps=1e-5, dtype=B):
    return (*(N if i in null else P for i in range(7)), rows, hidden, gates, scale, eps, dtype, N)


def norm_backward(*null, rows=4, hidden=8, gates=2, scale=1.0, eps=1e-5, dtype=B):
    return (*(N if i in null else P for i in range(12)), rows, hidden, gates, scale, eps, dtype, N)


BAD_SIZES = [dict(batch=0), dict(hq=0), dict(hkv=0), dict(hq=3, hkv=2), dict(d=0), dict(d=129), dict(scale=NAN), dict(scale=INF), dict(dtype=7), dict(dtype=-1),
             dict(batch=2**16), dict(hq=2**16, hkv=2**16), dict(batch=2**14, hq=2**7)]


@pytest.mark.parametrize("name,args", [
    *[("cgptx_linear_attention_forward", forward(i)) for i in (0, 2, 3, 4, 5)],
    *[("cgptx_linear_attention_forward", forward(**s)) for s in (*BAD_SIZES, dict(tokens=0), dict(tokens=2**31))],
    ("cgptx_linear_attention_forward", forward(same=True)),                       # the final state in the initial one's place
    *[("cgptx_linear_attention_backward", backward(i)) for i in (0, 1, 2, 4, 6, 7, 8, 9)],
    *[("cgptx_linear_attention_backward", backward(**s)) for s in (*BAD_SIZES, dict(tokens=0), dict(tokens=2**31))],
    ("cgptx_linear_attention_backward", backward(d_before=P)),
    *[("cgptx_linear_attention_step", step(i)) for i in range(7)],
    *[("cgptx_linear_attention_step", step(**s)) for s in BAD_SIZES],
    *[("cgptx_sandwich_norm_forward", norm(i)) for i in range(7)],               # gate without gate rows among them
    ("cgptx_sandwich_norm_forward", norm(gates=0)),
    ("cgptx_sandwich_norm_forward", norm(gates=3)),
    *[("cgptx_sandwich_norm_forward", norm(**s)) for s in (dict(rows=0), dict(hidden=0), dict(scale=NAN), dict(scale=-INF), dict(eps=0.0), dict(eps=-1.0),
                                                         dict(eps=NAN), dict(eps=INF), dict(dtype=9), dict(rows=2**31), dict(hidden=2**25 + 1))],
    *[("cgptx_sandwich_norm_backward", norm_backward(i)) for i in (0, 1, 2, 4, 6, 7, 8, 9, 10, 11)],
    ("cgptx_sandwich_norm_backward", norm_backward(10, gates=0)),                # a gate's gradient without a gate
    ("cgptx_sandwich_norm_backward", norm_backward(gates=3)),
    *[("cgptx_sandwich_norm_backward", norm_backward(**s)) for s in (dict(rows=0), dict(hidden=0), dict(scale=NAN), dict(eps=0.0), dict(dtype=9), dict(hidden=2**25 + 1))],
])
def test_invalid_arguments(name, args):
    with pytest.raises((ValueError, OverflowError)):
        capi.call(name, *args)


def test_python_mirror_refuses_host_tensors():
    q, k, s = torch.zeros(1, 4, 2, 8), torch.zeros(1, 4, 1, 8), torch.zeros(1, 1, 8, 8)
    o, decay, x, w = ops.FlashAttentionOptions(num_query_heads=2, num_kv_heads=1, head_dim=8), torch.zeros(1), torch.zeros(4, 8), torch.zeros(8)
    for call in (lambda: ops.linear_attention_forward(q, s, q, k, k, decay, None, None, o),
                 lambda: ops.linear_attention_backward(q, k, k, None, q, None, q, k, k, decay, None, None, o),
                 lambda: ops.linear_attention_step(q[:, :1], s, s, q[:, :1], k[:, :1], k[:, :1], decay, None, o),
                 lambda: ops.sandwich_norm_forward(x, x, x, x, w, None, w, 1.0, 1e-5),
                 lambda: ops.sandwich_norm_backward(x, x, w, None, w, None, x, x, x, w, None, w, 1.0, 1e-5)):
        with pytest.raises(ValueError):
            call()


def recurrence(q, k, v, log_decay, before, scale):
    group = q.shape[2] // k.shape[2]
    g, state, outs = torch.exp(log_decay).view(1, -1, 1, 1), before, []
    for t in range(q.shape[1]):
        state = g * state + k[:, t, :, :, None] * v[:, t, :, None, :]
        outs.append(scale * torch.matmul(q[:, t, :, None], state.repeat_interleave(group, 1)).squeeze(2))
    return torch.stack(outs, 1), state


def test_linear_oracle():
    torch.manual_seed(0)
    b, t, hq, hkv, d = 2, 9, 6, 2, 5
    q, k, v = (torch.randn(b, t, h, d, dtype=torch.float64, requires_grad=True) for h in (hq, hkv, hkv))
    before = torch.randn(b, hkv, d, d, dtype=torch.float64, requires_grad=True)
    log_decay = torch.tensor([-0.3, -0.01], dtype=torch.float64)
    out, after = recurrence(q, k, v, log_decay, before, 0.4)
    dout, d_after = torch.randn_like(out), torch.randn_like(after)
    grads = torch.autograd.grad((out * dout).sum() + (after * d_after).sum(), (q, k, v, before))
    data = [x.detach().float() for x in (q, k, v)]  # the formulas take storage types; their values are held in 64 bits
    with torch.no_grad():
        out, after = recurrence(*(x.double() for x in data), log_decay, before, 0.4)
        got = linear_forward(*data, log_decay, before.detach(), 0.4)
        back = linear_backward(*data, log_decay, before.detach(), dout, d_after, 0.4)
        one = linear_step(*(x[:, :1] for x in data), log_decay, before.detach(), 0.4)
        first, state = recurrence(*(x[:, :1].double() for x in data), log_decay, before, 0.4)
    for a, b_ in ((got["out"].value, out), (got["after"].value, after), (one["out"].value, first), (one["after"].value, state)):
        assert torch.allclose(a, b_, rtol=1e-12, atol=1e-12)
    for name, g in zip(("dq", "dk", "dv", "d_before"), grads):
        assert torch.allclose(back[name].value, g, rtol=1e-5, atol=1e-5), name  # inputs rounded to fp32 in one of the two
    # Bounds are of the magnitude of a few steps of the type.
    assert (got["out"].error / got["out"].value.abs().mean()).max() < 1e-3


def test_sandwich_oracle():
    torch.manual_seed(0)
    rows, hidden, eps, scale = 6, 11, 1e-5, 0.7
    x, f = (torch.randn(rows, hidden, dtype=torch.float64, requires_grad=True) for _ in range(2))
    u, w = (torch.randn(hidden, dtype=torch.float64, requires_grad=True) for _ in range(2))
    gate = torch.randn(3, hidden, dtype=torch.float64, requires_grad=True)

    def norm(t, weight):
        return t / torch.sqrt((t * t).mean(1, keepdim=True) + eps) * weight

    stream = scale * x + gate.repeat_interleave(2, 0) * norm(f, u)
    y = norm(stream, w)
    d_stream, dy = torch.randn_like(y), torch.randn_like(y)
    want = torch.autograd.grad((stream * d_stream).sum() + (y * dy).sum(), (x, f, u, gate, w))
    with torch.no_grad():
        got = sandwich_backward(stream, f, u, gate, w, scale, eps, d_stream, dy)
        there = sandwich_forward(x, f, u, gate, w, scale, eps, stream)
    assert torch.allclose(there["stream"].value, stream, rtol=1e-12, atol=1e-12) and torch.allclose(there["y"].value, y, rtol=1e-12, atol=1e-12)
    for name, g in zip(("dx", "df", "du", "d_gate", "dw"), want):
        assert torch.allclose(got[name].value, g, rtol=1e-10, atol=1e-10), name
