"""Calls whose rows or columns are more than one launch has threads for: a launch has less than 2^32 of them along a grid's axis, and a
wavefront to a row, or 1024 threads to 32 columns, are more than that from 2^26 rows, or 2^27 columns, on. Each result is one that can be written
down for every element."""
import pytest
import torch

from cgpt_amd import ops
from tests.util import randn

pytestmark = pytest.mark.gpu


def attention(heads, d, causal):
    return ops.FlashAttentionOptions(num_query_heads=heads, num_kv_heads=heads, head_dim=d, causal=causal)


def pattern(shape, dtype, device):
    """Numbers of few bits that differ between neighbours."""
    count = 1
    for n in shape:
        count *= n
    return ((torch.arange(count, device=device, dtype=torch.int64) * 37 % 61 - 30).to(torch.float32) / 8).to(dtype).view(shape)


@pytest.mark.parametrize("dtype,d,batch,queries", [(torch.bfloat16, 2, 8192, 8193), (torch.float32, 6, 16384, 4097), (torch.float32, 8, 1, (1 << 27) + 5)],
                         ids=["bf16-2", "f32-6", "f32-8"])
def test_more_queries_than_threads(device, dtype, d, batch, queries):
    """One key: its share is 1 in either map, out = (1 - lambda) v, dv = (1 - lambda) sum dO, dlambda = -sum dO.v."""
    q = torch.zeros((batch, queries, 1, d), dtype=dtype, device=device)
    q[-1, -5:] = randn((5, 1, d), dtype, 1).to(device)
    k, v = randn((batch, 1, 1, d), dtype, 2).to(device), pattern((batch, 1, 1, d), dtype, device)
    lambdas = torch.tensor([0.25], device=device)
    out, second, lse = torch.full_like(q, 7.0), torch.full_like(q, 7.0), torch.full((2, batch, queries, 1), 7.0, device=device)
    ops.differential_attention_forward(out, second, lse, q, k, v, lambdas, None, attention(1, d, False))
    # A score less itself may leave what its product with the scale was rounded by: e of 1 + x, and e v / e in three roundings, of either map.
    for got, want in ((second, v.float()), (out, v.float() * 0.75)):
        assert ((got.float() - want).abs() <= 8 * 2.0 ** -24 * v.float().abs()).all()
        assert torch.equal(got[:-1], want[:-1].to(dtype).expand_as(got[:-1])) and torch.equal(got[-1, :-5], want[-1].to(dtype).expand_as(got[-1, :-5]))
    assert not lse[:, :-1].any() and not lse[:, :, :-5].any()
    if queries > 1 << 20:
        return  # one key's gradient is a sum over them all by one wavefront
    dout, grads = torch.zeros_like(q), [torch.full_like(t, 7.0) for t in (q, k, v, lambdas)]
    dout[:, 0], dout[:, queries // 2], dout[:, -1] = 1.0, 2.0, 4.0
    ops.differential_attention_backward(*grads, dout, out, second, lse, q, k, v, lambdas, None, attention(1, d, False))
    assert not grads[0].any() and not grads[1].any()
    assert torch.equal(grads[2], torch.full_like(v, 0.75 * 7.0))
    want, size = -7.0 * v.double().sum().item(), 7.0 * v.double().abs().sum().item()
    assert abs(grads[3].item() - want) <= 2.0 ** -20 * size


@pytest.mark.parametrize("dtype,d,keys", [(torch.bfloat16, 2, (1 << 26) + 7), (torch.float32, 6, (1 << 26) + 3), (torch.float32, 8, (1 << 27) + 5)],
                         ids=["bf16-2", "f32-6", "f32-8"])
def test_more_keys_than_threads(device, dtype, d, keys):
    """One query that sees the first key alone: the others' gradients are 0, or what they were."""
    q, dout = randn((1, 1, 1, d), dtype, 1).to(device), pattern((1, 1, 1, d), dtype, device)
    k = torch.zeros((1, keys, 1, d), dtype=dtype, device=device)
    v, lambdas = torch.zeros_like(k), torch.tensor([0.25], device=device)
    v[0, 0] = 1.0
    out, second, lse = torch.full_like(q, 7.0), torch.full_like(q, 7.0), torch.full((2, 1, 1, 1), 7.0, device=device)
    ops.differential_attention_forward(out, second, lse, q, k, v, lambdas, None, attention(1, d, True))
    assert (out == 0.75).all() and (second == 1.0).all() and not lse.any()
    grads = [torch.full_like(t, 7.0) for t in (q, k, v, lambdas)]
    ops.differential_attention_backward(*grads, dout, out, second, lse, q, k, v, lambdas, None, attention(1, d, True))
    assert not grads[0].any() and not grads[1][:, 1:].any() and not grads[2][:, 1:].any()
    assert torch.equal(grads[2][0, 0], (dout[0, 0].float() * 0.75).to(dtype))
    grads[1].fill_(3.0)
    grads[2].fill_(5.0)
    ops.differential_attention_backward(*grads, dout, out, second, lse, q, k, v, lambdas, None, attention(1, d, True), True)
    assert (grads[1][:, 1:] == 3.0).all() and (grads[2][:, 1:] == 5.0).all()


def test_layernorm_of_more_columns_than_threads(device):
    """Values of 1 and -1 by turns: the mean is 0 and the variance 1, exactly. dx = dy - mean(dy) - x mean(dy x) but for epsilon and rounding:
    in fp32 a mean of n terms in n/1024 + 30 additions one after the other is off by 2^-24 of the mean magnitude for each."""
    hidden = (1 << 27) + 70
    dtype = torch.bfloat16
    x = torch.ones((1, hidden), dtype=dtype, device=device)
    x[:, 1::2] = -1.0
    dy, w = pattern((1, hidden), dtype, device), torch.ones(hidden, dtype=dtype, device=device)
    dx, dw, db = torch.full_like(x, 99.0), torch.full_like(w, 99.0), torch.full_like(w, 99.0)
    ops.layernorm_backward(dx, dw, db, dy, x, w, 1e-9)
    assert torch.equal(db, dy[0]) and torch.equal(dw, (dy * x)[0])
    off = 2 * 2.0 ** -24 * (hidden / 1024 + 30) * dy.float().abs().mean().item()
    want = dy.float() - dy.double().mean().float() - x.float() * (dy.double() * x).mean().float()
    assert ((dx.float() - want).abs() <= want.abs() * 2.0 ** -8 * 1.01 + off).all()
