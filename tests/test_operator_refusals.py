"""Arguments that layer norm, dropout and differential attention refuse, through the C entries and the Python mirror, before
anything is launched (so these run without a GPU)."""
import ctypes

import pytest
import torch

from cgpt_amd import capi, ops

N = ctypes.c_void_p(0)
P = ctypes.c_void_p(0x1000)  # never dereferenced: validation fails first
NAN, INF = float("nan"), float("inf")
F, B, H = capi.F32, capi.BF16, capi.F16
QKV = (P, P, P, P)  # query, key, value, lambda


def attention(batch=1, qs=8, ks=8, hq=2, hkv=1, d=32, scale=0.0, causal=1, offset=0, dtype=B):
    return (batch, qs, ks, hq, hkv, d, scale, causal, offset, dtype, N)


def attention_backward(*null, **shape):
    pointers = [N if i in null else P for i in range(12)]
    a = attention(**shape)
    return (*pointers, *a[:9], 0, *a[9:])


@pytest.mark.parametrize("name,args", [
    ("cgptx_layernorm_forward", (P, P, P, N, 4, 8, 0.0, B, N)),
    ("cgptx_layernorm_forward", (P, P, P, N, 4, 8, NAN, B, N)),
    ("cgptx_layernorm_forward", (P, P, P, N, 4, 8, INF, B, N)),
    ("cgptx_layernorm_forward", (P, P, P, N, 4, 8, 1e-5, 9, N)),
    ("cgptx_layernorm_forward", (P, P, P, N, 0, 8, 1e-5, B, N)),
    ("cgptx_layernorm_forward", (P, P, P, N, 4, 0, 1e-5, B, N)),
    ("cgptx_layernorm_forward", (P, P, P, N, 2**40, 8, 1e-5, B, N)),
    ("cgptx_layernorm_forward", (N, P, P, P, 4, 8, 1e-5, B, N)),
    ("cgptx_layernorm_forward", (P, N, P, P, 4, 8, 1e-5, B, N)),
    ("cgptx_layernorm_forward", (P, P, N, P, 4, 8, 1e-5, B, N)),
    ("cgptx_layernorm_backward", (P, P, P, P, P, P, N, 4, 8, -1.0, F, N)),
    ("cgptx_layernorm_backward", (P, P, P, P, P, P, N, 4, 8, 1e-5, -1, N)),
    ("cgptx_layernorm_backward", (P, N, P, P, P, P, N, 4, 8, 1e-5, F, N)),
    ("cgptx_layernorm_backward", (P, P, P, N, P, P, N, 4, 8, 1e-5, F, N)),
    ("cgptx_layernorm_backward", (P, P, P, P, P, N, N, 4, 8, 1e-5, F, N)),
    ("cgptx_dropout_forward", (P, P, N, 8, -0.1, 0, 0, N, B, N)),
    ("cgptx_dropout_forward", (P, P, N, 8, 1.1, 0, 0, N, B, N)),
    ("cgptx_dropout_forward", (P, P, N, 8, NAN, 0, 0, N, B, N)),
    ("cgptx_dropout_forward", (P, P, N, 8, 0.1, 0, 0, N, 5, N)),
    ("cgptx_dropout_forward", (N, P, N, 8, 0.1, 0, 0, N, B, N)),
    ("cgptx_dropout_forward", (P, N, N, 8, 0.1, 0, 0, N, B, N)),
    ("cgptx_dropout_forward", (P, P, N, 8, 0.1, 0, 0, ctypes.c_void_p(0x1004), B, N)),
    ("cgptx_dropout_backward", (P, P, 8, 2.0, 0, 0, N, 0, B, N)),
    ("cgptx_dropout_backward", (P, N, 8, 0.5, 0, 0, N, 0, B, N)),
    ("cgptx_differential_lambda_forward", (P, P, P, P, P, 0.2, 3, 8, 16, F, N)),   # neither one set nor one for each
    ("cgptx_differential_lambda_forward", (P, P, P, P, P, 0.2, 0, 0, 16, F, N)),
    ("cgptx_differential_lambda_forward", (P, P, P, P, P, 0.2, 8, 8, 0, F, N)),
    ("cgptx_differential_lambda_forward", (P, P, P, P, P, NAN, 8, 8, 16, F, N)),
    ("cgptx_differential_lambda_forward", (P, P, N, P, P, 0.2, 8, 8, 16, F, N)),
    ("cgptx_differential_lambda_forward", (N, P, P, P, P, 0.2, 8, 8, 16, F, N)),
    ("cgptx_differential_lambda_backward", (P, P, P, P, N, P, P, P, P, 8, 8, 16, F, N)),
    ("cgptx_differential_lambda_backward", (P, P, P, N, P, P, P, P, P, 8, 8, 16, F, N)),
    ("cgptx_differential_lambda_backward", (P, P, P, P, P, P, P, P, P, 2, 8, 16, F, N)),
    ("cgptx_differential_attention_forward", (P, P, P, *QKV, *attention(d=33))),
    ("cgptx_differential_attention_forward", (P, P, P, *QKV, *attention(d=130))),
    ("cgptx_differential_attention_forward", (P, P, P, *QKV, *attention(hq=3, hkv=2))),
    ("cgptx_differential_attention_forward", (P, P, P, *QKV, *attention(qs=0))),
    ("cgptx_differential_attention_forward", (P, P, P, *QKV, *attention(ks=0, causal=0))),
    ("cgptx_differential_attention_forward", (P, P, P, *QKV, *attention(qs=9))),        # queries that see no key of their own
    ("cgptx_differential_attention_forward", (P, P, P, *QKV, *attention(offset=1))),
    ("cgptx_differential_attention_forward", (P, P, P, *QKV, *attention(offset=2**63))),
    ("cgptx_differential_attention_forward", (P, P, P, *QKV, *attention(scale=INF))),
    ("cgptx_differential_attention_forward", (P, P, P, *QKV, *attention(dtype=3))),
    ("cgptx_differential_attention_forward", (N, P, P, *QKV, *attention())),
    ("cgptx_differential_attention_forward", (P, P, P, P, P, P, N, *attention())),
    *[("cgptx_differential_attention_backward", attention_backward(i)) for i in range(12)],
    ("cgptx_differential_attention_backward", attention_backward(d=7)),
    ("cgptx_differential_attention_backward", attention_backward(hkv=0)),
])
def test_invalid_arguments(name, args):
    with pytest.raises(ValueError):
        capi.call(name, *args)


@pytest.mark.parametrize("shape", [dict(batch=70000), dict(hq=70000, hkv=1), dict(qs=2**31, ks=2**31), dict(batch=65535, qs=2**20, ks=2**20)])
def test_sizes_past_the_range(shape):
    with pytest.raises(OverflowError):
        capi.call("cgptx_differential_attention_forward", P, P, P, *QKV, *attention(**shape))
    with pytest.raises(OverflowError):
        capi.call("cgptx_differential_attention_backward", *attention_backward(**shape))


def test_no_elements_need_no_tensors():
    capi.call("cgptx_dropout_forward", N, N, N, 0, 0.5, 1, 2, N, B, N)
    capi.call("cgptx_dropout_backward", N, N, 0, 0.5, 1, 2, N, 0, B, N)


def test_tensors_that_are_not_on_a_device():
    x, w = torch.zeros(4, 8), torch.zeros(8)
    q, lam, lse = torch.zeros(1, 4, 2, 32), torch.zeros(2), torch.zeros(2, 1, 4, 2)
    options = ops.FlashAttentionOptions(num_query_heads=2, num_kv_heads=2, head_dim=32)
    vectors = [torch.zeros(2, 16) for _ in range(4)]
    for call in (lambda: ops.layernorm_forward(x, x, w, w, 1e-5), lambda: ops.layernorm_backward(x, w, w, x, x, w, 1e-5),
                 lambda: ops.dropout_forward(x, x), lambda: ops.dropout_backward(x, x),
                 lambda: ops.differential_attention_forward(q, q, lse, q, q, q, lam, None, options),
                 lambda: ops.differential_attention_backward(q, q, q, lam, q, q, q, lse, q, q, q, lam, None, options),
                 lambda: ops.differential_lambda_forward(lam, *vectors, 0.2),
                 lambda: ops.differential_lambda_backward(*vectors, lam, *vectors)):
        with pytest.raises(ValueError, match="device"):
            call()


@pytest.mark.gpu
def test_shapes_and_types_that_do_not_fit(device):
    def t(*shape, dtype=torch.bfloat16):
        return torch.zeros(shape, dtype=dtype, device=device)

    x, w, f = t(4, 8), t(8), torch.float32
    q, k, lam, lse = t(1, 4, 2, 32), t(1, 4, 1, 32), t(2, dtype=f), t(2, 1, 4, 2, dtype=f)
    att = ops.FlashAttentionOptions(num_query_heads=2, num_kv_heads=1, head_dim=32)
    odd = ops.FlashAttentionOptions(num_query_heads=2, num_kv_heads=1, head_dim=31)
    v = [t(2, 16) for _ in range(4)]
    calls = [
        lambda: ops.layernorm_forward(x, x, t(7), None, 1e-5), lambda: ops.layernorm_forward(x, x, w, t(9), 1e-5),
        lambda: ops.layernorm_forward(t(4, 9), x, w, None, 1e-5), lambda: ops.layernorm_forward(x, x, w.float(), None, 1e-5),
        lambda: ops.layernorm_forward(x, x, w, None, 0.0), lambda: ops.layernorm_forward(x.t(), x.t(), t(4), None, 1e-5),
        lambda: ops.layernorm_backward(x, w, t(9), x, x, w, 1e-5), lambda: ops.layernorm_backward(x, w, w, x, x, w, 1e-5, None, t(4, 9)),
        lambda: ops.layernorm_backward(x, w, w, t(5, 8), x, w, 1e-5), lambda: ops.layernorm_backward(x, w, w, x, x, w, NAN),
        lambda: ops.dropout_forward(x, t(5, 8)), lambda: ops.dropout_forward(x, x, t(4, 9)), lambda: ops.dropout_forward(x, x.float()),
        lambda: ops.dropout_forward(x, x, None, None, ops.DropoutOptions(1.5)), lambda: ops.dropout_forward(x, x, None, None, ops.DropoutOptions(NAN)),
        lambda: ops.dropout_forward(x, x, None, None, ops.DropoutOptions(0.1, -1)),
        lambda: ops.dropout_forward(x, x, None, None, ops.DropoutOptions(0.1, 0, 2**64)),
        lambda: ops.dropout_backward(x, x, None, ops.DropoutOptions(0.1, counter=t(1))),
        lambda: ops.dropout_backward(x, x, None, ops.DropoutOptions(0.1, counter=torch.zeros(1, dtype=torch.int64))),
        lambda: ops.dropout_backward(x, x, None, ops.DropoutOptions(0.1, counter=torch.zeros(2, dtype=torch.int64, device=device))),
        lambda: ops.differential_attention_forward(q, None, None, q, k, k, lam, None, odd),
        lambda: ops.differential_attention_forward(q, None, None, q, k, k, t(3, dtype=f), None, att),
        lambda: ops.differential_attention_forward(q, None, None, q, k, k, t(2), None, att),
        lambda: ops.differential_attention_forward(q, k, None, q, k, k, lam, None, att),
        lambda: ops.differential_attention_forward(q, q, t(1, 4, 2, dtype=f), q, k, k, lam, None, att),
        lambda: ops.differential_attention_backward(q, k, k, t(3, dtype=f), q, q, q, lse, q, k, k, lam, None, att),
        lambda: ops.differential_attention_backward(q, q, k, lam, q, q, q, lse, q, k, k, lam, None, att),
        lambda: ops.differential_attention_backward(q, k, k, lam, q, q, k, lse, q, k, k, lam, None, att),
        lambda: ops.differential_lambda_forward(lam, *v[:3], t(2, 15), 0.2), lambda: ops.differential_lambda_forward(t(3, dtype=f), *v, 0.2),
        lambda: ops.differential_lambda_forward(t(2), *v, 0.2), lambda: ops.differential_lambda_forward(lam, *v, NAN),
        lambda: ops.differential_lambda_backward(*v[:3], t(1, 16), lam, *v),
    ]
    for i, call in enumerate(calls):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was taken")
