"""Cases of the operators of an attention branch around a residual stream: layer norm in front of it, differential attention
with its learned weights inside, dropout onto the stream behind it. Each is measured in training, forward and backward.

  layernorm_forward     y = (x - mean) / sqrt(var + epsilon) * w + b, row by row
  layernorm_backward    its gradient (added to the stream's where a case has one), with those of w and b
  dropout               forward (onto the stream where a case has one) and backward with the same mask, which is never stored
  lambda                the weight of each head's second map from its learned vectors, and their gradient
  attention_forward     (softmax(q1 k1') - lambda softmax(q2 k2')) v with what its backward pass needs
  attention_backward    the gradient of q, k, v and lambda

Where `own` is false, `run` computes the operators with elementary torch operations in 32 bits, rounded once at the end; where it
is true it calls the library. `exact` computes them in 64 bits in another way: the gradients by differentiation of the forward
formula, the generator of the masks in numpy.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False  # whether `run` calls the library

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
EPSILON = 1e-5


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # One short prompt through a norm of the narrow decoder: what counts is the way to the kernel and back.
        {"name": "layernorm_forward_f16_r16_h768", "path": "layernorm_forward", "rows": 16, "hidden": 768, "bias": True, "dtype": "f16"},
        # A norm of the training batch, 32 sequences of 1024 tokens.
        {"name": "layernorm_forward_bf16_r32768_h1024", "path": "layernorm_forward", "rows": 32768, "hidden": 1024, "bias": True,
         "dtype": "bf16"},
        # A width that no vector divides, in the precision that numerics are checked in, without a bias.
        {"name": "layernorm_backward_f32_r5005_h1001", "path": "layernorm_backward", "rows": 5005, "hidden": 1001, "bias": False,
         "residual": False, "dtype": "f32"},
        # The gradient of a norm of the training batch, added to the gradient that the stream carries past the branch.
        {"name": "layernorm_backward_bf16_r32768_h1024", "path": "layernorm_backward", "rows": 32768, "hidden": 1024, "bias": True,
         "residual": True, "dtype": "bf16"},
        # A first experiment's activations, an odd number of them.
        {"name": "dropout_f16_n76799", "path": "dropout", "count": 76799, "probability": 0.2, "residual": False, "dtype": "f16"},
        # A branch of the training batch dropped out onto the stream.
        {"name": "dropout_bf16_n33554432", "path": "dropout", "count": 32768 * 1024, "probability": 0.1, "residual": True, "dtype": "bf16"},
        # The weights of one layer's heads, vectors of half a head each: every head its own, and one set for all heads.
        {"name": "lambda_f32_h8_d64", "path": "lambda", "sets": 8, "heads": 8, "width": 64, "dtype": "f32"},
        {"name": "lambda_bf16_h12_shared_d32", "path": "lambda", "sets": 1, "heads": 12, "width": 32, "dtype": "bf16"},
        # A small model's micro-batch of a length that is no multiple of anything.
        {"name": "attention_forward_f16_b3_t100", "path": "attention_forward", "batch": 3, "queries": 100, "keys": 100, "heads": 4,
         "kv_heads": 2, "head_dim": 64, "causal": True, "dtype": "f16"},
        # The training batch.
        {"name": "attention_forward_bf16_b32_t1024", "path": "attention_forward", "batch": 32, "queries": 1024, "keys": 1024, "heads": 8,
         "kv_heads": 2, "head_dim": 128, "causal": True, "dtype": "bf16"},
        {"name": "attention_backward_bf16_b32_t1024", "path": "attention_backward", "batch": 32, "queries": 1024, "keys": 1024, "heads": 8,
         "kv_heads": 2, "head_dim": 128, "causal": True, "dtype": "bf16"},
        # A ragged micro-batch of the narrow decoder.
        {"name": "attention_backward_f16_b5_t1001", "path": "attention_backward", "batch": 5, "queries": 1001, "keys": 1001, "heads": 12,
         "kv_heads": 4, "head_dim": 64, "causal": True, "dtype": "f16"},
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    """One more case: the same operators over sizes from a few values to those of the training batch."""
    path = rng.choice(["layernorm_forward", "layernorm_backward", "dropout", "lambda", "attention_forward", "attention_forward",
                       "attention_backward", "attention_backward"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if path.startswith("layernorm"):
        hidden = _log_int(rng, 32, 8192)
        if rng.random() < 0.6:
            hidden = max(32, hidden // 32 * 32)
        rows = _log_int(rng, 1, max(1, 32768 * 1024 // hidden // (2 if dtype == "f32" else 1)))
        case = {"path": path, "rows": rows, "hidden": hidden, "bias": rng.random() < 0.7, "dtype": dtype}
        if path == "layernorm_backward":
            case["residual"] = rng.random() < 0.5
        return case
    if path == "dropout":
        return {"path": path, "count": _log_int(rng, 1000, 32768 * 1024 // (2 if dtype == "f32" else 1)),
                "probability": rng.choice([0.05, 0.1, 0.2, 0.3, 0.5]), "residual": rng.random() < 0.5, "dtype": dtype}
    if path == "lambda":
        heads = rng.randint(1, 64)
        return {"path": path, "sets": rng.choice([1, heads]), "heads": heads, "width": rng.choice([16, 24, 32, 40, 48, 64, 100, 128]),
                "dtype": dtype}
    kv_heads, group = rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 2, 3, 4])
    heads = kv_heads * group
    head_dim = rng.choice([32, 64, 64, 80, 96, 128, 128])
    causal = rng.random() < 0.75
    queries = _log_int(rng, 1, 512 if dtype == "f32" else 4096)
    keys = queries + (rng.choice([0, 0, 64, 333]) if causal else 0)
    if not causal:
        keys = _log_int(rng, 1, 512 if dtype == "f32" else 4096)
    limit = 32 * 8 * 1024 * 1024 // (16 if dtype == "f32" else 1)  # entries of the score matrices
    batch = min(32, max(1, _log_int(rng, 1, max(1, limit // (heads * queries * keys)))))
    if batch * heads * queries * keys > limit:
        batch, heads, kv_heads = 1, kv_heads, kv_heads
        if heads * queries * keys > limit:
            heads = kv_heads = 1
    return {"path": path, "batch": batch, "queries": queries, "keys": keys, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "causal": causal, "dtype": dtype}


# ------------------------------------------------------------------------------------------------ inputs
def _normal(generator, shape, dtype, deviation=1.0):
    return (torch.randn(shape, generator=generator, device="cuda", dtype=torch.float32) * deviation).to(dtype)


def prepare(case, seed):
    """Normal activations and gradients, norm weights around 1; a few channels of the stream are larger than the rest, as they are in
    trained models. What a backward pass is given of its forward pass comes from the plain form."""
    generator = torch.Generator(device="cuda").manual_seed(seed)
    dtype, path = DTYPES[case["dtype"]], case["path"]
    state = {"case": case}
    if path.startswith("layernorm"):
        rows, hidden = case["rows"], case["hidden"]
        channel = 1.0 + 4.0 * (torch.rand(hidden, generator=generator, device="cuda") < 0.02)
        state["x"] = (torch.randn((rows, hidden), generator=generator, device="cuda") * channel + 0.3).to(dtype)
        state["w"] = (1.0 + 0.1 * torch.randn(hidden, generator=generator, device="cuda")).to(dtype)
        state["b"] = _normal(generator, hidden, dtype, 0.1) if case["bias"] else None
        state["out"] = torch.empty_like(state["x"])
        if path == "layernorm_backward":
            state["dy"] = _normal(generator, (rows, hidden), dtype, 0.1)
            state["residual"] = _normal(generator, (rows, hidden), dtype, 0.1) if case["residual"] else None
            state["dw"] = torch.empty_like(state["w"])
            state["db"] = torch.empty_like(state["w"]) if case["bias"] else None
    elif path == "dropout":
        state["x"] = _normal(generator, case["count"], dtype)
        state["residual"] = _normal(generator, case["count"], dtype) if case["residual"] else None
        state["dy"] = _normal(generator, case["count"], dtype, 0.1)
        state["seed"] = seed * 0x9E3779B9 % 2**63  # of the run, and how far its masks have come
        state["offset"] = seed * 1_000_003 % 2**40
        state["out"], state["dx"] = torch.empty_like(state["x"]), torch.empty_like(state["x"])
    elif path == "lambda":
        shape = (case["sets"], case["width"])
        state["vectors"] = [_normal(generator, shape, dtype, 0.1) for _ in range(4)]  # q1, k1, q2, k2
        state["initial"] = 0.8 - 0.6 * math.exp(-0.3 * (seed % 12))  # by the layer's depth
        state["dlambda"] = _normal(generator, case["heads"], torch.float32, 1.0)
        state["out"] = torch.empty(case["heads"], device="cuda")
        state["grads"] = [torch.empty_like(v) for v in state["vectors"]]
    else:
        q_shape = (case["batch"], case["queries"], case["heads"], case["head_dim"])
        kv_shape = (case["batch"], case["keys"], case["kv_heads"], case["head_dim"])
        state["q"], state["k"], state["v"] = (_normal(generator, shape, dtype) for shape in (q_shape, kv_shape, kv_shape))
        state["lambdas"] = 0.2 + 0.6 * torch.rand(case["heads"], generator=generator, device="cuda")
        state["out"], state["second"] = torch.empty_like(state["q"]), torch.empty_like(state["q"])
        state["lse"] = torch.empty((2, *q_shape[:3]), device="cuda")
        if path == "attention_backward":
            out, second, lse = _attention_forward(state)
            state["out"].copy_(out)
            state["second"].copy_(second)
            state["lse"].copy_(lse)
            state["dout"] = _normal(generator, q_shape, dtype)
            state["dq"], state["dk"], state["dv"] = (torch.empty_like(state[name]) for name in ("q", "k", "v"))
            state["dlambdas"] = torch.empty_like(state["lambdas"])
    return state


# ------------------------------------------------------------------------------------------------ plain forms
def _layernorm_forward(state):
    x = state["x"].float()
    centred = x - x.mean(dim=1, keepdim=True)
    y = centred * (1.0 / torch.sqrt((centred * centred).mean(dim=1, keepdim=True) + EPSILON)) * state["w"].float()
    if state["b"] is not None:
        y = y + state["b"].float()
    return [y.to(state["x"].dtype)]


def _layernorm_backward(state):
    x, dy, w = state["x"].float(), state["dy"].float(), state["w"].float()
    centred = x - x.mean(dim=1, keepdim=True)
    inverse = 1.0 / torch.sqrt((centred * centred).mean(dim=1, keepdim=True) + EPSILON)
    normed = centred * inverse
    scaled = dy * w
    dx = inverse * (scaled - scaled.mean(dim=1, keepdim=True) - normed * (scaled * normed).mean(dim=1, keepdim=True))
    if state["residual"] is not None:
        dx = dx + state["residual"].float()
    out = [dx.to(state["x"].dtype), (dy * normed).sum(dim=0).to(state["w"].dtype)]
    if state["db"] is not None:
        out.append(dy.sum(dim=0).to(state["w"].dtype))
    return out


def _multiply_32(constant, word):
    """High and low 32 bits of the product of two 32-bit numbers, in 64-bit integers that it would overflow."""
    low = constant * (word & 0xFFFF)
    high = constant * (word >> 16) + (low >> 16)
    return high >> 16, ((high & 0xFFFF) << 16) | (low & 0xFFFF)


def _random_16(count, seed, offset):
    """`count` numbers of 16 bits: Philox 4x32 with ten rounds (Salmon, Moraes, Dror and Shaw, 2011), its key the seed, eight numbers from
    each value of its counter, of which the first is the offset."""
    n = torch.arange((count + 7) // 8, device="cuda", dtype=torch.int64) + offset
    c0, c1, c2, c3 = n & 0xFFFFFFFF, n >> 32, torch.zeros_like(n), torch.zeros_like(n)
    k0, k1 = seed & 0xFFFFFFFF, seed >> 32
    for _ in range(10):
        high0, low0 = _multiply_32(0xD2511F53, c0)
        high1, low1 = _multiply_32(0xCD9E8D57, c2)
        c0, c1, c2, c3 = high1 ^ c1 ^ k0, low1, high0 ^ c3 ^ k1, low0
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    halves = [part for c in (c0, c1, c2, c3) for part in (c & 0xFFFF, c >> 16)]
    return torch.stack(halves, dim=1).reshape(-1)[:count]


def _dropout(state):
    x, case = state["x"], state["case"]
    threshold = int(case["probability"] * 65536 + 0.5)
    kept = _random_16(x.numel(), state["seed"], state["offset"]) >= threshold
    factor = torch.where(kept, 65536.0 / (65536 - threshold), 0.0)
    out = x.float() * factor
    if state["residual"] is not None:
        out = out + state["residual"].float()
    return [out.to(x.dtype), (state["dy"].float() * factor).to(x.dtype)]


def _lambda(state):
    q1, k1, q2, k2 = (v.float() for v in state["vectors"])
    case, dlambda = state["case"], state["dlambda"]
    first = torch.exp((q1 * k1).sum(dim=1, keepdim=True))
    second = torch.exp((q2 * k2).sum(dim=1, keepdim=True))
    lambdas = (first - second + state["initial"]).reshape(-1).expand(case["heads"])
    of_set = dlambda.reshape(-1, 1) if case["sets"] > 1 else dlambda.sum().reshape(1, 1)
    first, second = of_set * first, of_set * second
    dtype = state["vectors"][0].dtype
    return [lambdas.contiguous(), *(g.to(dtype) for g in (first * k1, first * q1, -second * k2, -second * q2))]


def _heads_first(t, group=1):
    """[batch, tokens, heads, width] as fp32 [batch * heads * group, tokens, width]."""
    t = t.float().permute(0, 2, 1, 3)
    if group > 1:
        t = t.unsqueeze(2).expand(-1, -1, group, -1, -1)
    return t.reshape(-1, *t.shape[-2:]).contiguous()


def _tokens_first(t, batch):
    return t.reshape(batch, -1, *t.shape[1:]).permute(0, 2, 1, 3)


def _hidden(case):
    """[queries, keys], true where the causal mask hides a key from a query; the last query sees all keys."""
    q = torch.arange(case["queries"], device="cuda").reshape(-1, 1) + (case["keys"] - case["queries"])
    return torch.arange(case["keys"], device="cuda").reshape(1, -1) > q


def _maps(state):
    """The two softmax maps and the logarithms of their sums, and v: fp32, heads first."""
    case = state["case"]
    group, half = case["heads"] // case["kv_heads"], case["head_dim"] // 2
    q, k, v = _heads_first(state["q"]), _heads_first(state["k"], group), _heads_first(state["v"], group)
    hidden = _hidden(case) if case["causal"] else None
    maps, sums = [], []
    for columns in (slice(0, half), slice(half, 2 * half)):
        scores = torch.matmul(q[..., columns].contiguous(), k[..., columns].transpose(1, 2).contiguous()) * (1.0 / math.sqrt(half))
        if hidden is not None:
            scores = scores.masked_fill_(hidden, -math.inf)
        top = scores.max(dim=-1, keepdim=True).values
        scores = scores.sub_(top).exp_()
        total = scores.sum(dim=-1, keepdim=True)
        maps.append(scores.div_(total))
        sums.append((top + torch.log(total)).squeeze(-1))
    return maps, sums, q, k, v


def _per_head(state):
    return state["lambdas"].repeat(state["case"]["batch"]).reshape(-1, 1, 1)


def _attention_forward(state):
    case, dtype = state["case"], state["q"].dtype
    (p1, p2), sums, _, _, v = _maps(state)
    first, second = torch.matmul(p1, v), torch.matmul(p2, v)
    out = first - _per_head(state) * second
    lse = torch.stack([s.reshape(case["batch"], case["heads"], -1).permute(0, 2, 1) for s in sums])
    return [_tokens_first(out, case["batch"]).to(dtype).contiguous(), _tokens_first(second, case["batch"]).to(dtype).contiguous(),
            lse.contiguous()]


def _attention_backward(state):
    case, dtype = state["case"], state["q"].dtype
    batch, kv_heads, half = case["batch"], case["kv_heads"], case["head_dim"] // 2
    group, scale = case["heads"] // kv_heads, 1.0 / math.sqrt(half)
    (p1, p2), _, q, k, v = _maps(state)
    dout = _heads_first(state["dout"])
    lambdas = _per_head(state)
    dp = torch.matmul(dout, v.transpose(1, 2).contiguous())
    dv = torch.matmul((p1 - lambdas * p2).transpose(1, 2).contiguous(), dout)
    delta1, delta2 = (p1 * dp).sum(dim=-1, keepdim=True), (p2 * dp).sum(dim=-1, keepdim=True)
    dlambdas = -delta2.reshape(batch, case["heads"], -1).sum(dim=(0, 2))
    ds1 = p1.mul_(dp - delta1).mul_(scale)
    ds2 = p2.mul_(dp - delta2).mul_(-scale * lambdas)
    k1, k2 = k[..., :half].contiguous(), k[..., half:].contiguous()
    dq = torch.cat([torch.matmul(ds1, k1), torch.matmul(ds2, k2)], dim=-1)
    q1, q2 = q[..., :half].contiguous(), q[..., half:].contiguous()
    dk = torch.cat([torch.matmul(ds1.transpose(1, 2).contiguous(), q1), torch.matmul(ds2.transpose(1, 2).contiguous(), q2)], dim=-1)
    dk, dv = (t.reshape(batch * kv_heads, group, *t.shape[1:]).sum(dim=1) for t in (dk, dv))
    return [_tokens_first(t, batch).to(dtype).contiguous() for t in (dq, dk, dv)] + [dlambdas]


_PLAIN = {"layernorm_forward": _layernorm_forward, "layernorm_backward": _layernorm_backward, "dropout": _dropout, "lambda": _lambda,
          "attention_forward": _attention_forward, "attention_backward": _attention_backward}


# ------------------------------------------------------------------------------------------------ the library
def _own(state):
    from cgpt_amd import ops

    case = state["case"]
    path = case["path"]
    if path == "layernorm_forward":
        ops.layernorm_forward(state["out"], state["x"], state["w"], state["b"], EPSILON)
        return [state["out"]]
    if path == "layernorm_backward":
        ops.layernorm_backward(state["out"], state["dw"], state["db"], state["dy"], state["x"], state["w"], EPSILON, None, state["residual"])
        return [t for t in (state["out"], state["dw"], state["db"]) if t is not None]
    if path == "dropout":
        options = ops.DropoutOptions(probability=case["probability"], seed=state["seed"], offset=state["offset"])
        ops.dropout_forward(state["out"], state["x"], state["residual"], None, options)
        ops.dropout_backward(state["dx"], state["dy"], None, options)
        return [state["out"], state["dx"]]
    if path == "lambda":
        ops.differential_lambda_forward(state["out"], *state["vectors"], state["initial"])
        ops.differential_lambda_backward(*state["grads"], state["dlambda"], *state["vectors"])
        return [state["out"], *state["grads"]]
    options = ops.FlashAttentionOptions(num_query_heads=case["heads"], num_kv_heads=case["kv_heads"], head_dim=case["head_dim"],
                                        causal=case["causal"],
                                        query_position_offset=case["keys"] - case["queries"] if case["causal"] else 0)
    if path == "attention_forward":
        ops.differential_attention_forward(state["out"], state["second"], state["lse"], state["q"], state["k"], state["v"],
                                           state["lambdas"], None, options)
        return [state["out"], state["second"], state["lse"]]
    ops.differential_attention_backward(state["dq"], state["dk"], state["dv"], state["dlambdas"], state["dout"], state["out"],
                                        state["second"], state["lse"], state["q"], state["k"], state["v"], state["lambdas"], None, options)
    return [state["dq"], state["dk"], state["dv"], state["dlambdas"]]


def run(state):
    return _own(state) if own else _PLAIN[state["case"]["path"]](state)


# ------------------------------------------------------------------------------------------------ work
def work(case):
    """Bytes: every input read once, every output written once. Flops: two for each multiply-add of the products, one for each other
    operation of the formulas; the 32-bit integer operations of the generator are not counted."""
    size = 4 if case["dtype"] == "f32" else 2
    path = case["path"]
    if path == "layernorm_forward":
        values, hidden = case["rows"] * case["hidden"], case["hidden"]
        return {"bytes": size * (2 * values + hidden * (2 if case["bias"] else 1)), "flops": 7 * values}
    if path == "layernorm_backward":
        values, hidden = case["rows"] * case["hidden"], case["hidden"]
        return {"bytes": size * (values * (4 if case["residual"] else 3) + hidden * (3 if case["bias"] else 2)), "flops": 15 * values}
    if path == "dropout":
        return {"bytes": size * case["count"] * (5 if case["residual"] else 4), "flops": 4 * case["count"]}
    if path == "lambda":
        vectors = case["sets"] * case["width"]
        return {"bytes": size * 4 * vectors * 2 + 4 * 2 * case["heads"], "flops": 8 * vectors}
    queries, keys = case["queries"], case["keys"]
    pairs = queries * (keys - queries) + queries * (queries + 1) // 2 if case["causal"] else queries * keys
    pairs *= case["batch"] * case["heads"]
    q_values = case["batch"] * queries * case["heads"] * case["head_dim"]
    kv_values = case["batch"] * keys * case["kv_heads"] * case["head_dim"]
    rows = case["batch"] * queries * case["heads"]
    if path == "attention_forward":  # two score maps of half the width, two products with v
        return {"bytes": size * (3 * q_values + 2 * kv_values) + 8 * rows + 4 * case["heads"], "flops": 6 * pairs * case["head_dim"]}
    # the score maps again, the gradient of the maps, and of q, k and v
    return {"bytes": size * (5 * q_values + 4 * kv_values) + 8 * rows + 8 * case["heads"], "flops": 10 * pairs * case["head_dim"]}


# ------------------------------------------------------------------------------------------------ 64 bits
def _exact_mask(count, seed, offset, threshold):
    n = (np.arange((count + 7) // 8, dtype=np.uint64) + np.uint64(offset))
    words = [n & np.uint64(0xFFFFFFFF), n >> np.uint64(32), np.zeros_like(n), np.zeros_like(n)]
    key = [np.uint64(seed & 0xFFFFFFFF), np.uint64(seed >> 32)]
    mask = np.uint64(0xFFFFFFFF)
    for _ in range(10):
        a, b = words[0] * np.uint64(0xD2511F53), words[2] * np.uint64(0xCD9E8D57)
        words = [(b >> np.uint64(32)) ^ words[1] ^ key[0], b & mask, (a >> np.uint64(32)) ^ words[3] ^ key[1], a & mask]
        key = [(key[0] + np.uint64(0x9E3779B9)) & mask, (key[1] + np.uint64(0xBB67AE85)) & mask]
    numbers = np.empty((n.size, 4), dtype="<u4")
    for i, word in enumerate(words):
        numbers[:, i] = word
    return torch.from_numpy(numbers.view("<u2").reshape(-1)[:count].astype(np.int32) >= threshold).cuda()


def _exact_attention(state, backward):
    """One batch entry at a time, the gradients by differentiation."""
    case = state["case"]
    group, width = case["heads"] // case["kv_heads"], case["head_dim"]
    causal_bias = torch.zeros((case["queries"], case["keys"]), dtype=torch.float64, device="cuda")
    if case["causal"]:
        causal_bias[_hidden(case)] = -math.inf
    results, dlambdas = [], torch.zeros(case["heads"], dtype=torch.float64, device="cuda")
    for b in range(case["batch"]):
        q, k, v = (state[name][b].double().requires_grad_(backward) for name in ("q", "k", "v"))
        lambdas = state["lambdas"].double().requires_grad_(backward)
        outs, seconds, sums = [], [], []
        for h in range(case["heads"]):
            kv = h // group
            parts = []
            for columns in (slice(0, width // 2), slice(width // 2, width)):
                logits = torch.mm(q[:, h, columns], k[:, kv, columns].T) / math.sqrt(width // 2) + causal_bias
                parts.append(torch.mm(torch.softmax(logits, dim=1), v[:, kv]))
                sums.append(torch.logsumexp(logits, dim=1).detach())
            outs.append(parts[0] - lambdas[h] * parts[1])
            seconds.append(parts[1].detach())
        out = torch.stack(outs, dim=1)
        if not backward:
            lse = torch.stack(sums, dim=1).reshape(case["queries"], case["heads"], 2).permute(2, 0, 1)
            results.append((out.detach(), torch.stack(seconds, dim=1), lse))
            continue
        grads = torch.autograd.grad(out, (q, k, v, lambdas), state["dout"][b].double())
        results.append(grads[:3])
        dlambdas += grads[3]
    joined = [torch.stack(parts) for parts in zip(*results)]
    if backward:
        return [*joined, dlambdas]
    return [joined[0], joined[1], joined[2].transpose(0, 1).contiguous()]


def exact(case, seed):
    state = prepare(case, seed)
    path = case["path"]
    if path.startswith("layernorm"):
        x, w = state["x"].double(), state["w"].double()
        b = state["b"].double() if state["b"] is not None else torch.zeros_like(w)
        leaves = [t.requires_grad_(path == "layernorm_backward") for t in (x, w, b)]
        variance = torch.var(x, dim=1, unbiased=False, keepdim=True)
        y = (x - torch.mean(x, dim=1, keepdim=True)) * torch.rsqrt(variance + EPSILON) * w + b
        if path == "layernorm_forward":
            return [y]
        dx, dw, db = torch.autograd.grad(y, leaves, state["dy"].double())
        if state["residual"] is not None:
            dx = dx + state["residual"].double()
        return [dx, dw, db] if case["bias"] else [dx, dw]
    if path == "dropout":
        threshold = int(case["probability"] * 65536 + 0.5)
        kept = _exact_mask(case["count"], state["seed"], state["offset"], threshold)
        keep = (65536 - threshold) / 65536
        out, dx = (torch.where(kept, t.double() / keep, torch.zeros((), dtype=torch.float64, device="cuda")) for t in (state["x"], state["dy"]))
        return [out + state["residual"].double() if case["residual"] else out, dx]
    if path == "lambda":
        vectors = [v.double().requires_grad_() for v in state["vectors"]]
        q1, k1, q2, k2 = vectors
        lambdas = torch.exp((q1 * k1).sum(1)) - torch.exp((q2 * k2).sum(1)) + state["initial"]
        lambdas = lambdas.expand(case["heads"])
        return [lambdas.detach().clone(), *torch.autograd.grad(lambdas, vectors, state["dlambda"].double())]
    return _exact_attention(state, path == "attention_backward")
