"""Cases of the operators of a decoder block whose mixer is linear attention: the attention itself, in training, for prompts and for
single tokens, and the norms that stand between two branches of such a block.

  attention_forward    o_t = scale sum_{s <= t} decay^(t - s) (q_t . k_s) v_s (+ the same of the state that came before), the decay one
                       per key/value head; the state behind the last token where a case keeps it
  attention_backward   the gradient of q, k, v, of the state before where a case has one, from those of o and of the last state
  attention_step       one new token for every sequence: S' = decay S + k' v, o = scale q S'
  norm_forward         x' = a x + gate * rmsnorm(f) u,  y = rmsnorm(x') w: the norm behind a branch, its gate and the scale of the stream,
                       and the norm in front of the next branch
  norm_backward        the gradients of x, f, u, gate and w from those of x' and y

Where `own` is false, `run` computes the operators with elementary torch operations in 32 bits (powers of the decay in 64), rounded
once at the end; where it is true it calls the library. `exact` computes them in 64 bits in another way: the recurrence token by token,
the gradients by differentiation of the definition.
"""
from __future__ import annotations

import math

import torch

own = False  # whether `run` calls the library

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
EPSILON = 1e-5
CHUNK = 64  # tokens that the plain form takes at a time


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # A small model's first prompt: what counts is the way to the kernel and back.
        {"name": "attention_forward_f16_b1_t77", "path": "attention_forward", "batch": 1, "tokens": 77, "heads": 4, "kv_heads": 2,
         "head_dim": 64, "state": True, "dtype": "f16"},
        # The training batch, 32 sequences of 1024 tokens.
        {"name": "attention_forward_bf16_b32_t1024", "path": "attention_forward", "batch": 32, "tokens": 1024, "heads": 8, "kv_heads": 2,
         "head_dim": 128, "state": False, "dtype": "bf16"},
        # One long prompt of the narrow decoder, of which the state is kept for the tokens to come.
        {"name": "attention_forward_bf16_b1_t32768", "path": "attention_forward", "batch": 1, "tokens": 32768, "heads": 12, "kv_heads": 4,
         "head_dim": 64, "state": True, "dtype": "bf16"},
        # The training batch, backward.
        {"name": "attention_backward_bf16_b32_t1024", "path": "attention_backward", "batch": 32, "tokens": 1024, "heads": 8, "kv_heads": 2,
         "head_dim": 128, "state": False, "dtype": "bf16"},
        # A ragged micro-batch of the narrow decoder that goes on from a state and hands one on.
        {"name": "attention_backward_f16_b5_t1001", "path": "attention_backward", "batch": 5, "tokens": 1001, "heads": 12, "kv_heads": 4,
         "head_dim": 64, "state": True, "dtype": "f16"},
        # A head width that is no power of two, in the precision that numerics are checked in.
        {"name": "attention_backward_f32_b2_t333_d40", "path": "attention_backward", "batch": 2, "tokens": 333, "heads": 4, "kv_heads": 4,
         "head_dim": 40, "state": False, "dtype": "f32"},
        # The next token of one conversation, and of many at once.
        {"name": "attention_step_bf16_b1", "path": "attention_step", "batch": 1, "heads": 8, "kv_heads": 2, "head_dim": 128, "dtype": "bf16"},
        {"name": "attention_step_bf16_b512", "path": "attention_step", "batch": 512, "heads": 8, "kv_heads": 2, "head_dim": 128,
         "dtype": "bf16"},
        # One short prompt between two branches of the narrow decoder.
        {"name": "norm_forward_f16_r16_h768", "path": "norm_forward", "rows": 16, "hidden": 768, "gates": 1, "scale": 1.0, "dtype": "f16"},
        # Between two branches of the training batch.
        {"name": "norm_forward_bf16_r32768_h1024", "path": "norm_forward", "rows": 32768, "hidden": 1024, "gates": 1, "scale": 0.9,
         "dtype": "bf16"},
        # The same backward, each sequence with a gate of its own (a condition that the model is given).
        {"name": "norm_backward_bf16_r32768_h1024_g32", "path": "norm_backward", "rows": 32768, "hidden": 1024, "gates": 32, "scale": 1.0,
         "dtype": "bf16"},
        # A width that no vector divides, a gate for every token, in the precision that numerics are checked in.
        {"name": "norm_backward_f32_r5005_h1001_g5005", "path": "norm_backward", "rows": 5005, "hidden": 1001, "gates": 5005, "scale": 0.5,
         "dtype": "f32"},
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    """One more case: the same operators over sizes from a few values to those of the training batch."""
    path = rng.choice(["attention_forward", "attention_forward", "attention_backward", "attention_backward", "attention_step", "norm_forward",
                       "norm_backward"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if path.startswith("norm"):
        hidden = _log_int(rng, 32, 8192)
        if rng.random() < 0.6:
            hidden = max(32, hidden // 32 * 32)
        sequences = _log_int(rng, 1, 64)
        most = max(1, 32768 * 1024 // hidden // sequences // (2 if dtype == "f32" else 1))
        rows = sequences * _log_int(rng, 1, most)
        return {"path": path, "rows": rows, "hidden": hidden, "gates": rng.choice([0, 1, 1, sequences, sequences, rows]),
                "scale": rng.choice([1.0, 1.0, 0.5, 0.9, 1.2]), "dtype": dtype}
    kv_heads, group = rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 2, 3, 4])
    heads, head_dim = kv_heads * group, rng.choice([32, 40, 64, 64, 80, 96, 128, 128])
    if path == "attention_step":
        most = 512 * 2 * 128 * 128 // (kv_heads * head_dim * head_dim)
        return {"path": path, "batch": min(1024, _log_int(rng, 1, most)), "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
                "dtype": dtype}
    tokens = _log_int(rng, 1, 16384 if path == "attention_forward" else 4096)
    limit = 32 * 1024 * 8 * 128 // (8 if dtype == "f32" else 1)  # values of q
    batch = min(32, max(1, _log_int(rng, 1, max(1, limit // (heads * head_dim * tokens)))))
    return {"path": path, "batch": batch, "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "state": rng.random() < 0.5, "dtype": dtype}


# ------------------------------------------------------------------------------------------------ inputs
def _normal(generator, shape, dtype, deviation=1.0):
    return (torch.randn(shape, generator=generator, device="cuda", dtype=torch.float32) * deviation).to(dtype)


def prepare(case, seed):
    """Normal activations and gradients; decays that forget half of what was said within one token to seven hundred; norm weights around
    1; a few channels of the stream are larger than the rest, as they are in trained models."""
    generator = torch.Generator(device="cuda").manual_seed(seed)
    dtype, path = DTYPES[case["dtype"]], case["path"]
    state = {"case": case}
    if path.startswith("norm"):
        rows, hidden, gates = case["rows"], case["hidden"], case["gates"]
        channel = 1.0 + 4.0 * (torch.rand(hidden, generator=generator, device="cuda") < 0.02)
        state["x"] = (torch.randn((rows, hidden), generator=generator, device="cuda") * channel).to(dtype)
        state["f"] = _normal(generator, (rows, hidden), dtype, 0.5)
        state["u"], state["w"] = ((1.0 + 0.1 * torch.randn(hidden, generator=generator, device="cuda")).to(dtype) for _ in range(2))
        state["gate"] = (0.5 + 0.2 * torch.randn((gates, hidden), generator=generator, device="cuda")).to(dtype) if gates else None
        if path == "norm_forward":
            state["stream"], state["y"] = torch.empty_like(state["x"]), torch.empty_like(state["x"])
        else:  # the stream behind the forward pass is what the backward pass is given
            state["d_stream"], state["d_y"] = (_normal(generator, (rows, hidden), dtype, 0.1) for _ in range(2))
            state["dx"], state["df"] = torch.empty_like(state["x"]), torch.empty_like(state["x"])
            state["du"], state["dw"] = torch.empty_like(state["u"]), torch.empty_like(state["w"])
            state["d_gate"] = torch.empty_like(state["gate"]) if gates else None
        return state
    batch, tokens, width = case["batch"], case.get("tokens", 1), case["head_dim"]
    q_shape, kv_shape = (batch, tokens, case["heads"], width), (batch, tokens, case["kv_heads"], width)
    state_shape = (batch, case["kv_heads"], width, width)
    state["q"], state["k"], state["v"] = (_normal(generator, shape, dtype) for shape in (q_shape, kv_shape, kv_shape))
    forget = torch.rand(case["kv_heads"], generator=generator, device="cuda")
    state["log_decay"] = -torch.exp(math.log(1e-3) + forget * (math.log(0.7) - math.log(1e-3)))
    before = path == "attention_step" or case["state"]
    state["before"] = _normal(generator, state_shape, torch.float32, 3.0) if before else None
    if path == "attention_backward":
        state["dout"] = _normal(generator, q_shape, dtype)
        state["d_after"] = _normal(generator, state_shape, torch.float32) if before else None
        state["dq"], state["dk"], state["dv"] = (torch.empty_like(state[name]) for name in ("q", "k", "v"))
        state["d_before"] = torch.empty_like(state["before"]) if before else None
    else:
        state["out"] = torch.empty_like(state["q"])
        state["after"] = torch.empty_like(state["before"]) if before else None
    return state


# ------------------------------------------------------------------------------------------------ plain forms
def _powers(log_decay, exponents):
    """decay^n for every head, computed in 64 bits: fp32 [heads, *exponents.shape]."""
    log_decay = log_decay.double().reshape(-1, *([1] * exponents.dim()))
    return torch.exp(log_decay * exponents.double()).float()


def _chunks(t, kv_heads):
    """[batch, tokens, heads, width] as fp32 [batch, kv_heads, group, chunks, CHUNK, width], zeros behind the last token."""
    batch, tokens, heads, width = t.shape
    chunks = -(-tokens // CHUNK)
    padded = torch.zeros((batch, chunks * CHUNK, heads, width), device=t.device)
    padded[:, :tokens] = t
    return padded.reshape(batch, chunks, CHUNK, kv_heads, heads // kv_heads, width).permute(0, 3, 4, 1, 2, 5)


def _scan(x, y, z, log_decay, carry):
    """out_i = sum_{j <= i} decay^(i - j) (x_i . y_j) z_j + decay^i x_i . carry for [batch, tokens, heads, width], a decay and a carry for
    every kv head; heads of y and z that meet one of x are added up. With it sum_j decay^(tokens - 1 - j) y_j z_j + decay^(tokens - 1) carry."""
    kv_heads, tokens = log_decay.numel(), x.shape[1]
    xs, ys, zs = (_chunks(t, kv_heads) for t in (x, y, z))
    batch, _, _, chunks, _, width = xs.shape
    device = x.device
    i = torch.arange(CHUNK, device=device)
    apart = i.reshape(-1, 1) - i.reshape(1, -1)
    inside = torch.where(apart >= 0, _powers(log_decay, apart.clamp(min=0)), 0.0)  # [kv_heads, CHUNK, CHUNK]
    scores = torch.matmul(xs, ys.transpose(-1, -2)) * inside.reshape(1, kv_heads, 1, 1, CHUNK, CHUNK)
    out = torch.matmul(scores, zs)
    if out.shape[2] > xs.shape[2]:
        out = out.sum(dim=2, keepdim=True)
    # What each chunk adds, seen from its last token, and what all chunks before one leave at its first.
    from_end = _powers(log_decay, CHUNK - 1 - i).reshape(1, kv_heads, 1, 1, CHUNK, 1)
    added = torch.matmul((ys * from_end).transpose(-1, -2), zs).sum(dim=2)  # [batch, kv_heads, chunks, width, width]
    c = torch.arange(chunks, device=device)
    between = (c.reshape(-1, 1) - 1 - c.reshape(1, -1)) * CHUNK
    weights = torch.where(between >= 0, _powers(log_decay, between.clamp(min=0) + 1), 0.0)
    before = torch.matmul(weights, added.reshape(batch, kv_heads, chunks, width * width)).reshape(added.shape)
    if carry is not None:
        before = before + _powers(log_decay, c * CHUNK).reshape(1, kv_heads, chunks, 1, 1) * carry.unsqueeze(2)
    from_start = _powers(log_decay, i).reshape(1, kv_heads, 1, 1, CHUNK, 1)
    out = out + torch.matmul(xs * from_start, before.unsqueeze(2))
    out = out.permute(0, 3, 4, 1, 2, 5).reshape(batch, chunks * CHUNK, -1, width)[:, :tokens]
    left = tokens - 1 - (chunks - 1) * CHUNK  # the last token's place in its chunk
    from_last = torch.where(i <= left, _powers(log_decay, (left - i).clamp(min=0)), 0.0).reshape(1, kv_heads, 1, CHUNK, 1)
    last = torch.matmul((ys[:, :, :, -1] * from_last).transpose(-1, -2), zs[:, :, :, -1]).sum(dim=2)
    last = last + _powers(log_decay, torch.tensor([left], device=device)).reshape(1, kv_heads, 1, 1) * before[:, :, -1]
    return out, last


def _decay(state):
    return torch.exp(state["log_decay"]).reshape(1, -1, 1, 1)


def _attention_forward(state):
    q, before = state["q"], state["before"]
    out, after = _scan(q, state["k"], state["v"], state["log_decay"], None if before is None else _decay(state) * before)
    out = (out * (1.0 / math.sqrt(q.shape[-1]))).to(q.dtype)
    return [out] if before is None else [out, after]


def _attention_backward(state):
    q, k, v, dout, log_decay = state["q"].float(), state["k"].float(), state["v"].float(), state["dout"].float(), state["log_decay"]
    before, dtype, scale = state["before"], state["q"].dtype, 1.0 / math.sqrt(state["q"].shape[-1])
    carry = None if before is None else (_decay(state) * before).transpose(-1, -2)
    dq, _ = _scan(dout, v, k, log_decay, carry)
    # Time runs backwards for what reaches a key and a value, and the last state's gradient is what comes before.
    qr, kr, vr, dr = (t.flip(1) for t in (q * scale, k, v, dout))
    d_after = state["d_after"]
    dv, d_first = _scan(kr, qr, dr, log_decay, d_after)
    dk, _ = _scan(vr, dr, qr, log_decay, None if d_after is None else d_after.transpose(-1, -2))
    out = [(dq * scale).to(dtype), dk.flip(1).to(dtype), dv.flip(1).to(dtype)]
    return out if before is None else [*out, _decay(state) * d_first]


def _attention_step(state):
    q, k, v = state["q"].float(), state["k"].float(), state["v"].float()
    batch, _, heads, width = q.shape
    kv_heads = k.shape[2]
    after = _decay(state) * state["before"] + k.reshape(batch, kv_heads, width, 1) * v.reshape(batch, kv_heads, 1, width)
    out = torch.matmul(q.reshape(batch, kv_heads, heads // kv_heads, width), after) * (1.0 / math.sqrt(width))
    return [out.reshape(q.shape).to(state["q"].dtype), after]


def _of_rows(state):
    """The gate of every row, or 1."""
    gate, rows = state["gate"], state["x"].shape[0]
    return 1.0 if gate is None else gate.float().repeat_interleave(rows // gate.shape[0], dim=0)


def _inverse_rms(x):
    return 1.0 / torch.sqrt((x * x).mean(dim=1, keepdim=True) + EPSILON)


def _norm_forward(state):
    x, f, dtype = state["x"].float(), state["f"].float(), state["x"].dtype
    stream = (state["case"]["scale"] * x + _of_rows(state) * (f * _inverse_rms(f) * state["u"].float())).to(dtype)
    seen = stream.float()  # the next branch's norm reads the stream as it is stored
    return [stream, (seen * _inverse_rms(seen) * state["w"].float()).to(dtype)]


def _norm_gradient(d, x, inverse, w):
    """Of an RMS norm: what reaches x from d, and the terms of the weight's gradient."""
    normed, scaled = x * inverse, d * w
    return inverse * (scaled - normed * (scaled * normed).mean(dim=1, keepdim=True)), d * normed


def _norm_backward(state):
    stream, f, u, w = (state[name].float() for name in ("x", "f", "u", "w"))
    dtype, gate = state["x"].dtype, state["gate"]
    through, dw = _norm_gradient(state["d_y"].float(), stream, _inverse_rms(stream), w)
    d_stream = state["d_stream"].float() + through
    inverse = _inverse_rms(f)
    df, du = _norm_gradient(d_stream * _of_rows(state), f, inverse, u)
    out = [(state["case"]["scale"] * d_stream).to(dtype), df.to(dtype), du.sum(dim=0).to(dtype), dw.sum(dim=0).to(dtype)]
    if gate is not None:
        of_gate = d_stream * (f * inverse * u)
        out.append(of_gate.reshape(gate.shape[0], -1, gate.shape[1]).sum(dim=1).to(dtype))
    return out


_PLAIN = {"attention_forward": _attention_forward, "attention_backward": _attention_backward, "attention_step": _attention_step,
          "norm_forward": _norm_forward, "norm_backward": _norm_backward}


# ------------------------------------------------------------------------------------------------ the library
def _own(state):
    from cgpt_amd import ops

    case, path = state["case"], state["case"]["path"]
    if path == "norm_forward":
        ops.sandwich_norm_forward(state["stream"], state["y"], state["x"], state["f"], state["u"], state["gate"], state["w"], case["scale"],
                                  EPSILON)
        return [state["stream"], state["y"]]
    if path == "norm_backward":
        ops.sandwich_norm_backward(state["dx"], state["df"], state["du"], state["d_gate"], state["dw"], state["d_stream"], state["d_y"],
                                   state["x"], state["f"], state["u"], state["gate"], state["w"], case["scale"], EPSILON)
        return [t for t in (state["dx"], state["df"], state["du"], state["dw"], state["d_gate"]) if t is not None]
    options = ops.FlashAttentionOptions(num_query_heads=case["heads"], num_kv_heads=case["kv_heads"], head_dim=case["head_dim"])
    q, k, v, log_decay, before = state["q"], state["k"], state["v"], state["log_decay"], state["before"]
    if path == "attention_step":
        ops.linear_attention_step(state["out"], state["after"], before, q, k, v, log_decay, None, options)
        return [state["out"], state["after"]]
    if path == "attention_forward":
        ops.linear_attention_forward(state["out"], state["after"], q, k, v, log_decay, before, None, options)
        return [t for t in (state["out"], state["after"]) if t is not None]
    ops.linear_attention_backward(state["dq"], state["dk"], state["dv"], state["d_before"], state["dout"], state["d_after"], q, k, v, log_decay,
                                  before, None, options)
    return [t for t in (state["dq"], state["dk"], state["dv"], state["d_before"]) if t is not None]


def run(state):
    return _own(state) if own else _PLAIN[state["case"]["path"]](state)


# ------------------------------------------------------------------------------------------------ work
def work(case):
    """Bytes: every input read once, every output written once. Flops: two for each multiply-add of the recurrence, which is the form with
    the fewest, one for each other operation."""
    size = 4 if case["dtype"] == "f32" else 2
    path = case["path"]
    if path.startswith("norm"):
        values, hidden, gates = case["rows"] * case["hidden"], case["hidden"], case["gates"] * case["hidden"]
        if path == "norm_forward":
            return {"bytes": size * (4 * values + 2 * hidden + gates), "flops": 11 * values}
        return {"bytes": size * (6 * values + 4 * hidden + 2 * gates), "flops": 27 * values}
    tokens = case["batch"] * case.get("tokens", 1)
    q_values, kv_values = tokens * case["heads"] * case["head_dim"], tokens * case["kv_heads"] * case["head_dim"]
    states = 4 * case["batch"] * case["kv_heads"] * case["head_dim"] ** 2
    flops = case["head_dim"] * (2 * q_values + 3 * kv_values)
    if path == "attention_step":
        return {"bytes": size * (2 * q_values + 2 * kv_values) + 2 * states, "flops": flops}
    if path == "attention_forward":
        return {"bytes": size * (2 * q_values + 2 * kv_values) + (2 * states if case["state"] else 0), "flops": flops}
    # the states again, their gradients, and of q, k and v
    return {"bytes": size * (3 * q_values + 4 * kv_values) + (3 * states if case["state"] else 0),
            "flops": case["head_dim"] * (4 * q_values + 10 * kv_values)}


# ------------------------------------------------------------------------------------------------ 64 bits
def _exact_recurrence(state):
    """Token by token."""
    q, k, v = (state[name].double() for name in ("q", "k", "v"))
    batch, tokens, heads, width = q.shape
    kv_heads = k.shape[2]
    decay = torch.exp(state["log_decay"].double()).reshape(1, kv_heads, 1, 1)
    memory = torch.zeros((batch, kv_heads, width, width), dtype=torch.float64, device="cuda")
    if state["before"] is not None:
        memory += state["before"].double()
    q = q.reshape(batch, tokens, kv_heads, heads // kv_heads, width) / math.sqrt(width)
    out = torch.empty_like(q)
    for t in range(tokens):
        memory.mul_(decay).add_(k[:, t].unsqueeze(-1) * v[:, t].unsqueeze(-2))
        out[:, t] = torch.matmul(q[:, t], memory)
    return out.reshape(batch, tokens, heads, width), memory


def _exact_gradients(state):
    """One sequence at a time, by differentiation of the sums over all pairs of tokens."""
    tokens, heads, width = state["q"].shape[1:]
    kv_heads = state["k"].shape[2]
    place = torch.arange(tokens, device="cuda", dtype=torch.float64)
    apart = place.reshape(-1, 1) - place.reshape(1, -1)
    results = []
    for b in range(state["q"].shape[0]):
        leaves = [state[name][b].double().requires_grad_() for name in ("q", "k", "v")]
        if state["before"] is not None:
            leaves.append(state["before"][b].double().requires_grad_())
        grads = [torch.zeros_like(leaf) for leaf in leaves]
        for h in range(heads):
            kv = h // (heads // kv_heads)
            g = state["log_decay"][kv].double()
            weights = torch.exp(g * apart).masked_fill(apart < 0, 0.0)
            q, k, v = leaves[0][:, h], leaves[1][:, kv], leaves[2][:, kv]
            out = torch.mm(torch.mm(q, k.T) * weights, v)
            if len(leaves) == 4:
                out = out + torch.exp(g * (place + 1)).reshape(-1, 1) * torch.mm(q, leaves[3][kv])
            total = (out * state["dout"][b, :, h].double()).sum() / math.sqrt(width)
            if len(leaves) == 4 and h % (heads // kv_heads) == 0:
                after = torch.mm((k * torch.exp(g * (tokens - 1 - place)).reshape(-1, 1)).T, v) + torch.exp(g * tokens) * leaves[3][kv]
                total = total + (after * state["d_after"][b, kv].double()).sum()
            for grad, part in zip(grads, torch.autograd.grad(total, leaves)):
                grad += part
        results.append(grads)
    return [torch.stack(parts) for parts in zip(*results)]


def _exact_norms(state, names):
    """The two norms from leaves in 64 bits: x, f, u, w and, where there is one, the gate."""
    leaves = [state[name].double() for name in names]
    x, f, u, w = leaves[:4]
    gate = leaves[4].repeat_interleave(x.shape[0] // leaves[4].shape[0], dim=0) if len(leaves) == 5 else torch.ones_like(x)
    return leaves, x, gate * f * torch.rsqrt(torch.mean(f * f, dim=1, keepdim=True) + EPSILON) * u, w


def exact(case, seed):
    state = prepare(case, seed)
    path = case["path"]
    if path in ("attention_forward", "attention_step"):
        out, after = _exact_recurrence(state)
        return [out] if state["before"] is None else [out, after]
    if path == "attention_backward":
        return _exact_gradients(state)
    names = ["x", "f", "u", "w"] + (["gate"] if case["gates"] else [])
    if path == "norm_forward":
        _, x, branch, w = _exact_norms(state, names)
        stream = case["scale"] * x + branch
        seen = stream.to(state["x"].dtype).double()  # the norm reads the stream as it is stored
        return [stream, seen * torch.rsqrt(torch.mean(seen * seen, dim=1, keepdim=True) + EPSILON) * w]
    # Differentiation needs the stream as a function of x, whose value is that of the stream itself: the stream given, less the branch.
    state = {name: t.double().requires_grad_() if name in names else t for name, t in state.items() if t is not None}
    leaves, given, branch, w = _exact_norms(state, names)
    stream = given + (branch - branch.detach())
    y = stream * torch.rsqrt(torch.mean(stream * stream, dim=1, keepdim=True) + EPSILON) * w
    total = (stream * state["d_stream"].double()).sum() + (y * state["d_y"].double()).sum()
    grads = list(torch.autograd.grad(total, leaves))
    grads[0] = grads[0] * case["scale"]
    return [grads[0], grads[1], grads[2], grads[3], *grads[4:]]
