"""Linear attention with a decay and the sandwich norm in 64 bits, with bounds of what the kernels may be off by.

u is half a step of the storage type, f = 2^-24 that of fp32. Every result of linear attention is one sum over pairs of tokens,
  sum_r w(t - r) (x_t . y_r) z_r + w x_t C,    A: the same of the magnitudes.
16-bit storage rounds a pair's score and the matrix C once each before their products: u A; the decayed z that C is made of keeps 2^-16 in
bfloat16 and 2^-22 in half precision; the result is rounded once: u |result|. Sums of T tokens, d products and a chunk's few are fp32:
f (T + d + 300) A. A weight g^n = 2^(n log2 g) carries the roundings of log2 g and of the product, each f |n log g| of the weight, and exp2's
own; four of them meet on the way from a pair to its result (table, matrix, since, carry): 8 f sum (1 + |n log g|) |term|. Stored matrices
keep 2^-22 of each token's product and the fp32 terms. A weight below 2^-126, the smallest normal number of fp32, may be off by that much
whatever it is: 2^-126 of the largest term for each token. In half precision a chunk's weighted z are brought to 2^14 .. 2^15 by the largest of
them, 2^-39 of which is what the others may be off by.

Half precision rounds what is below 2^-14 by 2^-25 whatever its size. Scores of a tile and the matrix of a wavefront are brought to
2^-3 .. 2^15 by their largest value: 2^-22 of it is what the others may be off by, times 64 z or d x. Results that are that small themselves: 2^-25."""
import math

import torch

FP32 = 2.0 ** -24


def half_step(dtype):
    return 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2


def product(a, b):
    return torch.matmul(a.contiguous(), b.contiguous())


def powers(log_decay, n):
    """g^n, [heads, *n.shape], zero where n < 0, and the same times 1 + |n log g|."""
    ld = torch.clamp(log_decay.double(), max=0.0, min=-1e4).view(-1, *[1] * n.dim())
    x = -ld * n.clamp(min=0)
    w = torch.where(n >= 0, torch.exp(-x), torch.zeros((), dtype=torch.float64, device=n.device))
    return w, w * (1 + x)


def heads_first(t, group=1):
    t = t.double().permute(0, 2, 1, 3)
    return t.repeat_interleave(group, dim=1) if group > 1 else t


class Sum:
    """A result, [batch, heads, tokens, width] or a matrix for each head, and its bound."""

    def __init__(self, value, error):
        self.value, self.error = value, error


def pairs_sum(x, y, z, carry, log_decay, group, scale, carry_scale, reverse, dtype, grouped):
    """All heads as query heads; carry [batch, heads, width of x, width of z], weight g^(t+1), or g^(T-1-t) in reverse. grouped: the heads of a
    group are summed in the result."""
    tokens, d = x.shape[2], x.shape[3]
    at = torch.arange(tokens, device=x.device)
    apart = at.view(1, -1) - at.view(-1, 1) if reverse else at.view(-1, 1) - at.view(1, -1)
    ld = log_decay.repeat_interleave(group)
    w, w2 = powers(ld, apart)
    c, c2 = powers(ld, tokens - 1 - at if reverse else at + 1)

    def summed(x, y, z, carry, w, c):
        r = scale * product(w * product(x, y.transpose(2, 3)), z)
        if carry is not None:
            r = r + carry_scale * c[None, ..., None] * product(x, carry)
        return r.view(x.shape[0], -1, group, tokens, d).sum(2) if grouped else r

    value = summed(x, y, z, carry, w, c)
    size = (x.abs(), y.abs(), z.abs(), None if carry is None else carry.abs())
    a, a2 = summed(*size, w, c), summed(*size, w2, c2)
    u = half_step(dtype)
    split = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -16, torch.float16: 2.0 ** -22}[dtype]
    error = (u * (1 + 2.0 ** -6) + split) * a + u * value.abs() + FP32 * ((tokens + d + 300) * a + 8 * a2 + value.abs())
    error = error + 2.0 ** -126 * tokens * group * d * (1 + scale) * x.abs().max() * (y.abs().max() * z.abs().max() + (0.0 if carry is None else carry.abs().max()))
    if dtype == torch.float16:
        scores = (scale * product(x.abs(), y.abs().transpose(2, 3))).max().item()
        matrix = product(y.abs().transpose(2, 3), z.abs()).max().item() * max(scale, 1.0) + (0.0 if carry is None else carry.abs().max().item())
        error = error + 2.0 ** -21 * (64 * scores * z.abs().max().item() + d * matrix * x.abs().max().item()) * (group if grouped else 1) + 2.0 ** -25
    return Sum(value, error)


def matrix_sum(y, z, ahead, log_decay, group, scale, reverse, dtype):
    """sum_r w y_r z_r' over tokens (and a group's heads) + g^T ahead."""
    tokens = y.shape[2]
    at = torch.arange(tokens, device=y.device)
    ld = log_decay if not reverse else log_decay.repeat_interleave(group)
    w, w2 = powers(ld, at + 1 if reverse else tokens - 1 - at)
    last, last2 = powers(log_decay, torch.full((1,), tokens, device=y.device))

    def summed(y, z, ahead, w, last):
        r = scale * product((w[None, ..., None] * y).transpose(2, 3), z)
        if reverse:
            r = r.view(r.shape[0], -1, group, *r.shape[2:]).sum(2)
        return r if ahead is None else r + last[None, ..., None] * ahead

    value = summed(y, z, ahead, w, last)
    size = (y.abs(), z.abs(), None if ahead is None else ahead.abs())
    a, a2 = summed(*size, w, last), summed(*size, w2, last2)
    split = 0.0 if dtype == torch.float32 else 2.0 ** -22
    tiny = 2.0 ** -126 * (tokens * group * (1 + scale) * y.abs().max() * z.abs().max() + (0.0 if ahead is None else ahead.abs().max()))
    return Sum(value, tiny + split * a + FP32 * ((tokens * (group if reverse else 1) + 200) * a + 8 * a2) + (2.0 ** -35 if dtype == torch.float16 else 0.0) * a.max())


def rows_of(s):
    return Sum(s.value.permute(0, 2, 1, 3), s.error.permute(0, 2, 1, 3))


def linear_forward(q, k, v, log_decay, before, scale):
    group = q.shape[2] // k.shape[2]
    scale = scale if scale > 0 else 1 / math.sqrt(q.shape[3])
    state = None if before is None else before.double()
    each = None if state is None else state.repeat_interleave(group, dim=1)
    out = pairs_sum(heads_first(q), heads_first(k, group), heads_first(v, group), each, log_decay, group, scale, scale, False, q.dtype, False)
    after = matrix_sum(heads_first(k), heads_first(v), state, log_decay, group, 1.0, False, q.dtype)
    return {"out": rows_of(out), "after": after}


def linear_backward(q, k, v, log_decay, before, dout, d_after, scale):
    group = q.shape[2] // k.shape[2]
    scale = scale if scale > 0 else 1 / math.sqrt(q.shape[3])
    qh, kh, vh, do = heads_first(q), heads_first(k, group), heads_first(v, group), heads_first(dout)

    def each(t, transposed=False):
        if t is None:
            return None
        t = t.double().repeat_interleave(group, dim=1)
        return t.transpose(2, 3) if transposed else t

    # The state's gradient reaches a kv head once, not once for each query head of its group.
    behind = None if d_after is None else d_after.double() / group
    more = (log_decay, group, scale)
    dq = pairs_sum(do, vh, kh, each(before, True), *more, scale, False, q.dtype, False)
    dv = pairs_sum(kh, qh, do, each(behind), *more, 1.0, True, q.dtype, True)
    dk = pairs_sum(vh, do, qh, each(behind, True), *more, 1.0, True, q.dtype, True)
    d_before = matrix_sum(qh, do, None if d_after is None else d_after.double(), log_decay, group, scale, True, q.dtype)
    return {"dq": rows_of(dq), "dk": rows_of(dk), "dv": rows_of(dv), "d_before": d_before}


def linear_step(q, k, v, log_decay, state, scale):
    """One token: [batch, 1, heads, d]."""
    q, k, v = (t.squeeze(1) for t in (q, k, v))
    group = q.shape[1] // k.shape[1]
    scale = scale if scale > 0 else 1 / math.sqrt(q.shape[2])
    g = torch.exp(torch.clamp(log_decay.double(), max=0.0)).view(1, -1, 1, 1)
    kept, new = g * state.double(), k.double()[..., None] * v.double()[..., None, :]
    after = kept + new
    size = kept.abs() + new.abs()
    x = q.double()[..., None, :]
    out = scale * product(x, after.repeat_interleave(group, 1)).squeeze(2)
    a = scale * product(x.abs(), size.repeat_interleave(group, 1)).squeeze(2)
    decay = FP32 * 8 * (1 + torch.clamp(log_decay.double(), min=-100, max=0).abs()).view(1, -1, 1, 1)
    after_error = (decay + 4 * FP32) * size
    d = q.shape[2]
    lost = scale * product(x.abs(), after_error.repeat_interleave(group, 1)).squeeze(2)
    tiny = 2.0 ** -25 if q.dtype == torch.float16 else 0.0
    error = half_step(q.dtype) * out.abs() + FP32 * (d + 10) * a + lost + tiny
    return {"out": Sum(out[:, None], error[:, None]), "after": Sum(after, after_error)}


# ------------------------------------------------------------------------------------------------ sandwich norm
# Sums over a row are at most hidden / 64 + 8 elements a lane and a tree: n f of their magnitudes with n = hidden/64 + 32. The stream that
# is stored is rounded once and the second norm is of what is stored.
def expand_gate(gate, rows):
    return 1.0 if gate is None else gate.double().repeat_interleave(rows // gate.shape[0], 0)


def stored(value, error, dtype):
    return Sum(value, error + max(half_step(dtype), FP32) * (value.abs() + error) + (2.0 ** -25 if dtype == torch.float16 else 0.0))


def sandwich_forward(x, f, u, gate, w, scale, eps, stream):
    """stream: the kernel's, which the second norm is of."""
    rows, hidden = x.shape
    n = hidden / 64 + 32
    g = expand_gate(gate, rows)
    rf = 1 / torch.sqrt((f.double() ** 2).mean(1, keepdim=True) + eps)
    branch = g * f.double() * rf * u.double()
    xs = scale * x.double() + branch
    s = stream.double()
    y = s / torch.sqrt((s ** 2).mean(1, keepdim=True) + eps) * w.double()
    return {"stream": stored(xs, FP32 * ((n + 10) * branch.abs() + 4 * (scale * x.double()).abs()), x.dtype), "y": stored(y, FP32 * (n + 10) * y.abs(), x.dtype)}


def sandwich_backward(stream, f, u, gate, w, scale, eps, d_stream, dy):
    rows, hidden = stream.shape
    n = hidden / 64 + 32
    g = expand_gate(gate, rows)
    s, f, u, w, dy = (t.double() for t in (stream, f, u, w, dy))
    past = torch.zeros_like(s) if d_stream is None else d_stream.double()
    rs, rf = (1 / torch.sqrt((t ** 2).mean(1, keepdim=True) + eps) for t in (s, f))

    def all_of(sign, past, dy, w, s, f, g, u):
        grad = past + rs * (dy * w + sign * s * rs ** 2 * (dy * w * s).mean(1, keepdim=True))
        h = g * u * grad
        df = rf * (h + sign * f * rf ** 2 * (h * f).mean(1, keepdim=True))
        by_row = grad * f * rf
        dw, du = (dy * s * rs).sum(0), (g * by_row).sum(0)
        dgate = None if gate is None else u * by_row.view(gate.shape[0], -1, hidden).sum(1)
        return {"dx": scale * grad, "df": df, "dw": dw, "du": du, "d_gate": dgate}

    value = all_of(-1.0, past, dy, w, s, f, g, u)
    a = all_of(1.0, past.abs(), dy.abs(), w.abs(), s.abs(), f.abs(), abs(g), u.abs())
    factor = {"dx": 2 * n + 20, "df": 4 * n + 60, "dw": rows + n + 20, "du": rows + 3 * n + 60, "d_gate": rows + 3 * n + 60}
    return {name: stored(v, FP32 * factor[name] * a[name].abs(), stream.dtype) for name, v in value.items() if v is not None}


def check(got, want, name):
    """Every element within its bound. A result beyond the storage type's largest number has no value in it (half precision: 65504) and is stored as
    an infinity, which stands for that number here."""
    largest = torch.finfo(got.dtype).max
    assert bool((torch.isfinite(got) | (got.isinf() & (want.value.abs() + want.error >= largest))).all()), f"{name}: not finite"
    error = (got.double().clamp(-largest, largest) - want.value.clamp(-largest, largest)).abs()
    worst = (error / want.error.clamp(min=1e-300)).max().item() if error.numel() else 0.0
    assert bool((error <= want.error).all()), f"{name}: {worst:.3g} times its bound"
