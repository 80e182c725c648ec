"""Bounds of linear attention in half precision that follow the decays, head by head and chunk by chunk of 64 tokens. linear_oracle.py bounds scores and
matrices by the largest there are, undecayed, which is loose over long sequences and strong decays.

What half precision leaves of an operand, beside its half step u that linear_oracle.py counts: a tile's scores and a wavefront's part of the matrix C are
brought to 2^-3 or more by their largest, so 2^-25 absolute is 2^-22 of that,
  2^-22 max|P| sum |z_r| over the chunk's tokens that are seen,  2^-22 max|C| sum |x_t| since;
the weighted z are brought to 2^14 or more by the chunk's largest z times its largest weight, in two parts, by at most 2^30 and by no more than leaves
2^110 (of a matrix at 2^14) for the matrix they are added to: 2^-39 of that largest, 2^-55, or 2^-149 of the matrix's largest, times sum |y_r|, decaying
with the matrix. Matrices that are stored: 2^-39 of the chunk's largest weighted z, or 2^-145 of what the matrix cannot exceed (2^22 times the sum of
those largest), times sum |y_r|, decaying. All of it twice rounded: times 1 + 2^-6.

A matrix instruction aligns products by their operands' exponents, which of a number below 2^-14, half precision's smallest normal one, is that one's: to the
fp32 terms such operands count as 2^-14."""
import math

import torch

from tests import linear_oracle
from tests.linear_oracle import Sum, half_step, heads_first, matrix_sum, pairs_sum, product, rows_of

CHUNK = 64


def decays(log_decay, n):
    return torch.exp(torch.clamp(log_decay.double(), max=0.0, min=-1e4).view(-1, 1) * n.double())


def magnitude(t):
    return None if t is None else torch.where(t != 0, t.abs().clamp(min=2.0 ** -14), t.abs())


def half_slack(x, y, z, carry, log_decay, scale, reverse):
    """[batch, query heads, tokens, width of z]; magnitudes in, log_decay of every query head."""
    tokens, device = x.shape[2], x.device
    one = torch.ones(1, device=device)
    g = decays(log_decay, one).view(1, -1, 1)
    out_scale, matrix_scale = (1.0, scale) if reverse else (scale, 1.0)
    matrix = torch.zeros((*x.shape[:2], y.shape[3], z.shape[3]), dtype=torch.float64, device=device)
    if carry is not None:
        matrix = matrix + carry * (1.0 if reverse else g[..., None])
    lost = torch.zeros(matrix.shape[:3], dtype=torch.float64, device=device)
    slack = torch.zeros((*x.shape[:3], z.shape[3]), dtype=torch.float64, device=device)
    starts = range(0, tokens, CHUNK)
    for first in reversed(starts) if reverse else starts:
        rows = slice(first, min(first + CHUNK, tokens))
        xs, ys, zs = x[:, :, rows], y[:, :, rows], z[:, :, rows]
        n = xs.shape[2]
        at = torch.arange(n, device=device)
        since = decays(log_decay, n - 1 - at if reverse else at)[None]
        largest = matrix.amax((2, 3))[..., None]
        of_matrix = out_scale * since * (2.0 ** -22 * largest * xs.sum(-1) + (xs * lost[:, :, None]).sum(-1))
        apart = at.view(1, -1) - at.view(-1, 1) if reverse else at.view(-1, 1) - at.view(1, -1)
        seen = (apart >= 0).double()
        w = seen * decays(log_decay, apart.clamp(min=0).reshape(-1)).view(-1, n, n)
        scores = (scale * w * product(xs, ys.transpose(2, 3))).amax((2, 3))[..., None, None]
        slack[:, :, rows] = 2.0 ** -22 * scores * product(seen.expand(*xs.shape[:2], n, n), zs) + of_matrix[..., None]
        weights = matrix_scale * decays(log_decay, at + 1 if reverse else CHUNK - at)[None, ..., None]
        passed = decays(log_decay, one * n).view(1, -1, 1)
        left = 2.0 ** -39 * zs.amax((2, 3))[..., None] * (matrix_scale * g if reverse else 1.0) + 2.0 ** -55 + 2.0 ** -148 * largest
        lost = passed * lost + left * ys.sum(2)
        matrix = passed[..., None] * matrix + product(ys.transpose(2, 3), weights * zs)
    return slack * (1 + 2.0 ** -6)


def half_sum(x, y, z, carry, log_decay, group, scale, carry_scale, reverse, grouped):
    more = (log_decay, group, scale, carry_scale, reverse, torch.float32, grouped)
    size = (x.abs(), y.abs(), z.abs(), None if carry is None else carry.abs())
    value, a, u = pairs_sum(x, y, z, carry, *more).value, pairs_sum(*size, *more).value, half_step(torch.float16)
    error = pairs_sum(*(magnitude(t) for t in (x, y, z)), size[3], *more).error
    slack = half_slack(*size, log_decay.repeat_interleave(group), scale, reverse)
    if grouped:
        slack = slack.view(x.shape[0], -1, group, *slack.shape[2:]).sum(2)
    return Sum(value, error + (u * (1 + 2.0 ** -6) + 2.0 ** -22) * a + u * value.abs() + 2.0 ** -25 + slack)


def half_matrix(y, z, ahead, log_decay, group, scale, reverse):
    """A stored matrix, of tokens and a group's heads; the bound is linear_oracle.matrix_sum's with these terms for its last one."""
    tokens, device, more = y.shape[2], y.device, (log_decay, group, scale, reverse)
    size = (y.abs(), z.abs(), None if ahead is None else ahead.abs())
    value, a = (matrix_sum(*t, *more, torch.float32).value for t in ((y, z, ahead), size))
    error = matrix_sum(magnitude(y), magnitude(z), size[2], *more, torch.float32).error
    each = log_decay.repeat_interleave(group) if reverse else log_decay
    lost = torch.zeros(y.shape[:2] + y.shape[3:], dtype=torch.float64, device=device)
    room = torch.zeros((*y.shape[:2], 1), dtype=torch.float64, device=device)
    starts = range(0, tokens, CHUNK)
    for first in reversed(starts) if reverse else starts:
        rows = slice(first, min(first + CHUNK, tokens))
        ys, zs = size[0][:, :, rows], size[1][:, :, rows]
        n = ys.shape[2]
        at = torch.arange(n, device=device)
        end = n - 1 if not reverse and rows.stop == tokens else n  # what is stored is the matrix as the last token sees it
        w = (scale if reverse else 1.0) * decays(each, at + 1 if reverse else end - at)
        largest = (w[None, ..., None] * zs).amax((2, 3))[..., None]
        passed = decays(each, torch.full((1,), end, device=device)).view(1, -1, 1)
        room = passed * room
        if reverse:  # of the heads before, which are added to the same matrix
            room = room.view(room.shape[0], -1, group, 1).sum(2).repeat_interleave(group, 1)
        lost = passed * lost + (2.0 ** -39 * largest + 2.0 ** -145 * room) * ys.sum(2)
        room = room / (group if reverse else 1) + 2.0 ** 22 * largest
    if reverse:
        lost = lost.view(lost.shape[0], -1, group, lost.shape[2]).sum(2)
    return Sum(value, error + 2.0 ** -22 * a + (1 + 2.0 ** -6) * lost[..., None])


def linear_forward(q, k, v, log_decay, before, scale):
    want = linear_oracle.linear_forward(q, k, v, log_decay, before, scale)
    if q.dtype == torch.float16:
        group = q.shape[2] // k.shape[2]
        scale = scale if scale > 0 else 1 / math.sqrt(q.shape[3])
        state = None if before is None else before.double()
        each = None if before is None else state.repeat_interleave(group, dim=1)
        want["out"] = rows_of(half_sum(heads_first(q), heads_first(k, group), heads_first(v, group), each, log_decay, group, scale, scale, False, False))
        want["after"] = half_matrix(heads_first(k), heads_first(v), state, log_decay, group, 1.0, False)
    return want


def linear_backward(q, k, v, log_decay, before, dout, d_after, scale):
    want = linear_oracle.linear_backward(q, k, v, log_decay, before, dout, d_after, scale)
    if q.dtype != torch.float16:
        return want
    group = q.shape[2] // k.shape[2]
    scale = scale if scale > 0 else 1 / math.sqrt(q.shape[3])
    qh, kh, vh, do = heads_first(q), heads_first(k, group), heads_first(v, group), heads_first(dout)

    def each(t, parts=1, transposed=False):
        if t is None:
            return None
        t = t.double().repeat_interleave(group, dim=1) / parts
        return t.transpose(2, 3) if transposed else t

    more = (log_decay, group, scale)
    want["dq"] = rows_of(half_sum(do, vh, kh, each(before, transposed=True), *more, scale, False, False))
    want["dv"] = rows_of(half_sum(kh, qh, do, each(d_after, group), *more, 1.0, True, True))
    want["dk"] = rows_of(half_sum(vh, do, qh, each(d_after, group, True), *more, 1.0, True, True))
    want["d_before"] = half_matrix(qh, do, None if d_after is None else d_after.double(), *more, True)
    return want
