"""Attention and its gradient from the definition, in 64 bits on the CPU, with bounds of what the kernels may be off.

The bounds are arithmetic.  With ``u`` half a step of the operands' type (relative), ``e = 2^-24`` that of fp32:

* a score of K products is off by at most ``(K + 4) e sum |q k|`` times the scale, the argument of its exponential by as much plus
  its own rounding, so a weight is off by the relative ``E = 2 (K + 4) e S + 16 e``, S the largest scale sum |q k| of the row;
* sums of N weights or products in fp32 add at most ``(N + 16) e`` of the sum of magnitudes;
* weights are rounded to the operands' type in front of the product with the values: ``u`` each (fp16: at least 2^-25, half a step of its
  smallest numbers, below the row's largest weight, which is at least 1 before the division).
"""
import math

import torch

UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
FLOOR = {torch.float32: 0.0, torch.float16: 2.0 ** -25, torch.bfloat16: 0.0}       # of a rounded number, absolute
E32 = 2.0 ** -24


def keep_of(L, M, N, key_lengths=None, key_mask=None, causal=False):
    """[L, M, N]: the keys that each query meets."""
    keep = torch.ones(L, M, N, dtype=torch.bool)
    if key_lengths is not None:
        lengths = key_lengths.cpu().long().clamp(0, N)
        keep &= (torch.arange(N)[None] < lengths[:, None])[:, None]
        if causal:
            position = lengths[:, None] - M + torch.arange(M)
            keep &= torch.arange(N)[None, None] <= position[..., None]
    if key_mask is not None:
        keep &= key_mask.cpu().expand(L, N)[:, None]
    return keep


def forward(q, k, v, keep, scale):
    """(out, lse, bound of out, bound of lse) of q [L, M, H, K], k [L, N, G, K], v [L, N, G, O], keep [L, M, N]."""
    unit, floor = UNIT[q.dtype], FLOOR[q.dtype]
    L, M, H, K = q.shape
    N, G, O = v.shape[1:]
    q, k, v = (x.detach().cpu().double() for x in (q, k, v))
    used = keep.any(1)                                              # what no query of an entry meets may hold anything
    k = torch.where(used[..., None, None], k.expand(L, N, G, K), torch.zeros(()).double()).repeat_interleave(H // G, 2)
    v = torch.where(used[..., None, None], v.expand(L, N, G, O), torch.zeros(()).double()).repeat_interleave(H // G, 2)
    q, k, v = (x.transpose(1, 2).contiguous() for x in (q, k, v))                       # [L, H, tokens, features]
    s = torch.matmul(q, k.transpose(2, 3)) * scale
    magnitude = torch.matmul(q.abs(), k.abs().transpose(2, 3)) * abs(scale)
    s = s.masked_fill(~keep[:, None], -math.inf)
    top = s.amax(-1, keepdim=True) if N else torch.full((L, H, M, 1), -math.inf).double()
    weights = torch.exp(s - top.clamp_min(-1e300))
    total = weights.sum(-1, keepdim=True)
    p = weights / total.clamp_min(1e-300)
    out = torch.matmul(p, v)
    lse = (torch.log(total) + top.clamp_min(-1e300)).masked_fill(total == 0, -math.inf)[..., 0]
    S = magnitude.amax(-1, keepdim=True) if N else torch.zeros(L, H, M, 1).double()
    E = 2 * (K + 4) * E32 * S + 16 * E32
    sums = (N + 16) * E32
    A = torch.matmul(p, v.abs())
    bound = unit * 1.01 * (out.abs() + A) + 2 * (E + sums) * A + floor * (v.abs().sum(2, keepdim=True) + 1)
    lse_bound = (E + sums)[..., 0] + 4 * E32 * lse.abs().nan_to_num(posinf=0.0)
    return out.transpose(1, 2), lse.transpose(1, 2), bound.transpose(1, 2), lse_bound.transpose(1, 2)


def gradients(grad_out, q, k, v, keep, scale):
    """(grad_q, grad_k, grad_v) and their bounds.  On top of the forward's errors: lse is off by its bound, the result that delta is
    made of by its own, ds is rounded to the operands' type in front of the two products with keys and queries, p in front of the one with d."""
    unit, floor = UNIT[q.dtype], FLOOR[q.dtype]
    L, M, H, K = q.shape
    N, G, O = v.shape[1:]
    R, shared = H // G, k.shape[0] == 1 and L > 1
    out, lse, out_bound, lse_bound = forward(q, k, v, keep, scale)
    q, k, v, d = (x.detach().cpu().double() for x in (q, k, v, grad_out))
    used = keep.any(1)[..., None, None]
    k, v = (torch.where(used, x.expand(L, *x.shape[1:]), torch.zeros(()).double()).repeat_interleave(R, 2) for x in (k, v))
    q, k, v, d, out, out_bound = (x.transpose(1, 2).contiguous() for x in (q, k, v, d, out, out_bound))
    lse, lse_bound = lse.transpose(1, 2)[..., None], lse_bound.transpose(1, 2)[..., None]
    s = torch.matmul(q, k.transpose(2, 3)) * scale
    S = torch.matmul(q.abs(), k.abs().transpose(2, 3)) * abs(scale)
    p = torch.exp(s - lse).masked_fill(~keep[:, None], 0.0)
    p_error = p * 2 * (2 * (K + 4) * E32 * S + 16 * E32 + lse_bound + 4 * E32 * lse.abs().nan_to_num(posinf=0.0))
    dp = torch.matmul(d, v.transpose(2, 3))
    dp_magnitude = torch.matmul(d.abs(), v.abs().transpose(2, 3))
    delta = (d * out).sum(-1, keepdim=True)
    delta_error = (d.abs() * out_bound).sum(-1, keepdim=True) + (O + 16) * E32 * (d.abs() * out.abs()).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    ds_error = p_error * (dp - delta).abs() + p * ((O + 16) * E32 * dp_magnitude + delta_error)
    ds_error = ds_error + unit * 1.01 * (ds.abs() + ds_error) + floor * keep[:, None]
    p_rounded_error = p_error + unit * 1.01 * p + floor * keep[:, None]

    def result(value, bound):
        return value, bound + unit * 1.01 * (value.abs() + bound) + floor

    def over_rows(x):
        """[L, H, N, D] -> [L or 1, N, G, D]: the sum over heads and entries that share the keys"""
        x = x.reshape(L, G, R, N, -1).sum(2).transpose(1, 2)
        return x.sum(0, keepdim=True) if shared else x

    rows = M * R * (L if shared else 1) + 16
    grad_q = (scale * torch.matmul(ds, k)).transpose(1, 2)
    grad_q_bound = (abs(scale) * (torch.matmul(ds_error, k.abs()) + (N + 16) * E32 * torch.matmul(ds.abs(), k.abs()))).transpose(1, 2)
    grad_k = over_rows(scale * torch.matmul(ds.transpose(2, 3), q))
    grad_k_bound = over_rows(abs(scale) * (torch.matmul(ds_error.transpose(2, 3), q.abs()) + rows * E32 * torch.matmul(ds.abs().transpose(2, 3), q.abs())))
    grad_v = over_rows(torch.matmul(p.transpose(2, 3), d))
    grad_v_bound = over_rows(torch.matmul(p_rounded_error.transpose(2, 3), d.abs()) + rows * E32 * torch.matmul(p.transpose(2, 3), d.abs()))
    results = [result(*x) for x in ((grad_q, grad_q_bound), (grad_k, grad_k_bound), (grad_v, grad_v_bound))]
    return [value for value, _ in results], [bound for _, bound in results]


def prefix(q, pk, pv, k, v, lengths, scale):
    """(out, bound) of prefix_attention: the prefix and the own keys of an entry as one sequence of keys."""
    L, M = q.shape[:2]
    P, N = pk.shape[0], k.shape[1]
    keep = torch.cat((torch.ones(L, M, P, dtype=torch.bool), keep_of(L, M, N, lengths, causal=True)), 2)
    own = torch.arange(N)[None] < lengths.cpu().long().clamp(0, N)[:, None]
    zero = torch.zeros((), dtype=q.dtype)
    k, v = (torch.where(own[..., None, None], x.cpu(), zero) for x in (k, v))
    joined = [torch.cat((x.cpu()[None].expand(L, *x.shape), y), 1) for x, y in ((pk, k), (pv, v))]
    out, _, bound, _ = forward(q.cpu(), *joined, keep, scale)
    # parts of the keys are joined in fp32: a rounding of every part and of its weight
    return out, bound + 64 * E32 * out.abs() + 64 * E32 * bound


def assert_within(got, truth, bound, what):
    got = got.detach().cpu().double()
    assert got.shape == truth.shape, f"{what}: shape {tuple(got.shape)} instead of {tuple(truth.shape)}"
    infinite = torch.isinf(truth)
    assert torch.equal(got[infinite], truth[infinite]), f"{what}: infinities differ"
    error = (got - truth).abs()
    error[infinite] = 0.0
    worst = (error - bound).nan_to_num(nan=math.inf, posinf=math.inf, neginf=-math.inf)
    if worst.numel() and worst.max() > 0:
        at = worst.flatten().argmax()
        raise AssertionError(f"{what}: {int((worst > 0).sum())} of {worst.numel()} values out of bounds, the worst {got.flatten()[at]:.9g} "
                             f"instead of {truth.flatten()[at]:.9g} (bound {bound.expand_as(truth).flatten()[at]:.3g}), index {int(at)}")
