"""Attention: the product of a kernel matrix with coefficients whose rows are divided by their sums.

``run_kernel(..., coefficients=...)`` contracts a kernel matrix with coefficients; here the kernel is
``exp(scale <query, key>)``, every row of it is normalised, and the values are the coefficients.  The matrix never
reaches memory.  None of it has a counterpart in the reference.

``cross_attention``       queries against the keys and values of another sequence
``cross_attention_grad``  its gradient
``prefix_attention``      a batch of sequences that all continue one long prefix, which is walked once for all of them

Tensors are ``[L?, tokens, heads, features]`` with the last dimension contiguous and any strides in front of it, in fp32, fp16 or
bf16; sums, maxima and exponentials are fp32.  The operators are functions of tensors, not recorded by autograd: a training
step calls ``cross_attention_grad`` with the result and the row sums that ``cross_attention`` returned.
"""
from __future__ import annotations

import math
from typing import Optional

import torch

from . import _backend
from . import _scratch
from .build_a_kernel import _current_stream_for

_TYPES = {torch.float32: _backend.FP32, torch.float16: _backend.FP16, torch.bfloat16: _backend.BF16}
_MAX_WIDTH = 256


def _check_tensors(named, device, dtype, require_device):
    for name, x in named:
        if not isinstance(x, torch.Tensor):
            raise TypeError(f"{name} must be a PyTorch tensor")
        if x.dtype is not dtype:
            raise TypeError(f"{name} must have dtype {dtype}, got {x.dtype}")
        if require_device and not x.is_cuda:
            raise ValueError(f"{name} must be on a CUDA device")
        if x.device != device:
            raise ValueError(f"{name} must be on the same CUDA device as inputs: got {x.device}, expected {device}")


def _layout(name, x):
    """(batch entries, tokens, heads, features, strides of the first three) of a [tokens, heads, features] tensor or a batch of them."""
    shape, strides = x.shape, x.stride()
    if len(shape) == 4:
        (L, tokens, heads, width), (ls, ts, hs, ws) = shape, strides
        if L == 1:
            ls = 0
    elif len(shape) == 3:
        (tokens, heads, width), (ts, hs, ws) = shape, strides
        L, ls = 1, 0
    else:
        raise ValueError(f"{name} must be 3-dimensional or 4-dimensional with a batch mode")
    if ws != 1 and width > 1:
        raise ValueError(f"{name} must have stride 1 in last dimension")
    if not 1 <= width <= _MAX_WIDTH:
        raise ValueError(f"the last dimension of {name} must be 1 .. {_MAX_WIDTH}, got {width}")
    return L, tokens, heads, width, ls, ts, hs


def _result(name, out, shape, like, require_device):
    """`out`, checked, or a new tensor of `shape`."""
    if out is None:
        return torch.empty(shape, dtype=like.dtype, device=like.device)
    _check_tensors(((name, out),), like.device, like.dtype, require_device)
    if tuple(out.shape) != tuple(shape) and not (out.dim() == 3 and shape[0] == 1 and tuple(out.shape) == tuple(shape[1:])):
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(out.shape)}")
    if any(stride == 0 and extent > 1 for extent, stride in zip(out.shape, out.stride())):
        raise ValueError(f"{name} must not be an expanded tensor")
    return out


def _scale(scale, width):
    scale = width ** -0.5 if scale is None else float(scale)
    if not math.isfinite(scale):
        raise ValueError(f"scale must be finite, got {scale}")
    return scale


def _lengths(name, lengths, L, device, require_device):
    _check_tensors(((name, lengths),), device, torch.int32, require_device)
    if tuple(lengths.shape) != (L,) or (L > 1 and lengths.stride(0) != 1):
        raise ValueError(f"{name} must be contiguous with shape (L={L},), got {tuple(lengths.shape)}")
    return lengths.data_ptr()


def _check_types(x):
    if not isinstance(x, torch.Tensor):
        raise TypeError("queries must be a PyTorch tensor")
    if x.dtype not in _TYPES:
        raise TypeError(f"queries must have dtype torch.float32, torch.float16 or torch.bfloat16, got {x.dtype}")


class _AttentionPlan:
    __slots__ = ("params", "out", "lse", "keepalive")


def _plan_attention(queries, keys, values, out, scale, key_lengths, key_mask, return_lse, prefix=None, require_device=True) -> _AttentionPlan:
    """Validation and parameter marshalling, without the launch.  `prefix`: the prefix's keys and values; the queries are then
    the last tokens of `key_lengths`."""
    _check_types(queries)
    device, dtype = queries.device, queries.dtype
    inputs = [("queries", queries), ("keys", keys), ("values", values)]
    if prefix is not None:
        inputs += [("prefix_keys", prefix[0]), ("prefix_values", prefix[1])]
    _check_tensors(inputs, device, dtype, require_device)
    L, M, H, K, q_ls, q_ms, q_hs = _layout("queries", queries)
    L_k, N, G, K_k, k_ls, k_ns, k_gs = _layout("keys", keys)
    L_v, N_v, G_v, O, v_ls, v_ns, v_gs = _layout("values", values)
    if L_k != L_v or (L_k != L and (L_k != 1 or prefix is not None)):
        raise ValueError(f"keys and values must both have the batch size of queries (L={L})"
                         + (" or both 1" if prefix is None else "") + f", got {L_k} and {L_v}")
    if K_k != K:
        raise ValueError(f"keys must have as many features as queries (K={K}), got {K_k}")
    if (N_v, G_v) != (N, G):
        raise ValueError(f"values must have as many tokens and heads as keys (N={N}, G={G}), got {N_v} and {G_v}")
    if G == 0 and H > 0 or G > 0 and H % G != 0:
        raise ValueError(f"the heads of queries (H={H}) must be a multiple of the heads of keys (G={G})")
    scale = _scale(scale, K)

    params = _backend.AttentionParams(_TYPES[dtype], 0, L, M, N, H, G, K, O, scale, queries.data_ptr(), q_ls, q_ms, q_hs,
                                      keys.data_ptr(), k_ls, k_ns, k_gs, values.data_ptr(), v_ls, v_ns, v_gs)
    plan = _AttentionPlan()
    plan.keepalive = [queries, keys, values, key_lengths, key_mask, prefix]
    if key_lengths is not None:
        params.key_lengths = _lengths("lengths" if prefix is not None else "key_lengths", key_lengths, L, device, require_device)
    if key_mask is not None:
        _check_tensors((("key_mask", key_mask),), device, torch.bool, require_device)
        if tuple(key_mask.shape) not in ((N,), (1, N), (L, N)):
            raise ValueError(f"key_mask must have shape (N={N},) or (L={L}, N={N}), got {tuple(key_mask.shape)}")
        batched = key_mask.dim() == 2 and key_mask.size(0) > 1
        params.key_mask, params.key_mask_ls, params.key_mask_ns = key_mask.data_ptr(), key_mask.stride(0) if batched else 0, key_mask.stride(-1)
    if prefix is not None:
        prefix_k, prefix_v = prefix
        if prefix_k.dim() != 3 or prefix_v.dim() != 3:
            raise ValueError("prefix_keys and prefix_values must be 3-dimensional: they have no batch mode")
        _, P, G_p, K_p, _, pk_ns, pk_gs = _layout("prefix_keys", prefix_k)
        _, P_v, G_pv, O_p, _, pv_ns, pv_gs = _layout("prefix_values", prefix_v)
        if (G_p, K_p) != (G, K):
            raise ValueError(f"prefix_keys must have the heads and features of keys (G={G}, K={K}), got {G_p} and {K_p}")
        if (P_v, G_pv, O_p) != (P, G, O):
            raise ValueError(f"prefix_values must have the tokens of prefix_keys and the heads and features of values (P={P}, G={G}, O={O}), "
                             f"got {P_v}, {G_pv} and {O_p}")
        params.prefix_n, params.causal = P, 1
        params.prefix_key, params.prefix_key_ns, params.prefix_key_gs = prefix_k.data_ptr(), pk_ns, pk_gs
        params.prefix_value, params.prefix_value_ns, params.prefix_value_gs = prefix_v.data_ptr(), pv_ns, pv_gs

    plan.out = out = _result("out", out, (L, M, H, O), queries, require_device)
    strides = out.stride()
    if strides[-1] != 1 and O > 1:
        raise ValueError("out must have stride 1 in last dimension")
    params.out, params.out_ls, params.out_ms, params.out_hs = out.data_ptr(), strides[0] if len(strides) == 4 else 0, strides[-3], strides[-2]
    plan.lse = None
    if return_lse:
        plan.lse = torch.empty((L, M, H), dtype=torch.float32, device=device)
        params.lse = plan.lse.data_ptr()
    plan.params = params
    return plan


def _launch(plan, device, debug):
    stream = _current_stream_for(device)
    params = plan.params
    needed = _backend.attention_workspace_bytes(params)
    workspace = _scratch.allocate(needed, device) if needed else None
    if workspace is not None:           # refused: one pass over the keys per tile of rows
        params.workspace, params.workspace_bytes = workspace.data_ptr(), needed
    if debug:
        print(f"(Kermac Debug) Launching kernel: attention_forward{' and attention_join' if workspace is not None else ''}")
    _backend.attention(params, stream)
    # the launches are queued: the allocator hands the workspace on in stream order


@_scratch.operator
def cross_attention(
    queries: torch.Tensor,                  # [L?, M, H, K]
    keys: torch.Tensor,                     # [L?, N, G, K]
    values: torch.Tensor,                   # [L?, N, G, O]
    out: Optional[torch.Tensor] = None,     # [L?, M, H, O]
    *,
    scale: Optional[float] = None,
    key_lengths: Optional[torch.Tensor] = None,
    key_mask: Optional[torch.Tensor] = None,
    return_lse: bool = False,
    debug=False,
):
    """Attention of queries to the keys and values of a sequence of another length::

        out[l, m, h, o] = sum_n softmax_n(scale * sum_k queries[l, m, h, k] * keys[l, n, g, k]) * values[l, n, g, o]

    with ``g = h // (H // G)``: ``H`` is a multiple of ``G``, consecutive heads of queries share a head of keys and values.
    All of them have one dtype (fp32, fp16 or bf16), ``K`` and ``O`` up to 256, and the last dimension contiguous; keys and
    values of batch size 1 serve all entries of the batch.

    Args:
        scale: ``K ** -0.5`` when None; any finite number.
        key_lengths: int32 ``[L]``: the first so many keys of an entry take part (taken as 0 .. N where outside).
        key_mask: bool ``[N]`` or ``[L, N]``: the keys that take part.  With both, a key has to pass both.
        out: optional result, ``[L, M, H, O]``, written in place and returned; it must not share memory with the inputs.
        return_lse: also return ``log sum exp`` of every row, fp32 ``[L, M, H]``, for ``cross_attention_grad``.

    What keys and values hold where they do not take part does not matter, infinities and NaN included.  A row
    without a key (or with scores of -inf alone) gets zeros, and -inf for its ``lse``.  Returns ``out`` (allocated
    ``[L, M, H, O]`` when None), or ``(out, lse)``.

    Raises:
        TypeError: non-tensor inputs or a wrong dtype.
        ValueError: bad shapes, strides, batch sizes or devices, a scale that is not finite.
    """
    plan = _plan_attention(queries, keys, values, out, scale, key_lengths, key_mask, return_lse)
    _launch(plan, queries.device, debug)
    return (plan.out, plan.lse) if return_lse else plan.out


def _plan_attention_grad(grad_out, queries, keys, values, out, lse, scale, key_lengths, key_mask, require_device=True):
    """The checks of the forward call, whose result `out` and `lse` are, and the gradient's parameters."""
    forward = _plan_attention(queries, keys, values, out, scale, key_lengths, key_mask, False, require_device=require_device)
    of = forward.params
    device = queries.device
    shape = (of.l, of.m, of.h, of.o)
    _check_tensors((("grad_out", grad_out),), device, queries.dtype, require_device)
    if tuple(grad_out.shape) != shape and not (grad_out.dim() == 3 and of.l == 1 and tuple(grad_out.shape) == shape[1:]):
        raise ValueError(f"grad_out must have shape {shape}, got {tuple(grad_out.shape)}")
    _, _, _, _, d_ls, d_ms, d_hs = _layout("grad_out", grad_out)
    _check_tensors((("lse", lse),), device, torch.float32, require_device)
    if tuple(lse.shape) != shape[:3] or not lse.is_contiguous():
        raise ValueError(f"lse must be contiguous with shape {shape[:3]}, got {tuple(lse.shape)}")
    make = torch.zeros if queries.numel() == 0 else torch.empty         # no query: nothing is launched
    key_entries = keys.size(0) if keys.dim() == 4 else 1
    grads = (torch.empty(queries.shape, dtype=queries.dtype, device=device), make(keys.shape, dtype=keys.dtype, device=device),
             make(values.shape, dtype=values.dtype, device=device))
    params = _backend.AttentionGradientParams(
        of.type, 0, of.l, of.m, of.n, of.h, of.g, of.k, of.o, key_entries, of.scale, of.q, of.q_ls, of.q_ms, of.q_hs, of.key, of.key_ls, of.key_ns, of.key_gs,
        of.value, of.value_ls, of.value_ns, of.value_gs, of.out, of.out_ls, of.out_ms, of.out_hs, grad_out.data_ptr(), d_ls, d_ms, d_hs, lse.data_ptr(),
        of.key_lengths, of.key_mask, of.key_mask_ls, of.key_mask_ns, grads[0].data_ptr(), grads[1].data_ptr(), grads[2].data_ptr())
    plan = _AttentionPlan()
    plan.params, plan.out, plan.lse = params, grads, None
    plan.keepalive = [forward, grad_out, lse]
    return plan


@_scratch.operator
def cross_attention_grad(
    grad_out: torch.Tensor,                 # [L?, M, H, O]
    queries: torch.Tensor,                  # [L?, M, H, K]
    keys: torch.Tensor,                     # [L?, N, G, K]
    values: torch.Tensor,                   # [L?, N, G, O]
    out: torch.Tensor,                      # [L?, M, H, O]
    lse: torch.Tensor,                      # [L, M, H]
    *,
    scale: Optional[float] = None,
    key_lengths: Optional[torch.Tensor] = None,
    key_mask: Optional[torch.Tensor] = None,
    debug=False,
):
    """Gradients of ``cross_attention`` with respect to queries, keys and values, given the gradient of its result.

    ``out`` and ``lse`` are what ``cross_attention(..., return_lse=True)`` returned for the same tensors, scale, lengths and
    mask.  The gradient of a head of keys and values is the sum over the heads of queries that share it; that of keys and
    values of batch size 1 is the sum over the batch.  Keys that do not take part have a gradient of zero, and so has a query without
    keys.  Sums are fp32 in an order that does not depend on timing; in fp16 the products of weights and gradients are
    numbers of that type, so gradients far below 1e-4 want a loss scale.

    Returns ``(grad_queries, grad_keys, grad_values)``, new contiguous tensors with the shapes of the inputs.  Takes 4 bytes of
    scratch memory per row at least.

    Raises:
        TypeError: non-tensor inputs or a wrong dtype.
        ValueError: bad shapes, strides, batch sizes or devices, a scale that is not finite.
        RuntimeError: the limit on scratch memory, or the supplied buffer, does not allow those bytes.
    """
    plan = _plan_attention_grad(grad_out, queries, keys, values, out, lse, scale, key_lengths, key_mask)
    params, device = plan.params, queries.device
    stream = _current_stream_for(device)
    needed = _backend.attention_gradient_workspace_bytes(params)
    if needed:
        workspace = _scratch.allocate(needed, device)
        if workspace is None:           # refused: uncut launches, with room for one sum per row
            needed = -(-4 * params.l * params.m * params.h // 16) * 16
            workspace = _scratch.allocate(needed, device)
        if workspace is None:
            raise RuntimeError(f"cross_attention_grad needs {needed} bytes of scratch memory: the limit, the supplied buffer or the device does not allow them")
        params.workspace, params.workspace_bytes = workspace.data_ptr(), needed
    if debug:
        print("(Kermac Debug) Launching kernel: attention_grad_queries, attention_grad_keys")
    _backend.attention_gradient(params, stream)
    return plan.out


@_scratch.operator
def prefix_attention(
    queries: torch.Tensor,                  # [L, M, H, K]
    prefix_keys: torch.Tensor,              # [P, G, K]
    prefix_values: torch.Tensor,            # [P, G, O]
    keys: torch.Tensor,                     # [L, N, G, K]
    values: torch.Tensor,                   # [L, N, G, O]
    lengths: torch.Tensor,                  # [L]
    out: Optional[torch.Tensor] = None,     # [L, M, H, O]
    *,
    scale: Optional[float] = None,
    debug=False,
):
    """Attention of a batch of sequences that continue one common prefix, whose keys and values are read once for all of them.

    Sequence ``l`` consists of the ``P`` tokens of the prefix and ``lengths[l]`` tokens of its own, whose keys and values stand in the first
    ``lengths[l]`` rows of ``keys[l]`` and ``values[l]``.  Its queries are its last ``M`` tokens: query ``m`` is its own token
    ``lengths[l] - M + m`` and meets the whole prefix and its own tokens up to itself.  ``M = 1`` is one step of generation, a
    larger ``M`` a prompt behind the prefix.  Where ``lengths[l] < M``, the first queries are tokens that do not exist: they meet
    the prefix alone.  What ``keys`` and ``values`` hold behind ``lengths[l]`` does not matter.

    Types, heads, ``scale``, ``out`` and errors are those of ``cross_attention``; ``lengths`` is int32, taken as 0 .. N where outside.
    Returns ``out`` (allocated ``[L, M, H, O]`` when None).
    """
    if not isinstance(lengths, torch.Tensor):
        raise TypeError("lengths must be a PyTorch tensor")
    plan = _plan_attention(queries, keys, values, out, scale, lengths, None, False, prefix=(prefix_keys, prefix_values))
    _launch(plan, queries.device, debug)
    return plan.out
