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

import functools
import struct
from typing import Optional

import torch

from . import _backend
from . import _scratch
from .build_a_kernel import _current_stream_for

_TYPES = {torch.float32: _backend.FP32, torch.float16: _backend.FP16, torch.bfloat16: _backend.BF16}
_MAX_WIDTH = 256
_MAX_EXTENT = 2_000_000_000
_MAX_SCALE = 2e38                       # times log2(e) still a number of fp32

# A call on one token costs the GPU a few microseconds, so its host side counts: the parameter blocks are packed in one step (a field by
# field structure takes four times as long), and what a shape asks of the workspace is asked of the library once.
_PARAMS = struct.Struct(_backend.struct_format(_backend.AttentionParams))
_GRADIENT_PARAMS = struct.Struct(_backend.struct_format(_backend.AttentionGradientParams))


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(element, L, M, N, H, G, K, O, P, causal, with_lengths):
    """kmc_attention_workspace_bytes: a function of these alone."""
    one = 16                            # stands for any address: nothing is read
    return _backend.attention_workspace_bytes(_backend.AttentionParams(
        element, 0, L, M, N, H, G, K, O, 1.0, q=one, key=one, value=one, out=one, key_lengths=one if with_lengths else None, prefix_n=P, causal=causal,
        prefix_key=one, prefix_value=one))


@functools.lru_cache(maxsize=4096)
def _gradient_workspace_bytes(element, L, M, N, H, G, K, O, key_entries):
    one = 16
    return _backend.attention_gradient_workspace_bytes(_backend.AttentionGradientParams(
        element, 0, L, M, N, H, G, K, O, key_entries, 1.0, q=one, key=one, value=one, out=one, grad_out=one, lse=one, grad_q=one, grad_key=one,
        grad_value=one))


def _check(name, x, device, dtype):
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{name} must be a PyTorch tensor")
    if x.dtype is not dtype:
        raise TypeError(f"{name} must have dtype {dtype}, got {x.dtype}")
    if x.device != device:
        raise ValueError(f"{name} must be on the same CUDA device as inputs: got {x.device}, expected {device}")


def _operand(name, x, device, dtype):
    """(batch entries, tokens, heads, features, strides of the first three) of a [tokens, heads, features] tensor or a batch of them."""
    _check(name, x, device, dtype)
    shape, strides = x.shape, x.stride()
    if len(strides) == 4:
        (L, tokens, heads, width), (ls, ts, hs, ws) = shape, strides
        if L == 1:
            ls = 0
    elif len(strides) == 3:
        (tokens, heads, width), (ts, hs, ws) = shape, strides
        L, ls = 1, 0
    else:
        raise ValueError(f"{name} must be 3-dimensional or 4-dimensional with a batch mode")
    if ws != 1 and width > 1:
        raise ValueError(f"{name} must have stride 1 in last dimension")
    if not 1 <= width <= _MAX_WIDTH:
        raise ValueError(f"the last dimension of {name} must be 1 .. {_MAX_WIDTH}, got {width}")
    return L, tokens, heads, width, ls, ts, hs


def _strides_of_result(name, out, shape, device, dtype):
    _check(name, out, device, dtype)
    if tuple(out.shape) != shape and not (out.dim() == 3 and shape[0] == 1 and tuple(out.shape) == shape[1:]):
        raise ValueError(f"{name} must have shape {shape}, got {tuple(out.shape)}")
    strides = out.stride()
    if any(stride == 0 and extent > 1 for extent, stride in zip(out.shape, strides)):
        raise ValueError(f"{name} must not be an expanded tensor")
    if strides[-1] != 1 and shape[-1] > 1:
        raise ValueError(f"{name} must have stride 1 in last dimension")
    return strides[0] if len(strides) == 4 else 0, strides[-3], strides[-2]


def _mask(key_mask, L, N, device):
    """(address, stride of an entry, stride of a key)"""
    _check("key_mask", key_mask, device, torch.bool)
    if tuple(key_mask.shape) not in ((N,), (1, N), (L, N)):
        raise ValueError(f"key_mask must have shape (N={N},) or (L={L}, N={N}), got {tuple(key_mask.shape)}")
    return key_mask.data_ptr(), key_mask.stride(0) if key_mask.dim() == 2 and key_mask.size(0) > 1 else 0, key_mask.stride(-1)


class _AttentionPlan:
    """A checked call: `fields` are those of the parameter block in front of the workspace's."""
    __slots__ = ("fields", "extents", "out", "lse", "device")

    @property
    def params(self) -> _backend.AttentionParams:
        """The block as a structure."""
        return _backend.AttentionParams.from_buffer_copy(_PARAMS.pack(*self.fields, 0, 0))


def _plan_attention(queries, keys, values, out, scale, key_lengths, key_mask, return_lse, prefix=None, require_device=True) -> _AttentionPlan:
    """Validation and parameter marshalling, without the launch.  `prefix`: the prefix's keys and values; the queries are then
    the last tokens of `key_lengths`."""
    if not isinstance(queries, torch.Tensor):
        raise TypeError("queries must be a PyTorch tensor")
    device, dtype = queries.device, queries.dtype
    element = _TYPES.get(dtype)
    if element is None:
        raise TypeError(f"queries must have dtype torch.float32, torch.float16 or torch.bfloat16, got {dtype}")
    if require_device and not queries.is_cuda:
        raise ValueError("queries must be on a CUDA device")
    L, M, H, K, q_ls, q_ms, q_hs = _operand("queries", queries, device, dtype)
    L_k, N, G, K_k, k_ls, k_ns, k_gs = _operand("keys", keys, device, dtype)
    L_v, N_v, G_v, O, v_ls, v_ns, v_gs = _operand("values", values, device, dtype)
    if L_k != L_v or (L_k != L and (L_k != 1 or prefix is not None)):
        raise ValueError(f"keys and values must both have the batch size of queries (L={L})"
                         + (" or both 1" if prefix is None else "") + f", got {L_k} and {L_v}")
    if K_k != K:
        raise ValueError(f"keys must have as many features as queries (K={K}), got {K_k}")
    if N_v != N or G_v != G:
        raise ValueError(f"values must have as many tokens and heads as keys (N={N}, G={G}), got {N_v} and {G_v}")
    if G == 0 and H > 0 or G > 0 and H % G != 0:
        raise ValueError(f"the heads of queries (H={H}) must be a multiple of the heads of keys (G={G})")
    if L * M * H > _MAX_EXTENT or max(L, M, N, H) > _MAX_EXTENT:
        raise ValueError(f"at most {_MAX_EXTENT} keys, and rows over the batch and the heads: got N={N}, L={L}, M={M}, H={H}")
    scale = K ** -0.5 if scale is None else float(scale)
    if not abs(scale) <= _MAX_SCALE:
        raise ValueError(f"scale must be finite and at most {_MAX_SCALE:g}, got {scale}")
    lengths_ptr = mask_ptr = mask_ls = mask_ns = 0
    if key_lengths is not None:
        name = "key_lengths" if prefix is None else "lengths"
        _check(name, key_lengths, device, torch.int32)
        if key_lengths.dim() != 1 or key_lengths.size(0) != L or (L > 1 and key_lengths.stride(0) != 1):
            raise ValueError(f"{name} must be contiguous with shape (L={L},), got {tuple(key_lengths.shape)}")
        lengths_ptr = key_lengths.data_ptr()
    if key_mask is not None:
        mask_ptr, mask_ls, mask_ns = _mask(key_mask, L, N, device)
    P = causal = pk_ptr = pk_ns = pk_gs = pv_ptr = pv_ns = pv_gs = 0
    if prefix is not None:
        prefix_k, prefix_v = prefix
        L_p, P, G_p, K_p, _, pk_ns, pk_gs = _operand("prefix_keys", prefix_k, device, dtype)
        L_pv, P_v, G_pv, O_p, _, pv_ns, pv_gs = _operand("prefix_values", prefix_v, device, dtype)
        if prefix_k.dim() != 3 or prefix_v.dim() != 3:
            raise ValueError("prefix_keys and prefix_values must be 3-dimensional: they have no batch mode")
        if G_p != G or K_p != K:
            raise ValueError(f"prefix_keys must have the heads and features of keys (G={G}, K={K}), got {G_p} and {K_p}")
        if P > _MAX_EXTENT:
            raise ValueError(f"at most {_MAX_EXTENT} keys: got P={P}")
        if P_v != P or G_pv != G or O_p != O:
            raise ValueError(f"prefix_values must have the tokens of prefix_keys and the heads and features of values (P={P}, G={G}, O={O}), "
                             f"got {P_v}, {G_pv} and {O_p}")
        causal, pk_ptr, pv_ptr = 1, prefix_k.data_ptr(), prefix_v.data_ptr()

    if out is None:
        # (a dense tensor of that shape either way; the first form is the quicker call)
        out = torch.empty_like(queries, memory_format=torch.contiguous_format) if O == K and len(queries.shape) == 4 else torch.empty(
            (L, M, H, O), dtype=dtype, device=device)
        o_hs = O
        o_ms = H * o_hs
        o_ls = M * o_ms
    else:
        o_ls, o_ms, o_hs = _strides_of_result("out", out, (L, M, H, O), device, dtype)
    plan = _AttentionPlan()
    plan.lse, lse_ptr = None, 0
    if return_lse:
        plan.lse = torch.empty((L, M, H), dtype=torch.float32, device=device)
        lse_ptr = plan.lse.data_ptr()
    plan.out, plan.device = out, device
    plan.extents = (element, L, M, N, H, G, K, O, P, causal, lengths_ptr != 0)
    plan.fields = (element, 0, L, M, N, H, G, K, O, scale, queries.data_ptr(), q_ls, q_ms, q_hs, keys.data_ptr(), k_ls, k_ns, k_gs,
                   values.data_ptr(), v_ls, v_ns, v_gs, out.data_ptr(), o_ls, o_ms, o_hs, lse_ptr, lengths_ptr, mask_ptr, mask_ls, mask_ns, P, causal,
                   pk_ptr, pk_ns, pk_gs, pv_ptr, pv_ns, pv_gs)
    return plan


def _launch(plan, debug):
    stream = _current_stream_for(plan.device)
    needed = _workspace_bytes(*plan.extents)
    workspace = _scratch.allocate(needed, plan.device) if needed else None
    if debug:
        print(f"(Kermac Debug) Launching kernel: attention_forward{' and attention_join' if workspace is not None else ''}")
    if workspace is not None:
        _backend.attention(_PARAMS.pack(*plan.fields, workspace.data_ptr(), needed), stream)
    else:                               # none needed, or refused: one pass over the keys per tile of rows
        _backend.attention(_PARAMS.pack(*plan.fields, 0, 0), stream)
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
        scale: ``K ** -0.5`` when None; any number up to 2e38 in magnitude.
        key_lengths: int32 ``[L]``: the first so many keys of an entry take part (taken as 0 .. N where outside).
        key_mask: bool ``[N]`` or ``[L, N]``: the keys that take part.  With both, a key has to pass both.
        out: optional result, ``[L, M, H, O]``, written in place and returned; it must not share memory with the inputs.
        return_lse: also return ``log sum exp`` of every row, fp32 ``[L, M, H]``, for ``cross_attention_grad``.

    What keys and values hold where they do not take part does not matter, infinities and NaN included.  A row
    without a key (or with scores of -inf alone) gets zeros, and -inf for its ``lse``, which no other row has: one below fp32's
    numbers is the lowest of them.  Scores of any size give a softmax, with all the weight on the largest where they are far apart.  Returns ``out``
    (allocated ``[L, M, H, O]`` when None), or ``(out, lse)``.

    Raises:
        TypeError: non-tensor inputs or a wrong dtype.
        ValueError: bad shapes, strides, batch sizes or devices, a scale that is not finite or beyond 2e38.
    """
    plan = _plan_attention(queries, keys, values, out, scale, key_lengths, key_mask, return_lse)
    _launch(plan, debug)
    return (plan.out, plan.lse) if return_lse else plan.out


class _GradientPlan:
    __slots__ = ("fields", "extents", "out", "device")

    @property
    def params(self) -> _backend.AttentionGradientParams:
        return _backend.AttentionGradientParams.from_buffer_copy(_GRADIENT_PARAMS.pack(*self.fields, 0, 0))


def _plan_attention_grad(grad_out, queries, keys, values, out, lse, scale, key_lengths, key_mask, require_device=True) -> _GradientPlan:
    """The checks of the forward call, whose result `out` and `lse` are, and the gradient's parameters."""
    if out is None:
        raise TypeError("out must be a PyTorch tensor")
    of = _plan_attention(queries, keys, values, out, scale, key_lengths, key_mask, False, require_device=require_device)
    element, L, M, N, H, G, K, O = of.extents[:8]
    device, dtype = of.device, queries.dtype
    L_d, M_d, H_d, O_d, d_ls, d_ms, d_hs = _operand("grad_out", grad_out, device, dtype)
    if (L_d, M_d, H_d, O_d) != (L, M, H, O):
        raise ValueError(f"grad_out must have shape {(L, M, H, O)}, got {tuple(grad_out.shape)}")
    _check("lse", lse, device, torch.float32)
    if tuple(lse.shape) != (L, M, H) or not lse.is_contiguous():
        raise ValueError(f"lse must be contiguous with shape {(L, M, H)}, got {tuple(lse.shape)}")
    key_entries = keys.size(0) if keys.dim() == 4 else 1
    contiguous = torch.contiguous_format
    make = torch.empty_like if L * M * H else torch.zeros_like         # no query: nothing is launched
    grad_q = torch.empty_like(queries, memory_format=contiguous)
    grad_k, grad_v = make(keys, memory_format=contiguous), make(values, memory_format=contiguous)
    plan = _GradientPlan()
    plan.out, plan.device = (grad_q, grad_k, grad_v), device
    plan.extents = (element, L, M, N, H, G, K, O, key_entries)
    # type .. o of the forward block, key_entries, scale, then its operands up to out's strides
    plan.fields = (*of.fields[:9], key_entries, *of.fields[9:26], grad_out.data_ptr(), d_ls, d_ms, d_hs, lse.data_ptr(), *of.fields[27:31],
                   grad_q.data_ptr(), grad_k.data_ptr(), grad_v.data_ptr())
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
    keys.  Sums are fp32 in an order that does not depend on timing.  In fp16, the gradients of the scores, ``p * (d v - sum p d v)`` with
    ``d`` the gradient of the result and without ``scale``, are numbers of that type: what passes 65504 becomes infinite, what is below ``6e-8`` is lost,
    and a loss scale has to bring them in between.

    Returns ``(grad_queries, grad_keys, grad_values)``, new contiguous tensors with the shapes of the inputs.  Takes 8 bytes of
    scratch memory per row at least.  Scores of any size want 4 more (and 4 per 128 rows): where a limit leaves only those 8, weights of a row
    whose ``lse`` is 2839 or larger in magnitude are off by the relative ``2**-23 * |lse|``, as fp32 holds it.

    Raises:
        TypeError: non-tensor inputs or a wrong dtype.
        ValueError: bad shapes, strides, batch sizes or devices, a scale that is not finite or beyond 2e38.
        RuntimeError: the limit on scratch memory, or the supplied buffer, does not allow those bytes.
    """
    plan = _plan_attention_grad(grad_out, queries, keys, values, out, lse, scale, key_lengths, key_mask)
    stream = _current_stream_for(plan.device)
    needed, workspace = _gradient_workspace_bytes(*plan.extents), None
    if needed:
        workspace = _scratch.allocate(needed, plan.device)
        if workspace is None:           # refused: uncut launches, with room for the sums of a row, and for a shift of its scores if there is
            _, L, M, _, H, G = plan.extents[:6]
            least, shifts = (8 * L * M * H + 8 + 15) // 16 * 16, (4 * L * M * H + 4 * L * G * -(-M * (H // G) // 128) + 15) // 16 * 16
            for needed in (least + shifts, least):
                workspace = _scratch.allocate(needed, plan.device)
                if workspace is not None:
                    break
        if workspace is None:
            raise RuntimeError(f"cross_attention_grad needs {needed} bytes of scratch memory: the limit, the supplied buffer or the device does not allow them")
    if debug:
        print("(Kermac Debug) Launching kernel: attention_grad_queries, attention_grad_keys")
    _backend.attention_gradient(_GRADIENT_PARAMS.pack(*plan.fields, workspace.data_ptr() if needed else 0, needed), stream)
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
    the prefix alone.  What ``keys`` and ``values`` hold behind ``lengths[l]`` does not matter.  (In front of it it does: an infinity or NaN among
    the values of a sequence's own token may reach its queries in front of that token too, whose weight for it is 0.)

    Types, heads, ``scale``, ``out`` and errors are those of ``cross_attention``; ``lengths`` is int32, taken as 0 .. N where outside.
    Returns ``out`` (allocated ``[L, M, H, O]`` when None).
    """
    if not isinstance(lengths, torch.Tensor):
        raise TypeError("lengths must be a PyTorch tensor")
    plan = _plan_attention(queries, keys, values, out, scale, lengths, None, False, prefix=(prefix_keys, prefix_values))
    _launch(plan, debug)
    return plan.out
