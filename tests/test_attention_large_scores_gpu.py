"""Attention where scale times <query, key> is large: a softmax with all its weight on the largest scores, not an overflow.

Operands are small whole numbers, so that every score is exact in fp32 and what the kernels have to give follows from the definition without an error of
the scores: keys with the largest score share the weight, at these scales a key one below them has exp(-10^6) of it or less, which is 0.
"""
import math

import pytest
import torch

import kermac_amd as kermac
from tests import attention_reference as reference
from tests.attention_reference import E32, UNIT
from tests.test_attention_gpu import TYPES, normal

pytestmark = pytest.mark.gpu

SCALES = [1e6, 1e9, -1e9, 1e20, 2e38]


def whole(*shape, dtype, device, seed, largest=4):
    return torch.randint(-largest, largest + 1, shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(device)


def softmax(q, k, keep, scale):
    """(weights [L, H, M, N], log of the sum of exponentials [L, H, M]) in 64 bits, scale as fp32 holds it; rows without keys get zeros and -inf."""
    scale = torch.tensor(scale, dtype=torch.float32).double()
    H, G = q.shape[2], k.shape[2]
    q, k = q.cpu().double().transpose(1, 2), k.cpu().double().expand(q.shape[0], -1, -1, -1).repeat_interleave(H // G, 2).transpose(1, 2)
    scores = (torch.matmul(q, k.transpose(2, 3).contiguous()) * scale).masked_fill(~keep[:, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    weights = torch.exp(scores - top.clamp_min(-1e300))
    total = weights.sum(-1, keepdim=True)
    lse = (total.log() + top.clamp_min(-1e300)).masked_fill(total == 0, -math.inf)[..., 0]
    return weights / total.clamp_min(1e-300), lse


def check(got, q, k, v, keep, scale, what, lse=None):
    """The weights in front of the division are exactly 1 or 0, or off by `E` of themselves: a few roundings of an exponent of some units and of its exponential."""
    N, H, G = v.shape[1], q.shape[2], v.shape[2]
    weights, true_lse = softmax(q, k, keep, scale)
    v = v.cpu().double().expand(q.shape[0], -1, -1, -1).repeat_interleave(H // G, 2).transpose(1, 2).contiguous()
    truth, A = torch.matmul(weights, v).transpose(1, 2), torch.matmul(weights, v.abs()).transpose(1, 2)
    E, unit = 64 * E32, UNIT[q.dtype]
    bound = unit * 1.01 * (truth.abs() + A) + 2 * (E + (N + 16) * E32) * A
    reference.assert_within(got, truth, bound, what)
    if lse is not None:
        true_lse = true_lse.transpose(1, 2)
        held = true_lse.clamp(-torch.finfo(torch.float32).max, math.inf).masked_fill(true_lse == -math.inf, -math.inf)
        beyond = held > torch.finfo(torch.float32).max
        got = lse.cpu().double()
        assert got[beyond].eq(math.inf).all()
        # the scale and its product with log2(e), the product with the score and back to base e, the sum: a rounding each
        bound = 8 * E32 * held.abs() + 64 * E32
        reference.assert_within(lse.masked_fill(beyond.to(lse.device), 0.0), held.masked_fill(beyond, 0.0), bound.nan_to_num(posinf=0.0), what + " lse")


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("scale", SCALES)
@pytest.mark.parametrize("L, M, N", [(2, 1, 50), (2, 1, 5000), (3, 40, 200), (1, 200, 3001)])
def test_cross(device, dtype, scale, L, M, N):
    """Single tokens and tiles of rows, keys in one part and cut over workgroups; masks and a row without keys."""
    q, k = whole(L, M, 4, 64, dtype=dtype, device=device, seed=1), whole(L, N, 2, 64, dtype=dtype, device=device, seed=2)
    v = normal(L, N, 2, 64, dtype=dtype, seed=3).to(device)
    out, lse = kermac.cross_attention(q, k, v, scale=scale, return_lse=True)
    check(out, q, k, v, reference.keep_of(L, M, N), scale, "all", lse)
    mask = (torch.rand(L, N, generator=torch.Generator().manual_seed(5)) < 0.3).to(device)
    lengths = torch.tensor([N // 2, 0, N][:L], dtype=torch.int32, device=device)
    out, lse = kermac.cross_attention(q, k, v, scale=scale, key_mask=mask, key_lengths=lengths, return_lse=True)
    check(out, q, k, v, reference.keep_of(L, M, N, lengths, mask), scale, "masked", lse)
    kermac.set_max_scratch_bytes(0)
    try:
        check(kermac.cross_attention(q, k, v, scale=scale), q, k, v, reference.keep_of(L, M, N), scale, "uncut")
    finally:
        kermac.set_max_scratch_bytes(None)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("scale", SCALES)
@pytest.mark.parametrize("L, M, P, N", [(3, 1, 1000, 40), (2, 50, 300, 150)])
def test_prefix(device, dtype, scale, L, M, P, N):
    q, k = whole(L, M, 4, 64, dtype=dtype, device=device, seed=1), whole(L, N, 2, 64, dtype=dtype, device=device, seed=2)
    pk, pv = whole(P, 2, 64, dtype=dtype, device=device, seed=4), normal(P, 2, 64, dtype=dtype, seed=5).to(device)
    v = normal(L, N, 2, 64, dtype=dtype, seed=3).to(device)
    lengths = torch.tensor([N, N // 2, 0][:L], dtype=torch.int32, device=device)
    keep = torch.cat((torch.ones(L, M, P, dtype=torch.bool), reference.keep_of(L, M, N, lengths, causal=True)), 2)
    joined = [torch.cat((x[None].expand(L, *x.shape), y), 1) for x, y in ((pk, k), (pv, v))]
    for limit in (None, 0):
        kermac.set_max_scratch_bytes(limit)
        try:
            check(kermac.prefix_attention(q, pk, pv, k, v, lengths, scale=scale), q, *joined, keep, scale, f"limit {limit}")
        finally:
            kermac.set_max_scratch_bytes(None)


def far_operands(L, M, N, dtype, device, sign=1):
    """Scores 2^22 + {0 .. 5} (or minus that): the weights are spread over the keys, far from zero.  Values of one head of keys for two of queries."""
    q, k = torch.zeros(L, M, 2, 64), torch.zeros(L, N, 1, 64)
    q[..., 0], q[..., 1] = sign * 2.0 ** 11, 1.0
    k[..., 0] = 2.0 ** 11
    k[..., 1] = torch.randint(0, 6, (L, N, 1), generator=torch.Generator().manual_seed(7)).float()
    q[:, :, 1, 1] = -1.0
    return q.to(dtype).to(device), k.to(dtype).to(device), normal(L, N, 1, 64, dtype=dtype, seed=3).to(device)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("M, N", [(1, 70), (1, 4000), (40, 300), (130, 2500)])
def test_scores_far_from_zero(device, dtype, sign, M, N):
    q, k, v = far_operands(2, M, N, dtype, device, sign)
    out, lse = kermac.cross_attention(q, k, v, scale=1.0, return_lse=True)
    check(out, q, k, v, reference.keep_of(2, M, N), 1.0, "far", lse)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_rows_far_and_near_in_one_tile(device, dtype):
    """Rows whose scores are ordinary beside rows whose scores are far away, and keys that lift a row from one to the other."""
    L, M, N = 1, 40, 500
    q, k, v = far_operands(L, M, N, dtype, device)
    q[:, ::2, :, 0] = 0.0                       # scores 0 .. 5
    check(kermac.cross_attention(q, k, v, scale=1.0), q, k, v, reference.keep_of(L, M, N), 1.0, "rows")
    k[:, :, :, 0] = k[:, :, :, 0] * (torch.arange(N, device=device) // 100)[None, :, None].to(dtype) / 4
    check(kermac.cross_attention(q, k, v, scale=1.0), q, k, v, reference.keep_of(L, M, N), 1.0, "rising")
    check(kermac.cross_attention(q, k.flip(1), v, scale=1.0), q, k.flip(1), v, reference.keep_of(L, M, N), 1.0, "falling")
    check(kermac.cross_attention(-q[:, :1], k, v, scale=1.0), -q[:, :1], k, v, reference.keep_of(L, 1, N), 1.0, "below zero")


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("M", [1, 40])
@pytest.mark.parametrize("scale", [None, -7.0, 1e9, 2e38])
def test_one_key_is_its_value(device, dtype, M, scale):
    """In every type and at every scale, bit for bit: the weight of a row's only key is 1 in the operands' type."""
    q, k, v = (normal(2, n, h, 64, dtype=dtype, seed=i).to(device) for i, (n, h) in enumerate(((M, 4), (200, 2), (200, 2))))
    one = v[:, :1].repeat_interleave(2, 2).expand(2, M, 4, 64)
    assert torch.equal(kermac.cross_attention(q, k[:, :1], v[:, :1], scale=scale), one)
    lengths = torch.ones(2, dtype=torch.int32, device=device)
    assert torch.equal(kermac.cross_attention(q, k, v, scale=scale, key_lengths=lengths), one)
    nothing = torch.zeros(2, dtype=torch.int32, device=device)
    assert torch.equal(kermac.prefix_attention(q, k[0, :1], v[0, :1], k, v, nothing, scale=scale), v[:1, :1].repeat_interleave(2, 2).expand(2, M, 4, 64))
