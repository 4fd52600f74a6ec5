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


# ------------------------------------------------------------------------------------------------ gradients

def check_gradients(grads, d, q, k, v, keep, scale, what):
    """Against the formulas in 64 bits.  Scores are exact; weights are off by 2^-10 of themselves at most where the lse is below 4096 to base 2 (fp32 rounds it, and its
    product with log2(e), to 2^-13 each) and by a few roundings where it is larger.  What passes the operands' type may come back as an infinity, not as NaN."""
    unit, floor = UNIT[q.dtype], reference.FLOOR[q.dtype]
    L, M, H, _ = q.shape
    N, G, O = v.shape[1:]
    R, shared = H // G, k.shape[0] == 1 and L > 1
    p, lse = softmax(q, k, keep, scale)
    scale = torch.tensor(scale, dtype=torch.float32).double()
    k, v = (x.cpu().double().expand(L, -1, -1, -1).repeat_interleave(R, 2).transpose(1, 2).contiguous() for x in (k, v))
    q, d = (x.cpu().double().transpose(1, 2).contiguous() for x in (q, d))
    near = (lse.abs() < 4096 * math.log(2))[..., None]
    E = torch.where(near, 2.0 ** -10, 256 * E32)
    A = torch.matmul(p, v.abs())
    out = torch.matmul(p, v)
    dp, dp_magnitude = torch.matmul(d, v.transpose(2, 3)), torch.matmul(d.abs(), v.abs().transpose(2, 3))
    delta = (d * out).sum(-1, keepdim=True)
    delta_error = (d.abs() * (unit * 1.01 * (out.abs() + A) + 2 * (E + (N + 16) * E32) * A + floor)).sum(-1, keepdim=True) + (O + N + 16) * E32 * (d.abs() * A).sum(-1, keepdim=True)
    alone = p.amax(-1, keepdim=True) == 1.0                   # all weight on one key: its dp is delta, so that ds is 0, to the last bit
    ds = torch.where(alone, 0.0, p * (dp - delta))
    ds_error = E * p * (dp - delta).abs() + p * ((O + 16) * E32 * dp_magnitude + delta_error)
    ds_error = torch.where(alone, 0.0, ds_error + unit * 1.01 * (ds.abs() + ds_error) + floor * (p > 0))
    p_error = torch.where(alone, 0.0, E * p + unit * 1.01 * p + floor * (p > 0))
    if alone.any():
        assert grads[0].cpu().transpose(1, 2)[alone[..., 0] & ~near[..., 0]].eq(0).all(), what + ": the gradient of a query with one key is 0"

    def over_rows(x):
        x = x.reshape(L, G, R, N, -1).sum(2).transpose(1, 2)
        return x.sum(0, keepdim=True) if shared else x

    rows = M * R * (L if shared else 1) + 16
    values = ((scale * torch.matmul(ds, k)).transpose(1, 2), over_rows(scale * torch.matmul(ds.transpose(2, 3), q)), over_rows(torch.matmul(p.transpose(2, 3), d)))
    bounds = (scale.abs() * (torch.matmul(ds_error, k.abs()) + (N + 16) * E32 * torch.matmul(ds.abs(), k.abs())).transpose(1, 2),
              over_rows(scale.abs() * (torch.matmul(ds_error.transpose(2, 3), q.abs()) + rows * E32 * torch.matmul(ds.abs().transpose(2, 3), q.abs()))),
              over_rows(torch.matmul(p_error.transpose(2, 3), d.abs()) + rows * E32 * torch.matmul(p.transpose(2, 3), d.abs())))
    largest = torch.finfo(grads[0].dtype).max
    for name, got, truth, bound in zip(("queries", "keys", "values"), grads, values, bounds):
        bound = bound + unit * 1.01 * (truth.abs() + bound) + floor
        beyond = truth.abs() + bound > 0.99 * largest
        assert not got.isnan().any(), f"{what}: NaN in the gradient of {name}"
        reference.assert_within(got.masked_fill(beyond.to(got.device), 0.0), truth.masked_fill(beyond, 0.0), bound, f"{what} grad of {name}")


def step(d, q, k, v, **masks):
    out, lse = kermac.cross_attention(q, k, v, return_lse=True, **masks)
    return kermac.cross_attention_grad(d, q, k, v, out, lse, **masks)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("scale", SCALES)
@pytest.mark.parametrize("L, M, N, keys", [(2, 3, 20, 2), (2, 1, 5000, 2), (3, 40, 200, 3), (3, 40, 200, 1), (1, 200, 1001, 1)])
def test_gradient(device, dtype, scale, L, M, N, keys):
    """One tile of keys and many, whole and cut, sources of their own and a shared one; masks and a row without keys."""
    q, k = whole(L, M, 4, 64, dtype=dtype, device=device, seed=1), whole(keys, N, 2, 64, dtype=dtype, device=device, seed=2)
    v, d = normal(keys, N, 2, 64, dtype=dtype, seed=3).to(device), normal(L, M, 4, 64, dtype=dtype, seed=9).to(device)
    check_gradients(step(d, q, k, v, scale=scale), d, q, k, v, reference.keep_of(L, M, N), scale, "all")
    mask = (torch.rand(L, N, generator=torch.Generator().manual_seed(5)) < 0.3).to(device)
    lengths = torch.tensor([N // 2, 0, N][:L], dtype=torch.int32, device=device)
    check_gradients(step(d, q, k, v, scale=scale, key_mask=mask, key_lengths=lengths), d, q, k, v, reference.keep_of(L, M, N, lengths, mask), scale, "masked")


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("width", [64, 80, 128, 256])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("M, N", [(1, 30), (40, 300), (130, 900)])
def test_gradient_of_scores_far_from_zero(device, dtype, width, sign, M, N):
    """Rows far away beside ordinary ones, in aligned rows and in others."""
    L = 2
    for pad in (0, 1):
        q, k = torch.zeros(L, M, 2, width + pad, dtype=dtype, device=device)[..., pad:], torch.zeros(L, N, 1, width + pad, dtype=dtype, device=device)[..., pad:]
        few_q, few_k, _ = far_operands(L, M, N, dtype, device, sign)
        q[..., :2], k[..., :2] = few_q[..., :2], few_k[..., :2]
        q[:, 1::2, :, 0] = 0.0
        v, d = normal(L, N, 1, width, dtype=dtype, seed=3).to(device), normal(L, M, 2, width, dtype=dtype, seed=9).to(device)
        mask = (torch.rand(L, N, generator=torch.Generator().manual_seed(5)) < 0.7).to(device)
        for masks in ({}, dict(key_mask=mask)):
            check_gradients(step(d, q, k, v, scale=1.0, **masks), d, q, k, v, reference.keep_of(L, M, N, **masks), 1.0, f"pad={pad} {list(masks)}")


def test_gradient_with_the_least_scratch_memory(device):
    """Without room for shifts, ordinary rows have the gradients that they have with it."""
    q, k, v, d = (normal(2, n, h, 64, dtype=torch.bfloat16, seed=i).to(device) for i, (n, h) in enumerate(((40, 4), (130, 2), (130, 2), (40, 4))))
    q[0, 3] *= 1000.0
    out, lse = kermac.cross_attention(q, k, v, return_lse=True)
    assert lse.abs().max() > 2839 and lse[1].abs().max() < 2839
    roomy = kermac.cross_attention_grad(d, q, k, v, out, lse)
    kermac.set_max_scratch_bytes(8 * 2 * 40 * 4 + 16)
    try:
        least = kermac.cross_attention_grad(d, q, k, v, out, lse)
    finally:
        kermac.set_max_scratch_bytes(None)
    assert all(torch.equal(a[1], b[1]) for a, b in zip(roomy, least))


def test_a_row_without_keys_has_no_gradient(device):
    """Whatever the gradient of its result is."""
    q, k, v = (normal(2, n, 2, 64, dtype=torch.bfloat16, seed=i).to(device) for i, n in enumerate((5, 200, 200)))
    d = torch.full_like(q, math.inf)
    mask = torch.zeros(2, 200, dtype=torch.bool, device=device)
    for grad in step(d, q, k, v, key_mask=mask) + step(d, q, k, v, key_lengths=torch.zeros(2, dtype=torch.int32, device=device)):
        assert grad.eq(0).all()
