"""Attention in fp16 where weights are small: what the type's range takes from them, and what it must not."""
import math

import pytest
import torch

import kermac_amd as kermac
from tests import attention_reference as reference
from tests.attention_reference import E32, UNIT
from tests.test_attention_gpu import normal

pytestmark = pytest.mark.gpu
DTYPE = torch.float16


@pytest.mark.parametrize("M", [1, 40])
@pytest.mark.parametrize("N", [4096, 65536])
@pytest.mark.parametrize("above", [16.0, 18.0, 20.0])
@pytest.mark.parametrize("at", [0, 1000, -1])
def test_one_key_that_stands_out(device, M, N, above, at):
    """A key whose score is `above` higher than the others' and whose value is 0: the result is the others' share, N exp(-above) of their values.

    Weights are held to half a step of 2^-24, the type's smallest number, beside 2^7 for the largest: 2^-32 of it each, and to half of their own step."""
    q = torch.zeros(1, M, 1, 64)
    k = normal(1, N, 1, 64, dtype=torch.float32, seed=2)
    v = normal(1, N, 1, 64, dtype=torch.float32, seed=3).abs()
    q[..., 0], q[..., 1] = 1.0, 0.25
    k[..., 0] = 0.0
    k[:, at, :, 0], k[:, at, :, 1] = above, 0.0
    v[:, at] = 0.0
    q, k, v = (x.to(DTYPE) for x in (q, k, v))
    scores = (q[..., :2].double().transpose(1, 2) @ k[..., :2].double().permute(0, 2, 3, 1))
    weights = torch.softmax(scores, -1)
    truth = (weights @ v.double().transpose(1, 2)).transpose(1, 2)
    largest = weights.amax(-1).transpose(1, 2)[..., None]
    E = 2 * (64 + 4) * E32 * (above + 2) + 16 * E32 + (N + 16) * E32
    bound = 3.03 * UNIT[DTYPE] * truth + 2 * E * truth + 2.0 ** -32 * largest * v.double().sum(1, keepdim=True)
    out = kermac.cross_attention(*(x.to(device) for x in (q, k, v)), scale=1.0)
    reference.assert_within(out, truth, bound, f"M={M} N={N} above={above} at={at}")
    kermac.set_max_scratch_bytes(0)
    try:
        reference.assert_within(kermac.cross_attention(*(x.to(device) for x in (q, k, v)), scale=1.0), truth, bound, "uncut")
    finally:
        kermac.set_max_scratch_bytes(None)


@pytest.mark.parametrize("M", [1, 40])
def test_largest_values_and_weights(device, M):
    """The largest weights meet the type's largest values: nothing passes fp32, and the result is an average."""
    q, k = normal(2, M, 2, 64, dtype=DTYPE, seed=1).to(device), normal(2, 3000, 2, 64, dtype=DTYPE, seed=2).to(device)
    v = torch.full((2, 3000, 2, 64), 65504.0, dtype=DTYPE, device=device)
    # (an average of equal numbers: off by the sums' rounding, (N + 16) 2^-24, and that of the weights, 2^-11; not beyond the type)
    out = kermac.cross_attention(q, k * torch.linspace(0.1, 3.0, 3000, device=device).to(DTYPE)[None, :, None, None], v / 2)
    assert ((out.float() - 32752).abs() <= 32752 * (2.0 ** -11 * 2.02 + 3016 * E32)).all()
