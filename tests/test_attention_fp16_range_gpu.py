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


@pytest.mark.parametrize("M, N", [(1, 20000), (1, 150001), (2, 100003), (40, 70000)])
def test_gradient_of_values_of_many_keys(device, M, N):
    """Weights of 1 / N, rounded in front of the product with the gradient of the result: to half a step each, and a floor of 2^-40."""
    q, k = normal(1, M, 1, 64, dtype=DTYPE, seed=1) * 0.25, normal(1, N, 1, 64, dtype=DTYPE, seed=2)
    v, d = normal(1, N, 1, 64, dtype=DTYPE, seed=3), normal(1, M, 1, 64, dtype=DTYPE, seed=9) * 1024
    scores = q[0, :, 0].double() @ k[0, :, 0].double().t() / 8
    p = torch.softmax(scores, -1)
    truth, A = p.t() @ d[0, :, 0].double(), p.t() @ d[0, :, 0].double().abs()
    S = (q[0, :, 0].double().abs() @ k[0, :, 0].double().abs().t() / 8).max()
    E = 4 * (64 + 4) * E32 * S + 64 * E32 + 2 * (N + 16) * E32 * 2.0 ** -8          # (sums of N weights: their partial sums are 2^8 times as exact at least, N / 256 per lane)
    bound = (1.01 * UNIT[DTYPE] + E + (M + 16) * E32) * A + 2.0 ** -40 * d.double().abs().sum() + 1.01 * UNIT[DTYPE] * truth.abs() + 2.0 ** -25
    args = [x.to(device) for x in (q, k, v)]
    out, lse = kermac.cross_attention(*args, return_lse=True)
    grads = kermac.cross_attention_grad(d.to(device), *args, out, lse)
    reference.assert_within(grads[2][0, :, 0], truth, bound, f"M={M} N={N}")


def test_gradients_of_scores_at_the_ends_of_the_type(device):
    """ds in front of the scale is a number of the type: up to 65504 it comes back as it is, and p = 1 / 2 of a result of 2^-22 does too."""
    for size, exact in ((2.0 ** 14, True), (2.0 ** -21, True), (2.0 ** 18, False)):
        q = torch.zeros(1, 1, 1, 64, dtype=DTYPE, device=device)
        k, v = torch.zeros(1, 2, 1, 64, dtype=DTYPE, device=device), torch.zeros(1, 2, 1, 64, dtype=DTYPE, device=device)
        k[0, :, 0, 0], v[0, 0, 0, 0], v[0, 1, 0, 0] = 1.0, 4.0, -4.0
        k[0, 1, 0, 0] = -1.0
        d = torch.zeros(1, 1, 1, 64, dtype=DTYPE, device=device)
        d[..., 0] = min(size, 2.0 ** 15)
        if size > 2.0 ** 15:
            v *= size / 2.0 ** 15
        out, lse = kermac.cross_attention(q, k, v, scale=2.0 ** -4, return_lse=True)
        grad_q, grad_k, grad_v = kermac.cross_attention_grad(d, q, k, v, out, lse, scale=2.0 ** -4)
        # p = 1/2 each, dp = 4 d and -4 d, delta = 0: ds = 2 d and -2 d, grad_q = 2^-4 (2 d + 2 d)
        assert grad_q[0, 0, 0, 0].item() == (size * 2.0 ** -2 if exact else math.inf)
        assert grad_v[0, :, 0, 0].tolist() == [min(size, 2.0 ** 15) / 2] * 2
