"""Cross attention and prefix attention against the definition in 64 bits."""
import math

import pytest
import torch

import kermac_amd as kermac
from tests import attention_reference as reference

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]


def normal(*shape, dtype, seed):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def operands(L, M, N, H, G, K, O, dtype, device, key_batch=None):
    key_batch = L if key_batch is None else key_batch
    return (normal(L, M, H, K, dtype=dtype, seed=1).to(device), normal(key_batch, N, G, K, dtype=dtype, seed=2).to(device),
            normal(key_batch, N, G, O, dtype=dtype, seed=3).to(device))


def check_cross(q, k, v, what, scale=None, key_lengths=None, key_mask=None, **more):
    out, lse = kermac.cross_attention(q, k, v, scale=scale, key_lengths=key_lengths, key_mask=key_mask, return_lse=True, **more)
    L, M, N = q.shape[0], q.shape[1], k.shape[1]
    truth, truth_lse, bound, lse_bound = reference.forward(q, k, v, reference.keep_of(L, M, N, key_lengths, key_mask),
                                                           q.shape[-1] ** -0.5 if scale is None else scale)
    reference.assert_within(out, truth, bound, what)
    reference.assert_within(lse, truth_lse, lse_bound, what + " lse")
    return out


# one row, a tile of 32 that is just full or just passed, several workgroups; keys that end inside, at and behind a tile
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("M, N", [(1, 1), (1, 33), (2, 64), (31, 65), (33, 31), (129, 127), (40, 200), (300, 520)])
def test_lengths(device, dtype, M, N):
    q, k, v = operands(2, M, N, 2, 2, 64, 64, dtype, device)
    check_cross(q, k, v, f"M={M} N={N}")


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("K, O", [(1, 1), (7, 5), (16, 40), (32, 32), (80, 80), (96, 128), (128, 64), (128, 128), (200, 72), (256, 256), (251, 3)])
@pytest.mark.parametrize("M", [1, 70])
def test_features(device, dtype, K, O, M):
    q, k, v = operands(1, M, 150, 4, 2, K, O, dtype, device)
    check_cross(q, k, v, f"K={K} O={O} M={M}")


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("H, G, M", [(1, 1, 1), (8, 1, 1), (40, 1, 1), (33, 1, 3), (6, 2, 5), (20, 4, 17), (12, 12, 1)])
def test_heads(device, dtype, H, G, M):
    q, k, v = operands(3, M, 90, H, G, 64, 64, dtype, device)
    check_cross(q, k, v, f"H={H} G={G} M={M}")


# few rows against many keys: the keys are cut over workgroups and their partial results joined
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("L, M, N", [(1, 1, 5000), (2, 1, 4097), (1, 200, 3001)])
def test_cut_over_keys(device, dtype, L, M, N):
    q, k, v = operands(L, M, N, 4, 2, 64, 64, dtype, device)
    check_cross(q, k, v, f"L={L} M={M} N={N}")
    kermac.set_max_scratch_bytes(0)
    try:
        check_cross(q, k, v, f"uncut L={L} M={M} N={N}")
    finally:
        kermac.set_max_scratch_bytes(None)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("M", [1, 50, 140])
def test_key_lengths(device, dtype, M):
    """Lengths of zero, one, inside and at tiles, beyond the last key; what stands behind them is not a number."""
    lengths = torch.tensor([0, 1, 31, 32, 33, 64, 100, 257, 300, 1000, -5], dtype=torch.int32)
    N = 300
    q, k, v = operands(len(lengths), M, N, 2, 1, 64, 64, dtype, device)
    behind = torch.arange(N)[None] >= lengths[:, None]
    k[behind], v[behind] = math.nan, math.inf
    out = check_cross(q, k, v, f"M={M}", key_lengths=lengths.to(device))
    assert out[0].eq(0).all() and out[-1].eq(0).all()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("M", [1, 50, 140])
@pytest.mark.parametrize("kind", ["scattered", "left", "none", "one", "shared"])
def test_key_mask(device, dtype, M, kind):
    L, N = 3, 333
    mask = torch.rand(L, N, generator=torch.Generator().manual_seed(5)) < 0.7
    if kind == "left":
        mask = torch.arange(N)[None] >= torch.tensor([[0], [70], [332]])
    elif kind == "none":
        mask = torch.zeros(L, N, dtype=torch.bool)
        mask[1] = True
    elif kind == "one":
        mask = torch.zeros(L, N, dtype=torch.bool)
        mask[0, 0] = mask[1, 100] = mask[2, N - 1] = True
    elif kind == "shared":
        mask = mask[1]
    q, k, v = operands(L, M, N, 4, 4, 64, 64, dtype, device)
    if kind != "shared":
        k[~mask], v[~mask] = math.inf, math.nan
    check_cross(q, k, v, kind, key_mask=mask.to(device))
    lengths = torch.tensor([200, 333, 10], dtype=torch.int32, device=device)
    check_cross(q, k, v, kind + " and lengths", key_mask=mask.to(device), key_lengths=lengths)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_strides(device, dtype):
    """Heads in front of tokens, halves of one projection, a strided mask, a shared source, expanded queries, a result inside a larger tensor."""
    L, M, N, H, G, K = 3, 40, 100, 4, 2, 64
    q = normal(L, H, M, K, dtype=dtype, seed=1).to(device).transpose(1, 2)
    both = normal(L, N, 2, G, K, dtype=dtype, seed=2).to(device)
    mask = (torch.rand(N, L, generator=torch.Generator().manual_seed(5)) < 0.7).to(device).t()
    buffer = torch.full((L, M + 2, H, K + 8), 7.0, dtype=dtype, device=device)
    out = buffer[:, 1:-1, :, :K]
    assert check_cross(q, both[:, :, 0], both[:, :, 1], "views", key_mask=mask, out=out) is out
    assert buffer[:, 0].eq(7).all() and buffer[:, -1].eq(7).all() and buffer[..., K:].eq(7).all()
    # a source for the whole batch, queries that are one token seen by all entries, rows that start at odd addresses
    q1, k1, v1 = operands(1, 1, N, H, G, K, K, dtype, device)
    check_cross(q1.expand(L, M, H, K), k1, v1, "expanded")
    odd = normal(L, N, G, K + 1, dtype=dtype, seed=4).to(device)
    check_cross(q, odd[..., 1:], odd[..., :K], "odd addresses")


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("scale", [0.0, -0.125, 0.3, 1e-30])
@pytest.mark.parametrize("M", [1, 40])
def test_scale(device, dtype, scale, M):
    q, k, v = operands(2, M, 77, 2, 2, 64, 64, dtype, device)
    lengths = torch.tensor([50, 0], dtype=torch.int32, device=device)
    check_cross(q, k, v, f"scale={scale}", scale=scale, key_lengths=lengths)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("M", [1, 40])
def test_scores_that_grow(device, dtype, M):
    """Every tile's scores far above those before: the running maximum moves by hundreds, all weight ends up on the last keys."""
    q, k, v = operands(1, M, 400, 2, 2, 64, 64, dtype, device)
    q = q.abs()
    k = k.abs() * torch.linspace(0.1, 8.0, 400, device=device).to(dtype)[None, :, None, None]
    check_cross(q, k, v, "growing")
    check_cross(q, k.flip(1), v, "falling")


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_nothing_to_do(device, dtype):
    q, k, v = operands(2, 5, 7, 2, 2, 64, 32, dtype, device)
    assert kermac.cross_attention(q[:, :0], k, v).shape == (2, 0, 2, 32)
    assert kermac.cross_attention(q[:0], k[:0], v[:0]).shape == (0, 5, 2, 32)
    out, lse = kermac.cross_attention(q, k[:, :0], v[:, :0], return_lse=True)
    assert out.eq(0).all() and lse.eq(-math.inf).all()
    out = kermac.cross_attention(q[0], k[0], v[0])
    assert torch.equal(out, kermac.cross_attention(q[:1], k[:1], v[:1])) and out.shape == (1, 5, 2, 32)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("where", ["query", "key", "value"])
def test_not_a_number_stays(device, dtype, where):
    q, k, v = operands(1, 3, 200, 1, 1, 64, 64, dtype, device)
    {"query": q[0, 1], "key": k[0, 150], "value": v[0, 150]}[where].fill_(math.nan)
    out = kermac.cross_attention(q, k, v)
    rows = [1] if where == "query" else [0, 1, 2]
    assert out[0, rows].isnan().all() and out.isnan().sum() == len(rows) * 64


# ------------------------------------------------------------------------------------------------ prefix

def check_prefix(q, pk, pv, k, v, lengths, what, scale=None, **more):
    out = kermac.prefix_attention(q, pk, pv, k, v, lengths, scale=scale, **more)
    truth, bound = reference.prefix(q, pk, pv, k, v, lengths, q.shape[-1] ** -0.5 if scale is None else scale)
    reference.assert_within(out, truth, bound, what)
    return out


def prefix_operands(L, M, P, N, H, G, K, O, dtype, device):
    q, k, v = operands(L, M, N, H, G, K, O, dtype, device)
    return q, normal(P, G, K, dtype=dtype, seed=4).to(device), normal(P, G, O, dtype=dtype, seed=5).to(device), k, v


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("L, M, P, N", [(1, 1, 1, 1), (3, 1, 100, 40), (5, 1, 1000, 300), (4, 7, 65, 50), (2, 100, 300, 150), (40, 1, 31, 70),
                                        (2, 1, 0, 50), (3, 2, 50, 0)])
def test_prefix_lengths(device, dtype, L, M, P, N):
    q, pk, pv, k, v = prefix_operands(L, M, P, N, 4, 2, 64, 64, dtype, device)
    lengths = torch.randint(0, N + 1, (L,), generator=torch.Generator().manual_seed(6), dtype=torch.int32)
    behind = torch.arange(N)[None] >= lengths[:, None]
    k[behind], v[behind] = math.nan, math.nan
    check_prefix(q, pk, pv, k, v, lengths.to(device), f"L={L} M={M} P={P} N={N}")
    kermac.set_max_scratch_bytes(0)
    try:
        check_prefix(q, pk, pv, k, v, lengths.to(device), f"one pass, L={L} M={M} P={P} N={N}")
    finally:
        kermac.set_max_scratch_bytes(None)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("H, G, K, O", [(8, 1, 128, 128), (5, 5, 80, 40), (40, 1, 64, 64), (12, 3, 256, 256), (2, 1, 33, 7)])
@pytest.mark.parametrize("M", [1, 9])
def test_prefix_heads_and_features(device, dtype, H, G, K, O, M):
    q, pk, pv, k, v = prefix_operands(3, M, 200, 77, H, G, K, O, dtype, device)
    lengths = torch.tensor([77, 5, 200], dtype=torch.int32, device=device)
    check_prefix(q, pk, pv, k, v, lengths, f"H={H} G={G} K={K} O={O} M={M}", scale=-0.2)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_prefix_of_a_generation(device, dtype):
    """A prompt behind the prefix and tokens one by one, in a cache of heads in front of tokens: each step what the whole sequence gives."""
    L, P, N, H, G, K = 2, 150, 40, 4, 2, 64
    q, pk, pv, k, v = prefix_operands(L, N, P, N, H, G, K, K, dtype, device)
    cache_k, cache_v = (torch.full((L, G, N, K), math.nan, dtype=dtype, device=device).transpose(1, 2) for _ in range(2))
    whole = check_prefix(q, pk, pv, k, v, torch.full((L,), N, dtype=torch.int32, device=device), "whole")
    at = 0
    for step in (30, 1, 1, 5, 1, 2):
        cache_k[:, at:at + step], cache_v[:, at:at + step] = k[:, at:at + step], v[:, at:at + step]
        at += step
        lengths = torch.full((L,), at, dtype=torch.int32, device=device)
        out = check_prefix(q[:, at - step:at].contiguous(), pk, pv, cache_k, cache_v, lengths, f"step to {at}")
        # both are within one bound of the same truth
        assert torch.allclose(out.double(), whole[:, at - step:at].double(), rtol=8 * reference.UNIT[dtype], atol=8 * reference.UNIT[dtype] * 4)
    assert at == N


@pytest.mark.parametrize("dtype", TYPES[:2], ids=str)
@pytest.mark.parametrize("M", [1, 8, 40, 300])
@pytest.mark.parametrize("scale", [None, 0.3, -7.0])
def test_one_key_is_its_value(device, dtype, M, scale):
    """A softmax over one key is 1: the values come back bit for bit, alone, behind masked keys and through a length.

    Its weight is 1 up to fp32's rounding of the exponent (|scale q k| below 2^9 here, so off by less than 2^-14), which is less than
    half a step beside 1 of either type, and so is what the division by the sum leaves beside the value before it is rounded.
    """
    q, k, v = operands(2, M, 200, 4, 2, 64, 64, dtype, device)
    one = v[:, :1].repeat_interleave(2, 2).expand(2, M, 4, 64)
    assert torch.equal(kermac.cross_attention(q, k[:, :1], v[:, :1], scale=scale), one)
    lengths = torch.ones(2, dtype=torch.int32, device=device)
    assert torch.equal(kermac.cross_attention(q, k, v, scale=scale, key_lengths=lengths), one)
    mask = torch.zeros(200, dtype=torch.bool, device=device)
    mask[150] = True
    assert torch.equal(kermac.cross_attention(q, k, v, scale=scale, key_mask=mask), v[:, 150:151].repeat_interleave(2, 2).expand(2, M, 4, 64))
    nothing = torch.zeros(2, dtype=torch.int32, device=device)
    assert torch.equal(kermac.prefix_attention(q, k[0, :1], v[0, :1], k, v, nothing, scale=scale), v[:1, :1].repeat_interleave(2, 2).expand(2, M, 4, 64))


def test_prefix_of_no_sequences(device):
    q, pk, pv, k, v = prefix_operands(1, 3, 50, 7, 4, 2, 64, 64, torch.bfloat16, device)
    lengths = torch.zeros(1, dtype=torch.int32, device=device)
    assert kermac.prefix_attention(q[:0], pk, pv, k[:0], v[:0], lengths[:0]).shape == (0, 3, 4, 64)
    assert kermac.prefix_attention(q[:, :0], pk, pv, k, v, lengths).shape == (1, 0, 4, 64)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("K, O", [(96, 80), (128, 128), (256, 200), (33, 7)])
@pytest.mark.parametrize("M", [1, 9, 150])
def test_masked_keys_of_any_width_may_hold_anything(device, dtype, K, O, M):
    """Keys left out one by one, whole tiles of them, and all of an entry: what they hold stays out, in aligned rows and in others."""
    L, N = 4, 500
    mask = torch.rand(L, N, generator=torch.Generator().manual_seed(8)) < 0.6
    mask[1, 40:333], mask[2] = False, False
    mask[3] = torch.arange(N) == 499
    for pad in (0, 1):
        q, k, v = operands(L, M, N, 4, 2, K + pad, O + pad, dtype, device)
        q, k, v = q[..., pad:], k[..., pad:], v[..., pad:]
        k[~mask], v[~mask] = math.nan, math.inf
        out = check_cross(q, k, v, f"pad={pad}", key_mask=mask.to(device))
        assert out[2].eq(0).all()
        check_cross(q, k, v, f"pad={pad} and lengths", key_mask=mask.to(device), key_lengths=torch.tensor([350, 500, 2, 0], dtype=torch.int32, device=device))
