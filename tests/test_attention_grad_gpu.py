"""The gradient of cross attention against its formulas in 64 bits, against differences, and against itself."""
import math

import pytest
import torch

import kermac_amd as kermac
from tests import attention_reference as reference
from tests.test_attention_gpu import TYPES, normal, operands

pytestmark = pytest.mark.gpu


def step(grad_out, q, k, v, **masks):
    out, lse = kermac.cross_attention(q, k, v, return_lse=True, **masks)
    return kermac.cross_attention_grad(grad_out, q, k, v, out, lse, **masks)


def check(q, k, v, what, scale=None, key_lengths=None, key_mask=None, grad_out=None):
    L, M, H, K = q.shape
    N, O = v.shape[1], v.shape[3]
    if grad_out is None:
        grad_out = normal(L, M, H, O, dtype=q.dtype, seed=9).to(q.device)
    grads = step(grad_out, q, k, v, scale=scale, key_lengths=key_lengths, key_mask=key_mask)
    truth, bounds = reference.gradients(grad_out, q, k, v, reference.keep_of(L, M, N, key_lengths, key_mask), K ** -0.5 if scale is None else scale)
    for name, got, of, expected, bound in zip(("queries", "keys", "values"), grads, (q, k, v), truth, bounds):
        assert got.shape == of.shape and got.dtype == of.dtype and got.is_contiguous()
        reference.assert_within(got, expected, bound, f"{what} grad of {name}")
    return grads


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("M, N", [(1, 1), (1, 33), (2, 64), (31, 65), (33, 31), (129, 127), (40, 200), (300, 520)])
def test_lengths(device, dtype, M, N):
    check(*operands(2, M, N, 2, 2, 64, 64, dtype, device), f"M={M} N={N}")


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("K, O", [(1, 1), (7, 5), (16, 40), (80, 80), (96, 128), (128, 64), (128, 128), (200, 72), (256, 256), (251, 3)])
def test_features(device, dtype, K, O):
    check(*operands(1, 70, 150, 4, 2, K, O, dtype, device), f"K={K} O={O}")


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("H, G, M", [(8, 1, 1), (40, 1, 1), (33, 1, 3), (6, 2, 5), (20, 4, 17), (3, 3, 40)])
def test_shared_heads(device, dtype, H, G, M):
    check(*operands(3, M, 90, H, G, 64, 64, dtype, device), f"H={H} G={G} M={M}")


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("kind", ["all", "lengths", "holes"])
def test_one_source_for_the_batch(device, dtype, kind):
    """Keys and values of batch size 1: their gradient is the sum over the entries, each with keys of its own left out."""
    L, N = 5, 150
    q, k, v = operands(L, 40, N, 4, 2, 64, 64, dtype, device, key_batch=1)
    lengths = torch.tensor([150, 0, 1, 149, 77], dtype=torch.int32, device=device) if kind == "lengths" else None
    mask = (torch.rand(L, N, generator=torch.Generator().manual_seed(5)) < 0.5).to(device) if kind == "holes" else None
    check(q, k, v, kind, key_lengths=lengths, key_mask=mask)
    grads = step(q, q, k[0], v[0], key_lengths=lengths, key_mask=mask)
    assert grads[1].shape == k[0].shape and grads[2].shape == v[0].shape


# few rows against many keys, and many rows against few: the work is cut and partial sums are added in a fixed order
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("L, M, N, key_batch", [(1, 3, 3001, 1), (1, 1500, 5, 1), (1, 300, 1000, 1), (6, 130, 40, 1)])
def test_cut(device, dtype, L, M, N, key_batch):
    q, k, v = operands(L, M, N, 4, 2, 64, 64, dtype, device, key_batch=key_batch)
    first = check(q, k, v, "cut")
    again = check(q, k, v, "again")
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    kermac.set_max_scratch_bytes((8 * L * M * 4 + 8 + 15) // 16 * 16)
    try:
        check(q, k, v, "uncut")
        out, lse = kermac.cross_attention(q, k, v, return_lse=True)
        kermac.set_max_scratch_bytes(0)
        with pytest.raises(RuntimeError, match="scratch"):
            kermac.cross_attention_grad(q, q, k, v, out, lse)
    finally:
        kermac.set_max_scratch_bytes(None)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_key_lengths(device, dtype):
    lengths = torch.tensor([0, 1, 31, 32, 33, 64, 100, 128, 129, 257, 300, 1000, -5], dtype=torch.int32)
    L, N = len(lengths), 300
    q, k, v = operands(L, 50, N, 2, 1, 64, 64, dtype, device)
    behind = torch.arange(N)[None] >= lengths[:, None]
    k[behind], v[behind] = math.nan, math.inf
    grads = check(q, k, v, "lengths", key_lengths=lengths.to(device))
    assert grads[0][0].eq(0).all() and grads[1].cpu()[behind].eq(0).all() and grads[2].cpu()[behind].eq(0).all()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("kind", ["scattered", "left", "none", "one"])
def test_key_mask(device, dtype, kind):
    L, N = 3, 333
    mask = torch.rand(L, N, generator=torch.Generator().manual_seed(5)) < 0.7
    if kind == "left":
        mask = torch.arange(N)[None] >= torch.tensor([[0], [170], [332]])
    elif kind == "none":
        mask = torch.zeros(L, N, dtype=torch.bool)
        mask[1] = True
    elif kind == "one":
        mask = torch.zeros(L, N, dtype=torch.bool)
        mask[0, 0] = mask[1, 200] = mask[2, N - 1] = True
    q, k, v = operands(L, 140, N, 4, 4, 64, 64, dtype, device)
    k[~mask], v[~mask] = math.inf, math.nan
    check(q, k, v, kind, key_mask=mask.to(device))
    check(q, k, v, kind + " and lengths", key_mask=mask.to(device), key_lengths=torch.tensor([200, 333, 10], dtype=torch.int32, device=device))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("scale", [0.0, -0.125, 0.3])
def test_scale(device, dtype, scale):
    check(*operands(2, 40, 77, 2, 2, 64, 64, dtype, device), f"scale={scale}", scale=scale)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_strides(device, dtype):
    L, M, N, H, G, K = 3, 40, 100, 4, 2, 64
    q = normal(L, H, M, K, dtype=dtype, seed=1).to(device).transpose(1, 2)
    both = normal(L, N, 2, G, K, dtype=dtype, seed=2).to(device)
    mask = (torch.rand(N, L, generator=torch.Generator().manual_seed(5)) < 0.7).to(device).t()
    grad_out = normal(1, 1, H, K, dtype=dtype, seed=3).to(device).expand(L, M, H, K)
    check(q, both[:, :, 0], both[:, :, 1], "views", key_mask=mask, grad_out=grad_out)
    odd = normal(L, N, G, K + 1, dtype=dtype, seed=4).to(device)
    check(q, odd[..., 1:], odd[..., :K], "odd addresses")


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_nothing_to_do(device, dtype):
    q, k, v = operands(2, 5, 7, 2, 2, 64, 32, dtype, device)
    grads = step(torch.empty(2, 0, 2, 32, dtype=dtype, device=device), q[:, :0], k, v)
    assert [g.shape for g in grads] == [(2, 0, 2, 64), k.shape, v.shape] and grads[1].eq(0).all() and grads[2].eq(0).all()
    grads = step(torch.ones(2, 5, 2, 32, dtype=dtype, device=device), q, k[:, :0], v[:, :0])
    assert [g.shape for g in grads] == [q.shape, (2, 0, 2, 64), (2, 0, 2, 32)] and grads[0].eq(0).all()


def test_against_differences(device):
    """fp32 gradients along random directions against central differences of the definition in 64 bits.  The difference with half the
    step is off by at most what it differs from the one with the whole step, plus 64-bit rounding."""
    L, M, N, H, G, K, O = 2, 9, 37, 4, 2, 24, 16
    q, k, v = operands(L, M, N, H, G, K, O, torch.float32, device)
    grad_out = normal(L, M, H, O, dtype=torch.float32, seed=9).to(device)
    lengths = torch.tensor([37, 20], dtype=torch.int32, device=device)
    keep = reference.keep_of(L, M, N, lengths)
    grads = step(grad_out, q, k, v, key_lengths=lengths)
    _, bounds = reference.gradients(grad_out, q, k, v, keep, K ** -0.5)
    exact = [x.cpu().double() for x in (q, k, v)]
    weights = grad_out.cpu().double()

    def value(at):
        rows = at[0].transpose(1, 2)
        keys, values = (x.repeat_interleave(H // G, 2).transpose(1, 2) for x in at[1:])
        s = (torch.matmul(rows, keys.transpose(2, 3).contiguous()) * K ** -0.5).masked_fill(~keep[:, None], -math.inf)
        return (torch.matmul(torch.softmax(s, -1), values.contiguous()).transpose(1, 2) * weights).sum()

    for which in range(3):
        direction = torch.randn(exact[which].shape, generator=torch.Generator().manual_seed(20 + which), dtype=torch.float64)

        def difference(h):
            at = [[x + sign * h * direction if i == which else x for i, x in enumerate(exact)] for sign in (1, -1)]
            return (value(at[0]) - value(at[1])) / (2 * h)

        whole, half = difference(2e-4), difference(1e-4)
        got = (grads[which].cpu().double() * direction).sum()
        allowed = (bounds[which] * direction.abs()).sum() + (whole - half).abs() + 1e-11 * weights.abs().sum()
        assert (got - half).abs() <= allowed, (which, got.item(), half.item(), allowed.item())


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("K, O", [(64, 64), (128, 96), (200, 256), (33, 64)])
@pytest.mark.parametrize("kind", ["lengths", "holes", "both"])
def test_what_takes_no_part_may_hold_anything(device, dtype, K, O, kind):
    """Keys left out of every entry hold infinities and NaN, for entries with keys of their own and for a source that they share; those that one
    entry leaves out and another one meets are numbers.  M and the heads end inside tiles and parts."""
    L, M, N = 3, 45, 300
    lengths = torch.tensor([290, 129, 7], dtype=torch.int32) if kind != "holes" else None
    mask = torch.rand(L, N, generator=torch.Generator().manual_seed(8)) < 0.4 if kind != "lengths" else None
    keep = reference.keep_of(L, 1, N, lengths, mask)[:, 0]
    for key_batch in (L, 1):
        q, k, v = operands(L, M, N, 6, 2, K, O, dtype, device, key_batch=key_batch)
        unused = ~keep if key_batch == L else ~keep.any(0, keepdim=True)
        k[unused], v[unused] = math.nan, math.inf
        masks = dict(key_lengths=None if lengths is None else lengths.to(device), key_mask=None if mask is None else mask.to(device))
        grads = check(q, k, v, f"{kind} of {key_batch}", **masks)
        assert grads[1].cpu()[unused].eq(0).all() and grads[2].cpu()[unused].eq(0).all()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("K, O", [(64, 64), (80, 96), (128, 128), (128, 40), (256, 256)])
@pytest.mark.parametrize("M, N", [(5, 700), (200, 150), (333, 31)])
def test_rows_at_odd_addresses(device, dtype, K, O, M, N):
    """Rows that start and end between 16-byte pieces are read by elements, in kernels of their own."""
    q, k, v = (x[..., 1:] for x in operands(2, M, N, 4, 2, K + 1, O + 1, dtype, device))
    lengths = torch.tensor([N, N - 20], dtype=torch.int32, device=device)
    check(q, k, v, "odd", key_lengths=lengths)
    out = torch.empty(2, M, 4, O + 1, dtype=dtype, device=device)[..., 1:]
    assert torch.equal(kermac.cross_attention(q, k, v, out, key_lengths=lengths), kermac.cross_attention(q, k, v, key_lengths=lengths))
