"""Attention operators as programs run them: in captured graphs, on other streams, in a caller's scratch memory, in caches whose offsets pass 32 bits, and in
a training step."""
import math

import pytest
import torch

import kermac_amd as kermac
from tests import attention_reference as reference
from tests.helpers import kernels_of
from tests.test_attention_gpu import TYPES, check_cross, normal, operands, prefix_operands

pytestmark = pytest.mark.gpu


def calls(dtype, device):
    """{name: (inputs, a function of nothing that returns a tuple of results)}: cut and uncut launches of every operator."""
    made = {}
    for name, (L, M, N) in dict(cut=(2, 1, 3000), rows=(2, 150, 700), small=(1, 3, 5)).items():
        q, k, v = operands(L, M, N, 4, 2, 64, 64, dtype, device)
        lengths = torch.full((L,), N - 1, dtype=torch.int32, device=device)
        grad_out = normal(L, M, 4, 64, dtype=dtype, seed=9).to(device)

        def step(q=q, k=k, v=v, lengths=lengths, grad_out=grad_out):
            out, lse = kermac.cross_attention(q, k, v, key_lengths=lengths, return_lse=True)
            return (out, lse, *kermac.cross_attention_grad(grad_out, q, k, v, out, lse, key_lengths=lengths))

        made[f"step {name}"] = ((q, k, v, grad_out), step)
    q, pk, pv, k, v = prefix_operands(3, 2, 2000, 300, 4, 2, 64, 64, dtype, device)
    lengths = torch.tensor([300, 7, 150], dtype=torch.int32, device=device)
    made["prefix"] = ((q, pk, pv, k, v), lambda: (kermac.prefix_attention(q, pk, pv, k, v, lengths),))
    return made


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_captured_and_replayed(device, dtype):
    """A graph replayed on new values, eager work and synchronisations in between, gives the bits of the eager calls every time."""
    for name, (inputs, call) in calls(dtype, device).items():
        call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            results = call()
        for turn in range(4):
            for x in inputs:
                x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(100 + turn)).to(dtype))
            graph.replay()
            torch.cuda.synchronize()
            got = [r.clone() for r in results]
            expected = call()
            torch.cuda.synchronize()
            for i, (a, b) in enumerate(zip(got, expected)):
                assert torch.equal(a, b), f"{name}, replay {turn}, result {i}"


def test_two_graphs_one_after_the_other(device):
    """Two captured graphs with workspaces of their own, replayed in turns."""
    made = list(calls(torch.bfloat16, device).values())[:2]
    expected = [call() for _, call in made]
    graphs = []
    for _, call in made:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            results = call()
        graphs.append((graph, results))
    for _ in range(3):
        for graph, _ in graphs:
            graph.replay()
    torch.cuda.synchronize()
    for (_, results), truth in zip(graphs, expected):
        assert all(torch.equal(a, b) for a, b in zip(results, truth))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_another_stream(device, dtype):
    for name, (inputs, call) in calls(dtype, device).items():
        expected = call()
        torch.cuda.synchronize()
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for x in inputs:
                x.mul_(1.0)                     # the operators follow in this stream's order
            results = call()
        stream.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(results, expected)), name


def test_a_callers_scratch_memory(device):
    """Workspaces from the caller's buffer, whatever it holds; a buffer that is too small for cuts costs only the cuts."""
    q, k, v = operands(2, 1, 3000, 4, 2, 64, 64, torch.bfloat16, device)
    grad_out = normal(2, 1, 4, 64, dtype=torch.bfloat16, seed=9).to(device)
    out, lse = kermac.cross_attention(q, k, v, return_lse=True)
    grads = kermac.cross_attention_grad(grad_out, q, k, v, out, lse)
    big, small = (torch.full((n,), 255, dtype=torch.uint8, device=device) for n in (64 << 20, 1024))
    with kermac.scratch(big):
        assert torch.equal(kermac.cross_attention(q, k, v), out)
        assert all(torch.equal(a, b) for a, b in zip(kermac.cross_attention_grad(grad_out, q, k, v, out, lse), grads))
        names = kernels_of(lambda: kermac.cross_attention(q, k, v))
        assert any("attention_join" in name for name in names)
    with kermac.scratch(small):
        names = kernels_of(lambda: check_cross(q, k, v, "small buffer"))
        assert not any("attention_join" in name for name in names)
        kermac.cross_attention_grad(grad_out, q, k, v, out, lse)
    with kermac.scratch(small[:64]), pytest.raises(RuntimeError, match="scratch"):
        kermac.cross_attention_grad(grad_out, q, k, v, out, lse)


@pytest.mark.parametrize("token_stride, N", [(1 << 22, 600), (1 << 26, 40)], ids=["aligned", "far apart"])
@pytest.mark.parametrize("M", [1, 40])
def test_offsets_beyond_32_bits(device, token_stride, N, M):
    """Keys whose last tokens stand more than 2^31 elements behind the first: 5 GB of a cache, of which the tokens alone are written."""
    K = 64
    cache = torch.empty(N * token_stride, dtype=torch.bfloat16, device=device)
    k, v = cache.as_strided((1, N, 1, K), (0, token_stride, K, 1)), cache.as_strided((1, N, 1, K), (0, token_stride, K, 1), K)
    assert (N - 1) * token_stride > 1 << 31
    q, dense_k, dense_v = operands(1, M, N, 2, 1, K, K, torch.bfloat16, device)
    k.copy_(dense_k)
    v.copy_(dense_v)
    out, lse = kermac.cross_attention(q, k, v, return_lse=True)
    dense, dense_lse = kermac.cross_attention(q, dense_k, dense_v, return_lse=True)
    assert torch.equal(out, dense) and torch.equal(lse, dense_lse)
    lengths = torch.tensor([N], dtype=torch.int32, device=device)
    check = kermac.prefix_attention(q, k[0], v[0], dense_k, dense_v, lengths)
    assert torch.equal(check, kermac.prefix_attention(q, dense_k[0], dense_v[0], dense_k, dense_v, lengths))
    for a, b in zip(kermac.cross_attention_grad(out, q, k, v, out, lse), kermac.cross_attention_grad(out, q, dense_k, dense_v, out, lse)):
        assert torch.equal(a, b)


def test_a_single_token_of_any_stride(device):
    """The stride of a dimension of one token means nothing, 0 included, and an infinite value of it stays one."""
    q, k, v = operands(1, 2, 1, 2, 2, 64, 64, torch.float32, device)
    v.fill_(math.inf)
    odd_k, odd_v = (x.as_strided(x.shape, (0, 0, 64, 1)) for x in (k, v))
    assert kermac.cross_attention(q, odd_k, odd_v).eq(math.inf).all()
    q1 = q[:, :1].as_strided((1, 1, 2, 64), (0, 0, 64, 1))
    v.normal_()
    out, lse = kermac.cross_attention(q1, k, v, return_lse=True)
    for a, b in zip(kermac.cross_attention_grad(out, q1, odd_k, odd_v, out, lse), kermac.cross_attention_grad(out.clone(), q1.contiguous(), k, v, out, lse)):
        assert torch.equal(a, b)


def test_a_training_step_of_a_layer(device):
    """Decoder states attend to an encoder's: projections by torch, attention and its gradient by the operators.  The projections' gradients
    against those of the whole layer in 64 bits by autograd."""
    L, M, N, width, H, G, D = 3, 21, 50, 96, 4, 2, 32
    decoder, encoder = normal(L, M, width, dtype=torch.float32, seed=1).to(device), normal(L, N, width, dtype=torch.float32, seed=2).to(device)
    w_q, w_k, w_v = (normal(width, heads * D, dtype=torch.float32, seed=3 + i).to(device) * width ** -0.5 for i, heads in enumerate((H, G, G)))
    lengths = torch.tensor([50, 33, 1], dtype=torch.int32, device=device)
    target = normal(L, M, H, D, dtype=torch.float32, seed=7).to(device)

    q, k, v = (decoder @ w_q).unflatten(-1, (H, D)), (encoder @ w_k).unflatten(-1, (G, D)), (encoder @ w_v).unflatten(-1, (G, D))
    out, lse = kermac.cross_attention(q, k, v, key_lengths=lengths, return_lse=True)
    grad_q, grad_k, grad_v = kermac.cross_attention_grad(out - target, q, k, v, out, lse, key_lengths=lengths)      # of half the squared distance
    grads = [x.flatten(0, 1).t() @ g.flatten(2).flatten(0, 1) for x, g in ((decoder, grad_q), (encoder, grad_k), (encoder, grad_v))]

    weights = [w.cpu().double().requires_grad_() for w in (w_q, w_k, w_v)]
    states = [x.cpu().double() for x in (decoder, encoder, encoder)]
    rows, keys, values = (x @ w for x, w in zip(states, weights))
    rows = rows.unflatten(-1, (H, D)).transpose(1, 2)
    keys, values = (x.unflatten(-1, (G, D)).repeat_interleave(H // G, 2).transpose(1, 2) for x in (keys, values))
    keep = reference.keep_of(L, M, N, lengths)
    scores = (rows @ keys.transpose(2, 3) * D ** -0.5).masked_fill(~keep[:, None], -math.inf)
    distance = ((torch.softmax(scores, -1) @ values).transpose(1, 2) - target.cpu().double()).square().sum() / 2
    distance.backward()
    # every product of the layer is a sum of at most `width`, L M or L N terms in fp32 (2^-24 each), and six of them stand behind one another
    for name, got, weight in zip("qkv", grads, weights):
        error = (got.cpu().double() - weight.grad).norm() / weight.grad.norm()
        assert error < 6 * math.sqrt(max(width, L * N)) * 2.0 ** -24 * 8, (name, error.item())


@pytest.mark.parametrize("L, M, P, N", [(2, 5, 100, 40), (1, 70, 30, 90)])
def test_a_prefix_through_the_c_abi_is_causal_by_itself(device, L, M, P, N):
    """A C caller who sets prefix_n alone gets what one gets who sets causal too: no query meets the tokens behind it."""
    from kermac_amd import _backend
    from kermac_amd.attention import _plan_attention
    q, pk, pv, k, v = prefix_operands(L, M, P, N, 4, 2, 64, 64, torch.bfloat16, device)
    lengths = torch.full((L,), N - 3, dtype=torch.int32, device=device)
    plan = _plan_attention(q, k, v, torch.empty_like(q), None, lengths, None, False, prefix=(pk, pv))
    params = plan.params
    params.causal = 0
    _backend.attention(params, torch.cuda.current_stream().cuda_stream)
    truth, bound = reference.prefix(q, pk, pv, k, v, lengths, 64 ** -0.5)
    reference.assert_within(plan.out, truth, bound, "prefix_n alone")


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32], ids=str)
def test_more_workgroups_than_a_launch_holds(device, dtype):
    """2^24 workgroups of 256 threads are one more than a grid takes: the first, the last and the entries around the border of the launches are looked at."""
    L, N, K = (1 << 24) + 77, 3, 8
    q = torch.randn(L, 1, 1, K, device=device, dtype=dtype, generator=torch.Generator(device=device).manual_seed(1))
    k, v = normal(1, N, 1, K, dtype=dtype, seed=2).to(device), normal(1, N, 1, K, dtype=dtype, seed=3).to(device)
    out, lse = kermac.cross_attention(q, k, v, return_lse=True)
    grads = kermac.cross_attention_grad(out, q, k, v, out, lse)
    border = (1 << 24) - 8
    for some in (slice(0, 50), slice(border // 8 - 20, border // 8 + 20), slice(border - 20, border + 20), slice(L - 50, L)):
        part, part_lse = kermac.cross_attention(q[some], k, v, return_lse=True)
        assert torch.equal(out[some], part) and torch.equal(lse[some], part_lse)
        # (a row's gradient of its query is its own)
        assert torch.equal(grads[0][some], kermac.cross_attention_grad(part, q[some], k, v, part, part_lse)[0])
    scores = (q.double() * K ** -0.5 @ k[0, :, 0].double().t()).squeeze(2)
    truth = torch.softmax(scores, -1) @ v[0, :, 0].double()
    unit = reference.UNIT[dtype]
    assert ((out.double() - truth[:, :, None].reshape(out.shape)).abs() <= 2 * unit * v.double().abs().max() + 2.0 ** -18).all()


def test_more_rows_than_a_launch_of_the_join_holds(device):
    """2^26 rows, whose parts one wave each joins, behind a prefix that all of them share."""
    L, M, P, N, K = 2, (1 << 25) + 3, 5, 2, 8
    make = torch.Generator(device=device).manual_seed(1)
    q = torch.randn(L, M, 1, K, device=device, dtype=torch.float16, generator=make)
    pk, pv = normal(P, 1, K, dtype=torch.float16, seed=4).to(device), normal(P, 1, K, dtype=torch.float16, seed=5).to(device)
    k, v = normal(L, N, 1, K, dtype=torch.float16, seed=2).to(device), normal(L, N, 1, K, dtype=torch.float16, seed=3).to(device)
    lengths = torch.tensor([0, 2], dtype=torch.int32, device=device)
    out = kermac.prefix_attention(q, pk, pv, k, v, lengths)
    # the queries in front of an entry's own tokens meet the prefix alone
    shared = kermac.cross_attention(q.reshape(1, L * M, 1, K), pk, pv).reshape(L, M, 1, K)
    far = 2 * reference.UNIT[torch.float16] * pv.float().abs().max()
    assert ((out[:, :-2].float() - shared[:, :-2].float()).abs() <= far).all()
    last = kermac.prefix_attention(q[:, -2:].contiguous(), pk, pv, k, v, lengths)
    assert ((out[:, -2:].float() - last.float()).abs() <= 2 * reference.UNIT[torch.float16] * max(pv.float().abs().max(), v.float().abs().max())).all()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("M, N", [(3, 5000), (200, 3001)])
def test_not_a_number_stays_in_parts(device, dtype, M, N):
    """Rows whose scores are all NaN, in every part that the keys are cut into, and keys whose score is NaN or infinite in one of them."""
    q, k, v = operands(2, M, N, 2, 2, 64, 64, dtype, device)
    q[0, 1] = math.nan
    names = kernels_of(lambda: kermac.cross_attention(q, k, v))
    assert any("attention_join" in name for name in names)
    out, lse = kermac.cross_attention(q, k, v, return_lse=True)
    assert out[0, 1].isnan().all() and lse[0, 1].isnan().all() and out.isnan().sum() == 2 * 64
    prefixed = kermac.prefix_attention(q, k[0], v[0], k, v, torch.zeros(2, dtype=torch.int32, device=device))
    assert prefixed[0, 1].isnan().all() and prefixed.isnan().sum() == 2 * 64
    q[0, 1] = 1.0
    for value in (math.nan, math.inf):
        k[1, N - 2] = value                     # (infinity: the scores of the entry's rows are infinities of their sums' signs, or NaN)
        out = kermac.cross_attention(q.abs() + 0.1, k, v)
        assert out[1].isnan().all() and not out[0].isnan().any()
