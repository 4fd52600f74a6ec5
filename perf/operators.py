"""The calls that the speed of the attention operators is measured on, and the same operators in elementary torch operations.

Attention is a product of a kernel matrix with coefficients whose rows are normalised: the matrix is
``exp(scale <query, key>)``, every row is divided by its sum, the values are the coefficients.  Three operators:

* ``cross``: queries of one length against the keys and values of another sequence (an encoder's states);
* ``cross_grad``: the same with its gradient, as one training step runs them;
* ``prefix``: a batch whose sequences all continue one long prefix, each from keys and values of its own behind it.

A case is a plain dict: ``L`` batch entries, ``M`` queries and ``N`` keys each, ``H`` query heads on ``G`` heads of
keys and values, ``K`` features of queries and keys and ``O`` of values, ``P`` keys of the shared prefix.  ``mask``: all
keys take part (``"none"``), every batch entry has a length (``"lengths"``), or a truth value per key (``"holes"``).
``layout``: the storage of keys and values, ``"tokens"`` ([L, N, G, K]) or ``"heads"`` ([L, G, N, K]).  ``shared``: one
set of keys and values for the whole batch (several candidates that answer one source).
"""
import math
import random

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # The next token of one sequence against a short source: nothing but latency.
        dict(name="cross_one_token_short", op="cross", dtype="fp16", L=1, M=1, N=100, H=8, G=8, K=64, O=64, mask="none", layout="tokens"),
        # The next token of a batch of 32 against padded sources of up to 4000 states: bound by reading keys and values.
        dict(name="cross_one_token_batch", op="cross", dtype="bf16", L=32, M=1, N=4000, H=16, G=16, K=64, O=64, mask="lengths", layout="tokens"),
        # An ordinary batch of ragged sources in single precision, keys left out one by one.
        dict(name="cross_fp32_holes", op="cross", dtype="fp32", L=2, M=1000, N=2900, H=8, G=8, K=64, O=64, mask="holes", layout="tokens"),
        # A long document against a longer one, four query heads on each head of keys.
        dict(name="cross_large", op="cross", dtype="bf16", L=8, M=4096, N=8192, H=32, G=8, K=128, O=128, mask="none", layout="tokens"),
        # A small training step, as at the end of a data set.
        dict(name="grad_small", op="cross_grad", dtype="bf16", L=2, M=100, N=200, H=8, G=8, K=64, O=64, mask="lengths", layout="tokens"),
        # An ordinary training step: padded sources, as many heads of keys as of queries.
        dict(name="grad_medium", op="cross_grad", dtype="bf16", L=8, M=1000, N=1500, H=16, G=16, K=64, O=64, mask="lengths", layout="tokens"),
        # A training step in single precision, sizes that are no multiples of anything.
        dict(name="grad_fp32", op="cross_grad", dtype="fp32", L=2, M=777, N=1333, H=8, G=4, K=80, O=80, mask="none", layout="tokens"),
        # A training step on long sequences with shared heads.
        dict(name="grad_large", op="cross_grad", dtype="bf16", L=4, M=4096, N=4096, H=32, G=8, K=128, O=128, mask="none", layout="tokens"),
        # Four sequences behind a short common instruction: latency.
        dict(name="prefix_few", op="prefix", dtype="bf16", L=4, M=1, P=1000, N=100, H=16, G=4, K=128, O=128, layout="tokens"),
        # The next token of 64 sequences that share 8192 tokens and have up to 1000 of their own.
        dict(name="prefix_batch", op="prefix", dtype="bf16", L=64, M=1, P=8192, N=1000, H=32, G=8, K=128, O=128, layout="heads"),
        # The next token of 128 sequences that share a very long prefix.
        dict(name="prefix_long", op="prefix", dtype="bf16", L=128, M=1, P=65536, N=1024, H=32, G=8, K=128, O=128, layout="heads"),
        # 16 questions of up to 100 tokens each about one shared document.
        dict(name="prefix_questions", op="prefix", dtype="fp16", L=16, M=100, P=10000, N=300, H=16, G=4, K=128, O=128, layout="tokens"),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    """Another call of the same operators: sizes over the whole range, odd ones among them."""
    limit = max(_price(case) for case in listed())
    while True:
        op = rng.choice(("cross", "cross", "cross_grad", "cross_grad", "prefix", "prefix"))
        G = rng.choice((1, 2, 4, 8, 16))
        K = rng.choice((32, 64, 64, 80, 96, 128, 128, 256))
        case = dict(op=op, dtype=rng.choice(("bf16", "bf16", "fp16", "fp32")), L=_log_int(rng, 1, 128), H=G * rng.choice((1, 1, 2, 4, 5, 8)),
                    G=G, K=K, O=K if rng.random() < 0.8 else rng.choice((40, 64, 128)), layout=rng.choice(("tokens", "heads")))
        if op == "prefix":
            case.update(M=1 if rng.random() < 0.6 else _log_int(rng, 2, 300), P=_log_int(rng, 1, 65536))
            case.update(N=case["M"] + _log_int(rng, 1, 4096))
        else:
            single = op == "cross" and rng.random() < 0.4
            case.update(M=1 if single else _log_int(rng, 2, 8192), N=_log_int(rng, 1, 32768 if single else 8192),
                        mask=rng.choice(("none", "lengths", "lengths", "holes")), shared=rng.random() < 0.2)
        if _price(case) <= limit:
            return case


def _price(case):
    """Microseconds, roughly, in elementary operations: it only keeps drawn cases below the largest listed one."""
    rows, keys = case["L"] * case["M"] * case["H"], case["N"] + case.get("P", 0)
    passes = 3.5 if case["op"] == "cross_grad" else 1.0
    stored = case["L"] * case["N"] * case["G"] + case.get("P", 0) * case["G"]
    return passes * (rows * keys * (4e-8 * (case["K"] + case["O"]) + 1e-5) + 4e-6 * stored * (case["K"] + case["O"]))


def work(case):
    """Bytes that have to be read and written once, and operations of the products that have to be made, of one pass."""
    L, M, N, H, G, K, O = (case[name] for name in "LMNHGKO")
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "prefix":
        P = case["P"]
        own_keys = L * (0.75 * (N - M) + M)                               # lengths are spread over half the range
        seen = own_keys - L * (M - 1) / 2.0                               # a query does not see the tokens behind it
        return {"bytes": size * (L * M * H * (K + O) + (P + own_keys) * G * (K + O)), "flops": 2.0 * H * (K + O) * M * (L * P + seen)}
    part = {"none": 1.0, "lengths": 0.75, "holes": 0.8}[case["mask"]]
    read = part if case["mask"] == "lengths" else 1.0
    sources = 1 if case.get("shared") else L
    pairs = part * L * M * N * H
    tokens, stored = L * M * H * (K + O), sources * N * G * (K + O)
    if case["op"] == "cross":
        return {"bytes": size * (tokens + (stored if case.get("shared") else read * stored)), "flops": 2.0 * pairs * (K + O)}
    return {"bytes": size * (2 * tokens + L * M * H * O + 2 * stored), "flops": 2.0 * pairs * (4 * K + 3 * O)}


def prepare(case, seed):
    """Queries, keys, values and masks as a program holds them before the call."""
    device = torch.device("cuda")
    gen = torch.Generator(device=device)
    gen.manual_seed(seed)
    rng = random.Random(seed)
    dtype = _TYPES[case["dtype"]]
    L, M, N, H, G, K, O = (case[name] for name in "LMNHGKO")

    def normal(*shape):
        return torch.randn(*shape, device=device, generator=gen, dtype=dtype)

    def keys_and_values(batch, n):
        """[batch, n, G, K] and [batch, n, G, O]: one projection's two halves where the storage allows it."""
        if case["layout"] == "heads":
            return normal(batch, G, n, K).transpose(1, 2), normal(batch, G, n, O).transpose(1, 2)
        both = normal(batch, n, G * (K + O))
        return both[:, :, :G * K].unflatten(2, (G, K)), both[:, :, G * K:].unflatten(2, (G, O))

    state = dict(case=case, scale=K ** -0.5, q=normal(L, M, H, K))
    if case["op"] == "prefix":
        prefix_k, prefix_v = keys_and_values(1, case["P"])
        state.update(prefix_k=prefix_k[0], prefix_v=prefix_v[0])
        lengths = [M + rng.randint((N - M) // 2, N - M) for _ in range(L)]
        state["k"], state["v"] = keys_and_values(L, N)
        state["lengths"] = torch.tensor(lengths, dtype=torch.int32, device=device)
        return state
    state["k"], state["v"] = keys_and_values(1 if case.get("shared") else L, N)
    state["lengths"] = state["mask"] = None
    if case["mask"] == "lengths":
        lengths = [rng.randint((N + 1) // 2, N) for _ in range(L)]
        if L >= 4:
            lengths[rng.randrange(L)] = 0                                 # a slot of the batch that holds no source
        state["lengths"] = torch.tensor(lengths, dtype=torch.int32, device=device)
    elif case["mask"] == "holes":
        state["mask"] = torch.rand(L, N, device=device, generator=gen) < 0.8
    if case["op"] == "cross_grad":
        state["grad_out"] = normal(L, M, H, O)
    return state


def run(state):
    """One pass: the result, for a training step the result and the gradients of queries, keys and values."""
    return _run_own(state) if own else _run_plain(state)


def _run_own(state):
    import kermac_amd as kermac
    op = state["case"]["op"]
    if op == "prefix":
        return kermac.prefix_attention(state["q"], state["prefix_k"], state["prefix_v"], state["k"], state["v"], state["lengths"],
                                       scale=state["scale"])
    masks = dict(scale=state["scale"], key_lengths=state["lengths"], key_mask=state["mask"])
    if op == "cross":
        return kermac.cross_attention(state["q"], state["k"], state["v"], **masks)
    out, lse = kermac.cross_attention(state["q"], state["k"], state["v"], return_lse=True, **masks)
    return (out, *kermac.cross_attention_grad(state["grad_out"], state["q"], state["k"], state["v"], out, lse, **masks))


# ------------------------------------------------------------------------------------------------ the plain form

_SCORES_AT_ONCE = 1 << 30


def _rows_of_heads(x, G):
    """[B, M, H, D] -> [B, G, M * H / G, D] in fp32: the rows that meet one head of keys."""
    B, M, H, D = x.shape
    return x.float().reshape(B, M, G, H // G, D).transpose(1, 2).reshape(B, G, M * (H // G), D)


def _tokens_of_rows(x, M):
    """The inverse of _rows_of_heads."""
    B, G, rows, D = x.shape
    return x.reshape(B, G, M, rows // M, D).transpose(1, 2).reshape(B, M, G * (rows // M), D)


def _kept(state, first, last, N, device):
    """[B, 1, 1, N] truth values of the keys that take part, or None."""
    if state["lengths"] is not None:
        return (torch.arange(N, device=device) < state["lengths"][first:last, None])[:, None, None]
    if state["mask"] is not None:
        return state["mask"][first:last, None, None]
    return None


def _weights(scores):
    """Softmax over the last dimension; a row without keys gets zeros."""
    top = scores.amax(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).min)
    weights = scores.sub_(top).exp_()
    return weights.div_(weights.sum(-1, keepdim=True).clamp_min(1e-30))


def _run_plain(state):
    if state["case"]["op"] == "prefix":
        return _plain_prefix(state)
    q, k, v = state["q"], state["k"], state["v"]
    L, M, H, _ = q.shape
    N, G = k.shape[1:3]
    step = max(1, _SCORES_AT_ONCE // (M * H * N))
    outs, grad_qs, grad_ks, grad_vs = [], [], [], []
    for first in range(0, L, step):
        last = min(L, first + step)
        rows = _rows_of_heads(q[first:last], G)
        some_k, some_v = (x.float().transpose(1, 2) if x.shape[0] == 1 else x[first:last].float().transpose(1, 2) for x in (k, v))
        scores = torch.matmul(rows, some_k.transpose(2, 3)).mul_(state["scale"])
        kept = _kept(state, first, last, N, q.device)
        if kept is not None:
            scores.masked_fill_(~kept, -math.inf)
        weights = _weights(scores)
        outs.append(_tokens_of_rows(torch.matmul(weights, some_v), M).to(q.dtype))
        if state["case"]["op"] == "cross":
            continue
        grad = _rows_of_heads(state["grad_out"][first:last], G)
        grad_v = torch.matmul(weights.transpose(2, 3), grad)
        grad_w = torch.matmul(grad, some_v.transpose(2, 3))
        grad_s = grad_w.sub_((grad_w * weights).sum(-1, keepdim=True)).mul_(weights).mul_(state["scale"])
        grad_qs.append(_tokens_of_rows(torch.matmul(grad_s, some_k), M).to(q.dtype))
        grad_ks.append(torch.matmul(grad_s.transpose(2, 3), rows).transpose(1, 2))
        grad_vs.append(grad_v.transpose(1, 2))
    out = torch.cat(outs)
    if state["case"]["op"] == "cross":
        return out
    grad_k, grad_v = torch.cat(grad_ks), torch.cat(grad_vs)
    if k.shape[0] == 1:
        grad_k, grad_v = grad_k.sum(0, keepdim=True), grad_v.sum(0, keepdim=True)
    return out, torch.cat(grad_qs), grad_k.to(k.dtype), grad_v.to(v.dtype)


def _plain_prefix(state):
    q, k, v, lengths = state["q"], state["k"], state["v"], state["lengths"]
    L, M, H, K = q.shape
    N, G = k.shape[1:3]
    P, O = state["prefix_k"].shape[0], v.shape[3]
    rows = _rows_of_heads(q, G)                                                                  # [L, G, M H / G, K]
    some = rows.shape[2]
    prefix_k, prefix_v = (x.float().transpose(0, 1) for x in (state["prefix_k"], state["prefix_v"]))
    step = max(1, _SCORES_AT_ONCE // (some * G * (P + N)))
    outs = []
    for first in range(0, L, step):
        last = min(L, first + step)
        mine, count = rows[first:last], last - first
        # the prefix: the rows of all sequences against one set of keys, one product per head
        together = mine.transpose(0, 1).reshape(G, count * some, K)
        shared = torch.matmul(together, prefix_k.transpose(1, 2)).reshape(G, count, some, P).transpose(0, 1)
        ours = torch.matmul(mine, k[first:last].float().permute(0, 2, 3, 1))
        # query m is token lengths - M + m of its sequence: it sees itself and what stands before it
        position = lengths[first:last, None] - M + torch.arange(M, device=q.device)
        seen = torch.arange(N, device=q.device) <= position.repeat_interleave(H // G, 1)[:, None, :, None]
        scores = torch.cat((shared, ours.masked_fill_(~seen, -math.inf)), -1).mul_(state["scale"])
        weights = _weights(scores)
        from_prefix = torch.matmul(weights[..., :P].transpose(0, 1).reshape(G, count * some, P), prefix_v)
        out = from_prefix.reshape(G, count, some, O).transpose(0, 1) + torch.matmul(weights[..., P:], v[first:last].float().transpose(1, 2))
        outs.append(_tokens_of_rows(out, M).to(q.dtype))
    return torch.cat(outs)


# ------------------------------------------------------------------------------------- the definition in 64 bits

def exact(case, seed):
    """What run returns, from the definition in 64 bits, one batch entry and head of keys at a time."""
    if work(case)["flops"] > 2e13 or case["L"] * case["G"] > 4096:
        return None
    state = prepare(case, seed)
    L, M, N, H, G, K, O = (case[name] for name in "LMNHGKO")
    device, R, P = state["q"].device, H // G, case.get("P", 0)
    q, k, v = state["q"], state["k"], state["v"]
    training = case["op"] == "cross_grad"
    out = torch.zeros(L, M, H, O, dtype=torch.float64, device=device)
    if training:
        grad_q = torch.zeros(L, M, H, K, dtype=torch.float64, device=device)
        grad_k, grad_v = torch.zeros(k.shape, dtype=torch.float64, device=device), torch.zeros(v.shape, dtype=torch.float64, device=device)
    block = max(1, (1 << 28) // (R * (N + P)))                                         # queries at a time
    for entry in range(L):
        source = 0 if k.shape[0] == 1 else entry
        for head in range(G):
            keys, values = k[source, :, head].double(), v[source, :, head].double()
            if case["op"] == "prefix":
                length = int(state["lengths"][entry])
                keys = torch.cat((state["prefix_k"][:, head].double(), keys[:length]))
                values = torch.cat((state["prefix_v"][:, head].double(), values[:length]))
                members = torch.arange(P + length, device=device)
            elif state["lengths"] is not None:
                members = torch.arange(int(state["lengths"][entry]), device=device)
            elif state["mask"] is not None:
                members = state["mask"][entry].nonzero()[:, 0]
            else:
                members = torch.arange(N, device=device)
            if case["op"] != "prefix":
                keys, values = keys[members], values[members]
            if members.numel() == 0:
                continue
            heads = slice(head * R, (head + 1) * R)
            for begin in range(0, M, block):
                some = slice(begin, min(M, begin + block))
                rows = q[entry, some, heads].double().reshape(-1, K)
                logits = rows @ keys.t() * state["scale"]
                if case["op"] == "prefix":
                    query = torch.arange(some.start, some.stop, device=device).repeat_interleave(R)
                    logits[members[None] > (P + length - M + query)[:, None]] = -math.inf
                probabilities = torch.softmax(logits, -1)
                out[entry, some, heads] = (probabilities @ values).reshape(-1, R, O)
                if training:
                    grad = state["grad_out"][entry, some, heads].double().reshape(-1, O)
                    inner = grad @ values.t()
                    inner = probabilities * (inner - (probabilities * inner).sum(1, keepdim=True)) * state["scale"]
                    grad_q[entry, some, heads] = (inner @ keys).reshape(-1, R, K)
                    grad_k[source, :, head].index_add_(0, members, inner.t() @ rows)
                    grad_v[source, :, head].index_add_(0, members, probabilities.t() @ grad)
    return (out, grad_q, grad_k, grad_v) if training else out
