"""Attention over another sequence's states, and over a prefix that a batch shares, as measurable cases.

A case is a flat dict.  `op` names what one pass does:

  cross    kermac.cross_attention(q, k, v, lengths=...)
  train    the same with its log-sum-exp kept, then kermac.cross_attention_grad(...) for a given gradient of the output
  prefix   kermac.prefix_attention(q, k_prefix, v_prefix, k, v, lengths=...)

L sequences of N queries with H heads of D channels meet M keys (own keys behind a prefix of P) with Hk heads, H / Hk query
heads to a key head.  `fill` is the share of the M keys that the shortest sequence has (1.0: all have M, no lengths are
passed); `empty`: one sequence has none.  `layout` is how the caller holds heads: "nhd" tokens first, as projections leave
them, "hnd" heads first, passed as transposed views, "fused" keys and values side by side in one tensor.
"""
import math

import torch

own = False          # False: the operators in elementary torch operations; True: the package's own

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def listed():
    return [
        # One new token of a few sequences against an encoder's states: a decoding step, where latency counts.
        dict(name="cross_token", op="cross", dtype="bfloat16", L=4, N=1, M=1000, P=0, H=16, Hk=16, D=64, fill=1.0,
             empty=False, layout="fused"),
        # The same step of a large batch with shared key heads and ragged lengths: bound by reading the keys.
        dict(name="cross_token_batch", op="cross", dtype="float16", L=64, N=1, M=4096, P=0, H=32, Hk=8, D=128, fill=0.25,
             empty=True, layout="nhd"),
        # A decoder's whole target against padded encoder states, odd extents.
        dict(name="cross_ragged", op="cross", dtype="float16", L=8, N=509, M=1009, P=0, H=16, Hk=4, D=80, fill=0.3,
             empty=False, layout="hnd"),
        # Long queries over long states: the largest one, bound by the products.
        dict(name="cross_long", op="cross", dtype="bfloat16", L=4, N=4096, M=8192, P=0, H=16, Hk=16, D=128, fill=1.0,
             empty=False, layout="nhd"),
        # 32-bit tensors, the type of this package's other operators.
        dict(name="cross_float32", op="cross", dtype="float32", L=2, N=1000, M=1500, P=0, H=8, Hk=8, D=64, fill=0.5,
             empty=False, layout="nhd"),
        # A training step of a small model.
        dict(name="train_small", op="train", dtype="bfloat16", L=2, N=77, M=300, P=0, H=8, Hk=8, D=64, fill=0.5,
             empty=False, layout="nhd"),
        # An ordinary training step: padded states, shared key heads.
        dict(name="train_ragged", op="train", dtype="float16", L=8, N=512, M=1030, P=0, H=16, Hk=4, D=128, fill=0.25,
             empty=True, layout="fused"),
        # Training on long sequences.
        dict(name="train_long", op="train", dtype="bfloat16", L=2, N=4096, M=4096, P=0, H=16, Hk=8, D=128, fill=1.0,
             empty=False, layout="nhd"),
        # Training in 32 bits.
        dict(name="train_float32", op="train", dtype="float32", L=2, N=300, M=500, P=0, H=4, Hk=4, D=64, fill=1.0,
             empty=False, layout="nhd"),
        # A few answers being written below one short prompt.
        dict(name="prefix_few", op="prefix", dtype="bfloat16", L=4, N=1, M=64, P=500, H=8, Hk=8, D=64, fill=0.2,
             empty=False, layout="nhd"),
        # Several proposed tokens a sequence, an odd width.
        dict(name="prefix_proposed", op="prefix", dtype="float16", L=16, N=5, M=300, P=2001, H=16, Hk=2, D=80, fill=0.2,
             empty=False, layout="hnd"),
        # A server's batch below one long prompt.
        dict(name="prefix_batch", op="prefix", dtype="bfloat16", L=128, N=1, M=1024, P=32768, H=32, Hk=8, D=128, fill=0.1,
             empty=False, layout="nhd"),
    ]


# ------------------------------------------------------------------------------------ drawing
def _log_int(rng, low, high):
    """An integer spread evenly over the logarithm of [low, high]; every second one a multiple of 8."""
    v = min(high, max(low, int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))
    if rng.random() < 0.5 and v >= 16:
        v -= v % 8
    return v


def _elements(case):
    L, N, M, P, H, Hk, D = (case[x] for x in ("L", "N", "M", "P", "H", "Hk", "D"))
    return D * (L * N * H + 2 * Hk * (L * M + P))


def _fits(case):
    """Costs no more than the largest listed case (32-bit products counted by what they take), in time and memory."""
    heavy = 16.0 if case["dtype"] == "float32" else 1.0
    return work(case)["flops"] * heavy <= 1.0e12 and _elements(case) <= 3.5e8


def draw(rng):
    """One more case of the ranges above: single tokens to long queries, odd extents, every type and layout."""
    while True:
        op = rng.choice(["cross", "cross", "train", "train", "prefix", "prefix"])
        Hk = rng.choice([1, 2, 4, 8, 16])
        case = dict(op=op, dtype=rng.choice(["bfloat16", "bfloat16", "float16", "float16", "float32"]),
                    L=_log_int(rng, 1, 64 if op != "train" else 16), N=_log_int(rng, 1, 4096), M=_log_int(rng, 1, 16384),
                    P=0, H=Hk * rng.choice([1, 1, 2, 4, 5, 8]), Hk=Hk,
                    D=rng.choice([64, 128, 64, 128, 32, 40, 80, 96, 112]),
                    fill=rng.choice([1.0, round(rng.uniform(0.05, 0.9), 2)]), empty=False,
                    layout=rng.choice(["nhd", "hnd", "fused"]))
        if op == "train":
            case["N"], case["M"] = _log_int(rng, 8, 4096), _log_int(rng, 8, 8192)
        if op == "prefix":
            case["N"], case["M"], case["P"] = rng.choice([1, 1, 1, rng.randint(2, 40)]), _log_int(rng, 40, 4096), _log_int(rng, 1, 65536)
            case["L"] = _log_int(rng, 1, 256)
        if case["H"] > 64:
            continue
        case["empty"] = case["fill"] < 1.0 and case["L"] > 2 and op != "prefix" and rng.random() < 0.3
        # a pass of a few microseconds is the cost of the call alone: the listed small cases stand for that end
        if _fits(case) and work(case)["flops"] >= 1.0e6:
            return case


# ------------------------------------------------------------------------------------ inputs
def _lengths(case):
    """How many of its M keys each sequence has, evenly spread from fill * M to M; prepare() shuffles them."""
    L, M, N = case["L"], case["M"], case["N"]
    low = max(1, int(M * case["fill"]))
    if case["op"] == "prefix":
        low = min(M, max(low, N))          # the new tokens' own keys are there
    lengths = [low + (M - low) * (i + 1) // L for i in range(L)]
    if case["empty"]:
        lengths[0] = 0
    return lengths


def prepare(case, seed):
    dtype, L, N, M, P, H, Hk, D = (case[x] for x in ("dtype", "L", "N", "M", "P", "H", "Hk", "D"))
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, by=1.0):
        return (torch.randn(*shape, generator=gen, device="cuda") * by).to(DTYPES[dtype])

    def heads(n, h, by=1.0):
        return normal(L, h, n, D, by=by).transpose(1, 2) if case["layout"] == "hnd" else normal(L, n, h, D, by=by)

    state = {"op": case["op"], "q": heads(N, H, 1.5), "lengths": None}
    if case["layout"] == "fused":
        both = normal(L, M, 2, Hk, D)
        state["k"], state["v"] = both[:, :, 0], both[:, :, 1]
    else:
        state["k"], state["v"] = heads(M, Hk), heads(M, Hk)
    if case["fill"] < 1.0 or case["empty"]:
        order = torch.randperm(L, generator=gen, device="cuda")
        state["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")[order]
    if case["op"] == "train":
        state["grad_out"] = heads(N, H, 0.5)
    if case["op"] == "prefix":
        state["k_prefix"], state["v_prefix"] = normal(P, Hk, D), normal(P, Hk, D)
    return state


# ------------------------------------------------------------------------------------ plain form
def _weights(q, k, allowed, scale):
    """softmax over the allowed keys, (H, N, M) in 32 bits; rows without an allowed key are zero."""
    group = q.shape[1] // k.shape[1]
    qh = q.float().transpose(0, 1)
    kh = k.float().transpose(0, 1).repeat_interleave(group, dim=0)
    s = torch.matmul(qh, kh.transpose(1, 2)) * scale
    if allowed is not None:
        s = s.masked_fill(~allowed, -math.inf)
    top = s.amax(dim=-1, keepdim=True)
    p = torch.exp(s - top.masked_fill(top == -math.inf, 0.0))
    total = p.sum(dim=-1, keepdim=True)
    return p / total.masked_fill(total == 0.0, 1.0)


def _answer(p, v):
    vh = v.float().transpose(0, 1).repeat_interleave(p.shape[0] // v.shape[1], dim=0)
    return torch.matmul(p, vh).transpose(0, 1)


def _plain_cross(state):
    q, k, v, lengths = state["q"], state["k"], state["v"], state["lengths"]
    scale = 1.0 / math.sqrt(q.shape[-1])
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    grads = None
    if state["op"] == "train":
        grads = tuple(torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))
    at = torch.arange(k.shape[1], device=q.device)
    for l in range(q.shape[0]):
        allowed = None if lengths is None else at < lengths[l]
        if allowed is not None:
            allowed = allowed.expand(1, 1, -1)
        p = _weights(q[l], k[l], allowed, scale)
        o = _answer(p, v[l])
        out[l] = o.to(q.dtype)
        if grads is None:
            continue
        Hk, group = k.shape[2], q.shape[2] // k.shape[2]
        do = state["grad_out"][l].float().transpose(0, 1)
        vh = v[l].float().transpose(0, 1).repeat_interleave(group, dim=0)
        kh = k[l].float().transpose(0, 1).repeat_interleave(group, dim=0)
        qh = q[l].float().transpose(0, 1)
        dp = torch.matmul(do, vh.transpose(1, 2))
        ds = p * (dp - (do * o.transpose(0, 1)).sum(dim=-1, keepdim=True)) * scale
        grads[0][l] = torch.matmul(ds, kh).transpose(0, 1).to(q.dtype)
        for grad, left, right in ((grads[1], ds, qh), (grads[2], p, do)):
            each = torch.matmul(left.transpose(1, 2), right)
            grad[l] = each.reshape(Hk, group, each.shape[1], each.shape[2]).sum(dim=1).transpose(0, 1).to(q.dtype)
    if grads is None:
        return out
    return {"out": out, "grad_q": grads[0], "grad_k": grads[1], "grad_v": grads[2]}


def _plain_prefix(state):
    q, k, v, lengths, kp, vp = (state[x] for x in ("q", "k", "v", "lengths", "k_prefix", "v_prefix"))
    N, M, P = q.shape[1], k.shape[1], kp.shape[0]
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    at = torch.arange(P + M, device=q.device)
    new = torch.arange(N, device=q.device).reshape(1, N, 1)
    for l in range(q.shape[0]):
        length = M if lengths is None else lengths[l]
        allowed = at < P + length - N + new + 1
        p = _weights(q[l], torch.cat([kp, k[l]]), allowed, 1.0 / math.sqrt(q.shape[-1]))
        out[l] = _answer(p, torch.cat([vp, v[l]])).to(q.dtype)
    return out


# ------------------------------------------------------------------------------------ one pass
def run(state):
    if not own:
        return _plain_prefix(state) if state["op"] == "prefix" else _plain_cross(state)
    import kermac_b200 as kermac
    q, k, v, lengths = state["q"], state["k"], state["v"], state["lengths"]
    if state["op"] == "prefix":
        return kermac.prefix_attention(q, state["k_prefix"], state["v_prefix"], k, v, lengths=lengths)
    if state["op"] == "cross":
        return kermac.cross_attention(q, k, v, lengths=lengths)
    out, lse = kermac.cross_attention(q, k, v, lengths=lengths, return_lse=True)
    grad_q, grad_k, grad_v = kermac.cross_attention_grad(q, k, v, out, lse, state["grad_out"], lengths=lengths)
    return {"out": out, "grad_q": grad_q, "grad_k": grad_k, "grad_v": grad_v}


# ------------------------------------------------------------------------------------ work
def work(case):
    """Bytes: each input read once (keys and values up to each sequence's length), each result written once.  Operations:
    two products a (query, key) pair forwards, five more backwards, the softmax not counted."""
    L, N, M, P, H, Hk, D = (case[x] for x in ("L", "N", "M", "P", "H", "Hk", "D"))
    size = 4 if case["dtype"] == "float32" else 2
    lengths = _lengths(case) if case["fill"] < 1.0 or case["empty"] else [M] * L
    keys = sum(lengths)
    queries = L * N * H * D
    if case["op"] == "prefix":
        pairs = sum(N * (P + n) - N * (N - 1) // 2 for n in lengths)
        return {"bytes": size * (2 * queries + 2 * Hk * D * (keys + P)), "flops": 4 * H * D * pairs}
    pairs = N * keys
    if case["op"] == "cross":
        return {"bytes": size * (2 * queries + 2 * Hk * D * keys), "flops": 4 * H * D * pairs}
    return {"bytes": size * (4 * queries + 2 * Hk * D * keys + 2 * Hk * D * L * M), "flops": 14 * H * D * pairs}


# ------------------------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    """The same outputs from the definition, head by head in 64 bits."""
    s = prepare(case, seed)
    q, k, v = s["q"].double(), s["k"].double(), s["v"].double()
    L, N, H, D = q.shape
    M, Hk = k.shape[1], k.shape[2]
    out, dq, dk, dv = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    do = s["grad_out"].double() if case["op"] == "train" else None
    counts = [M] * L if s["lengths"] is None else s["lengths"].tolist()
    P = case["P"]
    for l in range(L):
        n_keys = counts[l]
        for hk in range(Hk):
            keys, values = k[l, :n_keys, hk], v[l, :n_keys, hk]
            hidden = None
            if case["op"] == "prefix":
                keys = torch.cat([s["k_prefix"][:, hk].double(), keys])
                values = torch.cat([s["v_prefix"][:, hk].double(), values])
                last = P + n_keys - N + torch.arange(N, device=q.device)
                hidden = torch.arange(P + n_keys, device=q.device)[None, :] > last[:, None]
            if keys.shape[0] == 0:
                continue
            for h in range(hk * (H // Hk), (hk + 1) * (H // Hk)):
                score = (q[l, :, h] @ keys.T) / math.sqrt(D)
                if hidden is not None:
                    score[hidden] = -math.inf
                e = torch.exp(score - score.max(dim=1, keepdim=True).values)
                w = e / e.sum(dim=1, keepdim=True)
                out[l, :, h] = w @ values
                if do is None:
                    continue
                g = do[l, :, h]
                dw = g @ values.T
                dscore = w * (dw - (w * dw).sum(dim=1, keepdim=True)) / math.sqrt(D)
                dq[l, :, h] = dscore @ keys
                dk[l, :n_keys, hk] += dscore.T @ q[l, :, h]
                dv[l, :n_keys, hk] += w.T @ g
    if case["op"] == "train":
        return {"out": out, "grad_q": dq, "grad_k": dk, "grad_v": dv}
    return out
