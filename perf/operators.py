"""What is measured of the decoder's operators in front of the MoE layer: ``picotron_amd.decoder_ops``.

Three operators, in the order a decoder calls them:

* ``embedding``      -- scaled token lookup; its gradient summed by sorted tokens
* ``qk_norm_rope``   -- RMS norm of each query and key head and the position rotation in one pass, and its gradient
* ``attention``      -- grouped-query attention with capped scores, distance bias, document, prefix and window masks, its
                        gradient, and its form for single tokens over a long cache

``own`` False: ``run`` computes them with elementary torch operations in 32 bits, rounded once at the end.  ``own`` True:
``run`` makes the calls a user makes.  ``exact`` gives the same outputs from the definitions in 64 bits.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
NORM_EPS = 1e-5
ROPE_BASE = 500000.0


# ------------------------------------------------------------------------------------------------
# Cases
# ------------------------------------------------------------------------------------------------
def _embedding_case(name, dtype, tokens, vocab, hidden, scale, padding, train):
    return {"name": name, "op": "embedding", "dtype": dtype, "tokens": tokens, "vocab": vocab, "hidden": hidden, "scale": scale,
            "padding": padding, "train": train}


def _rotate_case(name, dtype, batch, seq, heads, kv_heads, head_dim, norm, positions, packed, train):
    return {"name": name, "op": "qk_norm_rope", "dtype": dtype, "batch": batch, "seq": seq, "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "norm": norm, "positions": positions, "packed": packed, "train": train}


def _attention_case(name, dtype, batch, q_len, kv_len, heads, kv_heads, head_dim, train, softcap=0.0, window=0, slopes=False,
                    documents=0, prefix=0, packed=False):
    return {"name": name, "op": "attention", "dtype": dtype, "batch": batch, "q_len": q_len, "kv_len": kv_len, "heads": heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "train": train, "softcap": softcap, "window": window, "slopes": slopes,
            "documents": documents, "prefix": prefix, "packed": packed}


def listed():
    return [
        # the token lookup and its gradient in one step of the 4-layer training benchmark, four micro-batches in one
        _embedding_case("embedding train 8192", "bf16", 8192, 32000, 2048, 1.0, -1, True),
        # a large vocabulary and a large batch; scaled by sqrt(hidden), padding tokens without gradient
        _embedding_case("embedding train 32768", "bf16", 32768, 131072, 4096, 64.0, 0, True),
        # a small fp32 model of odd sizes
        _embedding_case("embedding train fp32 odd", "fp32", 777, 5003, 200, 14.0, 0, True),
        # queries and keys of one training step: 8192 tokens, 32 query and 8 key heads
        _rotate_case("rotate train 8192", "bf16", 1, 8192, 32, 8, 128, True, "range", False, True),
        # one new token for each of 16 sequences, each at its own position: latency
        _rotate_case("rotate one token x 16", "bf16", 16, 1, 32, 8, 128, True, "given", False, False),
        # fp32, odd length, heads cut out of one fused projection, positions restarting with each document
        _rotate_case("rotate train fp32 odd", "fp32", 3, 333, 6, 2, 72, True, "given", True, True),
        # causal attention of the 4-layer training benchmark: 2048 tokens, 16 / 4 heads
        _attention_case("attention train 2048", "bf16", 1, 2048, 2048, 16, 4, 128, True),
        # packed training: eight documents in a row of 8192 tokens, heads cut out of one fused projection
        _attention_case("attention train documents", "bf16", 2, 8192, 8192, 16, 4, 128, True, documents=8, packed=True),
        # the largest: a long sequence with capped scores
        _attention_case("attention train 16384 capped", "bf16", 1, 16384, 16384, 16, 4, 128, True, softcap=30.0),
        # fp32, odd sizes, prefix mask and distance bias
        _attention_case("attention train fp32 prefix", "fp32", 2, 777, 777, 4, 2, 64, True, slopes=True, prefix=200),
        # one new token for each of 8 sequences over a cache of 32768 keys
        _attention_case("attention one token", "bf16", 8, 1, 32768, 32, 8, 128, False),
        # a few tokens behind a cache, sliding window, capped scores
        _attention_case("attention 5 tokens window", "bf16", 3, 5, 10007, 16, 4, 64, False, softcap=50.0, window=4096),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, spread over its logarithm."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(["embedding", "qk_norm_rope", "attention", "attention"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    if op == "embedding":
        case = _embedding_case("", dtype, _spread(rng, 1, 32768), _spread(rng, 1000, 131072), 8 * _spread(rng, 8, 512),
                               rng.choice([1.0, round(rng.uniform(0.5, 64.0), 2)]), rng.choice([-1, 0, 7]), rng.random() < 0.7)
    elif op == "qk_norm_rope":
        kv_heads = rng.choice([1, 2, 4, 8])
        batch = _spread(rng, 1, 16)
        train = rng.random() < 0.7
        case = _rotate_case("", dtype, batch, _spread(rng, 1, 16384 // batch), kv_heads * rng.choice([1, 2, 3, 4]), kv_heads,
                            8 * rng.randint(1, 16), rng.random() < 0.8, rng.choice(["range", "given"]), rng.random() < 0.4, train)
    else:
        train = rng.random() < 0.6
        kv_heads = rng.choice([1, 2, 4])
        heads = kv_heads * rng.choice([1, 2, 3, 4])
        batch = _spread(rng, 1, 8)
        head_dim = rng.choice([64, 128, 128, 8 * rng.randint(1, 16)])
        mask = rng.choice(["plain", "documents", "prefix", "window"])
        options = {"softcap": rng.choice([0.0, 0.0, round(rng.uniform(5.0, 60.0), 1)]), "slopes": rng.random() < 0.25,
                   "packed": rng.random() < 0.3}
        if train:
            # pairs of all heads stay under those of the largest listed case; fp32 runs at a fraction of its rate
            top = 16384.0 if dtype == "bf16" else 4096.0
            q_len = _spread(rng, 1, int(top * math.sqrt(16.0 / (heads * batch)) / 2))
            kv_len = q_len
        else:
            q_len = rng.choice([1, 1, rng.randint(2, 16)])
            kv_len = q_len + _spread(rng, 16, 65536 // batch)
        if mask == "documents":
            options["documents"] = rng.randint(1, max(1, min(16, kv_len // 4)))
        elif mask == "prefix":
            options["prefix"] = rng.randint(1, kv_len)
        elif mask == "window":
            options["window"] = _spread(rng, 1, kv_len)
        case = _attention_case("", dtype, batch, q_len, kv_len, heads, kv_heads, head_dim, train, **options)
    del case["name"]
    return case


# ------------------------------------------------------------------------------------------------
# Inputs
# ------------------------------------------------------------------------------------------------
def _normal(gen, shape, dtype, std=1.0, mean=0.0):
    return torch.randn(shape, generator=gen, device="cuda").mul_(std).add_(mean).to(dtype)


def _documents(gen, batch, length, count):
    """[batch, length] document numbers: `count` documents of about the same length in a row, the last eighth of one document's
    length at the end of each row left without a document (-1), as padding."""
    at = torch.arange(1, count, device="cuda", dtype=torch.float64)
    cuts = (at + 0.6 * (torch.rand(batch, count - 1, generator=gen, device="cuda", dtype=torch.float64) - 0.5)) * (length / count)
    token = torch.arange(length, device="cuda", dtype=torch.float64)
    ids = (token[None, :, None] >= cuts[:, None, :]).sum(-1)
    ids[:, length - length // (8 * count):] = -1
    return ids.int()


def _parts(gen, case, dtype, lengths, heads):
    """Head tensors [batch, length, heads, head_dim]; with case["packed"] and one length, cut out of one fused projection's output."""
    if case["packed"] and len(set(lengths)) == 1:
        fused = _normal(gen, (case["batch"], lengths[0], sum(heads), case["head_dim"]), dtype)
        return list(fused.split(heads, dim=2))
    return [_normal(gen, (case["batch"], n, h, case["head_dim"]), dtype) for n, h in zip(lengths, heads)]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    state = {"case": case}
    if case["op"] == "embedding":
        # token frequencies fall as 1 / rank, ranks in no order of the ids
        u = torch.rand(case["tokens"], generator=gen, device="cuda", dtype=torch.float64)
        rank = (torch.exp(u * math.log(case["vocab"] + 1)) - 1).long().clamp_(0, case["vocab"] - 1)
        state["ids"] = torch.randperm(case["vocab"], generator=gen, device="cuda")[rank]
        state["weight"] = _normal(gen, (case["vocab"], case["hidden"]), dtype, 0.02)
        leaves = ["weight"]
        shapes = [(case["tokens"], case["hidden"])]
    elif case["op"] == "qk_norm_rope":
        b, s, d = case["batch"], case["seq"], case["head_dim"]
        limit = 4 * s if s > 1 else 8192
        freq = ROPE_BASE ** (-torch.arange(0, d, 2, dtype=torch.float64, device="cuda") / d)
        angle = torch.arange(limit, dtype=torch.float64, device="cuda")[:, None] * freq
        state["cos"], state["sin"] = torch.cos(angle).repeat(1, 2).float(), torch.sin(angle).repeat(1, 2).float()
        state["positions"] = torch.randint(0, limit, (b, s), generator=gen, device="cuda") if case["positions"] == "given" else None
        state["q"], state["k"] = _parts(gen, case, dtype, [s, s], [case["heads"], case["kv_heads"]])
        leaves = ["q", "k"]
        if case["norm"]:
            state["q_weight"], state["k_weight"] = _normal(gen, (d,), dtype, 0.1, 1.0), _normal(gen, (d,), dtype, 0.1, 1.0)
            leaves += ["q_weight", "k_weight"]
        shapes = [(b, s, case["heads"], d), (b, s, case["kv_heads"], d)]
    else:
        b, heads, kv_heads, d = case["batch"], case["heads"], case["kv_heads"], case["head_dim"]
        state["q"], state["k"], state["v"] = _parts(gen, case, dtype, [case["q_len"], case["kv_len"], case["kv_len"]], [heads, kv_heads, kv_heads])
        state["slopes"] = 2.0 ** (-8.0 * torch.arange(1, heads + 1, device="cuda") / heads) if case["slopes"] else None
        state["documents"] = _documents(gen, b, case["kv_len"], case["documents"]) if case["documents"] else None
        state["prefix"] = None
        if case["prefix"]:
            state["prefix"] = torch.randint(case["prefix"] // 2, case["prefix"] + 1, (b,), generator=gen, device="cuda").int()
        leaves = ["q", "k", "v"]
        shapes = [(b, case["q_len"], heads, d)]
    if case["train"]:
        state["grads"] = [_normal(gen, shape, dtype) for shape in shapes]
        state["leaves"] = leaves
        for name in leaves:
            state[name] = state[name].detach().requires_grad_(True)
    return state


# ------------------------------------------------------------------------------------------------
# One pass
# ------------------------------------------------------------------------------------------------
def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return {"embedding": _plain_embedding, "qk_norm_rope": _plain_rotate, "attention": _plain_attention}[state["case"]["op"]](state)


def _own(state):
    from picotron_amd import decoder_ops

    case = state["case"]
    if case["op"] == "embedding":
        outs = [decoder_ops.embedding(state["ids"], state["weight"], scale=case["scale"], padding_idx=case["padding"] if case["padding"] >= 0 else None)]
    elif case["op"] == "qk_norm_rope":
        outs = list(decoder_ops.qk_norm_rope(state["q"], state["k"], state["cos"], state["sin"], state.get("q_weight"), state.get("k_weight"),
                                             eps=NORM_EPS, positions=state["positions"]))
    else:
        outs = [decoder_ops.attention(state["q"], state["k"], state["v"], causal=True, softcap=case["softcap"], window=case["window"],
                                      slopes=state["slopes"], document_ids=state["documents"], prefix_lengths=state["prefix"])]
    if not case["train"]:
        return outs
    grads = torch.autograd.grad(outs, [state[name] for name in state["leaves"]], state["grads"])
    return [o.detach() for o in outs] + list(grads)


def _plain_embedding(state):
    case, weight, ids = state["case"], state["weight"], state["ids"]
    out = (weight[ids].float() * case["scale"]).to(weight.dtype)
    if not case["train"]:
        return [out]
    grad = state["grads"][0].float() * case["scale"]
    if case["padding"] >= 0:
        grad = torch.where((ids == case["padding"])[:, None], torch.zeros_like(grad), grad)
    d_weight = torch.zeros(weight.shape, dtype=torch.float32, device=weight.device).index_add_(0, ids, grad)
    return [out, d_weight.to(weight.dtype)]


def _half_turned(x):
    a, b = x.chunk(2, dim=-1)
    return torch.cat([-b, a], dim=-1)


def _plain_rotate_one(x, weight, cos, sin, grad):
    """Outputs of one of q and k; with grad: the gradients of x and of the weight too, from the formulas."""
    dtype, x = x.dtype, x.float()
    if weight is not None:
        rms = torch.rsqrt(x.square().mean(-1, keepdim=True) + NORM_EPS)
        normed = x * rms
        y = normed * weight.float()
    else:
        y = x
    out = (y * cos + _half_turned(y) * sin).to(dtype)
    if grad is None:
        return out, None, None
    grad = grad.float()
    dy = grad * cos - _half_turned(grad * sin)
    if weight is None:
        return out, dy.to(dtype), None
    dn = dy * weight.float()
    dx = rms * (dn - normed * (dn * normed).mean(-1, keepdim=True))
    return out, dx.to(dtype), (dy * normed).sum((0, 1, 2)).to(dtype)


def _plain_rotate(state):
    case = state["case"]
    at = state["positions"] if state["positions"] is not None else torch.arange(case["seq"], device="cuda")[None]
    cos, sin = state["cos"][at][:, :, None], state["sin"][at][:, :, None]
    grads = state["grads"] if case["train"] else (None, None)
    q, dq, dqw = _plain_rotate_one(state["q"], state.get("q_weight"), cos, sin, grads[0])
    k, dk, dkw = _plain_rotate_one(state["k"], state.get("k_weight"), cos, sin, grads[1])
    if not case["train"]:
        return [q, k]
    return [q, k, dq, dk] + ([dqw, dkw] if case["norm"] else [])


def _seen(state):
    """[batch, q_len, kv_len]: which keys each query sees."""
    case = state["case"]
    at = torch.arange(case["q_len"], device="cuda")[:, None] + (case["kv_len"] - case["q_len"])
    key = torch.arange(case["kv_len"], device="cuda")[None]
    seen = (key <= at)[None].expand(case["batch"], -1, -1)
    if state["prefix"] is not None:
        seen = seen | (key[None] < state["prefix"][:, None, None])
    if case["window"]:
        seen = seen & ((at - key).abs() < case["window"])[None]
    if state["documents"] is not None:
        ids = state["documents"]
        mine = ids[:, case["kv_len"] - case["q_len"]:]
        seen = seen & (mine[:, :, None] == ids[:, None, :]) & (mine[:, :, None] >= 0)
    return seen


def _plain_attention(state):
    case, dtype = state["case"], state["q"].dtype
    b, sq, sk, h, g, d = case["batch"], case["q_len"], case["kv_len"], case["heads"], case["kv_heads"], case["head_dim"]
    scale = 1.0 / math.sqrt(d)
    # heads of one key-value head side by side: [b, g, heads per key head * sq, .]
    rows = lambda x: x.float().transpose(1, 2).reshape(b, g, (h // g) * sq, d)
    q = rows(state["q"])
    k, v = (state[n].float().transpose(1, 2).contiguous() for n in ("k", "v"))
    s = (q @ k.transpose(2, 3)).mul_(scale)
    if case["softcap"]:
        capped = torch.tanh(s.div_(case["softcap"]))
        s = capped * case["softcap"]
    s = s.view(b, h, sq, sk)
    if state["slopes"] is not None:
        at = torch.arange(sq, device="cuda")[:, None] + (sk - sq)
        s = s - state["slopes"].float()[:, None, None] * (at - torch.arange(sk, device="cuda")[None]).abs().float()
    seen = _seen(state)[:, None]
    s = s.masked_fill(~seen, float("-inf"))
    top = s.amax(-1, keepdim=True)
    top = torch.where(top > float("-inf"), top, torch.zeros_like(top))
    p = s.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    p = p.div_(torch.where(total > 0, total, torch.ones_like(total))).view(b, g, (h // g) * sq, sk)
    o = p @ v
    back = lambda x: x.reshape(b, h, sq, d).transpose(1, 2).to(dtype)
    if not case["train"]:
        return [back(o)]
    do = rows(state["grads"][0])
    dv = p.transpose(2, 3) @ do
    ds = (do @ v.transpose(2, 3)).sub_((do * o).sum(-1, keepdim=True)).mul_(p)
    if case["softcap"]:
        ds.mul_(1.0 - capped.square_())
    ds.mul_(scale)
    dq, dk = ds @ k, ds.transpose(2, 3) @ q
    return [back(o), back(dq), dk.transpose(1, 2).to(dtype), dv.transpose(1, 2).to(dtype)]


# ------------------------------------------------------------------------------------------------
# The definitions in 64 bits
# ------------------------------------------------------------------------------------------------
def exact(case, seed):
    state = prepare(case, seed)
    leaf = lambda name: state[name].detach().double().requires_grad_(case["train"]) if state.get(name) is not None else None
    if case["op"] == "embedding":
        weight = leaf("weight")
        outs = [torch.nn.functional.embedding(state["ids"], weight, padding_idx=case["padding"] if case["padding"] >= 0 else None) * case["scale"]]
        leaves = [weight]
    elif case["op"] == "qk_norm_rope":
        at = state["positions"] if state["positions"] is not None else torch.arange(case["seq"], device="cuda").expand(case["batch"], -1)
        half = case["head_dim"] // 2
        turn = torch.complex(state["cos"].double(), state["sin"].double())[at][:, :, None, :half]
        outs, leaves, weights = [], [], []
        for name in ("q", "k"):
            x, w = leaf(name), leaf(name + "_weight")
            y = x if w is None else x / torch.sqrt((x * x).sum(-1, keepdim=True) / case["head_dim"] + NORM_EPS) * w
            z = torch.complex(y[..., :half].contiguous(), y[..., half:].contiguous()) * turn
            outs.append(torch.cat([z.real, z.imag], dim=-1))
            leaves.append(x)
            weights += [] if w is None else [w]
        leaves += weights
    else:
        return _exact_attention(state)
    if not case["train"]:
        return [o.detach() for o in outs]
    return [o.detach() for o in outs] + list(torch.autograd.grad(outs, leaves, [g.double() for g in state["grads"]]))


def _exact_attention(state):
    """Head by head and row block by row block."""
    case = state["case"]
    sq, sk, per = case["q_len"], case["kv_len"], case["heads"] // case["kv_heads"]
    q, k, v = (state[n].detach().double() for n in ("q", "k", "v"))
    o, dq, dk, dv = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    key = torch.arange(sk, device="cuda")
    block = max(1, (1 << 27) // sk)
    for b in range(case["batch"]):
        for first in range(0, sq, block):
            r = slice(first, min(sq, first + block))
            at = torch.arange(sq, device="cuda")[r] + sk - sq
            away = at[:, None] - key[None]
            hidden = away < 0
            if state["prefix"] is not None:
                hidden &= key[None] >= state["prefix"][b]
            if case["window"]:
                hidden |= away.abs() >= case["window"]
            if state["documents"] is not None:
                ids = state["documents"][b]
                hidden |= (ids[at][:, None] != ids[None]) | (ids[at] < 0)[:, None]
            nothing = hidden.all(1, keepdim=True)
            for h in range(case["heads"]):
                x = [t.clone().requires_grad_(case["train"]) for t in (q[b, r, h], k[b, :, h // per], v[b, :, h // per])]
                s = (x[0] @ x[1].T) / math.sqrt(case["head_dim"])
                if case["softcap"]:
                    s = torch.tanh(s / case["softcap"]) * case["softcap"]
                if state["slopes"] is not None:
                    s = s - state["slopes"][h].double() * away.abs()
                p = torch.softmax(s.masked_fill(hidden, -math.inf).masked_fill(nothing, 0.0), dim=1).masked_fill(hidden, 0.0)
                out = p @ x[2]
                o[b, r, h] = out.detach()
                if case["train"]:
                    a, c, e = torch.autograd.grad(out, x, state["grads"][0][b, r, h].double())
                    dq[b, r, h] = a
                    dk[b, :, h // per] += c
                    dv[b, :, h // per] += e
    return [o, dq, dk, dv] if case["train"] else [o]


# ------------------------------------------------------------------------------------------------
# What a pass cannot do without
# ------------------------------------------------------------------------------------------------
def _pairs(case):
    """Query-key pairs of one head that the masks leave, over the batch (documents of equal length)."""
    sq, sk, off = case["q_len"], case["kv_len"], case["kv_len"] - case["q_len"]
    reach = case["window"] or sk
    documents = case["documents"] or 1
    length = sk / documents
    total = 0
    for i in range(sq):
        at = i + off
        before = min(at + 1, reach, int(at % length) + 1)
        after = max(0, min(0.75 * case["prefix"], at + reach) - at - 1)
        total += before + after
    return case["batch"] * total


def work(case):
    size = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "embedding":
        rows = case["tokens"] * case["hidden"] * size
        table = min(case["tokens"], case["vocab"]) * case["hidden"] * size
        nbytes = table + rows + 8 * case["tokens"]
        flops = case["tokens"] * case["hidden"]
        if case["train"]:
            nbytes += rows + case["vocab"] * case["hidden"] * size
            flops *= 3
        return {"bytes": nbytes, "flops": flops}
    heads = case["heads"] + case["kv_heads"]
    if case["op"] == "qk_norm_rope":
        elements = case["batch"] * case["seq"] * heads * case["head_dim"]
        # forward: x in, out out; backward: x and the gradient in, dx out
        return {"bytes": elements * size * (5 if case["train"] else 2) + 8 * case["seq"] * case["head_dim"],
                "flops": elements * (25 if case["train"] else 8)}
    reach = min(case["kv_len"], (case["window"] or case["kv_len"]) + case["q_len"])
    q = case["batch"] * case["q_len"] * case["heads"] * case["head_dim"] * size
    kv = 2 * case["batch"] * reach * case["kv_heads"] * case["head_dim"] * size
    products = 7 if case["train"] else 2   # forward two; backward five
    return {"bytes": 2 * q + kv + ((2 * q + kv + kv) if case["train"] else 0),
            "flops": 2 * products * _pairs(case) * case["heads"] * case["head_dim"]}
