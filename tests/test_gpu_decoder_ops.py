"""The decoder's operators (picotron_amd.decoder_ops) against the 64-bit oracle, which also says elementwise how far fp32
arithmetic with one rounding at the end (and, for bf16 attention, roundings of P and dx to bf16) may be off."""

import itertools
import math
import types

import pytest
import torch

from oracle import decoder_ops_oracle as O

pytestmark = pytest.mark.gpu

BF16, FP32 = torch.bfloat16, torch.float32


def _ops():
    from picotron_amd import decoder_ops

    return decoder_ops


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(gen, *shape, dtype=BF16):
    return torch.randn(*shape, generator=gen, device="cuda").to(dtype)


def _within(name, got, pair):
    value, bound = pair
    assert got.shape == value.shape, (name, got.shape, value.shape)
    off = (got.double() - value).abs()
    finite = torch.isfinite(value)
    assert torch.equal(torch.isfinite(got), finite), f"{name}: {int((torch.isfinite(got) != finite).sum())} values finite on one side only"
    # values below the type's normal range are rounded to its absolute steps
    over = (off - bound - 2.0 ** -126)[finite]
    if over.numel():
        worst = int(over.argmax())
        assert float(over.max()) <= 0, f"{name}: off by {float(off[finite][worst]):.3e}, bound {float(bound[finite][worst]):.3e}"


# ------------------------------------------------------------------------------------------------
# Embedding
# ------------------------------------------------------------------------------------------------
def _ids(kind, tokens, vocab, gen):
    if kind == "uniform":
        return torch.randint(0, vocab, (tokens,), generator=gen, device="cuda")
    if kind == "one":
        return torch.full((tokens,), vocab - 1, device="cuda")
    if kind == "few":  # runs of every length around the 64 that are summed in one go
        lengths = list(itertools.islice(itertools.cycle([63, 64, 65, 1, 127, 128, 129, 200]), tokens))
        ids = torch.arange(len(lengths)).repeat_interleave(torch.tensor(lengths))[:tokens] % vocab
        return ids.cuda()[torch.randperm(tokens, generator=gen, device="cuda")]
    ids = torch.randint(0, vocab, (tokens,), generator=gen, device="cuda")  # some outside the table
    ids[::5] = -1
    ids[3::7] = vocab
    ids[4::11] = 1 << 40
    return ids


EMBEDDINGS = [
    # dtype, tokens, vocab, hidden, scale, padding, ids
    (BF16, 1, 1, 8, 1.0, None, "uniform"), (BF16, 777, 500, 64, 8.0, 0, "uniform"), (BF16, 4097, 32000, 200, 1.0, None, "uniform"),
    (FP32, 5000, 70, 36, 0.3, 5, "few"), (BF16, 5000, 70, 264, 3.7, None, "few"), (BF16, 3000, 300000, 8, 1.0, None, "uniform"),
    (BF16, 9000, 11, 2056, 1.0, None, "one"), (FP32, 64, 3, 7, 2.0, None, "one"), (FP32, 65, 3, 5, 2.0, None, "one"), (BF16, 130, 9, 13, 1.5, 8, "few"),
    (BF16, 1000, 50, 64, 1.0, 2, "bad"), (FP32, 1, 5, 4, 1.0, None, "bad"), (BF16, 20000, 511, 16, 1.0, None, "uniform"),
    (BF16, 0, 20, 16, 1.0, None, "uniform"),
    # sorts of one block (8192 tokens), of blocks of 1, 4 and 16 rounds; digits of one to four passes
    (BF16, 8192, 600, 8, 1.0, None, "uniform"), (FP32, 8193, 3, 4, 1.0, 1, "uniform"), (BF16, 70000, 40000, 8, 1.0, None, "uniform"),
    (BF16, 300000, 1000, 8, 1.0, 3, "bad"), (FP32, 300000, 600000, 4, 2.0, None, "few"), (BF16, 500, 1 << 27, 1, 1.0, None, "uniform"),
]


@pytest.mark.parametrize("dtype,tokens,vocab,hidden,scale,padding,kind", EMBEDDINGS)
def test_embedding_against_the_oracle(gpu, dtype, tokens, vocab, hidden, scale, padding, kind):
    gen = _gen(tokens + hidden)
    ids = _ids(kind, tokens, vocab, gen)
    weight = _randn(gen, vocab, hidden, dtype=dtype).requires_grad_(True)
    g = _randn(gen, tokens, hidden, dtype=dtype)
    out = _ops().embedding(ids, weight, scale=scale, padding_idx=padding)
    (dw,) = torch.autograd.grad(out, weight, g)
    want = O.embedding(ids, weight.detach(), scale, padding, g)
    _within("out", out.detach(), want["out"])
    _within("d_weight", dw, want["d_weight"])
    again = torch.autograd.grad(_ops().embedding(ids, weight, scale=scale, padding_idx=padding), weight, g)[0]
    assert torch.equal(dw, again)


def test_embedding_views_shapes_and_types(gpu):
    gen = _gen(1)
    table = _randn(gen, 40, 50)
    ids = torch.randint(0, 40, (3, 4), generator=gen, device="cuda", dtype=torch.int32)
    for weight in (table[:, 1:49], table.t()[:, :30], table[3:, 2:]):  # odd starts, transposed
        weight = weight.detach().requires_grad_(True)
        use = ids % weight.shape[0]
        out = _ops().embedding(use, weight, scale=0.5)
        assert out.shape == (3, 4, weight.shape[1]) and torch.equal(out, (weight[use.long()].float() * 0.5).to(BF16))
        g = _randn(gen, 4, 3, weight.shape[1]).transpose(0, 1)
        (dw,) = torch.autograd.grad(out, weight, g)
        _within("d_weight", dw, O.embedding(use, weight.detach(), 0.5, None, g)["d_weight"])


# ------------------------------------------------------------------------------------------------
# Norm + rotation
# ------------------------------------------------------------------------------------------------
ROTATIONS = [
    # dtype, batch, seq, heads, kv_heads, head_dim, q norm, k norm, positions, packed
    (BF16, 1, 1, 1, 1, 8, True, True, None, False), (BF16, 2, 100, 16, 4, 128, True, True, None, False), (FP32, 2, 37, 6, 2, 72, True, True, "given", True),
    (BF16, 3, 33, 5, 5, 72, True, True, "row", True), (BF16, 1, 257, 3, 1, 256, True, False, None, False), (FP32, 1, 65, 4, 2, 256, False, True, "given", False),
    (BF16, 2, 50, 4, 2, 64, False, False, None, True), (FP32, 4, 9, 2, 1, 16, True, True, None, False), (BF16, 2, 30, 7, 1, 24, True, True, "given", False),
    (BF16, 1, 3000, 20, 12, 128, True, True, "given", True), (BF16, 2, 11, 4, 2, 64, True, True, "bad", False), (BF16, 0, 5, 2, 1, 64, True, True, None, False),
    (BF16, 3, 0, 2, 1, 64, True, True, None, False),
]


@pytest.mark.parametrize("dtype,batch,seq,heads,kv_heads,D,q_norm,k_norm,kind,packed", ROTATIONS)
def test_norm_rope_against_the_oracle(gpu, dtype, batch, seq, heads, kv_heads, D, q_norm, k_norm, kind, packed):
    gen = _gen(seq * D + heads)
    if packed:
        q, k, _ = _randn(gen, batch, seq, heads + 2 * kv_heads, D, dtype=dtype).split([heads, kv_heads, kv_heads], dim=2)
    else:
        q, k = _randn(gen, batch, seq, heads, D, dtype=dtype), _randn(gen, batch, seq, kv_heads, D, dtype=dtype)
    cos, sin = torch.randn(max(1, 2 * seq), D, generator=gen, device="cuda"), torch.randn(max(1, 2 * seq), D, generator=gen, device="cuda")
    positions = None
    if kind in ("given", "bad"):
        positions = torch.randint(0, 2 * seq, (batch, seq), generator=gen, device="cuda")
    elif kind == "row":
        positions = torch.randint(0, 2 * seq, (seq,), generator=gen, device="cuda", dtype=torch.int32)
    if kind == "bad":
        positions[0, 3], positions[1, 0] = -1, 2 * seq
    at = torch.arange(seq, device="cuda").expand(batch, seq) if positions is None else positions.expand(batch, seq)
    weights = [(_randn(gen, D, dtype=torch.float32) * 0.2 + 1).to(dtype).requires_grad_(True) if on else None for on in (q_norm, k_norm)]
    q, k = q.detach().requires_grad_(True), k.detach().requires_grad_(True)
    gq, gk = _randn(gen, *q.shape, dtype=dtype), _randn(gen, *k.shape, dtype=dtype)
    run = lambda: _ops().qk_norm_rope(q, k, cos, sin, *weights, eps=1e-5, positions=positions)
    outs = run()
    leaves = [q, k] + [w for w in weights if w is not None]
    grads = torch.autograd.grad(outs, leaves, [gq, gk])
    bad = (at < 0) | (at >= cos.shape[0])
    if bad.any():
        for t in (*outs, *grads[:2]):
            assert torch.isnan(t[bad]).all() and torch.isfinite(t[~bad]).all()
        assert all(torch.isnan(t).all() for t in grads[2:])
        at = at.clamp(0, cos.shape[0] - 1)
    got = dict(zip(["dq", "dk"] + [n for n, w in zip(("dqw", "dkw"), weights) if w is not None], grads))
    for n, x, w, out, g in (("q", q, weights[0], outs[0], gq), ("k", k, weights[1], outs[1], gk)):
        want = O.norm_rope(x.detach(), None if w is None else w.detach(), cos, sin, at, 1e-5, g)
        keep = ~bad
        _within(n, out.detach()[keep], tuple(t[keep] for t in want["out"]))
        _within("d" + n, got["d" + n][keep], tuple(t[keep] for t in want["dx"]))
        if w is not None and not bad.any():
            _within(f"d{n}w", got[f"d{n}w"], want["dw"])
    for a, b in zip(grads, torch.autograd.grad(run(), leaves, [gq, gk])):
        assert torch.equal(a, b) or bad.any()


# ------------------------------------------------------------------------------------------------
# Attention
# ------------------------------------------------------------------------------------------------
def _documents(kind, batch, length, gen):
    if kind == "runs":
        cuts = torch.sort(torch.randint(1, max(2, length), (batch, 3), generator=gen, device="cuda"), dim=1).values
        ids = (torch.arange(length, device="cuda")[None, :, None] >= cuts[:, None]).sum(-1).int()
        ids[:, length - length // 7:] = -1
        return ids
    if kind == "mixed":  # in no order
        return torch.randint(-1, 3, (batch, length), generator=gen, device="cuda", dtype=torch.int32)
    return torch.full((batch, length), -1, device="cuda", dtype=torch.int32)  # nobody sees anything


def _options(spec, batch, kv_len, heads, gen):
    options = dict(spec)
    if "documents" in options:
        options["document_ids"] = _documents(options.pop("documents"), batch, kv_len, gen)
    if "prefix" in options:
        options["prefix_lengths"] = torch.randint(0, options.pop("prefix") + 1, (batch,), generator=gen, device="cuda", dtype=torch.int32)
    if options.pop("slopes", False):
        options["slopes"] = 2.0 ** (-8.0 * torch.arange(1, heads + 1, device="cuda") / heads)
    return options


def _qkv(gen, dtype, batch, q_len, kv_len, heads, kv_heads, D, packed=False):
    if packed:
        parts = _randn(gen, batch, kv_len, heads + 2 * kv_heads, D, dtype=dtype).split([heads, kv_heads, kv_heads], dim=2)
    else:
        parts = [_randn(gen, batch, n, h, D, dtype=dtype) for n, h in ((q_len, heads), (kv_len, kv_heads), (kv_len, kv_heads))]
    return [t.detach().requires_grad_(True) for t in parts]


ATTENTIONS = [
    # dtype, batch, q_len, kv_len, heads, kv_heads, head_dim, options
    (BF16, 1, 1, 1, 1, 1, 8, {}), (BF16, 2, 40, 40, 4, 2, 16, {}), (FP32, 2, 40, 40, 4, 2, 16, {}), (BF16, 1, 300, 300, 4, 1, 128, {}),
    (FP32, 1, 130, 130, 2, 2, 128, {}), (BF16, 2, 129, 129, 6, 2, 64, {"softcap": 5.0}), (FP32, 1, 150, 150, 3, 1, 72, {"softcap": 2.0, "slopes": True}),
    (BF16, 1, 257, 257, 8, 2, 128, {"documents": "runs"}), (BF16, 2, 200, 200, 2, 1, 64, {"documents": "mixed"}), (FP32, 2, 100, 100, 2, 1, 64, {"documents": "mixed", "softcap": 3.0}),
    (BF16, 1, 90, 90, 2, 1, 64, {"documents": "none"}), (BF16, 3, 200, 200, 4, 2, 64, {"prefix": 150}), (FP32, 2, 77, 77, 4, 2, 64, {"prefix": 77, "slopes": True}),
    (BF16, 1, 400, 400, 2, 1, 128, {"window": 50}), (BF16, 1, 200, 200, 2, 1, 128, {"window": 1}), (FP32, 1, 200, 200, 2, 1, 32, {"window": 70, "causal": False}),
    (BF16, 2, 100, 170, 4, 4, 64, {}), (BF16, 2, 170, 100, 4, 4, 64, {}), (FP32, 1, 70, 33, 4, 2, 64, {"window": 20}), (BF16, 2, 60, 90, 3, 3, 128, {"causal": False}),
    (BF16, 1, 120, 120, 16, 1, 128, {"slopes": True, "window": 64, "prefix": 100, "documents": "runs", "softcap": 20.0}),
    (BF16, 1, 70, 70, 5, 1, 256, {"softcap": 9.0}), (FP32, 1, 50, 50, 2, 1, 200, {}), (BF16, 1, 64, 64, 2, 2, 24, {"documents": "runs"}),
    (BF16, 4, 1, 500, 8, 2, 128, {}), (FP32, 2, 1, 300, 8, 2, 64, {"window": 100}), (BF16, 2, 5, 1000, 16, 4, 64, {"softcap": 10.0, "documents": "runs"}),
    (BF16, 1, 3, 777, 40, 1, 128, {"slopes": True}), (BF16, 1, 1, 4000, 4, 4, 128, {"causal": False}), (FP32, 1, 2, 2500, 3, 3, 72, {"prefix": 2000}),
    (BF16, 2, 90, 90, 6, 2, 64, {"softcap": 1e5}), (FP32, 1, 80, 80, 2, 1, 64, {"softcap": 1e7}), (BF16, 1, 140, 140, 2, 1, 128, {"scale": -0.2}),
    (BF16, 1, 140, 140, 2, 1, 64, {"scale": 0.0}), (BF16, 1, 150, 150, 24, 1, 128, {"window": 33}), (FP32, 1, 1, 900, 1, 1, 128, {"slopes": True, "softcap": 3.0}),
    (BF16, 1, 33, 3000, 1, 1, 128, {}), (BF16, 1, 1, 130, 33, 1, 64, {"window": 7}), (BF16, 2, 260, 260, 4, 2, 120, {"documents": "runs", "softcap": 6.0}),
    (BF16, 1, 300, 300, 4, 2, 256, {}), (BF16, 2, 1, 700, 8, 2, 256, {}), (BF16, 1, 150, 150, 3, 1, 200, {"documents": "runs"}),
    (BF16, 1, 5, 2000, 4, 1, 136, {"softcap": 20.0, "slopes": True}), (BF16, 1, 1300, 1300, 2, 1, 256, {"window": 400}), (BF16, 2, 65, 129, 1, 1, 248, {"softcap": 2e3}),
    (BF16, 5, 7, 7, 2, 1, 128, {}), (BF16, 1, 700, 700, 12, 4, 128, {"documents": "runs"}), (FP32, 1, 520, 520, 4, 2, 128, {"softcap": 4.0}),
]


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("dtype,batch,q_len,kv_len,heads,kv_heads,D,spec", ATTENTIONS)
def test_attention_against_the_oracle(gpu, dtype, batch, q_len, kv_len, heads, kv_heads, D, spec, packed):
    if packed and q_len != kv_len:
        pytest.skip("one projection has one length")
    gen = _gen(q_len * D + heads)
    q, k, v = _qkv(gen, dtype, batch, q_len, kv_len, heads, kv_heads, D, packed)
    options = _options(spec, batch, kv_len, heads, gen)
    g = _randn(gen, *q.shape, dtype=dtype)
    out = _ops().attention(q, k, v, **options)
    grads = torch.autograd.grad(out, (q, k, v), g)
    want = O.attention(q.detach(), k.detach(), v.detach(), d_out=g, **options)
    for name, got in zip(("out", "dq", "dk", "dv"), (out.detach(), *grads)):
        _within(name, got, want[name])
    again = _ops().attention(q, k, v, **options)
    assert torch.equal(out, again)
    for a, b in zip(grads, torch.autograd.grad(again, (q, k, v), g)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype,D,q_len", [(BF16, 128, 200), (FP32, 64, 200), (BF16, 64, 1), (BF16, 256, 70), (BF16, 72, 90)])
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_what_is_hidden_reaches_nothing(gpu, dtype, D, q_len, value):
    """NaN or infinity in the keys, values, queries and output gradients of one document: the other documents' outputs and gradients
    are, bit for bit, what they are without."""
    gen = _gen(D)
    L = max(q_len, 200)
    ids = torch.zeros(1, L, device="cuda", dtype=torch.int32)
    ids[:, 30:50], ids[:, 70:71], ids[:, L - 20:] = 1, 1, -1
    ids[:, L - 21] = 0
    other = ids[0] != 0
    q, k, v = _qkv(gen, dtype, 1, q_len, L, 4, 2, D)
    g = _randn(gen, *q.shape, dtype=dtype)
    if q_len == 1:
        ids[:, -1] = 0
        other = ids[0] != 0
    mine = other[L - q_len:]

    def run():
        out = _ops().attention(q, k, v, document_ids=ids, softcap=8.0)
        return (out.detach(), *torch.autograd.grad(out, (q, k, v), g))

    clean = run()
    with torch.no_grad():
        for t, hide in ((q, mine), (k, other), (v, other), (g, mine)):
            t[:, hide] = value
            if value == math.inf:
                t[:, hide, :, ::2] = -value
    dirty = run()
    for name, a, b, hide in zip(("out", "dq", "dk", "dv"), clean, dirty, (mine, mine, other, other)):
        assert torch.equal(a[:, ~hide], b[:, ~hide]), name
        assert torch.isfinite(b[:, ~hide]).all()
    # padding sees nothing and is seen by nobody
    pad = ids[0] == -1
    for t, hide in zip(dirty, (pad[L - q_len:], pad[L - q_len:], pad, pad)):
        assert not t[:, hide].any()


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_nan_shows_where_it_is_seen(gpu, dtype):
    gen = _gen(9)
    q, k, v = _qkv(gen, dtype, 1, 100, 100, 2, 2, 64)
    with torch.no_grad():
        v[0, 40, 0, 3] = math.nan
        k[0, 60, 1, 5] = math.nan
    out = _ops().attention(q, k, v).detach()
    assert torch.isnan(out[0, 40:, 0, 3]).all() and torch.isfinite(out[0, :40, 0]).all()
    assert torch.isfinite(out[0, :, 0, :3]).all() and torch.isfinite(out[0, :, 0, 4:]).all()
    assert torch.isnan(out[0, 60:, 1]).all() and torch.isfinite(out[0, :60, 1]).all()


def test_large_scores(gpu):
    """Scores of thousands: the running maximum carries them."""
    gen = _gen(4)
    q, k, v = _qkv(gen, FP32, 1, 150, 150, 2, 1, 64)
    with torch.no_grad():
        q.mul_(40.0)
        k.mul_(40.0)
    g = _randn(gen, *q.shape, dtype=FP32)
    out = _ops().attention(q, k, v)
    want = O.attention(q.detach(), k.detach(), v.detach(), d_out=g)
    for name, got in zip(("out", "dq", "dk", "dv"), (out.detach(), *torch.autograd.grad(out, (q, k, v), g))):
        _within(name, got, want[name])


def test_empty_lengths(gpu):
    q = torch.randn(2, 3, 4, 64, device="cuda", dtype=BF16, requires_grad=True)
    k = torch.randn(2, 0, 2, 64, device="cuda", dtype=BF16, requires_grad=True)
    out = _ops().attention(q, k, k, document_ids=torch.zeros(2, 0, device="cuda", dtype=torch.int32))
    assert out.shape == q.shape and not out.any()
    dq, dk = torch.autograd.grad(out.sum(), (q, k))
    assert not dq.any() and dk.shape == k.shape
    none = torch.randn(2, 0, 4, 64, device="cuda", dtype=BF16, requires_grad=True)
    keys = torch.randn(2, 5, 2, 64, device="cuda", dtype=BF16, requires_grad=True)
    out = _ops().attention(none, keys, keys)
    assert out.shape == none.shape
    assert not torch.autograd.grad(out.sum(), keys)[0].any()
    out = _ops().attention(q[:0], keys[:0], keys[:0])
    assert out.shape == (0, 3, 4, 64) and torch.autograd.grad(out.sum(), q)[0].shape == q.shape


def test_strides_and_broadcasts(gpu):
    """Heads first in memory, every other token, a cache broadcast over the batch, rows off the 16-byte grid."""
    gen = _gen(5)
    B, S, H, G, D = 3, 70, 4, 2, 64
    q = _randn(gen, B, H, S, D).transpose(1, 2)
    k = _randn(gen, 1, 2 * S, G, D)[:, ::2].expand(B, S, G, D)
    v = _randn(gen, B, S, G, D + 4)[..., 3:D + 3]
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    g = _randn(gen, B, H, S, D).transpose(1, 2)
    out = _ops().attention(*leaves)
    want = O.attention(q, k, v, d_out=g)
    for name, got in zip(("out", "dq", "dk", "dv"), (out.detach(), *torch.autograd.grad(out, leaves, g))):
        _within(name, got, want[name])
    # a broadcast leaf's gradient is the sum over what it was broadcast to
    shared = k[:1].detach().requires_grad_(True)
    (dk,) = torch.autograd.grad(_ops().attention(q, shared.expand(B, S, G, D), v), shared, g)
    value, bound = want["dk"]
    _within("dk", dk, (value.sum(0, keepdim=True), bound.sum(0, keepdim=True) + 2.0 ** -8 * value.abs().sum(0, keepdim=True)))


@pytest.mark.parametrize("B,S,H,G,D,options", [(6, 2, 1, 1, 128, {"slopes": True}), (3, 6, 4, 1, 128, {"window": 2}), (2, 2, 16, 4, 128, {}),
                                               (7, 15, 2, 2, 120, {"softcap": 36.5}), (2, 45, 4, 1, 24, {"softcap": 49.4}), (1, 300, 2, 1, 64, {"window": 4}),
                                               (2, 5, 4, 2, 256, {})])
def test_rows_with_few_keys_are_off_by_their_rounding(gpu, B, S, H, G, D, options):
    """bf16: P and dx of rows with few keys enter the products in two parts, so that what is left is off by 2^-17 of each term, by fp32 sums and
    by 2^-16 in d_out . out: some 2^-14 of the result, a tenth of the rms of its own rounding (some 2^-9.2).  With one part the rounding of
    a row's one or two large dx, as large as the result's own, would add to it: 1.4 times and more."""
    gen = _gen(12)
    q, k, v = _qkv(gen, BF16, B, S, S, H, G, D)
    options = dict(options)
    if options.pop("slopes", False):
        options["slopes"] = torch.rand(H, generator=gen, device="cuda")
    g = _randn(gen, *q.shape)
    out = _ops().attention(q, k, v, **options)
    want = O.attention(q.detach(), k.detach(), v.detach(), d_out=g, **options)
    for name, got in zip(("out", "dq", "dk", "dv"), (out.detach(), *torch.autograd.grad(out, (q, k, v), g))):
        value = want[name][0]
        rounding = (value.to(BF16).double() - value).norm()
        assert (got.double() - value).norm() <= 1.2 * rounding, name


def test_document_ids_of_any_value(gpu):
    """The lowest and highest int32 as document ids, in and out of order: negative is padding, every other value is a document."""
    gen = _gen(6)
    q, k, v = _qkv(gen, BF16, 1, 300, 300, 4, 2, 64)
    ids = torch.full((1, 300), 2 ** 31 - 1, device="cuda", dtype=torch.int32)
    ids[:, 40:90], ids[:, 90:150:3], ids[:, 200:203] = -2 ** 31, 0, -1
    g = _randn(gen, *q.shape)
    out = _ops().attention(q, k, v, document_ids=ids)
    want = O.attention(q.detach(), k.detach(), v.detach(), document_ids=ids, d_out=g)
    for name, got in zip(("out", "dq", "dk", "dv"), (out.detach(), *torch.autograd.grad(out, (q, k, v), g))):
        _within(name, got, want[name])


@pytest.mark.parametrize("D", [64, 128])
def test_rows_far_apart(gpu, D):
    """Strides of 2^22 elements and more, for which the kernels' 32-bit offsets inside a tile are not used."""
    gen = _gen(7)
    far = (1 << 22) + 8
    keys = _randn(gen, 70 * far // 64, 64).view(-1)
    k = keys.as_strided((1, 70, 2, D), (0, far, D, 1))
    v = keys.as_strided((1, 70, 2, D), (0, far, D, 1), 1024)
    q = keys.as_strided((1, 70, 4, D), (0, D, 2 * far, 1), 4096)
    g = _randn(gen, 1, 70, 4, D)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = _ops().attention(*leaves)
    want = O.attention(q, k, v, d_out=g)
    for name, got in zip(("out", "dq", "dk", "dv"), (out.detach(), *torch.autograd.grad(out, leaves, g))):
        _within(name, got, want[name])


def test_a_long_cache(gpu):
    """Keys and values whose last rows lie beyond 2^31 elements of the tensor: the new token's attention is that of those keys alone."""
    gen = _gen(8)
    length, heads, D = 1_060_000, 16, 128   # 2.17e9 elements
    if torch.cuda.get_device_properties(0).total_memory < 40 << 30:
        pytest.skip("needs 20 GB")
    k, v = (torch.zeros(1, length, heads, D, device="cuda", dtype=BF16) for _ in range(2))
    last = 300
    k[:, -last:], v[:, -last:] = _randn(gen, 1, last, heads, D), _randn(gen, 1, last, heads, D)
    q = _randn(gen, 1, 2, 2 * heads, D)
    got = _ops().attention(q, k, v, window=last - 1)
    want = O.attention(q, k[:, -last:], v[:, -last:], window=last - 1)["out"]
    _within("out", got, want)


def test_norm_rope_of_a_strided_table(gpu):
    gen = _gen(3)
    q, k = _randn(gen, 2, 4, 2, 64), _randn(gen, 2, 4, 1, 64)
    cos, sin = torch.rand(9, 128, generator=gen, device="cuda")[:, ::2], torch.rand(9, 64, generator=gen, device="cuda")
    got = _ops().qk_norm_rope(q, k, cos, sin)       # a strided table
    want = O.norm_rope(q, None, cos, sin, torch.arange(4, device="cuda").expand(2, 4), 1e-5, q)
    _within("q", got[0], want["out"])


def test_prefixes_and_windows_of_any_value(gpu):
    """Prefix lengths from the lowest int32 to the highest; a window wider than any integer of the kernels."""
    gen = _gen(9)
    q, k, v = _qkv(gen, BF16, 5, 90, 130, 4, 2, 64)
    prefix = torch.tensor([-2 ** 31, -1, 0, 100, 2 ** 31 - 1], device="cuda", dtype=torch.int32)
    g = _randn(gen, *q.shape)
    out = _ops().attention(q, k, v, prefix_lengths=prefix, window=1 << 70)
    want = O.attention(q.detach(), k.detach(), v.detach(), prefix_lengths=prefix.clamp(min=0), d_out=g)
    for name, got in zip(("out", "dq", "dk", "dv"), (out.detach(), *torch.autograd.grad(out, (q, k, v), g))):
        _within(name, got, want[name])


def test_wide_float32_heads_are_reported_once(gpu):
    import warnings

    q = torch.zeros(1, 2, 2, 136, device="cuda")
    _ops()._warned_generic.discard(136)
    with pytest.warns(RuntimeWarning, match="head_dim 136"):
        _ops().attention(q, q, q)
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        _ops().attention(q, q, q)
        _ops().attention(q.to(BF16), q.to(BF16), q.to(BF16))


def test_refused_values(gpu):
    from picotron_amd._lib import PicomoeError

    q = torch.zeros(1, 2, 2, 64, device="cuda")
    table = torch.zeros(4, 64, device="cuda")
    for bad in (lambda: _ops().attention(q, q, q, scale=1e39), lambda: _ops().attention(q, q, q, softcap=1e-50), lambda: _ops().attention(q, q, q, softcap=1e39),
                lambda: _ops().attention(q, q, q, scale=1e10, softcap=1e-30), lambda: _ops().qk_norm_rope(q, q, table, table, eps=-1e-6),
                lambda: _ops().qk_norm_rope(q, q, table, table, eps=math.nan), lambda: _ops().embedding(torch.zeros(3, device="cuda", dtype=torch.int64), table, scale=1e39)):
        with pytest.raises(PicomoeError):
            bad()


def test_refusals(gpu):
    from picotron_amd._lib import PicomoeError

    ops = _ops()
    t = lambda *s, dtype=BF16: torch.zeros(*s, device="cuda", dtype=dtype)
    q, k = t(2, 4, 4, 64), t(2, 4, 2, 64)
    i32 = torch.int32
    for bad in (lambda: ops.attention(q, t(2, 4, 3, 64), t(2, 4, 3, 64)), lambda: ops.attention(q, k, t(2, 5, 2, 64)), lambda: ops.attention(q, k, k.float()),
                lambda: ops.attention(q.half(), k.half(), k.half()), lambda: ops.attention(t(2, 4, 4, 60), t(2, 4, 2, 60), t(2, 4, 2, 60)),
                lambda: ops.attention(t(2, 4, 4, 264), t(2, 4, 2, 264), t(2, 4, 2, 264)), lambda: ops.attention(q, k, k, softcap=-1.0),
                lambda: ops.attention(q, k, k, window=-1), lambda: ops.attention(q, k, k, scale=math.nan), lambda: ops.attention(q, k, k, causal=False, prefix_lengths=t(2, dtype=i32)),
                lambda: ops.attention(q, k, k, prefix_lengths=t(3, dtype=i32)), lambda: ops.attention(q, k, k, document_ids=t(2, 4, dtype=torch.int64)),
                lambda: ops.attention(q, k, k, document_ids=t(2, 5, dtype=i32)), lambda: ops.attention(q, k, k, slopes=t(4)),
                lambda: ops.attention(q, k, k, slopes=t(4, dtype=FP32).requires_grad_(True)), lambda: ops.attention(q, k, k.cpu()),
                lambda: ops.qk_norm_rope(q, k, t(4, 64), t(4, 64)), lambda: ops.qk_norm_rope(q, k, t(3, 64, dtype=FP32), t(3, 64, dtype=FP32)),
                lambda: ops.qk_norm_rope(q, t(2, 5, 2, 64), t(9, 64, dtype=FP32), t(9, 64, dtype=FP32)),
                lambda: ops.qk_norm_rope(q, k, t(9, 64, dtype=FP32), t(9, 64, dtype=FP32), q_weight=t(32)),
                lambda: ops.qk_norm_rope(q, k, t(9, 64, dtype=FP32), t(9, 64, dtype=FP32), k_weight=t(64, dtype=FP32)),
                lambda: ops.qk_norm_rope(q, k, t(9, 64, dtype=FP32), t(9, 64, dtype=FP32), positions=t(2, 4)),
                lambda: ops.qk_norm_rope(q, k, t(9, 64, dtype=FP32), t(9, 64, dtype=FP32), positions=t(2, 3, dtype=i32)),
                lambda: ops.embedding(t(3, dtype=FP32), t(5, 8)), lambda: ops.embedding(t(3, dtype=i32), t(5, 8).half()), lambda: ops.embedding(t(3, dtype=i32), t(8)),
                lambda: ops.embedding(t(3, dtype=i32), t(5, 8), padding_idx=5), lambda: ops.embedding(t(3, dtype=i32), t(5, 8), scale=math.inf)):
        with pytest.raises(PicomoeError):
            bad()


# ------------------------------------------------------------------------------------------------
# Together
# ------------------------------------------------------------------------------------------------
def _front(state):
    """Lookup, projections by one weight, norms + rotation, attention: the operators in a row, with their gradients."""
    ops, (ids, table, fused, qw, kw, cos, sin, docs, g) = _ops(), state
    x = ops.embedding(ids, table, scale=4.0, padding_idx=0)
    B, S, _ = x.shape
    q, k, v = (x @ fused).view(B, S, 8, 64).split([4, 2, 2], dim=2)
    q, k = ops.qk_norm_rope(q, k, cos, sin, qw, kw)
    out = ops.attention(q, k, v, softcap=10.0, document_ids=docs)
    return [out, *torch.autograd.grad(out, (table, fused, qw, kw), g)]


def _front_state(seed):
    gen = _gen(seed)
    leaf = lambda t: t.to(BF16).requires_grad_(True)
    docs = torch.zeros(2, 150, device="cuda", dtype=torch.int32)
    docs[:, 60:], docs[:, 140:] = 1, -1
    return (torch.randint(0, 50, (2, 150), generator=gen, device="cuda"), leaf(_randn(gen, 50, 96)), leaf(_randn(gen, 96, 512) / 10),
            leaf(_randn(gen, 64) * 0.1 + 1), leaf(_randn(gen, 64) * 0.1 + 1), torch.rand(150, 64, generator=gen, device="cuda"),
            torch.rand(150, 64, generator=gen, device="cuda"), docs, _randn(gen, 2, 150, 4, 64))


def test_operators_replay_in_a_hip_graph(gpu):
    states = [_front_state(s) for s in range(3)]
    want = [[t.detach().clone() for t in _front(s)] for s in states]
    static = [t.detach().clone().requires_grad_(t.requires_grad) for t in states[0]]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _front(static)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = _front(static)
    for i in (1, 2, 0, 1):
        with torch.no_grad():
            for to, t in zip(static, states[i]):
                to.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, want[i]):
            assert torch.equal(a, b), i
        eager = _front(states[(i + 1) % 3])   # eager work between the replays
        for a, b in zip(eager, want[(i + 1) % 3]):
            assert torch.equal(a, b)


def test_operators_on_two_streams_at_once(gpu):
    states = [_front_state(s) for s in range(2)]
    want = [[t.detach().clone() for t in _front(s)] for s in states]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in states]
    for _ in range(5):
        got = []
        for stream, state in zip(streams, states):
            with torch.cuda.stream(stream):
                got.append(_front(state))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


def _config(**kw):
    base = dict(vocab_size=97, hidden_size=256, intermediate_size=128, num_attention_heads=4, num_key_value_heads=2, num_hidden_layers=2,
                max_position_embeddings=128, rms_norm_eps=1e-5, rope_theta=10000.0, num_experts=4, num_experts_per_tok=2, num_shared_experts=1)
    base.update(kw)
    return types.SimpleNamespace(**base)


def _model(cfg, dtype, seed=0):
    from picotron_amd.model import Llama

    torch.manual_seed(seed)
    model = Llama(cfg)
    gen = torch.Generator().manual_seed(seed)
    with torch.no_grad():
        for name, p in model.named_parameters():
            base = 1.0 if "norm" in name else 0.0
            p.copy_(base + (1.0 if name == "embedding.weight" else 0.1 if base else 0.05) * torch.randn(p.shape, generator=gen))
    return model.to(dtype).cuda()


def test_fused_decoder_equals_the_plain_one(gpu):
    """The same fp32 weights through the library's attention and through the kernels: logits and gradients agree to fp32 rounding."""
    ids = torch.randint(0, 97, (2, 100), generator=_gen(1), device="cuda")
    g = torch.randn(2, 100, 97, generator=_gen(2), device="cuda")
    found = []
    for kw in ({}, dict(fused_attention=True, embedding_scale=1.0)):
        model = _model(_config(**kw), FP32)
        logits = model(ids)
        logits.backward(g)
        found.append((logits.detach(), {n: p.grad for n, p in model.named_parameters()}))
    (a, ga), (b, gb) = found
    assert torch.allclose(a, b, atol=2e-4, rtol=1e-4)
    assert ga.keys() == gb.keys()
    for n in ga:
        assert torch.allclose(ga[n], gb[n], atol=2e-5 + 1e-3 * float(ga[n].abs().max())), n


@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_decoder_with_everything(gpu, dtype):
    """Packed documents through a model with every option on: each document's logits are those of the document alone."""
    cfg = _config(qk_norm=True, attention_softcap=20.0, attention_window=30, attention_bias="distance", embedding_scale=2.0, num_experts=1, num_shared_experts=0)
    model = _model(cfg, dtype)
    names = [n for n, _ in model.named_parameters()]
    assert "decoder_layers.1.attention.q_norm.weight" in names and "decoder_layers.0.attention.k_norm.weight" in names
    ids = torch.randint(0, 97, (1, 90), generator=_gen(3), device="cuda")
    docs = torch.zeros(1, 90, device="cuda", dtype=torch.int32)
    docs[:, 40:], docs[:, 85:] = 1, -1
    positions = torch.cat([torch.arange(40), torch.arange(50)])[None].cuda()
    packed = model(ids, position_ids=positions, document_ids=docs)
    packed.float().sum().backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in model.parameters())
    # the same arithmetic on the same rows but for the order of sums inside the kernels: fp32 rounding, or a few bf16 roundings
    tol = dict(atol=1e-4, rtol=1e-4) if dtype == FP32 else dict(atol=0.1, rtol=0.05)
    for part in (slice(0, 40), slice(40, 85)):
        alone = model(ids[:, part])
        assert torch.allclose(packed[:, part], alone, **tol), float((packed[:, part] - alone).abs().max())
    prefix = model(ids, prefix_lengths=torch.tensor([40], device="cuda", dtype=torch.int32))
    assert torch.isfinite(prefix).all() and not torch.equal(prefix[:, :39], model(ids)[:, :39])


def test_layers_share_their_tables(gpu):
    """The fused path's fp32 tables are on the device once, and no layer holds a copy on the host after its first call; the plain path then still runs."""
    model = _model(_config(fused_attention=True), FP32)
    ids = torch.randint(0, 97, (2, 20), generator=_gen(5), device="cuda")
    first = model(ids)
    layers = list(model.decoder_layers)
    assert all(layer.cos is layers[0].cos and layer.sin is layers[0].sin and layer.cos.is_cuda for layer in layers)
    for layer in layers:
        layer.attention.fused = False
    plain = model(ids)
    assert torch.allclose(first, plain, atol=2e-4, rtol=1e-4)   # fp32 rounding, as above
    for layer in layers:
        layer.attention.fused = True
    assert torch.equal(model(ids), first)


def test_positions_of_one_row_for_a_batch(gpu):
    """[1, seq] positions serve every row of a batch, in the operator and through the model."""
    gen = _gen(11)
    q, k = _randn(gen, 3, 5, 4, 64), _randn(gen, 3, 5, 2, 64)
    cos, sin = torch.rand(9, 64, generator=gen, device="cuda"), torch.rand(9, 64, generator=gen, device="cuda")
    row = torch.tensor([[8, 0, 3, 3, 1]], device="cuda")
    for at in (row, row.int(), row[0], row.expand(3, 5)):
        for got, want in zip(_ops().qk_norm_rope(q, k, cos, sin, positions=at), _ops().qk_norm_rope(q, k, cos, sin, positions=row.repeat(3, 1))):
            assert torch.equal(got, want)
    model = _model(_config(fused_attention=True), FP32)
    ids = torch.randint(0, 97, (2, 30), generator=gen, device="cuda")
    row = torch.arange(30, device="cuda")[None] + 7
    assert torch.equal(model(ids, position_ids=row), model(ids, position_ids=row.repeat(2, 1)))


def test_head_norms_under_autocast(gpu):
    """fp32 parameters and bf16 heads: the norm weights are taken in the heads' type, their gradients come back in fp32."""
    import torch.nn.functional as F

    model = _model(_config(qk_norm=True), FP32)
    layer = model.decoder_layers[0]
    attention = layer.attention
    cos, sin = layer.tables.on(torch.device("cuda", torch.cuda.current_device()))
    x, g = torch.randn(2, 40, 256, generator=_gen(1), device="cuda"), _randn(_gen(2), 2, 40, 256)
    leaves = [attention.q_norm.weight, attention.k_norm.weight]
    with torch.autocast("cuda", dtype=BF16):
        got = attention.forward_fused(x, cos, sin)
    grads = torch.autograd.grad(got, leaves, g)
    heads = [F.linear(x.to(BF16), p.weight.to(BF16)).view(2, 40, -1, 64) for p in (attention.q_proj, attention.k_proj, attention.v_proj)]
    low = [w.detach().to(BF16).requires_grad_(True) for w in leaves]
    q, k = _ops().qk_norm_rope(heads[0], heads[1], cos, sin, *low, eps=1e-5)
    want = F.linear(_ops().attention(q, k, heads[2]).reshape(2, 40, 256), attention.out_proj.weight.to(BF16))
    assert got.dtype == BF16 and torch.equal(got, want)
    for a, b in zip(grads, torch.autograd.grad(want, low, g)):
        assert a.dtype == FP32 and torch.equal(a, b.float())
    with torch.autocast("cuda", dtype=BF16):
        logits = model(torch.randint(0, 97, (2, 40), generator=_gen(3), device="cuda"))
    logits.float().sum().backward()
    assert all(p.grad is not None and p.grad.dtype == FP32 and torch.isfinite(p.grad).all() for p in leaves)


def test_training_after_inference(gpu):
    """A model whose first call ran under inference mode trains afterwards: what the layers keep from that call are ordinary tensors."""
    for kw in ({}, dict(qk_norm=True, attention_bias="distance", embedding_scale=2.0)):
        model = _model(_config(rope_theta=4321.0, num_experts=1, num_shared_experts=0, **kw), FP32)
        ids = torch.randint(0, 97, (2, 20), generator=_gen(6), device="cuda")
        with torch.inference_mode():
            first = model(ids)
        logits = model(ids)
        logits.sum().backward()
        assert torch.equal(logits, first) and all(p.grad is not None for p in model.parameters())
