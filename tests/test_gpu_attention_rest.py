"""bf16 attention, rows of fewer than 128 keys: P and dx enter the products in two parts, so that what their rounding to bf16 leaves is added.  The
forward keeps out and what out's own rounding left, so that its sums can be looked at to 2^-16."""

import pytest
import torch

from oracle import decoder_ops_oracle as O

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def _inputs(seed, batch, q_len, kv_len, heads, kv_heads, D, size=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    shapes = ((q_len, heads), (kv_len, kv_heads), (kv_len, kv_heads), (q_len, heads))
    q, k, v, g = (torch.randn(batch, n, h, D, generator=gen, device="cuda") for n, h in shapes)
    q, k = q * size, k * size
    return [t.to(BF16).requires_grad_(True) for t in (q, k, v)], g.to(BF16)


def _sums(out):
    """out before its rounding, to 2^-16: what the forward keeps for the backward."""
    residual = out.grad_fn.saved_tensors[4]
    assert residual.dtype == BF16 and residual.shape == out.shape
    return out.detach().double() + residual.double()


# Terms that enter a sum in two parts are off by 2^-16 at most.  Rows whose maximum moves after a tile has been added form P of that tile a second
# time, against the last maximum; the two differ by fp32 rounding, some 2^-22, which crosses one of bf16's rounding borders, 2^-7 apart, for one
# of 2^15 terms, off by 2^-7 then.  Over many rows: sqrt(2^-32 + 2^-15 2^-14) = 2^-14.2 of the sums.  (Where the second forming is of another
# number than the one that was rounded, 2^-9.3 of those terms is left: 2^-12 to 2^-13 of the sums of rows that cross a tile.)
LEFT = 2.0 ** -14


@pytest.mark.parametrize("window,size", [(20, 1.0), (20, 3.0), (60, 1.0), (60, 3.0), (100, 2.0)])
@pytest.mark.parametrize("D,batch,q_len,kv_len", [(64, 1, 300, 300), (128, 2, 200, 457), (256, 1, 150, 150), (128, 3, 4, 330)])
def test_windows_across_tiles(gpu, window, size, D, batch, q_len, kv_len):
    """Rows whose keys lie in two tiles: their running maximum moves, and that of the rows beside them."""
    (q, k, v), _ = _inputs(window + D, batch, q_len, kv_len, 4, 2, D, size)
    out = _call(q, k, v, window=window)
    value = O.attention(q.detach(), k.detach(), v.detach(), window=window)["out"][0]
    last = torch.arange(q_len, device="cuda") + kv_len - q_len
    first = (last - window + 1).clamp(min=0)
    crossing = first // 64 != last // 64
    off = _sums(out) - value
    for rows in (crossing, ~crossing):
        if rows.any():
            assert off[:, rows].norm() <= LEFT * value[:, rows].norm(), float(off[:, rows].norm() / value[:, rows].norm())


def _call(q, k, v, **options):
    from picotron_amd import decoder_ops

    return decoder_ops.attention(q, k, v, **options)


@pytest.mark.parametrize("size", [1.0, 8.0, 30.0])
def test_large_scores_in_bf16(gpu, size):
    """Scores up to thousands: the running maximum is moved many times, by any factor."""
    (q, k, v), g = _inputs(4, 1, 150, 150, 2, 1, 64, size)
    out = _call(q, k, v)
    want = O.attention(q.detach(), k.detach(), v.detach(), d_out=g)
    for name, got in zip(("out", "dq", "dk", "dv"), (out.detach(), *torch.autograd.grad(out, (q, k, v), g))):
        value, bound = want[name]
        assert ((got.double() - value).abs() <= bound + 2.0 ** -126).all(), name


@pytest.mark.parametrize("S,window,heads,kv_heads,D", [(300, 100, 2, 2, 64), (300, 100, 4, 1, 128), (420, 90, 6, 2, 128), (290, 110, 1, 1, 256)])
def test_last_rows_of_a_window_without_causality(gpu, S, window, heads, kv_heads, D):
    """At the end of a sequence a window's rows see fewer and fewer keys: those of fewer than 128 alone have an output gradient, so that dk and dv are
    their sums.  What is left of terms that enter in two parts, of fp32 sums and of d_out . out (2^-16) is a tenth of the rms of a gradient's own
    rounding (2^-9.3); terms in one part would add another 2^-9.3."""
    (q, k, v), g = _inputs(S, 1, S, S, heads, kv_heads, D)
    p = torch.arange(S, device="cuda")
    keys = (p + window - 1).clamp(max=S - 1) - (p - window + 1).clamp(min=0) + 1
    few = (keys < 128) & (p > S // 2)
    assert 0 < int(few.sum()) < 64
    g = torch.where(few[None, :, None, None], g, torch.zeros((), device="cuda", dtype=BF16))
    out = _call(q, k, v, window=window, causal=False)
    grads = torch.autograd.grad(out, (q, k, v), g)
    want = O.attention(q.detach(), k.detach(), v.detach(), d_out=g, window=window, causal=False)
    for name, got in zip(("dq", "dk", "dv"), grads):
        value = want[name][0]
        rounding = (value.to(BF16).double() - value).norm()
        assert (got.double() - value).norm() <= 1.2 * rounding, (name, float((got.double() - value).norm() / rounding))


def _documents(kind, batch, length):
    """[batch, length]: runs of tokens, some short, some begun inside a tile of 64, with padding among them; "scattered" has every document in two
    pieces."""
    lengths = {"short": [40, 5, 64, 1, 100, 30, 90, 127, 2, 60], "long": [300, 200, 140, 400, 129], "unequal": [700, 20, 128, 127, 3, 260]}[
        "short" if kind == "scattered" else kind]
    ids, number = [], 0
    while len(ids) < length:
        n = lengths[number % len(lengths)]
        ids += [-7 if number % 6 == 4 else (number * 37 % 101 if kind != "scattered" else number // 4 * 2 + number % 2)] * n
        number += 1
    rows = [ids[:length], ids[-length:] if kind == "short" else ids[:length][::-1]]
    return torch.tensor([rows[b % 2] for b in range(batch)], dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("kind,batch,q_len,kv_len,heads,kv_heads,D,options", [
    ("short", 2, 700, 700, 4, 1, 128, {}), ("short", 1, 500, 500, 2, 2, 64, {"softcap": 20.0}), ("long", 1, 1000, 1000, 6, 2, 64, {}),
    ("unequal", 2, 1200, 1200, 2, 1, 128, {"slopes": True}), ("short", 1, 300, 300, 2, 1, 256, {}), ("long", 1, 2600, 2600, 2, 1, 64, {}),
    ("long", 2, 700, 700, 4, 2, 128, {"window": 150}), ("short", 2, 400, 400, 5, 1, 72, {"causal": False}), ("long", 1, 600, 600, 2, 1, 128, {"prefix": 350}),
    ("scattered", 2, 600, 600, 4, 2, 128, {}), ("short", 2, 3, 700, 8, 2, 128, {}), ("unequal", 1, 200, 2000, 4, 2, 64, {}), ("short", 2, 150, 60, 4, 2, 64, {}),
    ("long", 1, 1, 700, 1, 1, 64, {"softcap": 5.0})])
def test_documents_in_a_row(gpu, kind, batch, q_len, kv_len, heads, kv_heads, D, options):
    """The first tokens of a document, wherever it begins, and all of a short one see few keys.  Their rows of out, to 2^-16, and of dq; dk and dv with
    an output gradient for them alone: each off by its own rounding, as above."""
    (q, k, v), g = _inputs(q_len + kv_len, batch, q_len, kv_len, heads, kv_heads, D)
    options = dict(options, document_ids=_documents(kind, batch, kv_len))
    if options.pop("slopes", False):
        options["slopes"] = 2.0 ** (-8.0 * torch.arange(1, heads + 1, device="cuda") / heads)
    if "prefix" in options:
        options["prefix_lengths"] = torch.full((batch,), options.pop("prefix"), dtype=torch.int32, device="cuda")
    masks = {n: options.get(n) for n in ("window", "document_ids", "prefix_lengths")}
    seen = O.seen(batch, q_len, kv_len, options.get("causal", True), masks["window"], masks["document_ids"], masks["prefix_lengths"], q.device).sum(-1)
    few = (seen > 0) & (seen < 128)
    assert few.any()
    g = torch.where(few[..., None, None], g, torch.zeros((), device="cuda", dtype=BF16))
    out = _call(q, k, v, **options)
    sums = _sums(out)
    grads = torch.autograd.grad(out, (q, k, v), g)
    want = O.attention(q.detach(), k.detach(), v.detach(), d_out=g, **options)
    value = want["out"][0]
    assert (sums - value)[few].norm() <= LEFT * value[few].norm(), float((sums - value)[few].norm() / value[few].norm())
    assert not out.detach()[seen == 0].any()
    for name, got in zip(("dq", "dk", "dv"), grads):
        value = want[name][0]
        rounding = (value.to(BF16).double() - value).norm()
        assert (got.double() - value).norm() <= 1.2 * rounding, (name, float((got.double() - value).norm() / rounding))


def test_a_document_packed_is_as_exact_as_alone(gpu):
    """40 tokens behind 500 others, and the same 40 alone: the same sums to 2^-16, the same gradients but for a rounding."""
    (q, k, v), g = _inputs(3, 1, 540, 540, 4, 2, 128)
    ids = torch.zeros(1, 540, dtype=torch.int32, device="cuda")
    ids[:, 500:] = 1
    last = [t.detach()[:, 500:].clone().requires_grad_(True) for t in (q, k, v)]
    packed, alone = _call(q, k, v, document_ids=ids), _call(*last)
    a, b = _sums(packed)[:, 500:], _sums(alone)
    assert (a - b).norm() <= 2 * LEFT * b.norm()
    for x, y in zip(torch.autograd.grad(packed, (q, k, v), g), torch.autograd.grad(alone, last, g[:, 500:].contiguous())):
        x, y = x[:, 500:].double(), y.double()
        assert ((x - y).abs() <= 2.0 ** -7 * y.abs() + 2.0 ** -12 * y.abs().max()).all()


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
@pytest.mark.parametrize("scale,softcap", [(0.125, 1e30), (0.125, 1e20), (1e-7, 1e30), (0.0, 1e30), (1e-37, 2.0)])
def test_the_largest_caps(gpu, dtype, scale, softcap):
    """Caps up to the largest that is taken: far above every score they change nothing."""
    from picotron_amd import _lib

    (q, k, v), g = _inputs(8, 1, 90, 90, 2, 1, 64)
    q, k, v = (t.detach().to(dtype).requires_grad_(True) for t in (q, k, v))
    g = g.to(dtype)
    out = _call(q, k, v, scale=scale, softcap=softcap)
    want = O.attention(q.detach(), k.detach(), v.detach(), scale=scale, softcap=softcap, d_out=g)
    for name, got in zip(("out", "dq", "dk", "dv"), (out.detach(), *torch.autograd.grad(out, (q, k, v), g))):
        value, bound = want[name]
        assert ((got.double() - value).abs() <= bound + 2.0 ** -126).all(), name
    for bad in ((0.125, 3e38), (0.125, 1.1e30), (1e-9, 1e30)):
        with pytest.raises(_lib.PicomoeError):
            _call(q, k, v, scale=bad[0], softcap=bad[1])


@pytest.mark.parametrize("batch,q_len,kv_len,heads,kv_heads,D,options", [
    (1, 1, 3000, 4, 4, 64, {}), (8, 1, 4096, 32, 8, 128, {}), (2, 1, 20000, 2, 1, 128, {"softcap": 20.0}), (1, 5, 1003, 8, 2, 64, {"window": 400}),
    (3, 2, 777, 6, 2, 72, {"slopes": True}), (1, 1, 700, 8, 2, 256, {}), (2, 7, 900, 4, 1, 128, {"documents": 150}), (1, 32, 500, 1, 1, 128, {"causal": False})])
def test_a_few_tokens_over_a_cache(gpu, batch, q_len, kv_len, heads, kv_heads, D, options):
    """Up to 32 rows of a key head take P in two parts whatever their number of keys: sums to 2^-16 of the terms."""
    (q, k, v), _ = _inputs(kv_len, batch, q_len, kv_len, heads, kv_heads, D)
    options = dict(options)
    if options.pop("slopes", False):
        options["slopes"] = 2.0 ** (-8.0 * torch.arange(1, heads + 1, device="cuda") / heads)
    if "documents" in options:
        options["document_ids"] = (torch.arange(kv_len, device="cuda") // options.pop("documents")).int().expand(batch, -1).contiguous()
    out = _call(q, k, v, **options)
    value = O.attention(q.detach(), k.detach(), v.detach(), **options)["out"][0]
    off = _sums(out) - value
    assert off.norm() <= LEFT * value.norm(), float(off.norm() / value.norm())


@pytest.mark.parametrize("slope", [0.5, 1.0, 2.0, 4.0])
@pytest.mark.parametrize("D,S", [(64, 800), (128, 800), (256, 400)])
def test_one_key_that_outweighs_many(gpu, slope, D, S):
    """Steep distance biases: every row sees hundreds of keys and one or two have all the weight.  Its P is 1, which bf16 holds; dx of the others, of
    the order of their P, must not carry the rounding of the large one through d_out . out.  Three roundings of 2^-9.3 are left, of the gradient, of
    dx, and of the lesser P in d_out . out: sqrt(3) times the gradient's own."""
    (q, k, v), g = _inputs(5, 2, S, S, 4, 2, D)
    options = {"slopes": torch.full((4,), slope, device="cuda")}
    out = _call(q, k, v, **options)
    want = O.attention(q.detach(), k.detach(), v.detach(), d_out=g, **options)
    for name, got in zip(("dq", "dk", "dv"), torch.autograd.grad(out, (q, k, v), g)):
        value = want[name][0]
        rounding = (value.to(BF16).double() - value).norm()
        assert (got.double() - value).norm() <= 3 ** 0.5 * rounding, (name, float((got.double() - value).norm() / rounding))


@pytest.mark.parametrize("gap", [5.3, 6.6, 7.8])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_a_later_key_that_outweighs_another(gpu, gap, D):
    """Two keys count, key 3 and, 2^gap times its weight, key 140, in a tile of its own; the others are 2^-20 of it.  dP - D of the heavy key is 2^-gap of
    dP: its P's rounding may not reach D.  dx of the two is off by its own rounding and by that of the light key's P in D, dq by its rounding
    besides: three times 2^-8 at most (the rows' scores are nearly the same, and so are their roundings)."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    S, late = 250, 140
    q, k, v, g = (torch.randn(1, S, n, D, generator=gen, device="cuda") for n in (2, 1, 1, 2))
    q, k = q * 0.02, k * 0.02
    q[..., 0], k[..., 0], k[:, 3, :, 0], k[:, late, :, 0] = D ** 0.5 * 0.6931, -20.0, 0.0, gap
    q, k, v = (t.to(BF16).requires_grad_(True) for t in (q, k, v))
    g = torch.where((torch.arange(S, device="cuda") >= late)[None, :, None, None], g, torch.zeros((), device="cuda")).to(BF16)
    want = O.attention(q.detach(), k.detach(), v.detach(), d_out=g)
    (dq,) = torch.autograd.grad(_call(q, k, v), q, g)
    value = want["dq"][0]
    assert (dq.double() - value).norm() <= 3 * 2.0 ** -8 * value.norm(), float((dq.double() - value).norm() / value.norm())


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
@pytest.mark.parametrize("q_len", [1, 40])
def test_scores_of_minus_infinity_weigh_nothing(gpu, dtype, q_len):
    """A key whose score is -inf has no weight; a query that has only such scores gets zeros, like one that sees no key."""
    gen = torch.Generator(device="cuda").manual_seed(2)
    q, k, v = (torch.randn(1, n, h, 64, generator=gen, device="cuda").to(dtype) for n, h in ((q_len, 2), (200, 1), (200, 1)))
    q[..., 0] = 1.0
    k[:, 50:100, :, 0] = -torch.inf
    got = _call(q, k, v, causal=False)
    keep = torch.cat([torch.arange(50), torch.arange(100, 200)]).cuda()
    value, bound = O.attention(q, k[:, keep], v[:, keep], causal=False)["out"]
    assert ((got.double() - value).abs() <= bound).all()
    k[..., 0] = -torch.inf
    assert not _call(q, k, v, causal=False).any()
