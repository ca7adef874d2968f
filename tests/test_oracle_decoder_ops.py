"""Pins oracle/decoder_ops_oracle.py on the CPU: gradients of the formulas against finite differences, masks against a loop,
softmax attention against the library's, and what is hidden having no influence."""

import math

import pytest
import torch
import torch.nn.functional as F

from oracle import decoder_ops_oracle as O


def _rand(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64)


def _differences(fn, x, d_out, step=1e-6):
    """d (fn(x) . d_out) / dx, central differences."""
    flat, grad = x.reshape(-1), torch.zeros(x.numel(), dtype=torch.float64)
    for i in range(x.numel()):
        keep = float(flat[i])
        flat[i] = keep + step
        up = float((fn() * d_out).sum())
        flat[i] = keep - step
        down = float((fn() * d_out).sum())
        flat[i] = keep
        grad[i] = (up - down) / (2 * step)
    return grad.view_as(x)


def test_embedding():
    ids = torch.tensor([[3, 0, 3], [9, -1, 2]])
    w, g = _rand(1, 5, 4), _rand(2, 2, 3, 4)
    found = O.embedding(ids, w, 2.0, 0, g)
    out = found["out"][0]
    assert torch.equal(out[0, 0], 2 * w[3]) and torch.isnan(out[1, :2]).all() and torch.equal(out[1, 2], 2 * w[2])
    dw = found["d_weight"][0]
    assert torch.allclose(dw[3], 2 * (g[0, 0] + g[0, 2])) and torch.allclose(dw[2], 2 * g[1, 2]) and not dw[[0, 1, 4]].any()


@pytest.mark.parametrize("weighted", [True, False])
def test_norm_rope_gradients(weighted):
    x, w, g = _rand(3, 2, 3, 2, 8), (_rand(4, 8) if weighted else None), _rand(5, 2, 3, 2, 8)
    cos, sin = _rand(6, 7, 8), _rand(7, 7, 8)
    pos = torch.tensor([[0, 6, 2], [3, 3, 1]])
    run = lambda: O.norm_rope(x, w, cos, sin, pos, 1e-5, g)["out"][0]
    found = O.norm_rope(x, w, cos, sin, pos, 1e-5, g)
    assert torch.allclose(found["dx"][0], _differences(run, x, g), atol=1e-6)
    if weighted:
        assert torch.allclose(found["dw"][0], _differences(run, w, g), atol=1e-6)
        n = x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-5) * w
    else:
        n = x
    a, b = n[..., :4], n[..., 4:]
    c, s = cos[pos][:, :, None], sin[pos][:, :, None]
    want = torch.cat([a * c[..., :4] - b * s[..., :4], b * c[..., 4:] + a * s[..., 4:]], dim=-1)
    assert torch.allclose(found["out"][0], want)


MASKS = [dict(), dict(causal=False), dict(window=2), dict(softcap=1.5), dict(causal=False, window=3, softcap=0.7),
         dict(prefix_lengths=torch.tensor([3, 0], dtype=torch.int32)),
         dict(document_ids=torch.tensor([[0, 0, 1, 1, 1], [2, -1, 2, 5, 2]], dtype=torch.int32)),
         dict(slopes=torch.tensor([0.5, 0.25, 0.1, 0.0]))]


@pytest.mark.parametrize("options", MASKS, ids=lambda o: ",".join(o) or "causal")
@pytest.mark.parametrize("q_len", [5, 3, 1, 7])
def test_attention_gradients(options, q_len):
    B, Sk, H, G, D = 2, 5, 4, 2, 8
    q, k, v, g = _rand(1, B, q_len, H, D), _rand(2, B, Sk, G, D), _rand(3, B, Sk, G, D), _rand(4, B, q_len, H, D)
    found = O.attention(q, k, v, d_out=g, **options)
    run = lambda: O.attention(q, k, v, **options)["out"][0]
    for name, x in (("dq", q), ("dk", k), ("dv", v)):
        assert torch.allclose(found[name][0], _differences(run, x, g), atol=1e-6), name
    # query by query
    for b in range(B):
        for h in range(H):
            for i in range(q_len):
                p, scores, rows = i + Sk - q_len, [], []
                for j in range(Sk):
                    ok = not options.get("causal", True) or j <= p or ("prefix_lengths" in options and j < int(options["prefix_lengths"][b]))
                    if options.get("window"):
                        ok = ok and abs(p - j) < options["window"]
                    if "document_ids" in options:
                        ids = options["document_ids"][b]
                        ok = ok and p >= 0 and int(ids[p]) >= 0 and int(ids[p]) == int(ids[j])
                    if not ok:
                        continue
                    s = float(q[b, i, h] @ k[b, j, h // 2]) / math.sqrt(D)
                    if options.get("softcap"):
                        s = options["softcap"] * math.tanh(s / options["softcap"])
                    if "slopes" in options:
                        s -= float(options["slopes"][h]) * abs(p - j)
                    scores.append(s)
                    rows.append(v[b, j, h // 2])
                want = torch.zeros(D, dtype=torch.float64)
                if rows:
                    want = torch.softmax(torch.tensor(scores, dtype=torch.float64), 0) @ torch.stack(rows)
                assert torch.allclose(found["out"][0][b, i, h], want, atol=1e-12)


def test_attention_is_the_librarys():
    q, k, v = _rand(1, 2, 9, 4, 16), _rand(2, 2, 9, 4, 16), _rand(3, 2, 9, 4, 16)
    want = F.scaled_dot_product_attention(*(t.transpose(1, 2) for t in (q, k, v)), is_causal=True).transpose(1, 2)
    assert torch.allclose(O.attention(q, k, v)["out"][0], want)


def test_what_is_hidden_reaches_nothing():
    ids = torch.tensor([[0, 0, 0, 1, 1, -1]], dtype=torch.int32)
    q, k, v, g = (_rand(i, 1, 6, 2, 8) for i in range(4))
    clean = O.attention(q, k, v, document_ids=ids, d_out=g)
    for t in (q, k, v, g):
        t[:, 5] = math.nan
        t[:, 3] = math.inf
    dirty = O.attention(q, k, v, document_ids=ids, d_out=g)
    for name in clean:
        for i in (0, 1):
            assert torch.equal(clean[name][i][:, :3], dirty[name][i][:, :3]), name
        assert not dirty[name][0][:, 5].any()
