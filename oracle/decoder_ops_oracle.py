"""64-bit oracle for the decoder's operators in front of the MoE layer.  TEST INFRASTRUCTURE ONLY.

Each function evaluates the definition and its gradient from the formulas, in float64 on the device of its inputs, and bounds
how far a result may be off that was computed in fp32 from the same inputs, with the roundings that the kernels' comments
state, and rounded once to the inputs' type: ``(value, bound)`` pairs, the bound elementwise and absolute.

Unit roundoffs: u = 2^-24 for fp32 arithmetic; r = ``torch.finfo(dtype).eps / 2`` for a rounding to the inputs' type.  A sum of
n terms computed in any order is off by at most n u times the sum of the absolute terms.

tests/test_oracle_decoder_ops.py pins the formulas' gradients against finite differences and the masks against a loop.
"""

from __future__ import annotations

import math

import torch

U = 2.0 ** -24
# what an exponential or a product below fp32's normal range may lose: the hardware's exponential returns zero there
FLUSH = 2.0 ** -126


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


# ------------------------------------------------------------------------------------------------
def embedding(ids, weight, scale, padding_idx, d_out):
    """{"out", "d_weight"}: (value, bound).  ids outside the table: NaN rows, no gradient."""
    r, w = half_step(weight.dtype), weight.double()
    flat = ids.reshape(-1).long()
    good = (flat >= 0) & (flat < weight.shape[0])
    out = torch.where(good[:, None], w[flat.clamp(0, weight.shape[0] - 1)] * scale, torch.full((), math.nan, dtype=torch.float64, device=w.device))
    counted = good if padding_idx is None else good & (flat != padding_idx)
    g = d_out.double().reshape(len(flat), weight.shape[1])[counted] * scale
    rows = flat[counted]
    d_weight, total = torch.zeros_like(w).index_add_(0, rows, g), torch.zeros_like(w).index_add_(0, rows, g.abs())
    count = torch.bincount(rows, minlength=weight.shape[0]).double()[:, None]
    return {"out": (out.view(*ids.shape, w.shape[1]), (r + 2 * U) * out.abs().nan_to_num().view(*ids.shape, w.shape[1])),
            "d_weight": (d_weight, r * d_weight.abs() + (count + 3) * U * total)}


# ------------------------------------------------------------------------------------------------
def _turn(x):
    a, b = x.chunk(2, dim=-1)
    return torch.cat([-b, a], dim=-1)


def norm_rope(x, weight, cos, sin, positions, eps, d_out):
    """One of q and k: {"out", "dx", "dw"}: (value, bound); "dw" only with a weight.  positions [batch, seq]."""
    r, D = half_step(x.dtype), x.shape[-1]
    xd, g = x.double(), d_out.double()
    c, s = cos.double()[positions][:, :, None], sin.double()[positions][:, :, None]
    ac, as_ = c.abs(), s.abs()
    if weight is not None:
        w = weight.double()
        rms = torch.rsqrt(xd.square().mean(-1, keepdim=True) + eps)
        n = xd * rms
        y = n * w
        e_rms = (D + 8) * U          # relative: D-term sum of squares halved by the root, division, root, reciprocal
    else:
        n, y, e_rms, w, rms = xd, xd, 0.0, None, None
    out = y * c + _turn(y) * s
    swapped = lambda t: torch.cat(t.chunk(2, dim=-1)[::-1], dim=-1)
    size = y.abs() * ac + swapped(y.abs()) * as_
    found = {"out": (out, r * out.abs() + (e_rms + 6 * U) * size)}
    dy = g * c - _turn(g * s)
    dy_size = g.abs() * ac + swapped(g.abs() * as_)
    e_dy = 4 * U * dy_size
    if weight is None:
        found["dx"] = (dy, r * dy.abs() + e_dy)
        return found
    dn, dn_size = dy * w, dy_size * w.abs()
    mean = (dn * n).mean(-1, keepdim=True)
    mean_size = (dn_size * n.abs()).mean(-1, keepdim=True)
    dx = rms * (dn - n * mean)
    dx_size = rms * (dn_size + n.abs() * mean_size)
    found["dx"] = (dx, r * dx.abs() + (3 * e_rms + (D + 16) * U) * dx_size)
    rows = dy.shape[0] * dy.shape[1] * dy.shape[2]
    dw, dw_size = (dy * n).sum((0, 1, 2)), (dy_size * n.abs()).sum((0, 1, 2))
    found["dw"] = (dw, r * dw.abs() + (e_rms + (rows + 8) * U) * dw_size)
    return found


# ------------------------------------------------------------------------------------------------
def seen(batch, q_len, kv_len, causal, window, document_ids, prefix_lengths, device):
    """[batch, q_len, kv_len]: which keys each query sees."""
    p = torch.arange(q_len, device=device)[:, None] + (kv_len - q_len)
    j = torch.arange(kv_len, device=device)[None]
    m = (j <= p) if causal else torch.ones(q_len, kv_len, dtype=torch.bool, device=device)
    m = m[None].expand(batch, -1, -1)
    if prefix_lengths is not None:
        m = m | (j[None] < prefix_lengths[:, None, None])
    if window:
        m = m & ((p - j).abs() < window)[None]
    if document_ids is not None:
        at = p[:, 0].clamp(min=0)
        mine = torch.where((p[:, 0] >= 0)[None], document_ids[:, at], torch.full((), -1, dtype=document_ids.dtype, device=device)) if kv_len else \
            torch.full((batch, q_len), -1, device=device)
        m = m & (mine[:, :, None] == document_ids[:, None, :]) & (mine >= 0)[:, :, None]
    return m


def attention(q, k, v, *, causal=True, scale=None, softcap=0.0, window=0, slopes=None, document_ids=None, prefix_lengths=None, d_out=None):
    """{"out", "dq", "dk", "dv"}: (value, bound).  Keys that a query does not see take no part, NaN included: hidden factors
    are replaced by zeros pair by pair, which needs [.., q_len, kv_len, head_dim] only where k, v, q or d_out are not finite."""
    dtype, r = q.dtype, half_step(q.dtype)
    B, Sq, H, D = q.shape
    Sk, G = k.shape[1:3]
    scale = D ** -0.5 if scale is None else scale
    Q = q.double().transpose(1, 2)
    K, V = (t.double().transpose(1, 2).repeat_interleave(H // G, dim=1) for t in (k, v))
    m = seen(B, Sq, Sk, causal, window, document_ids, prefix_lengths, q.device)[:, None].expand(B, H, Sq, Sk)
    zero = torch.zeros((), dtype=torch.float64, device=q.device)

    def pairs(a, b):
        """a [.., Sq, D] . b [.., Sk, D] -> [.., Sq, Sk] on seen pairs, zero elsewhere"""
        return torch.where(m, a @ b.transpose(2, 3).contiguous(), zero)

    def over(w, b, mask):
        """sum over the last axis of w (zero where hidden) times rows of b, hidden pairs left out"""
        if bool(torch.isfinite(b).all()):
            return w @ b
        return torch.where(mask[..., None], w[..., None] * b[:, :, None], zero).sum(-2)

    x = pairs(Q, K) * scale
    size = abs(scale)
    e_z = (D + 4) * U * size * pairs(Q.abs(), K.abs())
    t = torch.tanh(x / softcap) if softcap else None
    z = softcap * t if softcap else x
    if softcap:
        # tanh from an exponential and a quotient: absolute error of some steps at 1; for large caps, whose scores that would
        # swamp, tanh itself: some steps of the value
        e_z = e_z + (16 * U * softcap if softcap <= 1024 else 8 * U * z.abs())
    if slopes is not None:
        away = (torch.arange(Sq, device=q.device)[:, None] + (Sk - Sq) - torch.arange(Sk, device=q.device)[None]).abs().double()
        z = z - slopes.double()[:, None, None] * away
        e_z = e_z + 2 * U * slopes.double().abs()[:, None, None] * away
    e_z = e_z + 6 * U * z.abs()
    top = torch.where(m, z, zero - math.inf).amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, zero, top)
    p = torch.where(m, torch.exp(z - top), zero)
    total = p.sum(-1, keepdim=True)
    P = torch.where(m, p / torch.where(total == 0, zero + 1, total), zero)
    # relative error of P: its own score, the scores in the normaliser, the exponentials, the sum
    e_p = e_z + torch.where(m, e_z, zero).amax(-1, keepdim=True) + (Sk + 32) * U + 2 * U * top.abs()
    o = over(P, V, m)
    o_size = over(P, V.abs(), m)
    e_o = r * o.abs() + over(torch.where(m, P * (e_p + r) + FLUSH, zero), V.abs(), m) + (Sk + 8) * U * o_size
    back = lambda a: a.transpose(1, 2)
    found = {"out": (back(o), back(e_o))}
    if d_out is None:
        return found
    g = d_out.double().transpose(1, 2)
    dP = pairs(g, V)
    delta = (g * o).sum(-1, keepdim=True)
    e_delta = (g.abs() * e_o).sum(-1, keepdim=True) + (D + 2) * U * (g.abs() * o.abs()).sum(-1, keepdim=True)
    slope = (1 - t * t) if softcap else torch.ones_like(x)
    dx = torch.where(m, P * (dP - delta) * slope * scale, zero)
    raw = torch.where(m, P * size, zero)
    e_dx = raw * slope * ((D + 2) * U * pairs(g.abs(), V.abs()) + e_delta) + (e_p + 8 * U) * dx.abs()
    if softcap:
        e_dx = e_dx + raw * (dP - delta).abs() * (2 * e_z / softcap + 16 * U)
    e_dx = torch.where(m, e_dx + r * dx.abs() + FLUSH * (1 + size * (dP - delta).abs()), zero)
    dq = over(dx, K, m)
    e_dq = r * dq.abs() + over(e_dx + (Sk + 8) * U * dx.abs(), K.abs(), m)
    mt = m.transpose(2, 3)
    group = lambda a: a.view(B, G, H // G, Sk, D).sum(2)
    dk = group(over(dx.transpose(2, 3), Q, mt))
    n = Sq * (H // G)
    e_dk = r * dk.abs() + group(over((e_dx + (n + 8) * U * dx.abs()).transpose(2, 3), Q.abs(), mt))
    dv = group(over(P.transpose(2, 3), g, mt))
    e_dv = r * dv.abs() + group(over(torch.where(m, P * (e_p + r + (n + 8) * U) + FLUSH, zero).transpose(2, 3), g.abs(), mt))
    found.update(dq=(back(dq), back(e_dq)), dk=(back(dk), back(e_dk)), dv=(back(dv), back(e_dv)))
    return found
