"""The operators of the decoder in front of the MoE layer, on this library's kernels.

* :func:`embedding` -- scaled token lookup (picotron/model.py:343-360); gradient summed by sorted tokens
* :func:`qk_norm_rope` -- RMS norm of each query and key head with the position rotation (picotron/model.py:29-36) in one pass
* :func:`attention` -- grouped-query attention (picotron/model.py:199-233) with capped scores, distance bias, document, prefix and
  window masks; also for a few new tokens over a long cache

All run on the GPU only, in float32 or bfloat16, compute in fp32, and give the same bits on every run.  Head tensors are
``[batch, length, heads, head_dim]`` -- as a projection's output viewed by heads -- and may be strided (slices of one fused
projection, an expanded batch); results are dense.  Nothing synchronises with the host, so every call can be captured into a
HIP graph.  Arguments that the kernels do not take raise ``PicomoeError``; values on the device are not looked at by the
host: token ids and positions outside their tables give NaN rows.
"""

import contextlib
import ctypes
import functools
import math
import warnings

import torch
from torch.autograd.function import once_differentiable

from picotron_amd import _lib


def _fail(message):
    raise _lib.PicomoeError(message)


def _same_device(what, first, *others):
    if not first.is_cuda:
        _lib.require_cuda(first)
    for t in others:
        if t is not None and t.device != first.device:
            _lib.require_cuda(t)
            _fail(f"{what}: tensors on {first.device} and {t.device}")


def _on(t):
    """Context in which t's device is the current one (the calls below are short: entering one costs as much as a launch)."""
    return _HERE if t.device.index == torch.cuda.current_device() else torch.cuda.device(t.device)


_HERE = contextlib.nullcontext()


def _stream():
    return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device())  # a tenth of what current_stream().cuda_stream costs


def _ptr(t):
    return None if t is None else t.data_ptr()


def _rows16(t):
    """t, or a copy of it, with a dense last dimension and rows that start on 16-byte boundaries."""
    if t.data_ptr() % 16 == 0 and (t.is_contiguous() or _strided16(t.shape, t.stride(), 16 // t.element_size())):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _strided16(shape, stride, step):
    return stride[-1] == 1 and all(n == 1 or s % step == 0 for n, s in zip(shape[:-1], stride[:-1]))


def _dense16(t):
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _strides(t):
    """{batch, length, head} strides for the C ABI; a dimension of one element has none."""
    return _stride_array(tuple(t.shape[:3]), t.stride()[:3])


@functools.lru_cache(maxsize=256)
def _stride_array(shape, stride):
    return (ctypes.c_int64 * 3)(*(0 if n == 1 else s for n, s in zip(shape, stride)))


def _integer(what, t):
    if t.dtype == torch.int64:
        return t.contiguous()
    if t.dtype != torch.int32:
        _fail(f"{what} must be int32 or int64, got {t.dtype}")
    return t.to(torch.int64).contiguous()


def _workspace(n_bytes, like, what):
    if n_bytes < 0:
        _fail(f"{what}: sizes that the kernels do not take")
    return torch.empty(max(n_bytes, 16), dtype=torch.uint8, device=like.device)


# ------------------------------------------------------------------------------------------------
# Embedding
# ------------------------------------------------------------------------------------------------
class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, weight, ids, scale, padding_idx):
        lib = _lib.load()
        dt = _lib.dtype_code(weight.dtype)
        vocab, hidden = weight.shape
        with _on(weight):
            table = weight.contiguous()
            out = table.new_empty((ids.numel(), hidden))
            _lib.check(
                lib.picomoe_embedding_fwd(_ptr(table), dt, vocab, hidden, _ptr(ids), ids.numel(), scale, _ptr(out), _stream()),
                "picomoe_embedding_fwd",
            )
        ctx.save_for_backward(ids)
        ctx.meta = (vocab, hidden, scale, padding_idx)
        return out.view(*ids.shape, hidden)

    @staticmethod
    @once_differentiable
    def backward(ctx, d_out):
        (ids,) = ctx.saved_tensors
        vocab, hidden, scale, padding_idx = ctx.meta
        lib = _lib.load()
        dt = _lib.dtype_code(d_out.dtype)
        with _on(d_out):
            d_out = d_out.contiguous()
            d_weight = d_out.new_empty((vocab, hidden))
            ws = _workspace(lib.picomoe_embedding_bwd_workspace_bytes(dt, ids.numel(), vocab, hidden), d_out, "embedding")
            _lib.check(
                lib.picomoe_embedding_bwd(_ptr(d_out), dt, _ptr(ids), ids.numel(), vocab, hidden, scale, padding_idx, _ptr(d_weight),
                                          _ptr(ws), ws.numel(), _stream()),
                "picomoe_embedding_bwd",
            )
        return d_weight, None, None, None


def embedding(ids, weight, scale=1.0, padding_idx=None):
    """``scale * weight[ids]``: ids (int64 or int32, any shape), weight ``[vocab, hidden]`` -> ``[*ids.shape, hidden]``.

    ``padding_idx``: a row that is looked up like any other and gets no gradient.  An id outside the table gives a row of NaN
    and no gradient.  The gradient of the table is dense; every row of it is the sum over its tokens in token order."""
    _same_device("embedding", weight, ids)
    if weight.dim() != 2 or weight.shape[0] < 1 or weight.shape[1] < 1:
        _fail(f"embedding: the table must be [vocab, hidden], got {tuple(weight.shape)}")
    if padding_idx is not None and not 0 <= padding_idx < weight.shape[0]:
        _fail(f"embedding: padding_idx {padding_idx} outside the table of {weight.shape[0]} rows")
    scale = float(scale)
    if not abs(scale) <= 3e38:
        _fail(f"embedding: scale {scale}")
    return _Embedding.apply(weight, _integer("embedding: ids", ids), scale, -1 if padding_idx is None else int(padding_idx))


# ------------------------------------------------------------------------------------------------
# Norm of query and key heads + position rotation
# ------------------------------------------------------------------------------------------------
class _QkNormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, cos, sin, positions, eps):
        lib = _lib.load()
        B, S, _, D = q.shape
        with _on(q):
            q, k = _rows16(q), _rows16(k)
            q_out, k_out = q.new_empty(q.shape), k.new_empty(k.shape)
            _lib.check(
                lib.picomoe_qk_norm_rope_fwd(
                    _ptr(q), _strides(q), q.shape[2], _ptr(k), _strides(k), k.shape[2], _lib.dtype_code(q.dtype), B, S, D,
                    _ptr(q_weight), _ptr(k_weight), eps, _ptr(cos), _ptr(sin), cos.shape[0], _ptr(positions),
                    _ptr(q_out), _ptr(k_out), _stream(),
                ),
                "picomoe_qk_norm_rope_fwd",
            )
        ctx.save_for_backward(q, k, q_weight, k_weight, cos, sin, positions)
        ctx.eps = eps
        return q_out, k_out

    @staticmethod
    @once_differentiable
    def backward(ctx, dq_out, dk_out):
        q, k, q_weight, k_weight, cos, sin, positions = ctx.saved_tensors
        lib = _lib.load()
        B, S, _, D = q.shape
        dt = _lib.dtype_code(q.dtype)
        with _on(q):
            dq_out, dk_out = _dense16(dq_out), _dense16(dk_out)
            dq, dk = q.new_empty(q.shape), k.new_empty(k.shape)
            dqw = q.new_empty((D,)) if q_weight is not None and ctx.needs_input_grad[2] else None
            dkw = q.new_empty((D,)) if k_weight is not None and ctx.needs_input_grad[3] else None
            ws = _workspace(lib.picomoe_qk_norm_rope_bwd_workspace_bytes(dt, B, S, q.shape[2], k.shape[2], D), q, "qk_norm_rope")
            _lib.check(
                lib.picomoe_qk_norm_rope_bwd(
                    _ptr(dq_out), _ptr(dk_out), _ptr(q), _strides(q), q.shape[2], _ptr(k), _strides(k), k.shape[2], dt, B, S, D,
                    _ptr(q_weight), _ptr(k_weight), ctx.eps, _ptr(cos), _ptr(sin), cos.shape[0], _ptr(positions),
                    _ptr(dq), _ptr(dk), _ptr(dqw), _ptr(dkw), _ptr(ws), ws.numel(), _stream(),
                ),
                "picomoe_qk_norm_rope_bwd",
            )
        return dq, dk, dqw, dkw, None, None, None, None


def _check_heads(what, head_dim, dtype, *named):
    _lib.dtype_code(dtype)
    if head_dim % 8 or not 8 <= head_dim <= 256:
        _fail(f"{what}: head_dim {head_dim}: a multiple of 8 up to 256 is needed")
    for name, t in named:
        if t.dtype != dtype:
            _fail(f"{what}: {name} is {t.dtype}, the others {dtype}")


def qk_norm_rope(q, k, cos, sin, q_weight=None, k_weight=None, eps=1e-5, positions=None):
    """``(rotate(norm(q)), rotate(norm(k)))``, dense, in the shapes of q ``[batch, seq, heads, head_dim]`` and k
    ``[batch, seq, kv_heads, head_dim]``.

    ``norm``: RMS norm over head_dim times the weight ``[head_dim]`` (None: no norm).  ``rotate``: rotate-half with the rows of
    the fp32 tables ``cos``, ``sin`` ``[n_positions, head_dim]`` (``model.rope_tables``) that ``positions`` (int64 or int32,
    ``[batch, seq]``, ``[1, seq]`` or ``[seq]``; None: 0, 1, 2, ...) names.  fp32 arithmetic, rounded once.  Gradients for q, k and the weights."""
    what = "qk_norm_rope"
    _same_device(what, q, k, cos, sin, q_weight, k_weight, positions)
    if q.dim() != 4 or k.dim() != 4 or q.shape[:2] != k.shape[:2] or q.shape[3] != k.shape[3] or q.shape[2] < 1 or k.shape[2] < 1:
        _fail(f"{what}: q {tuple(q.shape)} and k {tuple(k.shape)}: [batch, seq, heads, head_dim] with the same batch, seq and head_dim are needed")
    B, S, _, D = q.shape
    weights = [(n, w) for n, w in (("q_weight", q_weight), ("k_weight", k_weight)) if w is not None]
    _check_heads(what, D, q.dtype, ("k", k), *weights)
    for name, w in weights:
        if w.shape != (D,):
            _fail(f"{what}: {name} {tuple(w.shape)}, [{D}] is needed")
    if not 0 <= eps <= 3e38:
        _fail(f"{what}: eps {eps}")
    for name, t in (("cos", cos), ("sin", sin)):
        if t.dtype != torch.float32 or t.dim() != 2 or t.shape[1] != D or t.shape != cos.shape:
            _fail(f"{what}: {name} must be float32 [n_positions, {D}] like the other table, got {t.dtype} {tuple(t.shape)}")
        if t.requires_grad:
            _fail(f"{what}: no gradient for {name}")
    if positions is not None:
        if positions.shape not in ((B, S), (1, S), (S,)):
            _fail(f"{what}: positions {tuple(positions.shape)}, [{B}, {S}], [1, {S}] or [{S}] is needed")
        positions = _integer(f"{what}: positions", positions.expand(B, S))
    elif S > cos.shape[0]:
        _fail(f"{what}: {S} tokens, tables of {cos.shape[0]} positions")
    q_weight, k_weight = (w if w is None else _dense16(w) for w in (q_weight, k_weight))
    return _QkNormRope.apply(q, k, q_weight, k_weight, _dense16(cos), _dense16(sin), positions, float(eps))


# ------------------------------------------------------------------------------------------------
# Attention
# ------------------------------------------------------------------------------------------------
_warned_generic = set()


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, scale, softcap, causal, window, slopes, document_ids, prefix_lengths):
        lib = _lib.load()
        B, Sq, H, D = q.shape
        Sk, G = k.shape[1:3]
        dt = _lib.dtype_code(q.dtype)
        with _on(q):
            q, k, v = _rows16(q), _rows16(k), _rows16(v)
            out = q.new_empty((B, Sq, H, D))
            lse = q.new_empty((B, H, Sq), dtype=torch.float32)
            # what out's rounding left makes the backward's d_out . out exact; nothing else reads it
            residual = q.new_empty(q.shape) if q.dtype == torch.bfloat16 and any(ctx.needs_input_grad[:3]) else None
            ws = _workspace(lib.picomoe_attention_fwd_workspace_bytes(dt, B, Sq, Sk, H, G, D), q, "attention")
            _lib.check(
                lib.picomoe_attention_fwd(
                    _ptr(q), _strides(q), _ptr(k), _strides(k), _ptr(v), _strides(v), dt, B, Sq, Sk, H, G, D, scale, softcap, causal,
                    window, _ptr(slopes), _ptr(document_ids), _ptr(prefix_lengths), _ptr(out), _ptr(residual),
                    _ptr(lse), _ptr(ws), ws.numel(), _stream(),
                ),
                "picomoe_attention_fwd",
            )
        ctx.save_for_backward(q, k, v, out, residual, lse, slopes, document_ids, prefix_lengths)
        ctx.meta = (scale, softcap, causal, window)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, d_out):
        q, k, v, out, residual, lse, slopes, document_ids, prefix_lengths = ctx.saved_tensors
        scale, softcap, causal, window = ctx.meta
        lib = _lib.load()
        B, Sq, H, D = q.shape
        Sk, G = k.shape[1:3]
        dt = _lib.dtype_code(q.dtype)
        with _on(q):
            if Sq == 0 or Sk == 0:
                return tuple(torch.zeros(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v)) + (None,) * 7
            d_out = _dense16(d_out)
            dq, dk, dv = q.new_empty(q.shape), k.new_empty(k.shape), v.new_empty(v.shape)
            ws = _workspace(lib.picomoe_attention_bwd_workspace_bytes(dt, B, Sq, Sk, H, G, D), q, "attention")
            _lib.check(
                lib.picomoe_attention_bwd(
                    _ptr(d_out), _ptr(q), _strides(q), _ptr(k), _strides(k), _ptr(v), _strides(v), _ptr(out), _ptr(residual),
                    _ptr(lse), dt, B, Sq, Sk, H, G, D, scale, softcap, causal, window, _ptr(slopes), _ptr(document_ids), _ptr(prefix_lengths),
                    _ptr(dq), _ptr(dk), _ptr(dv), _ptr(ws), ws.numel(), _stream(),
                ),
                "picomoe_attention_bwd",
            )
        return (dq, dk, dv) + (None,) * 7


def attention(q, k, v, *, causal=True, scale=None, softcap=0.0, window=0, slopes=None, document_ids=None, prefix_lengths=None):
    """``softmax(scores) @ v``, dense, in the shape of q ``[batch, q_len, heads, head_dim]``; k and v
    ``[batch, kv_len, kv_heads, head_dim]``, head ``h`` reads key head ``h // (heads // kv_heads)``.  Gradients for q, k, v.

    The queries are the last ones: query ``s`` stands at position ``p = s + kv_len - q_len`` (one new token over a cache: q_len 1).

    Scores, for key position ``j``: ``x = scale * q.k`` (``scale`` default ``head_dim ** -0.5``); ``softcap > 0``:
    ``softcap * tanh(x / softcap)`` (1e-30 to 1e30, and ``scale / softcap`` not below float32's normal numbers); ``slopes`` (fp32 ``[heads]``): minus ``slopes[h] * |p - j|``.

    A query sees key j when all of these hold: ``causal`` is off or ``j <= p`` or ``j < prefix_lengths[b]`` (int32 ``[batch]``); ``window``
    is 0 or ``|p - j| < window``; ``document_ids`` (int32 ``[batch, kv_len]``, in any order) is None or
    ``document_ids[b, j] == document_ids[b, p] >= 0`` (negative: padding).  A query that sees nothing gets zeros and no gradient.
    What a query does not see has no influence on it, NaN and infinities included.

    Runs on the matrix pipes, except float32 heads wider than 128 (generic kernels: the same results, a one-time ``RuntimeWarning``)."""
    what = "attention"
    _same_device(what, q, k, v, slopes, document_ids, prefix_lengths)
    if q.dim() != 4 or k.dim() != 4 or k.shape != v.shape or q.shape[0] != k.shape[0] or q.shape[3] != k.shape[3]:
        _fail(f"{what}: q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}: [batch, length, heads, head_dim] with the same batch and "
              "head_dim, k and v of one shape, are needed")
    B, Sq, H, D = q.shape
    Sk, G = k.shape[1:3]
    if G < 1 or H < 1 or H % G:
        _fail(f"{what}: {H} query heads over {G} key heads")
    _check_heads(what, D, q.dtype, ("k", k), ("v", v))
    if q.dtype == torch.float32 and D > 128 and D not in _warned_generic:
        _warned_generic.add(D)   # once per width: the results are the same, only the speed is not
        warnings.warn(f"picotron_amd: float32 attention with head_dim {D} runs the generic kernels, not the matrix pipes (up to 128 does)",
                      RuntimeWarning, stacklevel=2)
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    softcap, window = float(softcap or 0.0), int(window or 0)
    if not abs(scale) <= 3e38 or not (softcap == 0 or 1e-30 <= softcap <= 1e30) or window < 0:
        _fail(f"{what}: scale {scale}, softcap {softcap} (0 or from 1e-30 to 1e30), window {window}")
    window = min(window, Sq + Sk)  # no query is that far from a key
    if slopes is not None:
        if slopes.dtype != torch.float32 or slopes.shape != (H,):
            _fail(f"{what}: slopes must be float32 [{H}], got {slopes.dtype} {tuple(slopes.shape)}")
        if slopes.requires_grad:
            _fail(f"{what}: no gradient for the slopes")
        slopes = slopes.contiguous()
    if document_ids is not None:
        if document_ids.dtype != torch.int32 or document_ids.shape != (B, Sk):
            _fail(f"{what}: document_ids must be int32 [{B}, {Sk}], got {document_ids.dtype} {tuple(document_ids.shape)}")
        document_ids = document_ids.contiguous()
    if prefix_lengths is not None:
        if not causal:
            _fail(f"{what}: prefix_lengths without causal")
        if prefix_lengths.dtype != torch.int32 or prefix_lengths.shape != (B,):
            _fail(f"{what}: prefix_lengths must be int32 [{B}], got {prefix_lengths.dtype} {tuple(prefix_lengths.shape)}")
        prefix_lengths = prefix_lengths.contiguous()
    return _Attention.apply(q, k, v, scale, softcap, int(bool(causal)), window, slopes, document_ids, prefix_lengths)
