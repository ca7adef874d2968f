"""Arguments of the decoder's operators that are refused before anything reaches the GPU: through the C ABI with pointers that are
never dereferenced on the host, and through the Python wrappers with CPU tensors."""

import copy
import ctypes
import gc
import types
import weakref

import pytest
import torch

from picotron_amd import _lib, decoder_ops

P = ctypes.c_void_p(64)          # never dereferenced: these calls return before any launch
ODD = ctypes.c_void_p(72)        # off the 16-byte grid
STRIDES = (ctypes.c_int64 * 3)(4 * 4 * 64, 4 * 64, 64)
ODD_STRIDES = (ctypes.c_int64 * 3)(4 * 4 * 64, 4 * 64 + 2, 64)


def test_embedding_arguments():
    lib = _lib.load()
    assert lib.picomoe_embedding_fwd(P, 7, 10, 64, P, 4, 1.0, P, None) == 1           # dtype
    assert lib.picomoe_embedding_fwd(P, 1, 0, 64, P, 4, 1.0, P, None) == 1            # empty table
    assert lib.picomoe_embedding_fwd(P, 1, 1 << 31, 64, P, 4, 1.0, P, None) == 1      # table rows beyond 31 bits
    assert lib.picomoe_embedding_fwd(P, 1, 10, (1 << 20) + 1, P, 4, 1.0, P, None) == 1
    assert lib.picomoe_embedding_fwd(None, 1, 10, 64, P, 4, 1.0, P, None) == 1
    assert lib.picomoe_embedding_fwd(None, 1, 10, 64, None, 0, 1.0, None, None) == 0  # no tokens
    need = lib.picomoe_embedding_bwd_workspace_bytes(1, 5000, 100, 64)
    # two buffers of keys and of tokens, two partial rows for each of 79 pieces
    assert need == 4 * 20000 + 79 * 2 * 64 * 4
    assert lib.picomoe_embedding_bwd_workspace_bytes(1, -1, 100, 64) == -1
    assert lib.picomoe_embedding_bwd_workspace_bytes(1, 1 << 31, 100, 64) == -1
    assert lib.picomoe_embedding_bwd(P, 1, P, 5000, 100, 64, 1.0, -1, P, P, need - 1, None) == 1   # workspace too small
    assert lib.picomoe_embedding_bwd(P, 1, P, 5000, 100, 64, 1.0, -1, P, ODD, need, None) == 1
    assert lib.picomoe_embedding_bwd(P, 1, P, 5000, 100, 64, 1.0, -1, None, P, need, None) == 1
    assert lib.picomoe_embedding_bwd(None, 1, P, 5000, 100, 64, 1.0, -1, P, P, need, None) == 1


def test_norm_rope_arguments():
    lib = _lib.load()

    def fwd(q=P, qs=STRIDES, heads=4, dtype=1, batch=2, seq=4, D=64, weight=None, cos=P, k=P):
        return lib.picomoe_qk_norm_rope_fwd(q, qs, heads, k, STRIDES, 4, dtype, batch, seq, D, weight, None, 1e-5, cos, P, 8, None, P, P, None)

    assert fwd(batch=0) == 0 and fwd(seq=0) == 0
    for bad in (dict(q=None), dict(qs=None), dict(qs=ODD_STRIDES), dict(heads=0), dict(heads=5000), dict(dtype=3), dict(batch=-1), dict(D=60), dict(D=264),
                dict(D=0), dict(cos=None), dict(cos=ODD), dict(q=ctypes.c_void_p(66)), dict(weight=ctypes.c_void_p(66)), dict(batch=1 << 16, seq=1 << 16)):
        assert fwd(**bad) == 1, bad
    assert lib.picomoe_qk_norm_rope_bwd_workspace_bytes(1, 2, 4, 4, 4, 60) == -1
    need = lib.picomoe_qk_norm_rope_bwd_workspace_bytes(1, 2, 4, 4, 4, 64)
    assert need > 0

    def bwd(dq_out=P, qw=P, dqw=P, ws=P, size=need):
        return lib.picomoe_qk_norm_rope_bwd(dq_out, P, P, STRIDES, 4, P, STRIDES, 4, 1, 2, 4, 64, qw, P, 1e-5, P, P, 8, None, P, P, dqw, None, ws, size, None)

    for bad in (dict(dq_out=None), dict(dq_out=ODD), dict(qw=None), dict(ws=None), dict(size=need - 1)):
        assert bwd(**bad) == 1, bad


def test_attention_arguments():
    lib = _lib.load()

    def fwd(q=P, qs=STRIDES, ks=STRIDES, dtype=1, batch=2, q_len=4, kv_len=4, heads=4, kv_heads=4, D=64, scale=0.1, softcap=0.0, causal=1, window=0, prefix=None,
            out=P, lse=P, ws=P, size=1 << 40):
        return lib.picomoe_attention_fwd(q, qs, P, ks, P, STRIDES, dtype, batch, q_len, kv_len, heads, kv_heads, D, scale, softcap, causal, window, None, None,
                                         prefix, out, None, lse, ws, size, None)

    assert fwd(batch=0) == 0 and fwd(q_len=0) == 0
    nan = float("nan")
    for bad in (dict(q=None), dict(q=ODD), dict(qs=None), dict(qs=ODD_STRIDES), dict(ks=ODD_STRIDES), dict(dtype=2), dict(batch=-1), dict(q_len=-1), dict(kv_len=-1),
                dict(kv_len=(1 << 28) + 1), dict(heads=6), dict(kv_heads=0), dict(heads=8192, kv_heads=1), dict(D=60), dict(D=264), dict(scale=nan), dict(scale=float("inf")),
                dict(softcap=-1.0), dict(softcap=nan), dict(softcap=float("inf")), dict(window=-1), dict(causal=0, prefix=P), dict(out=None), dict(out=ODD),
                dict(lse=None), dict(ws=None), dict(ws=ODD), dict(size=0), dict(q_len=1 << 28, heads=32, kv_heads=4)):
        assert fwd(**bad) == 1, bad
    for call in (lib.picomoe_attention_fwd_workspace_bytes, lib.picomoe_attention_bwd_workspace_bytes):
        assert call(1, 2, 4, 4, 4, 2, 64) >= 16 and call(1, 2, 4, 4, 4, 3, 64) == -1 and call(5, 2, 4, 4, 4, 2, 64) == -1
    need = lib.picomoe_attention_bwd_workspace_bytes(1, 2, 4, 4, 4, 4, 64)

    def bwd(g=P, out=P, lse=P, dq=P, dv=P, size=need, kv_len=4, q_len=4):
        return lib.picomoe_attention_bwd(g, P, STRIDES, P, STRIDES, P, STRIDES, out, None, lse, 1, 2, q_len, kv_len, 4, 4, 64, 0.1, 0.0, 1, 0, None, None, None, dq, P, dv,
                                         P, size, None)

    for bad in (dict(g=None), dict(g=ODD), dict(out=None), dict(lse=None), dict(dq=None), dict(dv=ODD), dict(size=need - 1), dict(kv_len=0), dict(q_len=0)):
        assert bwd(**bad) == 1, bad


def test_values_that_reach_no_kernel():
    """Strides below zero (offsets inside a tile are unsigned), factors that float32 does not hold, an eps that makes a norm NaN."""
    lib = _lib.load()
    for at in range(3):
        back = (ctypes.c_int64 * 3)(*(-64 if i == at else 64 for i in range(3)))
        assert lib.picomoe_attention_fwd(P, back, P, STRIDES, P, STRIDES, 1, 2, 4, 4, 4, 4, 64, 0.1, 0.0, 1, 0, None, None, None, P, None, P, P, 1 << 40, None) == 1
        assert lib.picomoe_attention_fwd(P, STRIDES, P, STRIDES, P, back, 1, 2, 4, 4, 4, 4, 64, 0.1, 0.0, 1, 0, None, None, None, P, None, P, P, 1 << 40, None) == 1
        assert lib.picomoe_attention_bwd(P, P, STRIDES, P, back, P, STRIDES, P, None, P, 1, 2, 4, 4, 4, 4, 64, 0.1, 0.0, 1, 0, None, None, None, P, P, P, P, 1 << 40, None) == 1
    assert lib.picomoe_attention_fwd(P, STRIDES, P, STRIDES, P, STRIDES, 1, 2, 4, 4, 4, 4, 64, -1e10, 1e-30, 1, 0, None, None, None, P, None, P, P, 1 << 40, None) == 1
    for eps in (-1e-5, float("nan"), float("inf")):
        assert lib.picomoe_qk_norm_rope_fwd(P, STRIDES, 4, P, STRIDES, 4, 1, 2, 4, 64, None, None, eps, P, P, 8, None, P, P, None) == 1
    for scale in (float("nan"), float("-inf")):
        assert lib.picomoe_embedding_fwd(P, 1, 10, 64, P, 4, scale, P, None) == 1
        assert lib.picomoe_embedding_bwd(P, 1, P, 4, 10, 64, scale, -1, P, P, 1 << 30, None) == 1


def test_caps_beyond_the_factors_range():
    """softcap log2(e) and scale / softcap are float32 factors: a cap that makes the first infinite or the second less than normal is refused."""
    lib = _lib.load()

    def refused(scale, softcap):
        fwd = lib.picomoe_attention_fwd(P, STRIDES, P, STRIDES, P, STRIDES, 1, 2, 4, 4, 4, 4, 64, scale, softcap, 1, 0, None, None, None, P, None, P, P, 1 << 40, None)
        bwd = lib.picomoe_attention_bwd(P, P, STRIDES, P, STRIDES, P, STRIDES, P, None, P, 1, 2, 4, 4, 4, 4, 64, scale, softcap, 1, 0, None, None, None, P, P, P, P, 1 << 40,
                                        None)
        return fwd == 1 and bwd == 1

    for scale, softcap in ((0.125, 3e38), (0.125, 2.4e38), (0.125, 1e37), (0.125, 1.1e30), (1e-9, 1e30), (-1e-9, 1e30), (1e-38, 2.0), (0.0, 2e30)):
        assert refused(scale, softcap), (scale, softcap)


def test_cpu_tensors_are_refused():
    q = torch.zeros(1, 2, 2, 64)
    table = torch.zeros(4, 64)
    for call in (lambda: decoder_ops.attention(q, q, q), lambda: decoder_ops.qk_norm_rope(q, q, table, table), lambda: decoder_ops.embedding(torch.tensor([1]), table)):
        with pytest.raises(_lib.PicomoeError):
            call()


@pytest.mark.parametrize("flag", [None, False, True])
def test_a_projection_bias_flag_is_no_distance_bias(flag):
    """Llama configurations carry attention_bias: False; such models are built as without the option."""
    from picotron_amd.model import Llama

    config = types.SimpleNamespace(vocab_size=50, hidden_size=64, intermediate_size=32, num_attention_heads=4, num_key_value_heads=2, num_hidden_layers=1,
                                   max_position_embeddings=8, rms_norm_eps=1e-5, rope_theta=10000.0, attention_bias=flag)
    attention = Llama(config).decoder_layers[0].attention
    assert not attention.fused and attention.slopes is None


def test_model_options():
    from picotron_amd.model import Llama

    base = dict(vocab_size=50, hidden_size=64, intermediate_size=32, num_attention_heads=4, num_key_value_heads=2, num_hidden_layers=1, max_position_embeddings=8,
                rms_norm_eps=1e-5, rope_theta=10000.0)
    plain = Llama(types.SimpleNamespace(**base))
    attention = plain.decoder_layers[0].attention
    assert not attention.fused and attention.q_norm is None and plain.embedding.scale is None
    model = Llama(types.SimpleNamespace(**base, qk_norm=True, attention_bias="distance", embedding_scale=8.0))
    attention = model.decoder_layers[0].attention
    assert attention.fused and attention.q_norm.weight.shape == (16,) and attention.slopes.tolist() == [0.25, 0.0625, 0.015625, 0.00390625]
    assert model.embedding.scale == 8.0
    extra = set(n for n, _ in model.named_parameters()) - set(n for n, _ in plain.named_parameters())
    assert extra == {"decoder_layers.0.attention.q_norm.weight", "decoder_layers.0.attention.k_norm.weight"}
    for option in (dict(fused_attention=True), dict(attention_softcap=30.0), dict(attention_window=4)):
        assert Llama(types.SimpleNamespace(**base, **option)).decoder_layers[0].attention.fused
    with pytest.raises(ValueError):
        Llama(types.SimpleNamespace(**base, attention_bias="alibi"))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float64])
def test_slopes_are_float32_whatever_the_default_type(dtype):
    """A model built with another default type has the fp32 slopes that the attention takes."""
    from picotron_amd.model import Llama

    config = types.SimpleNamespace(vocab_size=50, hidden_size=96, intermediate_size=32, num_attention_heads=12, num_key_value_heads=2, num_hidden_layers=1,
                                   max_position_embeddings=8, rms_norm_eps=1e-5, rope_theta=10000.0, attention_bias="distance")
    before = torch.get_default_dtype()
    torch.set_default_dtype(dtype)
    try:
        slopes = Llama(config).decoder_layers[0].attention.slopes
    finally:
        torch.set_default_dtype(before)
    assert slopes.dtype == torch.float32
    assert torch.equal(slopes, 2.0 ** (-8.0 * torch.arange(1, 13, dtype=torch.float32) / 12))


def test_no_layer_keeps_tables_that_it_does_not_read():
    """A layer that rotates by tables of the activations' type holds no others once it has run; the fp32 tables of the fused path are one copy per
    device for all layers, and go with the last of them."""
    from picotron_amd.model import Llama, rope_tables

    config = types.SimpleNamespace(vocab_size=50, hidden_size=64, intermediate_size=32, num_attention_heads=4, num_key_value_heads=2, num_hidden_layers=3,
                                   max_position_embeddings=40, rms_norm_eps=1e-5, rope_theta=12345.0)
    model = Llama(config)
    layers = list(model.decoder_layers)
    host = [weakref.ref(t) for layer in layers for t in (layer.cos, layer.sin)]
    for layer in layers:
        cos, sin = layer._rope(torch.zeros(1, 7, 64, dtype=torch.bfloat16))
        assert cos.dtype == sin.dtype == torch.bfloat16 and cos.shape == (7, 16)
    gc.collect()
    assert all(t() is None for t in host)
    cpu = torch.device("cpu")
    shared = layers[0].tables.on(cpu)
    assert all(layer.tables.on(cpu)[0] is shared[0] and layer.tables.on(cpu)[1] is shared[1] for layer in layers)
    for a, b in zip(shared, rope_tables(40, 16, 12345.0)):
        assert a.dtype == torch.float32 and torch.equal(a, b)
    twin = copy.deepcopy(model)   # holds its own
    assert torch.equal(twin.decoder_layers[1].tables.on(cpu)[0], shared[0])
    gone = weakref.ref(shared[0])
    del model, layers, layer, shared, a, b
    gc.collect()
    assert gone() is None


def test_tables_of_a_first_call_under_inference_mode_can_be_trained_with():
    from picotron_amd.model import Llama

    config = types.SimpleNamespace(vocab_size=50, hidden_size=64, intermediate_size=32, num_attention_heads=4, num_key_value_heads=2, num_hidden_layers=1,
                                   max_position_embeddings=40, rms_norm_eps=1e-5, rope_theta=54321.0)
    layer = Llama(config).decoder_layers[0]
    with torch.inference_mode():
        cos, sin = layer._rope(torch.zeros(1, 7, 64, dtype=torch.bfloat16))
        shared = layer.tables.on(torch.device("cpu"))
    for t in (layer.cos, layer.sin, *shared):
        assert not t.is_inference()
        x = torch.ones(t.shape, requires_grad=True)
        (x * t).sum().backward()


@pytest.mark.parametrize("parallel", [False, True])
def test_the_plain_paths_tables_are_in_the_type_of_the_layers_input(parallel):
    """Norm weights kept in fp32 make the norm's output fp32; the rotation tables stay in the type of the hidden states."""
    from picotron_amd.model import Llama

    config = types.SimpleNamespace(vocab_size=50, hidden_size=64, intermediate_size=32, num_attention_heads=4, num_key_value_heads=2, num_hidden_layers=1,
                                   max_position_embeddings=40, rms_norm_eps=1e-5, rope_theta=10000.0, parallel_block=parallel)
    layer = Llama(config).decoder_layers[0]
    seen = []
    layer.attention.forward = lambda n, cos, sin, *rest: seen.append((n.dtype, cos.dtype, sin.dtype)) or torch.zeros_like(n)
    layer.mlp.forward = torch.zeros_like
    layer(torch.ones(1, 5, 64, dtype=torch.bfloat16))
    assert seen == [(torch.float32, torch.bfloat16, torch.bfloat16)]
