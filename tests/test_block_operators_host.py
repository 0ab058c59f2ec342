"""CPU: refusals of the block operators by name, the layer's construction, and the C-ABI argument block."""
import ctypes as C
import re
import os

import pytest
import torch

import orbitssm_b200 as ob
from orbitssm_b200 import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
F32, BF = torch.float32, torch.bfloat16


def _qkv(B=1, L=4, H=2, Dk=8, Dv=8, dtype=F32):
    return torch.zeros(B, L, H, Dk, dtype=dtype), torch.zeros(B, L, H, Dk, dtype=dtype), torch.zeros(B, L, H, Dv, dtype=dtype)


def test_cpu_tensors_are_refused_by_name():
    q, k, v = _qkv()
    ld, s = torch.zeros(2), torch.zeros(1, 2, 8, 8)
    for who, call in (("linear_attention", lambda: ob.linear_attention(q, k, v, ld)),
                      ("linear_attention_step", lambda: ob.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], ld, s)),
                      ("block_norm", lambda: ob.block_norm(torch.zeros(2, 8), torch.zeros(2, 8))),
                      ("pack_activation", lambda: ob.pack_activation(torch.zeros(2, 8))),
                      ("unpack_activation", lambda: ob.unpack_activation(ob.PackedActivation(
                          torch.zeros(2, 8, dtype=torch.int8), torch.ones(2, 1, dtype=torch.uint8), F32)))):
        with pytest.raises(ValueError, match=who + ": got a CPU tensor"):
            call()


@pytest.mark.parametrize("change,error,text", [
    (dict(k=torch.zeros(1, 4, 1, 8)), ValueError, "as many key heads"),
    (dict(v=torch.zeros(1, 3, 2, 8)), ValueError, "expected q, k"),
    (dict(q=torch.zeros(1, 4, 2, 8, dtype=torch.float16)), NotImplementedError, "float32 or bfloat16"),
    (dict(k=torch.zeros(1, 4, 2, 8, dtype=BF)), ValueError, "one dtype"),
    (dict(log_decay=torch.zeros(3)), ValueError, "log_decay must be float32"),
    (dict(log_decay=torch.zeros(2, dtype=BF)), ValueError, "log_decay must be float32"),
    (dict(log_decay=torch.zeros(2, requires_grad=True)), ValueError, "constant of the layer"),
    (dict(state=torch.zeros(1, 2, 8, 4)), ValueError, "state must be float32"),
    (dict(state=torch.zeros(1, 2, 8, 8, dtype=BF)), ValueError, "state must be float32"),
])
def test_linear_attention_refusals(change, error, text):
    q, k, v = _qkv()
    args = dict(q=q, k=k, v=v, log_decay=torch.zeros(2), state=None) | change
    with pytest.raises(error, match=text):
        ob.linear_attention(**args)


def test_linear_attention_refuses_wide_heads_and_bad_scales():
    q, k, v = _qkv(Dk=257)
    with pytest.raises(NotImplementedError, match="widths 1..256"):
        ob.linear_attention(q, k, v, torch.zeros(2))
    with pytest.raises(NotImplementedError, match="widths 1..256"):
        ob.linear_attention(*_qkv(Dv=0), torch.zeros(2))
    lib = _lib.load()
    a = _lib.LaArgs(B=1, L=4, H=1, Dk=8, Dv=300, scale=1.0)
    assert lib.orbit_la_fwd(C.byref(a), _lib.F32, None) == 2 and b"1..256" in lib.orbit_last_error()
    a = _lib.LaArgs(B=1, L=4, H=1, Dk=8, Dv=8, scale=0.0)
    assert lib.orbit_la_fwd(C.byref(a), _lib.F32, None) == 1 and b"scale" in lib.orbit_last_error()
    a = _lib.LaArgs(B=1, L=4, H=1, Dk=8, Dv=8, scale=1.0)
    assert lib.orbit_la_fwd(C.byref(a), _lib.F32, None) == 1 and b"null" in lib.orbit_last_error()
    assert lib.orbit_la_bwd(C.byref(a), 7, None) == 1 and b"dtype" in lib.orbit_last_error()
    # no tokens, no sequences: nothing to launch
    assert lib.orbit_la_fwd(C.byref(_lib.LaArgs(B=0, L=4, H=1, Dk=8, Dv=8, scale=1.0)), _lib.F32, None) == 0


def test_step_refusals():
    q, k, v = (t[:, 0] for t in _qkv())
    ld, s = torch.zeros(2), torch.zeros(1, 2, 8, 8)
    with pytest.raises(ValueError, match="state is required"):
        ob.linear_attention_step(q, k, v, ld, None)
    with pytest.raises(ValueError, match="expected q, k"):
        ob.linear_attention_step(q[0], k[0], v[0], ld, s)


@pytest.mark.parametrize("kw,text", [
    (dict(h=torch.zeros(2, 4)), "h must have the shape"), (dict(gate=torch.zeros(2, 8, dtype=BF)), "gate must have the shape and dtype"),
    (dict(scale=torch.zeros(7)), "scale must be"), (dict(post_weight=torch.zeros(1, 8)), "post_weight must be"),
    (dict(pre_weight=torch.zeros(8, dtype=torch.int64)), "pre_weight must be"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"),
])
def test_block_norm_refusals(kw, text):
    args = dict(x=torch.zeros(2, 8), h=torch.zeros(2, 8)) | kw
    with pytest.raises(ValueError, match=text):
        ob.block_norm(**args)
    with pytest.raises(NotImplementedError, match="float32 or bfloat16"):
        ob.block_norm(torch.zeros(2, 8).double(), torch.zeros(2, 8).double())


def test_pack_refusals():
    with pytest.raises(NotImplementedError, match="float32 or bfloat16"):
        ob.pack_activation(torch.zeros(2, 8, dtype=torch.float16))
    for x in (torch.zeros(()), torch.zeros(3, 0)):
        with pytest.raises(ValueError, match="D > 0"):
            ob.pack_activation(x)
    q, e = torch.zeros(2, 40, dtype=torch.int8), torch.ones(2, 2, dtype=torch.uint8)
    for bad in ((q, e[:, :1], F32), (q.to(torch.int16), e, F32), (q, e.to(torch.int8), F32)):
        with pytest.raises(ValueError, match="int8 q"):
            ob.unpack_activation(ob.PackedActivation(*bad))
    with pytest.raises(NotImplementedError, match="float32 or bfloat16"):
        ob.unpack_activation(ob.PackedActivation(q, e, torch.float16))


def test_argument_block_mirrors_the_header():
    text = open(os.path.join(ROOT, "include", "orbit_b200.h")).read()
    body = re.search(r"typedef struct orbit_la_args \{(.*?)\} orbit_la_args;", text, flags=re.S).group(1)
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
    fields = []
    for decl in body.split(";"):
        if decl.strip():
            names = decl.strip().split(",")
            fields += [names[0].split()[-1].lstrip("*")] + [n.strip().lstrip("*") for n in names[1:]]
    assert fields == [f[0] for f in _lib.LaArgs._fields_]


def test_layer_configuration():
    c = ob.LinearAttentionConfig(64, 4)
    assert (c.d_key, c.d_value) == (16, 16)
    layer = ob.LinearAttention(c.to_dict())
    assert layer.init_state(3)["hidden_state"].shape == (3, 4, 16, 16) and layer.hidden_state_shape() == (4, 16, 16)
    assert bool((layer.log_decay < 0).all()) and bool((layer.log_decay.diff() > 0).all())
    for kw in (dict(d_model=65, n_heads=4), dict(d_model=64, n_heads=0), dict(d_model=64, n_heads=4, d_key=300),
               dict(d_model=64, n_heads=4, span_min=1.0), dict(d_model=64, n_heads=4, span_min=9.0, span_max=8.0),
               dict(d_model=2048, n_heads=4)):
        with pytest.raises(ValueError):
            ob.LinearAttentionConfig(**kw)
    with pytest.raises(TypeError):
        ob.LinearAttentionConfig.from_dict({"d_model": 64, "n_heads": 4, "width": 3})
    for ex in ({"precision": "ieee"}, {"chunk_size": 64}, {"checkpoint": True}, {"kernel_options": {"a": 1}}, {"backend": "torch"}):
        with pytest.raises(ValueError):
            ob.LinearAttention(c, ex)
    kept = layer.log_decay.clone()
    layer.to(BF)
    assert layer.q_proj.weight.dtype == BF and layer.log_decay.dtype == F32 and torch.equal(layer.log_decay, kept)
    layer.load_state_dict(ob.LinearAttention(c).state_dict())
    layer.float()
    with pytest.raises(ValueError, match="CPU tensor"):
        layer(torch.zeros(1, 3, 64))
    with pytest.raises(ValueError, match="expected x"):
        layer(torch.zeros(1, 3, 32))


def test_stack_checkpoint_modes():
    stack = ob.BlockStack.from_mixers([ob.LinearAttention(ob.LinearAttentionConfig(32, 2)) for _ in range(2)], 32, post_norm=True,
                                      gate=True, residual_scale=0.5)
    assert stack.checkpoint is None and stack.set_checkpoint("int8").checkpoint == "int8" and stack.set_checkpoint(None).checkpoint is None
    with pytest.raises(ValueError, match="None or 'int8'"):
        stack.set_checkpoint("fp8")
    assert {"layers.0.post_norm.weight", "layers.1.gate_proj.weight", "layers.1.scale"} <= set(stack.state_dict())
    stack.layers[0].mixer._cp = object()
    with pytest.raises(ValueError, match="context-parallel"):
        stack.set_checkpoint("int8")
