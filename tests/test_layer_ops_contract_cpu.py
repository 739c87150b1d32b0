"""What the documentation of the encoder-layer operators promises and needs no GPU to be seen (contexts are never looked
into beyond the number of CUs)."""
import ctypes as C
import struct

import pytest
import torch

from hybrid_rag_system_amd import _native as N
from hybrid_rag_system_amd.engine import Engine
from test_layer_ops_cpu import _attention_args, _p

CTX = C.create_string_buffer(4096)
struct.pack_into("ii", CTX, 0, 0, 256)  # device 0 of 256 CUs


def _workspace(a):
    size = C.c_size_t(77)
    assert N.lib().hrs_attention_workspace(CTX, C.byref(a), C.byref(size)) == 0, N.last_error()
    return size.value


@pytest.mark.parametrize("shape", [dict(q_rows=1, k_rows=32768), dict(q_rows=300, k_rows=5000, batch=2), dict(q_rows=40, k_rows=100)])
def test_workspace_size_does_not_depend_on_addresses(shape):
    """Asked before the tensors exist, with any placeholders, it is enough for the call with the real ones."""
    need = _workspace(_attention_args(**shape))
    assert (need > 0) == (shape["k_rows"] > 1024)
    odd = {name: _p(2).value for name in ("q", "k", "v", "out")}
    for other in (odd, {name: 1 for name in odd}, {"out": _attention_args().q}):
        assert _workspace(_attention_args(**shape, **other)) == need
    # the aligned call takes that size, and no less
    for given in (0, need - 1):
        if need:
            a = _attention_args(**shape, workspace=_p(2048).value, workspace_bytes=given)
            assert N.lib().hrs_attention(CTX, C.byref(a), None) == -1 and f"workspace of {need} bytes" in N.last_error()


def test_inputs_that_require_a_gradient_are_refused():
    """While gradients are recorded, by name; without recording the same call goes on (here to the check of its device)."""
    eng = object.__new__(Engine)
    eng.device, eng._ctx = torch.device("cuda", 0), None
    b = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)
    calls = {
        "linear": (eng.linear, dict(x=b(2, 8), weight=b(4, 8), bias=torch.zeros(4), residual=b(2, 4))),
        "layer_norm": (eng.layer_norm, dict(x=b(2, 8), weight=torch.zeros(8), bias=torch.zeros(8), residual=b(2, 8))),
        "attention": (eng.attention, dict(q=b(1, 2, 1, 8), k=b(1, 2, 1, 8), v=b(1, 2, 1, 8), slopes=torch.zeros(1))),
        "attention with a table": (eng.attention, dict(q=b(1, 2, 1, 8), k=b(1, 2, 1, 8), v=b(1, 2, 1, 8), bias_table=torch.zeros(1, 3))),
    }
    for name, (call, kw) in calls.items():
        for arg in kw:
            with_grad = {**kw, arg: kw[arg].clone().requires_grad_()}
            with pytest.raises(ValueError, match="requires a gradient"):
                call(**with_grad)
            with torch.no_grad(), pytest.raises(ValueError, match="must be on cuda:0|bias_table"):
                call(**with_grad)
        with pytest.raises(ValueError, match="must be on cuda:0|bias_table"):
            call(**kw)


def test_a_geometry_that_is_not_built_is_refused_before_its_weights_are_read():
    """w holds as many pointers as the geometry says; a refused one says nothing."""
    w, out = (C.c_void_p * 8192)(), C.c_void_p()
    good = dict(vocab=100, hidden=128, layers=1, heads=2, inter=64, max_pos=16, eps=1e-12)
    for kw, word in ((dict(hidden=100, heads=4), "hidden=100"), (dict(hidden=8192), "hidden=8192"), (dict(heads=3), "heads=3"), (dict(inter=0), "intermediate"), (dict(layers=257), "layers=257"),
                     (dict(layers=0), "layers=0"), (dict(vocab=0), "vocabulary"), (dict(max_pos=0), "position"), ({}, "weight tensor 0 is null")):
        cfg = N.EncoderConfigC(**{**good, **kw})
        assert N.lib().hrs_encoder_load(CTX, C.byref(cfg), w, None, C.byref(out)) == -1 and word in N.last_error(), N.last_error()
