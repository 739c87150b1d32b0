"""Refusals of the encoder-layer operators: arguments are checked before the device is touched, so none of this needs a
GPU (the context handed in is never looked into)."""
import ctypes as C

import pytest
import torch

from hybrid_rag_system_amd import _native as N
from hybrid_rag_system_amd.engine import Engine
from oracle import layer_oracle as LO

ERR_ARG = -1
CTX = C.create_string_buffer(4096)
BUF = C.create_string_buffer(4096)


def _p(off=0):
    return C.c_void_p((C.addressof(BUF) + 63) // 64 * 64 + off)


def _refused(rc, *words):
    assert rc == ERR_ARG
    msg = N.last_error()
    assert all(w in msg for w in words), msg


def test_linear_refusals():
    f = N.lib().hrs_linear
    good = dict(ctx=CTX, dtype=0, x=_p(0), ldx=8, w=_p(256), ldw=8, bias=None, r=None, ldr=0, act=0, y=_p(512), ldy=8, m=2, n=8, k=8)
    call = lambda **kw: f(*{**good, **kw}.values(), None)
    _refused(call(ctx=None), "null ctx")
    for t in (2, 3, -1):
        _refused(call(dtype=t), "hrs_linear", "type")
    for a in (-1, 6):
        _refused(call(act=a), "activation")
    for kw in ({"m": -1}, {"n": -1}, {"k": -1}, {"m": 1 << 31}, {"n": 1 << 30}, {"k": 1 << 30}):
        _refused(call(**kw), "M=")
    for kw in ({"x": None}, {"w": None}, {"y": None}):
        _refused(call(**kw), "null operand")
    _refused(call(ldx=-8), "stride")
    _refused(call(ldy=7), "overlap")
    _refused(call(y=_p(0)), "may not be x")
    _refused(call(y=_p(256)), "may not be x")
    for kw in ({"x": _p(1)}, {"w": _p(257)}, {"y": _p(513)}, {"r": _p(1)}, {"bias": _p(2)}):
        _refused(call(**kw), "aligned")
    _refused(call(r=_p(512), ldr=16), "in place of the residual")
    assert call(m=0, x=None, w=None, y=None) == 0 and call(n=0, w=None, y=None) == 0  # nothing to do


def test_layer_norm_refusals():
    f = N.lib().hrs_layer_norm
    good = dict(ctx=CTX, dtype=0, x=_p(0), ldx=8, r=None, ldr=0, g=_p(256), b=None, eps=1e-5, y=_p(512), ldy=8, m=2, n=8)
    call = lambda **kw: f(*{**good, **kw}.values(), None)
    _refused(call(ctx=None), "null ctx")
    for t in (3, -1):
        _refused(call(dtype=t), "type")
    _refused(call(eps=-1e-9), "eps")
    _refused(call(eps=float("nan")), "eps")
    for kw in ({"x": None}, {"g": None}, {"y": None}):
        _refused(call(**kw), "null operand")
    for kw in ({"m": -1}, {"n": -1}, {"m": 1 << 31}, {"n": 1 << 30}):
        _refused(call(**kw), "M=")
    _refused(call(ldr=-1), "stride")
    _refused(call(ldy=4), "overlap")
    for kw in ({"x": _p(1)}, {"dtype": 2, "y": _p(514)}, {"g": _p(258)}, {"b": _p(1)}):
        _refused(call(**kw), "aligned")
    _refused(call(y=_p(0), ldy=16), "in place")
    _refused(call(r=_p(512), ldr=16), "in place")
    assert call(m=0, x=None, y=None, g=None) == 0 and call(n=0, x=None, y=None, g=None) == 0


def _attention_args(**kw):
    a = N.AttentionArgsC()
    a.q, a.k, a.v, a.out = (_p(i * 512).value for i in range(4))
    a.dtype, a.batch, a.q_heads, a.kv_heads, a.head_dim, a.scale = 0, 1, 2, 2, 16, 0.25
    a.q_stride[:], a.k_stride[:], a.v_stride[:] = (32, 32, 16), (32, 32, 16), (32, 32, 16)
    a.q_rows, a.k_rows = 4, 4
    for k, v in kw.items():
        if k.endswith("stride"):
            getattr(a, k)[:] = v
        else:
            setattr(a, k, v)
    return a


@pytest.mark.parametrize("entry", ["hrs_attention", "hrs_attention_workspace"])
def test_attention_refusals(entry):
    L = N.lib()
    size = C.c_size_t()
    call = lambda a, ctx=CTX: L.hrs_attention(ctx, C.byref(a), None) if entry == "hrs_attention" else L.hrs_attention_workspace(ctx, C.byref(a), C.byref(size))
    ptr = _p(2048).value
    _refused(call(_attention_args(), ctx=None), "null")
    for kw, word in (
        ({"dtype": 2}, "type"),
        ({"batch": -1}, "batch"),
        ({"q_heads": 3}, "multiple"),
        ({"q_heads": 0}, "heads"),
        ({"kv_heads": 0}, "heads"),
        ({"head_dim": 12}, "head_dim"),
        ({"head_dim": 0}, "head_dim"),
        ({"head_dim": 264}, "head_dim"),
        ({"q_rows": -1}, "q_rows"),
        ({"k_rows": 1 << 30}, "k_rows"),
        ({"scale": 0.0}, "scale"),
        ({"scale": -1.0}, "scale"),
        ({"scale": float("nan")}, "scale"),
        ({"scale": float("inf")}, "scale"),
        ({"softcap": -1.0}, "softcap"),
        ({"scale": 1e31}, "range"),
        ({"softcap": 1e-35}, "range"),
        ({"softcap": 1e32}, "range"),
        ({"softcap": float("nan")}, "softcap"),
        ({"slopes": ptr, "bias_table": ptr}, "exclude"),
        ({"bias_table": ptr, "bias_reach": -1}, "bias_reach"),
        ({"prefix_lens": ptr}, "causal"),
        ({"q_offs": ptr, "q_lens": ptr}, "exclude"),
        ({"k_stride": (32, -32, 16)}, "stride"),
    ):
        _refused(call(_attention_args(**kw)), "hrs_attention", word)
    if entry == "hrs_attention":
        for name in "qkv":
            _refused(call(_attention_args(**{name: None})), "null operand")
            _refused(call(_attention_args(out=getattr(_attention_args(), name))), "may not be an input")
            _refused(call(_attention_args(**{name: _p(1025).value})), "aligned")
        _refused(call(_attention_args(out=None)), "null operand")
        assert call(_attention_args(batch=0)) == 0 and call(_attention_args(q_rows=0, q=None, out=None)) == 0
    else:
        assert call(_attention_args()) == 0
        assert L.hrs_attention_workspace(CTX, C.byref(_attention_args()), None) == ERR_ARG


def test_attention_arguments_are_packed_as_the_header_lays_them_out():
    """Engine.attention packs hrs_attention_args in one go: the same bytes as the structure filled field by field."""
    a = _attention_args(softcap=3.0, bias_reach=7, q_offs=11 << 33, prefix_lens=5, bias_table=9, max_q=1 << 40, max_k=3, workspace=77, workspace_bytes=1 << 35)
    flat = []
    for name, _ in N.AttentionArgsC._fields_:
        v = getattr(a, name)
        flat += list(v) if hasattr(v, "__len__") else [v or 0]
    assert bytes(a) == N.ATTENTION_ARGS.pack(*flat)


def test_wrapper_refuses_host_tensors():
    eng = object.__new__(Engine)
    eng.device, eng._ctx = torch.device("cuda", 0), None
    x = torch.zeros(2, 8, dtype=torch.bfloat16)
    for call in (lambda: eng.linear(x, x), lambda: eng.layer_norm(x, torch.zeros(8)), lambda: eng.attention(x.view(1, 2, 1, 8), x.view(1, 2, 1, 8), x.view(1, 2, 1, 8))):
        with pytest.raises(ValueError, match="must be on cuda:0"):
            call()


def test_geometry_of_a_model_directory(tmp_path):
    from hybrid_rag_system_amd import weights as W

    assert W.EncoderConfig.from_dir(str(tmp_path)) == W.EncoderConfig() and not W.EncoderConfig().packs
    f = tmp_path / "config.json"
    f.write_text('{"model_type": "bert", "hidden_size": 1024, "num_attention_heads": 16, "num_hidden_layers": 24, "intermediate_size": 4096, "hidden_act": "gelu"}')
    cfg = W.EncoderConfig.from_dir(str(tmp_path))
    assert (cfg.hidden, cfg.heads, cfg.layers, cfg.inter, cfg.vocab, cfg.eps) == (1024, 16, 24, 4096, 30522, 1e-12) and cfg.packs
    for bad in ('{"model_type": "t5"}', '{"hidden_act": "relu"}', '{"position_embedding_type": "relative_key"}'):
        f.write_text(bad)
        with pytest.raises(ValueError, match="not the encoder"):
            W.EncoderConfig.from_dir(str(tmp_path))


def test_oracle_bounds_hold_for_a_plain_evaluation_and_catch_mistakes():
    """The bounds the GPU tests use, on the CPU: an fp32 evaluation rounded once keeps them, small planted mistakes (a
    key too many, a wrong alignment of the last query, the residual inside the activation) do not."""
    g = torch.Generator()
    g.manual_seed(0)
    rnd = lambda *s: torch.randn(s, generator=g)
    for t in (torch.bfloat16, torch.float16):
        x, w, b, r = rnd(9, 72).to(t), (rnd(33, 72) / 8).to(t), rnd(33), rnd(9, 33).to(t)
        y, bound = LO.linear(x, w, b, "gelu", r, t)
        z = x.float() @ w.float().t() + b
        assert ((torch.nn.functional.gelu(z) + r.float()).to(t).double() - y).abs().le(bound).all()
        assert not (torch.nn.functional.gelu(z + r.float()).to(t).double() - y).abs().le(bound).all()
        y, bound = LO.layer_norm(x, 1 + rnd(72) * 0.1, None, 1e-12, x, t)
        assert (bound < 0.1).all()
        q, k, v = rnd(20, 2, 16).to(t), rnd(30, 1, 16).to(t), rnd(30, 1, 16).to(t)
        o, bound = LO.attention(q, k, v, 20, 30, causal=True, prefix=7, slopes=torch.tensor([0.5, 0.1]), dtype=t)
        for shift, ok in ((0, True), (1, False)):
            pos = torch.arange(20)[:, None] + 10 + shift
            j = torch.arange(30)[None, :]
            s = torch.einsum("ihd,jd->hij", q.float(), k[:, 0].float()) / 4 - torch.tensor([0.5, 0.1])[:, None, None] * (j - pos).abs()
            s = s.masked_fill(~((j <= pos) | (j < 7)), float("-inf"))
            got = torch.einsum("hij,jd->ihd", torch.softmax(s, -1), v[:, 0].float()).to(t)
            assert bool((got.double() - o).abs().le(bound + 1e-30).all()) == ok
