"""hrs_linear, hrs_attention and hrs_layer_norm at the ends of what their documentation allows: score caps of any size,
infinities and NaN, weights far below a row's largest, very wide outputs.  Definitions and bounds: oracle/layer_oracle.py."""
import itertools
import math

import pytest
import torch

from oracle import layer_oracle as LO
from test_gpu_layer_ops import TYPES, _attention_case, _close, _gen, eng  # noqa: F401 (eng: a fixture)

pytestmark = pytest.mark.gpu


def _unaligned(t):
    """The same values at strides that are no multiple of 8 elements: the kernel for any alignment."""
    return torch.cat([t, t[..., :1]], -1)[..., : t.shape[-1]]


# ---- activations -------------------------------------------------------------------------------------
@pytest.mark.parametrize("act", ["none", "relu", "gelu", "gelu_tanh", "silu", "tanh"])
@pytest.mark.parametrize("m,k", [(3, 64), (40, 64), (40, 63), (700, 64)])
def test_linear_activations_of_infinities(eng, act, m, k):
    """A sum of +-inf goes through every activation as its definition says (gelu, its tanh form and silu have 0 * inf below
    zero), in every kernel; NaN stays NaN; large finite sums stay themselves or go to zero."""
    inf, nan = float("inf"), float("nan")
    b = torch.tensor([inf, -inf, nan, 3e4, -3e4, 1e38, -1e38, 0.0] * 32)
    x, w = torch.zeros(m, k, dtype=torch.bfloat16, device="cuda"), torch.zeros(256, k, dtype=torch.bfloat16, device="cuda")
    got = eng.linear(x, w, b.cuda(), activation=act).cpu().float()
    want = torch.tensor([inf, -inf, nan, 3e4, -3e4, 1e38, -1e38, 0.0]).double()
    if act in ("none", "relu", "tanh"):
        want = LO.activate(want, act)
    else:
        want[1], want[4], want[6] = nan, 0.0, 0.0
    want = want.float().bfloat16().float()
    assert torch.equal(torch.nan_to_num(got, nan=77.0), torch.nan_to_num(want, nan=77.0).repeat(32).expand(m, -1)), got[0, :8]


# ---- score caps --------------------------------------------------------------------------------------
@pytest.mark.parametrize("t", ["bf16", "fp16"])
@pytest.mark.parametrize("cap", [66.0, 100.0, 1e3, 1e4, 1e6, 1e9, 1e29])
def test_attention_large_caps(eng, t, cap):
    """A cap far above the scores changes them little and must not round them to its own size: documents, single tokens,
    scores on both sides of tanh's bend (66: scores reach 100)."""
    size = 5.0 if cap < 1e3 else 2.0
    _attention_case(eng, "packed", [70, 33, 130], [70, 150, 20], 2, 1, 64, t, True, None, cap, size=size, seed=1)
    _attention_case(eng, "padded", [1, 1], [700, 33], 4, 2, 128, t, True, None, cap, "slope", size=size, seed=2)
    _attention_case(eng, "padded", [40], [90], 2, 2, 32, t, False, None, cap, "table", 7, size=size, seed=3)
    rnd = _gen(4)
    q, k, v = (rnd(90, 2, 64).to(TYPES[t]) * f for f in (size, size, 1.0))
    got = eng.attention(*(_unaligned(x.cuda())[None] for x in (q, k, v)), softcap=cap)
    want, bound = LO.attention(q, k, v, 90, 90, cap=cap, dtype=TYPES[t])
    _close(got[0], want, bound)


# ---- infinities and NaN in a bias table ----------------------------------------------------------------
@pytest.mark.parametrize("cap", [0.0, 30.0])
@pytest.mark.parametrize("queries,aligned", [(200, True), (2, True), (200, False)])
def test_attention_table_with_nan_and_the_largest_value(eng, cap, queries, aligned):
    """NaN at one distance reaches every query that sees a key there and no other; at the table's end it stands for all
    distances beyond.  The type's largest value gives its key the whole weight."""
    rnd, nan, keys = _gen(3), float("nan"), 300
    q, k, v = rnd(1, queries, 2, 64).bfloat16(), rnd(1, keys, 2, 64).bfloat16(), rnd(1, keys, 2, 64).bfloat16()
    dq, dk, dv = q.cuda(), k.cuda() if aligned else _unaligned(k.cuda()), v.cuda()
    pos = torch.arange(queries) + keys - queries
    for at, value in ((-20, nan), (5, nan), (-21, nan), (21, nan), (-3, torch.finfo(torch.float32).max), (-21, float("-inf")), (0, float("-inf"))):
        table = rnd(2, 43) * 0.1
        table[1, at + 21] = value
        got = eng.attention(dq, dk, dv, causal=True, softcap=cap, bias_table=table.cuda())[0].cpu()
        want, bound = LO.attention(q[0], k[0], v[0], queries, keys, causal=True, cap=cap, table=torch.nan_to_num(table, nan=0.0), dtype=torch.bfloat16)
        if value != value:
            hit = pos + at >= 0 if at <= 0 else torch.zeros(queries, dtype=torch.bool)  # (keys behind are not seen)
            assert torch.isnan(got[:, 1]).all(-1).equal(hit) and torch.isnan(got[:, 1]).any(-1).equal(hit), at
            got[hit, 1], want[hit, 1] = 0.0, 0.0
        elif value > 0:
            has = pos + at >= 0
            assert torch.equal(got[has, 1], v[0, (pos + at)[has], 1])
            got[has, 1], want[has, 1] = 0.0, 0.0
        _close(got, want, bound + 1e-30, at)


# ---- infinities in keys and values that every query sees -------------------------------------------------
@pytest.mark.parametrize("t", ["bf16", "fp16"])
@pytest.mark.parametrize("queries,aligned", [(70, True), (1, True), (70, False)])
@pytest.mark.parametrize("dim", [64, 80])
def test_attention_infinite_value_of_the_last_key(eng, queries, aligned, dim, t):
    """A weight above zero times inf is inf, in that column alone, whether the last key ends a tile or not."""
    for keys in (1, 33, 64, 65, 70, 127, 2000):
        rnd = _gen(keys)
        q, k, v = ((rnd(1, n, 2, dim) * 0.5).to(TYPES[t]) for n in (queries, keys, keys))
        dq, dk, dv = q.cuda(), k.cuda(), v.cuda()
        dv[0, -1, 1, 3] = float("inf")
        if not aligned:
            dk, dv = _unaligned(dk), _unaligned(dv)
        got = eng.attention(dq, dk, dv)[0].cpu()
        assert (got[:, 1, 3] == float("inf")).all(), keys
        got[:, 1, 3] = 0
        want, bound = LO.attention(q[0], k[0], v[0], queries, keys, dtype=TYPES[t])
        want[:, 1, 3] = 0
        _close(got, want, bound, keys)


@pytest.mark.parametrize("t", ["bf16", "fp16"])
@pytest.mark.parametrize("queries,heads,aligned", [(70, 2, True), (1, 2, True), (70, 2, False), (20, 6, True)])
@pytest.mark.parametrize("dim", [8, 16, 40, 64, 80, 120, 136, 256])
def test_attention_infinite_key_has_no_weight(eng, queries, heads, aligned, dim, t):
    """A key whose products with every query are -inf weighs nothing, at every head width: as if it were not there."""
    rnd = _gen(dim)
    for keys, gone in ((90, 3), (70, 69), (1500, 777)):
        q, k, v = ((rnd(1, n, h, dim) * 0.5).to(TYPES[t]) for n, h in ((queries, heads), (keys, 2), (keys, 2)))
        q = q.abs() + 0.25
        dq, dk, dv = q.cuda(), k.cuda(), v.cuda()
        dk[0, gone, :, 0] = dk[0, gone, :, dim - 1] = dk[0, gone, :, dim // 2] = -float("inf")
        if not aligned:
            dk, dv = _unaligned(dk), _unaligned(dv)
        got = eng.attention(dq, dk, dv)[0].cpu()
        rest = [j for j in range(keys) if j != gone]
        want, bound = LO.attention(q[0], k[0, rest], v[0, rest], queries, keys - 1, dtype=TYPES[t])
        _close(got, want, bound, (keys, gone))


# ---- weights -----------------------------------------------------------------------------------------
@pytest.mark.parametrize("t", ["bf16", "fp16"])
@pytest.mark.parametrize("queries,aligned", [(70, True), (1, True), (70, False), (1, False)])
def test_attention_of_one_value_is_that_value(eng, queries, aligned, t):
    """All values alike: the weights' rounding cancels between numerator and denominator, in every kernel.  All but one of
    the weights stand just above the middle of two numbers of the type, the value just below a power of two."""
    step = torch.finfo(TYPES[t]).eps / 2  # of the numbers in [0.5, 1)
    weight, value = 0.5 + 0.55 * step, 2 - 2 * step
    q, k = torch.zeros(1, queries, 1, 64), torch.zeros(1, 101, 1, 64)
    q[..., 0], k[:, 1:, :, 0] = 1, -1
    v = torch.full((1, 101, 1, 64), value)
    q, k, v = (x.to(TYPES[t]).cuda() for x in (q, k, v))
    if not aligned:
        k, v = _unaligned(k), _unaligned(v)
    got = eng.attention(q, k, v, scale=-math.log(weight))
    assert (got == value).all(), got[0, 0, 0, 0].item()


@pytest.mark.parametrize("t", ["bf16", "fp16"])
@pytest.mark.parametrize("queries,heads,aligned", [(70, 520, True), (1, 520, True), (70, 1, True), (70, 1, False), (1, 1, False)])
def test_attention_many_small_weights_are_not_lost(eng, queries, heads, aligned, t):
    """One key of weight 1 and 2^17 of 2^-26 each, half of what rounds to nothing in fp16: together 2^-9, which moves the
    result by 2^-8.  520 heads (of the same numbers): a row's keys are not cut into chunks, which have maxima of their own."""
    n = 1 << 17
    q, k, v = torch.zeros(1, queries, 1, 32), torch.zeros(1, n + 1, 1, 32), torch.full((1, n + 1, 1, 32), -1.0)
    q[..., 0], k[:, 1:, :, 0], v[:, 0] = 1, -1, 1
    q, k, v = (x.to(TYPES[t]).cuda() for x in (q, k, v))
    if not aligned:
        k, v = _unaligned(k), _unaligned(v)
    got = eng.attention(*(x.expand(-1, -1, heads, -1) for x in (q, k, v)), scale=26 * math.log(2)).double()
    mass = n * 2.0**-26
    # The weights are exact but for the scale's rounding (2^-23 of an exponent of 26).  The running sum of weights takes a
    # tile of 32 keys at least with one rounding of 2^-24, the products 16 keys with one of 2^-23 at most.
    tol = LO.half_step(TYPES[t]) + (n / 32 + 2 * n / 16) * 2.0**-24 + 2 * mass * 2.0**-18
    assert (got - (1 - mass) / (1 + mass)).abs().max() <= tol


# ---- very wide outputs -------------------------------------------------------------------------------
@pytest.mark.parametrize("m,k,ld", [(1, 8, 8), (3, 40, 1), (2, 2048, 8), (17, 8, 8)])
def test_linear_more_features_than_one_launch_takes(eng, m, k, ld):
    """2^27 features and some: the rows of W overlap, so that they need little memory.  Equal to the products of their parts."""
    n = (1 << 27) + 40
    base, x = torch.randn(n * ld + k, device="cuda").bfloat16(), torch.randn(m, k, device="cuda").bfloat16()
    w, b, r = base.as_strided((n, k), (ld, 1)), torch.randn(n, device="cuda"), torch.randn(m, n, device="cuda").bfloat16()
    y = eng.linear(x, w, b, "relu", r)
    for at in (0, (1 << 25) - 100, (1 << 26) - 100, 3 * (1 << 25) - 100, n - 200):
        part = slice(at, at + 200)
        assert torch.equal(y[:, part], eng.linear(x, w[part], b[part], "relu", r[:, part])), at
    eng.linear(x, w, b, "relu", r, out=r)  # in place of the residual
    assert torch.equal(r, y)


@pytest.mark.parametrize("t", ["bf16", "fp16"])
@pytest.mark.parametrize("queries,aligned", [(150, True), (7, True), (150, False)])
def test_attention_keys_that_a_query_does_not_see_may_hold_anything(eng, queries, aligned, t):
    """NaN and infinities in keys behind a query (v stays finite): with every bias and cap, as if they were zero."""
    rnd = _gen(queries)
    keys = 200
    q, k, v = (rnd(1, n, 2, 64).to(TYPES[t]) for n in (queries, keys, keys))
    for i, (cap, kw) in enumerate(itertools.product((0.0, 30.0, 100.0), ({}, {"slopes": torch.tensor([0.5, 0.01])}, {"table": rnd(2, 31)}))):
        seen = keys - queries + 1 + i  # keys that query i sees
        bad = k.clone()
        bad[0, seen:, 0, i], bad[0, seen:, 1, 63] = float("nan"), float("inf")
        dk, dv = bad.cuda(), v.cuda()
        if not aligned:
            dk, dv = _unaligned(dk), _unaligned(dv)
        given = {("bias_table" if n == "table" else n): x.cuda() for n, x in kw.items()}
        got = eng.attention(q.cuda(), dk, dv, causal=True, softcap=cap, **given)[0, : i + 1].cpu()
        want, bound = LO.attention(q[0], k[0], v[0], queries, keys, causal=True, cap=cap, dtype=TYPES[t], **kw)
        if i < queries:
            _close(got, want[: i + 1], bound[: i + 1], (cap, list(kw)))
