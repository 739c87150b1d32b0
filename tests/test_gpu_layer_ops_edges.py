"""hrs_linear, hrs_attention and hrs_layer_norm at the ends of what their documentation allows: score caps of any size,
infinities and NaN, weights far below a row's largest, very wide outputs.  Definitions and bounds: oracle/layer_oracle.py."""
import pytest
import torch

from oracle import layer_oracle as LO
from test_gpu_layer_ops import TYPES, _attention_case, _close, _gen, eng  # noqa: F401 (eng: a fixture)

pytestmark = pytest.mark.gpu


def _unaligned(t):
    """The same values at strides that are no multiple of 8 elements: the kernel for any alignment."""
    return torch.cat([t, t[..., :1]], -1)[..., : t.shape[-1]]


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
