"""What the documentation of the encoder-layer operators promises and needs no GPU to be seen (contexts are never looked
into beyond the number of CUs)."""
import ctypes as C
import struct

import pytest

from hybrid_rag_system_amd import _native as N
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
