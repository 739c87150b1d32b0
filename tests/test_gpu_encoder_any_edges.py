"""Encoders of other geometries than the built-in one at the ends of what hrs_encode and hrs_encode_packed take."""

import pytest
import torch

from hybrid_rag_system_amd import weights as W
from test_gpu_encoder_any import eng  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu


def test_more_texts_than_one_launch_takes(eng):
    """2^24 texts of one token and some, padded and packed: the same rows as a part of them alone."""
    cfg = W.EncoderConfig(vocab=500, hidden=8, layers=1, heads=1, inter=8, max_pos=4)
    enc = eng.encoder(W.generate(cfg, 3), cfg)
    n = (1 << 24) + 5
    ids = torch.randint(0, 500, (n, 1), dtype=torch.int32, device="cuda")
    lens, offs = torch.ones(n, dtype=torch.int32, device="cuda"), torch.arange(n + 1, dtype=torch.int32, device="cuda")
    for out in (enc.encode_ids(ids, lens), enc.encode_packed(ids.view(-1), offs, 1)):
        for at in (0, (1 << 23) - 50, n - 100):
            assert torch.equal(out[at : at + 100], enc.encode_ids(ids[at : at + 100].contiguous(), lens[:100])), at
    enc.close()
