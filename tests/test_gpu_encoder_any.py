"""Encoders of other geometries than the built-in one (hrs_encode and hrs_encode_packed on the engine's layer operators)
against the fp32 CPU oracle; tolerance as for the built-in geometry: cosine >= 0.999."""
import json
import os

import numpy as np
import pytest
import torch

from hybrid_rag_system_amd import weights as W
from oracle import encoder_oracle as EO

pytestmark = pytest.mark.gpu

COS_TOL = 0.999
GEOMETRIES = [
    dict(vocab=5000, hidden=1024, layers=3, heads=16, inter=4096, max_pos=512),  # the width of the 1024-deep collections
    dict(vocab=3000, hidden=768, layers=2, heads=12, inter=2048, max_pos=512),
    dict(vocab=2000, hidden=384, layers=2, heads=6, inter=1536, max_pos=300),  # built-in width, other heads
    dict(vocab=2000, hidden=384, layers=18, heads=12, inter=1536, max_pos=64),  # built-in geometry, more layers
    dict(vocab=1500, hidden=320, layers=2, heads=5, inter=777, max_pos=256),  # odd inner width
    dict(vocab=1200, hidden=64, layers=1, heads=8, inter=100, max_pos=40),
]


@pytest.fixture(scope="module")
def eng():
    from hybrid_rag_system_amd.engine import Engine

    e = Engine(0)
    yield e
    e.close()


def _cos(a, b):
    return (a * b).sum(1) / np.maximum(np.linalg.norm(a, axis=1) * np.linalg.norm(b, axis=1), 1e-30)


@pytest.mark.parametrize("g", GEOMETRIES, ids=lambda g: f"{g['hidden']}x{g['heads']}x{g['layers']}")
def test_padded_and_packed_match_the_oracle(eng, g):
    cfg = W.EncoderConfig(**g)
    assert cfg.packs
    w = W.generate(cfg, seed=7)
    enc = eng.encoder(w, cfg)
    rng = np.random.default_rng(g["hidden"])
    for lens in ([min(40, cfg.max_pos)], [3, 1, 17, 33, min(200, cfg.max_pos), 64 if cfg.max_pos >= 64 else 8, 2]):
        lens = np.asarray(lens, np.int32)
        S = int(lens.max()) + (5 if cfg.max_pos >= lens.max() + 5 else 0)
        ids = rng.integers(0, cfg.vocab, (len(lens), S)).astype(np.int32)
        want = EO.forward(w, ids, lens, cfg).numpy()
        padded = enc.encode_ids(torch.from_numpy(ids).cuda(), torch.from_numpy(lens).cuda())
        flat = np.concatenate([ids[b, :n] for b, n in enumerate(lens)])
        offs = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
        packed = enc.encode_packed(torch.from_numpy(flat).cuda(), torch.from_numpy(offs).cuda(), int(lens.max()))
        unhinted = enc.encode_packed(torch.from_numpy(flat).cuda(), torch.from_numpy(offs).cuda())
        for name, got in (("padded", padded), ("packed", packed), ("unhinted", unhinted)):
            got = got.cpu().numpy()
            assert np.isfinite(got).all() and np.abs(np.linalg.norm(got, axis=1) - 1).max() < 1e-5, name
            assert _cos(got, want).min() >= COS_TOL, (name, _cos(got, want))
            assert np.abs(got - want).max() < 5e-3 * np.sqrt(384 / cfg.hidden) + 2e-3, name
        # padding does not leak, an empty text is zeros, the others keep their rows
        ids2 = ids.copy()
        for b, n in enumerate(lens):
            ids2[b, n:] = rng.integers(0, cfg.vocab, S - n)
        assert torch.equal(enc.encode_ids(torch.from_numpy(ids2).cuda(), torch.from_numpy(lens).cuda()), padded)
        l2 = np.append(lens, 0).astype(np.int32)
        more = enc.encode_ids(torch.from_numpy(np.vstack([ids, ids[:1]])).cuda(), torch.from_numpy(l2).cuda())
        assert (more[-1] == 0).all() and _cos(more[:-1].cpu().numpy(), want).min() >= COS_TOL
    enc.close()


def test_calls_that_do_not_fit(eng):
    from hybrid_rag_system_amd._native import HrsError

    small = dict(vocab=100, layers=1, inter=64, max_pos=16)
    for bad in (dict(hidden=100, heads=4), dict(hidden=128, heads=3), dict(hidden=1040, heads=2)):
        cfg = W.EncoderConfig(**small, **bad)
        with pytest.raises(HrsError, match="hidden="):
            eng.encoder(W.generate(cfg, 1), cfg)
    cfg = W.EncoderConfig(**small, hidden=64, heads=2)
    enc = eng.encoder(W.generate(cfg, 1), cfg)
    ids, lens = torch.zeros((2, 17), dtype=torch.int32, device="cuda"), torch.ones(2, dtype=torch.int32, device="cuda")
    with pytest.raises(HrsError, match="positions"):
        enc.encode_ids(ids, lens)
    with pytest.raises(ValueError, match="offs"):
        enc.encode_packed(ids[0], lens.long())
    assert enc.encode_packed(ids[0, :0].contiguous(), torch.zeros(1, dtype=torch.int32, device="cuda")).shape == (0, 64)
    # offsets outside the ids are cut to them
    a = enc.encode_packed(ids[0, :10].contiguous(), torch.tensor([-3, 4, 1 << 30], dtype=torch.int32, device="cuda"))
    b = enc.encode_packed(ids[0, :10].contiguous(), torch.tensor([0, 4, 10], dtype=torch.int32, device="cuda"))
    assert torch.equal(a, b)
    enc.close()
    builtin = W.EncoderConfig(vocab=200, layers=1)
    assert not builtin.packs
    enc = eng.encoder(W.generate(builtin, 1), builtin)
    with pytest.raises(HrsError, match="padded"):
        enc.encode_packed(ids[0], torch.tensor([0, 17], dtype=torch.int32, device="cuda"))
    enc.close()


def test_model_directory_of_another_geometry(tmp_path):
    """HRS_MODEL_DIR with a config.json: the embedding function loads that geometry and embeds packed batches."""
    from safetensors.numpy import save_file

    from hybrid_rag_system_amd import store

    words = ["restart", "the", "nginx", "container", "backup", "disk", "array", "of", "server", "a"]
    vocab = ["[PAD]", "[UNK]", "[CLS]", "[SEP]"] + words + list("abcdefghijklmnopqrstuvwxyz") + ["##" + c for c in "abcdefghijklmnopqrstuvwxyz"]
    vocab += [f"[unused{i}]" for i in range(100 - len(vocab))]
    cfg = W.EncoderConfig(vocab=100, hidden=128, layers=2, heads=2, inter=320, max_pos=256)
    gen = W.generate(cfg, 5)
    save_file({W.hf_name(n): t for n, t in gen.items()}, os.path.join(tmp_path, "model.safetensors"))
    (tmp_path / "vocab.txt").write_text("\n".join(vocab) + "\n")
    (tmp_path / "config.json").write_text(json.dumps({"model_type": "bert", "vocab_size": 100, "hidden_size": 128, "num_hidden_layers": 2, "num_attention_heads": 2, "intermediate_size": 320,
                                                      "max_position_embeddings": 256, "layer_norm_eps": 1e-12, "hidden_act": "gelu"}))
    ef = store.HrsEmbeddingFunction(model_dir=str(tmp_path), batch_size=4)
    assert ef.cfg == cfg
    texts = ["restart the nginx container", "backup of the array", "a", "server " * 60, "the disk of a server", "container"]
    got = ef.embed_tensor(texts).cpu().numpy()
    assert got.shape == (6, 128)
    ids, lens = ef.tokenizer.encode_batch_python(texts)
    want = EO.forward(gen, ids, lens, cfg).numpy()
    assert _cos(got, want).min() >= COS_TOL
    assert len(ef(texts[:1])[0]) == 128
