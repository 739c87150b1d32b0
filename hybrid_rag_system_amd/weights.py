"""MiniLM-L6 geometry and weight sources for the encoder.

The reference loads `all-MiniLM-L6-v2` by NAME through sentence-transformers
(scripts/chromadb_helper.py:58-71), i.e. from the Hugging Face hub.  No weights or vocabulary exist
offline, so two sources are offered: a local directory with `model.safetensors` (real weights,
BERT key names), or a deterministic counter-based generator (same numbers on every machine; used by
tests and benchmarks, where only the arithmetic matters).

Tensor order (101 tensors, the order of `hrs_weights` in include/hrs.h):
  word_emb [V,H], pos_emb [P,H], type_emb [2,H], emb_ln_g [H], emb_ln_b [H], then per layer
  q_w [H,H], q_b, k_w, k_b, v_w, v_b, o_w [H,H], o_b, ln1_g, ln1_b, i_w [I,H], i_b [I], d_w [H,I], d_b, ln2_g, ln2_b
Linear weights are [out, in] (y = x @ w.T + b), as BERT stores them.
"""
import json
import os
import warnings
from dataclasses import dataclass, replace

import numpy as np


@dataclass(frozen=True)
class EncoderConfig:
    vocab: int = 30522
    hidden: int = 384
    layers: int = 6
    heads: int = 12
    inter: int = 1536
    max_pos: int = 512
    eps: float = 1e-12
    max_seq: int = 256  # sentence-transformers truncates all-MiniLM-L6-v2 inputs to 256 tokens

    @property
    def packs(self):
        """Whether the encoder takes texts back to back (Encoder.encode_packed): every geometry but the built-in one."""
        return not (self.hidden == 384 and self.heads == 12 and self.inter % 192 == 0 and self.inter <= 8 * 384 and self.layers <= 16)

    @classmethod
    def from_dir(cls, path):
        """The geometry a local model directory names in its `config.json` (BERT's keys); without that file, or without a
        key, the default's.  What the directory's sentence-transformers files say of pooling is checked (check_modules)."""
        check_modules(path)
        file = os.path.join(path, "config.json")
        raw = read_json(path, "config.json")
        keys = {"vocab": "vocab_size", "hidden": "hidden_size", "layers": "num_hidden_layers", "heads": "num_attention_heads", "inter": "intermediate_size",
                "max_pos": "max_position_embeddings", "eps": "layer_norm_eps"}
        for key, want in (("model_type", "bert"), ("hidden_act", "gelu"), ("position_embedding_type", "absolute")):
            if raw.get(key, want) != want:
                raise ValueError(f"{file}: {key} {raw[key]!r} is not the encoder built here ({want})")
        cfg = cls(**{ours: type(getattr(cls, ours))(raw[theirs]) for ours, theirs in keys.items() if theirs in raw})
        # texts are cut where the directory says, at 256 tokens where it does not, and never behind the last position
        length = read_json(path, "sentence_bert_config.json").get("max_seq_length") or read_json(path, "tokenizer_config.json").get("model_max_length") or cfg.max_seq
        length = min(int(length), cfg.max_pos)
        if length > 256 and not cfg.packs:
            warnings.warn(f"{path}: texts are cut at 256 tokens, the longest this geometry's kernels take, not at {length}", stacklevel=2)
            length = 256
        return replace(cfg, max_seq=length)


def read_json(path, *names):
    """A directory's JSON file, {} where it has none."""
    file = os.path.join(path, *names)
    if not os.path.exists(file):
        return {}
    with open(file, encoding="utf-8") as f:
        return json.load(f)


def check_modules(path):
    """What stands behind the transformer in a model directory (modules.json, the pooling's config.json): the encoder here
    takes the mean over the tokens and gives rows of unit length.  Another pooling or another module is another embedding:
    ValueError.  Without a Normalize module the model's own rows have other lengths (and the same directions): a warning."""
    modules = read_json(path, "modules.json") or [{"type": "Transformer", "path": ""}, {"type": "Pooling", "path": "1_Pooling"}, {"type": "Normalize"}]
    for m in modules:
        kind = m["type"].split(".")[-1]
        if kind not in ("Transformer", "Pooling", "Normalize"):
            raise ValueError(f"{path}: module {m['type']} is not built here (a mean over tokens, of unit length, is)")
        if kind == "Pooling":
            raw = read_json(path, m["path"], "config.json")
            modes = [k[len("pooling_mode_") :] for k, v in raw.items() if k.startswith("pooling_mode_") and v]
            modes += [raw["pooling_mode"]] if "pooling_mode" in raw else []
            if raw and modes not in (["mean_tokens"], ["mean"]):
                raise ValueError(f"{os.path.join(path, m['path'])}: pooling by {' and '.join(modes) or 'nothing'} is not built here (the mean over tokens is)")
    if not any(m["type"].split(".")[-1] == "Normalize" for m in modules):
        warnings.warn(f"{path}: the model does not normalise its embeddings, the rows given here have unit length", stacklevel=3)


def tensor_specs(cfg):
    H, I = cfg.hidden, cfg.inter
    specs = [("word_emb", (cfg.vocab, H)), ("pos_emb", (cfg.max_pos, H)), ("type_emb", (2, H)), ("emb_ln_g", (H,)), ("emb_ln_b", (H,))]
    for l in range(cfg.layers):
        p = f"l{l}."
        specs += [
            (p + "q_w", (H, H)), (p + "q_b", (H,)), (p + "k_w", (H, H)), (p + "k_b", (H,)), (p + "v_w", (H, H)), (p + "v_b", (H,)),
            (p + "o_w", (H, H)), (p + "o_b", (H,)), (p + "ln1_g", (H,)), (p + "ln1_b", (H,)),
            (p + "i_w", (I, H)), (p + "i_b", (I,)), (p + "d_w", (H, I)), (p + "d_b", (H,)), (p + "ln2_g", (H,)), (p + "ln2_b", (H,)),
        ]
    return specs


def _mix(x):
    x = (x + np.uint64(0x9E3779B97F4A7C15)) & np.uint64(0xFFFFFFFFFFFFFFFF)
    x = ((x ^ (x >> np.uint64(30))) * np.uint64(0xBF58476D1CE4E5B9)) & np.uint64(0xFFFFFFFFFFFFFFFF)
    x = ((x ^ (x >> np.uint64(27))) * np.uint64(0x94D049BB133111EB)) & np.uint64(0xFFFFFFFFFFFFFFFF)
    return x ^ (x >> np.uint64(31))


def _uniform(seed, tensor_index, n):
    """n uniforms in (-1, 1), keyed (seed, tensor, element) -- pure integer hashing, so bit-identical everywhere."""
    with np.errstate(over="ignore"):
        idx = np.arange(n, dtype=np.uint64)
        h = _mix(_mix(np.uint64(seed) ^ (np.uint64(tensor_index + 1) * np.uint64(0xD1B54A32D192ED03))) + idx)
    return ((h >> np.uint64(11)).astype(np.float64) / float(1 << 53) * 2.0 - 1.0).astype(np.float32)


def generate(cfg=EncoderConfig(), seed=2026):
    """Deterministic weights, uniform with per-kind scales chosen so that the random network behaves like an
    embedding model rather than collapsing every input onto one direction: word embeddings dominate the
    position / type embeddings and the biases (the part common to all inputs), and the sub-layers add to the
    residual stream without swamping it.  Unrelated random inputs then embed at cosine ~0.2 (with equal
    scales everywhere it is ~0.99 and bf16-vs-fp32 rank comparisons are meaningless)."""
    out = {}
    for t, (name, shape) in enumerate(tensor_specs(cfg)):
        n = int(np.prod(shape))
        u = _uniform(seed, t, n).reshape(shape)
        base = name.split(".")[-1]
        if base.endswith("_g"):
            w = 1.0 + 0.1 * u
        elif base.endswith("_b"):
            w = 0.01 * u
        elif base == "word_emb":
            w = 0.5 * u
        elif base in ("pos_emb", "type_emb"):
            w = 0.02 * u
        else:
            w = u * np.float32(0.6 / np.sqrt(shape[1]))  # var = 0.12 / fan_in
        out[name] = np.ascontiguousarray(w.astype(np.float32))
    return out


_HF_LAYER = {
    "q_w": "attention.self.query.weight", "q_b": "attention.self.query.bias",
    "k_w": "attention.self.key.weight", "k_b": "attention.self.key.bias",
    "v_w": "attention.self.value.weight", "v_b": "attention.self.value.bias",
    "o_w": "attention.output.dense.weight", "o_b": "attention.output.dense.bias",
    "ln1_g": "attention.output.LayerNorm.weight", "ln1_b": "attention.output.LayerNorm.bias",
    "i_w": "intermediate.dense.weight", "i_b": "intermediate.dense.bias",
    "d_w": "output.dense.weight", "d_b": "output.dense.bias",
    "ln2_g": "output.LayerNorm.weight", "ln2_b": "output.LayerNorm.bias",
}
_HF_TOP = {
    "word_emb": "embeddings.word_embeddings.weight", "pos_emb": "embeddings.position_embeddings.weight",
    "type_emb": "embeddings.token_type_embeddings.weight", "emb_ln_g": "embeddings.LayerNorm.weight", "emb_ln_b": "embeddings.LayerNorm.bias",
}


def hf_name(name):
    """Our tensor name -> the key BertModel.state_dict() uses."""
    if name in _HF_TOP:
        return _HF_TOP[name]
    layer, base = name.split(".")
    return f"encoder.layer.{int(layer[1:])}.{_HF_LAYER[base]}"


def load_safetensors(path, cfg=EncoderConfig()):
    """Real weights from a LOCAL model.safetensors (BERT key names, optional 'bert.' prefix)."""
    from safetensors.numpy import load_file

    if os.path.isdir(path):
        path = os.path.join(path, "model.safetensors")
    raw = load_file(path)
    out = {}
    for name, shape in tensor_specs(cfg):
        key = hf_name(name)
        for cand in (key, "bert." + key, "0.auto_model." + key):
            if cand in raw:
                w = raw[cand]
                break
        else:
            raise KeyError(f"{path}: tensor {key} not found")
        if tuple(w.shape) != tuple(shape):
            raise ValueError(f"{key}: shape {w.shape}, expected {shape}")
        out[name] = np.ascontiguousarray(w.astype(np.float32))
    return out
