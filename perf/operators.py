"""Cases for timing the encoder-layer operators of the engine: `linear` (matrix product with bias, activation and
residual), `attention` (documents packed into one batch, score cap, distance bias, prefix) and `layer_norm` (with the
residual's addition).  With `own` false `run` computes them in elementary torch operations in 32 bits, with `own` true
it calls the engine."""
import math
import random

import torch

own = False

_ENGINE = None
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _engine():
    global _ENGINE
    if _ENGINE is None:
        from hybrid_rag_system_amd.engine import Engine

        _ENGINE = Engine(0)
    return _ENGINE


# ---- cases -----------------------------------------------------------------------------------------
def _linear(rows, k, n, act, residual, dtype):
    return {"op": "linear", "rows": rows, "k": k, "n": n, "act": act, "residual": residual, "type": dtype}


def _attention(layout, batch, queries, keys, ragged, heads, kv_heads, dim, dtype, causal=False, prefix=0, cap=0.0, bias="none", reach=0, lens_seed=1):
    """layout "packed": `batch` documents back to back, lengths 1 .. `keys` (ragged) or all `keys`.  "padded": the same
    documents in rows of `keys` tokens.  "tail": the last `queries` tokens of every document over all its keys."""
    return {"op": "attention", "layout": layout, "batch": batch, "queries": queries, "keys": keys, "ragged": ragged, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "type": dtype, "causal": causal, "prefix": prefix, "cap": cap, "bias": bias, "reach": reach, "lens_seed": lens_seed}


def _norm(rows, n, residual, dtype):
    return {"op": "layer_norm", "rows": rows, "n": n, "residual": residual, "type": dtype}


def listed():
    cases = [
        # up projection of one short query in the 384-wide encoder: the latency of a search request
        dict(_linear(12, 384, 1536, "gelu", False, "bf16"), name="linear_query_up"),
        # up projection of an indexing batch (256 chunks x 256 tokens) in an encoder for the 1024-deep collections
        dict(_linear(65536, 1024, 4096, "gelu", False, "bf16"), name="linear_chunks_up"),
        # down projection with the residual of a smaller indexing batch
        dict(_linear(16384, 4096, 1024, "none", True, "fp16"), name="linear_chunks_down"),
        # a dense head behind the pooling: no dimension is a multiple of anything
        dict(_linear(4999, 773, 1537, "tanh", True, "bf16"), name="linear_odd_head"),
        # one short query in the 384-wide encoder
        dict(_attention("packed", 1, 12, 12, False, 12, 12, 32, "bf16"), name="attention_query"),
        # an indexing batch of ragged chunks, packed without padding, 1024-wide encoder
        dict(_attention("packed", 1024, 256, 256, True, 16, 16, 64, "bf16"), name="attention_packed_chunks"),
        # two whole documents in an encoder whose positions are a linear distance bias
        dict(_attention("packed", 2, 8192, 8192, False, 16, 16, 64, "bf16", bias="slope"), name="attention_long_documents"),
        # padded chunks in an encoder with a learned bias per distance
        dict(_attention("padded", 48, 512, 512, True, 12, 12, 64, "fp16", bias="table", reach=128), name="attention_table_padded"),
        # a causal embedder with capped scores, shared key heads and an instruction in front that all tokens see
        dict(_attention("padded", 2, 4096, 4096, False, 16, 8, 128, "bf16", causal=True, prefix=500, cap=50.0), name="attention_capped_prefix"),
        # one token at a time over long kept keys
        dict(_attention("tail", 8, 1, 32768, True, 32, 8, 128, "bf16", causal=True, cap=30.0, bias="slope"), name="attention_single_token"),
        # the norm between the blocks, for one query and for an indexing batch
        dict(_norm(12, 384, True, "bf16"), name="norm_query"),
        dict(_norm(65536, 1024, True, "bf16"), name="norm_chunks"),
    ]
    return cases


def _spread(rng, lo, hi):
    """A whole number in [lo, hi], even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng):
    """A layer's width: a multiple of 8 (or, one time in four, any number)."""
    n = _spread(rng, 64, 4096)
    return n if rng.random() < 0.25 else max(64, n // 8 * 8)


def draw(rng):
    kind = rng.choice(["linear", "linear", "attention", "attention", "attention", "layer_norm"])
    dtype = rng.choice(["bf16", "fp16"])
    if kind == "linear":
        k, n = _width(rng), _width(rng)
        rows = _spread(rng, 1, min(65536, max(1, 65536 * 1024 * 4096 // (k * n))))
        return _linear(rows, k, n, rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu", "tanh"]), rng.random() < 0.5, dtype)
    if kind == "layer_norm":
        n = _width(rng)
        return _norm(_spread(rng, 1, min(65536, 65536 * 1024 // n)), n, rng.random() < 0.5, dtype)
    dim = rng.choice([32, 64, 80, 128, 256])
    kv_heads = rng.choice([1, 2, 4, 8, 12])
    heads = kv_heads * rng.choice([1, 1, 2, 4])
    bias = rng.choice(["none", "slope", "table"])
    common = {"bias": bias, "reach": rng.randint(1, 200) if bias == "table" else 0, "cap": rng.choice([0.0, 0.0, 30.0, 50.0]), "lens_seed": rng.randint(1, 10**6)}
    form = rng.choice(["packed", "padded", "tail"])
    if form == "tail":
        keys = _spread(rng, 16, 32768)
        batch = _spread(rng, 1, max(1, min(64, 8 * 32768 * 8 * 128 // (keys * kv_heads * dim))))
        return _attention(form, batch, rng.choice([1, 1, 3, 16]), keys, True, heads, kv_heads, dim, dtype, causal=True, **common)
    causal = rng.random() < 0.5
    seq = _spread(rng, 2, min(8192, int((2 * 8192 * 8192 * 16 * 64 / max(heads * dim, 512)) ** 0.5)))
    batch = _spread(rng, 1, max(1, min(1024, 2 * 8192 * 8192 * 16 * 64 // (seq * seq * max(heads * dim, 512)), 2**27 // (seq * heads * dim))))
    prefix = rng.randint(1, seq) if causal and rng.random() < 0.5 else 0
    return _attention(form, batch, seq, seq, rng.random() < 0.7, heads, kv_heads, dim, dtype, causal=causal, prefix=prefix, **common)


def _lens(case):
    """Keys of every document (packed: its queries too), at least one of them the longest."""
    r = random.Random(case["lens_seed"])
    top = case["keys"]
    lens = [r.randint(1, top) if case["ragged"] else top for _ in range(case["batch"])]
    lens[0] = top
    return lens


def _visible(case):
    """Pairs of a query and a key that it sees, over all documents (of one head)."""
    triangle = lambda n: n * (n + 1) // 2
    total = 0
    for lk in _lens(case):
        lq = case["queries"] if case["layout"] == "tail" else lk
        if not case["causal"]:
            total += lq * lk
            continue
        p, first = min(case["prefix"], lk), lk - lq  # the query at position t sees max(t + 1, p) keys, or none
        total += max(0, p - first) * p + triangle(lk) - triangle(max(p, first))
    return total


def work(case):
    """The least one pass reads, writes and computes."""
    if case["op"] == "linear":
        m, k, n = case["rows"], case["k"], case["n"]
        return {"bytes": 2 * (m * k + n * k + m * n * (2 if case["residual"] else 1)) + 4 * n, "flops": 2 * m * k * n}
    if case["op"] == "layer_norm":
        return {"bytes": 2 * case["rows"] * case["n"] * (3 if case["residual"] else 2) + 8 * case["n"], "flops": 8 * case["rows"] * case["n"]}
    keys = sum(_lens(case))
    queries = case["batch"] * case["queries"] if case["layout"] == "tail" else keys
    row = 2 * case["dim"]
    table = 4 * case["heads"] * (2 * case["reach"] + 1 if case["bias"] == "table" else 1 if case["bias"] == "slope" else 0)
    return {"bytes": 2 * queries * case["heads"] * row + 2 * keys * case["kv_heads"] * row + table, "flops": 4 * case["dim"] * case["heads"] * _visible(case)}


# ---- inputs ----------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    t = TYPES[case["type"]]
    normal = lambda *shape: torch.randn(shape, generator=g, device="cuda")
    s = {"case": case, "eng": _engine() if own else None}
    if case["op"] == "linear":
        m, k, n = case["rows"], case["k"], case["n"]
        s["x"] = normal(m, k).to(t)  # normalised activations
        s["w"] = (normal(n, k) * k**-0.5).to(t)
        s["b"] = normal(n) * 0.1
        s["r"] = normal(m, n).to(t) if case["residual"] else None
        return s
    if case["op"] == "layer_norm":
        m, n = case["rows"], case["n"]
        s["x"] = (normal(m, n) * 2 + 0.3).to(t)
        s["r"] = normal(m, n).to(t) if case["residual"] else None
        s["g"] = 1 + 0.1 * normal(n)
        s["b"] = 0.1 * normal(n)
        return s
    lens, h, hk, d = _lens(case), case["heads"], case["kv_heads"], case["dim"]
    if case["layout"] == "packed":
        total = sum(lens)
        qs, ks = (total, h, d), (total, hk, d)
        offs = [0]
        for n in lens:
            offs.append(offs[-1] + n)
        s["offs"] = torch.tensor(offs, dtype=torch.int32, device="cuda")
    else:
        qs, ks = (case["batch"], case["queries"], h, d), (case["batch"], case["keys"], hk, d)
        s["k_lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    s["q"] = (normal(*qs) * (4 if case["cap"] else 1)).to(t)  # capped models are those whose scores grow large
    s["k"], s["v"] = normal(*ks).to(t), normal(*ks).to(t)
    s["slopes"] = torch.tensor([2.0 ** (-8.0 * (i + 1) / h) for i in range(h)], device="cuda") if case["bias"] == "slope" else None
    s["table"] = normal(h, 2 * case["reach"] + 1) if case["bias"] == "table" else None
    s["prefix"] = torch.tensor([min(case["prefix"], n) for n in lens], dtype=torch.int32, device="cuda") if case["prefix"] else None
    return s


# ---- one pass --------------------------------------------------------------------------------------
def run(state):
    case = state["case"]
    if own:
        eng = state["eng"]
        if case["op"] == "linear":
            return eng.linear(state["x"], state["w"], state["b"], activation=case["act"], residual=state["r"])
        if case["op"] == "layer_norm":
            return eng.layer_norm(state["x"], state["g"], state["b"], eps=1e-12, residual=state["r"])
        shared = {"causal": case["causal"], "prefix_lens": state["prefix"], "softcap": case["cap"], "slopes": state["slopes"], "bias_table": state["table"]}
        if case["layout"] == "packed":
            return eng.attention(state["q"], state["k"], state["v"], q_offs=state["offs"], max_q=case["queries"], **shared)
        q_lens = state["k_lens"] if case["layout"] == "padded" else None
        return eng.attention(state["q"], state["k"], state["v"], q_lens=q_lens, k_lens=state["k_lens"], **shared)
    if case["op"] == "linear":
        return _plain_linear(state)
    if case["op"] == "layer_norm":
        return _plain_norm(state)
    return _plain_attention(state)


def _activate(z, act):
    if act == "relu":
        return z.clamp(min=0)
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * 0.5**0.5))
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh((2 / math.pi) ** 0.5 * (z + 0.044715 * z * z * z)))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    if act == "tanh":
        return torch.tanh(z)
    return z


def _plain_linear(s):
    z = s["x"].float() @ s["w"].float().t() + s["b"]
    z = _activate(z, s["case"]["act"])
    if s["r"] is not None:
        z = z + s["r"].float()
    return z.to(s["x"].dtype)


def _plain_norm(s):
    z = s["x"].float()
    if s["r"] is not None:
        z = z + s["r"].float()
    c = z - z.mean(-1, keepdim=True)
    y = c * torch.rsqrt((c * c).mean(-1, keepdim=True) + 1e-12)
    return (y * s["g"] + s["b"]).to(s["x"].dtype)


def _plain_attention(s):
    case = s["case"]
    q, k, v = s["q"], s["k"], s["v"]
    dev, group = q.device, case["heads"] // case["kv_heads"]
    if case["layout"] == "packed":
        lens = s["offs"][1:] - s["offs"][:-1]
        at = torch.arange(case["keys"], device=dev)
        index = (s["offs"][:-1, None] + at).clamp(max=q.shape[0] - 1)
        inside = at < lens[:, None]
        q, k, v = q[index], k[index], v[index]
        lq, lk = lens, lens
    else:
        lk = s["k_lens"]
        lq = lk if case["layout"] == "padded" else torch.full_like(lk, case["queries"])
    i, j = torch.arange(q.shape[1], device=dev), torch.arange(k.shape[1], device=dev)
    pos = i + (lk - lq)[:, None]  # [B, Sq]
    seen = (j < lk[:, None])[:, None, :] & (i < lq[:, None])[:, :, None]
    if case["causal"]:
        order = j <= pos[:, :, None]
        if s["prefix"] is not None:
            order = order | (j < s["prefix"][:, None])[:, None, :]
        seen = seen & order
    out = torch.empty_like(q)
    step = max(1, 2**30 // max(1, q.shape[0] * q.shape[1] * k.shape[1])) // group * group or group
    for h0 in range(0, case["heads"], step):  # some heads at a time, so that the scores fit
        h1 = min(case["heads"], h0 + step)
        qf = q[:, :, h0:h1].float().transpose(1, 2).contiguous()
        kf = k[:, :, h0 // group : (h1 + group - 1) // group].float().permute(0, 2, 3, 1).repeat_interleave(group, 1).contiguous()
        vf = v[:, :, h0 // group : (h1 + group - 1) // group].float().transpose(1, 2).repeat_interleave(group, 1).contiguous()
        x = torch.matmul(qf, kf) * case["dim"] ** -0.5
        if case["cap"]:
            x = case["cap"] * torch.tanh(x / case["cap"])
        if s["slopes"] is not None:
            x = x - s["slopes"][h0:h1, None, None] * (j - pos[:, :, None]).abs().float()[:, None]
        if s["table"] is not None:
            r = case["reach"]
            d = (j - pos[:, :, None]).clamp(-r, r) + r
            x = x + s["table"][h0:h1][:, d].transpose(0, 1)
        x = torch.where(seen[:, None], x, float("-inf"))
        top = x.amax(-1, keepdim=True)
        top = torch.where(top == float("-inf"), 0.0, top)
        p = torch.exp(x - top)
        total = p.sum(-1, keepdim=True)
        p = p / torch.where(total == 0, 1.0, total)
        out[:, :, h0:h1] = torch.matmul(p, vf).transpose(1, 2).to(q.dtype)
    return out[inside] if case["layout"] == "packed" else out


# ---- the definition in 64 bits ---------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "linear":
        w = s["w"].double()
        parts = []
        for m0 in range(0, case["rows"], 8192):
            z = torch.nn.functional.linear(s["x"][m0 : m0 + 8192].double(), w, s["b"].double())
            a = case["act"]
            if a == "relu":
                z = torch.maximum(z, torch.zeros_like(z))
            elif a == "gelu":
                z = z * (0.5 * torch.special.erfc(-z / math.sqrt(2.0)))
            elif a == "gelu_tanh":
                u = math.sqrt(2 / math.pi) * (z + 0.044715 * z**3)
                z = z * torch.sigmoid(2 * u)
            elif a == "silu":
                z = z * torch.sigmoid(z)
            elif a == "tanh":
                z = z.tanh()
            parts.append(z if s["r"] is None else z + s["r"][m0 : m0 + 8192].double())
        return torch.cat(parts)
    if case["op"] == "layer_norm":
        z = s["x"].double() + (s["r"].double() if s["r"] is not None else 0)
        var, mean = torch.var_mean(z, dim=1, unbiased=False, keepdim=True)
        return (z - mean) / torch.sqrt(var + 1e-12) * s["g"].double() + s["b"].double()
    group = case["heads"] // case["kv_heads"]
    packed = case["layout"] == "packed"
    result = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    first = 0
    for b, lk in enumerate(_lens(case)):
        lq = case["queries"] if case["layout"] == "tail" else lk
        mine = slice(first, first + lk)
        q = s["q"][mine] if packed else s["q"][b, :lq]
        k = s["k"][mine] if packed else s["k"][b, :lk]
        v = s["v"][mine] if packed else s["v"][b, :lk]
        o = result[mine] if packed else result[b, :lq]
        first += lk
        distance = torch.arange(lk, device="cuda")[None, :] - (torch.arange(lq, device="cuda")[:, None] + (lk - lq))
        hidden = None
        if case["causal"]:
            hidden = distance > 0
            if case["prefix"]:
                hidden[:, : min(case["prefix"], lk)] = False
        per = max(1, 2**27 // (lq * lk))  # heads at a time
        for h0 in range(0, case["heads"], per):
            hs = list(range(h0, min(case["heads"], h0 + per)))
            ks = [h // group for h in hs]
            a = torch.bmm(q[:, hs].double().permute(1, 0, 2).contiguous(), k[:, ks].double().permute(1, 2, 0).contiguous()) / math.sqrt(case["dim"])
            if case["cap"]:
                a = torch.tanh(a / case["cap"]) * case["cap"]
            if case["bias"] == "slope":
                a -= distance.abs().double() * torch.tensor([2.0 ** (-8.0 * (h + 1) / case["heads"]) for h in hs], dtype=torch.float64, device="cuda").float().double()[:, None, None]
            elif case["bias"] == "table":
                near = distance.clamp(-case["reach"], case["reach"]) + case["reach"]
                a += s["table"][hs].double()[:, near.reshape(-1)].view(len(hs), lq, lk)
            if hidden is not None:
                a.masked_fill_(hidden, -math.inf)
            weight = torch.nan_to_num(torch.softmax(a, -1), nan=0.0)  # a row that sees nothing stays zero
            o[:, hs] = torch.bmm(weight, v[:, ks].double().permute(1, 0, 2).contiguous()).permute(1, 0, 2)
    return result
