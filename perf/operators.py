"""Cases of the operators that an encoder-decoder Transformer's training and
decoding add to the GPT step: the scaled embedding lookup and its gradient,
attention of queries over the states of another sequence (forward, gradient,
one query per sequence), and the global gradient norm with clipping over many
tensors. Each case runs in a plain form or through magma_b200.ops.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
PAD = 0  # the padding token of the embedding gradient


# ---------------------------------------------------------------------- cases
def listed():
    return [
        # one new token of each of 16 sequences that are being decoded
        {"name": "embed_step", "op": "embed", "batch": 16, "seq": 1, "dim": 512, "vocab": 32000,
         "dtype": "bf16", "pos": True},
        # a batch of source sentences with learned positions
        {"name": "embed_batch", "op": "embed", "batch": 32, "seq": 1024, "dim": 1024,
         "vocab": 50257, "dtype": "f32", "pos": True},
        # the character model's batch: 16384 rows share 65 tokens
        {"name": "embed_grad_chars", "op": "embed_grad", "batch": 64, "seq": 256, "dim": 384,
         "vocab": 65, "dtype": "f32", "pos": True},
        # a batch of padded source sentences with word frequencies as in text
        {"name": "embed_grad_text", "op": "embed_grad", "batch": 32, "seq": 1024, "dim": 1024,
         "vocab": 50257, "dtype": "bf16", "pos": False},
        # a decoder of ordinary size over short, ragged sources in F32
        {"name": "cross_f32", "op": "cross", "batch": 8, "heads": 12, "kv_heads": 12, "q_len": 200,
         "kv_len": 333, "dim": 64, "dtype": "f32", "ragged": True},
        # long ragged sources, wide heads that share keys and values
        {"name": "cross_long", "op": "cross", "batch": 4, "heads": 32, "kv_heads": 8,
         "q_len": 2048, "kv_len": 4096, "dim": 128, "dtype": "bf16", "ragged": True},
        # gradients of a decoder training batch of ordinary size
        {"name": "cross_grad_batch", "op": "cross_grad", "batch": 8, "heads": 16, "kv_heads": 16,
         "q_len": 512, "kv_len": 1024, "dim": 64, "dtype": "bf16", "ragged": True},
        # gradients over long sources with shared keys and values
        {"name": "cross_grad_long", "op": "cross_grad", "batch": 2, "heads": 32, "kv_heads": 8,
         "q_len": 2048, "kv_len": 4096, "dim": 128, "dtype": "bf16", "ragged": False},
        # one decoding step of a single request
        {"name": "step_one", "op": "cross_step", "batch": 1, "heads": 16, "kv_heads": 16,
         "q_len": 1, "kv_len": 777, "dim": 64, "dtype": "bf16", "ragged": False},
        # one decoding step of a full batch over long sources
        {"name": "step_many", "op": "cross_step", "batch": 64, "heads": 32, "kv_heads": 8,
         "q_len": 1, "kv_len": 4096, "dim": 128, "dtype": "bf16", "ragged": True},
        # the gradients of the 784-128-10 classifier: two weights, two biases
        {"name": "clip_classifier", "op": "clip", "layers": 0, "width": 128, "vocab": 10,
         "dtype": "f32", "out": "f32", "odd": False},
        # the gradients of an encoder-decoder model, one tensor per parameter
        {"name": "clip_model", "op": "clip", "layers": 16, "width": 1024, "vocab": 32000,
         "dtype": "f32", "out": "f32", "odd": False},
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["embed", "embed_grad", "cross", "cross_grad", "cross_step", "clip"])
    case = {"op": op}
    if op in ("embed", "embed_grad"):
        seq = _spread(rng, 1, 2048)
        case |= {"batch": _spread(rng, 1, max(1, 32768 // seq)), "seq": seq,
                 "dim": rng.choice([384, 512, 777, 1024]), "vocab": _spread(rng, 65, 50257),
                 "dtype": rng.choice(["f32", "bf16"]), "pos": rng.random() < 0.5}
    elif op == "clip":
        case |= {"layers": _spread(rng, 1, 15), "width": 4 * _spread(rng, 16, 255),
                 "vocab": _spread(rng, 65, 32000), "dtype": rng.choice(["f32", "bf16"]),
                 "out": rng.choice(["f32", "bf16"]), "odd": rng.random() < 0.5}
    else:
        kv_heads = rng.choice([1, 2, 4, 6, 8])
        dtype = rng.choice(["bf16", "bf16", "f32"])
        heads = kv_heads * rng.choice([1, 1, 2, 3, 4])
        dim = rng.choice([32, 64, 64, 80, 96, 128, 128])
        kv_len = _spread(rng, 1, 4000)
        q_len = 1 if op == "cross_step" else _spread(rng, 2, 1024)
        batch = _spread(rng, 1, 48 if op == "cross_step" else 8)
        if dtype == "f32":
            batch = min(batch, 2 if op == "cross_grad" else 4)
        case |= {"batch": batch, "heads": heads, "kv_heads": kv_heads, "q_len": q_len,
                 "kv_len": kv_len, "dim": dim, "dtype": dtype, "ragged": rng.random() < 0.7,
                 "empty": rng.random() < 0.15}
    return case


def _lengths(case):
    """Source lengths of a batch: a quarter of kv_len up to all of it, or one of them nothing."""
    b, n = case["batch"], case["kv_len"]
    if not case["ragged"]:
        return [n] * b
    lens = [round(n * (0.25 + 0.75 * (i + 1) / b)) for i in range(b)]
    return [0] + lens[1:] if case.get("empty") and b > 1 else lens


def _sizes(case):
    """Parameter sizes of a model: per layer four projections and a two-layer
    network with their biases and a norm's weight and bias, then the embedding.
    Without layers: a classifier of 784 inputs."""
    w = case["width"]
    if case["layers"] == 0:
        return [784 * w, w, w * case["vocab"], case["vocab"]]
    layer = [w * w, w] * 4 + [4 * w * w, 4 * w, 4 * w * w, w, w, w]
    return layer * case["layers"] + [case["vocab"] * w] + ([1, 17, w + 3] if case["odd"] else [])


# --------------------------------------------------------------------- inputs
def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    op, dt = case["op"], DTYPES[case["dtype"]]

    def normal(*shape, dtype=dt, std=1.0):
        return torch.randn(*shape, generator=gen, device=dev).mul_(std).to(dtype)

    s = {"case": case}
    if op in ("embed", "embed_grad"):
        b, n, d, v = case["batch"], case["seq"], case["dim"], case["vocab"]
        # word frequencies fall as the inverse of the word's rank
        u = torch.rand(b, n, generator=gen, device=dev, dtype=torch.float64)
        tokens = (torch.exp(u * math.log(v)).long() - 1).clamp_(0, v - 1)
        if op == "embed_grad" and n > 1:
            # every sequence is padded behind its own length
            ends = torch.randint((n + 1) // 2, n + 1, (b, 1), generator=gen, device=dev)
            tokens[torch.arange(n, device=dev)[None, :] >= ends] = PAD
        s |= {"tokens": tokens.int(), "scale": math.sqrt(d)}
        if op == "embed":
            s["table"] = normal(v, d, std=d ** -0.5)
            s["pos"] = normal(n, d, std=0.02) if case["pos"] else None
        else:
            s["dout"] = normal(b * n, d, std=1e-2)
    elif op == "clip":
        sizes = _sizes(case)
        flat = normal(sum(sizes), std=1e-3)
        out = torch.empty(sum(sizes), dtype=DTYPES[case["out"]], device=dev)
        s |= {"grads": list(flat.split(sizes)), "flat": out, "out": list(out.split(sizes)),
              "max_norm": 1.0, "grad_scale": 0.125}
    else:
        b, h, g = case["batch"], case["heads"], case["kv_heads"]
        m, n, d = case["q_len"], case["kv_len"], case["dim"]
        # heads are views of the projections' outputs
        s["q"] = normal(b, m, h, d).transpose(1, 2)
        kv = normal(b, n, 2, g, d)
        s["k"], s["v"] = kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2)
        lens = torch.tensor(_lengths(case), device=dev)
        order = torch.randperm(b, generator=gen, device=dev)
        s["lens"] = lens[order].int() if case["ragged"] else None
        s["scale"] = d ** -0.5
        if op == "cross_grad":
            # the forward pass is behind the call: its outputs are at hand
            s["do"] = normal(b, m, h, d).transpose(1, 2)
            o, s["lse"] = _cross(s)
            s["o"] = o.to(dt)
    return s


# ---------------------------------------------------------------- plain forms
def _mask(s):
    """[B, 1, 1, 1, Skv]: the keys that a sequence has."""
    n = s["k"].shape[2]
    at = torch.arange(n, device=s["k"].device)
    lens = s["lens"] if s["lens"] is not None else torch.full(
        (s["k"].shape[0],), n, device=at.device)
    return (at[None, :] < lens[:, None])[:, None, None, None, :]


def _grouped(x, kv_heads):
    """[B, H, S, D] -> [B, Hkv, H / Hkv, S, D] in F32."""
    b, h, n, d = x.shape
    return x.float().reshape(b, kv_heads, h // kv_heads, n, d)


def _probs(s):
    """Softmax over the keys that are there (zeros where none is), and its log-sum-exp."""
    g = s["k"].shape[1]
    scores = _grouped(s["q"], g) @ _grouped(s["k"], g).transpose(-1, -2) * s["scale"]
    scores = scores.masked_fill(~_mask(s), -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    lse = (top + torch.log(total)).squeeze(-1)
    return p / torch.where(total == 0, torch.ones_like(total), total), lse


def _values(s):
    g = s["v"].shape[1]
    return torch.where(_mask(s).transpose(-1, -2), _grouped(s["v"], g), 0.0)


def _cross(s):
    p, lse = _probs(s)
    return (p @ _values(s)).reshape(s["q"].shape), lse.reshape(s["q"].shape[:3])


def _cross_grad(s):
    g = s["k"].shape[1]
    p, _ = _probs(s)
    do, q = _grouped(s["do"], g), _grouped(s["q"], g)
    k = torch.where(_mask(s).transpose(-1, -2), _grouped(s["k"], g), 0.0)
    dv = (p.transpose(-1, -2) @ do).sum(2)
    dp = do @ _values(s).transpose(-1, -2)
    ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * s["scale"]
    dq = (ds @ k).reshape(s["q"].shape)
    dk = (ds.transpose(-1, -2) @ q).sum(2)
    return dq, dk, dv


def _embed(s):
    rows = s["table"][s["tokens"].reshape(-1).long()].float() * s["scale"]
    if s["pos"] is None:
        return rows
    b, n = s["tokens"].shape
    return rows + s["pos"].float().repeat(b, 1)


def _embed_grad(s):
    case, t = s["case"], s["tokens"].reshape(-1).long()
    b, n = s["tokens"].shape
    dout = s["dout"].double()
    kept = torch.where((t != PAD)[:, None], dout, 0.0)
    dtable = torch.zeros(case["vocab"], case["dim"], dtype=torch.float64, device=t.device)
    dtable.index_add_(0, t, kept)
    dpos = dout.reshape(b, n, -1).sum(0).float() if case["pos"] else None
    return (dtable * s["scale"]).float(), dpos


def _clip(s):
    scaled = [g.float() * s["grad_scale"] for g in s["grads"]]
    norm = torch.stack([g.double().square().sum() for g in scaled]).sum().sqrt().float()
    c = torch.clamp(s["max_norm"] / (norm + 1e-6), max=1.0)
    return norm.reshape(1), torch.cat(scaled) * c


def run(state):
    s, case = state, state["case"]
    op, dt = case["op"], DTYPES[case["dtype"]]
    if own:
        from magma_b200 import ops
        if op == "embed":
            return ops.embedding_scaled_fwd(s["tokens"], s["table"], s["pos"], scale=s["scale"])
        if op == "embed_grad":
            return ops.embedding_scaled_bwd(s["tokens"], s["dout"], case["vocab"],
                                            scale=s["scale"], padding_idx=PAD, pos=case["pos"])
        if op == "clip":
            return ops.clip_grad_norm(s["grads"], s["max_norm"], grad_scale=s["grad_scale"],
                                      out=s["out"]), s["flat"]
        if op == "cross_grad":
            return ops.cross_attention_bwd(s["q"], s["k"], s["v"], s["o"], s["do"], s["lse"],
                                           s["scale"], s["lens"])
        return ops.cross_attention_fwd(s["q"], s["k"], s["v"], s["scale"], s["lens"])
    if op == "embed":
        return _embed(s).to(dt)
    if op == "embed_grad":
        return _embed_grad(s)
    if op == "clip":
        norm, flat = _clip(s)
        return norm, flat.to(DTYPES[case["out"]])
    if op == "cross_grad":
        return tuple(t.to(dt) for t in _cross_grad(s))
    o, lse = _cross(s)
    return o.to(dt), lse


def work(case):
    op = case["op"]
    size = {"f32": 4, "bf16": 2}
    e = size[case["dtype"]]
    if op in ("embed", "embed_grad"):
        rows, d, v = case["batch"] * case["seq"], case["dim"], case["vocab"]
        pos = case["seq"] * d if case["pos"] else 0
        if op == "embed":
            return {"bytes": 4 * rows + e * (min(rows, v) * d + pos + rows * d),
                    "flops": 2 * rows * d}
        return {"bytes": 4 * rows + e * rows * d + 4 * (v * d + pos), "flops": 2 * rows * d}
    if op == "clip":
        n = sum(_sizes(case))
        return {"bytes": n * (e + size[case["out"]]), "flops": 4 * n}
    b, h, g = case["batch"], case["heads"], case["kv_heads"]
    m, d, keys = case["q_len"], case["dim"], sum(_lengths(case))
    rows, pairs = b * h * m, h * m * keys
    if op == "cross_grad":
        return {"bytes": e * d * (4 * rows + 2 * g * keys + 2 * g * b * case["kv_len"]) + 4 * rows,
                "flops": 10 * pairs * d}
    return {"bytes": e * d * (2 * rows + 2 * g * keys) + 4 * rows, "flops": 4 * pairs * d}


# --------------------------------------------------------------------- exact
def _exact_heads(s, b, j):
    """Probabilities, log-sum-exp and operands of one sequence's key head, in 64 bits."""
    group = s["q"].shape[1] // s["k"].shape[1]
    n = s["k"].shape[2] if s["lens"] is None else int(s["lens"][b])
    q = s["q"][b, j * group:(j + 1) * group].double()
    k, v = s["k"][b, j, :n].double(), s["v"][b, j, :n].double()
    scores = torch.einsum("hmd,nd->hmn", q, k) * s["scale"]
    return torch.softmax(scores, -1), torch.logsumexp(scores, -1), q, k, v


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "embed":
        b, n = s["tokens"].shape
        out = torch.nn.functional.embedding(s["tokens"].long(), s["table"].double()) * s["scale"]
        if s["pos"] is not None:
            out = out + s["pos"].double()[None]
        return out.reshape(b * n, -1)
    if op == "embed_grad":
        b, n = s["tokens"].shape
        tokens, order = s["tokens"].reshape(-1).long().sort(stable=True)
        counts = torch.bincount(tokens, minlength=case["vocab"])
        total = torch.segment_reduce(s["dout"].double()[order], "sum", lengths=counts, axis=0,
                                     initial=0.0)
        total[PAD] = 0.0
        dpos = None
        if case["pos"]:
            dpos = torch.einsum("bnd->nd", s["dout"].double().reshape(b, n, -1))
        return total * s["scale"], dpos
    if op == "clip":
        flat = torch.cat(s["grads"]).double() * s["grad_scale"]
        norm = torch.linalg.vector_norm(flat)
        c = min(1.0, s["max_norm"] / (float(norm) + 1e-6))
        return norm.reshape(1), flat * c
    b, h, m, d = s["q"].shape
    g, n = s["k"].shape[1], s["k"].shape[2]
    full = dict(dtype=torch.float64, device=s["q"].device)
    group = h // g
    if op == "cross_grad":
        dq, dk, dv = (torch.zeros(*x, **full) for x in ((b, h, m, d), (b, g, n, d), (b, g, n, d)))
    else:
        o, lse = torch.zeros(b, h, m, d, **full), torch.zeros(b, h, m, **full)
    for i in range(b):
        for j in range(g):
            at = slice(j * group, (j + 1) * group)
            p, l, q, k, v = _exact_heads(s, i, j)
            if op != "cross_grad":
                o[i, at], lse[i, at] = torch.einsum("hmn,nd->hmd", p, v), l
                continue
            do = s["do"][i, at].double()
            dp = torch.einsum("hmd,nd->hmn", do, v)
            ds = p * (dp - torch.einsum("hmn,hmn->hm", p, dp)[..., None]) * s["scale"]
            dq[i, at] = torch.einsum("hmn,nd->hmd", ds, k)
            dk[i, j, :k.shape[0]] = torch.einsum("hmn,hmd->nd", ds, q)
            dv[i, j, :k.shape[0]] = torch.einsum("hmn,hmd->nd", p, do)
    return (dq, dk, dv) if op == "cross_grad" else (o, lse)
