"""The language-model operators of this package whose speed matters, as data.

They are the projection, the attention and the norm of one encoder layer in the
forms that a server of many fine-tuned variants and a cached, causal decoder
need, on the rows ([B*T, C]) and valid lengths that the rest of the package uses:

  linear     a shared projection with a low-rank adapter per request,
             y = act(x W^T + bias + s_e (x A_e^T) B_e^T)
  residual   the same into the fp32 stream, out = y + x W^T + s_e (x A_e^T) B_e^T
  attention  differential attention, the difference of two softmax maps with a
             learned weight, with an optional norm of each head's output
  norm       group norm with an activation, channels last, over valid frames

``listed()`` names the fixed cases, ``draw(rng)`` gives another one of the same
ranges, ``prepare`` / ``run`` make and run a case: its plain form, or where
``own`` is set this package's entry points.  ``work`` counts what a case cannot
do without and ``exact`` computes it in 64 bits.  Sizes are the encoder's
(hidden 1024, feed-forward 4096, 50 frames a second, chunks of up to 96 s).
"""

from __future__ import annotations

import math

import torch

own = False

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
EPS = 1e-5
LAMBDA_INIT = 0.5


# ---- cases ------------------------------------------------------------------------


def listed():
    return [
        # One frame of one stream through a square projection: latency.
        {"name": "adapter 1 frame", "op": "linear", "items": 1, "rows": 1, "n": 1024, "k": 1024, "rank": 16,
         "adapters": 8, "bare": 0, "type": "fp16", "act": "none"},
        # 48 streams of one frame each, most with an adapter of their own, into the feed-forward.
        {"name": "adapter 48 frames", "op": "linear", "items": 48, "rows": 1, "n": 4096, "k": 1024, "rank": 16,
         "adapters": 64, "bare": 5, "type": "bf16", "act": "silu"},
        # A small batch of 8 s utterances, query and key projections together.
        {"name": "adapter 4 x 400", "op": "linear", "items": 4, "rows": 400, "n": 2048, "k": 1024, "rank": 32,
         "adapters": 6, "bare": 1, "type": "fp16", "act": "none"},
        # The feed-forward output into the stream, items of no round length.
        {"name": "adapter residual 3 x 1463", "op": "residual", "items": 3, "rows": 1463, "n": 1024, "k": 4096,
         "rank": 16, "adapters": 4, "bare": 0, "type": "fp16", "act": "none"},
        # The feed-forward input of a full batch at a large rank.
        {"name": "adapter 8 x 600", "op": "linear", "items": 8, "rows": 600, "n": 4096, "k": 1024, "rank": 64,
         "adapters": 8, "bare": 0, "type": "bf16", "act": "silu"},
        # One new frame against 96 s of cache.
        {"name": "attention 1 of 4800", "op": "attention", "batch": 1, "heads": 8, "kv": 8, "dim": 64, "length": 1,
         "keys": 4800, "shortest": 4800, "causal": True, "norm": True, "type": "fp16"},
        # One new token of 32 streams of very different age, heads in groups of four.
        {"name": "attention 32 x 1 of 6000", "op": "attention", "batch": 32, "heads": 16, "kv": 4, "dim": 64,
         "length": 1, "keys": 6000, "shortest": 97, "causal": True, "norm": True, "type": "bf16"},
        # A whole 96 s chunk, both directions: the encoder's own attention shape.
        {"name": "attention 4800", "op": "attention", "batch": 1, "heads": 8, "kv": 8, "dim": 64, "length": 4800,
         "keys": 4800, "shortest": 4800, "causal": False, "norm": True, "type": "fp16"},
        # A ragged batch of prompts, wide heads in groups.
        {"name": "attention 3 x 1037 causal", "op": "attention", "batch": 3, "heads": 8, "kv": 2, "dim": 128,
         "length": 1037, "keys": 1037, "shortest": 211, "causal": True, "norm": False, "type": "bf16"},
        # A 3 s chunk: latency.
        {"name": "norm 150", "op": "norm", "items": 1, "rows": 150, "channels": 1024, "groups": 32, "shortest": 150,
         "type": "fp16", "act": "silu"},
        # A small ragged batch.
        {"name": "norm 3 x 1463", "op": "norm", "items": 3, "rows": 1463, "channels": 1024, "groups": 16,
         "shortest": 800, "type": "bf16", "act": "gelu"},
        # A full batch of whole chunks in fp32.
        {"name": "norm 8 x 4800", "op": "norm", "items": 8, "rows": 4800, "channels": 1024, "groups": 32,
         "shortest": 4800, "type": "fp32", "act": "silu"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case: 1 to 4800 rows in all in 1 to 64 items for the
    projections, 1 to 4800 queries against up to 8192 keys, up to 8 x 4800
    frames for the norm."""
    op = rng.choice(["linear", "linear", "residual", "attention", "attention", "attention", "norm", "norm"])
    if op in ("linear", "residual"):
        items = _log(rng, 1, 64)
        rows = _log(rng, 1, max(1, 4800 // items)) if rng.random() < 0.7 else 1
        n, k = rng.choice([(1024, 1024), (2048, 1024), (4096, 1024), (1024, 4096), (64 * rng.randint(1, 32),
                                                                                  64 * rng.randint(1, 32))])
        adapters = _log(rng, 1, 64)
        return {"op": op, "items": items, "rows": rows, "n": n, "k": k, "rank": 8 * rng.randint(1, 8),
                "adapters": adapters, "bare": rng.randint(0, items // 2), "type": rng.choice(["fp16", "bf16"]),
                "act": rng.choice(["none", "silu"]) if op == "linear" else "none"}
    if op == "attention":
        dim = rng.choice([64, 64, 128])
        kv = rng.choice([1, 2, 4, 8])
        heads = kv * rng.choice([1, 2, 4]) if kv < 8 else 8
        batch = _log(rng, 1, 32)
        causal = rng.random() < 0.6
        keys = _log(rng, 1, 8192)
        # new tokens against a cache, or as many queries as keys
        length = rng.choice([1, 1, rng.randint(1, 8), keys])
        if length == keys:
            # no more query-key products than the largest listed case has
            keys = length = min(keys, 4800)
            while heads * dim > 8 * 64:
                heads, kv = heads // 2, max(1, kv // 2)
            batch = max(1, min(batch, 4800 * 4800 * 64 * 8 // (keys * keys * dim * heads)))
        # no more cache than the largest listed one has
        keys = max(keys, length)
        batch = max(1, min(batch, 32 * 3000 * 4 * 64 // (keys * kv * dim)))
        return {"op": op, "batch": batch, "heads": heads, "kv": kv, "dim": dim, "length": length, "keys": keys,
                "shortest": keys if batch == 1 else rng.randint(0, keys), "causal": causal,
                "norm": rng.random() < 0.7, "type": rng.choice(["fp16", "bf16"])}
    channels, groups = rng.choice([(1024, 32), (1024, 16), (1024, 1), (512, 32), (160, 10), (320, 32),
                                   (8 * rng.randint(1, 128), 1), (8 * rng.randint(1, 128), 8)])
    items = _log(rng, 1, 8)
    rows = _log(rng, 1, 4800)
    return {"op": op, "items": items, "rows": rows, "channels": channels, "groups": groups,
            "shortest": rows if items == 1 else rng.randint(0, rows), "type": rng.choice(["fp16", "bf16", "fp32"]),
            "act": rng.choice(["none", "silu", "gelu", "relu"])}


def _lens(items, longest, shortest):
    """Valid lengths from the longest down to the shortest, evenly."""
    if items == 1:
        return [shortest]
    return [longest - (longest - shortest) * i // (items - 1) for i in range(items)]


def _ids(case):
    """The adapter of each item: the last ``bare`` items have none."""
    used = case["items"] - case["bare"]
    return [i % case["adapters"] for i in range(used)] + [-1] * case["bare"]


# ---- inputs -----------------------------------------------------------------------


def prepare(case, seed):
    """What a server has in hand: activations, packed weights, cache and lengths."""
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    kind = TYPES[case["type"]]

    def randn(*shape, std=1.0, dtype=kind):
        return (torch.randn(*shape, generator=gen, device=dev) * std).to(dtype)

    if case["op"] in ("linear", "residual"):
        m, n, k, r, e = case["items"] * case["rows"], case["n"], case["k"], case["rank"], case["adapters"]
        state = {"x": randn(m, k), "w": randn(n, k, std=k ** -0.5), "a": randn(e, r, k, std=k ** -0.5),
                 "b": randn(e, n, r, std=0.3 * r ** -0.5),
                 "scale": torch.rand(e, generator=gen, device=dev) + 0.5,
                 "ids": torch.tensor(_ids(case), dtype=torch.int32, device=dev)}
        if case["op"] == "linear":
            state["bias"] = randn(n, std=0.1)
        else:
            state["y"] = randn(m, n, dtype=torch.float32)
    elif case["op"] == "attention":
        b, h, g, d = case["batch"], case["heads"], case["kv"], case["dim"]
        l, s = case["length"], case["keys"]
        # Rows of the fused projections, as the encoder lays its q | k | v out:
        # a head's two maps side by side, its values twice as wide.
        state = {"q": randn(b, l, h, 2, d).permute(0, 2, 3, 1, 4), "k": randn(b, s, g, 2, d).permute(0, 2, 3, 1, 4),
                 "v": randn(b, s, g, 2 * d).permute(0, 2, 1, 3),
                 "lam": randn(4, d, std=0.1, dtype=torch.float32),
                 "lens": torch.tensor(_lens(b, s, case["shortest"]), dtype=torch.int32, device=dev),
                 "norm_w": None}
        if case["norm"]:
            state["norm_w"] = 1 + randn(2 * d, std=0.1, dtype=torch.float32)
    else:
        t, c = case["rows"], case["channels"]
        state = {"x": randn(case["items"] * t, c, std=1.5) + randn(1, c, std=0.5),
                 "w": 1 + randn(c, std=0.1, dtype=torch.float32), "b": randn(c, std=0.1, dtype=torch.float32),
                 "lens": torch.tensor(_lens(case["items"], t, case["shortest"]), dtype=torch.int32, device=dev)}
    state["case"] = dict(case)
    if own:
        from __graft_entry__ import load_package

        state["sidon"] = load_package()
    return state


# ---- one pass ---------------------------------------------------------------------


def run(state):
    case = state["case"]
    if own:
        return _own(state["sidon"], case, state)
    if case["op"] in ("linear", "residual"):
        return _plain_adapter(case, state)
    if case["op"] == "attention":
        return _plain_attention(case, state)
    return _plain_norm(case, state)


def _own(sidon, case, s):
    if case["op"] == "linear":
        return sidon.adapters.adapter_linear(s["x"], s["w"], s["bias"], s["a"], s["b"], s["scale"], s["ids"],
                                             act=None if case["act"] == "none" else case["act"])
    if case["op"] == "residual":
        return sidon.adapters.adapter_residual(s["y"], s["x"], s["w"], s["a"], s["b"], s["scale"], s["ids"],
                                               out=torch.empty_like(s["y"]))
    if case["op"] == "attention":
        return sidon.diff_attention.diff_attention(s["q"], s["k"], s["v"], s["lam"], LAMBDA_INIT, lens=s["lens"],
                                                   causal=case["causal"], norm_w=s["norm_w"], eps=EPS)
    return sidon.conformer.group_norm_act(s["x"], case["items"], case["groups"], s["w"], s["b"], EPS,
                                          lens=s["lens"], act=None if case["act"] == "none" else case["act"])


def _act(y, act):
    if act == "silu":
        return y * torch.sigmoid(y)
    if act == "gelu":
        return 0.5 * y * (1 + torch.erf(y * math.sqrt(0.5)))
    if act == "relu":
        return y.clamp_min(0)
    return y


def _plain_adapter(case, s):
    items, rows = case["items"], case["rows"]
    x = s["x"].float()
    y = x @ s["w"].float().t()
    ids = s["ids"].long()
    have = (ids >= 0).float().view(items, 1, 1)
    pick = ids.clamp_min(0)
    a = s["a"][pick].float().transpose(1, 2).contiguous()
    b = s["b"][pick].float().transpose(1, 2).contiguous()
    low = torch.matmul(x.view(items, rows, -1), a) * (s["scale"][pick].view(items, 1, 1) * have)
    y = y + torch.matmul(low, b).view(items * rows, -1)
    if case["op"] == "residual":
        return s["y"] + y
    return _act(y + s["bias"].float(), case["act"]).to(s["x"].dtype)


def _plain_attention(case, s):
    b, h, g, d = case["batch"], case["heads"], case["kv"], case["dim"]
    l, n = case["length"], case["keys"]
    lens = s["lens"].view(b, 1, 1)
    key = torch.arange(n, device=lens.device).view(1, 1, n)
    seen = key < lens
    if case["causal"]:
        seen = seen & (key <= lens - l + torch.arange(l, device=lens.device).view(1, l, 1))
    seen = seen.expand(b, l, n)
    lam = s["lam"]
    weight = torch.exp((lam[0] * lam[1]).sum()) - torch.exp((lam[2] * lam[3]).sum()) + LAMBDA_INIT
    used = (torch.arange(n, device=lens.device).view(1, 1, n, 1) < lens.view(b, 1, 1, 1))
    v = torch.where(used, s["v"].float(), 0.0)
    out = torch.empty(b, h, l, 2 * d, device=lens.device, dtype=s["q"].dtype)
    # a key head at a time, so that the maps of long sequences fit
    per = h // g
    for head in range(g):
        maps = []
        k = s["k"][:, head].float().transpose(2, 3).contiguous()
        for which in range(2):
            q = s["q"][:, head * per:(head + 1) * per, which].float().reshape(b, per * l, d)
            score = torch.matmul(q, k[:, which].contiguous()).view(b, per, l, n) * d ** -0.5
            score = score.masked_fill(~seen.unsqueeze(1), float("-inf"))
            top = score.amax(-1, keepdim=True)
            p = torch.exp(score - torch.where(top == float("-inf"), 0.0, top))
            total = p.sum(-1, keepdim=True)
            maps.append(p / torch.where(total == 0, 1.0, total))
        o = torch.matmul((maps[0] - weight * maps[1]).view(b, per * l, n), v[:, head].contiguous())
        o = o.view(b, per, l, 2 * d)
        if s["norm_w"] is not None:
            o = o * torch.rsqrt((o * o).mean(-1, keepdim=True) + EPS) * (s["norm_w"] * (1 - LAMBDA_INIT))
        out[:, head * per:(head + 1) * per] = o.to(out.dtype)
    return out


def _plain_norm(case, s):
    items, t, c, groups = case["items"], case["rows"], case["channels"], case["groups"]
    x = s["x"].float().view(items, t, groups, c // groups)
    valid = (torch.arange(t, device=x.device).view(1, t) < s["lens"].view(items, 1)).view(items, t, 1, 1)
    count = s["lens"].clamp_min(1).view(items, 1, 1, 1).float() * (c // groups)
    mean = torch.where(valid, x, 0.0).sum((1, 3), keepdim=True) / count
    centred = torch.where(valid, x - mean, 0.0)
    var = (centred * centred).sum((1, 3), keepdim=True) / count
    y = (centred * torch.rsqrt(var + EPS)).view(items, t, c) * s["w"] + s["b"]
    y = torch.where(valid.view(items, t, 1), _act(y, case["act"]), 0.0)
    return y.view(items * t, c).to(s["x"].dtype)


# ---- what a case cannot do without -------------------------------------------------


def _pairs(case):
    """Query-key pairs that the masks leave, over the batch, per head."""
    total = 0
    for n in _lens(case["batch"], case["keys"], case["shortest"]):
        if not case["causal"]:
            total += n * case["length"]
            continue
        # query i sees n - length + i + 1 keys, where positive
        last, count = n, min(case["length"], n)
        total += count * (last + last - count + 1) // 2
    return total


def work(case):
    size = 4 if case["type"] == "fp32" else 2
    if case["op"] in ("linear", "residual"):
        m, n, k, r = case["items"] * case["rows"], case["n"], case["k"], case["rank"]
        used = len({i for i in _ids(case) if i >= 0})
        adapted = case["rows"] * (case["items"] - case["bare"])
        moved = 2 * (m * k + n * k + used * r * (n + k)) + 4 * used + 4 * case["items"]
        moved += 8 * m * n if case["op"] == "residual" else 2 * n + 2 * m * n
        return {"bytes": moved, "flops": 2 * m * n * k + 2 * adapted * r * (n + k)}
    if case["op"] == "attention":
        b, h, g, d = case["batch"], case["heads"], case["kv"], case["dim"]
        keys = sum(_lens(b, case["keys"], case["shortest"]))
        return {"bytes": 2 * (keys * g * 4 * d + b * h * case["length"] * 4 * d) + 16 * d,
                "flops": 12 * d * h * _pairs(case)}
    c = case["channels"]
    valid = c * sum(_lens(case["items"], case["rows"], case["shortest"]))
    return {"bytes": size * (valid + case["items"] * case["rows"] * c) + 8 * c, "flops": 10 * valid}


# ---- the definitions in 64 bits ----------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("linear", "residual"):
        return _exact_adapter(case, s)
    if case["op"] == "attention":
        return _exact_attention(case, s)
    return _exact_norm(case, s)


def _exact_adapter(case, s):
    x, w = s["x"].double(), s["w"].double()
    out = x @ w.t()
    for item, e in enumerate(_ids(case)):
        if e >= 0:
            lo, hi = item * case["rows"], (item + 1) * case["rows"]
            low = x[lo:hi] @ s["a"][e].double().t()
            out[lo:hi] += s["scale"][e].double() * (low @ s["b"][e].double().t())
    if case["op"] == "residual":
        return out + s["y"].double()
    out += s["bias"].double()
    return out / (1 + torch.exp(-out)) if case["act"] == "silu" else out


def _exact_attention(case, s):
    d, l = case["dim"], case["length"]
    lam = s["lam"].double()
    weight = math.exp(float(lam[0] @ lam[1])) - math.exp(float(lam[2] @ lam[3])) + LAMBDA_INIT
    out = torch.zeros(case["batch"], case["heads"], l, 2 * d, dtype=torch.float64, device=lam.device)
    for b, n in enumerate(_lens(case["batch"], case["keys"], case["shortest"])):
        limit = torch.full((l,), n, device=lam.device)
        if case["causal"]:
            limit = torch.arange(l, device=lam.device) + (n - l + 1)
        hidden = torch.arange(n, device=lam.device) >= limit.view(l, 1)
        empty = (limit <= 0).view(l, 1)
        for h in range(case["heads"]):
            g = h // (case["heads"] // case["kv"])
            v = s["v"][b, g, :n].double()
            o = torch.zeros(l, 2 * d, dtype=torch.float64, device=lam.device)
            for which, factor in ((0, 1.0), (1, -weight)):
                logits = s["q"][b, h, which].double() @ s["k"][b, g, which, :n].double().t() / math.sqrt(d)
                p = torch.softmax(logits.masked_fill(hidden, float("-inf")), -1)
                o += factor * (torch.where(empty, 0.0, p) @ v)
            if s["norm_w"] is not None:
                rms = torch.sqrt(o.square().mean(-1, keepdim=True) + EPS)
                o = o / rms * s["norm_w"].double() * (1 - LAMBDA_INIT)
            out[b, h] = o
    return out


def _exact_norm(case, s):
    t, c, groups = case["rows"], case["channels"], case["groups"]
    out = torch.zeros(case["items"] * t, c, dtype=torch.float64, device=s["x"].device)
    for i, n in enumerate(_lens(case["items"], t, case["shortest"])):
        if n == 0:
            continue
        x = s["x"][i * t:i * t + n].double().view(n, groups, c // groups)
        var, mean = torch.var_mean(x, dim=(0, 2), correction=0, keepdim=True)
        y = ((x - mean) / torch.sqrt(var + EPS)).reshape(n, c) * s["w"].double() + s["b"].double()
        if case["act"] == "silu":
            y = y / (1 + torch.exp(-y))
        elif case["act"] == "gelu":
            y = y * 0.5 * torch.erfc(-y / math.sqrt(2))
        elif case["act"] == "relu":
            y = torch.relu(y)
        out[i * t:i * t + n] = y
    return out
