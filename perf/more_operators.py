"""The operators of a text decoder over the encoder's frames, as data.

A decoder that reads the encoder's hidden states (frames at 50 a second, chunks
of up to 96 s) needs them in each of its layers, in training and a token at a time:

  norms    the norm of queries and keys for each head with the position rotation
  cross    attention of the decoder's tokens over the encoder's frames
  int4     the projections of single tokens with 4-bit weights and group scales

The first two have a backward direction ("train": the forward call and the
gradients from it), the last one serves.  ``listed()`` names the fixed cases,
``draw(rng)`` gives another one of the same ranges, ``prepare`` / ``run`` make and
run a case: its plain form, or where ``own`` is set this package's entry points.
``work`` counts what a case cannot do without and ``exact`` computes it in 64
bits.
"""

from __future__ import annotations

import math

import torch

own = False

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
EPS = 1e-6
PLACES = 8192   # rows of the rotation's table


# ---- cases ------------------------------------------------------------------------


def listed():
    return [
        # The new token of one stream late in a chunk: latency.
        {"name": "norms 1 token", "op": "norms", "batch": 1, "length": 1, "heads": 16, "kv": 16, "dim": 64, "rot": 64,
         "pairs": False, "shortest": 1, "type": "fp16", "train": False},
        # A ragged batch of chunks, wide heads in groups, half of each head rotated.
        {"name": "norms 3 x 1463", "op": "norms", "batch": 3, "length": 1463, "heads": 16, "kv": 4, "dim": 128,
         "rot": 64, "pairs": True, "shortest": 800, "type": "bf16", "train": False},
        # A training batch of whole chunks, with its gradients.
        {"name": "norms 8 x 4800 train", "op": "norms", "batch": 8, "length": 4800, "heads": 16, "kv": 16, "dim": 64,
         "rot": 64, "pairs": False, "shortest": 3900, "type": "bf16", "train": True},
        # One new token over 30 s of frames: latency.
        {"name": "cross 1 of 1500", "op": "cross", "batch": 1, "length": 1, "keys": 1500, "heads": 16, "kv": 16,
         "dim": 64, "shortest": 1500, "type": "fp16", "train": False},
        # One new token of 32 streams, each over its own chunk, heads in groups of four.
        {"name": "cross 32 x 1 of 4800", "op": "cross", "batch": 32, "length": 1, "keys": 4800, "heads": 16, "kv": 4,
         "dim": 64, "shortest": 150, "type": "bf16", "train": False},
        # The prompts of a small batch over 30 s chunks.
        {"name": "cross 4 x 224 of 1500", "op": "cross", "batch": 4, "length": 224, "keys": 1500, "heads": 16,
         "kv": 16, "dim": 64, "shortest": 731, "type": "fp16", "train": False},
        # Long texts over 96 s chunks, wide heads in groups.
        {"name": "cross 2 x 1037 of 4800", "op": "cross", "batch": 2, "length": 1037, "keys": 4800, "heads": 8,
         "kv": 2, "dim": 128, "shortest": 4091, "type": "bf16", "train": False},
        # A small training batch of no round sizes.
        {"name": "cross 2 x 300 of 1463 train", "op": "cross", "batch": 2, "length": 300, "keys": 1463, "heads": 16,
         "kv": 16, "dim": 64, "shortest": 1100, "type": "bf16", "train": True},
        # A training batch of whole chunks, heads in groups.
        {"name": "cross 4 x 1200 of 4800 train", "op": "cross", "batch": 4, "length": 1200, "keys": 4800,
         "heads": 16, "kv": 4, "dim": 64, "shortest": 3000, "type": "fp16", "train": True},
        # One token into the feed-forward: latency.
        {"name": "int4 1 x 4096 x 1024", "op": "int4", "rows": 1, "n": 4096, "k": 1024, "group": 64, "zeros": False,
         "type": "fp16", "act": "silu"},
        # The tokens of 7 streams out of the feed-forward.
        {"name": "int4 7 x 1024 x 4096", "op": "int4", "rows": 7, "n": 1024, "k": 4096, "group": 128, "zeros": True,
         "type": "bf16", "act": "none"},
        # The tokens of 32 streams into a vocabulary's logits.
        {"name": "int4 32 x 32768 x 4096", "op": "int4", "rows": 32, "n": 32768, "k": 4096, "group": 128,
         "zeros": True, "type": "bf16", "act": "none"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case: 1 to 8 x 4800 tokens for the norms, 1 to 1200 tokens of 1 to
    32 items over 1 to 6000 frames, 1 to 64 rows through up to 32768 x 4096 weights."""
    op = rng.choice(["norms", "norms", "cross", "cross", "cross", "cross", "int4", "int4"])
    if op == "norms":
        dim = rng.choice([64, 64, 128, 16 * rng.randint(2, 16)])
        kv = rng.choice([1, 2, 4, 8, 16])
        heads = kv * rng.choice([1, 2, 3, 4])
        batch, length = _log(rng, 1, 32), rng.choice([1, _log(rng, 1, 4800), _log(rng, 1, 4800)])
        kind = rng.choice(["fp16", "bf16", "bf16", "fp32"])
        # no more bytes than the largest listed case has
        size = 4 if kind == "fp32" else 2
        length = max(1, min(length, 8 * 4800 * 32 * 64 * 2 // (batch * (heads + kv) * dim * size)))
        return {"op": op, "batch": batch, "length": length, "heads": heads, "kv": kv, "dim": dim,
                "rot": rng.choice([dim, dim, 16 * rng.randint(0, dim // 16)]), "pairs": rng.random() < 0.4,
                "shortest": length if batch == 1 else rng.randint(0, length), "type": kind,
                "train": rng.random() < 0.4}
    if op == "cross":
        dim = rng.choice([64, 64, 128])
        kv = rng.choice([1, 2, 4, 8, 16])
        heads = kv * (rng.choice([1, 2, 4]) if kv < 16 else 1)
        train = rng.random() < 0.4
        batch, keys = _log(rng, 1, 32), _log(rng, 1, 6000)
        length = _log(rng, 1, 1200) if train or rng.random() < 0.5 else rng.choice([1, 1, rng.randint(2, 8)])
        # no more query-key products and no more frames than the largest listed cases have
        most = 4 * 1200 * 4800 * 16 * 64 * 7 // (7 if train else 2)
        length = max(1, min(length, most // (batch * keys * heads * dim)))
        batch = max(1, min(batch, 32 * 4800 * 4 * 64 // (keys * kv * dim)))
        return {"op": op, "batch": batch, "length": length, "keys": keys, "heads": heads, "kv": kv, "dim": dim,
                "shortest": keys if batch == 1 else rng.randint(0, keys), "type": rng.choice(["fp16", "bf16"]),
                "train": train}
    n, k = rng.choice([(4096, 1024), (1024, 4096), (4096, 4096), (rng.randint(1, 4096), 128 * rng.randint(1, 32)),
                       (_log(rng, 1000, 32768), 32 * rng.randint(1, 128))])
    return {"op": op, "rows": rng.choice([1, _log(rng, 1, 64)]), "n": n, "k": k,
            "group": rng.choice([g for g in (32, 64, 128) if k % g == 0]), "zeros": rng.random() < 0.6,
            "type": rng.choice(["fp16", "bf16"]), "act": rng.choice(["none", "silu"])}


def _lens(items, longest, shortest):
    """Valid lengths from the longest down to the shortest, evenly."""
    if items == 1:
        return [shortest]
    return [longest - (longest - shortest) * i // (items - 1) for i in range(items)]


def _query_lens(case):
    """Valid tokens of each item: all of the longest one's, fewer of the others in training and prompts."""
    length = case["length"]
    return [length - (length - 1) * i // (2 * case["batch"]) for i in range(case["batch"])]


# ---- inputs -----------------------------------------------------------------------


def prepare(case, seed):
    """What a decoder has in hand: its projections' rows, weights, positions and lengths."""
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    kind = TYPES[case["type"]]

    def randn(*shape, std=1.0, dtype=kind):
        return (torch.randn(*shape, generator=gen, device=dev) * std).to(dtype)

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device=dev)

    if case["op"] == "norms":
        b, l, h, g, d, rot = (case[n] for n in ("batch", "length", "heads", "kv", "dim", "rot"))
        # rows of a fused projection q | k | v
        rows = randn(b, l, h + 2 * g, d, std=1.5).permute(0, 2, 1, 3)
        state = {"q": rows[:, :h], "k": rows[:, h:h + g], "q_w": 1 + randn(d, std=0.1, dtype=torch.float32),
                 "k_w": 1 + randn(d, std=0.1, dtype=torch.float32), "cos": None, "sin": None}
        if rot:
            angle = (torch.arange(PLACES, dtype=torch.float64).view(-1, 1)
                     * 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot))
            state["cos"], state["sin"] = angle.cos().float().to(dev), angle.sin().float().to(dev)
        # each item begins at a place of its own; padded rows have none
        first = torch.randint(0, PLACES - l + 1, (b, 1), generator=gen, device=dev)
        at = torch.arange(l, device=dev).view(1, l)
        state["pos"] = torch.where(at < ints(_lens(b, l, case["shortest"])).view(b, 1), first + at, -1).to(torch.int32)
        if case["train"]:
            state["dq"] = randn(b, l, h, d).permute(0, 2, 1, 3)
            state["dk"] = randn(b, l, g, d).permute(0, 2, 1, 3)
    elif case["op"] == "cross":
        b, l, s, h, g, d = (case[n] for n in ("batch", "length", "keys", "heads", "kv", "dim"))
        kv = randn(b, s, 2, g, d).permute(2, 0, 3, 1, 4)   # rows of the frames' fused projection k | v
        state = {"q": randn(b, l, h, d).permute(0, 2, 1, 3), "k": kv[0], "v": kv[1],
                 "lens": ints(_lens(b, s, case["shortest"])), "q_lens": ints(_query_lens(case))}
        if case["train"]:
            state["dout"] = randn(b, l, h, d).permute(0, 2, 1, 3)
    else:
        m, n, k, group = case["rows"], case["n"], case["k"], case["group"]
        state = {"x": randn(m, k), "bias": randn(n, std=0.1),
                 "w": torch.randint(0, 16, (n, k), generator=gen, device=dev, dtype=torch.uint8),
                 "scale": (randn(n, k // group, std=0.3, dtype=torch.float32).exp() * (0.2 * k ** -0.5)).to(kind),
                 "zero": None}
        if case["zeros"]:
            state["zero"] = torch.randint(5, 11, (n, k // group), generator=gen, device=dev, dtype=torch.uint8)
    state["case"] = dict(case)
    if own:
        from __graft_entry__ import load_package

        state["sidon"] = load_package()
        if case["op"] == "int4":
            # laid out once, when the weights are loaded
            state["packed"] = state["sidon"].int4.pack_int4(state["w"], state["scale"], state["zero"])
    return state


# ---- one pass ---------------------------------------------------------------------


def run(state):
    case = state["case"]
    if own:
        return _own(state["sidon"], case, state)
    if case["op"] == "norms":
        return _plain_norms(case, state)
    if case["op"] == "cross":
        return _plain_cross(case, state)
    return _plain_int4(case, state)


def _own(sidon, case, s):
    if case["op"] == "norms":
        turn = {"cos": s["cos"], "sin": s["sin"], "q_pos": s["pos"], "k_pos": s["pos"], "eps": EPS,
                "interleaved": case["pairs"]}
        q, k = sidon.head_norm.qk_norm_rotary(s["q"], s["k"], s["q_w"], s["k_w"], **turn)
        if not case["train"]:
            return {"q": q, "k": k}
        dq, dk, dq_w, dk_w = sidon.head_norm.qk_norm_rotary_backward(s["dq"], s["dk"], s["q"], s["k"], s["q_w"],
                                                                     s["k_w"], **turn)
        return {"q": q, "k": k, "dq": dq, "dk": dk, "dq_w": dq_w, "dk_w": dk_w}
    if case["op"] == "cross":
        cross = sidon.cross_attention
        if not case["train"]:
            return {"out": cross.cross_attention(s["q"], s["k"], s["v"], lens=s["lens"], q_lens=s["q_lens"])}
        lse = torch.empty(s["q"].shape[:3], device=s["q"].device)
        out = cross.cross_attention(s["q"], s["k"], s["v"], lens=s["lens"], q_lens=s["q_lens"], lse=lse)
        dq, dk, dv = cross.cross_attention_backward(s["dout"], s["q"], s["k"], s["v"], out, lse, lens=s["lens"],
                                                    q_lens=s["q_lens"])
        return {"out": out, "dq": dq, "dk": dk, "dv": dv}
    return sidon.int4.int4_linear(s["x"], s["packed"], bias=s["bias"], act=None if case["act"] == "none" else "silu")


def _turn(x, cos, sin, pairs, back=False):
    """x [B, H, L, D] with its first 2 * cos.shape[-1] dimensions rotated (cos, sin [B, 1, L, R / 2])."""
    half = cos.shape[-1]
    if back:
        sin = -sin
    head, rest = x[..., :2 * half], x[..., 2 * half:]
    if pairs:
        a, b = head[..., 0::2], head[..., 1::2]
        return torch.cat((torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2), rest), -1)
    a, b = head[..., :half], head[..., half:]
    return torch.cat((a * cos - b * sin, a * sin + b * cos, rest), -1)


def _plain_norms(case, s):
    valid = (s["pos"] >= 0).view(case["batch"], 1, case["length"], 1)
    cos = sin = torch.empty(case["batch"], 1, case["length"], 0, device=s["q"].device)
    if case["rot"]:
        at = s["pos"].clamp_min(0).long()
        cos, sin = s["cos"][at].unsqueeze(1), s["sin"][at].unsqueeze(1)
    out = {}
    for name in ("q", "k"):
        x = s[name].float()
        r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
        y = _turn(x * r * s[name + "_w"], cos, sin, case["pairs"])
        out[name] = torch.where(valid, y, 0.0).to(s[name].dtype)
        if case["train"]:
            g = torch.where(valid, _turn(s["d" + name].float(), cos, sin, case["pairs"], back=True), 0.0)
            n = torch.where(valid, x * r, 0.0)
            out[f"d{name}_w"] = (g * n).sum((0, 1, 2))
            g = g * s[name + "_w"]
            out["d" + name] = (r * (g - n * (g * n).mean(-1, keepdim=True))).to(s[name].dtype)
    return out


def _plain_cross(case, s):
    b, l, n, h, g, d = (case[name] for name in ("batch", "length", "keys", "heads", "kv", "dim"))
    dev, kind = s["q"].device, s["q"].dtype
    seen = torch.arange(n, device=dev).view(1, 1, 1, n) < s["lens"].view(b, 1, 1, 1)
    here = (torch.arange(l, device=dev).view(1, 1, l, 1) < s["q_lens"].view(b, 1, 1, 1))
    out = {"out": torch.empty(b, h, l, d, device=dev, dtype=kind)}
    if case["train"]:
        out["dq"] = torch.empty(b, h, l, d, device=dev, dtype=kind)
        out["dk"] = torch.empty(b, g, n, d, device=dev, dtype=kind)
        out["dv"] = torch.empty(b, g, n, d, device=dev, dtype=kind)
    per = h // g
    # a key head at a time, so that the maps of long sequences fit
    for head in range(g):
        block = slice(head * per, (head + 1) * per)
        used = seen.view(b, n, 1)
        k = torch.where(used, s["k"][:, head].float(), 0.0)
        v = torch.where(used, s["v"][:, head].float(), 0.0)
        q = torch.where(here, s["q"][:, block].float(), 0.0).reshape(b, per * l, d)
        score = torch.matmul(q, k.transpose(1, 2).contiguous()).view(b, per, l, n) * d ** -0.5
        score = score.masked_fill(~seen, float("-inf"))
        top = score.amax(-1, keepdim=True)
        p = torch.exp(score - torch.where(top == float("-inf"), 0.0, top))
        total = p.sum(-1, keepdim=True)
        p = torch.where(here, p / torch.where(total == 0, 1.0, total), 0.0)
        out["out"][:, block] = torch.matmul(p.view(b, per * l, n), v).view(b, per, l, d).to(kind)
        if case["train"]:
            p = p.view(b, per * l, n)
            do = torch.where(here, s["dout"][:, block].float(), 0.0).reshape(b, per * l, d)
            out["dv"][:, head] = torch.matmul(p.transpose(1, 2).contiguous(), do).to(kind)
            dp = torch.matmul(do, v.transpose(1, 2).contiguous())
            ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * d ** -0.5
            out["dq"][:, block] = torch.matmul(ds, k).view(b, per, l, d).to(kind)
            out["dk"][:, head] = torch.matmul(ds.transpose(1, 2).contiguous(), q).to(kind)
    return out


def _plain_int4(case, s):
    n, k, group = case["n"], case["k"], case["group"]
    zero = 8.0 if s["zero"] is None else s["zero"].float().unsqueeze(-1)
    w = (s["w"].view(n, k // group, group).float() - zero) * s["scale"].float().unsqueeze(-1)
    y = s["x"].float() @ w.view(n, k).t() + s["bias"].float()
    if case["act"] == "silu":
        y = y * torch.sigmoid(y)
    return y.to(s["x"].dtype)


# ---- what a case cannot do without -------------------------------------------------


def work(case):
    size = 4 if case["type"] == "fp32" else 2
    if case["op"] == "norms":
        width = (case["heads"] + case["kv"]) * case["dim"]
        rows = case["batch"] * case["length"]
        valid = sum(_lens(case["batch"], case["length"], case["shortest"]))
        small = 8 * case["dim"] + 4 * rows + 4 * case["rot"] * min(valid, PLACES)
        if not case["train"]:
            return {"bytes": size * width * (valid + rows) + small, "flops": 8 * width * valid}
        return {"bytes": size * width * (2 * valid + 2 * rows) + small + 8 * case["dim"],
                "flops": 24 * width * valid}
    if case["op"] == "cross":
        b, h, g, d = case["batch"], case["heads"], case["kv"], case["dim"]
        lens, q_lens = _lens(b, case["keys"], case["shortest"]), _query_lens(case)
        pairs = sum(i * j for i, j in zip(lens, q_lens))
        rows, valid, keys = b * case["length"] * h * d, sum(q_lens) * h * d, sum(lens) * g * d
        if not case["train"]:
            return {"bytes": 2 * (valid + rows + 2 * keys) + 8 * b, "flops": 4 * d * h * pairs}
        return {"bytes": 2 * (2 * valid + 2 * rows + 2 * keys + 2 * b * case["keys"] * g * d) + 8 * b,
                "flops": 14 * d * h * pairs}
    m, n, k, group = case["rows"], case["n"], case["k"], case["group"]
    return {"bytes": n * k // 2 + n * k // group * (3 if case["zeros"] else 2) + 2 * (m * k + n + m * n),
            "flops": 2 * m * n * k}


# ---- the definitions in 64 bits ----------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norms":
        return _exact_norms(case, s)
    if case["op"] == "cross":
        return _exact_cross(case, s)
    return _exact_int4(case, s)


def _exact_norms(case, s):
    b, l, d, half = case["batch"], case["length"], case["dim"], case["rot"] // 2
    out = {}
    for name, heads in (("q", case["heads"]), ("k", case["kv"])):
        y = torch.zeros(b, heads, l, d, dtype=torch.float64, device=s["q"].device)
        dx, dw = torch.zeros_like(y), torch.zeros(d, dtype=torch.float64, device=y.device)
        for i, n in enumerate(_lens(b, l, case["shortest"])):
            if n == 0:
                continue
            with torch.enable_grad():
                x = s[name][i, :, :n].double().requires_grad_(case["train"])
                w = s[name + "_w"].double().requires_grad_(case["train"])
                z = x / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS) * w
                if half:
                    at = s["pos"][i, :n].long()
                    cos, sin = s["cos"][at].double(), s["sin"][at].double()
                    # as complex numbers
                    head = z[..., :2 * half]
                    head = head.unflatten(-1, (half, 2)) if case["pairs"] else head.unflatten(-1, (2, half)).transpose(-1, -2)
                    turned = torch.view_as_real(torch.view_as_complex(head.contiguous()) * torch.complex(cos, sin))
                    turned = turned.flatten(-2) if case["pairs"] else turned.transpose(-1, -2).flatten(-2)
                    z = torch.cat((turned, z[..., 2 * half:]), -1)
                y[i, :, :n] = z.detach()
                if case["train"]:
                    gx, gw = torch.autograd.grad(z, (x, w), s["d" + name][i, :, :n].double())
                    dx[i, :, :n] = gx
                    dw += gw
        out[name] = y
        if case["train"]:
            out["d" + name], out[f"d{name}_w"] = dx, dw
    return out


def _exact_cross(case, s):
    b, l, h, g, d = (case[n] for n in ("batch", "length", "heads", "kv", "dim"))
    zeros = lambda t: torch.zeros(t.shape, dtype=torch.float64, device=t.device)  # noqa: E731
    out = {"out": zeros(s["q"])}
    if case["train"]:
        out.update(dq=zeros(s["q"]), dk=zeros(s["k"]), dv=zeros(s["v"]))
    for i, (n, m) in enumerate(zip(_lens(b, case["keys"], case["shortest"]), _query_lens(case))):
        for head in range(h if n and m else 0):
            kv = head // (h // g)
            with torch.enable_grad():
                q, k, v = (t.double().requires_grad_(case["train"])
                           for t in (s["q"][i, head, :m], s["k"][i, kv, :n], s["v"][i, kv, :n]))
                o = torch.softmax(q @ k.t() / math.sqrt(d), -1) @ v
                out["out"][i, head, :m] = o.detach()
                if case["train"]:
                    dq, dk, dv = torch.autograd.grad(o, (q, k, v), s["dout"][i, head, :m].double())
                    out["dq"][i, head, :m] = dq
                    out["dk"][i, kv, :n] += dk
                    out["dv"][i, kv, :n] += dv
    return out


def _exact_int4(case, s):
    group = case["group"]
    out = torch.zeros(case["rows"], case["n"], dtype=torch.float64, device=s["x"].device)
    for j in range(case["k"] // group):
        part = slice(j * group, (j + 1) * group)
        w = s["w"][:, part].double()
        w -= 8 if s["zero"] is None else s["zero"][:, j:j + 1].double()
        out += (s["x"][:, part].double() @ w.t()) * s["scale"][:, j].double()
    out += s["bias"].double()
    return out / (1 + torch.exp(-out)) if case["act"] == "silu" else out
