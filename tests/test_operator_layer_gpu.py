"""The language-model operators run together, as a layer and as the encoder use
them (needs an MI355X).

Bars.  Each 16-bit rounding between two operators is a relative error of about
2^-12 rms (fp16; 2^-9 bf16); a layer has five of them (normed rows, low-rank products,
projected rows, probabilities, context), each passed on with a gain of about one,
so the output's relative error is near sqrt(5) 2^-12 of the branch: 65 dB (47 in
bf16).  10 dB are left for gains above one (small denominators of the norms).  The
encoder's bar is that of its own tests against the oracle."""

from __future__ import annotations

import sys

import pytest
import torch

from conftest import ROOT

sys.path.insert(0, str(ROOT / "tests" / "golden"))

from make_encoder_golden import encoder_features, encoder_weights  # noqa: E402
from oracle.encoder_oracle import encoder_reference  # noqa: E402
from oracle.flexrel_oracle import errors  # noqa: E402
from test_diff_attention_gpu import reference as attention_reference  # noqa: E402
from test_group_norm_gpu import reference as norm_reference  # noqa: E402

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")


def snr(want, got):
    return errors(want.double().cpu().numpy(), got.double().cpu().numpy())["snr_db"]


class Layer:
    """group norm -> adapted q | k | v -> differential attention -> adapted
    projection into the stream, for H heads of two 64-wide maps."""

    def __init__(self, sidon, heads, kv, hidden, kind, adapters, seed):
        gen = torch.Generator().manual_seed(seed)

        def randn(*shape, std=1.0, dtype=kind):
            return (torch.randn(*shape, generator=gen) * std).to(dtype).to(DEV)

        self.sidon, self.h, self.g, self.hid, self.kind = sidon, heads, kv, hidden, kind
        n = heads * 128 + kv * 256
        self.gn = (1 + randn(hidden, std=0.1, dtype=torch.float32), randn(hidden, std=0.1, dtype=torch.float32))
        self.qkv_w, self.qkv_b = randn(n, hidden, std=hidden ** -0.5), randn(n, std=0.1)
        self.out_w = randn(hidden, heads * 128, std=(heads * 128) ** -0.5)
        self.qkv_low = (randn(adapters, 16, hidden, std=hidden ** -0.5), randn(adapters, n, 16, std=0.1),
                        randn(adapters, dtype=torch.float32).abs())
        self.out_low = (randn(adapters, 8, heads * 128, std=(heads * 128) ** -0.5), randn(adapters, hidden, 8, std=0.1),
                        randn(adapters, dtype=torch.float32).abs())
        self.lam = randn(heads, 4, 64, std=0.1, dtype=torch.float32)
        self.norm_w = 1 + randn(128, std=0.1, dtype=torch.float32)

    def split(self, qkv, batch):
        q, k, v = qkv.view(batch, -1, qkv.shape[1]).split([self.h * 128, self.g * 128, self.g * 128], -1)
        return (q.unflatten(-1, (self.h, 2, 64)).permute(0, 2, 3, 1, 4),
                k.unflatten(-1, (self.g, 2, 64)).permute(0, 2, 3, 1, 4),
                v.unflatten(-1, (self.g, 128)).permute(0, 2, 1, 3))

    def project(self, xn, ids):
        return self.sidon.adapters.adapter_linear(xn, self.qkv_w, self.qkv_b, *self.qkv_low, ids)

    def attend(self, q, k, v, lens, causal):
        batch, _, _, length, _ = q.shape
        ctx = torch.empty(batch, length, self.h, 128, dtype=self.kind, device=DEV)
        self.sidon.diff_attention.diff_attention(q, k, v, self.lam, 0.3, lens=lens, causal=causal, norm_w=self.norm_w,
                                                 out=ctx.permute(0, 2, 1, 3))
        return ctx.view(batch * length, self.h * 128)

    def __call__(self, x, batch, lens, ids):
        xn = self.sidon.conformer.group_norm_act(x.to(self.kind), batch, 8, *self.gn, lens=lens, act="silu")
        q, k, v = self.split(self.project(xn, ids), batch)
        return self.sidon.adapters.adapter_residual(x, self.attend(q, k, v, lens, False), self.out_w, *self.out_low, ids)

    def exact(self, x, batch, lens, ids):
        def projection(a, w, bias, low):
            y = a @ w.double().t() + (0 if bias is None else bias.double())
            rows = a.shape[0] // batch
            for i, e in enumerate(ids.tolist()):
                if 0 <= e < low[0].shape[0]:
                    at = slice(i * rows, (i + 1) * rows)
                    y[at] += low[2][e].double() * (a[at] @ low[0][e].double().t()) @ low[1][e].double().t()
            return y

        xn, _ = norm_reference(x.to(self.kind), batch, 8, *self.gn, 1e-5, lens.tolist(), "silu")
        q, k, v = self.split(projection(xn, self.qkv_w, self.qkv_b, self.qkv_low), batch)
        ctx, _ = attention_reference(Cast(q, self.kind), k, v, self.lam, 0.3, lens.tolist(), False, self.norm_w, 1e-5)
        ctx = ctx.permute(0, 2, 1, 3).reshape(-1, self.h * 128)
        return x.double() + projection(ctx, self.out_w, None, self.out_low)


class Cast:
    """A float64 tensor that says it is of another type (for the tolerances that
    the reference computes beside its result)."""

    def __init__(self, t, dtype):
        self.t, self.dtype, self.shape, self.device = t, dtype, t.shape, t.device

    def __getitem__(self, at):
        return self.t[at]


@pytest.mark.parametrize("kind,bar", [(torch.float16, 55), (torch.bfloat16, 37)], ids=str)
def test_layer_against_float64(sidon, kind, bar):
    layer = Layer(sidon, 4, 2, 256, kind, 3, seed=5)
    lens = torch.tensor([150, 97, 1, 0], dtype=torch.int32, device=DEV)
    ids = torch.tensor([2, -1, 0, 1], dtype=torch.int32, device=DEV)
    x = torch.randn(4 * 150, 256, generator=torch.Generator().manual_seed(6)).to(DEV)
    want = layer.exact(x, 4, lens, ids)
    before = x.clone()
    got = layer(x, 4, lens, ids)
    assert got is x and torch.isfinite(got).all()
    for b, n in enumerate(lens.tolist()):
        at = slice(b * 150, b * 150 + n)
        if n > 1:
            # (the branch alone, so that the stream does not hide it)
            assert snr(want[at] - before[at].double(), got[at].double() - before[at].double()) > bar, b


@pytest.mark.parametrize("kind", [torch.float16, torch.bfloat16], ids=str)
def test_prompt_and_single_tokens_are_one_sequence(sidon, kind):
    """A causal prompt into a cache, then single tokens of three streams of
    different age, each with its adapter, against the whole sequences at once."""
    layer = Layer(sidon, 4, 2, 256, kind, 3, seed=8)
    prompts, steps, cap = [70, 33, 1], 5, 96
    total = [n + steps for n in prompts]
    ids = torch.tensor([1, -1, 2], dtype=torch.int32, device=DEV)
    gen = torch.Generator().manual_seed(9)
    x = torch.randn(3, cap, 256, generator=gen).to(kind).to(DEV)
    # all at once
    lens = torch.tensor(total, dtype=torch.int32, device=DEV)
    q, k, v = layer.split(layer.project(x.view(-1, 256), ids), 3)
    whole = []
    for b in range(3):
        n = total[b]
        whole.append(layer.attend(q[b:b + 1, :, :, :n], k[b:b + 1], v[b:b + 1], lens[b:b + 1], True))
    # prompts, then tokens against the cache
    k_cache, v_cache = torch.full_like(k, float("nan")), torch.full_like(v, float("nan"))
    for b, n in enumerate(prompts):
        qp, kp, vp = layer.split(layer.project(x[b, :n], ids[b:b + 1]), 1)
        k_cache[b, :, :, :n], v_cache[b, :, :n] = kp[0], vp[0]
        out = layer.attend(qp, k_cache[b:b + 1], v_cache[b:b + 1],
                           torch.tensor([n], dtype=torch.int32, device=DEV), True)
        # the same arithmetic but for the shared projection's tile and the order of sums
        assert snr(whole[b][:n], out) > (55 if kind == torch.float16 else 37)
    at = torch.tensor(prompts, device=DEV)
    rows = torch.arange(3, device=DEV)
    for step in range(steps):
        token = x[rows, at + step]
        qt, kt, vt = layer.split(layer.project(token, ids), 3)
        k_cache[rows, :, :, at + step] = kt[:, :, :, 0]
        v_cache[rows, :, at + step] = vt[:, :, 0]
        out = layer.attend(qt, k_cache, v_cache, (at + step + 1).to(torch.int32), True)
        for b in range(3):
            assert snr(whole[b][prompts[b] + step], out[b]) > (55 if kind == torch.float16 else 37), (b, step)


# ---- the encoder ---------------------------------------------------------------------


def variants(weights, seed):
    """Three variants: all projections at rank 4, some at other ranks, none."""
    gen = torch.Generator().manual_seed(seed)

    def pair(w, r):
        return (torch.randn(r, w.shape[1], generator=gen) * w.shape[1] ** -0.5,
                torch.randn(w.shape[0], r, generator=gen) * 0.5 * r ** -0.5)

    names = ("ffn1_w1", "ffn1_w2", "q_w", "k_w", "v_w", "out_w", "pw2_w", "ffn2_w1", "ffn2_w2")
    full = [{n: pair(p[n], 4) for n in names} for p in weights["layers"]]
    some = [{n: pair(p[n], r) for n, r in (("q_w", 3), ("v_w", 9), ("ffn2_w2", 16))} for p in weights["layers"]]
    return [(0.5, full), (0.25, some), (1.0, [{} for _ in weights["layers"]])]


def merged(weights, variant):
    scale, layers = variant
    out = dict(weights, layers=[dict(p) for p in weights["layers"]])
    for p, low in zip(out["layers"], layers):
        for name, (a, b) in low.items():
            p[name] = p[name].double() + scale * b.double() @ a.double()
    return out


def test_adapted_encoder_against_merged_weights(sidon):
    weights = encoder_weights(2, 2, seed=4)
    packed = sidon.encoder.pack_weights(weights)
    enc = sidon.encoder.HipEncoder(packed, DEV)
    tuned = variants(weights, 3)
    adapters = sidon.encoder.pack_adapters(packed, tuned, device=DEV)
    assert set(adapters[0]) == {"ffn1_w1", "ffn1_w2", "qkv_w", "out_w", "pw2_w", "ffn2_w1", "ffn2_w2"}
    lens, ids = [90, 71, 90, 33, 90], [1, 0, -1, 0, 2]
    feats = encoder_features(5, 90, 7).float().to(DEV)
    frames = torch.tensor(lens, dtype=torch.int32, device=DEV)
    which = torch.tensor(ids, dtype=torch.int32, device=DEV)
    ws = enc.workspace(5 * 90, rank=32)
    got = enc(feats, frames, workspace=ws, adapters=adapters, ids=which)
    plain = enc(feats, frames)
    for b, (n, e) in enumerate(zip(lens, ids)):
        w = weights if e < 0 else merged(weights, tuned[e])
        want = encoder_reference(feats[b:b + 1].double().cpu(), w, [n], dtype=torch.float64)[0, :n]
        assert snr(want, got[b, :n]) > 60, b
        if e in (0, 1):   # (the adapters matter)
            assert snr(want, plain[b, :n]) < 30, b
    # captured, with other variants written between the replays
    out = torch.empty_like(got)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        enc(feats, frames, out=out, workspace=ws, adapters=adapters, ids=which)
    for turn in range(3):
        which.copy_(torch.tensor([(e + turn) % 3 for e in range(5)], dtype=torch.int32))
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        want = enc(feats, frames, adapters=adapters, ids=which)
        for b, n in enumerate(lens):
            assert torch.equal(out[b, :n], want[b, :n])


def test_adapted_encoder_at_its_own_width(sidon):
    """Hidden 1024 (16 heads), feed-forward 4096, one layer, where the projections
    take the wide tiles, with a captured call on the encoder's own workspace."""
    weights = encoder_weights(16, 1, seed=6, inter_mult=4)
    packed = sidon.encoder.pack_weights(weights)
    enc = sidon.encoder.HipEncoder(packed, DEV)
    gen = torch.Generator().manual_seed(5)
    low = {n: (torch.randn(8, w.shape[1], generator=gen) * w.shape[1] ** -0.5, torch.randn(w.shape[0], 8, generator=gen) * 0.2)
           for n in ("ffn1_w1", "ffn1_w2", "q_w", "k_w", "v_w", "out_w", "pw2_w", "ffn2_w1", "ffn2_w2")
           for w in (weights["layers"][0][n],)}
    tuned = (0.5, [low])
    adapters = sidon.encoder.pack_adapters(packed, [(1.0, [{}]), tuned], device=DEV)
    lens, ids = [400, 333, 150], [1, -1, 1]
    feats = encoder_features(3, 400, 9).float().to(DEV)
    frames = torch.tensor(lens, dtype=torch.int32, device=DEV)
    which = torch.tensor(ids, dtype=torch.int32, device=DEV)
    ws = enc.workspace(3 * 400, rank=24)
    got = enc(feats, frames, workspace=ws, adapters=adapters, ids=which).clone()
    for b, (n, e) in enumerate(zip(lens, ids)):
        want = encoder_reference(feats[b:b + 1].double().cpu(), weights if e < 0 else merged(weights, tuned), [n],
                                 dtype=torch.float64)[0, :n]
        assert snr(want, got[b, :n]) > 60, b
    out = torch.empty_like(got)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        enc(feats, frames, out=out, workspace=ws, adapters=adapters, ids=which)
    for _ in range(3):
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        for b, n in enumerate(lens):
            assert torch.equal(out[b, :n], got[b, :n])


def test_adapted_encoder_refusals(sidon):
    weights = encoder_weights(2, 2, seed=4)
    packed = sidon.encoder.pack_weights(weights)
    enc = sidon.encoder.HipEncoder(packed, DEV)
    adapters = sidon.encoder.pack_adapters(packed, variants(weights, 1), device=DEV)
    feats = torch.zeros(2, 10, 160, device=DEV)
    ids = torch.zeros(2, dtype=torch.int32, device=DEV)
    for bad in (dict(adapters=adapters), dict(ids=ids), dict(adapters=adapters[:1], ids=ids),
                dict(adapters=adapters, ids=ids[:1])):
        with pytest.raises(ValueError):
            enc(feats, **bad)
    with pytest.raises(ValueError, match="no adapters"):
        sidon.encoder.pack_adapters(packed, [(1.0, [{"pw1_w": None}, {}])])
    with pytest.raises(ValueError, match="layers"):
        sidon.encoder.pack_adapters(packed, [(1.0, [{}])])
    with pytest.raises(ValueError, match="q_w"):
        sidon.encoder.pack_adapters(packed, [(1.0, [{"q_w": (torch.ones(2, 64), torch.ones(128, 2))}, {}])])
