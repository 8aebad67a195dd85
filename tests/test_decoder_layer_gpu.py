"""The decoder's operators run together over the encoder's frames: 4-bit
projections, norms with rotation, cross attention and their gradients (needs an
MI355X).

Bars.  Each 16-bit rounding between two operators is a relative error of about
2^-12 rms (fp16; 2^-9 bf16).  A layer's branch has eight: q and k as projected and as
normed (four, each moving the scores, which have a deviation near one, and with them
the probabilities, by as much), v, probabilities, context and output, passed on with a gain of
about one: sqrt(8) 2^-12 of the branch, 63 dB (45 in bf16).  10 dB are left for gains above one.
Gradients: the normed q and k, out, probabilities, dS, the gradients of the normed and
those of the inputs, seven or eight of the same size."""

from __future__ import annotations

import sys

import pytest
import torch

from conftest import ROOT

sys.path.insert(0, str(ROOT / "tests" / "golden"))

from make_encoder_golden import encoder_features, encoder_weights  # noqa: E402
from oracle import decoder_oracle as oracle  # noqa: E402
from oracle.flexrel_oracle import errors  # noqa: E402

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
BARS = [(torch.float16, 53), (torch.bfloat16, 35)]


def snr(want, got):
    return errors(want.detach().double().cpu().numpy(), got.double().cpu().numpy())["snr_db"]


class Layer:
    """q from tokens, k | v from frames by 4-bit projections, normed and (tokens only)
    rotated heads, attention of the tokens over the frames, 4-bit projection back."""

    def __init__(self, sidon, heads, kv, dim, hidden, kind, seed, zeros=True, group=64):
        gen = torch.Generator().manual_seed(seed)
        self.sidon, self.h, self.g, self.d, self.kind = sidon, heads, kv, dim, kind
        self.parts, self.packed = {}, {}
        for name, n, k in (("q", heads * dim, hidden), ("kv", 2 * kv * dim, hidden), ("o", hidden, heads * dim)):
            w = (torch.randn(n, k, generator=gen) * k ** -0.5).to(kind).to(DEV)
            self.parts[name] = (*sidon.int4.quantize_int4(w, group, zeros), (0.1 * torch.randn(n, generator=gen)).to(kind).to(DEV))
            self.packed[name] = sidon.int4.pack_int4(*self.parts[name][:3])
        self.w = [(1 + 0.1 * torch.randn(dim, generator=gen)).to(DEV) for _ in range(2)]
        angle = torch.arange(300).view(-1, 1) * 10000 ** (-torch.arange(dim // 2) / (dim // 2))
        self.cos, self.sin = angle.cos().to(DEV), angle.sin().to(DEV)

    def linear(self, x, name):
        return self.sidon.int4.int4_linear(x, self.packed[name], self.parts[name][3])

    def states(self, frames, lens):
        """frames [B, S, hidden] -> k | v rows [B, S, 2 Hk D], k normed in place; kept for all tokens."""
        b, s, hid = frames.shape
        kv = self.linear(frames.reshape(-1, hid), "kv").view(b, s, 2, self.g, self.d)
        k, v = kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2)
        self.sidon.head_norm.qk_norm_rotary(k, None, self.w[1], None, out_q=k)
        return k, v

    def __call__(self, x, k, v, lens, pos, q_lens=None):
        """x [B, L, hidden], pos [B, L] places -> [B, L, hidden]."""
        b, l, hid = x.shape
        q = self.linear(x.reshape(-1, hid), "q").view(b, l, self.h, self.d).transpose(1, 2)
        self.sidon.head_norm.qk_norm_rotary(q, None, self.w[0], None, self.cos, self.sin, pos, out_q=q)
        ctx = torch.empty(b, l, self.h, self.d, dtype=self.kind, device=DEV)
        self.sidon.cross_attention.cross_attention(q, k, v, lens, q_lens, out=ctx.transpose(1, 2))
        return self.linear(ctx.view(b * l, -1), "o").view(b, l, -1)

    def exact(self, x, frames, lens, pos):
        def linear(a, name):
            values, scales, zero, bias = self.parts[name]
            return oracle.int4(a.reshape(-1, a.shape[-1]), values, scales, zero, bias, None)[0].view(*a.shape[:-1], -1)

        b, l, _ = x.shape
        s = frames.shape[1]
        q = linear(x, "q").view(b, l, self.h, self.d).transpose(1, 2)
        kv = linear(frames, "kv").view(b, s, 2, self.g, self.d)
        q = oracle.norm_rotary(q, self.w[0], self.cos, self.sin, pos, 1e-6, False)[0]
        k = oracle.norm_rotary(kv[:, :, 0].transpose(1, 2), self.w[1], None, None, None, 1e-6, False)[0]
        ctx = oracle.cross(q, k, kv[:, :, 1].transpose(1, 2), lens.tolist(), None, self.d ** -0.5)[0]
        return linear(ctx.transpose(1, 2).reshape(b, l, -1), "o")


@pytest.mark.parametrize("kind,bar", BARS, ids=str)
@pytest.mark.parametrize("heads,kv,dim", [(4, 2, 64), (2, 2, 128)])
def test_layer_against_float64(sidon, kind, bar, heads, kv, dim):
    layer = Layer(sidon, heads, kv, dim, 256, kind, 5)
    gen = torch.Generator().manual_seed(6)
    x = torch.randn(3, 40, 256, generator=gen).to(kind).to(DEV)
    frames = torch.randn(3, 150, 256, generator=gen).to(kind).to(DEV)
    lens = torch.tensor([150, 97, 0], dtype=torch.int32, device=DEV)
    pos = torch.arange(40, dtype=torch.int32, device=DEV) + torch.tensor([[0], [100], [7]], dtype=torch.int32, device=DEV)
    want = layer.exact(x, frames, lens, pos)
    got = layer(x, *layer.states(frames, lens), lens, pos)
    assert torch.isfinite(got).all()
    for b in range(2):
        assert snr(want[b], got[b]) > bar, b
    assert (got[2] == layer.parts["o"][3]).all()   # (without frames: the bias)


@pytest.mark.parametrize("kind,bar", BARS, ids=str)
def test_tokens_over_encoded_speech(sidon, kind, bar):
    """A prompt and then single tokens, captured, over frames that the encoder has
    just written, with its device lengths; padded tokens by negative places."""
    enc = sidon.encoder.HipEncoder(sidon.encoder.pack_weights(encoder_weights(2, 2, seed=4)), DEV)
    feats = encoder_features(3, 90, 7).float().to(DEV)
    lens = torch.tensor([90, 71, 33], dtype=torch.int32, device=DEV)
    hidden = enc(feats, lens).to(kind)
    layer = Layer(sidon, 4, 1, 64, hidden.shape[-1], kind, 8, zeros=False, group=128)
    k, v = layer.states(hidden, lens)
    gen = torch.Generator().manual_seed(9)
    prompts, steps = torch.tensor([7, 12, 1], device=DEV), 4
    x = torch.randn(3, 16, hidden.shape[-1], generator=gen).to(kind).to(DEV)
    at = torch.arange(16, dtype=torch.int32, device=DEV).expand(3, 16).contiguous()
    want = layer.exact(x, hidden, lens, at)
    # prompts of different lengths as one padded batch
    place = torch.where(at[:, :12] < prompts.view(3, 1), at[:, :12], -1).int().contiguous()
    padded = torch.where((place < 0).unsqueeze(-1), float("nan"), x[:, :12])
    got = layer(padded, k, v, lens, place, prompts.int())
    bias = layer.linear(torch.zeros(1, 256, dtype=kind, device=DEV), "o")[0]
    for b, n in enumerate(prompts.tolist()):
        assert snr(want[b, :n], got[b, :n]) > bar, b
        assert (got[b, n:] == bias).all()
    # tokens one after another
    token, pos = torch.empty(3, 1, hidden.shape[-1], dtype=kind, device=DEV), torch.empty(3, 1, dtype=torch.int32, device=DEV)
    token.zero_()
    pos.zero_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer(token, k, v, lens, pos)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer(token, k, v, lens, pos)
    rows = torch.arange(3, device=DEV)
    for step in range(steps):
        token[:, 0] = x[rows, prompts + step]
        pos[:, 0] = prompts + step
        graph.replay()
        eager = layer(token, k, v, lens, pos)
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
        for b in range(3):
            assert snr(want[b, prompts[b] + step], out[b, 0]) > bar, (b, step)


class Heads(torch.autograd.Function):
    """Norm, rotation and attention as one step of a training program's graph."""

    @staticmethod
    def forward(ctx, sidon, q, k, v, q_w, k_w, cos, sin, pos, lens):
        qn, kn = sidon.head_norm.qk_norm_rotary(q, k, q_w, k_w, cos, sin, q_pos=pos)
        lse = q.new_empty(q.shape[:3], dtype=torch.float32)
        out = sidon.cross_attention.cross_attention(qn, kn, v, lens, lse=lse)
        ctx.sidon, ctx.turn = sidon, (cos, sin, pos, lens)
        ctx.save_for_backward(q, k, v, q_w, k_w, qn, kn, out, lse)
        return out

    @staticmethod
    def backward(ctx, dout):
        q, k, v, q_w, k_w, qn, kn, out, lse = ctx.saved_tensors
        cos, sin, pos, lens = ctx.turn
        dqn, dkn, dv = ctx.sidon.cross_attention.cross_attention_backward(dout, qn, kn, v, out, lse, lens)
        dq, dk, dq_w, dk_w = ctx.sidon.head_norm.qk_norm_rotary_backward(dqn, dkn, q, k, q_w, k_w, cos, sin, q_pos=pos,
                                                                         dq=dqn, dk=dkn)
        return None, dq, dk, dv, dq_w, dk_w, None, None, None, None


def exact_heads(q, k, v, q_w, k_w, cos, sin, pos, lens):
    """The same in float64 torch operations, which autograd follows."""
    def norm(x, w):
        return w * x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6)

    half = cos.shape[1]
    qn, kn = norm(q, q_w), norm(k, k_w)

    def turn(x, at):
        c, s = cos[at].unsqueeze(1), sin[at].unsqueeze(1)
        a, b, rest = x[..., :half], x[..., half:2 * half], x[..., 2 * half:]
        return torch.cat((a * c - b * s, a * s + b * c, rest), -1)

    qn = turn(qn, pos)
    kn = turn(kn, torch.arange(k.shape[2]).expand(k.shape[0], -1))
    times = q.shape[1] // k.shape[1]
    kn, vv = kn.repeat_interleave(times, 1), v.repeat_interleave(times, 1)
    scores = q.shape[-1] ** -0.5 * qn @ kn.transpose(-1, -2)
    hide = torch.arange(k.shape[2]) >= lens.view(-1, 1, 1, 1)
    return torch.softmax(scores.masked_fill(hide, float("-inf")), -1) @ vv


@pytest.mark.parametrize("kind,bar", BARS, ids=str)
@pytest.mark.parametrize("shape", [(2, 4, 2, 70, 150, 64), (2, 2, 1, 33, 200, 128), (3, 2, 2, 300, 131, 64)], ids=str)
def test_training_step(sidon, shape, kind, bar):
    """Gradients through norm, rotation and attention by the backward calls, against
    float64 autograd of the plain formulas, twice (leaves that hold a gradient add to it)."""
    b, h, g, l, s, d = shape
    gen = torch.Generator().manual_seed(l)
    rows = torch.randn(b, l, h, d, generator=gen).to(kind)
    frames = torch.randn(b, s, 2, g, d, generator=gen).to(kind)
    w = [1 + 0.1 * torch.randn(d, generator=gen) for _ in range(2)]
    angle = torch.rand(400, d // 4, generator=gen) * 6
    pos = torch.randint(0, 400, (b, l), generator=gen, dtype=torch.int32)
    lens = torch.tensor([s, s // 2, s - 1][:b], dtype=torch.int32)
    dout = torch.randn(b, l, h, d, generator=gen).to(kind)
    leaves = [t.to(DEV).requires_grad_() for t in (rows, frames, *w)]
    wants = [t.double().requires_grad_() for t in (rows, frames, *w)]
    for _ in range(2):
        q, kv = leaves[0].transpose(1, 2), leaves[1]
        out = Heads.apply(sidon, q, kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2), leaves[2], leaves[3],
                          angle.cos().to(DEV), angle.sin().to(DEV), pos.to(DEV), lens.to(DEV))
        out.backward(dout.to(DEV).transpose(1, 2))
        q, kv = wants[0].transpose(1, 2), wants[1]
        want = exact_heads(q, kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2), wants[2], wants[3],
                           angle.cos().double(), angle.sin().double(), pos, lens)
        want.backward(dout.double().transpose(1, 2))
        assert snr(want, out.detach()) > bar
        for name, got, ref in zip(("rows", "frames", "q_w", "k_w"), leaves, wants):
            assert got.grad.dtype == got.dtype and snr(ref.grad, got.grad) > bar, name
    # a padded frame has no part
    assert (leaves[1].grad[1, s // 2:] == 0).all()


def test_training_step_in_a_graph(sidon):
    """Both directions captured while tensors of an eager step of the same leaves live."""
    b, h, g, l, s, d, kind = 2, 4, 2, 40, 130, 64, torch.bfloat16
    gen = torch.Generator().manual_seed(3)
    q = torch.randn(b, l, h, d, generator=gen).to(kind).to(DEV).transpose(1, 2)
    kv = torch.randn(b, s, 2, g, d, generator=gen).to(kind).to(DEV)
    k, v = kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2)
    w = torch.ones(2, d, device=DEV)
    lens = torch.tensor([130, 60], dtype=torch.int32, device=DEV)
    dout = torch.randn(b, h, l, d, generator=gen).to(kind).to(DEV)
    hn, ca = sidon.head_norm, sidon.cross_attention

    def step():
        qn, kn = hn.qk_norm_rotary(q, k, w[0], w[1])
        lse = torch.empty(b, h, l, device=DEV)
        out = ca.cross_attention(qn, kn, v, lens, lse=lse)
        dqn, dkn, dv = ca.cross_attention_backward(dout, qn, kn, v, out, lse, lens)
        return out, dv, *hn.qk_norm_rotary_backward(dqn, dkn, q, k, w[0], w[1])

    leaf = w.clone().requires_grad_()
    live = (leaf * 2).sum()   # (an eager graph of a leaf that is still to run backward)
    eager = step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for i in range(3):
        q.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(i)))
        lens[1] = 50 * i
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(outs, want))
    live.backward()
    assert all(torch.isfinite(t).all() for t in eager) and (leaf.grad == 2).all()
