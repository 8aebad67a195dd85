"""The decoder operators' refusals, before any launch (no GPU)."""

from __future__ import annotations

import ctypes

import pytest
import torch

MB = 1 << 20
I64 = ctypes.c_int64


def _strides(values):
    return None if values is None else (I64 * len(values))(*values)


# ---- norm and rotation -------------------------------------------------------------


def _norm(lib, backward=False, **over):
    # B=2 items of L=10 tokens (S=12) of 4 and 2 heads of 64, rows of their own tensors
    a = dict(q=MB, k=2 * MB, yq=3 * MB, yk=4 * MB, gq=5 * MB, gk=6 * MB, qw=16, kw=16, cos=1024, sin=8192, places=20, rot=64,
             pairs=0, qp=None, kp=None, eps=1e-6, B=2, H=4, Hk=2, L=10, S=12, D=64, dtype=1, dqw=7 * MB, dkw=7 * MB + 256,
             ws=8 * MB, wsb=MB, qs=(2560, 64, 256), ks=(1536, 64, 128), yqs=(2560, 64, 256), yks=(1536, 64, 128),
             gqs=(2560, 64, 256), gks=(1536, 64, 128))
    a.update(over)
    st = {n: _strides(a[n]) for n in ("qs", "ks", "yqs", "yks", "gqs", "gks")}
    sizes = [a[n] for n in ("B", "H", "Hk", "L", "S", "D", "dtype")]
    turn = [a["cos"], a["sin"], a["places"], a["rot"], a["pairs"], a["qp"], a["kp"], a["eps"]]
    if backward:
        return lib.sidon_qk_norm_rotary_bwd(a["gq"], a["gk"], a["q"], a["k"], a["yq"], a["yk"], a["dqw"], a["dkw"], a["qw"],
                                            a["kw"], *turn, a["ws"], a["wsb"], *sizes, st["gqs"], st["gks"], st["qs"],
                                            st["ks"], st["yqs"], st["yks"], None)
    return lib.sidon_qk_norm_rotary(a["q"], a["k"], a["yq"], a["yk"], a["qw"], a["kw"], *turn, *sizes, st["qs"], st["ks"],
                                    st["yqs"], st["yks"], None)


NORM = [
    (dict(q=None), -1), (dict(k=None), -1), (dict(yq=None), -1), (dict(yk=None), -1), (dict(qw=None), -1), (dict(kw=None), -1),
    (dict(cos=None), -1), (dict(sin=None), -1), (dict(qs=None), -1), (dict(yks=None), -1), (dict(dtype=3), -2),
    (dict(dtype=-1), -2), (dict(B=0), -2), (dict(H=0), -2), (dict(Hk=-1), -2), (dict(L=0), -2), (dict(S=0), -2), (dict(D=8), -2),
    (dict(D=72), -2), (dict(D=272), -2), (dict(rot=8), -2), (dict(rot=80), -2), (dict(rot=-16), -2), (dict(places=0), -2),
    (dict(places=11), -2), (dict(eps=0.0), -2), (dict(eps=-1e-6), -2), (dict(eps=float("nan")), -2), (dict(eps=float("inf")), -2),
    (dict(H=4097), -2), (dict(L=1 << 27, H=4, places=1 << 28), -2), (dict(qs=(2560, 60, 256)), -3), (dict(qs=(2560, 64, -256)), -3),
    (dict(ks=(1 << 41, 64, 128)), -3), (dict(yqs=(2560, 64, 0)), -3), (dict(yqs=(0, 64, 256)), -3), (dict(yks=(1536, 32, 128)), -3),
    (dict(q=MB + 8), -4), (dict(yk=4 * MB + 8), -4), (dict(qw=20), -4), (dict(cos=1028), -4), (dict(qp=6), -4), (dict(kp=5), -4),
    (dict(dtype=0, qs=(2560, 66, 256)), -3),
    # outputs over what is read: other strides, the other side's rows, weights, tables, places
    (dict(yq=MB, yqs=(2560, 640, 64)), -2), (dict(yq=MB + 128), -2), (dict(yq=2 * MB), -2), (dict(yk=MB), -2), (dict(yk=3 * MB + 512), -2),
    (dict(qw=3 * MB), -2), (dict(kw=4 * MB + 2048), -2), (dict(cos=3 * MB + 4096), -2), (dict(qp=3 * MB), -2), (dict(kp=4 * MB), -2),
]
BACK = [
    (dict(gq=None), -1), (dict(gk=None), -1), (dict(dqw=None), -1), (dict(dkw=None), -1), (dict(ws=None), -1), (dict(gqs=None), -1),
    (dict(wsb=0), -2), (dict(ws=8 * MB + 4), -4), (dict(dqw=7 * MB + 2), -4), (dict(gq=5 * MB + 2), -4), (dict(gks=(1536, 64, 4)), -3),
    (dict(yq=5 * MB, yqs=(5120, 64, 256)), -2), (dict(yq=6 * MB), -2), (dict(dkw=7 * MB + 128), -2), (dict(dqw=16), -2),
    (dict(dqw=MB), -2), (dict(dqw=3 * MB), -2), (dict(dkw=8 * MB), -2), (dict(ws=2 * MB), -2), (dict(ws=3 * MB), -2), (dict(ws=6 * MB), -2),
    (dict(ws=1024), -2),
]


@pytest.mark.parametrize("over,code", NORM)
def test_norm_refuses(sidon, over, code):
    # fake addresses, never dereferenced: validation returns before any HIP call
    lib = sidon._lib.load()
    for backward in (False, True):
        assert _norm(lib, backward, **over) == code, backward
        assert lib.sidon_last_error().decode()


@pytest.mark.parametrize("over,code", BACK)
def test_norm_gradients_refuse(sidon, over, code):
    lib = sidon._lib.load()
    assert _norm(lib, True, **over) == code
    assert lib.sidon_last_error().decode()


@pytest.mark.parametrize("over", [
    dict(), dict(Hk=0, k=None, yk=None, kw=None, ks=None, yks=None, gk=None, gks=None, dkw=None), dict(rot=0, cos=None, sin=None),
    dict(yq=MB), dict(yq=MB, yk=2 * MB),
    # q | k | v rows of 8 heads, in place; outputs as column blocks of one tensor with their inputs
    dict(q=MB, k=MB + 512, yq=MB, yk=MB + 512, qs=(5120, 64, 512), ks=(6144, 64, 512), yqs=(5120, 64, 512), yks=(6144, 64, 512)),
    dict(q=MB, yq=MB + 512, qs=(5120, 64, 512), yqs=(5120, 64, 512)),
])
def test_norm_takes(sidon, over):
    """What reaches the device check (no GPU here): in place, column blocks, without k, without rotation."""
    lib = sidon._lib.load()
    for backward in (False, True):
        if torch.cuda.is_available():
            pytest.skip("fake addresses")
        assert _norm(lib, backward, **over) == -6, lib.sidon_last_error()


def test_norm_workspace(sidon):
    ws = sidon.head_norm.workspace_bytes
    assert ws(0, 4, 2, 10, 10, 64) == 0 and ws(1, 4, 2, 10, 10, 24) == 0 and ws(1, 4, 2, 10, 0, 64) == 0
    assert ws(1, 1, 0, 1, 0, 64) == 256 and ws(1, 16, 0, 1, 7, 64) == ws(1, 16, 0, 1, 0, 64) == 16 * 256
    for sizes in ((8, 16, 16, 4800, 4800, 64), (1, 4096, 4096, 1, 1, 256), (3, 17, 5, 301, 77, 128)):
        assert 0 < ws(*sizes) <= 2 * max(1024, sizes[1]) * sizes[-1] * 4


def test_norm_rejects_wrong_tensors(sidon):
    call, back = sidon.head_norm.qk_norm_rotary, sidon.head_norm.qk_norm_rotary_backward
    q, k, w = torch.zeros(2, 4, 3, 64), torch.zeros(2, 2, 5, 64), torch.ones(64)
    with pytest.raises(ValueError, match="HIP device"):
        call(q, k, w, w)
    with pytest.raises(TypeError, match="float32, float16 or bfloat16"):
        call(q.double(), k.double(), w, w)
    with pytest.raises(TypeError, match="torch.Tensor"):
        call(None, k, w, w)
    with pytest.raises(ValueError, match="B, heads"):
        call(q[0], k, w, w)
    with pytest.raises(ValueError, match="multiple of 16"):
        call(q[..., :40], k, w, w)
    with pytest.raises(ValueError, match="empty"):
        call(q[:, :, :0], k, w, w)
    with pytest.raises(ValueError, match="HIP device"):
        back(q, k, q, k, w, w)


# ---- cross attention ---------------------------------------------------------------


def _cross(lib, backward=False, **over):
    # B=2, H=4 heads over Hk=2, L=10, S=100, D=64: q and out [B, L, H, D] rows, k | v rows of one tensor
    a = dict(dout=6 * MB, q=MB, k=2 * MB, v=2 * MB + 256, out=3 * MB, lse=4 * MB, lens=16, q_lens=32, scale=0.125, dq=7 * MB, dk=8 * MB,
             dv=8 * MB + 256, ws=5 * MB, wsb=MB, B=2, H=4, Hk=2, L=10, S=100, D=64, dtype=1, qs=(2560, 64, 256), ks=(25600, 64, 256),
             vs=(25600, 64, 256), os=(2560, 64, 256), gs=(2560, 64, 256), dqs=(2560, 64, 256), dks=(25600, 64, 256),
             dvs=(25600, 64, 256))
    a.update(over)
    st = {n: _strides(a[n]) for n in ("qs", "ks", "vs", "os", "gs", "dqs", "dks", "dvs")}
    sizes = [a[n] for n in ("B", "H", "Hk", "L", "S", "D", "dtype")]
    if backward:
        return lib.sidon_cross_attention_bwd(a["dout"], a["q"], a["k"], a["v"], a["out"], a["lse"], a["lens"], a["q_lens"], a["scale"],
                                             a["dq"], a["dk"], a["dv"], a["ws"], a["wsb"], *sizes, st["gs"], st["qs"], st["ks"], st["vs"],
                                             st["os"], st["dqs"], st["dks"], st["dvs"], None)
    return lib.sidon_cross_attention(a["q"], a["k"], a["v"], a["lens"], a["q_lens"], a["scale"], a["out"], a["lse"], a["ws"], a["wsb"],
                                     *sizes, st["qs"], st["ks"], st["vs"], st["os"], None)


CROSS = [
    (dict(q=None), -1), (dict(k=None), -1), (dict(v=None), -1), (dict(out=None), -1), (dict(qs=None), -1), (dict(os=None), -1),
    (dict(dtype=0), -2), (dict(dtype=3), -2), (dict(B=0), -2), (dict(H=5), -2), (dict(Hk=0), -2), (dict(L=0), -2), (dict(S=0), -2),
    (dict(D=32), -2), (dict(D=96), -2), (dict(L=1 << 24), -2), (dict(S=(1 << 30) + 1), -2), (dict(scale=0.0), -2), (dict(scale=-1.0), -2),
    (dict(scale=float("nan")), -2), (dict(scale=float("inf")), -2), (dict(qs=(2560, 60, 256)), -3), (dict(ks=(25600, -64, 256)), -3),
    (dict(ks=(25600, 64, 1 << 25)), -3), (dict(vs=(25600, 64, 1 << 25)), -3), (dict(os=(1 << 41, 64, 256)), -3),
    (dict(q=MB + 8), -4), (dict(v=2 * MB + 8), -4), (dict(out=3 * MB + 2), -4),
    (dict(lens=18), -4), (dict(q_lens=33), -4), (dict(lse=4 * MB + 2), -4), (dict(ws=5 * MB + 8), -4),
]
FORWARD = [
    # rows of out that share memory
    (dict(os=(2560, 64, 0)), -3), (dict(os=(0, 64, 256)), -3), (dict(os=(2560, 32, 256)), -3), (dict(os=(2304, 64, 256)), -3),
    (dict(os=(640, 640, 64)), -3), (dict(ks=(1 << 40, 1 << 40, 0), B=1 << 22, H=4, Hk=4, L=1), -3),
]
CROSS_BACK = [
    (dict(dout=None), -1), (dict(lse=None), -1), (dict(dq=None), -1), (dict(dk=None), -1), (dict(dv=None), -1), (dict(ws=None), -1),
    (dict(gs=None), -1), (dict(dvs=None), -1), (dict(wsb=0), -2), (dict(S=(1 << 24) + 1), -2), (dict(B=1 << 19), -2),
    (dict(qs=(2560, 64, 1 << 25)), -3), (dict(gs=(2560, 64, 1 << 25)), -3), (dict(gs=(2560, 4, 256)), -3), (dict(dqs=(2560, 64, 0)), -3),
    (dict(dks=(25600, 32, 256)), -3), (dict(dvs=(0, 64, 256)), -3), (dict(dk=8 * MB + 2), -4), (dict(dout=6 * MB + 8), -4),
    (dict(dq=MB), -2), (dict(dq=3 * MB), -2), (dict(dq=6 * MB), -2), (dict(dk=2 * MB), -2), (dict(dv=8 * MB), -2), (dict(dk=7 * MB), -2),
    (dict(ws=MB), -2), (dict(ws=7 * MB), -2), (dict(ws=4 * MB), -2), (dict(lse=7 * MB), -2), (dict(lens=8 * MB), -2), (dict(q_lens=8 * MB + 1024), -2),
]


@pytest.mark.parametrize("over,code", CROSS)
def test_cross_attention_refuses(sidon, over, code):
    lib = sidon._lib.load()
    for backward in (False, True):
        assert _cross(lib, backward, **over) == code, backward
        assert lib.sidon_last_error().decode()


@pytest.mark.parametrize("over,code", FORWARD)
def test_cross_attention_forward_refuses(sidon, over, code):
    lib = sidon._lib.load()
    assert _cross(lib, **over) == code
    assert lib.sidon_last_error().decode()


@pytest.mark.parametrize("over,code", CROSS_BACK)
def test_cross_attention_gradients_refuse(sidon, over, code):
    lib = sidon._lib.load()
    assert _cross(lib, True, **over) == code
    assert lib.sidon_last_error().decode()


@pytest.mark.parametrize("over", [
    # out over q, k, v, lse, the lengths; lse over them; q and out a column apart, but wider than that
    dict(out=MB), dict(out=2 * MB), dict(out=2 * MB + 25600), dict(lse=MB), dict(lse=3 * MB), dict(lse=2 * MB + 512), dict(lens=3 * MB),
    dict(q_lens=3 * MB + 512), dict(lens=4 * MB), dict(out=MB + 256, qs=(5120, 64, 512), os=(5120, 64, 512)),
])
def test_cross_attention_refuses_overlaps(sidon, over):
    lib = sidon._lib.load()
    assert _cross(lib, **over) == -2
    assert "apart" in lib.sidon_last_error().decode()


@pytest.mark.parametrize("over", [dict(), dict(lens=None, q_lens=None), dict(lse=None), dict(ws=None, wsb=0),
                                  dict(out=MB + 512, qs=(5120, 64, 512), os=(5120, 64, 512))])
def test_cross_attention_takes(sidon, over):
    """What reaches the device check (no GPU here)."""
    if torch.cuda.is_available():
        pytest.skip("fake addresses")
    assert _cross(sidon._lib.load(), **over) == -6, sidon._lib.load().sidon_last_error()


def test_cross_attention_gradients_take(sidon):
    if torch.cuda.is_available():
        pytest.skip("fake addresses")
    lib = sidon._lib.load()
    for over in (dict(), dict(lens=None, q_lens=None), dict(gs=(0, 0, 0)),
                 # dq beside q, dk | dv beside k | v in rows of one tensor each
                 dict(q=MB, dq=MB + 512, qs=(5120, 64, 512), dqs=(5120, 64, 512))):
        assert _cross(lib, True, **over) == -6, lib.sidon_last_error()


def test_cross_attention_workspaces(sidon):
    lib = sidon._lib.load()
    ws = lib.sidon_cross_attention_workspace_bytes
    assert ws(1, 8, 3, 1, 100, 64) == 0 and ws(8, 16, 16, 4800, 4800, 64) == 0
    one = ws(1, 8, 8, 1, 4800, 64)   # split over the chip
    assert one % (8 * (16 + 64 * 4)) == 0 and 1 < one // (8 * (16 + 64 * 4)) <= 64
    back = sidon.cross_attention.backward_workspace_bytes
    assert back(1, 8, 3, 1, 100, 64, torch.float16) == 0 and back(1, 8, 8, 1, 100, 64, torch.float32) == 0
    assert back(2, 4, 2, 33, 100, 64, torch.bfloat16) == 2 * 4 * 2 * 64 * 4
    assert back(2, 4, 2, 33, 100, 64, torch.float16) == 2 * 4 * 2 * (96 + 1) * 4 + 2 * 2 * 4 * 4


def test_cross_attention_rejects_wrong_tensors(sidon):
    call = sidon.cross_attention.cross_attention
    q, k = torch.zeros(1, 2, 3, 64, dtype=torch.float16), torch.zeros(1, 1, 5, 64, dtype=torch.float16)
    with pytest.raises(ValueError, match="HIP device"):
        call(q, k, k)
    with pytest.raises(TypeError, match="torch.Tensor"):
        call(q, k, None)
    with pytest.raises(ValueError, match="belong together"):
        call(q, k, k[..., :32])
    with pytest.raises(ValueError, match="share"):
        call(q, torch.zeros(1, 3, 5, 64, dtype=torch.float16), torch.zeros(1, 3, 5, 64, dtype=torch.float16))
    with pytest.raises(ValueError, match="H, L"):
        call(q[..., :32], k[..., :32], k[..., :32])
    with pytest.raises(TypeError, match="float16"):
        call(q.float(), k.float(), k.float())
    with pytest.raises(ValueError, match="empty"):
        call(q[:, :, :0], k, k)
    with pytest.raises(ValueError, match="HIP device"):
        sidon.cross_attention.cross_attention_backward(q, q, k, k, q, torch.zeros(1, 2, 3))


# ---- 4-bit projection --------------------------------------------------------------


def _int4(lib, **over):
    a = dict(x=MB, ldx=256, words=2 * MB, scales=3 * MB, bias=4 * MB, y=5 * MB, ldy=48, M=7, N=48, K=256, group=64, zeros=1, act=0, dtype=1)
    a.update(over)
    return lib.sidon_int4_linear(*[a[n] for n in ("x", "ldx", "words", "scales", "bias", "y", "ldy", "M", "N", "K", "group", "zeros",
                                                  "act", "dtype")], None)


@pytest.mark.parametrize("over,code", [
    (dict(x=None), -1), (dict(words=None), -1), (dict(scales=None), -1), (dict(y=None), -1), (dict(dtype=0), -2), (dict(dtype=3), -2),
    (dict(act=2), -2), (dict(act=-1), -2), (dict(M=0), -2), (dict(N=0), -2), (dict(K=0), -2), (dict(M=(1 << 21) + 1), -2),
    (dict(N=(1 << 24) + 1), -2), (dict(K=(1 << 20) + 128, ldx=1 << 21), -2), (dict(group=16), -2), (dict(group=256), -2), (dict(K=224), -2),
    (dict(K=192, group=128), -2), (dict(ldx=248), -3), (dict(ldx=260), -3), (dict(ldy=47), -3), (dict(ldx=1 << 41), -3),
    (dict(x=MB + 8), -4), (dict(words=2 * MB + 8), -4), (dict(scales=3 * MB + 4), -4), (dict(y=5 * MB + 1), -4), (dict(bias=4 * MB + 1), -4),
    (dict(y=MB), -2), (dict(y=MB + 256 * 2 * 6), -2), (dict(y=2 * MB + 64), -2), (dict(y=3 * MB), -2), (dict(y=4 * MB + 2), -2),
])
def test_int4_refuses(sidon, over, code):
    lib = sidon._lib.load()
    assert _int4(lib, **over) == code
    assert lib.sidon_last_error().decode()


def test_int4_takes(sidon):
    if torch.cuda.is_available():
        pytest.skip("fake addresses")
    lib = sidon._lib.load()
    for over in (dict(), dict(bias=None), dict(ldx=512, y=MB + 512, ldy=512), dict(N=1, ldy=1), dict(K=96, group=32)):
        assert _int4(lib, **over) == -6, lib.sidon_last_error()


def test_int4_packing(sidon):
    """Every weight and scale at the place that the header gives it, the rest zeros."""
    n, k, group = 19, 160, 32
    values = torch.randint(0, 16, (n, k), dtype=torch.uint8)
    zeros = torch.randint(0, 16, (n, k // group), dtype=torch.uint8)
    for kind in (torch.float16, torch.bfloat16):
        scales = torch.rand(n, k // group).to(kind)
        packed = sidon.int4.pack_int4(values, scales, zeros)
        assert packed.words.shape == (2, 2, 64, 4) and packed.scales.shape == (2, 2, 4, 16) and packed.words.is_contiguous()
        words = packed.words.view(2, 2, 4, 16, 4).tolist()
        pairs = packed.scales.contiguous().view(kind).view(2, 2, 4, 16, 2)
        order = (0, 2, 4, 6, 1, 3, 5, 7)
        for row in range(32):
            for col in range(256):
                b, i, q, e = col // 128, col % 128 // 32, col % 32 // 8, col % 8
                nibble = (words[row // 16][b][q][row % 16][i] >> (4 * order.index(e))) & 15
                assert nibble == (int(values[row, col]) if row < n and col < k else 0)
            for g in range(8):
                s, off = pairs[row // 16, g // 4, g % 4, row % 16].tolist()
                if row < n and g < k // group:
                    assert s == float(scales[row, g])
                    assert off == int(zeros[row, g]) + (-8 if kind == torch.float16 else 128)
                else:
                    assert s == 0


def test_int4_rejects_wrong_weights(sidon):
    int4 = sidon.int4
    v, s = torch.zeros(4, 128, dtype=torch.uint8), torch.ones(4, 1, dtype=torch.float16)
    with pytest.raises(TypeError, match="uint8"):
        int4.pack_int4(v.int(), s)
    with pytest.raises(TypeError, match="float16 or bfloat16"):
        int4.pack_int4(v, s.float())
    with pytest.raises(ValueError, match="0 to 15"):
        int4.pack_int4(v + 16, s)
    with pytest.raises(ValueError, match="0 to 15"):
        int4.pack_int4(v, s, torch.full((4, 1), 16, dtype=torch.uint8))
    with pytest.raises(ValueError, match="groups of 16"):
        int4.pack_int4(v, torch.ones(4, 8, dtype=torch.float16))
    with pytest.raises(ValueError, match="zeros"):
        int4.pack_int4(v, s, torch.zeros(4, 2, dtype=torch.uint8))
    with pytest.raises(ValueError, match="scales"):
        int4.pack_int4(v, s[:3])
    w = int4.pack_int4(v, s)
    with pytest.raises(ValueError, match="HIP device"):
        int4.int4_linear(torch.zeros(1, 128, dtype=torch.float16), w)
    with pytest.raises(TypeError, match="Int4Weight"):
        int4.int4_linear(torch.zeros(1, 128, dtype=torch.float16), v)
    with pytest.raises(ValueError, match="multiple"):
        int4.quantize_int4(torch.zeros(4, 100), 64)


@pytest.mark.parametrize("zeros", [False, True])
def test_quantize(sidon, zeros):
    w = torch.randn(6, 96) * torch.tensor([1e-3, 1.0, 100.0, 0.0, 1e-30, 5.0]).view(6, 1)
    values, scales, zero = sidon.int4.quantize_int4(w, 32, zeros)
    assert values.dtype == torch.uint8 and int(values.max()) <= 15 and scales.shape == (6, 3) and (scales > 0).all()
    back = (values.float().unflatten(1, (3, 32)) - (zero.float().unsqueeze(-1) if zeros else 8)) * scales.unsqueeze(-1)
    assert ((back.flatten(1) - w).abs() <= 1.01 * scales.repeat_interleave(32, 1)).all()
    assert (back.flatten(1)[3] == 0).all()


def test_int4_weights_of_other_sizes_are_refused(sidon):
    """Built or changed by hand, as from a file: what the kernel would read past its tensors."""
    import dataclasses

    w = sidon.int4.pack_int4(torch.zeros(20, 160, dtype=torch.uint8), torch.ones(20, 5, dtype=torch.float16))
    assert dataclasses.replace(w, n=17).n == 17   # (the same tiles)
    for bad in (dict(n=33), dict(n=0), dict(k=288), dict(k=170), dict(group=64), dict(group=256), dict(words=w.words[:1]),
                dict(words=w.words.long()), dict(scales=w.scales[:, :, :2]), dict(scales=w.scales.float()),
                dict(words=w.words.transpose(0, 1).contiguous().transpose(0, 1))):
        with pytest.raises(ValueError):
            dataclasses.replace(w, **bad)
    with pytest.raises(TypeError):
        dataclasses.replace(w, dtype=torch.float32)
