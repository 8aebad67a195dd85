"""The language-model operators' refusals, before any launch (no GPU)."""

from __future__ import annotations

import ctypes

import pytest
import torch


def _norm(lib, **over):
    a = dict(x=1 << 20, ldx=64, lens=None, w=16, b=16, eps=1e-5, y=1 << 22, ldy=64, ws=16, wsb=1 << 20, B=2, T=10, C=64,
             G=4, dtype=1, act=1)
    a.update(over)
    return lib.sidon_group_norm_act(a["x"], a["ldx"], a["lens"], a["w"], a["b"], a["eps"], a["y"], a["ldy"], a["ws"],
                                    a["wsb"], a["B"], a["T"], a["C"], a["G"], a["dtype"], a["act"], None)


@pytest.mark.parametrize("over,code", [
    (dict(x=None), -1), (dict(w=None), -1), (dict(b=None), -1), (dict(y=None), -1), (dict(ws=None), -1),
    (dict(dtype=3), -2), (dict(dtype=-1), -2), (dict(act=4), -2), (dict(B=0), -2), (dict(T=0), -2), (dict(T=(1 << 30) + 1), -2), (dict(C=0), -2),
    (dict(G=0), -2), (dict(G=5), -2), (dict(C=8256, ldx=8256, ldy=8256, G=1), -2), (dict(B=65536), -2),
    (dict(wsb=0), -2), (dict(ldx=63), -3), (dict(ldy=0), -3), (dict(ldx=-64), -3), (dict(x=(1 << 20) + 1), -4),
    (dict(w=18), -4), (dict(lens=6), -4), (dict(ws=20), -4),
    (dict(y=(1 << 20) + 128), -2), (dict(y=1 << 20, ldy=128), -2),
])
def test_group_norm_refuses(sidon, over, code):
    # fake addresses, never dereferenced: validation returns before any HIP call
    lib = sidon._lib.load()
    assert _norm(lib, **over) == code
    assert lib.sidon_last_error().decode()


def test_group_norm_workspace(sidon):
    ws = sidon.conformer.group_norm_workspace
    assert ws(0, 10, 64, 4, torch.float16) == 0 and ws(1, 10, 64, 5, torch.float16) == 0
    for shape in ((1, 1, 8, 1), (3, 1463, 1024, 16), (65535, 2, 64, 64)):
        assert 0 < ws(*shape, torch.float32) <= 8 * shape[0] * shape[3] * min(128, shape[1])


@pytest.mark.parametrize("dtype,vec", [(0, 4), (1, 8), (2, 8), (0, 1), (1, 1)])
def test_group_norm_statistics_fit_their_lds(sidon, dtype, vec):
    """Every column block's units, the last and narrower one's too, whose fewer
    columns leave a workgroup of 256 threads more row lanes."""
    lib = sidon._lib.load()
    block, chunks, lds = ctypes.c_int(), ctypes.c_int(), ctypes.c_int()
    short = 0
    for c in sorted({*range(vec, 1400, vec), *range(2048, 8193, 8 * vec), 8184, 8192}):
        for groups in range(1, min(c, 700) + 1):
            if c % groups:
                continue
            assert lib.sidon_group_norm_passes(2, 1500, c, groups, dtype, vec, *map(ctypes.byref, (block, chunks, lds))) == 0
            cg = c // groups
            assert 1 <= block.value <= groups and 1 <= chunks.value <= 64 and lds.value <= 64 << 10
            last = groups - (groups - 1) // block.value * block.value
            short += last < block.value
            for n in {block.value, last}:
                assert n * cg % vec == 0
                nv = n * cg // vec
                lanes = 256 // nv if nv < 256 else 1
                # a (mean, M2) of 8 bytes per vector, or per channel where a vector lies in two groups
                assert lanes * nv * (1 if cg % vec == 0 else vec) * 8 <= lds.value, (c, groups, n)
    assert short > 100
    assert lib.sidon_group_norm_passes(2, 10, 64, 5, dtype, vec, *map(ctypes.byref, (block, chunks, lds))) == -2
    assert lib.sidon_group_norm_passes(2, 10, 64, 4, dtype, 3, *map(ctypes.byref, (block, chunks, lds))) == -2
    assert lib.sidon_group_norm_passes(2, 10, 64, 4, dtype, vec, None, None, None) == -1


def test_group_norm_rejects_host_tensors(sidon):
    x = torch.zeros(4, 8)
    with pytest.raises(ValueError, match="HIP device"):
        sidon.conformer.group_norm_act(x, 1, 2, torch.ones(8), torch.zeros(8))


def _attention(lib, **over):
    i64 = ctypes.c_int64
    a = dict(q=16, k=16, v=16, lam=16, lam_heads=1, eps=1e-5, lens=None, norm_w=16, out=16, ws=None, wsb=0, B=2, H=4, Hk=2, L=10,
             S=100, D=64, causal=0, dtype=1, qs=(512, 128, 64, 1024), ks=(8192, 128, 64, 256), vs=(8192, 128, 256),
             os=(8192, 128, 512))
    a.update(over)
    st = [None if a[n] is None else (i64 * len(a[n]))(*a[n]) for n in ("qs", "ks", "vs", "os")]
    return lib.sidon_diff_attention(a["q"], a["k"], a["v"], a["lam"], a["lam_heads"], 0.5, a["lens"], a["norm_w"], a["eps"],
                                    a["out"], a["ws"], a["wsb"], a["B"], a["H"], a["Hk"], a["L"], a["S"], a["D"],
                                    a["causal"], a["dtype"], *st, None)


@pytest.mark.parametrize("over,code", [
    (dict(q=None), -1), (dict(k=None), -1), (dict(v=None), -1), (dict(lam=None), -1), (dict(out=None), -1),
    (dict(qs=None), -1), (dict(os=None), -1), (dict(dtype=0), -2), (dict(dtype=3), -2), (dict(B=0), -2), (dict(L=0), -2),
    (dict(S=0), -2), (dict(H=5), -2), (dict(Hk=0), -2), (dict(D=32), -2), (dict(D=96), -2), (dict(S=(1 << 30) + 1), -2),
    (dict(L=1 << 24), -2), (dict(lam_heads=2), -2), (dict(qs=(512, 128, 60, 1024)), -3), (dict(ks=(-8, 0, 0, 0)), -3),
    (dict(ks=(8192, 128, 64, 1 << 25)), -3), (dict(vs=(8192, 128, 1 << 25)), -3), (dict(vs=(8192, 4, 256)), -3),
    (dict(os=(1 << 41, 128, 512)), -3), (dict(q=24), -4), (dict(v=8), -4), (dict(out=8), -4), (dict(norm_w=20), -4),
    (dict(lam=18), -4), (dict(lens=6), -4), (dict(ws=24, wsb=1 << 20), -4),
])
def test_diff_attention_refuses(sidon, over, code):
    lib = sidon._lib.load()
    assert _attention(lib, **over) == code
    assert lib.sidon_last_error().decode()


@pytest.mark.parametrize("over,code", [
    (dict(os=(8192, 128, 0)), -3), (dict(os=(0, 128, 512)), -3), (dict(os=(8192, 64, 512)), -3),
    (dict(os=(8192, 128, 504)), -3), (dict(os=(2048, 128, 512)), -3), (dict(os=(128, 256, 64)), -3),
    (dict(out=1 << 30), -2), (dict(out=(1 << 30) + 2 * (512 + 3 * 128 + 9 * 1024)), -2), (dict(out=(1 << 31) + 4096), -2),
    (dict(out=(1 << 32) - 4096), -2), (dict(eps=0.0), -2), (dict(eps=-1e-5), -2), (dict(eps=float("nan")), -2),
    (dict(ks=(1 << 40, 1 << 40, 1 << 40, 0), L=1, Hk=4, B=1 << 22), -3),
])
def test_diff_attention_refuses_overlaps(sidon, over, code):
    """Rows of out that share memory, out across an input, and a norm without eps."""
    lib = sidon._lib.load()
    assert _attention(lib, **{**dict(q=1 << 30, k=1 << 31, v=1 << 32, out=1 << 33), **over}) == code
    assert lib.sidon_last_error().decode()


def test_diff_attention_workspace(sidon):
    lib = sidon._lib.load()
    ws = lib.sidon_diff_attention_workspace_bytes
    assert ws(1, 8, 3, 1, 100, 64) == 0 and ws(1, 8, 8, 4800, 4800, 64) == 0
    one = ws(1, 8, 8, 1, 4800, 64)   # split over the chip
    assert one % (8 * (16 + 64 * 16)) == 0 and 1 < one // (8 * (16 + 64 * 16)) <= 64


def test_diff_attention_rejects_wrong_tensors(sidon):
    call = sidon.diff_attention.diff_attention
    q = torch.zeros(1, 2, 2, 3, 64, dtype=torch.float16)
    k, v = torch.zeros(1, 1, 2, 5, 64, dtype=torch.float16), torch.zeros(1, 1, 5, 128, dtype=torch.float16)
    lam = torch.zeros(4, 64)
    with pytest.raises(ValueError, match="HIP device"):
        call(q, k, v, lam, 0.5)
    with pytest.raises(ValueError, match="belong together"):
        call(q, k, v[..., :64], lam, 0.5)
    with pytest.raises(ValueError, match="share"):
        call(q, torch.zeros(1, 3, 2, 5, 64, dtype=torch.float16), torch.zeros(1, 3, 5, 128, dtype=torch.float16), lam, 0.5)
    with pytest.raises(ValueError, match="H, 2, L"):
        call(q[..., :32], k[..., :32], v[..., :64], lam[:, :32], 0.5)
    with pytest.raises(TypeError, match="float16"):
        call(q.float(), k.float(), v.float(), lam, 0.5)
    with pytest.raises(ValueError, match="empty"):
        call(q[:, :, :, :0], k, v, lam, 0.5)


def _adapter(lib, residual, **over):
    mb = 1 << 20
    a = dict(x=16 * mb, ldx=128, w=32 * mb, ldw=128, bias=48 * mb, a=64 * mb, b=80 * mb, scale=16, ids=16, y=96 * mb,
             ldy=256, add=112 * mb, ldadd=256, ws=128 * mb, wsb=mb, M=12, N=256, K=128, R=16, adapters=3, items=4, act=0,
             dtype=1)
    a.update(over)
    if residual:
        return lib.sidon_adapter_residual(*[a[n] for n in (
            "x", "ldx", "w", "ldw", "a", "b", "scale", "ids", "add", "ldadd", "y", "ldy", "ws", "wsb", "M", "N", "K", "R",
            "adapters", "items", "dtype")], None)
    return lib.sidon_adapter_linear(*[a[n] for n in (
        "x", "ldx", "w", "ldw", "bias", "a", "b", "scale", "ids", "y", "ldy", "ws", "wsb", "M", "N", "K", "R", "adapters",
        "items", "act", "dtype")], None)


@pytest.mark.parametrize("over,code", [
    (dict(x=None), -1), (dict(w=None), -1), (dict(a=None), -1), (dict(b=None), -1), (dict(scale=None), -1),
    (dict(ids=None), -1), (dict(y=None), -1), (dict(ws=None), -1), (dict(M=0), -2), (dict(N=32), -2), (dict(N=250), -2),
    (dict(K=96), -2), (dict(R=0), -2), (dict(R=12), -2), (dict(R=136), -2), (dict(adapters=0), -2), (dict(items=0), -2),
    (dict(items=5), -2), (dict(dtype=0), -2), (dict(wsb=100), -2), (dict(ldx=120), -3), (dict(ldw=132), -3),
    (dict(ldy=255), -3), (dict(ldx=1 << 30), -2), (dict(x=8), -4), (dict(a=8), -4), (dict(ids=2), -4),
    (dict(y=16 * (1 << 20)), -2), (dict(y=32 * (1 << 20) + 64), -2), (dict(y=80 * (1 << 20)), -2),
    (dict(y=128 * (1 << 20)), -2),
])
@pytest.mark.parametrize("residual", [False, True])
def test_adapter_calls_refuse(sidon, residual, over, code):
    lib = sidon._lib.load()
    assert _adapter(lib, residual, **over) == code
    assert lib.sidon_last_error().decode()


def test_adapter_calls_refuse_their_own(sidon):
    lib = sidon._lib.load()
    assert _adapter(lib, False, act=2) == -2 and _adapter(lib, False, bias=12) == -4
    assert _adapter(lib, True, add=None) == -1 and _adapter(lib, True, ldadd=250) == -3
    assert _adapter(lib, True, add=96 * (1 << 20), ldadd=260) == -2   # the same memory, other rows


def test_column_blocks_of_one_tensor(sidon):
    """Rows side by side in a wider tensor are apart, a column of both is not:
    here the call gets as far as asking for a device (-6) or is refused (-2)."""
    lib = sidon._lib.load()
    mb = 1 << 20
    wide = dict(ldx=512, ldy=512)   # x 128 columns, y 256, of 512
    if torch.cuda.is_available():
        pytest.skip("fake addresses: only where no device would take the launch")
    assert _adapter(lib, False, y=16 * mb + 2 * 128, **wide) == -6
    assert _adapter(lib, False, y=16 * mb + 2 * 256, **wide) == -6
    assert _adapter(lib, False, x=96 * mb + 2 * 256, **wide) == -6
    assert _adapter(lib, False, y=16 * mb + 2 * 120, **wide) == -2
    assert _adapter(lib, False, y=16 * mb + 2 * 264, **wide) == -2
    assert _adapter(lib, False, y=16 * mb + 2 * 128, ldx=512, ldy=520) == -2
    assert _adapter(lib, True, add=96 * mb + 4 * 256, ldadd=512, ldy=512) == -6
    assert _adapter(lib, True, add=96 * mb + 4 * 252, ldadd=512, ldy=512) == -2
    assert _norm(lib, y=(1 << 20) + 128, ldx=128, ldy=128) == -6
    assert _norm(lib, y=(1 << 20) + 126, ldx=128, ldy=128) == -2
    assert _norm(lib, x=1 << 22, ldx=128, y=(1 << 22) - 256 * 3 + 128, ldy=128) == -6


MB = 1 << 20


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("over", [
    dict(ids=96 * MB), dict(ids=96 * MB + 1024), dict(scale=96 * MB + 2048), dict(scale=96 * MB - 4),
    *[dict(ws=n * MB + 64) for n in (16, 32, 64, 80)], dict(ws=16 * MB - 16), dict(ids=128 * MB + 16),
    dict(scale=128 * MB + 4),
], ids=str)
def test_adapter_calls_refuse_overlaps(sidon, residual, over):
    """y over what other workgroups still read, ws over an input."""
    lib = sidon._lib.load()
    assert _adapter(lib, residual, **over) == -2
    assert "overlap" in lib.sidon_last_error().decode()


def test_workspaces_and_outputs_refuse_overlaps(sidon):
    lib = sidon._lib.load()
    assert _adapter(lib, False, ws=48 * MB) == -2 and _adapter(lib, True, ws=112 * MB) == -2
    one = dict(w=8 * MB, b=9 * MB, ws=10 * MB)
    for over in (dict(w=1 << 22), dict(b=(1 << 22) + 16), dict(lens=(1 << 22) + 4)):
        assert _norm(lib, **{**one, **over}) == -2
    two = dict(x=16 * MB, y=64 * MB, T=100000, lens=11 * MB, **one)   # two launches
    for ws in (8 * MB, 9 * MB, 11 * MB, 16 * MB + 64, 64 * MB):
        assert _norm(lib, **{**two, "ws": ws}) == -2
        assert "overlap" in lib.sidon_last_error().decode()
    apart = dict(q=1 << 30, k=1 << 31, v=1 << 32, out=1 << 33, lam=16, norm_w=4096, lens=8192)
    for over in (dict(lam=(1 << 33) + 64), dict(norm_w=(1 << 33) + 64), dict(lens=(1 << 33) + 64)):
        assert _attention(lib, **{**apart, **over}) == -2
        assert "apart" in lib.sidon_last_error().decode()
    if torch.cuda.is_available():
        return   # (fake addresses: below, only where no device would take the launch)
    # between the rows of a wider tensor, and a workspace that the call does not use
    assert _adapter(lib, False, ldy=512, ids=96 * MB + 512, scale=96 * MB + 1024 + 512) == -6
    assert _adapter(lib, False, ldx=1 << 16, ws=16 * MB + 1024) == -6
    assert _norm(lib, **two) == -6 and _norm(lib, ws=1 << 20) == -6
    assert _attention(lib, **apart) == -6


def test_adapter_workspace_and_packing(sidon):
    ws = sidon.adapters.workspace_bytes
    assert ws(100, 16) == 3200 and ws(100, 16, True) == 6400 and ws(100, 16, True, torch.bfloat16) == 9600
    assert ws(0, 16) == 0 and ws(10, 12) == 0 and ws(10, 136) == 0
    a, b = torch.ones(3, 64), torch.ones(128, 3)
    pa, pb, sc = sidon.adapters.pack_adapters([(a, b), (torch.ones(9, 64), torch.ones(128, 9))], [1.0, 0.5])
    assert tuple(pa.shape) == (2, 16, 64) and tuple(pb.shape) == (2, 128, 16) and sc.tolist() == [1.0, 0.5]
    assert pa[0].sum() == 3 * 64 and pb[0].sum() == 3 * 128
    with pytest.raises(ValueError):
        sidon.adapters.pack_adapters([(a, b), (a[:, :32], b)], [1.0, 1.0])
    with pytest.raises(ValueError):
        sidon.adapters.pack_adapters([(a, b)], [])
    with pytest.raises(ValueError):
        sidon.adapters.pack_adapters([(torch.ones(129, 64), torch.ones(8, 129))], [1.0])


def test_adapter_linear_rejects_wrong_tensors(sidon):
    x, w = torch.zeros(4, 64, dtype=torch.float16), torch.zeros(64, 64, dtype=torch.float16)
    a, b = torch.zeros(1, 8, 64, dtype=torch.float16), torch.zeros(1, 64, 8, dtype=torch.float16)
    with pytest.raises(ValueError, match="HIP device"):
        sidon.adapters.adapter_linear(x, w, None, a, b, torch.ones(1), torch.zeros(1, dtype=torch.int32))


def test_encoder_adapters_of_the_largest_rank(sidon):
    """A part that a variant leaves out takes none of the rank that its fused
    projection has."""
    packed = {"layers": [{"qkv_w": torch.zeros(192, 64), "out_w": torch.zeros(64, 64)}]}
    pair = (torch.ones(128, 64), torch.ones(64, 128))
    packed_set = sidon.encoder.pack_adapters(packed, [(1.0, [{"k_w": pair}]), (2.0, [{"out_w": pair}])])
    a, b, scale = packed_set[0]["qkv_w"]
    assert tuple(a.shape) == (2, 128, 64) and tuple(b.shape) == (2, 192, 128) and scale.tolist() == [1.0, 2.0]
    assert (a[0] == 1).all() and (b[0, 64:128] == 1).all() and b[0].sum() == 64 * 128 and not b[1].any()
    assert not packed_set[0]["out_w"][1][0].any()


def test_sizes_past_32_bits_are_refused(sidon):
    """2^32 + n must not arrive as n."""
    far = 1 << 32
    for call in (lambda: sidon.adapters.workspace_bytes(far + 100, 16),
                 lambda: sidon.conformer.group_norm_workspace(1, far + 10, 64, 4, torch.float16),
                 lambda: sidon.conformer.group_norm_workspace(1, 10, far + 64, 4, torch.float16),
                 lambda: sidon.diff_attention.workspace_bytes(1, 8, 8, 1, far + 4800, 64),
                 lambda: sidon._lib.ints(row_stride=1 << 31)):
        with pytest.raises(ValueError, match="32 bits"):
            call()
    sidon._lib.ints(row_stride=(1 << 31) - 1, other=-5)


def test_layouts_are_bounded(sidon):
    kept = sidon._lib.Layouts()
    for i in range(3 * kept.MOST + 5):
        assert kept.keep((i,), (i, "found")) == (i, "found") and kept.get((i,)) == (i, "found")
        assert len(kept) <= kept.MOST
    assert kept.get((0,)) is None
