"""CPU: the streaming-layer descriptors match the C header, bad arguments are refused before any
device call, and the 64-bit restatement agrees with plain torch."""
import ctypes
import math
import os
import shutil
import subprocess
from fractions import Fraction

import pytest
import torch

from oracle import stream_ref as R

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("cls,name", [("QkNormRopeDesc", "m3s_qk_norm_rope_desc"),
                                      ("WindowAttentionDesc", "m3s_window_attention_desc"),
                                      ("GemmBlockDesc", "m3s_gemm_block_desc")])
def test_descriptor_layout_matches_header(tmp_path, cls, name):
    from monst3r_slam_amd import _lib
    if shutil.which("gcc") is None:
        pytest.skip("no gcc")
    c = getattr(_lib, cls)
    names = [f[0] for f in c._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "monst3r_slam_amd.h"\n'
                   f'int main(void) {{ printf("%zu\\n", sizeof({name}));\n' +
                   "".join(f'printf("%zu\\n", offsetof({name}, {n}));\n' for n in names) +
                   "return 0; }\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)],
                   check=True)
    out = [int(v) for v in subprocess.run([str(exe)], check=True, capture_output=True,
                                          text=True).stdout.split()]
    assert out[0] == ctypes.sizeof(c) and out[1:] == [getattr(c, n).offset for n in names]


P = 1 << 20   # a 16-byte aligned address that nothing reads: every call below is refused


def _norm(**kw):
    from monst3r_slam_amd import _lib
    d = _lib.QkNormRopeDesc()
    base = dict(q=P, ld_q=256, stride_q=1024, k=P, ld_k=128, stride_k=512, q_out=P, ld_qo=256,
                stride_qo=1024, k_out=P, ld_ko=128, stride_ko=512, pos=P, stride_pos=4, batch=1,
                rows=4, cache_rows=4, heads_q=4, heads_kv=2, head_dim=64, axes=1, eps=1e-6,
                base=100.0)
    for n, v in {**base, **kw}.items():
        setattr(d, n, v)
    return _lib.load().m3s_vit_qk_norm_rope(ctypes.byref(d), None)


@pytest.mark.parametrize("kw", [
    dict(q=0), dict(q=P + 8), dict(k=0), dict(k_out=0), dict(q_out=0), dict(pos=0), dict(ld_q=252),
    dict(ld_q=248), dict(stride_q=1020), dict(ld_k=64), dict(head_dim=96), dict(axes=3),
    dict(axes=0), dict(dtype=1), dict(dtype=7), dict(batch=-1), dict(rows=-1), dict(heads_q=-1),
    dict(cache_rows=3), dict(cache_rows=-1, kv_row=P), dict(v=P), dict(eps=-1.0), dict(base=0.0),
    dict(base=math.inf), dict(eps=math.nan), dict(stride_pos=-1)])
def test_norm_rope_refuses(kw):
    assert _norm(**kw) == -1


def _attn(**kw):
    from monst3r_slam_amd import _lib
    d = _lib.WindowAttentionDesc()
    base = dict(q=P, ld_q=256, stride_q=1024, k=P, ld_k=128, stride_k=512, v=P, ld_v=128,
                stride_v=512, o=P, ld_o=256, stride_o=1024, window=1, sinks=0, frame=1, batch=1,
                rows=4, cache_rows=4, heads_q=4, heads_kv=2, head_dim=64, scale=0.125)
    for n, v in {**base, **kw}.items():
        setattr(d, n, v)
    return _lib.load().m3s_vit_window_attention(ctypes.byref(d), None)


@pytest.mark.parametrize("kw", [
    dict(q=0), dict(o=0), dict(k=0), dict(v=0), dict(q=P + 2), dict(k=P + 8), dict(o=P + 4),
    dict(ld_q=250), dict(ld_q=128), dict(ld_k=120), dict(ld_v=64), dict(ld_o=254), dict(window=-1),
    dict(sinks=-1), dict(frame=0), dict(heads_kv=3), dict(heads_kv=0), dict(heads_q=0),
    dict(head_dim=32), dict(dtype=1), dict(batch=-1), dict(rows=-1), dict(cache_rows=-1),
    dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan), dict(scale=math.inf)])
def test_window_attention_refuses(kw):
    assert _attn(**kw) == -1


def test_window_attention_too_large():
    assert _attn(rows=1 << 30, heads_q=4) == -3
    assert _attn(ld_k=1 << 23) == -3
    assert _attn(cache_rows=0x7fffffff) == -3
    assert _attn(heads_q=1 << 16, heads_kv=1 << 16, ld_q=1 << 22, ld_k=1 << 22, ld_v=1 << 22,
                 ld_o=1 << 22) == -3
    assert _attn(batch=1 << 27, rows=128, heads_q=2) == -3     # more threads than a launch has


def test_norm_rope_too_large():
    assert _norm(batch=1 << 13, rows=1 << 13, cache_rows=1 << 13) == -3
    assert _norm(heads_q=1 << 16, ld_q=1 << 23, ld_qo=1 << 23) == -3


def test_block_scaled_too_large():
    from monst3r_slam_amd import _lib
    lib = _lib.load()
    big = 1 << 28
    assert lib.m3s_vit_quant_block(P, 0, 256, P, 256, P, big, big, 256, 0, None) == -3
    for kw in (dict(M=0x7fffffff, ld_sa=0x7fffffff), dict(N=0x7fffffff, ldc=0x7fffffff),
               dict(lda=1 << 23)):
        d = _lib.GemmBlockDesc(**{**dict(A=P, lda=256, scale_a=P, ld_sa=8, B=P, ldb=256,
                                         scale_b=P, ld_sb=2, C=P, ldc=100, M=8, N=100, K=256),
                                  **kw})
        assert lib.m3s_vit_gemm_block(ctypes.byref(d), None) == -3, kw


def test_window_attention_workspace():
    """Few query rows over a long cache ask for scratch, a large batch for none."""
    from monst3r_slam_amd import _lib
    d = _lib.WindowAttentionDesc(batch=1, rows=1, cache_rows=1 << 16, heads_q=8, heads_kv=2,
                                 head_dim=128, frame=1)
    f = _lib.load().m3s_vit_window_attention_workspace_bytes
    assert f(ctypes.byref(d)) > 0
    d.batch, d.rows, d.cache_rows = 8, 8192, 8192
    assert f(ctypes.byref(d)) == 0
    d.heads_kv = 3
    assert f(ctypes.byref(d)) == 0 and f(None) == 0


def test_quant_block_refuses():
    from monst3r_slam_amd import _lib
    f = _lib.load().m3s_vit_quant_block
    ok = [P, 0, 256, P, 256, P, 8, 8, 256, 0, None]
    for i, v in ((0, 0), (0, P + 8), (1, 3), (2, 248), (2, 252), (3, 0), (3, P + 4), (4, 248),
                 (5, 0), (5, P + 2), (6, 7), (7, -1), (8, 250), (8, -16)):
        a = list(ok)
        a[i] = v
        assert f(*a) == -1, (i, v)
    assert f(None, 0, 0, None, 0, None, 0, 0, 256, 0, None) == 0


def test_gemm_block_refuses():
    from monst3r_slam_amd import _lib
    base = dict(A=P, lda=256, scale_a=P, ld_sa=8, B=P, ldb=256, scale_b=P, ld_sb=2, C=P, ldc=100,
                M=8, N=100, K=256, out_type=0)
    for kw in (dict(A=0), dict(B=0), dict(C=0), dict(scale_a=0), dict(scale_b=0), dict(A=P + 8),
               dict(lda=240), dict(lda=264), dict(ldb=240), dict(ldc=99), dict(ld_sa=7),
               dict(ld_sb=1), dict(K=250), dict(K=0), dict(M=-1), dict(N=-1), dict(out_type=3),
               dict(C=P + 1), dict(R=P, ldr=99), dict(bias=P + 2)):
        d = _lib.GemmBlockDesc()
        for n, v in {**base, **kw}.items():
            setattr(d, n, v)
        assert _lib.load().m3s_vit_gemm_block(ctypes.byref(d), None) == -1, kw
    assert _lib.load().m3s_vit_gemm_block(None, None) == -1


def test_ops_refuse_cpu_tensors():
    from monst3r_slam_amd.model import Ops
    ops = Ops(torch.device("cuda", 0))
    z = torch.zeros
    q = z(1, 4, 4, 64, dtype=torch.bfloat16)
    for call in (lambda: ops.qk_norm_rope(q, q, z(4, 1, dtype=torch.int64), q, q),
                 lambda: ops.window_attn(q, q, q, q, 1),
                 lambda: ops.quant_block(z(4, 128), z(4, 128, dtype=torch.uint8), z(1, 4)),
                 lambda: ops.gemm_block(z(4, 128, dtype=torch.uint8), z(1, 4),
                                        z(4, 128, dtype=torch.uint8), z(1, 1), z(4, 4))):
        with pytest.raises(RuntimeError, match="GPU"):
            call()


@pytest.mark.parametrize("N,K", [(1, 16), (130, 272), (256, 128)])
def test_quant_e4m3_block(N, K):
    from monst3r_slam_amd.model import quant_e4m3_block
    g = torch.Generator().manual_seed(0)
    w = torch.randn(N, K, generator=g) * torch.exp(torch.randn(N, 1, generator=g))
    q, s = quant_e4m3_block(w)
    assert q.shape == (N, K) and s.shape == (-(-N // 128), -(-K // 128))
    sc = s.repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]
    back = q.view(torch.float8_e4m3fn).float() * sc
    # half a step of e4m3 (2^-4), or half its smallest step (2^-10) at the block's scale, and
    # the 32-bit roundings of the quotient and the product
    assert ((back - w).abs() <= 2.0 ** -4 * w.abs() * (1 + 2.0 ** -20) + 2.0 ** -10 * sc).all()


def test_restatement_against_torch():
    """The 64-bit window attention against torch's own softmax under the same mask."""
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(1, n, 2, 64, generator=g) for n in (9, 30, 30))
    got, _ = R.window_attn(q, k, v, torch.zeros_like(q), 6, 2, 1, None, None, 0.125)
    i, j = torch.arange(9)[:, None] + 21, torch.arange(30)[None]
    see = (j <= i) & ((j > i - 6) | (j < 2))
    x = torch.einsum("bihd,bjhd->bhij", q.double(), k.double()) * 0.125
    p = torch.softmax(x.masked_fill(~see, -math.inf), -1)
    assert torch.allclose(got, torch.einsum("bhij,bjhd->bihd", p, v.double()))
    assert not R.visible(4, 2, 5, 3, 2, 1)[:2].any()   # queries in front of the first key


def test_descriptor_pack():
    """pack() lays the values out as the ctypes fields do; what does not fit is refused."""
    from monst3r_slam_amd import _lib
    for c in (_lib.QkNormRopeDesc, _lib.WindowAttentionDesc, _lib.GemmBlockDesc):
        vals = [i + 1.0 if t is ctypes.c_float else (i << 33 if t in (ctypes.c_void_p,
                ctypes.c_int64) else i + 1) for i, (_, t) in enumerate(c._fields_)]
        d = c.from_buffer_copy(c.pack(*vals))
        assert [getattr(d, n) or 0 for n, _ in c._fields_] == vals
        big = list(vals)
        big[[t for _, t in c._fields_].index(ctypes.c_int32)] = 1 << 31
        with pytest.raises(RuntimeError, match="out of range"):
            c.pack(*big)


def test_angles():
    """f64's own angles where f64 is exact enough, in [-pi, pi]; one that cancels to 6e-5 (710
    is nearly 113 turns) keeps its digits."""
    pos = torch.tensor([[0], [1], [-7], [3000], [1 << 20]])
    t = R.angles(pos, 16, 100.0)
    f = pos.double()[..., None] * torch.tensor([100.0 ** (-i / 16) for i in range(16)],
                                               dtype=torch.float64)
    # a product and a table entry rounded to 53 bits each, and the reduction's own
    assert ((t.cos() - f.cos()).abs() <= 2.0 ** -51 * f.abs().clamp_min(1)).all()
    assert ((t.sin() - f.sin()).abs() <= 2.0 ** -51 * f.abs().clamp_min(1)).all()
    assert (t.abs() <= math.pi).all()
    # math.sin(math.pi) is what math.pi lacks of pi
    left = 710 - 226 * (Fraction(math.pi) + Fraction(math.sin(math.pi)))
    assert abs(float(R.angles(torch.tensor([710]), 1, 1.0)) - float(left)) < 1e-18


@pytest.mark.parametrize("K", [272, 1024, 4096])
def test_gemm_block_rms_tells_short_sums(K):
    """The bound on the product's rms error holds for the matrix instruction's cut octets and
    fails for a sum over the groups that is rounded to 14 bits."""
    g = torch.Generator().manual_seed(K)
    M, N, G = 24, 48, -(-K // 128)
    a, b = ((90 * torch.randn(r, K, generator=g)).clamp(-448, 448).to(torch.float8_e4m3fn)
            for r in (M, N))
    sa = torch.exp(torch.randn(G, M, generator=g)) / 90
    sb = torch.exp(torch.randn(1, G, generator=g)) / (90 * K ** 0.5)
    ref, tol = R.gemm_block(a, sa, b, sb, None, False, None, torch.float32)
    a, b, sa, sb = a.double(), b.double(), sa.double(), sb.double()
    cut, short = torch.zeros_like(ref), torch.zeros_like(ref)
    for i in range(G):
        k = slice(128 * i, 128 * i + 128)
        f = sa[i][:, None] * sb[0, i]
        cut += R.cut_octets(a[:, k], b[:, k]) * f
        m, e = torch.frexp(short + a[:, k] @ b[:, k].t() * f)
        short = torch.ldexp(torch.round(m * 2.0 ** 14) * 2.0 ** -14, e)
    rms = lambda x: float(x.square().mean().sqrt() / ref.square().mean().sqrt())  # noqa: E731
    assert ((cut - ref).abs() <= tol).all()
    assert rms(cut - ref) < R.GEMM_BLOCK_RMS < rms(short - ref)


def test_ops_follow_the_current_device(monkeypatch):
    """A device without an index is the one that is current at the call, not at the first one."""
    from monst3r_slam_amd.model import Ops
    ops = Ops(torch.device("cuda"))
    x, q, s = torch.zeros(4, 128), torch.zeros(4, 128, dtype=torch.uint8), torch.zeros(1, 4)
    for i in (0, 1):
        monkeypatch.setattr(torch.cuda, "current_device", lambda: i)
        with pytest.raises(RuntimeError, match=f"cuda:{i} "):
            ops.quant_block(x, q, s)


def test_zero_sizes():
    """What the header calls no work is, and what it refuses is refused."""
    from monst3r_slam_amd import _lib
    lib = _lib.load()
    for kw in (dict(batch=0), dict(rows=0), dict(heads_q=0, heads_kv=0)):
        assert _norm(**kw) == 0, kw
    for kw in (dict(batch=0), dict(rows=0)):
        assert _attn(**kw) == 0, kw
    for m, k in ((0, 256), (8, 0)):
        assert lib.m3s_vit_quant_block(P, 0, 256, P, 256, P, 8, m, k, 0, None) == 0
    base = dict(A=P, lda=256, scale_a=P, ld_sa=8, B=P, ldb=256, scale_b=P, ld_sb=2, C=P, ldc=100,
                M=8, N=100, K=256)
    for kw, want in ((dict(M=0), 0), (dict(N=0), 0), (dict(K=0), -1), (dict(K=0, M=0), -1)):
        d = _lib.GemmBlockDesc(**{**base, **kw})
        assert lib.m3s_vit_gemm_block(ctypes.byref(d), None) == want, kw
