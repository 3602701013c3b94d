"""GPU numerics of the streaming-layer operators (per-head norm + rotation, windowed attention,
block-scaled e4m3) against the 64-bit restatement (oracle/stream_ref.py) and its derived bounds."""
import math

import pytest
import torch

from oracle import stream_ref as R

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module")
def ops(dev):
    from monst3r_slam_amd.model import Ops
    return Ops(dev)


def _gen(dev, seed):
    g = torch.Generator(device=dev).manual_seed(seed)
    return lambda *s: torch.randn(*s, device=dev, generator=g)


def _within(got, ref, tol, what=""):
    err = (got.to(torch.float64) - ref).abs()
    bad = ~(err <= tol)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} off, worst "
                           f"{float((err - tol)[bad].max())} over {float(tol[bad].max())}")


# ---- norm + rotation -----------------------------------------------------------------------

def _norm_tol(ref, amp, dtype):
    # 32-bit norm: sums of 128 terms by halving, a root, a quotient, the products (< 32
    # roundings of numbers up to amp), cos / sin to 2^-22; one rounding to dtype
    return R.half_step(dtype) * ref.abs() + 2.0 ** -18 * amp


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("D,axes", [(64, 1), (64, 2), (128, 1), (128, 2)])
@pytest.mark.parametrize("B,S,hq,hk,layer", [(1, 1, 1, 1, False), (3, 7, 5, 1, True),
                                             (2, 700, 4, 2, False)])
def test_norm_rope(ops, dev, dtype, D, axes, B, S, hq, hk, layer):
    rand = _gen(dev, B * S + D)
    qkv = (rand(B, S, hq + 2 * hk, D) * 2 + 0.5).to(dtype)   # views of one projection
    q, k, v = qkv[:, :, :hq], qkv[:, :, hq:hq + hk], qkv[:, :, hq + hk:]
    w = [1 + 0.3 * rand(D), 0.2 * rand(D), 1 + 0.3 * rand(D), 0.2 * rand(D)]
    pos = torch.randint(0, 3000, (B, S, axes), device=dev)
    q_out = torch.empty(B, S, hq, D, dtype=dtype, device=dev)
    k_out, v_out = (torch.empty(B, S, hk, D, dtype=dtype, device=dev) for _ in range(2))
    ops.qk_norm_rope(q, k, pos, q_out, k_out, gamma_q=w[0], beta_q=w[1], gamma_k=w[2],
                     beta_k=w[3], layer=layer, eps=1e-5, base=10000.0, v=v, v_out=v_out)
    for got, x, g, b in ((q_out, q, w[0], w[1]), (k_out, k, w[2], w[3])):
        ref, amp = R.norm_rope(x, g, b, pos, layer, 1e-5, 10000.0)
        _within(got, ref, _norm_tol(ref, amp, dtype))
    assert torch.equal(v_out, v)


def test_norm_rope_plain_and_far_positions(ops, dev):
    """No gamma / beta, shared positions, positions up to 2^31 (angles keep their precision)."""
    rand = _gen(dev, 5)
    q, k = rand(2, 6, 3, 64).half(), rand(2, 6, 3, 64).half()
    pos = torch.tensor([0, 1, -7, 1 << 20, (1 << 24) + 1, (1 << 31) - 1], device=dev)[:, None]
    q_out, k_out = torch.empty_like(q), torch.empty_like(k)
    ops.qk_norm_rope(q, k, pos, q_out, k_out, base=10000.0)
    for got, x in ((q_out, q), (k_out, k)):
        ref, amp = R.norm_rope(x, None, None, pos.expand(2, 6, 1), False, 1e-6, 10000.0)
        # the restatement's own f64 angles are off by up to 2^31 2^-53 of a radian
        _within(got, ref, _norm_tol(ref, amp, F16))


@pytest.mark.parametrize("D,axes", [(64, 2), (128, 1)])
@pytest.mark.parametrize("base", [100.0, 10000.0])
def test_norm_rope_positions_up_to_2_40(ops, dev, D, axes, base):
    """Angles against 90 digits: off by 2^-23.7 of a half turn at most, 2.3e-7 radians, a
    sixteenth of _norm_tol's 2^-18."""
    rand = _gen(dev, D)
    far = [1 << 31, (1 << 33) + 5, (1 << 36) - 3, -(1 << 37) + 1, 987654321987, (1 << 40) - 1]
    pos = torch.tensor(far * axes, device=dev).reshape(axes, 1, 6).permute(1, 2, 0).contiguous()
    q, k = rand(1, 6, 3, D).half(), rand(1, 6, 3, D).half()
    q_out, k_out = torch.empty_like(q), torch.empty_like(k)
    ops.qk_norm_rope(q, k, pos, q_out, k_out, base=base)
    t = R.angles(pos, D // axes // 2, base)
    for got, x in ((q_out, q), (k_out, k)):
        ref, amp = R.norm_rope(x, None, None, pos, False, 1e-6, base, t)
        _within(got, ref, _norm_tol(ref, amp, F16))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("layer", [False, True])
def test_norm_rope_every_magnitude(ops, dev, D, layer):
    """bf16 heads whose squares or sums leave f32's range, up and down, beside ordinary ones."""
    rand = _gen(dev, D + layer)
    # one magnitude a token, most of them beside others in the wave's other heads
    for eps, low in ((0.0, -125), (1e-5, -100)):
        e = torch.arange(low, 126, device=dev)
        x = rand(1, len(e), 6, D) + 0.5
        x[:, :, 1::2] *= torch.exp2(e.float())[:, None, None]
        x = x.bfloat16()
        assert torch.isfinite(x).all()
        pos = torch.randint(0, 500, (len(e), 1), device=dev)
        q_out = torch.empty_like(x)
        k_out = torch.empty_like(x[:, :, 1:2])
        ops.qk_norm_rope(x, x[:, :, 1:2], pos, q_out, k_out, layer=layer, eps=eps, base=100.0)
        ref, amp = R.norm_rope(x, None, None, pos[None], layer, eps, 100.0)
        # the restatement's eps is the call's, rounded to f32: 2^-24 of it
        _within(q_out, ref, _norm_tol(ref, amp, BF16))
        assert torch.equal(k_out, q_out[:, :, 1:2])


def test_norm_rope_in_place_and_zero_rows(ops, dev):
    rand = _gen(dev, 6)
    qk = rand(1, 33, 6, 128).bfloat16()
    qk[0, 5] = 0                                   # an all-zero row: 0, not NaN
    pos = torch.arange(33, device=dev)[:, None]
    a, b = torch.empty(1, 33, 4, 128, dtype=BF16, device=dev), torch.empty(1, 33, 2, 128,
                                                                           dtype=BF16, device=dev)
    ops.qk_norm_rope(qk[:, :, :4], qk[:, :, 4:], pos, a, b)
    ops.qk_norm_rope(qk[:, :, :4], qk[:, :, 4:], pos, qk[:, :, :4], qk[:, :, 4:])
    assert torch.equal(qk[:, :, :4], a) and torch.equal(qk[:, :, 4:], b)
    assert (a[0, 5] == 0).all() and (b[0, 5] == 0).all()


def test_norm_rope_matches_2d_rope_layout(ops, dev):
    """Head dim 64 with (y, x) positions turns the pairs that Ops.rope turns."""
    rand = _gen(dev, 7)
    q = rand(1, 12, 2, 64).bfloat16()
    pos = torch.randint(0, 40, (1, 12, 2), device=dev)
    out, k = torch.empty_like(q), q.clone()
    ops.qk_norm_rope(q, k, pos, out, k, eps=0.0, base=100.0)
    ref = (q.float() / q.float().square().mean(-1, keepdim=True).sqrt()).bfloat16()
    ops.rope(ref, 128, 12 * 128, pos, 24, 1, 12, 2, 100.0)
    # ref is rounded before the rotation as well as after it
    assert (out.float() - ref.float()).abs().max() <= 3 * 2.0 ** -8 * ref.float().abs().max()


@pytest.mark.parametrize("D", [64, 128])
def test_norm_rope_cache_rows_and_lengths(ops, dev, D):
    """Append at kv_row; rows past seq_len, cache rows outside the cache and rows in front of and
    behind the new ones stay as they were."""
    rand = _gen(dev, 8)
    B, S, hq, hk, cache = 4, 9, 4, 2, 20
    q, k, v = (rand(B, S, h, D).bfloat16() for h in (hq, hk, hk))
    pos = torch.randint(0, 100, (B, S, 1), device=dev)
    row = torch.tensor([0, 5, 15, -3], device=dev, dtype=torch.int32)
    n = torch.tensor([9, 4, 9, 9], device=dev, dtype=torch.int32)
    q_out = torch.full_like(q, 7.0)
    k_out = torch.full((B, cache + 2, hk, D), 7.0, dtype=BF16, device=dev)
    v_out = k_out.clone()
    ops.qk_norm_rope(q, k, pos, q_out, k_out[:, :cache], v=v, v_out=v_out[:, :cache], kv_row=row,
                     seq_len=n)
    full_q, full_k = torch.empty_like(q), torch.empty_like(k)
    ops.qk_norm_rope(q, k, pos, full_q, full_k)
    for b in range(B):
        m = int(n[b])
        assert torch.equal(q_out[b, :m], full_q[b, :m]) and (q_out[b, m:] == 7).all()
        want_k, want_v = torch.full_like(k_out[b], 7.0), torch.full_like(k_out[b], 7.0)
        for s in range(m):
            r = int(row[b]) + s
            if 0 <= r < cache:
                want_k[r], want_v[r] = full_k[b, s], v[b, s]
        assert torch.equal(k_out[b], want_k) and torch.equal(v_out[b], want_v)


# ---- windowed attention --------------------------------------------------------------------

def _attn_case(ops, dev, dtype, B, S, L, hq, hk, D, window, sinks, frame, q_len=None, kv_len=None,
               seed=0, spread=1.5, scale=None):
    rand = _gen(dev, seed)
    q = (spread * rand(B, S, hq, D)).to(dtype)
    k, v = rand(B, L, hk, D).to(dtype), (rand(B, L, hk, D) + 0.5).to(dtype)
    lens = [None if t is None else torch.tensor(t, device=dev, dtype=torch.int32)
            for t in (q_len, kv_len)]
    if kv_len is not None:                          # behind a sequence's end: anything
        for b, n in enumerate(kv_len):
            k[b, max(n, 0):], v[b, max(n, 0):] = math.nan, math.inf
    o = torch.full((B, S, hq, D), 9.0, dtype=dtype, device=dev)
    ops.window_attn(q, k, v, o, window, sinks=sinks, frame=frame, q_len=lens[0], kv_len=lens[1],
                    scale=scale)
    ref, tol = R.window_attn(q, k, v, torch.full_like(o, 9.0), window, sinks, frame, q_len,
                             kv_len, D ** -0.5 if scale is None else scale)
    _within(o, ref, tol, f"{dtype} {B} {S} {L}")
    return q, k, v, o


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("S,L,hq,hk,window,sinks", [
    (1, 1, 1, 1, 0, 0), (1, 65, 4, 4, 0, 0), (1, 1000, 8, 1, 100, 3), (5, 333, 6, 2, 17, 1),
    (64, 64, 2, 2, 0, 0), (130, 257, 4, 2, 64, 70), (200, 200, 8, 2, 1, 0), (77, 500, 3, 3, 40, 9),
    (33, 33, 32, 1, 5, 2)])
def test_window_attn_tokens(ops, dev, dtype, D, S, L, hq, hk, window, sinks):
    _attn_case(ops, dev, dtype, 2, S, L, hq, hk, D, window, sinks, 1, seed=S + L)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("S,L,window,sinks,frame", [
    (48, 48 * 6, 3, 48, 48), (48, 48 * 6 + 20, 2, 0, 48), (96, 400, 1, 10, 33),
    (10, 300, 2, 700, 1000), (150, 150, 4, 1, 7)])
def test_window_attn_frames(ops, dev, D, S, L, window, sinks, frame):
    _attn_case(ops, dev, BF16, 2, S, L, 4, 4, D, window, sinks, frame, seed=S + L)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("S,L,hq,hk,D", [(1, 700, 8, 2, 128), (70, 300, 4, 1, 64),
                                         (300, 600, 4, 2, 128)])
@pytest.mark.parametrize("frame", [1, 50])
def test_window_attn_ragged_lengths(ops, dev, dtype, S, L, hq, hk, D, frame):
    """Lengths of zero, one, past the end; fewer keys than queries (rows that see nothing are 0);
    padding rows and whatever lies behind a sequence's keys untouched."""
    q_len = [S, 1, 0, S, S, S + 5, max(1, S - 3)]
    kv_len = [L, 1, 5, 0, max(1, S // 2), L + 9, L // 2 + 1]
    _attn_case(ops, dev, dtype, 7, S, L, hq, hk, D, 60 if frame == 1 else 2, 4, frame, q_len,
               kv_len, seed=S)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("S,L", [(1, 9000), (3, 20011), (40, 5000), (600, 3000)])
def test_window_attn_long(ops, dev, D, S, L):
    """Key ranges split over the grid and joined; no window, and one with sinks."""
    _attn_case(ops, dev, BF16, 1, S, L, 4, 2, D, 0, 0, 1, seed=S)
    _attn_case(ops, dev, F16, 1, S, L, 4, 2, D, 2500, 130, 1, seed=S)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_window_attn_peaked_scores(ops, dev, dtype):
    """Scores of some hundreds, one-hot rows, and keys far below the maximum that add up."""
    _attn_case(ops, dev, dtype, 1, 50, 300, 2, 2, 64, 0, 0, 1, spread=40.0)
    D, L = 128, 4096
    q = torch.zeros(1, 1, 1, D, dtype=dtype, device=dev)
    k = torch.zeros(1, L, 1, D, dtype=dtype, device=dev)
    q[..., 0], k[0, 0, 0, 0] = 8.0, 1.25           # one key e^10 above 4095 equal ones
    v = torch.zeros(1, L, 1, D, dtype=dtype, device=dev)
    v[0, 1:] = 1.0
    o = torch.empty_like(q)
    ops.window_attn(q, k, v, o, 0, scale=1.0)
    ref, tol = R.window_attn(q, k, v, o, 0, 0, 1, None, None, 1.0)
    _within(o, ref, tol)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("D,S", [(64, 40), (128, 40), (64, 300), (128, 300), (128, 2)])
def test_window_attn_not_finite_where_masked(ops, dev, dtype, D, S):
    """NaN and Inf in keys and values of positions that a row does not see do not reach it; a
    value that is not finite does reach the rows that see it."""
    rand = _gen(dev, S)
    L, window, sinks = S + 200, 30, 5
    q, k, v = (rand(1, n, 2, D).to(dtype) for n in (S, L, L))
    k[0, 5:L - S - window], v[0, 5:L - S - window] = math.nan, math.inf   # in front of the window
    j = L - S // 2 - 1                                                    # seen by some rows only
    v[0, j, 0, 3], v[0, j, 1, 7], v[0, j, 1, 40] = math.inf, -math.inf, math.nan
    o = torch.empty_like(q)
    ops.window_attn(q, k, v, o, window, sinks=sinks)
    ref, tol = R.window_attn(q, k, v, o, window, sinks, 1, None, None, D ** -0.5)
    assert torch.equal(torch.isfinite(o), torch.isfinite(ref))
    fin = torch.isfinite(ref)
    assert torch.equal(torch.nan_to_num(o.double(), 5.0, 3e300, -3e300)[~fin],
                       torch.nan_to_num(ref, 5.0, 3e300, -3e300)[~fin])
    _within(torch.where(fin, o.double(), 0), torch.where(fin, ref, 0), tol)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("frame", [1, 90])
def test_window_attn_many_blocks(ops, dev, dtype, D, frame):
    """Grids of more than 256 blocks of 128 rows take blocks without key splits."""
    _attn_case(ops, dev, dtype, 4, 700, 900, 16, 8, D, 60 if frame == 1 else 2, 4, frame,
               [700, 1, 0, 699], [900, 5, 7, 650], seed=frame)
    _attn_case(ops, dev, dtype, 5, 400, 400, 32, 16, D, 0, 0, 1, seed=frame + 1)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("frame", [1, 70])
def test_window_attn_middle_grids(ops, dev, dtype, D, frame):
    """More than 256 tiles of 32 rows, up to 256 of 128: several row waves and key splits a block;
    long keys split over the grid too."""
    _attn_case(ops, dev, dtype, 4, 320, 500, 16, 8, D, 60 if frame == 1 else 2, 4, frame,
               [320, 1, 0, 319], [500, 5, 7, 350], seed=frame)
    _attn_case(ops, dev, dtype, 1, 2100, 2300, 4, 4, D, 0, 0, frame, seed=frame + 1)
    _attn_case(ops, dev, dtype, 1, 2100, 2300, 4, 4, D, 0 if frame == 1 else 30, 9, frame,
               seed=frame + 2)


@pytest.mark.parametrize("D", [64, 128])
def test_window_attn_middle_grids_not_finite_where_masked(ops, dev, D):
    rand = _gen(dev, D + 1)
    S, L, h, window = 300, 500, 40, 30
    q, k, v = (rand(1, n, h, D).bfloat16() for n in (S, L, L))
    k[0, 5:L - S - window], v[0, 5:L - S - window] = math.nan, math.inf   # in front of the window
    j = L - S // 2 - 1                                                    # seen by some rows only
    v[0, j, 0, 3], v[0, j, 1, 7], v[0, j, 39, 40] = math.inf, -math.inf, math.nan
    o = torch.empty_like(q)
    ops.window_attn(q, k, v, o, window, sinks=5)
    ref, tol = R.window_attn(q, k, v, o, window, 5, 1, None, None, D ** -0.5)
    fin = torch.isfinite(ref)
    assert torch.equal(torch.isfinite(o), fin) and not fin.all()
    _within(torch.where(fin, o.double(), 0), torch.where(fin, ref, 0), tol)


@pytest.mark.parametrize("D", [64, 128])
def test_window_attn_many_blocks_not_finite_where_masked(ops, dev, D):
    rand = _gen(dev, D)
    S, L, h, window = 500, 700, 70, 30
    q, k, v = (rand(1, n, h, D).bfloat16() for n in (S, L, L))
    k[0, 5:L - S - window], v[0, 5:L - S - window] = math.nan, math.inf   # in front of the window
    j = L - S // 2 - 1                                                    # seen by some rows only
    v[0, j, 0, 3], v[0, j, 1, 7], v[0, j, 69, 40] = math.inf, -math.inf, math.nan
    o = torch.empty_like(q)
    ops.window_attn(q, k, v, o, window, sinks=5)
    ref, tol = R.window_attn(q, k, v, o, window, 5, 1, None, None, D ** -0.5)
    fin = torch.isfinite(ref)
    assert torch.equal(torch.isfinite(o), fin) and not fin.all()
    _within(torch.where(fin, o.double(), 0), torch.where(fin, ref, 0), tol)


@pytest.mark.parametrize("S,D", [(1, 128), (40, 64)])
def test_window_attn_without_workspace(ops, dev, S, D):
    """The C entry without scratch walks all keys in one block: slower, the same bound."""
    from monst3r_slam_amd import _lib
    rand = _gen(dev, 13)
    q, k, v = (rand(1, n, 4, D).bfloat16() for n in (S, 3000, 3000))
    o = torch.empty_like(q)
    d = _lib.WindowAttentionDesc(
        **{n: t.data_ptr() for n, t in dict(q=q, k=k, v=v, o=o).items()},
        **{"ld_" + n: 4 * D for n in "qkvo"}, frame=1, batch=1, rows=S, cache_rows=3000,
        heads_q=4, heads_kv=4, head_dim=D, scale=D ** -0.5)
    d = bytes(d)
    assert ops.lib.m3s_vit_window_attention_workspace_bytes(d) > 0
    assert ops.lib.m3s_vit_window_attention(d, _lib.raw_stream(0)) == 0
    ref, tol = R.window_attn(q, k, v, o, 0, 0, 1, None, None, D ** -0.5)
    _within(o, ref, tol)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B,S,L,hq,hk", [(2, 3, 900, 8, 2), (4, 320, 500, 16, 8),
                                         (4, 700, 900, 16, 8)])
def test_window_attn_not_finite_queries(ops, dev, D, B, S, L, hq, hk):
    """NaN and Inf in a query make its own row and head NaN and leave its neighbours, which share
    its tiles, as they are."""
    rand = _gen(dev, S + D)
    q, k, v = (rand(B, *n, D).bfloat16() for n in ((S, hq), (L, hk), (L, hk)))
    want, got = torch.empty_like(q), torch.empty_like(q)
    ops.window_attn(q, k, v, want, 600, sinks=70)
    bad = torch.zeros(B, S, hq, dtype=torch.bool, device=dev)
    for b, s, h, x in ((0, 0, 0, math.nan), (1, S - 1, hq - 1, math.inf), (1, S // 2, 3, math.nan)):
        q[b, s, h, 5], bad[b, s, h] = x, True
    ops.window_attn(q, k, v, got, 600, sinks=70)
    assert torch.isnan(got[bad]).all()
    assert torch.equal(got[~bad], want[~bad])


@pytest.mark.parametrize("D", [64, 128])
def test_norm_rope_not_finite(ops, dev, D):
    """NaN and Inf stay in their own head."""
    rand = _gen(dev, D)
    q, k = rand(2, 9, 5, D).bfloat16(), rand(2, 9, 20, D).bfloat16()
    pos = torch.arange(9, device=dev)[:, None]
    want, got = [[torch.empty_like(t) for t in (q, k)] for _ in range(2)]
    ops.qk_norm_rope(q, k, pos, *want)
    q[0, 3, 4, 7], q[1, 0, 0, D - 1], k[1, 8, 19, 0] = math.nan, math.inf, -math.inf
    ops.qk_norm_rope(q, k, pos, *got)
    for x, w, g in ((q, want[0], got[0]), (k, want[1], got[1])):
        bad = ~torch.isfinite(x).all(-1)
        assert bad.any() and (~torch.isfinite(g[bad])).any(-1).all()
        assert torch.equal(g[~bad], w[~bad])


def test_window_attn_infinite_scores(ops, dev):
    """Scores of -inf for every key a row sees: 0, as for a row that sees none; one finite key
    among them takes all the weight."""
    q = torch.ones(1, 2, 1, 64, dtype=F16, device=dev)
    k = torch.full((1, 70, 1, 64), -math.inf, dtype=F16, device=dev)
    v, o = torch.ones_like(k), torch.empty_like(q)
    ops.window_attn(q, k, v, o, 0)
    assert (o == 0).all()
    k[0, 69], v[0, 69] = 0.5, 3.0
    ops.window_attn(q, k, v, o, 0)
    assert (o[0, 0] == 0).all() and (o[0, 1] == 3).all()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B,S,L,hq,hk", [(4, 1, 9000, 8, 2), (1, 40, 5000, 4, 2),
                                         (1, 2100, 2300, 4, 4), (4, 700, 900, 16, 8),
                                         (2, 1001, 3, 12, 4)])
def test_window_attn_in_place(ops, dev, D, B, S, L, hq, hk):
    """o may be q itself: a block's rows are read before any of them is written, also where they
    see nothing (1,001 queries over 3 keys) and where rows past a length stay queries."""
    rand = _gen(dev, S + D)
    q, k, v = (rand(B, *n, D).bfloat16() for n in ((S, hq), (L, hk), (L, hk)))
    n = torch.tensor([S - S // 3 * (b % 2) for b in range(B)], device=dev, dtype=torch.int32)
    want = q.clone()
    ops.window_attn(q, k, v, want, 600, sinks=70, q_len=n)
    ops.window_attn(q, k, v, q, 600, sinks=70, q_len=n)
    assert torch.equal(q, want)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B,S,L,hq,hk", [(4, 1, 9000, 8, 2), (1, 40, 5000, 4, 2),
                                         (1, 2100, 2300, 4, 4), (4, 700, 900, 16, 8)])
def test_window_attn_repeats_exactly(ops, dev, D, B, S, L, hq, hk):
    """The same call gives the same bits on every launch shape, split over the grid or not, with
    other work on the card."""
    rand = _gen(dev, S + D)
    q, k, v = (rand(B, *n, D).bfloat16() for n in ((S, hq), (L, hk), (L, hk)))
    outs = [torch.empty_like(q) for _ in range(6)]
    side, x = torch.cuda.Stream(dev), rand(1024, 1024)
    torch.cuda.synchronize(dev)
    for o in outs:
        with torch.cuda.stream(side):
            _ = x @ x
        ops.window_attn(q, k, v, o, 600, sinks=70)
    torch.cuda.synchronize(dev)
    assert all(torch.equal(o, outs[0]) for o in outs)


def test_window_attn_strides(ops, dev):
    """Views of a fused projection, transposed batch order, a cache with wider rows."""
    rand = _gen(dev, 11)
    B, S, h, D = 2, 100, 4, 64
    qkv = rand(B, S, 3 * h, D).bfloat16()
    q, k, v = qkv[:, :, :h], qkv[:, :, h:2 * h], qkv[:, :, 2 * h:]
    wide = torch.full((S, B, h + 2, D), 3.0, dtype=BF16, device=dev)
    o = wide.transpose(0, 1)[:, :, 1:h + 1]
    ops.window_attn(q, k, v, o, 20, sinks=2)
    ref, tol = R.window_attn(q, k, v, o, 20, 2, 1, None, None, D ** -0.5)
    _within(o, ref, tol)
    assert (wide[:, :, 0] == 3).all() and (wide[:, :, h + 1] == 3).all()


def test_one_row_views(ops, dev):
    """One token of each sequence out of rows whose length suits nothing: the row stride of a
    single row is not used."""
    rand = _gen(dev, 14)
    B, h, D, L = 3, 2, 64, 40
    W = h * D + 4                                          # 132 a row, 264 a sequence
    view = lambda x: x.as_strided((B, 1, h, D), (2 * W, W, D, 1))  # noqa: E731
    wide = rand(B, 2, h * D + 4).bfloat16()
    q, out = view(wide), torch.full((B, 2, h * D + 4), 7.0, dtype=BF16, device=dev)
    k, v = rand(B, L, h, D).bfloat16(), rand(B, L, h, D).bfloat16()
    want, got = torch.empty(B, 1, h, D, dtype=BF16, device=dev), view(out)
    ops.window_attn(q.contiguous(), k, v, want, 9, sinks=2)
    ops.window_attn(q, k, v, got, 9, sinks=2)
    assert torch.equal(got, want) and (out[:, 1] == 7).all() and (out[:, 0, h * D:] == 7).all()
    pos = torch.arange(B, device=dev).reshape(B, 1, 1)
    wk, want_k = torch.empty_like(want), torch.empty_like(want)
    ops.qk_norm_rope(q.contiguous(), k[:, :1], pos, want, want_k)
    ops.qk_norm_rope(q, k[:, :1], pos, got, wk)
    assert torch.equal(got, want) and torch.equal(wk, want_k)
    assert (out[:, 1] == 7).all() and (out[:, 0, h * D:] == 7).all()


def test_window_attn_cache_past_32_bits(ops, dev):
    """A cache of more than 2^32 bytes: the newest keys lie behind the 32-bit offsets."""
    L, h, D = 2_200_000, 8, 128
    k = torch.zeros(1, L, h, D, dtype=BF16, device=dev)
    v = torch.zeros_like(k)
    rand = _gen(dev, 12)
    k[:, -300:], v[:, -300:] = rand(1, 300, h, D).bfloat16(), rand(1, 300, h, D).bfloat16()
    q = rand(1, 3, h, D).bfloat16()
    o = torch.empty_like(q)
    ops.window_attn(q, k, v, o, 290, sinks=4)
    o2 = torch.empty_like(q)
    kk, vv = (torch.cat([t[:, :4], t[:, -300:]], 1) for t in (k, v))
    ref, tol = R.window_attn(q, kk, vv, o2, 290, 4, 1, None, None, D ** -0.5)
    _within(o, ref, tol)


# ---- block-scaled e4m3 ---------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("pow2", [False, True])
@pytest.mark.parametrize("M,K", [(1, 16), (3, 128), (65, 1040), (257, 400), (1000, 4096)])
def test_quant_block_exact(ops, dev, dtype, pow2, M, K):
    rand = _gen(dev, M + K)
    x = (rand(M, K) * torch.exp(2 * rand(M, 1)) * torch.exp(rand(K))).to(dtype)
    x[M // 2, :min(K, 128)] = 0
    if dtype != F16:
        x[M - 1, :16] = 1e-38                      # scale at its smallest
    q = torch.empty(M, K, dtype=torch.float8_e4m3fn, device=dev)
    s = torch.empty(-(-K // 128), M, device=dev)
    ops.quant_block(x, q, s, pow2=pow2)
    rq, rs = R.quant_block(x, pow2)
    assert torch.equal(s.double(), rs)
    assert torch.equal(q.float().double(), rq)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("pow2", [False, True])
def test_quant_block_every_magnitude(ops, dev, dtype, pow2):
    rand = _gen(dev, 5)
    e = torch.arange(-149, 128, device=dev).double()     # a row each, down to denormal groups
    x = (rand(277, 256).double() % 1.0 * torch.exp2(e)[:, None])
    x[:, 1::2] = x[:, 1::2] * 2.0 ** -4
    x = x.to(dtype)
    q = torch.empty(277, 256, dtype=torch.float8_e4m3fn, device=dev)
    s = torch.empty(2, 277, device=dev)
    ops.quant_block(x, q, s, pow2=pow2)
    rq, rs = R.quant_block(x, pow2)
    assert torch.equal(s.double(), rs)
    assert torch.equal(q.float().double(), rq)


def test_quant_block_views_and_not_finite(ops, dev):
    rand = _gen(dev, 21)
    wide = rand(40, 512).bfloat16()
    x = wide[:, 64:320]
    x[3, 5], x[4, 200] = math.inf, math.nan
    qw = torch.full((40, 512), 7, dtype=torch.uint8, device=dev)
    sw = torch.full((2, 50), 7.0, device=dev)
    ops.quant_block(x, qw[:, 128:384], sw[:, :40])
    rq, rs = R.quant_block(x.nan_to_num(0, 0, 0), False)
    bad = torch.zeros(2, 40, dtype=torch.bool, device=dev)
    bad[0, 3] = bad[1, 4] = True                   # their groups' scales, and no others
    assert torch.equal(torch.isnan(sw[:, :40]), bad)
    assert torch.equal(sw[:, :40][~bad].double(), rs[~bad])
    assert (sw[:, 40:] == 7).all() and (qw[:, :128] == 7).all() and (qw[:, 384:] == 7).all()
    assert torch.equal(qw[0, 128:384].view(torch.float8_e4m3fn).float().double(), rq[0])


def _gemm_case(ops, dev, M, N, K, dtype, bias, gelu, res, seed=0, pad=0):
    rand = _gen(dev, seed)
    e4 = lambda r, c: (90 * rand(r, c + pad)).clamp(-448, 448).to(torch.float8_e4m3fn)[:, :c]  # noqa
    a, b = e4(M, K), e4(N, K)
    G = -(-K // 128)
    sa = torch.exp(rand(G, M)) / 90
    sb = torch.exp(rand(-(-N // 128), G)) / (90 * K ** 0.5)
    bi = rand(N) if bias else None
    R_ = rand(M, N) if res else None
    c = torch.full((M, N + pad), 5.0, dtype=dtype, device=dev)
    ops.gemm_block(a, sa, b, sb, c[:, :N], bias=bi, R=R_, gelu=gelu)
    ref, tol = R.gemm_block(a, sa, b, sb, bi, gelu, R_, dtype)
    _within(c[:, :N], ref, tol, f"{M} {N} {K}")
    assert (c[:, N:] == 5).all()


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("M,N,K", [(1, 1, 16), (1, 4096, 1024), (5, 130, 208), (16, 48, 2048),
                                   (17, 1000, 768), (33, 257, 400), (64, 64, 128), (100, 384, 8448),
                                   (129, 100, 9216), (200, 2050, 640), (768, 1024, 1024)])
def test_gemm_block(ops, dev, dtype, M, N, K):
    _gemm_case(ops, dev, M, N, K, dtype, M % 2 == 1, False, False, seed=M)


@pytest.mark.parametrize("groups", [1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11, 16, 17])
def test_gemm_block_every_ring_length(ops, dev, groups):
    """K-tiles fewer than, equal to and more than the stages, odd ones between two key groups."""
    K = 128 * groups
    for M, N, k in ((40, 96, K), (400, 1040, K), (700, 1030, K - 48), (700, 2100, K),
                    (1200, 2100, K)):
        _gemm_case(ops, dev, M, N, k, BF16, True, False, False, seed=groups)


@pytest.mark.parametrize("bias,gelu,res", [(True, True, False), (True, False, True),
                                           (False, True, True), (False, False, True)])
@pytest.mark.parametrize("M,N,K", [(7, 260, 512), (300, 515, 272), (520, 768, 256)])
def test_gemm_block_epilogues(ops, dev, bias, gelu, res, M, N, K):
    _gemm_case(ops, dev, M, N, K, F32, bias, gelu, res)
    _gemm_case(ops, dev, M, N, K, BF16, bias, gelu, res, pad=16)


@pytest.mark.parametrize("M,N,K", [(2300, 2100, 1040), (2048, 4096, 512), (4100, 1030, 144)])
def test_gemm_block_large_tiles(ops, dev, M, N, K):
    _gemm_case(ops, dev, M, N, K, BF16, True, False, False)
    _gemm_case(ops, dev, M, N, K, F32, False, True, True)


@pytest.mark.parametrize("K", [16, 128, 208, 256, 384, 512, 592, 640])
def test_gemm_block_256_tiles(ops, dev, K):
    """From 160 tiles of 256 x 256 on the two-group kernel takes over: one to five K-tiles, a cut
    one, odd and even counts, cut rows and columns, aligned rows and others."""
    _gemm_case(ops, dev, 3300, 3104, K, BF16, True, False, False, seed=K)
    _gemm_case(ops, dev, 3300, 3101, K, F16, True, True, False, seed=K + 1)
    _gemm_case(ops, dev, 3073, 3200, K, F32, False, False, True, seed=K + 2)


@pytest.mark.parametrize("bias,gelu,res", [(True, True, True), (True, False, True),
                                           (False, True, False), (False, False, False)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_gemm_block_256_tiles_epilogues(ops, dev, bias, gelu, res, dtype):
    """Every operand a view with strides of its own; then bias, residual and results that are not
    16-B aligned."""
    M, N, K = 2600, 4100, 272                            # 11 x 17 tiles
    _gemm_case(ops, dev, M, N, K, dtype, bias, gelu, res, seed=1, pad=16)
    rand = _gen(dev, 77)
    a, b = ((90 * rand(r, K)).clamp(-448, 448).to(torch.float8_e4m3fn) for r in (M, N))
    sa, sb = torch.rand(3, M + 7, device=dev)[:, 5:M + 5], torch.rand(33, 5, device=dev)[:, :3]
    wide = torch.full((M, N + 5), 5.0, dtype=dtype, device=dev)
    bi = rand(N + 3)[3:] if bias else None
    R_ = rand(M, N + 1)[:, 1:] if res else None
    ops.gemm_block(a, sa / 9e3, b, sb, wide[:, 3:N + 3], bias=bi, R=R_, gelu=gelu)
    ref, tol = R.gemm_block(a, sa / 9e3, b, sb, bi, gelu, R_, dtype)
    _within(wide[:, 3:N + 3], ref, tol)
    assert (wide[:, :3] == 5).all() and (wide[:, N + 3:] == 5).all()


@pytest.mark.parametrize("M,N", [(17, 40_961), (100, 41_000), (257, 20_500), (41_000, 40)])
def test_gemm_block_256_tiles_one_band(ops, dev, M, N):
    """Few rows of many columns, and the other way round: bands that are mostly padding."""
    _gemm_case(ops, dev, M, N, 400, BF16, True, False, False, seed=M)
    _gemm_case(ops, dev, M, N, 256, F32, False, False, True, seed=M)


def test_gemm_block_256_tiles_not_finite(ops, dev):
    """A NaN factor or operand reaches its own row or column only."""
    rand = _gen(dev, 78)
    M, N, K = 3300, 3100, 640
    a, b = ((90 * rand(r, K)).clamp(-448, 448).to(torch.float8_e4m3fn) for r in (M, N))
    sa, sb = torch.rand(5, M, device=dev), torch.rand(25, 5, device=dev)
    ref, tol = R.gemm_block(a, sa, b, sb, None, False, None, F32)
    sa[1, 300], sa[4, 3299], sb[3, 2] = math.nan, math.nan, math.nan
    a.view(torch.uint8)[700, 639], b.view(torch.uint8)[3099, 0] = 0x7f, 0x7f
    c = torch.empty(M, N, device=dev)
    ops.gemm_block(a, sa, b, sb, c)
    bad = torch.zeros(M, N, dtype=torch.bool, device=dev)
    bad[[300, 700, 3299]] = True
    bad[:, 384:512], bad[:, 3099] = True, True
    assert torch.equal(torch.isnan(c), bad)
    _within(torch.where(bad, 0, c), torch.where(bad, 0, ref), tol)


@pytest.mark.parametrize("K", [272, 1024, 4096])
@pytest.mark.parametrize("M,N", [(8, 4000), (100, 500), (700, 1000), (700, 2100), (1200, 2100),
                                 (3300, 3100)])
def test_gemm_block_f32_rms(ops, dev, M, N, K):
    """f32 results on each kernel: no sum but the instruction's own is kept in few bits."""
    rand = _gen(dev, M + K)
    G = -(-K // 128)
    a, b = ((90 * rand(r, K)).clamp(-448, 448).to(torch.float8_e4m3fn) for r in (M, N))
    sa, sb = torch.exp(rand(G, M)) / 90, torch.exp(rand(-(-N // 128), G)) / (90 * K ** 0.5)
    c = torch.empty(M, N, device=dev)
    ops.gemm_block(a, sa, b, sb, c)
    ref, _ = R.gemm_block(a, sa, b, sb, None, False, None, F32)
    rms = float((c.double() - ref).square().mean().sqrt() / ref.square().mean().sqrt())
    print(f"rms {rms:.3g}")
    assert rms <= R.GEMM_BLOCK_RMS


def test_gemm_block_residual_in_place_and_not_finite(ops, dev):
    """R may be C; a NaN scale (a group that held an Inf) makes its row NaN and no other."""
    rand = _gen(dev, 31)
    M, N, K = 70, 200, 384
    x = rand(M, K)
    x[9, 130] = math.inf
    q, s = torch.empty(M, K, dtype=torch.uint8, device=dev), torch.empty(3, M, device=dev)
    ops.quant_block(x, q, s)
    from monst3r_slam_amd.model import quant_e4m3_block
    w, sw = quant_e4m3_block(rand(N, K))
    c = rand(M, N)
    ref, tol = R.gemm_block(q.view(torch.float8_e4m3fn), s, w.view(torch.float8_e4m3fn), sw, None,
                            False, c, F32)
    ops.gemm_block(q, s, w, sw, c, R=c)
    rows = torch.arange(M, device=dev) != 9
    assert torch.isnan(c[9]).all()
    _within(c[rows], ref[rows], tol[rows])


@pytest.mark.parametrize("M,N,K", [(40, 60, 256), (300, 260, 272), (700, 1036, 640),
                                   (700, 2100, 400), (1200, 2100, 144), (3300, 3100, 384)])
def test_gemm_block_residual_in_place_at_a_cut_chunk(ops, dev, M, N, K):
    """Columns that end inside a chunk of 8, rows aligned: R as C on every tile kernel, and 16-bit
    rows of a padded C."""
    rand = _gen(dev, N)
    a, b = ((90 * rand(r, K)).clamp(-448, 448).to(torch.float8_e4m3fn) for r in (M, N))
    G = -(-K // 128)
    sa, sb = torch.exp(rand(G, M)) / 90, torch.exp(rand(-(-N // 128), G)) / (90 * K ** 0.5)
    bias, c = rand(N), 3 * rand(M, N)
    wide = torch.full((M, N + 4), 5.0, dtype=BF16, device=dev)
    ops.gemm_block(a, sa, b, sb, wide[:, :N], bias=bias, R=c)
    ref, tol = R.gemm_block(a, sa, b, sb, bias, False, c, BF16)
    _within(wide[:, :N], ref, tol, "16-bit")
    assert (wide[:, N:] == 5).all()
    ref, tol = R.gemm_block(a, sa, b, sb, bias, False, c, F32)
    ops.gemm_block(a, sa, b, sb, c, bias=bias, R=c)
    _within(c, ref, tol, "in place")


def test_gemm_block_deterministic(ops, dev):
    rand = _gen(dev, 33)
    M, N, K = 40, 512, 4096
    a, b = ((90 * rand(r, K)).to(torch.float8_e4m3fn) for r in (M, N))
    sa, sb = torch.rand(32, M, device=dev), torch.rand(4, 32, device=dev)
    outs = [torch.empty(M, N, device=dev) for _ in range(3)]
    for o in outs:
        ops.gemm_block(a, sa, b, sb, o)
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


# ---- offsets past 32 bits: more than 2^32 bytes of inputs and results; the last rows are held
# against the restatement of those rows alone ------------------------------------------------

def test_quant_and_gemm_past_32_bits(ops, dev):
    rand = _gen(dev, 61)
    M, K, N, last = 600_000, 8192, 64, slice(599_900, 600_000)
    x = torch.zeros(M, K, dtype=BF16, device=dev)
    x[last] = rand(100, K).bfloat16()
    q, s = torch.empty(M, K, dtype=torch.float8_e4m3fn, device=dev), torch.empty(64, M, device=dev)
    ops.quant_block(x, q, s)
    rq, rs = R.quant_block(x[last], False)
    assert torch.equal(q[last].float().double(), rq) and torch.equal(s[:, last].double(), rs)
    del x
    b = (90 * rand(N, K)).clamp(-448, 448).to(torch.float8_e4m3fn)
    sb = torch.rand(1, 64, device=dev) / 90
    c = torch.empty(M, N, device=dev)
    ops.gemm_block(q, s, b, sb, c)
    ref, tol = R.gemm_block(q[last], s[:, last], b, sb, None, False, None, F32)
    _within(c[last], ref, tol)
    assert (c[:599_900] == 0).all()


@pytest.mark.parametrize("vec", [True, False])
def test_gemm_block_results_past_32_bits(ops, dev, vec):
    rand = _gen(dev, 62)
    M, N, K, last = 70_000, 33_000 + (not vec), 128, slice(69_900, 70_000)
    a, b = ((90 * rand(r, K)).clamp(-448, 448).to(torch.float8_e4m3fn) for r in (M, N))
    sa, sb = torch.rand(1, M, device=dev) / 90, torch.rand(-(-N // 128), 1, device=dev) / 90
    c = torch.zeros(M, N, device=dev)
    c[last] = rand(100, N)
    ref, tol = R.gemm_block(a[last], sa[:, last], b, sb, None, False, c[last], F32)
    ops.gemm_block(a, sa, b, sb, c, R=c)
    _within(c[last], ref, tol)


def test_norm_and_attention_rows_past_32_bits(ops, dev):
    rand = _gen(dev, 63)
    S, h, D, L = 2_200_000, 8, 128, 300
    q = torch.zeros(1, S, h, D, dtype=BF16, device=dev)
    q[:, -L:] = rand(1, L, h, D).bfloat16()
    k, v = rand(1, L, 2, D).bfloat16(), rand(1, L, 2, D).bfloat16()
    o = torch.full_like(q, 3.0)
    ops.window_attn(q, k, v, o, 64, sinks=2)              # query S - L + j stands at key j
    ref, tol = R.window_attn(q[:, -L:], k, v, o[:, -L:], 64, 2, 1, None, None, D ** -0.5)
    _within(o[:, -L:], ref, tol)
    assert (o[:, :-L] == 0).all()
    pos = torch.arange(S, device=dev)[:, None]
    ko = torch.empty_like(q)
    ops.qk_norm_rope(q, q, pos, o, ko, base=10000.0)
    ref, amp = R.norm_rope(q[:, -L:], None, None, pos[None, -L:], False, 1e-6, 10000.0)
    _within(o[:, -L:], ref, _norm_tol(ref, amp, BF16))
    assert torch.equal(ko, o) and (o[:, :-L] == 0).all()


# ---- together ------------------------------------------------------------------------------

class _Layer:
    """A transformer layer over a stream, as a user writes it: block-scaled projections, head
    norm + rotation into the cache, windowed attention, residual."""

    def __init__(self, ops, dev, B, C, heads, kv_heads, D, cache, seed=41):
        from monst3r_slam_amd.model import quant_e4m3_block
        rand = _gen(dev, seed)
        self.ops, self.dev, self.dims = ops, dev, (B, C, heads, kv_heads, D)
        n = (heads + 2 * kv_heads) * D
        self.w, self.sw = quant_e4m3_block(rand(n, C) / C ** 0.5)
        self.p, self.sp = quant_e4m3_block(rand(C, heads * D) / (heads * D) ** 0.5)
        self.bias, self.gq, self.gk = rand(n), 1 + 0.1 * rand(D), 1 + 0.1 * rand(D)
        self.k = torch.full((B, cache, kv_heads, D), math.nan, dtype=BF16, device=dev)
        self.v = torch.full_like(self.k, math.nan)

    def __call__(self, x, row, kv_len, pos, window, sinks, frame):
        """x f32 [B, S, C] (the residual stream, updated in place)."""
        B, C, hq, hk, D = self.dims
        S = x.shape[1]
        M, n = B * S, (hq + 2 * hk) * D
        new = lambda *s, t=BF16: torch.empty(*s, dtype=t, device=self.dev)  # noqa: E731
        q8, s8 = new(M, C, t=torch.uint8), new(-(-C // 128), M, t=F32)
        self.ops.quant_block(x.view(M, C), q8, s8)
        qkv = new(M, n)
        self.ops.gemm_block(q8, s8, self.w, self.sw, qkv, bias=self.bias)
        h = qkv.view(B, S, -1, D)
        q = new(B, S, hq, D)
        self.ops.qk_norm_rope(h[:, :, :hq], h[:, :, hq:hq + hk], pos, q, self.k, gamma_q=self.gq,
                              gamma_k=self.gk, base=100.0, v=h[:, :, hq + hk:], v_out=self.v,
                              kv_row=row)
        o = new(B, S, hq, D)
        self.ops.window_attn(q, self.k, self.v, o, window, sinks=sinks, frame=frame,
                             kv_len=kv_len)
        o8, so = new(M, hq * D, t=torch.uint8), new(-(-hq * D // 128), M, t=F32)
        self.ops.quant_block(o.view(M, hq * D), o8, so, pow2=True)
        self.ops.gemm_block(o8, so, self.p, self.sp, x.view(M, C), R=x.view(M, C))
        self.seen = dict(q8=q8, s8=s8, qkv=qkv, q=q, o=o, o8=o8, so=so)
        return x


def _stream(layer, x, frame, window, sinks, step):
    """The layer over x [B, T, C], `step` tokens at a time."""
    B, T, _ = x.shape
    out = []
    for t in range(0, T, step):
        n = min(step, T - t)
        row = torch.full((B,), t, dtype=torch.int32, device=x.device)
        pos = torch.arange(t, t + n, device=x.device)
        pos = torch.stack([pos // 8, pos % 8], -1)
        out.append(layer(x[:, t:t + n].clone(), row, row + n, pos, window, sinks, frame))
    return torch.cat(out, 1)


@pytest.mark.parametrize("D,hq,hk", [(64, 4, 4), (128, 4, 2)])
def test_layer_over_a_stream(ops, dev, D, hq, hk):
    """Frame by frame through the cache; every operator against the 64-bit restatement on what
    the one before it wrote."""
    B, C, frame, window, sinks, T = 2, 320, 24, 2, 5, 120
    rand = _gen(dev, 40)
    layer = _Layer(ops, dev, B, C, hq, hk, D, T + 8)
    x = rand(B, T, C)
    for t in range(0, T, frame):
        row = torch.full((B,), t, dtype=torch.int32, device=dev)
        pos = torch.arange(t, t + frame, device=dev)
        pos = torch.stack([pos // 8, pos % 8], -1)
        xin = x[:, t:t + frame].contiguous()
        got = layer(xin.clone(), row, row + frame, pos, window, sinks, frame)
        z = layer.seen
        e8 = lambda a: a.view(torch.float8_e4m3fn)  # noqa: E731
        rq, rs = R.quant_block(xin.view(-1, C), False)
        assert torch.equal(e8(z["q8"]).float().double(), rq) and torch.equal(z["s8"].double(), rs)
        ref, tol = R.gemm_block(e8(z["q8"]), z["s8"], e8(layer.w), layer.sw, layer.bias, False,
                                None, BF16)
        _within(z["qkv"], ref, tol, "qkv")
        h = z["qkv"].view(B, frame, -1, D)
        bp = pos.expand(B, frame, 2)
        for out, part, g in ((z["q"], h[:, :, :hq], layer.gq),
                             (layer.k[:, t:t + frame], h[:, :, hq:hq + hk], layer.gk)):
            ref, amp = R.norm_rope(part, g, None, bp, False, 1e-6, 100.0)
            _within(out, ref, _norm_tol(ref, amp, BF16), "norm")
        assert torch.equal(layer.v[:, t:t + frame], h[:, :, hq + hk:])
        ref, tol = R.window_attn(z["q"], layer.k, layer.v, z["o"], window, sinks, frame, None,
                                 [t + frame] * B, D ** -0.5)
        _within(z["o"], ref, tol, "attention")
        rq, rs = R.quant_block(z["o"].reshape(B * frame, -1), True)
        assert torch.equal(e8(z["o8"]).float().double(), rq) and torch.equal(z["so"].double(), rs)
        ref, tol = R.gemm_block(e8(z["o8"]), z["so"], e8(layer.p), layer.sp, None, False,
                                xin.view(-1, C), F32)
        _within(got.view(-1, C), ref, tol, "proj")


def test_layer_captured_and_replayed(ops, dev):
    """Two captured graphs of the layer, one frame each, replayed in turn with eager work between
    the replays, equal the eager results bit by bit; device-side rows move between replays."""
    B, C, hq, hk, D, frame, T = 1, 256, 4, 2, 64, 32, 2048
    rand = _gen(dev, 42)
    make = lambda: _Layer(ops, dev, B, C, hq, hk, D, T)  # noqa: E731
    x = rand(B, frame, C)
    rows = [torch.full((B,), r, dtype=torch.int32, device=dev) for r in (0, 1500, 700)]
    pos = torch.randint(0, 50, (frame, 2), device=dev)
    layer = make()
    layer.k.zero_()
    layer.v.zero_()
    eager = [layer(x.clone(), r, r + frame, pos, 20, 10, frame).clone() for r in rows]
    graphs = []
    for i in range(2):
        cap = make()
        cap.k.zero_()
        cap.v.zero_()
        row, lens, xin = rows[0].clone(), rows[0] + frame, x.clone()
        side = torch.cuda.Stream(dev)
        side.wait_stream(torch.cuda.current_stream(dev))
        with torch.cuda.stream(side):
            cap(xin, row, lens, pos, 20, 10, frame)
        torch.cuda.current_stream(dev).wait_stream(side)
        cap.k.zero_()
        cap.v.zero_()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            cap(xin, row, lens, pos, 20, 10, frame)
        graphs.append((g, row, lens, xin, cap))   # a graph reads its layer's weights and cache
    streams = [torch.cuda.Stream(dev) for _ in graphs]
    for n, r in enumerate(rows):
        for (g, row, lens, xin, _), st in zip(graphs, streams):
            row.copy_(r)
            lens.copy_(r + frame)
            xin.copy_(x)
            st.wait_stream(torch.cuda.current_stream(dev))
            with torch.cuda.stream(st):   # both graphs in flight at once
                g.replay()
        torch.cuda.synchronize(dev)
        for _, _, _, xin, _ in graphs:
            assert torch.equal(xin, eager[n]), f"replay {n}"
        _ = (x @ x.transpose(1, 2).contiguous()).sum()


# ---- refusals (nothing is launched) --------------------------------------------------------

def test_refusals(ops, dev):
    z = lambda *s, t=BF16: torch.zeros(*s, dtype=t, device=dev)  # noqa: E731
    q, k = z(1, 4, 4, 64), z(1, 4, 2, 64)
    pos = z(4, 1, t=torch.int64)

    def refuse(fn, *a, **kw):
        with pytest.raises(RuntimeError):
            fn(*a, **kw)

    n = ops.qk_norm_rope
    refuse(n, q.cpu(), k, pos, q, k)
    refuse(n, q, k, pos.int(), q, k)
    refuse(n, q, k, pos[:3], q, k)
    refuse(n, q, k, z(4, 3, t=torch.int64), q, k)
    refuse(n, q, k.half(), pos, q, k)
    refuse(n, q.float(), k.float(), pos, q.float(), k.float())
    refuse(n, z(1, 4, 4, 32), z(1, 4, 2, 32), pos, z(1, 4, 4, 32), z(1, 4, 2, 32))
    refuse(n, q, k, pos, z(1, 5, 4, 64), k)
    refuse(n, q, k, pos, q, z(1, 3, 2, 64))
    refuse(n, q, k, pos, q, k, gamma_q=z(32, t=F32))
    refuse(n, q, k, pos, q, k, gamma_q=z(64))
    refuse(n, q, k, pos, q, k, v=k)
    refuse(n, q, k, pos, q, k, kv_row=z(1, t=torch.int64))
    refuse(n, q, k, pos, q, k, base=0.0)
    refuse(n, q, k, pos, q, k, eps=float("nan"))
    refuse(n, q.transpose(1, 2), k, pos, q, k)
    refuse(n, z(1, 4, 4 * 64 + 4)[:, :, 4:].unflatten(2, (4, 64)), k, pos, q, k)
    w = ops.window_attn
    o = z(1, 4, 4, 64)
    refuse(w, q, k, k, o, -1)
    refuse(w, q, k, k, o, 1, sinks=-1)
    refuse(w, q, k, k, o, 1, frame=0)
    refuse(w, q, k, k, o, 1, scale=0.0)
    refuse(w, q, k, k, o, 1, scale=float("inf"))
    refuse(w, q, z(1, 4, 3, 64), z(1, 4, 3, 64), o, 1)
    refuse(w, q, k, z(1, 5, 2, 64), o, 1)
    refuse(w, q, k, k, z(1, 4, 4, 128), 1)
    refuse(w, q, k, k, o.half(), 1)
    refuse(w, q, k, k, o, 1, kv_len=z(2, t=torch.int32))
    refuse(w, q, k, k, o, 1, q_len=z(1, t=torch.int64))
    refuse(w, q, z(2, 4, 2, 64), z(2, 4, 2, 64), o, 1)
    refuse(w, q.cpu(), k, k, o, 1)
    e8 = z(4, 128, t=torch.uint8)
    b = ops.quant_block
    refuse(b, z(4, 120), z(4, 120, t=torch.uint8), z(1, 4, t=F32))
    refuse(b, z(4, 128), e8, z(4, 1, t=F32))
    refuse(b, z(4, 128, t=torch.float64), e8, z(1, 4, t=F32))
    refuse(b, z(4, 128), z(4, 128), z(1, 4, t=F32))
    refuse(b, z(128, 4).t(), e8, z(1, 4, t=F32))
    m = ops.gemm_block
    s1, c = z(1, 4, t=F32), z(4, 4)
    refuse(m, e8, s1, z(4, 112, t=torch.uint8), z(1, 1, t=F32), c)
    refuse(m, e8, s1, e8, z(2, 1, t=F32), c)
    refuse(m, e8, z(4, 1, t=F32), e8, z(1, 1, t=F32), c)
    refuse(m, e8, s1, e8, z(1, 1, t=F32), z(4, 5))
    refuse(m, e8, s1, e8, z(1, 1, t=F32), c, bias=z(4))
    refuse(m, e8, s1, e8, z(1, 1, t=F32), c, R=z(4, 4))
    refuse(m, z(4, 8, t=torch.uint8), s1, z(4, 8, t=torch.uint8), z(1, 1, t=F32), c)


def test_empty_calls(ops, dev):
    z = lambda *s, t=BF16: torch.zeros(*s, dtype=t, device=dev)  # noqa: E731
    ops.qk_norm_rope(z(0, 4, 2, 64), z(0, 4, 1, 64), z(4, 1, t=torch.int64), z(0, 4, 2, 64),
                     z(0, 8, 1, 64))
    ops.window_attn(z(1, 0, 2, 64), z(1, 4, 1, 64), z(1, 4, 1, 64), z(1, 0, 2, 64), 1)
    o = torch.ones(1, 3, 2, 64, dtype=BF16, device=dev)
    ops.window_attn(z(1, 3, 2, 64), z(1, 0, 1, 64), z(1, 0, 1, 64), o, 1)   # an empty cache: 0
    assert (o == 0).all()
    ops.quant_block(z(0, 128), z(0, 128, t=torch.uint8), z(1, 0, t=F32))
    ops.gemm_block(z(0, 128, t=torch.uint8), z(1, 0, t=F32), z(4, 128, t=torch.uint8),
                   z(1, 1, t=F32), z(0, 4))
    torch.cuda.synchronize(dev)


def test_calls_on_another_stream(ops, dev):
    """Work goes to the current stream and scratch is the call's own: two streams at once."""
    rand = _gen(dev, 51)
    q = [rand(1, 1, 8, 128).bfloat16() for _ in range(2)]
    k, v = rand(1, 20000, 2, 128).bfloat16(), rand(1, 20000, 2, 128).bfloat16()
    want = [torch.empty_like(t) for t in q]
    for t, o in zip(q, want):
        ops.window_attn(t, k, v, o, 0)
    torch.cuda.synchronize(dev)
    streams = [torch.cuda.Stream(dev) for _ in q]
    got = [[torch.zeros_like(t) for _ in range(5)] for t in q]
    torch.cuda.synchronize(dev)
    for i in range(5):
        for t, os, st in zip(q, got, streams):
            with torch.cuda.stream(st):
                ops.window_attn(t, k, v, os[i], 0)
    torch.cuda.synchronize(dev)
    for os, w in zip(got, want):
        assert all(torch.equal(o, w) for o in os)
