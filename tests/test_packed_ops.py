"""The operators of a packed request batch -- per-head norm with rotation, attention over key ranges,
projections with per-row adapters -- against plain fp64 forms, and what they refuse.

Tolerances are elementwise bounds from the roundings that the kernels make: half a step of bf16 is
2^-8 of the value, of fp32 2^-24."""
import ctypes
import math

import pytest
import torch

from wanb200 import _lib as L
from wanb200 import ops, ranges

DEV = "cuda"
BF16 = torch.bfloat16
HALF = 2.0 ** -8  # half a bf16 step, relative


@pytest.fixture()
def word():
    """The device error word is clear before and after."""
    L.device_error(reset=True)
    yield
    assert L.device_error(reset=True) == 0, "a kernel reported a device-side error"


def randn(*shape, scale=1.0, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=DEV) * scale).to(BF16)


def within(got, ref, tol):
    d = (got.double() - ref).abs()
    bad = ~(d <= tol)
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} off, worst {float((d / tol.clamp_min(1e-300)).max()):.2f} x the bound"


# ---------------------------------------------------------------------------- key ranges (CPU)
@pytest.mark.parametrize("lengths,block,prefix,window", [
    ([5, 0, 1, 9], 0, None, 0), ([5, 0, 1, 9], 1, None, 0), ([7, 12], 4, None, 0), ([7, 12], 1, [3, 20], 0),
    ([7, 12], 1, 2, 3), ([7, 12], 0, None, 2), ([], 0, None, 0)])
def test_document_ranges_are_the_mask(lengths, block, prefix, window):
    lo, hi = ranges.document_ranges(lengths, "cpu", block=block, prefix=prefix, window=window)
    assert lo.dtype == torch.int32 and lo.shape == hi.shape == (sum(lengths),)
    pre = prefix if isinstance(prefix, list) else [prefix or 0] * len(lengths)
    doc = [(d, t) for d, n in enumerate(lengths) for t in range(n)]
    for i, (d, t) in enumerate(doc):
        seen = []
        for j, (e, u) in enumerate(doc):
            ok = d == e and (not block or u // block <= t // block or u < pre[d])
            if window:
                ok = ok and t - u < window and (block or u - t < window)
            if ok:
                seen.append(j)
        assert seen == list(range(int(lo[i]), int(hi[i]))), (i, seen)


def test_cache_and_padded_ranges():
    lo, hi, pos = ranges.cache_ranges(torch.tensor([3, 9], dtype=torch.int32), 2)
    assert hi.tolist() == [[2, 3], [8, 9]] and pos.tolist() == [[1, 2], [7, 8]] and not lo.any()
    lo, hi, _ = ranges.cache_ranges(torch.tensor([3, 9], dtype=torch.int32), 1, window=4)
    assert lo.tolist() == [[0], [5]] and hi.tolist() == [[3], [9]]
    lo, hi = ranges.padded_ranges([0, 2], 3, "cpu")
    assert hi.tolist() == [[0, 0, 0], [2, 2, 0]]
    with pytest.raises(ValueError):
        ranges.padded_ranges([4], 3, "cpu")
    with pytest.raises(ValueError):
        ranges.document_ranges([-1], "cpu")


@pytest.mark.parametrize("q_len,window", [(-1, 0), (1, -1)])
def test_cache_ranges_refuses_negative_sizes(q_len, window):
    with pytest.raises(ValueError):
        ranges.cache_ranges(torch.tensor([3], dtype=torch.int32), q_len, window=window)


# ---------------------------------------------------------------------------- refusals (CPU)
def _refused(fn, p, word):
    rc = fn(ctypes.byref(p), None)
    assert rc == -1
    assert word in L.load().wanb200_last_error().decode(), (word, L.load().wanb200_last_error())


def _norm_params():
    p = L.HeadNormParams()
    p.x = p.out = 256
    p.ldx = p.ldo = 512
    p.rows, p.nsections, p.head_dim, p.eps = 3, 2, 64, 1e-6
    p.col0[0], p.col0[1], p.heads[0], p.heads[1] = 0, 256, 4, 2
    p.gamma[0] = p.gamma[1] = 256
    p.cos = p.sin = 256
    p.rot, p.table_rows = 64, 10
    return p


@pytest.mark.parametrize("field,value,word", [
    ("x", None, "need x"), ("rows", 0, "rows > 0"), ("head_dim", 96, "head_dim"), ("nsections", 3, "nsections"),
    ("ldx", 500, "strides"), ("ldo", 1024, "in place"), ("x", 264, "16-byte"), ("sin", None, "together"),
    ("rot", 24, "rot"), ("rot", 128, "rot"), ("table_rows", 0, "table_rows")])
def test_head_norm_rope_refuses_on_host(field, value, word):
    p = _norm_params()
    setattr(p, field, value)
    _refused(L.load().wanb200_head_norm_rope, p, word)


def test_head_norm_rope_refuses_bad_sections_on_host():
    for i, field, value, word in ((0, "col0", 4, "section"), (1, "col0", 448, "section"), (1, "col0", 128, "overlap"),
                                  (0, "heads", 0, "section"), (1, "gamma", 264, "section")):
        p = _norm_params()
        getattr(p, field)[i] = value
        _refused(L.load().wanb200_head_norm_rope, p, word)
    p = _norm_params()
    p.cos = p.sin = p.gamma[0] = p.gamma[1] = None
    _refused(L.load().wanb200_head_norm_rope, p, "neither")


def _range_params():
    p = L.RangeAttnParams()
    p.q = p.k = p.v = p.o = 4096
    p.lo = p.hi = 4096
    p.batch, p.heads, p.kv_heads, p.q_len, p.kv_len, p.head_dim = 2, 4, 2, 5, 9, 64
    p.q_tok_stride = p.o_tok_stride = 256
    p.k_tok_stride = p.v_tok_stride = 128
    p.q_batch_stride = p.o_batch_stride = 256 * 5
    p.k_batch_stride = p.v_batch_stride = 128 * 9
    p.softmax_scale = 0.125
    return p


@pytest.mark.parametrize("field,value,word", [
    ("q", None, "null"), ("lo", None, "null"), ("head_dim", 96, "head_dim"), ("q_len", 0, "positive"),
    ("kv_len", 0, "positive"), ("kv_heads", 3, "multiple"), ("k_tok_stride", 100, "multiples of 8"),
    ("k_tok_stride", 64, "token stride"), ("v", 4104, "aligned"), ("softmax_scale", 0.0, "softmax_scale"),
    ("softmax_scale", float("nan"), "softmax_scale"), ("softmax_scale", float("inf"), "softmax_scale"),
    ("softcap", -1.0, "softcap"), ("softcap", 1e-20, "softcap"), ("softcap", float("nan"), "softcap"), ("softcap", float("inf"), "softcap"),
    ("range_batch_stride", -1, "range_batch_stride"), ("kv_len", 2 ** 31, "too large")])
def test_range_attention_refuses_on_host(field, value, word):
    p = _range_params()
    setattr(p, field, value)
    _refused(L.load().wanb200_range_attn_fwd, p, word)


def test_range_attention_refuses_two_biases_and_bad_reach_on_host():
    p = _range_params()
    p.slopes = p.dist_bias = 4096
    _refused(L.load().wanb200_range_attn_fwd, p, "not both")
    for reach in (-1, 8193):
        p.slopes, p.reach = None, reach
        _refused(L.load().wanb200_range_attn_fwd, p, "reach")
        assert L.load().wanb200_range_attn_workspace_bytes(ctypes.byref(p)) == 0


def _lora_params():
    p = L.LoraParams()
    g = p.gemm
    g.a = g.w = g.d = g.bias = 4096
    g.lda = g.ldw = 128
    g.ldd = 64
    g.M, g.N, g.K, g.epilogue = 10, 64, 128, L.EPI_BIAS
    p.down = p.up = p.ids = p.lora_workspace = 4096
    p.adapters, p.rank = 3, 16
    p.lora_workspace_bytes = 1 << 30
    return p


@pytest.mark.parametrize("field,value,word", [
    ("adapters", 0, "adapters"), ("rank", 12, "rank"), ("adapters", 300, "4096"), ("down", None, "down"),
    ("up", 4104, "aligned"), ("ids", None, "ids"), ("lora_workspace", None, "workspace"),
    ("lora_workspace_bytes", 100, "workspace"), ("lora_workspace", 4112, "workspace")])
def test_gemm_lora_refuses_on_host(field, value, word):
    p = _lora_params()
    setattr(p, field, value)
    _refused(L.load().wanb200_gemm_lora, p, word)


def test_gemm_lora_refuses_epilogues_and_gemm_limits_on_host():
    p = _lora_params()
    p.gemm.epilogue, p.gemm.rowss, p.gemm.ss_cols = L.EPI_BIAS_SUMSQ, 4096, 64
    _refused(L.load().wanb200_gemm_lora, p, "SUMSQ")
    p = _lora_params()
    p.gemm.K = 96
    _refused(L.load().wanb200_gemm_lora, p, "multiple of 64")
    assert L.load().wanb200_lora_workspace_bytes(10, 3, 12, 0) == 0
    assert L.load().wanb200_lora_workspace_bytes(100, 3, 16, 1) > L.load().wanb200_lora_workspace_bytes(100, 3, 16, 0) > 0


def test_ops_need_cuda_tensors():
    x = torch.zeros(2, 64, dtype=BF16)
    with pytest.raises(L.WanB200Error):
        ops.head_norm_rope(x, [(0, 1, x[0])], 64)
    q = torch.zeros(1, 2, 1, 64, dtype=BF16)
    r = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(L.WanB200Error):
        ops.range_attention(q, q, q, r, r)
    with pytest.raises(L.WanB200Error):
        ops.lora_linear(x, x, None, x, x, r)


def test_blocks_of_rows_that_share_no_byte():
    """ops._apart against the bytes themselves; it may refuse, but never pass a pair that shares one."""
    g = torch.Generator().manual_seed(3)
    passed = 0
    for _ in range(3000):
        a, b = ([int(x) for x in torch.randint(0, hi, (4,), generator=g)] for hi in (24, 24))
        if passed % 2:
            b[1] = a[1]  # one stride
        a[2], b[2], a[3], b[3] = a[2] % 6 + 1, b[2] % 6 + 1, a[3] % 4 + 1, b[3] % 4 + 1
        bytes_of = [{p + i * st + k for i in range(m) for k in range(w)} for p, st, w, m in (a, b)]
        if ops._apart(a, b):
            passed += 1
            assert not bytes_of[0] & bytes_of[1], (a, b)
        assert ops._apart(a, b) == ops._apart(b, a)
    assert passed > 300
    assert ops._apart((0, 16, 4, 9), (4, 16, 12, 9)) and not ops._apart((0, 16, 4, 9), (3, 16, 4, 9))


# ---------------------------------------------------------------------------- head norm
def head_norm_ref(x, secs, d, rot, cos, sin, pos, inter, eps=1e-6):
    """fp64 (values, bound): the bound is half a bf16 step plus fp32 steps of the pair's magnitude."""
    y = x.double().clone()
    mag = torch.zeros_like(y)
    for c0, heads, g in secs:
        for h in range(heads):
            c = slice(c0 + h * d, c0 + (h + 1) * d)
            v = x[:, c].double()
            if g is not None:
                v = v / (v.pow(2).mean(1, keepdim=True) + eps).sqrt() * g.double()
            m = v.abs()
            if cos is not None:
                half = rot // 2
                i = torch.arange(half, device=x.device)
                a, b = (2 * i, 2 * i + 1) if inter else (i, i + half)
                co, si = cos.double()[pos], sin.double()[pos]
                z, m = v.clone(), m.clone()
                z[:, a], z[:, b] = v[:, a] * co - v[:, b] * si, v[:, a] * si + v[:, b] * co
                m[:, a] = m[:, b] = v[:, a].abs() + v[:, b].abs()
                v = z
            y[:, c], mag[:, c] = v, m
    # fp32: the mean, rsqrt, two products of the gain and the rotation: at most 16 half steps
    return y, HALF * y.abs() + 16 * 2.0 ** -24 * mag


@pytest.mark.gpu
@pytest.mark.parametrize("M,hq,hk,d,rot,inter", [
    (1, 24, 24, 128, 128, True), (1, 1, 1, 64, 64, False), (77, 5, 3, 64, 48, False), (33, 32, 8, 128, 64, True),
    (130, 7, 1, 128, 96, False), (9, 3, 2, 256, 256, True), (9, 3, 2, 256, 80, False), (300, 24, 24, 128, 128, False)])
def test_head_norm_rope(M, hq, hk, d, rot, inter, word):
    x = randn(M, (hq + 2 * hk) * d + 8, seed=M)
    gq, gk = randn(d, seed=1), randn(d, seed=2)
    P = 50
    ang = torch.rand(P, rot // 2, device=DEV) * 6
    cos, sin = ang.cos(), ang.sin()
    pos = torch.randint(0, P, (M,), device=DEV, dtype=torch.int32)
    secs = [(8, hq, gq), (8 + hq * d, hk, gk)]
    ref, tol = head_norm_ref(x, secs, d, rot, cos, sin, pos.long(), inter)
    out = torch.full((M, (hq + hk) * d + 24), 7.0, dtype=BF16, device=DEV)
    ops.head_norm_rope(x, secs, d, out=out, cos=cos, sin=sin, positions=pos, interleaved=inter)
    w = slice(8, 8 + (hq + hk) * d)
    within(out[:, w], ref[:, w], tol[:, w])
    assert bool((out[:, :8] == 7).all()) and bool((out[:, w.stop:] == 7).all())
    y = x.clone()  # in place, and the other columns as they were
    assert ops.head_norm_rope(y, secs, d, cos=cos, sin=sin, positions=pos, interleaved=inter) is y
    assert torch.equal(y[:, w], out[:, w]) and torch.equal(y[:, w.stop:], x[:, w.stop:]) and torch.equal(y[:, :8], x[:, :8])


@pytest.mark.gpu
@pytest.mark.parametrize("M,hq,hk,d,rot,inter", [
    (1300, 24, 24, 128, 128, True), (1701, 21, 11, 128, 96, False), (2400, 23, 21, 64, 64, True), (2401, 6, 5, 256, 80, False),
    (2500, 32, 8, 64, 48, False), (700, 24, 24, 128, 128, True)])
def test_head_norm_rope_many_rows(M, hq, hk, d, rot, inter, word):
    """Rows enough for six passes a warp, with heads that fill them, leave some idle, or too many idle."""
    x, gq, gk = randn(M, (hq + hk) * d, seed=M), randn(d, seed=1), randn(d, seed=2)
    ang = torch.rand(M, rot // 2, device=DEV) * 6
    secs = [(0, hq, gq), (hq * d, hk, gk)]
    ref, tol = head_norm_ref(x, secs, d, rot, ang.cos(), ang.sin(), torch.arange(M, device=DEV), inter)
    out = torch.empty_like(x)
    ops.head_norm_rope(x, secs, d, out=out, cos=ang.cos(), sin=ang.sin(), interleaved=inter)
    within(out, ref, tol)


@pytest.mark.gpu
def test_head_norm_rope_forms(word):
    M, d = 40, 64
    x = randn(M, 6 * d, seed=3)
    g = randn(d, seed=4)
    ang = torch.rand(16, d // 2, device=DEV)
    cos, sin = ang.cos(), ang.sin()
    pos = torch.arange(M, device=DEV) % 16
    for secs, tabs in (([(0, 4, g)], True), ([(0, 4, None), (4 * d, 2, g)], True), ([(2 * d, 3, g)], False)):
        kw = dict(cos=cos, sin=sin) if tabs else {}
        ref, tol = head_norm_ref(x, secs, d, d, cos if tabs else None, sin, pos, True)
        within(ops.head_norm_rope(x.clone(), secs, d, **kw), ref, tol)
    assert ops.head_norm_rope(x[:0], [(0, 4, g)], d).shape == (0, 6 * d)
    # zeros norm to zero, an infinite head is not a number, its neighbours are untouched by it
    x[3] = 0
    x[5, :d] = math.inf
    y = ops.head_norm_rope(x.clone(), [(0, 6, g)], d)
    assert bool((y[3] == 0).all()) and bool(y[5, :d].isnan().all()) and bool(y[5, d:].isfinite().all())


@pytest.mark.gpu
def test_head_norm_rope_leaves_rows_with_bad_positions():
    L.device_error(reset=True)
    M, d = 6, 128
    x = randn(M, 2 * d, seed=5)
    g = randn(d, seed=6)
    cos = sin = torch.ones(10, d // 2, device=DEV)
    pos = torch.tensor([0, 10, 3, -1, 9, 2 ** 31 - 1], dtype=torch.int32, device=DEV)
    y = ops.head_norm_rope(x.clone(), [(0, 2, g)], d, cos=cos, sin=sin, positions=pos)
    assert L.device_error(reset=True) == 501
    good = torch.tensor([True, False, True, False, True, False], device=DEV)
    assert torch.equal(y[~good], x[~good]) and not bool((y[good] == x[good]).all(1).any())


@pytest.mark.gpu
def test_head_norm_rope_refuses_overlap():
    x = randn(8, 512, seed=1)
    g = randn(64, seed=2)
    with pytest.raises(ValueError, match="overlap"):
        ops.head_norm_rope(x[:4], [(0, 2, g)], 64, out=x[1:5])
    with pytest.raises(ValueError, match="outside"):
        ops.head_norm_rope(x, [(0, 9, g)], 64)
    with pytest.raises(ValueError, match="positions"):
        ops.head_norm_rope(x, [(0, 2, g)], 64, cos=torch.ones(4, 32, device=DEV), sin=torch.ones(4, 32, device=DEV),
                           positions=torch.zeros(8, dtype=torch.int64, device=DEV))


@pytest.mark.gpu
def test_head_norm_rope_offsets_past_32_bits(word):
    M, hq, d, ld = 700_000, 2, 128, 3200
    x = torch.zeros(M, ld, dtype=BF16, device=DEV)
    assert x.numel() > 2 ** 31
    x[-40:] = randn(40, ld, seed=7)
    g, ang = randn(d, seed=8), torch.rand(50, d // 2, device=DEV) * 6
    pos = (torch.arange(M, device=DEV) % 50).to(torch.int32)
    secs = [(ld - hq * d, hq, g)]
    ref, tol = head_norm_ref(x[-40:], secs, d, d, ang.cos(), ang.sin(), pos[-40:].long(), True)
    ops.head_norm_rope(x, secs, d, cos=ang.cos(), sin=ang.sin(), positions=pos)
    within(x[-40:], ref, tol)
    assert not bool(x[:-40].any())


# ---------------------------------------------------------------------------- range attention
def attn_ref(q, k, v, lo, hi, pos=None, cap=0.0, slopes=None, table=None, scale=None):
    """fp64 (o, bound).  The kernel rounds the weights to bf16 for the product with v (half a step of
    each, so 2^-8 sum w|v|) and the output (2^-8 |o|).  A score's fp32 error e moves its weight by
    e: the dot product, scale, cap and bias are good to 2^-20 of their magnitude, summed in `se`."""
    B, Lq, H, D = q.shape
    Lk, g = k.shape[1], H // k.shape[2]
    scale = D ** -0.5 if scale is None else scale
    j = torch.arange(Lk, device=q.device)
    lo, hi = (t.view(-1, Lq).long() for t in (lo, hi))
    pos = torch.arange(Lq, device=q.device)[None] if pos is None else pos.view(-1, Lq).long()
    out = torch.zeros(B, Lq, H, D, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    for b in range(B):
        l, u, p = (t[b if t.shape[0] > 1 else 0][:, None] for t in (lo, hi, pos))
        seen = (j >= l) & (j < u)
        dist = j - p
        for h in range(H):
            qd, kd = q[b, :, h].double(), k[b, :, h // g].double()
            vd = v[b, :, h // g].double()
            s = qd @ kd.t() * scale
            mag = qd.abs() @ kd.abs().t() * scale + cap
            if cap:
                s = cap * torch.tanh(s / cap)
            if slopes is not None:
                s = s - slopes[h].double() * dist.abs()
                mag = mag + slopes[h].double() * dist.abs()
            if table is not None:
                r = table.shape[1] // 2
                bias = table[h].double()[dist.clamp(-r, r) + r]
                s, mag = s + bias, mag + bias.abs()
            s = s.masked_fill(~seen, -math.inf)
            some = seen.any(1)
            w = torch.zeros_like(s)
            w[some] = torch.softmax(s[some], 1)
            for i in range(Lq):  # row by row over its own keys only: what others hold must not matter
                if bool(some[i]) and not bool(vd[seen.any(0)].isfinite().all()):
                    keys = seen[i]
                    out[b, i, h] = w[i, keys] @ vd[keys]
            if bool(vd.isfinite().all()):
                out[b, :, h] = w @ vd
            mag = torch.where(seen & mag.isfinite(), mag, torch.zeros_like(mag))
            av = torch.where(vd.isfinite(), vd.abs(), torch.zeros_like(vd))
            se = 2.0 ** -20 * mag.amax(1, keepdim=True) + 2.0 ** -20
            tol[b, :, h] = (HALF * 1.01 + 2 * se) * (w.nan_to_num() @ av) + HALF * out[b, :, h].abs()
    return out, tol + 1e-30


def check_attn(q, k, v, lo, hi, **kw):
    names = {"cap": "softcap", "table": "dist_bias", "scale": "softmax_scale"}
    got = ops.range_attention(q, k, v, lo, hi, **{names.get(n, n): x for n, x in kw.items()})
    ref, tol = attn_ref(q, k, v, lo, hi, **kw)
    within(got, ref, tol)
    return got


def ints(*rows):
    return torch.tensor(rows, dtype=torch.int32, device=DEV)


def random_ranges(B, Lq, Lk, seed):
    """Arbitrary ranges, some empty, some past the ends."""
    g = torch.Generator().manual_seed(seed)
    a = torch.randint(-5, Lk + 6, (2, B, Lq), generator=g)
    lo, hi = a.amin(0), a.amax(0)
    hi = torch.where(torch.rand(B, Lq, generator=g) < 0.2, lo - 1, hi)
    return lo.to(torch.int32).to(DEV), hi.to(torch.int32).to(DEV)


SHAPES = [(1, 1, 1, 1, 1, 64), (1, 1, 1, 2, 2, 128), (2, 1, 300, 4, 2, 128), (3, 1, 77, 6, 2, 64), (1, 3, 130, 4, 4, 64),
          (2, 5, 129, 8, 1, 128), (1, 17, 257, 3, 3, 128), (1, 127, 128, 2, 1, 64), (2, 129, 200, 4, 2, 128),
          (1, 300, 300, 6, 2, 64), (1, 260, 515, 2, 2, 128), (1, 70, 1000, 10, 2, 128), (1, 40, 90, 12, 1, 64)]


@pytest.mark.gpu
@pytest.mark.parametrize("B,Lq,Lk,H,Hkv,D", SHAPES)
def test_range_attention_arbitrary_ranges(B, Lq, Lk, H, Hkv, D, word):
    q, k, v = randn(B, Lq, H, D, seed=1), randn(B, Lk, Hkv, D, seed=2), randn(B, Lk, Hkv, D, seed=3)
    lo, hi = random_ranges(B, Lq, Lk, 7)
    got = check_attn(q, k, v, lo, hi)
    empty = (lo.clamp_min(0) >= hi.clamp_max(Lk))
    assert bool((got[empty] == 0).all())
    full = torch.zeros_like(lo), torch.full_like(hi, Lk)
    check_attn(q, k, v, *full)
    assert torch.equal(ops.range_attention(q, k, v, *full), ops.range_attention(q, k, v, *full))


@pytest.mark.gpu
@pytest.mark.parametrize("lengths,block,prefix,window,H,Hkv,D", [
    ([100, 1, 0, 260, 7], 1, None, 0, 4, 2, 128), ([100, 1, 260, 7], 0, None, 0, 2, 2, 64), ([200, 333], 1, 50, 0, 3, 1, 64),
    ([512], 1, None, 0, 2, 2, 128), ([300, 300], 22, None, 0, 2, 1, 128), ([600], 1, None, 40, 2, 2, 64),
    ([5] * 60, 0, None, 0, 2, 2, 128)])
def test_range_attention_documents(lengths, block, prefix, window, H, Hkv, D, word):
    T = sum(lengths)
    q, k, v = randn(1, T, H, D, seed=4), randn(1, T, Hkv, D, seed=5), randn(1, T, Hkv, D, seed=6)
    lo, hi = ranges.document_ranges(lengths, DEV, block=block, prefix=prefix, window=window)
    check_attn(q, k, v, lo, hi)


@pytest.mark.gpu
@pytest.mark.parametrize("lengths,block,prefix,H,Hkv,D", [
    ([2600], 374, None, 16, 16, 128), ([3000, 77, 900], 1, 130, 8, 4, 128), ([1500, 2000], 0, None, 24, 24, 64)])
def test_range_attention_many_units_a_block(lengths, block, prefix, H, Hkv, D, word):
    """More units than SMs, each with a run of fully seen key tiles before the partly seen ones."""
    T = sum(lengths)
    q, k, v = randn(1, T, H, D, seed=4), randn(1, T, Hkv, D, seed=5), randn(1, T, Hkv, D, seed=6)
    lo, hi = ranges.document_ranges(lengths, DEV, block=block, prefix=prefix)
    got = check_attn(q, k, v, lo, hi)
    assert torch.equal(got, ops.range_attention(q, k, v, lo, hi))


@pytest.mark.gpu
def test_range_attention_many_short_sequences(word):
    """More tile pairs than the plan sorts, and more (key head, batch element) pairs than the few-rows
    kernel deals out."""
    for B, Lq, H, Hkv in ((1100, 17, 2, 2), (500, 2, 4, 2)):
        q, k, v = randn(B, Lq, H, 64, seed=1), randn(B, 40, Hkv, 64, seed=2), randn(B, 40, Hkv, 64, seed=3)
        check_attn(q, k, v, *random_ranges(B, Lq, 40, 5))


@pytest.mark.gpu
@pytest.mark.parametrize("H,Hkv", [(10, 1), (7, 1), (96, 1), (24, 2)])
def test_range_attention_groups_that_do_not_fill_a_tile(H, Hkv, word):
    """Key heads shared by numbers of query heads that leave rows of the 128-row tile unused."""
    for Lq in (1, 3, 150):
        q, k, v = randn(1, Lq, H, 128, seed=1), randn(1, 300, Hkv, 128, seed=2), randn(1, 300, Hkv, 128, seed=3)
        lo, hi = random_ranges(1, Lq, 300, 6)
        check_attn(q, k, v, lo, hi, cap=20.0)
        check_attn(q, k, v, lo, hi, slopes=torch.rand(H, device=DEV))


@pytest.mark.gpu
@pytest.mark.parametrize("Lq", [1, 4, 130])
def test_range_attention_long_cache_of_unequal_lengths(Lq, word):
    """Caches from nothing to 5000 keys in one batch, views of a larger cache."""
    B, H, Hkv, D = 7, 8, 4, 64
    cache = randn(2, B, 5100, Hkv, D, seed=7)
    k, v = cache[0, :, 50:5050], cache[1, :, 50:5050]
    q = randn(B, Lq, H, D, seed=8)
    lens = torch.tensor([0, 1, 5000, 77, 64, 4097, 2048], dtype=torch.int32, device=DEV)
    lo, hi, pos = ranges.cache_ranges(lens, Lq)
    check_attn(q, k, v, lo, hi, pos=pos, slopes=torch.rand(H, device=DEV) * 0.1)
    lo, hi, pos = ranges.cache_ranges(lens, Lq, window=100)
    check_attn(q, k, v, lo, hi, pos=pos)


@pytest.mark.gpu
@pytest.mark.parametrize("B,Lq,H,Hkv,D", [(5, 3, 16, 4, 128), (5, 4, 16, 4, 64), (3, 16, 3, 3, 128), (2, 9, 2, 2, 64),
                                          (40, 5, 16, 8, 64), (60, 2, 64, 8, 64)])
def test_range_attention_nine_to_sixteen_rows_of_unequal_caches(B, Lq, H, Hkv, D, word):
    """Two column tiles a block, with one and with several blocks a cache."""
    Lk = 900 if B > 10 else 4000
    q, k, v = randn(B, Lq, H, D, seed=40), randn(B, Lk, Hkv, D, seed=41), randn(B, Lk, Hkv, D, seed=42)
    lens = torch.randint(0, Lk + 1, (B,), dtype=torch.int32, generator=torch.Generator().manual_seed(B))
    lens[0], lens[1] = Lk, 0
    lo, hi, pos = ranges.cache_ranges(lens.to(DEV), Lq)
    check_attn(q, k, v, lo, hi, pos=pos)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("cap", [0.0, 5.0, 50.0])
@pytest.mark.parametrize("bias", ["none", "slopes", "table", "short_table", "flat_table"])
@pytest.mark.parametrize("B,Lq,Lk,H,Hkv", [(2, 1, 150, 4, 2), (1, 150, 280, 4, 2), (2, 4, 260, 3, 3)])
def test_range_attention_cap_and_bias(B, Lq, Lk, H, Hkv, cap, bias, D, word):
    q, k, v = randn(B, Lq, H, D, scale=2.0, seed=8), randn(B, Lk, Hkv, D, scale=2.0, seed=9), randn(B, Lk, Hkv, D, seed=10)
    lo, hi = random_ranges(B, Lq, Lk, 11)
    pos = torch.randint(-20, Lk + 20, (B, Lq), dtype=torch.int32, device=DEV)
    slopes = table = None
    if bias == "slopes":
        slopes = torch.rand(H, device=DEV)
    elif bias != "none":
        table = torch.randn(H, 2 * {"table": 40, "short_table": 3, "flat_table": 0}[bias] + 1, device=DEV)
    check_attn(q, k, v, lo, hi, pos=pos, cap=cap, slopes=slopes, table=table)
    if bias == "slopes" and not cap:
        check_attn(q, k, v, lo, hi, slopes=slopes)  # positions default to the row


def capped_ref(q, k, v, lo, hi, cap):
    """fp64 (o, bound) of capped scores whose error goes with the score itself, whatever the cap: the dot
    product to 2^-20 of its magnitude (as attn_ref), the cap to 2^-16 of the capped score (its polynomial is
    9e-6 from tanh, the general form below that where it is used, above 0.6 of the cap)."""
    B, Lq, H, D = q.shape
    g, j = H // k.shape[2], torch.arange(k.shape[1], device=q.device)
    kd, vd = (t.double().repeat_interleave(g, 2) for t in (k, v))
    s = torch.einsum("bihd,bjhd->bhij", q.double(), kd) / math.sqrt(D)
    mag = torch.einsum("bihd,bjhd->bhij", q.double().abs(), kd.abs()) / math.sqrt(D)
    s = cap * torch.tanh(s / cap)
    seen = ((j >= lo.view(-1, Lq, 1)) & (j < hi.view(-1, Lq, 1)))[:, None]
    w = torch.softmax(s.masked_fill(~seen, -math.inf), 3).nan_to_num(0.0)
    o = torch.einsum("bhij,bjhd->bihd", w, vd)
    av = torch.einsum("bhij,bjhd->bihd", w, vd.abs())
    e = w * (2.0 ** -20 * (mag + 1) + 2.0 ** -16 * s.abs())  # a score off by e moves w by w e, and the sum by all of them
    moved = torch.einsum("bhij,bjhd->bihd", e, vd.abs()) + e.sum(3).transpose(1, 2)[..., None] * av
    return o, HALF * 1.01 * av + moved + HALF * o.abs() + 1e-30


@pytest.mark.gpu
@pytest.mark.parametrize("cap", [10.0, 256.0, 300.0, 1e3, 1e5, 1e6])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B,Lq,Lk,H,Hkv", [(2, 1, 300, 4, 2), (1, 3, 1000, 4, 1), (1, 16, 257, 2, 2), (1, 17, 257, 2, 2),
                                           (1, 150, 280, 4, 2)])
def test_range_attention_caps_far_above_the_scores(B, Lq, Lk, H, Hkv, D, cap, word):
    """A cap that no score comes near changes nothing: the weights are those of the plain scores."""
    q, k, v = randn(B, Lq, H, D, scale=2.0, seed=60), randn(B, Lk, Hkv, D, scale=1.5, seed=61), randn(B, Lk, Hkv, D, seed=62)
    lo, hi = random_ranges(B, Lq, Lk, 63)
    within(ops.range_attention(q, k, v, lo, hi, softcap=cap), *capped_ref(q, k, v, lo, hi, cap))


@pytest.mark.gpu
@pytest.mark.parametrize("cap", [30.0, 256.0, 1e4, 1e6])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Lq,Lk", [(2, 300), (12, 300), (150, 300), (300, 300)])
def test_range_attention_small_scores_beside_scores_above_the_cap(Lq, Lk, D, cap, word):
    """Rows with scores far above the cap, and single keys far below it, next to rows and keys with small
    scores, which must not lose their accuracy to them."""
    H = 2
    q, k, v = randn(1, Lq, H, D, scale=2.0, seed=64), randn(1, Lk, H, D, scale=1.5, seed=65), randn(1, Lk, H, D, seed=66)
    lo, hi = torch.zeros(1, Lq, dtype=torch.int32, device=DEV), torch.full((1, Lq), Lk, dtype=torch.int32, device=DEV)
    hi[0, ::3] -= 7
    # key 40 scores about -4 cap with the even rows: it points against a channel that only they have, large
    q[:, :, :, 0], k[:, :, :, 0] = 0, 0
    far = math.sqrt(4 * cap * math.sqrt(D))
    q[0, ::2, :, 0], k[0, 40, :, 0] = far, -far
    # the scores of row 5 are far above the cap on either side, all of the largest size
    if Lq > 5:
        q[0, 5] *= 2 * cap
    got = ops.range_attention(q, k, v, lo, hi, softcap=cap)
    ref, tol = capped_ref(q, k, v, lo, hi, cap)
    rows = torch.arange(Lq, device=DEV) != 5
    within(got[:, rows], ref[:, rows], tol[:, rows])
    if Lq > 5:
        # the keys at +cap weigh alike as far as fp32 tells them apart: convex combinations of v
        assert bool(got[0, 5].isfinite().all()) and bool((got[0, 5].abs() <= v.abs().amax(1)[0] * 1.01).all())


@pytest.mark.gpu
@pytest.mark.parametrize("Lq,Lk,H,Hkv", [(1, 200, 4, 2), (3, 200, 4, 4), (200, 200, 2, 2), (150, 400, 4, 2)])
def test_range_attention_hidden_keys_do_not_reach_a_row(Lq, Lk, H, Hkv, word):
    """NaN and infinities in keys and values that a row does not see; a row that sees them shows it."""
    D = 128
    q, k, v = randn(1, Lq, H, D, seed=12), randn(1, Lk, Hkv, D, seed=13), randn(1, Lk, Hkv, D, seed=14)
    i = torch.arange(Lq, device=DEV)
    hi = (Lk - Lq + i + 1).to(torch.int32)
    lo = (hi - 60).clamp_min(0).contiguous()
    v[0, 30, :, 5], k[0, 31], v[0, Lk - 1], k[0, Lk - 2] = math.nan, math.nan, -math.inf, math.inf
    v[0, 90, 0, 100] = math.inf
    got = ops.range_attention(q, k, v, lo, hi)
    for r in range(Lq):
        a, b = int(lo[r]), int(hi[r])
        one = ops.range_attention(q[:, r:r + 1].contiguous(), k[:, a:b].contiguous(), v[:, a:b].contiguous(),
                                  ints(0)[:1], ints(b - a)[:1])[0, 0]
        ka, va = k[0, a:b].double(), v[0, a:b].double()
        for h in range(H):
            s = (ka[:, h // (H // Hkv)] @ q[0, r, h].double()) / math.sqrt(D)
            ref = torch.softmax(s, 0) @ va[:, h // (H // Hkv)]
            assert torch.equal(got[0, r, h].isfinite(), ref.isfinite()), (r, h)
            assert torch.equal(one[h].isfinite(), ref.isfinite()), (r, h)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("cap", [0.0, 5.0, 1e4])
@pytest.mark.parametrize("bias", ["none", "slopes", "table"])
@pytest.mark.parametrize("Lq,Lk,H,Hkv", [(1, 200, 4, 2), (2, 200, 4, 2), (3, 200, 4, 1), (40, 200, 2, 2), (150, 300, 2, 1)])
def test_range_attention_non_finite_values_seen_and_hidden(Lq, Lk, H, Hkv, bias, cap, D, word):
    """Rows that do not see a NaN or an infinity keep their values; rows that do have what the formula gives,
    infinities with their sign, in every form of the score."""
    q, k, v = randn(1, Lq, H, D, seed=70), randn(1, Lk, Hkv, D, seed=71), randn(1, Lk, Hkv, D, seed=72)
    i = torch.arange(Lq, device=DEV)
    hi = (Lk - Lq + i + 1).to(torch.int32)[None]
    lo = (hi - 70).clamp_min(0)
    lo[0, ::7], hi[0, ::7] = 0, Lk  # some rows see all keys, the last and the first
    v[0, 20, :, 5], v[0, Lk - 1, 0, 7], v[0, Lk - 2, 0, 7], v[0, Lk - 40, Hkv - 1, D - 1] = math.nan, math.inf, -math.inf, math.inf
    k[0, 25], k[0, Lk - 30, 0, 3] = math.nan, math.inf
    kw = dict(cap=cap)
    if bias == "slopes":
        kw["slopes"] = torch.rand(H, device=DEV) * 0.2
    elif bias == "table":
        kw["table"] = torch.randn(H, 61, device=DEV)
    got = ops.range_attention(q, k, v, lo, hi, softcap=cap, slopes=kw.get("slopes"), dist_bias=kw.get("table"))
    ref, tol = attn_ref(q, k, v, lo, hi, **kw)
    fine = ref.isfinite()
    assert Lq == 1 or bool(fine.any())  # a row alone sees all keys
    assert torch.equal(got.isfinite(), fine) and torch.equal(got.isnan(), ref.isnan())
    assert torch.equal(got[ref.isinf()].double(), ref[ref.isinf()])
    within(torch.where(fine, got, torch.zeros_like(got)), torch.where(fine, ref, torch.zeros_like(ref)), tol.nan_to_num(1e-30))


@pytest.mark.gpu
@pytest.mark.parametrize("B,Lq,Lk,H,Hkv,D", [
    (1, 1, 9000, 24, 1, 128), (1, 40, 9000, 1, 1, 64), (1, 1, 12000, 40, 2, 64), (2, 1, 5000, 128, 1, 128), (1, 17, 20000, 1, 1, 128)])
def test_range_attention_few_tiles_over_long_caches(B, Lq, Lk, H, Hkv, D, word):
    """One or two pairs of row tiles over a cache of more key tiles than a pair is split into."""
    q, k, v = randn(B, Lq, H, D, seed=73), randn(B, Lk, Hkv, D, seed=74), randn(B, Lk, Hkv, D, seed=75)
    lens = torch.tensor([Lk, Lk // 3][:B], dtype=torch.int32, device=DEV)
    lo, hi, pos = ranges.cache_ranges(lens, Lq)
    check_attn(q, k, v, lo, hi, pos=pos)
    check_attn(q, k, v, lo, hi, pos=pos, slopes=torch.rand(H, device=DEV) * 0.01, cap=20.0)


@pytest.mark.gpu
@pytest.mark.parametrize("Lq", [1, 150])
def test_range_attention_batch_inside_tokens(Lq, word):
    """Tensors laid out [L, B, H, D]: the batch stride is the smaller one."""
    B, Lk, H, Hkv, D = 3, 200, 4, 2, 64
    q, k, v = (randn(n, B, h, D, seed=s).transpose(0, 1) for n, h, s in ((Lq, H, 76), (Lk, Hkv, 77), (Lk, Hkv, 78)))
    lo, hi = random_ranges(B, Lq, Lk, 79)
    ref, tol = attn_ref(q, k, v, lo, hi)
    out = torch.empty(Lq, B, H, D, dtype=BF16, device=DEV).transpose(0, 1)
    within(ops.range_attention(q, k, v, lo, hi, out=out), ref, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("Lq", [1, 60])
def test_range_attention_offsets_past_32_bits(Lq, word):
    """A cache of more than 2^31 values, seen at its start, its end and, in between, by rows with a few keys."""
    Lk, Hkv, H, D = 2 ** 21 + 1000, 8, 16, 128
    k, v = torch.zeros(1, Lk, Hkv, D, dtype=BF16, device=DEV), torch.zeros(1, Lk, Hkv, D, dtype=BF16, device=DEV)
    assert k.numel() > 2 ** 31
    k[:, -300:], v[:, -300:] = randn(1, 300, Hkv, D, seed=80), randn(1, 300, Hkv, D, seed=81)
    v[:, -400, :, 3] = math.nan  # a tile that is partly seen, its non-finite value hidden
    q = randn(1, Lq, H, D, seed=82)
    pos = (Lk - Lq + torch.arange(Lq, device=DEV)).to(torch.int32)
    lo, hi = pos - 240, pos + 1
    got = ops.range_attention(q, k, v, lo, hi, pos=pos, slopes=torch.full((H,), 0.01, device=DEV))
    cut = Lk - 300
    ref, tol = attn_ref(q, k[:, cut:], v[:, cut:], lo - cut, hi - cut, pos=pos - cut, slopes=torch.full((H,), 0.01, device=DEV))
    within(got, ref, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("low", [torch.finfo(torch.float32).min, -math.inf])
@pytest.mark.parametrize("cap", [0.0, 5.0])
@pytest.mark.parametrize("Lq,Lk,H,Hkv", [(1, 700, 4, 2), (3, 300, 4, 1), (200, 300, 4, 2)])
def test_range_attention_table_of_lowest_values(Lq, Lk, H, Hkv, cap, low, word):
    """A table that is 0 near the row and the lowest value, or -inf, from a distance of R on hides the far keys
    from rows that see a near one.  Where every key has the lowest value all weigh alike (in fp32 no
    score changes it); where every key has -inf the weights are 0 / 0."""
    D, R = 64, 20
    q, k, v = randn(1, Lq, H, D, seed=30), randn(1, Lk, Hkv, D, seed=31), randn(1, Lk, Hkv, D, seed=32)
    table = torch.zeros(H, 2 * R + 1, device=DEV)
    table[:, 0] = table[:, -1] = low
    lo, hi = ints([3] * Lq)[0].contiguous(), ints([Lk - 2] * Lq)[0].contiguous()
    for first in (5, Lk + 100):  # near keys for every row; none
        pos = torch.arange(Lq, dtype=torch.int32, device=DEV) + first
        got = ops.range_attention(q, k, v, lo, hi, pos=pos, softcap=cap, dist_bias=table)
        if first == 5:
            ref, tol = attn_ref(q, k, v, torch.maximum(lo, pos - R + 1), torch.minimum(hi, pos + R), cap=cap)
            within(got, ref, tol)
        elif low == -math.inf:
            assert bool(got.isnan().all())
        else:  # weights of exactly 1, fp32 sums of up to 700 values, one rounding to bf16
            seen = v[:, 3:Lk - 2].double()
            ref = seen.mean(1, keepdim=True).repeat_interleave(H // Hkv, 2).expand(1, Lq, H, D)
            mag = seen.abs().mean(1, keepdim=True).repeat_interleave(H // Hkv, 2).expand(1, Lq, H, D)
            within(got, ref, HALF * 1.01 * ref.abs() + 2.0 ** -14 * mag)


@pytest.mark.gpu
def test_range_attention_extreme_scores(word):
    """Scores far apart, all equal, and of the largest size: the running maximum keeps the sums finite."""
    D, Lk = 64, 300
    for Lq in (1, 200):
        q, k, v = randn(1, Lq, 2, D, scale=40, seed=15), randn(1, Lk, 2, D, scale=40, seed=16), randn(1, Lk, 2, D, seed=17)
        lo, hi = random_ranges(1, Lq, Lk, 18)
        got = ops.range_attention(q, k, v, lo, hi)
        ref, _ = attn_ref(q, k, v, lo, hi)
        # scores up to 1e4: an fp32 score is good to 2^-20 of that, so weights to one part in 100
        assert bool(got.isfinite().all()) and float((got.double() - ref).abs().max()) < 0.05 * float(v.abs().max())
        k.zero_()
        check_attn(q, k, v, lo, hi)


@pytest.mark.gpu
def test_range_attention_strided_views_and_out(word):
    T, H, D = 150, 4, 128
    buf = randn(2, T, 3 * H * D + 64, seed=19)
    q, k, v = (buf[:, :, i * H * D:(i + 1) * H * D].unflatten(2, (H, D)) for i in range(3))
    lo, hi = random_ranges(2, T, T, 20)
    ref, tol = attn_ref(q, k, v, lo, hi)
    big = torch.full((2, T + 3, H + 1, D), 3.0, dtype=BF16, device=DEV)
    out = big[:, 1:T + 1, :H]
    assert ops.range_attention(q, k, v, lo, hi, out=out) is out
    within(out, ref, tol)
    assert bool((big[:, 0] == 3).all()) and bool((big[:, T + 1:] == 3).all()) and bool((big[:, :, H] == 3).all())
    one = ops.range_attention(q[:, :1], k, v, lo[:, :1].contiguous(), hi[:, :1].contiguous())
    within(one, ref[:, :1], tol[:, :1])


@pytest.mark.gpu
@pytest.mark.parametrize("B", [1, 2])
def test_outputs_beside_inputs_in_one_buffer(B, word):
    """Columns of one buffer that do not meet: each call writes its own and leaves the others alone."""
    T, H, D, C = 150, 2, 64, 128
    buf = randn(B, T, 6 * C, seed=83)
    want = buf.clone()
    q, k, v, o = (buf[..., i * C:(i + 1) * C].unflatten(2, (H, D)) for i in range(4))
    lo, hi = random_ranges(B, T, T, 84)
    want[..., 3 * C:4 * C] = ops.range_attention(q.contiguous(), k.contiguous(), v.contiguous(), lo, hi).flatten(2)
    assert ops.range_attention(q, k, v, lo, hi, out=o) is o
    rows, wrows = buf.view(B * T, 6 * C), want.view(B * T, 6 * C)
    _, w, b, down, up, ids, scales = lora_case(B * T, C, C, 3, 16, 85)
    wrows[:, 4 * C:5 * C] = ops.lora_linear(wrows[:, 3 * C:4 * C].contiguous(), w, b, down, up, ids, scales=scales)
    ops.lora_linear(rows[:, 3 * C:4 * C], w, b, down, up, ids, scales=scales, out=rows[:, 4 * C:5 * C])
    g = randn(D, seed=86)
    wrows[:, 5 * C:] = ops.head_norm_rope(wrows[:, 4 * C:5 * C].contiguous(), [(0, H, g)], D)
    ops.head_norm_rope(rows[:, 4 * C:5 * C], [(0, H, g)], D, out=rows[:, 5 * C:])
    assert torch.equal(buf, want)
    for at in (3 * C - 8, 2 * C, 5):
        with pytest.raises(ValueError, match="overlap"):
            ops.range_attention(q, k, v, lo, hi, out=buf[..., at:at + C].unflatten(2, (H, D)))
    with pytest.raises(ValueError, match="overlap"):
        ops.lora_linear(rows[:, :C], w, b, down, up, ids, out=rows[:, C - 8:2 * C - 8])


@pytest.mark.gpu
@pytest.mark.parametrize("Lq", [1, 7, 140])
@pytest.mark.parametrize("two_dims", [False, True])
@pytest.mark.parametrize("D", [64, 128])
def test_range_attention_shared_ranges_and_other_scales(Lq, two_dims, D, word):
    """One range for all batch elements, given as [Lq] or [1, Lq]; scales other than the root's."""
    B, Lk, H, Hkv = 3, 333, 6, 2
    q, k, v = randn(B, Lq, H, D, seed=87), randn(B, Lk, Hkv, D, seed=88), randn(B, Lk, Hkv, D, seed=89)
    lo, hi = random_ranges(1, Lq, Lk, 90)
    pos = torch.randint(-20, Lk + 20, (1, Lq), dtype=torch.int32, device=DEV)
    if not two_dims:
        lo, hi, pos = lo[0], hi[0], pos[0]
    for scale in (1e-3, 0.3):
        check_attn(q, k, v, lo, hi, scale=scale)
        check_attn(q, k, v, lo, hi, pos=pos, scale=scale, cap=4.0, slopes=torch.rand(H, device=DEV))
        check_attn(q, k, v, lo, hi, pos=pos, scale=scale, table=torch.randn(H, 31, device=DEV))


@pytest.mark.gpu
def test_range_attention_empty_tensors_and_refusals(word):
    q, k = randn(2, 3, 4, 64), randn(2, 5, 2, 64)
    lo = hi = torch.zeros(3, dtype=torch.int32, device=DEV)
    assert bool((ops.range_attention(q, k[:, :0], k[:, :0], lo, hi) == 0).all())
    assert ops.range_attention(q[:, :0], k, k, lo[:0], hi[:0]).shape == (2, 0, 4, 64)
    for bad, match in ((dict(lo=lo.long()), "int32"), (dict(hi=hi[:2]), "one shape"), (dict(out=q), "overlap"),
                       (dict(slopes=torch.ones(3, device=DEV)), "slopes"),
                       (dict(dist_bias=torch.ones(4, 4, device=DEV)), "dist_bias"),
                       (dict(slopes=torch.ones(4, device=DEV), dist_bias=torch.ones(4, 3, device=DEV)), "not both")):
        with pytest.raises(ValueError, match=match):
            ops.range_attention(**{**dict(q=q, k=k, v=k, lo=lo, hi=hi), **bad})
    with pytest.raises(ValueError, match="mismatch"):
        ops.range_attention(q, k, k[:, :4], lo, hi)
    with pytest.raises(ValueError, match="multiple"):
        ops.range_attention(q, randn(2, 5, 3, 64), randn(2, 5, 3, 64), lo, hi)
    with pytest.raises(ValueError, match="head stride"):
        ops.range_attention(q, k.transpose(1, 2).contiguous().transpose(1, 2), k, lo, hi)


# ---------------------------------------------------------------------------- adapters
def lora_ref(x, w, bias, down, up, ids, scales, epi, residual=None, gate=None, f32=False):
    """fp64 (y, bound).  fp32 accumulation: a step (2^-23, the tensor core may truncate) of the sum of
    magnitudes for each 16-wide product; h in bf16 (2^-8 of each, 2^-16 in two planes), then the
    output's rounding; tanh and exp of the activations are good to 2^-10 of the input."""
    xd, wd = x.double(), w.double()
    K = x.shape[1]
    y = xd @ wd.t() + (0 if bias is None else bias.double())
    mag = xd.abs() @ wd.abs().t() + (0 if bias is None else bias.double().abs())
    hr = torch.zeros_like(y)
    for a in range(down.shape[0]):
        r = (ids == a).nonzero().squeeze(1)
        if r.numel():
            s = 1.0 if scales is None else scales[a].double()
            h = s * (xd[r] @ down[a].double().t())
            u = up[:, a].double()
            y[r] += h @ u.t()
            hr[r] = h.abs() @ u.abs().t()
            mag[r] += (s * (xd[r].abs() @ down[a].double().abs().t())) @ u.abs().t()
    err = (K / 16 + 8) * 2.0 ** -23 * mag + hr * (2.0 ** -16 if f32 else HALF)
    if epi == L.EPI_BIAS_GELU:
        err = 1.2 * err + 2.0 ** -10 * y.abs()
        y = torch.nn.functional.gelu(y, approximate="tanh")
    if epi == L.EPI_BIAS_SILU:
        err = 1.2 * err + 2.0 ** -20 * y.abs()
        y = torch.nn.functional.silu(y)
    if gate is not None:
        y, err = y * gate, err * gate.abs()
    if residual is not None:
        y = y + residual.double()
    return y, err + (2.0 ** -22 if f32 else HALF) * y.abs() + 1e-30


def lora_case(M, K, N, n, r, seed, order="mixed"):
    g = torch.Generator().manual_seed(seed)
    x, w, b = randn(M, K, seed=seed), randn(N, K, scale=K ** -0.5, seed=seed + 1), randn(N, seed=seed + 2)
    down, up = randn(n, r, K, scale=K ** -0.5, seed=seed + 3), randn(N, n, r, scale=r ** -0.5, seed=seed + 4)
    scales = torch.rand(n, generator=g).to(DEV) + 0.5
    ids = torch.randint(-1, n, (M,), generator=g)
    if order == "sorted":
        ids = ids.sort().values
    return x, w, b, down, up, ids.to(torch.int32).to(DEV), scales


@pytest.mark.gpu
@pytest.mark.parametrize("M,K,N,n,r,order", [
    (1, 64, 32, 1, 8, "mixed"), (1, 512, 96, 5, 16, "mixed"), (4, 1024, 256, 8, 16, "mixed"), (13, 256, 160, 3, 24, "mixed"),
    (16, 2048, 64, 20, 64, "mixed"), (17, 128, 64, 2, 8, "sorted"), (100, 320, 544, 9, 40, "mixed"), (129, 64, 64, 16, 16, "sorted"),
    (300, 704, 256, 4, 64, "sorted"), (400, 256, 1056, 32, 128, "mixed"), (1000, 192, 96, 3, 8, "sorted"),
    (509, 2048, 512, 16, 16, "mixed"), (60, 4096, 320, 7, 40, "mixed"), (2500, 512, 1024, 2, 64, "sorted")])
def test_lora_linear(M, K, N, n, r, order, word):
    x, w, b, down, up, ids, scales = lora_case(M, K, N, n, r, 21, order)
    got = ops.lora_linear(x, w, b, down, up, ids, scales=scales)
    within(got, *lora_ref(x, w, b, down, up, ids, scales, L.EPI_BIAS))
    assert torch.equal(got, ops.lora_linear(x, w, b, down, up, ids, scales=scales))
    none = torch.full_like(ids, -1)
    within(ops.lora_linear(x, w, b, down, up, none), *lora_ref(x, w, b, down, up, none, None, L.EPI_BIAS))
    same = torch.full_like(ids, n - 1)
    within(ops.lora_linear(x, w, None, down, up, same, epilogue=L.EPI_NONE),
           *lora_ref(x, w, None, down, up, same, None, L.EPI_NONE))


@pytest.mark.gpu
@pytest.mark.parametrize("M", [5, 150, 700])
@pytest.mark.parametrize("epi", [L.EPI_BIAS_GELU, L.EPI_BIAS_SILU, L.EPI_BIAS_RES, L.EPI_BIAS_GATE_RES])
@pytest.mark.parametrize("f32", [False, True])
def test_lora_linear_epilogues(M, epi, f32, word):
    K, N, n, r = 256, 512, 4, 16
    x, w, b, down, up, ids, scales = lora_case(M, K, N, n, r, 30)
    dt = torch.float32 if f32 else BF16
    kw, rf = {}, {}
    if epi in (L.EPI_BIAS_RES, L.EPI_BIAS_GATE_RES):
        kw["residual"] = randn(M, N, seed=40).to(dt)
        rf["residual"] = kw["residual"].clone()
    if epi == L.EPI_BIAS_GATE_RES:
        mod, e0 = randn(N, seed=41), torch.randn(5, N, device=DEV)
        kw["gate"], kw["frames"] = (mod, e0), (M, -(-M // 5))
        rf["gate"] = (mod.double() + e0.double())[(torch.arange(M, device=DEV) // -(-M // 5))]
    out = kw["residual"] if "residual" in kw else torch.empty(M, N, dtype=dt, device=DEV)
    got = ops.lora_linear(x, w, b, down, up, ids, scales=scales, epilogue=epi, out=out, **kw)
    within(got, *lora_ref(x, w, b, down, up, ids, scales, epi, f32=f32, **rf))


@pytest.mark.gpu
@pytest.mark.parametrize("M", [7, 260])
@pytest.mark.parametrize("r", [8, 16, 24])
def test_lora_linear_broken_adapters_stay_with_their_rows(M, r, word):
    """NaN and infinite weights: in an adapter that no row uses nothing shows; in one that is used, in
    its rows only, and there in the columns that it reaches."""
    K, N, n = 128, 96, 6
    x, w, b, down, up, ids, scales = lora_case(M, K, N, n, r, 50)
    ids[ids == 1] = 0
    ref, tol = lora_ref(x, w, b, down, up, ids, scales, L.EPI_BIAS)
    up[:, 1], down[1] = math.nan, math.nan
    within(ops.lora_linear(x, w, b, down, up, ids, scales=scales), ref, tol)
    up[5, 2, 3], down[3, 0] = math.inf, math.nan
    ids[0], ids[1] = 2, 3
    ref, tol = lora_ref(x, w, b, down, torch.where(up.isfinite(), up, torch.zeros_like(up)), ids, scales, L.EPI_BIAS)
    got = ops.lora_linear(x, w, b, down, up, ids, scales=scales)
    wrong = torch.zeros_like(ref, dtype=torch.bool)
    wrong[ids == 2, 5] = True
    wrong[ids == 3] = True
    assert torch.equal(~got.isfinite(), wrong)
    within(torch.where(wrong, torch.zeros_like(got), got), torch.where(wrong, torch.zeros_like(ref), ref), tol.nan_to_num(1.0))


def _broken_neighbours(K, N, n, r, M, order, seed=200):
    """Adapters 0, 2, 4, ... in use (or one of them alone), NaN and infinities in the weights of the others."""
    x, w, b, down, up, ids, scales = lora_case(M, K, N, n, r, seed)
    ids = ids.abs() // 2 * 2
    if order == "sorted":
        ids = ids.sort().values
    elif order != "mixed":
        ids = torch.full_like(ids, order)
    up[:, 1::2] = math.nan
    up[3, 1::2, 0] = math.inf
    up[4, 1::2, -1] = -math.inf
    down[1::2] = math.inf
    down[1::2, 0] = math.nan
    return x, w, b, down, up, ids, scales


def _spared(x, w, b, down, up, ids, scales, epi, f32=False, **rf):
    """(y, bound) of lora_ref, the broken adapters, which no row uses, replaced by zeros."""
    clean = [torch.where(t.isfinite(), t, torch.zeros_like(t)) for t in (down, up)]
    return lora_ref(x, w, b, *clean, ids, scales, epi, f32=f32, **rf)


@pytest.mark.gpu
@pytest.mark.parametrize("order", [0, 2, 4, "sorted", "mixed"])
@pytest.mark.parametrize("r", [8, 16, 24, 40])
@pytest.mark.parametrize("M,K", [(9, 128), (17, 128), (260, 128), (700, 128), (260, 2048), (700, 2048)])
def test_lora_linear_spares_rows_beside_broken_adapters(M, K, r, order, word):
    """Ranks that are no multiple of 16 put columns of two adapters into one K step, also where all rows of a
    tile use one adapter; K = 2048 with few tiles shares K over a cluster."""
    case = _broken_neighbours(K, 96, 6, r, M, order)
    within(ops.lora_linear(*case[:6], scales=case[6]), *_spared(*case, L.EPI_BIAS))
    out = torch.empty(M, 96, device=DEV)
    within(ops.lora_linear(*case[:6], scales=case[6], out=out), *_spared(*case, L.EPI_BIAS, f32=True))


@pytest.mark.gpu
@pytest.mark.parametrize("order", ["mixed", "sorted"])
@pytest.mark.parametrize("M,K,r,N", [(11, 64, 16, 64), (40, 64, 8, 64), (300, 64, 64, 96), (300, 2048, 24, 96), (1000, 192, 40, 64)])
def test_lora_linear_fp32_output_keeps_the_intermediate(M, K, r, N, order, word):
    """With w = 0 and one value a row of x the intermediate is a scaled product of two bf16 values, which fp32
    holds to half a step: an fp32 output is as good, up to the additions of its matrix products (a step of fp32
    of the sum of magnitudes for each K step of 16 that adds something, and each bf16 plane of h)."""
    x, w, _, down, up, ids, scales = lora_case(M, K, N, 3, r, 210, order)
    keep = torch.arange(M, device=DEV) * 7 % K
    x = torch.zeros_like(x).scatter_(1, keep[:, None], x.gather(1, keep[:, None]))
    up[:, :, 3:] = 0  # few terms, so that the error of each shows
    ref = torch.zeros(M, N, dtype=torch.float64, device=DEV)
    mag = torch.zeros_like(ref)
    for a in range(3):
        h = scales[a].double() * (x.double() @ down[a].double().t())
        on = (ids == a)[:, None]
        ref += on * (h @ up[:, a].double().t())
        mag += on * (h.abs() @ up[:, a].double().abs().t())
    got = ops.lora_linear(x, torch.zeros_like(w), None, down, up, ids, scales=scales, epilogue=L.EPI_NONE,
                          out=torch.empty(M, N, device=DEV))
    steps = 3 * 2  # planes x steps of 16 columns that hold an adapter's first three
    within(got, ref, (steps + 2) * 2.0 ** -23 * mag + 1e-30)


@pytest.mark.gpu
@pytest.mark.parametrize("M,K,N,n,r", [(9, 4096, 96, 3, 16), (150, 4096, 160, 3, 16), (300, 8192, 96, 4, 64), (1300, 4096, 1056, 4, 64),
                                       (5000, 4096, 512, 16, 16), (2600, 2048, 2048, 2, 8)])
@pytest.mark.parametrize("order", ["mixed", "sorted"])
def test_lora_linear_fp32_output_over_long_sums(M, K, N, n, r, order, word):
    """The tensor core cuts a sum off at each of its steps of 16 K values: a step of fp32 is 2^-24 to 2^-23 of the
    sum so far (0.72 x 2^-23 on average), half of it is cut on average, and the sum so far is 2/3 of the run's end
    (it grows with the root of its length).  A run of 512 values is thus short by 32 x 2/3 x 0.36 x 2^-23 = 9.2e-7,
    and so is the whole, a sum of runs (one sum over K = 4096 is short by 8 times that)."""
    x, w, b, down, up, ids, scales = lora_case(M, K, N, n, r, 240, order)
    y = x.double() @ w.double().t() + b.double()
    for a in range(n):
        on = ids == a
        y[on] += scales[a].double() * (x[on].double() @ down[a].double().t()) @ up[:, a].double().t()
    res = torch.randn(M, N, device=DEV)
    for kw, ref in ((dict(epilogue=L.EPI_BIAS), y), (dict(epilogue=L.EPI_BIAS_RES, residual=res), y + res.double())):
        got = ops.lora_linear(x, w, b, down, up, ids, scales=scales, out=torch.empty(M, N, device=DEV), **kw)
        assert float((got.double() - ref).norm() / ref.norm()) < 1e-6
        # none of it is lost to the order of the runs: the same bits again
        assert torch.equal(got, ops.lora_linear(x, w, b, down, up, ids, scales=scales, out=torch.empty(M, N, device=DEV), **kw))


@pytest.mark.gpu
@pytest.mark.parametrize("epi", [L.EPI_NONE, L.EPI_BIAS_GELU, L.EPI_BIAS_SILU, L.EPI_BIAS_RES, L.EPI_BIAS_GATE_RES])
@pytest.mark.parametrize("M,N,K,tile_n", [(2600, 1024, 1024, 0), (2500, 1056, 640, 256), (700, 544, 1024, 96), (1300, 2016, 1600, 224),
                                          (300, 1056, 1024, 64), (700, 256, 4096, 0)])
@pytest.mark.parametrize("broken", [False, True])
@pytest.mark.parametrize("res_bf16", [False, True])
def test_lora_linear_fp32_epilogues_over_several_runs(M, N, K, tile_n, epi, broken, res_bf16, word):
    """Tiles of every width whose sums come in several runs, whole and with non-finite weights, the residual in
    bf16, or in fp32 and overwritten by the output."""
    residual = epi in (L.EPI_BIAS_RES, L.EPI_BIAS_GATE_RES)
    if res_bf16 and not residual:
        pytest.skip("no residual")
    n, r = 5, 24
    x, w, b, down, up, ids, scales = lora_case(M, K, N, n, r, 250, "sorted")
    if broken:
        up[7, 2, 3], up[40, 2, 0], down[1, 2] = math.inf, math.nan, math.nan
    kw, rf = {}, {}
    out = torch.empty(M, N, device=DEV)
    if residual:
        rf["residual"] = randn(M, N, seed=40) if res_bf16 else torch.randn(M, N, device=DEV)
        kw["residual"] = rf["residual"].clone()
        out = out if res_bf16 else kw["residual"]
    if epi == L.EPI_BIAS_GATE_RES:
        mod, e0 = randn(N, seed=41), torch.randn(7, N, device=DEV)
        kw["gate"], kw["frames"] = (mod, e0), (M, -(-M // 7))
        rf["gate"] = (mod.double() + e0.double())[(torch.arange(M, device=DEV) // -(-M // 7))]
    bias = None if epi == L.EPI_NONE else b
    got = ops.lora_linear(x, w, bias, down, up, ids, scales=scales, epilogue=epi, out=out, tile_n=tile_n, **kw)
    clean = [torch.where(t.isfinite(), t, torch.zeros_like(t)) for t in (down, up)]
    ref, tol = lora_ref(x, w, bias, *clean, ids, scales, epi, f32=True, **rf)
    spared = torch.ones(M, N, dtype=torch.bool, device=DEV)
    if broken:
        spared[ids == 2, 7] = spared[ids == 2, 40] = False
        spared[ids == 1] = False
        assert not bool(got[~spared].isfinite().all())
    within(got[spared], ref[spared], tol[spared])


@pytest.mark.gpu
@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("M,K,frames", [(10, 128, (100, 25, 30, 0)), (10, 128, (100, 25, 30, 5)), (300, 1024, (100, 25, 30, 120)),
                                        (2600, 1024, (500, 50, 130, 0)), (700, 2048, (90, 7, 0, 350))])
def test_lora_linear_gate_of_a_row_s_frame(M, K, frames, f32, word):
    """Rows that start inside a sequence, and several sequences in the rows."""
    N, n, r = 544, 3, 16
    x, w, b, down, up, ids, scales = lora_case(M, K, N, n, r, 260)
    seq, tokens, offset, per = frames
    row = torch.arange(M, device=DEV)
    frame = ((row % per if per else row) + offset) % seq // tokens
    mod, e0 = randn(N, seed=41), torch.randn(-(-seq // tokens), N, device=DEV)
    dt = torch.float32 if f32 else BF16
    res = randn(M, N, seed=42).to(dt)
    got = ops.lora_linear(x, w, b, down, up, ids, scales=scales, epilogue=L.EPI_BIAS_GATE_RES, residual=res, gate=(mod, e0),
                          frames=frames, out=torch.empty(M, N, dtype=dt, device=DEV))
    within(got, *lora_ref(x, w, b, down, up, ids, scales, L.EPI_BIAS_GATE_RES, residual=res, f32=f32,
                          gate=(mod.double() + e0.double())[frame]))


@pytest.mark.gpu
@pytest.mark.parametrize("order", ["mixed", "one"])
@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("M,K,r", [(9, 128, 16), (150, 128, 16), (150, 128, 24), (260, 2048, 16)])
def test_lora_linear_infinite_weight_in_use(M, K, r, f32, order, word):
    """An infinite up-projection weight gives its rows an infinity of the intermediate's sign, whoever shares
    their tile."""
    x, w, b, down, up, ids, scales = lora_case(M, K, 64, 3, r, 220)
    if order == "one":
        ids = torch.full_like(ids, 1)
    up[5, 1, 3], up[6, 1, 0] = math.inf, -math.inf
    got = ops.lora_linear(x, w, b, down, up, ids, scales=scales, out=torch.empty(M, 64, dtype=torch.float32 if f32 else BF16, device=DEV))
    on = ids == 1
    h = x.double() @ down[1].double().t()
    sure = on & (h[:, [0, 3]].abs() > 1e-3).all(1)  # the sign of a value near zero is not settled in fp32
    assert bool(sure.any()) and bool(got[~on].isfinite().all())
    for col, i, sign in ((5, 3, 1.0), (6, 0, -1.0)):
        assert torch.equal(got[sure, col].double(), torch.copysign(torch.full_like(h[sure, i], math.inf), sign * h[sure, i]))
    rest = torch.ones(64, dtype=torch.bool, device=DEV)
    rest[5] = rest[6] = False
    ref, tol = lora_ref(x, w, b, down, torch.where(up.isfinite(), up, torch.zeros_like(up)), ids, scales, L.EPI_BIAS, f32=f32)
    within(got[:, rest], ref[:, rest], tol[:, rest])


@pytest.mark.gpu
@pytest.mark.parametrize("epi", [L.EPI_NONE, L.EPI_BIAS_GELU, L.EPI_BIAS_SILU, L.EPI_BIAS_RES, L.EPI_BIAS_GATE_RES])
@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("M,K", [(12, 128), (150, 128), (260, 2048)])
def test_lora_linear_epilogues_beside_broken_adapters(M, K, epi, f32, word):
    """Tiles with non-finite weights have an epilogue of their own, with and without K shared by a cluster: the
    rows of the other adapters get what they get without them."""
    N, n, r = 96, 4, 16
    x, w, b, down, up, ids, scales = lora_case(M, K, N, n, r, 230)
    up[7, 2, 3], up[40, 2, 0], down[1, 2] = math.inf, math.nan, math.nan
    dt = torch.float32 if f32 else BF16
    kw, rf = {}, {}
    if epi in (L.EPI_BIAS_RES, L.EPI_BIAS_GATE_RES):
        kw["residual"] = rf["residual"] = randn(M, N, seed=40).to(dt)
    if epi == L.EPI_BIAS_GATE_RES:
        mod, e0 = randn(N, seed=41), torch.randn(5, N, device=DEV)
        kw["gate"], kw["frames"] = (mod, e0), (M, -(-M // 5))
        rf["gate"] = (mod.double() + e0.double())[(torch.arange(M, device=DEV) // -(-M // 5))]
    bias = None if epi == L.EPI_NONE else b
    got = ops.lora_linear(x, w, bias, down, up, ids, scales=scales, epilogue=epi, out=torch.empty(M, N, dtype=dt, device=DEV), **kw)
    clean = [torch.where(t.isfinite(), t, torch.zeros_like(t)) for t in (down, up)]
    ref, tol = lora_ref(x, w, bias, *clean, ids, scales, epi, f32=f32, **rf)
    spared = ((ids != 2)[:, None] | ((torch.arange(N, device=DEV) != 7) & (torch.arange(N, device=DEV) != 40))) & (ids != 1)[:, None]
    assert bool((ids == 2).any()) and bool((ids == 1).any()) and not bool(got[~spared].isfinite().all())
    within(got[spared], ref[spared], tol[spared])


@pytest.mark.gpu
def test_lora_linear_bad_id_counts_as_none():
    L.device_error(reset=True)
    for M in (6, 200):
        x, w, b, down, up, ids, scales = lora_case(M, 128, 64, 3, 16, 60)
        ids[2], ids[3] = 3, 2 ** 31 - 1
        got = ops.lora_linear(x, w, b, down, up, ids, scales=scales)
        assert L.device_error(reset=True) == 502
        ids[2] = ids[3] = -1
        within(got, *lora_ref(x, w, b, down, up, ids, scales, L.EPI_BIAS))


@pytest.mark.gpu
def test_lora_linear_views_and_refusals(word):
    M, K, N, n, r = 40, 192, 64, 3, 16
    x, w, b, down, up, ids, scales = lora_case(M, K, N, n, r, 70)
    wide = randn(M, 2 * K, seed=71)
    wide[:, K:] = x
    out = torch.full((M, N + 32), 5.0, dtype=BF16, device=DEV)
    ops.lora_linear(wide[:, K:], w, b, down, up, ids, scales=scales, out=out[:, :N])
    within(out[:, :N], *lora_ref(x, w, b, down, up, ids, scales, L.EPI_BIAS))
    assert bool((out[:, N:] == 5).all())
    assert ops.lora_linear(x[:0], w, b, down, up, ids[:0]).shape == (0, N)
    for bad, match in ((dict(ids=ids.long()), "ids"), (dict(ids=ids[:5]), "ids"), (dict(up=up.transpose(0, 1)), "up"),
                       (dict(down=down[:, :, :64]), "down"), (dict(scales=scales[:2]), "scales"), (dict(out=x[:, :N]), "overlap"),
                       (dict(bias=b[:8]), "bias")):
        with pytest.raises(ValueError, match=match):
            ops.lora_linear(**{**dict(a=x, w=w, bias=b, down=down, up=up, ids=ids), **bad})
    with pytest.raises(L.WanB200Error, match="SUMSQ"):
        ops.lora_linear(x, w, b, down, up, ids, epilogue=L.EPI_SCATTER)


# ---------------------------------------------------------------------------- together
def packed_layer(x, res, P, lo, hi, pos, ids):
    """QKV projection with adapters -> per-head norm and rotation -> attention -> output projection
    with adapters into the residual stream, on rows of packed requests."""
    T, H, Hkv, D = x.shape[0], P["H"], P["Hkv"], P["D"]
    qkv = ops.lora_linear(x, P["wqkv"], P["bqkv"], P["dqkv"], P["uqkv"], ids, scales=P["scales"])
    ops.head_norm_rope(qkv, [(0, H, P["gq"]), (H * D, Hkv, P["gk"])], D, cos=P["cos"], sin=P["sin"], positions=pos)
    q = qkv[:, :H * D].view(1, T, H, D)
    k, v = (qkv[:, (H + i * Hkv) * D:(H + (i + 1) * Hkv) * D].unflatten(1, (Hkv, D))[None] for i in (0, 1))
    o = ops.range_attention(q.unflatten(2, (H, D)) if q.dim() == 3 else q, k, v, lo, hi)
    return ops.lora_linear(o.view(T, H * D), P["wo"], P["bo"], P["do"], P["uo"], ids, scales=P["scales"],
                           epilogue=L.EPI_BIAS_RES, residual=res, out=torch.empty_like(res))


def make_layer(C, H, Hkv, D, n, r, P=4000):
    w = {"H": H, "Hkv": Hkv, "D": D}
    N = (H + 2 * Hkv) * D
    w["wqkv"], w["bqkv"] = randn(N, C, scale=C ** -0.5, seed=80), randn(N, seed=81)
    w["dqkv"], w["uqkv"] = randn(n, r, C, scale=C ** -0.5, seed=82), randn(N, n, r, scale=r ** -0.5, seed=83)
    w["wo"], w["bo"] = randn(C, H * D, scale=(H * D) ** -0.5, seed=84), randn(C, seed=85)
    w["do"], w["uo"] = randn(n, r, H * D, scale=(H * D) ** -0.5, seed=86), randn(C, n, r, scale=r ** -0.5, seed=87)
    w["gq"], w["gk"], w["scales"] = randn(D, seed=88), randn(D, seed=89), torch.rand(n, device=DEV) + 0.5
    ang = torch.arange(P, device=DEV)[:, None] * 10000.0 ** (-torch.arange(D // 2, device=DEV) * 2 / D)
    w["cos"], w["sin"] = ang.cos(), ang.sin()
    return w


@pytest.mark.gpu
@pytest.mark.parametrize("D,H,Hkv", [(64, 6, 2), (128, 4, 4)])
def test_packed_requests_equal_single_requests(D, H, Hkv, word):
    """A packed batch gives each request what it gets alone (up to the roundings of other tile shapes),
    and the rows of a captured and replayed run are those of the eager one, bit for bit."""
    C, n, r = 256, 3, 16
    P = make_layer(C, H, Hkv, D, n, r)
    lengths = [130, 1, 57, 400]
    T = sum(lengths)
    x, res = randn(T, C, seed=90), randn(T, C, seed=91).float()
    lo, hi = ranges.document_ranges(lengths, DEV, block=1)
    pos = torch.cat([torch.arange(m) for m in lengths]).to(torch.int32).to(DEV)
    ids = torch.tensor([0, -1, 2, 1]).repeat_interleave(torch.tensor(lengths)).to(torch.int32).to(DEV)
    y = packed_layer(x, res, P, lo, hi, pos, ids)
    at = 0
    for m in lengths:
        s = slice(at, at + m)
        l1, h1 = ranges.document_ranges([m], DEV, block=1)
        one = packed_layer(x[s], res[s], P, l1, h1, pos[s].contiguous(), ids[s].contiguous())
        # bf16 qkv, weights and outputs in between, each within half a step of the other run's
        assert float((one - y[s]).norm() / (y[s] - res[s]).norm()) < 8 * HALF
        at += m
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        packed_layer(x, res, P, lo, hi, pos, ids)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            z = packed_layer(x, res, P, lo, hi, pos, ids)
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(z, y)
    # the graph reads the ids and ranges at every replay
    ids.fill_(-1)
    hi.copy_(lo)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(z, packed_layer(x, res, P, lo, hi, pos, ids)) and not torch.equal(z, y)


@pytest.mark.gpu
def test_two_streams_at_once(word):
    """The same calls on two streams, running at the same time, do not disturb each other."""
    P = make_layer(512, 8, 2, 128, 4, 16)
    T = 700
    lo, hi = ranges.document_ranges([300, 400], DEV, block=1)
    pos = torch.arange(T, device=DEV).to(torch.int32)
    ids = (torch.arange(T, device=DEV) % 5 - 1).to(torch.int32)
    xs = [(randn(T, 512, seed=s), randn(T, 512, seed=s + 1).float()) for s in (100, 102)]
    want = [packed_layer(x, r, P, lo, hi, pos, ids) for x, r in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(packed_layer(*xs[i], P, lo, hi, pos, ids))
    torch.cuda.synchronize()
    for i in (0, 1):
        assert all(torch.equal(g, want[i]) for g in got[i])


@pytest.mark.gpu
def test_two_captured_graphs_at_once(word):
    """Two captured graphs of the same layer, replayed at the same time, have workspaces of their own."""
    P = make_layer(512, 8, 2, 128, 4, 16)
    sets = []
    for T, seed in ((700, 104), (3, 106)):  # tiles; the few-rows kernels
        lo, hi = ranges.document_ranges([T], DEV, block=1)
        pos = torch.arange(T, device=DEV).to(torch.int32)
        ids = (torch.arange(T, device=DEV) % 5 - 1).to(torch.int32)
        for s in (seed, seed + 10):
            args = (randn(T, 512, seed=s), randn(T, 512, seed=s + 1).float(), P, lo, hi, pos, ids)
            want = packed_layer(*args).clone()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                out = packed_layer(*args)
            sets.append((g, out, want, torch.cuda.Stream(), args))  # the graph reads args
    torch.cuda.synchronize()
    for _ in range(10):
        for g, _, _, st, _ in sets:
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for _, out, want, _, _ in sets:
        assert torch.equal(out, want)
