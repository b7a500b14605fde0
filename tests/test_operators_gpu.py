"""Rotary positions, packed attention and request adapters against plain float64 forms.

Tolerances count roundings: u = 2^-24 for an f32 operation, 2^-22 for an operand carried as an f16
hi + lo pair (its lo part is rounded at 2^-11 of 2^-11 of it), half an ulp of f16 (2^-11 of the
value, 2^-25 below its normal range) for an f16 result. A product of n terms summed in f32 is off by
4 sqrt(n) u of the sum of the terms' magnitudes, the budget of test_gemm_gpu."""
import math

import numpy as np
import pytest

import tgo_amd
from tgo_amd import TgoError

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
HALF = 2.0 ** -11


def f16_step(y):
    return HALF * y.abs() + 2.0 ** -25


# ---------------------------------------------------------------------------
# rotary positions
# ---------------------------------------------------------------------------

SCALINGS = {"none": {}, "linear": dict(scaling=tgo_amd.ROPE_LINEAR, factor=3.0),
            "yarn": dict(scaling=tgo_amd.ROPE_YARN, factor=4.0, original=4096.0, fast=32.0, slow=1.0),
            "bands": dict(scaling=tgo_amd.ROPE_BANDS, factor=8.0, original=8192.0, fast=4.0, slow=1.0)}


def rope64(torch, x, pos, rd, layout, w, m):
    """The definition in float64, and each output's |a| + |b|."""
    x = x.double()
    ang = pos.double().cpu()[:, None] * torch.from_numpy(w)[None, :]
    c, s = (m * ang.cos()).to(x.device)[:, None], (m * ang.sin()).to(x.device)[:, None]
    y, mag = x.clone(), torch.zeros_like(x)
    ia = torch.arange(rd // 2, device=x.device)
    ia, ib = (ia, ia + rd // 2) if layout == tgo_amd.ROPE_HALF else (2 * ia, 2 * ia + 1)
    a, b = x[..., ia], x[..., ib]
    y[..., ia], y[..., ib] = a * c - b * s, a * s + b * c
    mag[..., ia] = mag[..., ib] = m * (a.abs() + b.abs())
    return y, mag


def check_rope(torch, got, x, pos, rd, layout, w, m):
    want, mag = rope64(torch, x, pos, rd, layout, w, m)
    # cos and sin in f32 to 2 ulp of 1 (the angle itself to 2^-30 turns at |position| < 2^31), two
    # products and a sum: 2^-23 + 2^-24 * 3 < 2^-21
    tol = 2.0 ** -21 * mag
    if got.dtype == torch.float16:
        tol = tol + f16_step(want)
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), float((err - tol).max())


@pytest.mark.parametrize("scaling", sorted(SCALINGS))
@pytest.mark.parametrize("layout", [tgo_amd.ROPE_INTERLEAVED, tgo_amd.ROPE_HALF])
@pytest.mark.parametrize("d,rd,T,H,Hkv", [(128, 128, 1, 32, 8), (128, 64, 37, 5, 3), (64, 64, 300, 2, 1),
                                          (80, 20, 65, 3, 1), (96, 96, 9, 24, 8), (256, 256, 130, 4, 2), (2, 2, 3, 1, 1),
                                          (10, 6, 5, 7, 1), (128, 32, 1153, 16, 8)])
def test_rope_over_a_fused_row(ctx, torch_gpu, d, rd, T, H, Hkv, layout, scaling):
    torch = torch_gpu
    g = torch.Generator(device="cuda").manual_seed(d * T + rd)
    row = torch.randn(T, H + 2 * Hkv, d, device="cuda", generator=g)
    pos = torch.randint(-70000, 200000, (T,), device="cuda", generator=g, dtype=torch.int32)
    w, m = tgo_amd.rope_freqs(d, 1e6, rotary_dim=rd, layout=layout, **SCALINGS[scaling])
    h = ctx.rope_new(d, 1e6, rotary_dim=rd, layout=layout, **SCALINGS[scaling])
    try:
        q = torch.full((T, H, d), float("nan"), device="cuda")
        k = torch.full((T, Hkv, d), float("nan"), device="cuda", dtype=torch.float16)
        v = torch.full((T, Hkv, d), float("nan"), device="cuda", dtype=torch.float16)
        xq, xk, xv = row[:, :H], row[:, H:H + Hkv], row[:, H + Hkv:]
        ctx.rope(h, pos, [(xq, q), (xk, k), (xv, v, False)])
        torch.cuda.synchronize()
        check_rope(torch, q, xq, pos, rd, layout, w, m)
        check_rope(torch, k, xk, pos, rd, layout, w, m)
        assert torch.equal(v, xv.half())
        # in place, f16, and apart: the same bits
        f = row.half()
        apart = torch.empty_like(f)
        ctx.rope(h, pos, [(f, apart)])
        ctx.rope(h, pos, [(f[:, :H], f[:, :H]), (f[:, H:], f[:, H:])])
        torch.cuda.synchronize()
        check_rope(torch, apart, row.half(), pos, rd, layout, w, m)
        assert torch.equal(f, apart)
    finally:
        ctx.rope_free(h)


@pytest.mark.parametrize("layout", [tgo_amd.ROPE_INTERLEAVED, tgo_amd.ROPE_HALF])
def test_rope_strides_orders_and_alignments(ctx, torch_gpu, layout):
    """Heads-major order, rows and heads apart by odd distances, starts off 16 bytes, one row or head
    read by all: the values of the dense call, to the bit, and nothing outside y written."""
    torch = torch_gpu
    T, H, d, rd = 33, 6, 64, 48
    w, m = tgo_amd.rope_freqs(d, 1e4, rotary_dim=rd, layout=layout)
    h = ctx.rope_new(d, 1e4, rotary_dim=rd, layout=layout)
    pos = torch.arange(T, device="cuda", dtype=torch.int32) * 977
    try:
        for xt in (torch.float32, torch.float16):
            for yt in (torch.float32, torch.float16):
                x = torch.randn(T, H, d, device="cuda").to(xt)
                dense = torch.empty(T, H, d, device="cuda", dtype=yt)
                ctx.rope(h, pos, [(x, dense)])
                check_rope(torch, dense, x, pos, rd, layout, w, m)
                for off, pad, order in ((0, 0, "hm"), (1, 3, "rm"), (2, 6, "rm"), (5, 1, "hm"), (4, 8, "rm")):
                    shape = (T, H, d + pad) if order == "rm" else (H, T, d + pad)

                    def strided(ty):
                        buf = torch.full((off + math.prod(shape),), -7.0, device="cuda", dtype=ty)
                        t = buf[off:].view(shape)[..., :d]
                        return buf, t if order == "rm" else t.transpose(0, 1)
                    _, xs = strided(xt)
                    xs.copy_(x)
                    buf, ys = strided(yt)
                    ctx.rope(h, pos, [(xs, ys)])
                    torch.cuda.synchronize()
                    assert torch.equal(ys, dense), (xt, yt, off, pad, order)
                    ys.fill_(-7.0)
                    assert bool((buf == -7.0).all())
        x = torch.randn(1, 1, d, device="cuda").expand(T, H, d)
        y = torch.empty(T, H, d, device="cuda")
        ctx.rope(h, pos, [(x, y)])
        check_rope(torch, y, x, pos, rd, layout, w, m)
    finally:
        ctx.rope_free(h)


@pytest.mark.parametrize("T,heads", [(20000, 1), (3000, 3), (2, 65536), (5000, 13)])
def test_rope_heads_and_rows_of_a_workgroup(ctx, torch_gpu, T, heads):
    torch = torch_gpu
    d = 8 if heads > 1000 else 64
    h = ctx.rope_new(d, 1e4, layout=tgo_amd.ROPE_HALF)
    try:
        w, m = tgo_amd.rope_freqs(d, 1e4)
        x = torch.randn(T, heads, d, device="cuda").half()
        pos = torch.randint(0, 100000, (T,), device="cuda", dtype=torch.int32)
        y = torch.full_like(x, float("nan"))
        ctx.rope(h, pos, [(x, y)])
        check_rope(torch, y, x, pos, d, tgo_amd.ROPE_HALF, w, m)
    finally:
        ctx.rope_free(h)


def test_rope_far_positions(ctx, torch_gpu):
    torch = torch_gpu
    pos = torch.tensor([0, 1, -1, 2 ** 31 - 1, -2 ** 31, 131071, 10 ** 9], dtype=torch.int32, device="cuda")
    h = ctx.rope_new(128, 1e6)
    try:
        w, m = tgo_amd.rope_freqs(128, 1e6)
        x = torch.randn(7, 4, 128, device="cuda")
        y = torch.empty_like(x)
        ctx.rope(h, pos, [(x, y)])
        check_rope(torch, y, x, pos, 128, tgo_amd.ROPE_INTERLEAVED, w, m)
        assert torch.equal(y[0], x[0])
    finally:
        ctx.rope_free(h)


def test_rope_nonfinite_values_stay_in_their_pair(ctx, torch_gpu):
    torch = torch_gpu
    h = ctx.rope_new(128, 1e6, rotary_dim=64, layout=tgo_amd.ROPE_HALF)
    try:
        x = torch.randn(5, 2, 128, device="cuda")
        pos = torch.arange(5, device="cuda", dtype=torch.int32)
        y0, y1 = torch.empty_like(x), torch.empty_like(x)
        ctx.rope(h, pos, [(x, y0)])
        x[2, 1, 3] = float("nan")
        x[3, 0, 100] = float("inf")
        ctx.rope(h, pos, [(x, y1)])
        torch.cuda.synchronize()
        same = torch.ones_like(x, dtype=torch.bool)
        same[2, 1, 3] = same[2, 1, 35] = same[3, 0, 100] = False
        assert torch.equal(y0[same], y1[same])
        assert y1[2, 1, 3].isnan() and y1[2, 1, 35].isnan() and y1[3, 0, 100] == float("inf")
    finally:
        ctx.rope_free(h)


def test_rope_refusals(ctx, torch_gpu):
    torch = torch_gpu
    h = ctx.rope_new(64, 1e4)
    L = tgo_amd.lib()
    try:
        x, y = torch.randn(4, 2, 64, device="cuda"), torch.zeros(4, 2, 64, device="cuda")
        pos = torch.zeros(4, device="cuda", dtype=torch.int32)
        xa, ya = x.data_ptr(), y.data_ptr()

        def call(n=1, T=4, p=pos.data_ptr(), handle=h, **kw):
            g = (tgo_amd.RopeHeads * 3)()
            for i in range(3):
                a = dict(x=xa, y=ya, x_row=128, x_head=64, y_row=128, y_head=64, heads=2, x_dtype=0, y_dtype=0, rotate=1)
                a.update(kw)
                for f, v in a.items():
                    setattr(g[i], f, v)
            rc = L.tgohip_rope(ctx.h, handle, p, T, g, n)
            return "" if rc == 0 else tgo_amd.last_error()

        for msg, kw in (("no handle 99999", dict(handle=99999)), ("rows; 0 to", dict(T=-1)), ("rows; 0 to", dict(T=1 << 24)),
                        ("1 to 3", dict(n=0)), ("1 to 3", dict(n=4)), ("positions is a device", dict(p=None)),
                        ("x and y are device", dict(x=None)), ("x and y are device", dict(y=None)), ("0 heads", dict(heads=0)),
                        ("f32 or f16", dict(x_dtype=2)), ("f32 or f16", dict(y_dtype=-1)), ("not aligned", dict(x=xa + 2)),
                        ("not aligned", dict(y=ya + 1)), ("strides are not negative", dict(x_row=-1)),
                        ("strides are not negative", dict(x_head=1 << 41)), ("heads of y overlap", dict(y_head=63)),
                        ("heads of y overlap", dict(y_row=127)), ("heads of y overlap", dict(y_row=0)),
                        ("meets x", dict(y=xa + 4)), ("meets x", dict(y=xa, y_dtype=1)), ("meets x", dict(y=xa, y_row=256)),
                        ("and 1 meet in memory", dict(n=2))):
            assert msg in call(**kw), (msg, kw, tgo_amd.last_error())
        assert call(T=0, p=None) == ""
        torch.cuda.synchronize()
        assert bool((y == 0).all())
        with pytest.raises(TgoError, match="float32 or float16"):
            ctx.rope(h, pos, [(x.bfloat16(), y)])
        with pytest.raises(TgoError, match="tensor 0 is"):
            ctx.rope(h, pos, [(x[:, :, :32], y[:, :, :32])])
        with pytest.raises(TgoError, match="dense head rows"):
            ctx.rope(h, pos, [(x.transpose(1, 2).contiguous().transpose(1, 2), y)])
        with pytest.raises(TgoError, match="positions is int32"):
            ctx.rope(h, pos.long(), [(x, y)])
    finally:
        ctx.rope_free(h)
    with pytest.raises(TgoError, match="no handle"):
        ctx.rope_free(h)


# ---------------------------------------------------------------------------
# packed attention
# ---------------------------------------------------------------------------

def attention64(torch, q, k, v, nq, nk, scale, causal):
    """(output, tolerance of an f32 result before its own rounding) in float64."""
    H, d = q.shape[1:]
    G = H // k.shape[1]
    f16 = q.dtype == torch.float16
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    tq = tk = 0
    for n, m in zip(nq, nk):
        for i0 in range(0, n if m else 0, 1024):
            i1 = min(n, i0 + 1024)
            qs = q[tq + i0:tq + i1].double()
            ks, vs = k[tk:tk + m].double(), v[tk:tk + m].double()
            for h in range(H):
                kh, vh = ks[:, h // G], vs[:, h // G]
                s = scale * (qs[:, h] @ kh.t())
                seen = torch.ones_like(s, dtype=torch.bool)
                if causal:
                    seen = torch.arange(m, device=q.device)[None] <= torch.arange(m - n + i0, m - n + i1, device=q.device)[:, None]
                s = s.masked_fill(~seen, -math.inf)
                top = s.max(1, keepdim=True)[0]
                live = seen.any(1, keepdim=True)
                p = torch.where(seen, (s - torch.where(live, top, 0.0)).exp(), 0.0)
                l = p.sum(1, keepdim=True).clamp_min(1e-300)
                o = p @ vh / l
                out[tq + i0:tq + i1, h] = torch.where(live, o, 0.0)
                # relative error of a probability: its score's (the operands' pairs, d terms summed, the
                # scaling and subtraction in log2 units up to |s| 1.45 each), the exponential's 2^-23 and the
                # rounding to f16 (or a pair)
                mag = scale * (qs[:, h].abs() @ kh.abs().t())
                ds = ((0 if f16 else 2.0 ** -22) + 4 * math.sqrt(d) * U) * mag + 3 * U * 1.45 * (s.abs() + top.abs())
                e = torch.where(seen, p * (ds + 2.0 ** -23 + (HALF if f16 else 2.0 ** -22)), 0.0)
                # an f16 probability's absolute floor (2^-32 of the largest), the f32 sums
                e = e + seen * 2.0 ** -32 + p * 4 * math.sqrt(m) * U
                bound = (e @ vh.abs() + (e.sum(1, keepdim=True) / l) * (p @ vh.abs())) / l
                tol[tq + i0:tq + i1, h] = torch.where(live, bound, 0.0)
        tq, tk = tq + n, tk + m
    return out, tol


def attend(ctx, torch, q, k, v, nq, nk, causal=True, out=None, scale=None, plan=0, free=True):
    H, d = q.shape[1:]
    plan = ctx.packed_plan(nq, nk, H, k.shape[1], head_dim=d, causal=causal,
                           q_dtype=tgo_amd.F16 if q.dtype == torch.float16 else tgo_amd.F32, plan=plan)
    if out is None:
        out = torch.full(q.shape, float("nan"), device="cuda", dtype=q.dtype)
    ctx.packed_attention(plan, q, k, v, out, scale or 1 / math.sqrt(d))
    if free:
        ctx.packed_free(plan)
    return out


def inputs(torch, nq, nk, H, Hkv, d, f16, seed=1, spread=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = torch.randn(sum(nq), H, d, device="cuda", generator=g) * spread
    k = torch.randn(sum(nk), Hkv, d, device="cuda", generator=g).half()
    v = torch.randn(sum(nk), Hkv, d, device="cuda", generator=g).half()
    return (q.half() if f16 else q), k, v


def check_attention(torch, got, q, k, v, nq, nk, causal, scale=None):
    want, tol = attention64(torch, q, k, v, nq, nk, scale or 1 / math.sqrt(q.shape[2]), causal)
    tol = tol + (f16_step(want) if got.dtype == torch.float16 else U * want.abs())
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), (float((err / (tol + 1e-30)).max()), int((~(err <= tol)).sum()))


BATCHES = {
    "one": ([1], [1]), "tiny": ([3, 1, 2], [3, 1, 2]), "edges": ([31, 32, 33, 63, 64, 65], [31, 32, 33, 63, 64, 65]),
    "empty": ([0, 5, 0, 7, 1], [4, 0, 0, 7, 300]), "decode": ([1] * 9, [1, 2, 63, 64, 65, 700, 127, 129, 2049]),
    "few": ([2, 5, 8, 1, 7], [500, 5, 1025, 33, 1000]), "chunks": ([100, 17, 257], [1000, 17, 700]),
    "more_queries": ([50, 130, 3], [20, 1, 2]), "prompt": ([777], [777]), "mixed": ([1, 300, 1, 40], [3000, 300, 64, 2000]),
}


@pytest.mark.parametrize("batch", sorted(BATCHES))
@pytest.mark.parametrize("H,Hkv,d", [(8, 2, 128), (4, 4, 64), (7, 1, 128), (64, 1, 64), (6, 2, 128), (10, 2, 64)])
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("causal", [True, False])
def test_packed_attention(ctx, torch_gpu, batch, H, Hkv, d, f16, causal):
    torch = torch_gpu
    nq, nk = BATCHES[batch]
    q, k, v = inputs(torch, nq, nk, H, Hkv, d, f16)
    out = attend(ctx, torch, q, k, v, nq, nk, causal)
    check_attention(torch, out, q, k, v, nq, nk, causal)


@pytest.mark.parametrize("nq,nk,H,Hkv,d,f16,causal", [
    ([1, 1], [40000, 9000], 32, 8, 128, False, True),    # long contexts of single tokens, split and merged
    ([4], [30011], 16, 2, 64, True, True),
    ([300], [20000], 8, 1, 128, True, True),             # a chunk far behind its keys
    ([64], [16001], 4, 2, 128, False, False),
    ([3000, 1100, 2047], [3000, 1100, 2047], 16, 8, 128, True, True),
    ([2500], [2500], 28, 4, 128, False, True),
    ([1500, 700], [1500, 700], 16, 16, 64, False, False),
])
def test_packed_attention_over_long_contexts(ctx, torch_gpu, nq, nk, H, Hkv, d, f16, causal):
    torch = torch_gpu
    q, k, v = inputs(torch, nq, nk, H, Hkv, d, f16, seed=3)
    out = attend(ctx, torch, q, k, v, nq, nk, causal)
    check_attention(torch, out, q, k, v, nq, nk, causal)
    again = attend(ctx, torch, q, k, v, nq, nk, causal)
    torch.cuda.synchronize()
    assert torch.equal(out, again)


@pytest.mark.parametrize("seed", range(12))
def test_packed_attention_over_random_batches(ctx, torch_gpu, seed):
    """Batches of single tokens, chunks and prompts, cut, merged and whole, both kernels in one call."""
    torch = torch_gpu
    r = np.random.default_rng(seed)
    n = int(r.integers(2, 14))
    nk = [int(x) for x in np.exp(r.uniform(0, math.log(9000), n))]
    nq = [int(r.choice([0, 1, 1, 2, r.integers(1, 9), r.integers(1, min(600, k) + 1)])) for k in nk]
    H, Hkv, d = [(32, 8, 128), (14, 2, 64), (8, 8, 128), (12, 1, 64)][seed % 4]
    f16, causal = bool(seed & 1), seed % 3 != 0
    print("packed: %s over %s, %d/%d heads of %d" % (nq, nk, H, Hkv, d), flush=True)
    q, k, v = inputs(torch, nq, nk, H, Hkv, d, f16, seed=seed)
    out = attend(ctx, torch, q, k, v, nq, nk, causal)
    check_attention(torch, out, q, k, v, nq, nk, causal)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("d", [64, 128])
def test_packed_attention_with_peaked_scores(ctx, torch_gpu, f16, d):
    """Scores of some tens: the largest key anywhere, rising and falling along the context, and one
    scale that makes every probability but one vanish."""
    torch = torch_gpu
    nq, nk = [200, 1, 6], [200, 1500, 900]
    q, k, v = inputs(torch, nq, nk, 4, 2, d, f16, seed=5, spread=4.0)
    slope = torch.linspace(0.2, 3.0, sum(nk), device="cuda")[:, None, None]
    for keys in (k, (k * slope).half(), (k * slope.flip(0)).half()):
        for scale in (1 / math.sqrt(d), 0.5):
            out = attend(ctx, torch, q, keys, v, nq, nk, True, scale=scale)
            check_attention(torch, out, q, keys, v, nq, nk, True, scale)


@pytest.mark.parametrize("q_f16", [False, True])
def test_packed_outputs_in_every_type(ctx, torch_gpu, q_f16):
    """An f16 result and a pair's planes are the f32 result, rounded."""
    torch = torch_gpu
    nq, nk = [70, 1, 5], [70, 3000, 40]
    q, k, v = inputs(torch, nq, nk, 8, 2, 128, q_f16)
    f32 = attend(ctx, torch, q, k, v, nq, nk, out=torch.full(q.shape, float("nan"), device="cuda"))
    f16 = attend(ctx, torch, q, k, v, nq, nk, out=torch.full(q.shape, float("nan"), device="cuda", dtype=torch.float16))
    pair = attend(ctx, torch, q, k, v, nq, nk, out=torch.full((2,) + q.shape, float("nan"), device="cuda", dtype=torch.float16))
    torch.cuda.synchronize()
    assert torch.equal(f16, f32.half()) and torch.equal(pair[0], f32.half())
    assert torch.equal(pair[1], (f32 - f32.half().float()).half())


@pytest.mark.parametrize("q_f16", [False, True])
@pytest.mark.parametrize("d", [64, 128])
def test_packed_rows_of_wider_buffers(ctx, torch_gpu, q_f16, d):
    """q, k, v and out as columns of wider rows; what lies between and behind the rows stays."""
    torch = torch_gpu
    nq, nk, H, Hkv = [40, 1, 9], [90, 1800, 9], 6, 2
    q, k, v = inputs(torch, nq, nk, H, Hkv, d, q_f16)
    dense = attend(ctx, torch, q, k, v, nq, nk)

    def wide(t, extra, rows=0):
        buf = torch.full((t.shape[0] + rows, t.shape[1] + extra, d), 3.0, device="cuda", dtype=t.dtype)
        buf[:t.shape[0], 1:1 + t.shape[1]] = t
        return buf, buf[:t.shape[0], 1:1 + t.shape[1]]
    _, qs = wide(q, 3)
    kv = torch.full((k.shape[0], 3 * Hkv, d), float("nan"), device="cuda", dtype=torch.float16)
    kv[:, :Hkv], kv[:, 2 * Hkv:] = k, v
    buf, out = wide(torch.full_like(dense, 3.0), 2, rows=5)
    attend(ctx, torch, qs, kv[:, :Hkv], kv[:, 2 * Hkv:], nq, nk, out=out)
    torch.cuda.synchronize()
    assert torch.equal(out, dense)
    out.fill_(3.0)
    assert bool((buf == 3.0).all())


@pytest.mark.parametrize("q_f16", [False, True])
@pytest.mark.parametrize("H,Hkv,d,nq,nk", [(8, 2, 128, [130, 5, 1, 64], [130, 70, 900, 64]), (3, 3, 64, [90, 33], [90, 33]),
                                           (2, 1, 128, [3, 1], [2500, 4000])])
def test_nothing_unseen_reaches_a_row(ctx, torch_gpu, H, Hkv, d, q_f16, nq, nk):
    """NaN and infinities in rows behind the sequences, in other sequences' rows and in later tokens'
    keys and values leave every row that does not see them as it was, to the bit; rows that see a value
    get it."""
    torch = torch_gpu
    q, k, v = inputs(torch, nq, nk, H, Hkv, d, q_f16)
    pad = torch.full((128, Hkv, d), float("nan"), device="cuda", dtype=torch.float16)
    kp, vp = torch.cat([k, pad]), torch.cat([v, -pad / 0])
    clean = attend(ctx, torch, q, kp[:len(k)], vp[:len(v)], nq, nk)
    tk = tq = 0
    for n, m in zip(nq, nk):
        for at, bad in ((m - 1, float("nan")), (m - max(1, n // 2), float("inf")), (m - n, float("-inf"))):
            for what in "kv":
                kb, vb = kp.clone(), vp.clone()
                (kb if what == "k" else vb)[tk + at, :, 3] = bad
                out = attend(ctx, torch, q, kb[:len(k)], vb[:len(v)], nq, nk)
                torch.cuda.synchronize()
                sees = torch.zeros(len(q), dtype=torch.bool, device="cuda")
                first = tq + max(0, at - (m - n))  # the first query at position `at` or later
                sees[first:tq + n] = True
                assert torch.equal(out[~sees], clean[~sees]), (m, at, bad, what)
                if what == "v":
                    hit = out[sees][..., 3]
                    # a pair's product with an infinity may be NaN (its lo part is 0 or of the other sign)
                    good = hit.isnan() if bad != bad else (hit == bad) | (hit.isnan() & (not q_f16))
                    assert bool(good.all()), (m, at, bad)
                    keep = [j for j in range(d) if j != 3]
                    assert torch.equal(out[sees][..., keep], clean[sees][..., keep])
                elif bad != bad:
                    assert bool(out[sees].isnan().all())
        tq, tk = tq + n, tk + m


def test_packed_offsets_past_32_bits(ctx, torch_gpu):
    """Key rows a megabyte apart: the last lie beyond 4 GiB (and 2^31 elements) of the first."""
    torch = torch_gpu
    nq, nk, H, Hkv, d = [1, 40], [2900, 1400], 4, 2, 128
    q, k, v = inputs(torch, nq, nk, H, Hkv, d, False)
    dense = attend(ctx, torch, q, k, v, nq, nk)
    buf = torch.empty(sum(nk), 1 << 19, device="cuda", dtype=torch.float16)
    ks, vs = buf[:, 256:512].view(-1, Hkv, d), buf[:, 1024:1280].view(-1, Hkv, d)
    ks.copy_(k)
    vs.copy_(v)
    out = attend(ctx, torch, q, ks, vs, nq, nk)
    torch.cuda.synchronize()
    assert torch.equal(out, dense)


def test_packed_plans_are_replaced_and_shared_by_layers(ctx, torch_gpu):
    torch = torch_gpu
    H, Hkv, d = 8, 2, 128
    plan, queued = 0, []
    for i, (nq, nk) in enumerate([([1] * 4, [500, 6000, 9, 40]), ([300], [300]), ([], []), ([2, 3], [2000, 7])]):
        layers = [inputs(torch, nq, nk, H, Hkv, d, False, seed=10 * i + l) for l in range(2)]
        plan = ctx.packed_plan(nq, nk, H, Hkv, plan=plan)
        for q, k, v in layers:
            out = torch.full(q.shape, float("nan"), device="cuda")
            ctx.packed_attention(plan, q, k, v, out, 0.1)
            queued.append((out, q, k, v, nq, nk))
    ctx.packed_free(plan)
    torch.cuda.synchronize()
    for out, q, k, v, nq, nk in queued:
        if len(q):
            check_attention(torch, out, q, k, v, nq, nk, True, 0.1)


def test_packed_attention_refusals(ctx, torch_gpu):
    torch = torch_gpu
    L = tgo_amd.lib()
    nq, nk, H, Hkv, d = [4, 3], [10, 3], 4, 2, 64
    q, k, v = inputs(torch, nq, nk, H, Hkv, d, False)
    out = torch.full_like(q, 5.0)
    plan = ctx.packed_plan(nq, nk, H, Hkv, head_dim=d)
    try:
        def call(handle=plan, q=q.data_ptr(), q_row=256, k=k.data_ptr(), k_row=128, v=v.data_ptr(), v_row=128, scale=0.1,
                 out=out.data_ptr(), out_row=256, out_dtype=0):
            rc = L.tgohip_packed_attention(ctx.h, handle, q, q_row, k, k_row, v, v_row, scale, out, out_row, out_dtype)
            return "" if rc == 0 else tgo_amd.last_error()
        for msg, kw in (("no handle 4444", dict(handle=4444)), ("scale is 0", dict(scale=0.0)), ("scale is -1", dict(scale=-1.0)),
                        ("scale is nan", dict(scale=float("nan"))), ("scale is inf", dict(scale=float("inf"))),
                        ("out_dtype is 3", dict(out_dtype=3)), ("q and out are device", dict(q=None)),
                        ("q and out are device", dict(out=None)), ("k and v are device", dict(v=None)),
                        ("q rows are 255", dict(q_row=255)), ("k rows are 16777224", dict(k_row=(1 << 24) + 8)), ("k rows are 64", dict(k_row=64)), ("v rows are -128", dict(v_row=-128)),
                        ("out rows are 0", dict(out_row=0)), ("16-byte", dict(q=q.data_ptr() + 4)), ("16-byte", dict(k_row=132)),
                        ("16-byte", dict(out_row=258)), ("rows are dense", dict(out_dtype=2, out_row=264)),
                        ("out meets q", dict(out=q.data_ptr())), ("out meets k", dict(out=k.data_ptr())),
                        ("out meets v", dict(out=v.data_ptr() + 16))):
            assert msg in call(**kw), (msg, kw, tgo_amd.last_error())
        with pytest.raises(TgoError, match="no handle 777"):
            ctx.packed_plan(nq, nk, H, Hkv, plan=777)
        with pytest.raises(TgoError, match="q is \\[7, 4, 64\\]"):
            ctx.packed_attention(plan, q[:6], k, v, out, 0.1)
        with pytest.raises(TgoError, match="q is float32"):
            ctx.packed_attention(plan, q.half(), k, v, out, 0.1)
        with pytest.raises(TgoError, match="k is float16"):
            ctx.packed_attention(plan, q, k.float(), v, out, 0.1)
        torch.cuda.synchronize()
        assert bool((out == 5.0).all())
    finally:
        ctx.packed_free(plan)
    empty = ctx.packed_plan([], [], H, Hkv, head_dim=d)
    ctx.packed_attention(empty, q[:0], k[:0], v[:0], out[:0], 0.1)
    ctx.packed_free(empty)


# ---------------------------------------------------------------------------
# adapters
# ---------------------------------------------------------------------------

def adapters64(torch, x, base, extents, who, loaded, K, N, x_pair):
    """(y, tolerance before y's own rounding) in float64; loaded: {index: (down, up, scale)}, float64."""
    y = base.double().clone() if base is not None else torch.zeros(sum(extents), N, dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(y)
    at = 0
    for n, a in zip(extents, who):
        if a in loaded and n:
            down, up, s = loaded[a]
            xs = x[at:at + n]
            u = xs @ down.t()
            du = ((2.0 ** -22 if x_pair else 0) + 4 * math.sqrt(K) * U) * (xs.abs() @ down.abs().t())
            top = u.abs().max(1, keepdim=True)[0]
            r = down.shape[0]
            y[at:at + n] += s * (u @ up.t())
            tol[at:at + n] = abs(s) * ((du + (2.0 ** -22) * (top + du)) @ up.abs().t()
                                       + (4 * math.sqrt(r) + 1) * U * (u.abs() @ up.abs().t()))
        at += n
    return y, tol + U * y.abs()


def make_adapter(torch, K, N, r, seed, spread=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    down = (torch.randn(r, K, device="cuda", generator=g) * spread / math.sqrt(K)).half()
    return down, (torch.randn(N, r, device="cuda", generator=g) * 0.05).half()


def stored(torch, x, xk):
    """(the stored activation, its dtype code, its values in float64)"""
    if xk == "f32":
        return x, tgo_amd.F32, x.double()
    hi = x.half()
    if xk == "f16":
        return hi, tgo_amd.F16, hi.double()
    lo = (x - hi.float()).half()
    return torch.stack([hi, lo]), tgo_amd.F16X2, hi.double() + lo.double()


def check_adapters(ctx, torch, K, N, ranks, extents, who, xk, yk, seed=1, base="apart", spread=1.0):
    loaded = {}
    h = ctx.adapters_new(K, N, max([len(ranks)] + [w + 1 for w in who]))
    rows = ctx.adapter_rows(extents, who)
    try:
        for i, r in enumerate(ranks):
            if r:
                down, up = make_adapter(torch, K, N, r, 100 * seed + i, spread)
                s = 0.5 + i
                ctx.adapters_put(h, i, down.cpu().numpy(), up.cpu().numpy(), s)
                loaded[i] = (down.double(), up.double(), s)
        T = sum(extents)
        x, xd, x64 = stored(torch, torch.randn(T, K, device="cuda"), xk)
        yt = torch.float16 if yk == "f16" else torch.float32
        b = torch.randn(T, N, device="cuda").to(yt) if base else None
        # behind the last row stays as it is
        buf = torch.full((T + 3, N), float("nan"), device="cuda", dtype=yt)
        if base == "same":
            buf[:T] = b
        buf[T:] = 9.0
        print("adapters: [%d,%d] ranks %s rows %d %s %s" % (K, N, ranks, T, xk, yk), flush=True)
        ctx.adapters(h, rows, x, buf[:T] if base == "same" else b, buf[:T], x_dtype=xd,
                     y_dtype=tgo_amd.F16 if yk == "f16" else tgo_amd.F32)
        torch.cuda.synchronize()
        want, tol = adapters64(torch, x64, b, extents, who, loaded, K, N, xk != "f16")
        if yk == "f16":
            tol = tol + f16_step(want)
        err = (buf[:T].double() - want).abs()
        assert bool((err <= tol).all()), (float((err / (tol + 1e-30)).max()), int((~(err <= tol)).sum()))
        assert bool((buf[T:] == 9.0).all())
        at = 0
        for n, a in zip(extents, who):
            if a not in loaded:
                assert torch.equal(buf[at:at + n], b[at:at + n] if b is not None else torch.zeros_like(buf[at:at + n]))
            at += n
    finally:
        ctx.adapter_rows_free(rows)
        ctx.adapters_free(h)


@pytest.mark.parametrize("xk,yk", [("f32", "f32"), ("x2", "f32"), ("f16", "f16"), ("f32", "f16"), ("f16", "f32")])
@pytest.mark.parametrize("K,N,ranks,extents,who", [
    (64, 32, [1], [1], [0]),
    (64, 32, [5], [70], [0]),
    (4096, 6144, [16, 8, 16], [1] * 13, [0, 1, 2, 2, 1, 0, -1, 0, 0, 0, 2, 1, 0]),
    (1024, 2048, [64, 128, 24, 1], [1, 40, 1, 129, 0, 31, 32, 33], [0, 1, -1, 2, 3, 3, 0, 1]),
    (640, 1056, [20, 0, 48], [17, 65, 3], [2, 1, 0]),
    (12288, 96, [100], [5, 5], [0, 0]),
    (192, 4128, [17], [257], [0]),
    (2048, 1024, [16, 32], [3, 4], [-1, -1]),
])
def test_adapters(ctx, torch_gpu, K, N, ranks, extents, who, xk, yk):
    check_adapters(ctx, torch_gpu, K, N, ranks, extents, who, xk, yk)


@pytest.mark.parametrize("base", ["apart", "same", None])
@pytest.mark.parametrize("yk", ["f32", "f16"])
def test_adapters_bases(ctx, torch_gpu, base, yk):
    check_adapters(ctx, torch_gpu, 256, 160, [8, 40], [9, 1, 50], [0, -1, 1], "f32", yk, base=base)


@pytest.mark.parametrize("spread", [2.0 ** -9, 2.0 ** 9])
def test_adapters_far_from_unit_size(ctx, torch_gpu, spread):
    """x . down^T of 1e-3 and of some thousands (its values as f16 hi + lo parts, scaled per row)."""
    check_adapters(ctx, torch_gpu, 1024, 512, [16, 64], [1, 70, 30], [0, 1, 0], "f32", "f32", spread=spread)


@pytest.mark.parametrize("extents", [[2000, 1, 700], [1] * 300])
def test_adapters_many_rows(ctx, torch_gpu, extents):
    who = [(7 * i) % 40 - 1 for i in range(len(extents))]
    check_adapters(ctx, torch_gpu, 1024, 1536, [8 + i for i in range(39)], extents, who, "x2", "f32")


@pytest.mark.parametrize("xk,yk", [("f32", "f32"), ("x2", "f32"), ("f16", "f16"), ("f32", "f16"), ("f16", "f32")])
@pytest.mark.parametrize("K,N,ranks", [(64, 32, [3, 16]), (192, 96, [30, 9]), (1088, 160, [64, 17, 50]), (4096, 2080, [128, 5, 70])])
def test_adapters_of_large_tiles(ctx, torch_gpu, K, N, ranks, xk, yk):
    """Beyond 512 rows tiles hold up to 64: full ones and ones of 1, 16, 17, 33, 48 and 63 rows, requests
    without an adapter between them, odd numbers of 64-element units in a share of K."""
    extents = [200, 1, 64, 81, 33, 16, 65, 112, 3]
    who = [0, 1, -1, 1, 0, len(ranks) - 1, -1, len(ranks) - 1, 0]
    check_adapters(ctx, torch_gpu, K, N, ranks, extents, who, xk, yk, base="same" if K == 192 else "apart")


def test_adapters_are_replaced_and_dropped(ctx, torch_gpu):
    torch = torch_gpu
    K, N = 256, 128
    h, rows = ctx.adapters_new(K, N, 3), ctx.adapter_rows([4, 3], [2, 0])
    x, base = torch.randn(7, K, device="cuda"), torch.randn(7, N, device="cuda")
    try:
        def run():
            y = torch.full((7, N), float("nan"), device="cuda")
            ctx.adapters(h, rows, x, base, y)
            return y
        assert torch.equal(run(), base)  # no adapter loaded yet
        for r in (16, 40, 3):
            down, up = make_adapter(torch, K, N, r, r)
            ctx.adapters_put(h, 2, down.float().cpu().numpy(), up.float().cpu().numpy(), 2.0)  # f32 planes
            want, tol = adapters64(torch, x.double(), base, [4, 3], [2, 0], {2: (down.double(), up.double(), 2.0)}, K, N, True)
            assert bool(((run().double() - want).abs() <= tol).all())
        ctx.adapters_drop(h, 2)
        assert torch.equal(run(), base)
        rows = ctx.adapter_rows([7], [1], rows=rows)
        down, up = make_adapter(torch, K, N, 8, 8)
        ctx.adapters_put(h, 1, down.cpu().numpy(), up.cpu().numpy(), -1.5)
        want, tol = adapters64(torch, x.double(), base, [7], [1], {1: (down.double(), up.double(), -1.5)}, K, N, True)
        assert bool(((run().double() - want).abs() <= tol).all())
        rows = ctx.adapter_rows([], [], rows=rows)
        ctx.adapters(h, rows, x[:0], base[:0], base[:0])
    finally:
        ctx.adapter_rows_free(rows)
        ctx.adapters_free(h)


def test_adapter_rows_do_not_depend_on_each_other(ctx, torch_gpu):
    """A row's result is the same bits alone, among others and with NaN in every other row."""
    torch = torch_gpu
    K, N = 512, 256
    h = ctx.adapters_new(K, N, 2)
    one, many = ctx.adapter_rows([1], [1]), ctx.adapter_rows([20, 1, 9], [0, 1, 1])
    try:
        for i in range(2):
            down, up = make_adapter(torch, K, N, 16, i)
            ctx.adapters_put(h, i, down.cpu().numpy(), up.cpu().numpy(), 1.0)
        x, base = torch.randn(30, K, device="cuda"), torch.randn(30, N, device="cuda")
        y1, y30, ynan = (torch.empty(n, N, device="cuda") for n in (1, 30, 30))
        ctx.adapters(h, one, x[20:21], base[20:21], y1)
        ctx.adapters(h, many, x, base, y30)
        xb = torch.full_like(x, float("nan"))
        xb[20] = x[20]
        ctx.adapters(h, many, xb, base, ynan)
        torch.cuda.synchronize()
        assert torch.equal(y30[20], ynan[20])
        want, tol = adapters64(torch, x[20:21].double(), base[20:21], [1], [0], {0: (down.double(), up.double(), 1.0)}, K, N, True)
        assert bool(((y1.double() - want).abs() <= tol).all()) and bool(((y30[20:21].double() - want).abs() <= tol).all())
        assert bool(ynan[:20].isnan().all()) and bool(ynan[21:].isnan().all())
    finally:
        for r in (one, many):
            ctx.adapter_rows_free(r)
        ctx.adapters_free(h)


def test_captured_adapters_see_later_puts(ctx, torch_gpu):
    """A replay reads the set as it is then; an adapter beyond the captured rank makes its rows NaN, loudly."""
    torch = torch_gpu
    K, N = 256, 320
    h, rows = ctx.adapters_new(K, N, 2), ctx.adapter_rows([3, 2], [0, 1])
    x, base, y = torch.randn(5, K, device="cuda"), torch.randn(5, N, device="cuda"), torch.zeros(5, N, device="cuda")
    try:
        def put(i, r, seed):
            down, up = make_adapter(torch, K, N, r, seed)
            ctx.adapters_put(h, i, down.cpu().numpy(), up.cpu().numpy(), 1.0)
            return down.double(), up.double(), 1.0
        loaded = {0: put(0, 16, 1), 1: put(1, 30, 2)}
        graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        ctx.adapters(h, rows, x, base, y)
        ctx.set_stream(side.cuda_stream)
        try:
            with torch.cuda.graph(graph, stream=side):
                ctx.adapters(h, rows, x, base, y)
        finally:
            ctx.set_stream(torch.cuda.current_stream().cuda_stream)
        for step in range(3):
            if step:
                loaded[0] = put(0, 32 if step == 1 else 7, 10 + step)
            graph.replay()
            torch.cuda.synchronize()
            want, tol = adapters64(torch, x.double(), base, [3, 2], [0, 1], loaded, K, N, True)
            assert bool(((y.double() - want).abs() <= tol).all())
        ctx.adapters_drop(h, 0)
        put(1, 33, 20)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y[:3], base[:3]) and bool(y[3:].isnan().all())
    finally:
        ctx.adapter_rows_free(rows)
        ctx.adapters_free(h)


def test_adapter_refusals(ctx, torch_gpu):
    torch = torch_gpu
    L, K, N = tgo_amd.lib(), 128, 64
    h, rows, far = ctx.adapters_new(K, N, 2), ctx.adapter_rows([5], [1]), ctx.adapter_rows([5, 0], [2, 1])
    x, b, y = torch.randn(5, K, device="cuda"), torch.randn(5, N, device="cuda"), torch.full((5, N), 4.0, device="cuda")
    try:
        def call(s=h, r=rows, x=x.data_ptr(), xd=0, base=b.data_ptr(), y=y.data_ptr(), yd=0):
            rc = L.tgohip_adapters(ctx.h, s, r, x, xd, base, y, yd)
            return "" if rc == 0 else tgo_amd.last_error()
        for msg, kw in (("set: no handle 9", dict(s=99999)), ("rows: no handle 9", dict(r=99999)), ("x_dtype is 3", dict(xd=3)),
                        ("y_dtype is 2", dict(yd=2)), ("rows name adapter 2 and the set holds 2", dict(r=far)),
                        ("x and y are device", dict(x=None)), ("x and y are device", dict(y=None)),
                        ("16-byte", dict(x=x.data_ptr() + 4)), ("16-byte", dict(base=b.data_ptr() + 8)),
                        ("16-byte", dict(y=y.data_ptr() + 2)), ("y meets x", dict(y=x.data_ptr() + 256)),
                        ("y meets base", dict(y=b.data_ptr() + 16))):
            assert msg in call(**kw), (msg, kw, tgo_amd.last_error())
        down, up = np.zeros((4, K), np.float32), np.zeros((N, 4), np.float32)
        with pytest.raises(TgoError, match="index 2 of a set of 2"):
            ctx.adapters_put(h, 2, down, up, 1.0)
        with pytest.raises(TgoError, match="index -1 of a set"):
            ctx.adapters_drop(h, -1)
        with pytest.raises(TgoError, match="down is"):
            ctx.adapters_put(h, 0, down[:, :64], up, 1.0)
        with pytest.raises(TgoError, match="down is"):
            ctx.adapters_put(h, 0, down, up[:, :3], 1.0)
        with pytest.raises(TgoError, match="past f16's range"):
            ctx.adapters_put(h, 0, down, up + 65536, 1.0)
        torch.cuda.synchronize()
        assert bool((y == 4.0).all())
    finally:
        for r in (rows, far):
            ctx.adapter_rows_free(r)
        ctx.adapters_free(h)


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------

def test_an_attention_block_of_adapted_requests(ctx, torch_gpu):
    """One layer's attention over packed prompts and a decoding request: projection, the requests'
    adapters, rotary positions (scaled, half layout), attention over the rotated rows."""
    torch = torch_gpu
    K, H, Hkv, d = 256, 4, 2, 128
    N = (H + 2 * Hkv) * d
    nq, who = [70, 1, 33, 128], [0, -1, 1, 0]
    T = sum(nq)
    g = torch.Generator(device="cuda").manual_seed(4)
    w = (torch.randn(K, N, device="cuda", generator=g) / 16).half()
    x = torch.randn(T, K, device="cuda", generator=g)
    pos = torch.cat([torch.arange(n) for n in nq]).int().cuda() + 5000
    wh = ctx.weight_upload(tgo_amd.FORM_F16, K, N, w.cpu())
    kw = dict(layout=tgo_amd.ROPE_HALF, **SCALINGS["yarn"])
    rope, s = ctx.rope_new(d, 1e6, **kw), ctx.adapters_new(K, N, 2)
    rows, plan = ctx.adapter_rows(nq, who), ctx.packed_plan(nq, nq, H, Hkv)
    try:
        loaded = {}
        for i, r in enumerate((8, 24)):
            down, up = make_adapter(torch, K, N, r, i)
            ctx.adapters_put(s, i, down.cpu().numpy(), up.cpu().numpy(), 2.0)
            loaded[i] = (down.double(), up.double(), 2.0)
        qkv = torch.empty(T, H + 2 * Hkv, d, device="cuda")
        q = torch.empty(T, H, d, device="cuda")
        k, v = (torch.empty(T, Hkv, d, device="cuda", dtype=torch.float16) for _ in "kv")
        out = torch.empty(T, H, d, device="cuda")

        def layer():
            ctx.linear(wh, x, T, qkv)
            ctx.adapters(s, rows, x, qkv, qkv)
            ctx.rope(rope, pos, [(qkv[:, :H], q), (qkv[:, H:H + Hkv], k), (qkv[:, H + Hkv:], v, False)])
            ctx.packed_attention(plan, q, k, v, out, d ** -0.5)
        layer()
        torch.cuda.synchronize()
        # each stage against float64 of what the stage before left, then the attention
        want, tol = adapters64(torch, x.double(), (x.double() @ w.double()), nq, who, loaded, K, N, True)
        lin = (4 * math.sqrt(K) * U + 2.0 ** -22) * (x.double().abs() @ w.double().abs())
        assert bool(((qkv.view(T, N).double() - want).abs() <= tol + lin + U * want.abs()).all())
        fr, m = tgo_amd.rope_freqs(d, 1e6, **kw)
        check_rope(torch, q, qkv[:, :H], pos, d, tgo_amd.ROPE_HALF, fr, m)
        check_rope(torch, k, qkv[:, H:H + Hkv], pos, d, tgo_amd.ROPE_HALF, fr, m)
        check_attention(torch, out, q, k, v, nq, nq, True)
        # the whole block against float64 throughout: k and v are rounded to f16 (2^-11 of scores and
        # values of size 1 to 10), everything else far below
        w64 = want.view(T, H + 2 * Hkv, d)
        q64, _ = rope64(torch, w64[:, :H], pos, d, tgo_amd.ROPE_HALF, fr, m)
        k64, _ = rope64(torch, w64[:, H:H + Hkv], pos, d, tgo_amd.ROPE_HALF, fr, m)
        v64 = w64[:, H + Hkv:]
        full, _ = attention64(torch, q64, k64, v64, nq, nq, d ** -0.5, True)
        shift = HALF * d ** -0.5 * float(q64.abs().sum(-1).max() * k64.abs().max())  # of a score, by k's rounding
        assert float((out.double() - full).abs().max()) <= (2.1 * shift + 1.1 * HALF) * float(v64.abs().max())
        # captured once and replayed: the eager bits, other calls between the replays
        eager = out.clone()
        graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        ctx.set_stream(side.cuda_stream)
        try:
            torch.cuda.synchronize()
            with torch.cuda.graph(graph, stream=side):
                ctx.rope(rope, pos, [(qkv[:, :H], q), (qkv[:, H:H + Hkv], k), (qkv[:, H + Hkv:], v, False)])
                ctx.packed_attention(plan, q, k, v, out, d ** -0.5)
        finally:
            ctx.set_stream(torch.cuda.current_stream().cuda_stream)
        for _ in range(4):
            for t in (q, k, v, out):
                t.fill_(float("nan"))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, eager)
            layer()
            torch.cuda.synchronize()
    finally:
        ctx.weight_free(wh)
        ctx.rope_free(rope)
        ctx.adapters_free(s)
        ctx.adapter_rows_free(rows)
        ctx.packed_free(plan)


def test_captured_adapters_and_split_attention_replay(ctx, torch_gpu):
    """Both kernels of the adapters and a context split over many workgroups, captured; a second plan and
    row handle run eagerly between the replays."""
    torch = torch_gpu
    K, N, H, Hkv, d = 1024, 512, 8, 2, 128
    nq, nk, who = [1, 1, 1], [6000, 90, 3000], [0, 1, 0]
    q, k, v = inputs(torch, nq, nk, H, Hkv, d, False)
    x, base = torch.randn(3, K, device="cuda"), torch.randn(3, N, device="cuda")
    s = ctx.adapters_new(K, N, 2)
    rows, rows2 = ctx.adapter_rows([1] * 3, who), ctx.adapter_rows([3], [1])
    plan, plan2 = ctx.packed_plan(nq, nk, H, Hkv), ctx.packed_plan([3], [500], H, Hkv)
    try:
        for i in range(2):
            down, up = make_adapter(torch, K, N, 16, i)
            ctx.adapters_put(s, i, down.cpu().numpy(), up.cpu().numpy(), 1.0)
        y, out, y2, out2 = torch.empty_like(base), torch.empty_like(q), torch.empty_like(base), torch.empty_like(q)

        def run():
            ctx.adapters(s, rows, x, base, y)
            ctx.packed_attention(plan, q, k, v, out, 0.09)
        run()
        torch.cuda.synchronize()
        ey, eo = y.clone(), out.clone()
        graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        ctx.set_stream(side.cuda_stream)
        try:
            with torch.cuda.graph(graph, stream=side):
                run()
        finally:
            ctx.set_stream(torch.cuda.current_stream().cuda_stream)
        for _ in range(4):
            y.fill_(float("nan"))
            out.fill_(float("nan"))
            graph.replay()
            ctx.adapters(s, rows2, x, base, y2)
            ctx.packed_attention(plan2, q, k[:500], v[:500], out2, 0.09)
            torch.cuda.synchronize()
            assert torch.equal(y, ey) and torch.equal(out, eo)
    finally:
        for f, a in ((ctx.adapters_free, s), (ctx.adapter_rows_free, rows), (ctx.adapter_rows_free, rows2),
                     (ctx.packed_free, plan), (ctx.packed_free, plan2)):
            f(a)


def test_rotary_and_adapter_offsets_past_32_bits(ctx, torch_gpu):
    """More than 2^31 elements of heads, of x and of y: the last rows are right, and the first ones too."""
    torch = torch_gpu
    T, K, r = 140000, 16384, 4
    assert T * K > 2 ** 31
    buf = torch.zeros(T, K, device="cuda", dtype=torch.float16)
    x = torch.zeros_like(buf)
    at = torch.tensor([0, 1, 77777, T - 65, T - 2, T - 1], device="cuda")
    g = torch.Generator(device="cuda").manual_seed(3)
    x[at] = torch.randn(len(at), K, device="cuda", generator=g).half()
    buf[at] = torch.randn(len(at), K, device="cuda", generator=g).half()
    base = buf[at].double()
    down, up = make_adapter(torch, K, K, r, 5)
    s, rows, h = ctx.adapters_new(K, K, 1), ctx.adapter_rows([T], [0]), ctx.rope_new(128, 1e4, layout=tgo_amd.ROPE_HALF)
    try:
        ctx.adapters_put(s, 0, down.cpu().numpy(), up.cpu().numpy(), 1.5)
        print("adapters: %d rows of [%d, %d]" % (T, K, K), flush=True)
        ctx.adapters(s, rows, x, buf, buf, x_dtype=tgo_amd.F16, y_dtype=tgo_amd.F16)
        torch.cuda.synchronize()
        loaded = {0: (down.double(), up.double(), 1.5)}
        want, tol = adapters64(torch, x[at].double(), base, [len(at)], [0], loaded, K, K, False)
        assert bool(((buf[at].double() - want).abs() <= tol + f16_step(want)).all())
        assert float(buf.abs().sum(1, dtype=torch.float32).count_nonzero()) == len(at)  # no row but these
        print("rope: %d rows of %d heads" % (T, K // 128), flush=True)
        positions = torch.arange(T, device="cuda", dtype=torch.int32)
        before = x[at].double().reshape(len(at), K // 128, 128)
        heads = x.view(T, K // 128, 128)
        ctx.rope(h, positions, [(heads, heads)])
        torch.cuda.synchronize()
        w, _ = tgo_amd.rope_freqs(128, 1e4, layout=tgo_amd.ROPE_HALF)
        angle = at.double()[:, None] * torch.tensor(w, device="cuda")[None]
        c, sn = angle.cos()[:, None], angle.sin()[:, None]
        a, b = before[..., :64], before[..., 64:]
        want = torch.cat([a * c - b * sn, a * sn + b * c], 2)
        # cos and sin within 2 ulp of 1, two f32 operations, one f16 rounding
        tol = 8 * U * (a.abs() + b.abs()).repeat(1, 1, 2) + f16_step(want)
        assert bool(((heads[at].double() - want).abs() <= tol).all())
    finally:
        for f, a in ((ctx.rope_free, h), (ctx.adapters_free, s), (ctx.adapter_rows_free, rows)):
            f(a)


def test_one_row_of_strange_strides_and_its_refusals(ctx, torch_gpu):
    """A single row's stride says nothing: the pair's lo plane is a row's width behind the hi plane, and the
    check of what it meets goes by that. A scale past 2^32 is refused."""
    torch, L = torch_gpu, tgo_amd.lib()
    H, Hkv, d, nk = 4, 2, 64, 50
    q, k, v = inputs(torch, [1], [nk], H, Hkv, d, False)
    out = torch.full((3, H * d), 5.0, device="cuda", dtype=torch.float16)
    want = attend(ctx, torch, q, k, v, [1], [nk], out=torch.empty_like(q), scale=0.1)
    plan = ctx.packed_plan([1], [nk], H, Hkv, head_dim=d)
    try:
        def call(q=q.data_ptr(), out=out.data_ptr(), out_row=0, scale=0.1):
            rc = L.tgohip_packed_attention(ctx.h, plan, q, -7, k.data_ptr(), 128, v.data_ptr(), 128, scale, out, out_row,
                                           tgo_amd.F16X2)
            return "" if rc == 0 else tgo_amd.last_error()
        joint = torch.zeros(4, H * d, device="cuda")  # q in the place of the lo plane
        for row in (0, -4096, 1 << 40):
            assert "out meets q" in call(q=joint.data_ptr() + 2 * H * d, out=joint.data_ptr(), out_row=row)
            assert call(out_row=row) == ""
            torch.cuda.synchronize()
            pair = out[0].double() + out[1].double()
            # the pair's own rounding: 2^-22 of the value and an f16 step of its lo part
            assert bool(((pair - want.reshape(-1).double()).abs() <= 2.0 ** -22 * want.reshape(-1).double().abs() + 2.0 ** -25).all())
            assert bool((out[2] == 5.0).all())
        assert "at most 2^32" in call(scale=2.0 ** 33)
    finally:
        ctx.packed_free(plan)


def test_operands_of_the_host_and_positions_as_an_output_are_refused(ctx, torch_gpu):
    torch = torch_gpu
    L = tgo_amd.lib()
    h = ctx.rope_new(64, 1e4)
    s, rows, plan = ctx.adapters_new(64, 32, 1), ctx.adapter_rows([2], [0]), ctx.packed_plan([2], [2], 1, 1, head_dim=64)
    try:
        x, pos = torch.zeros(2, 1, 64, device="cuda"), torch.zeros(2, device="cuda", dtype=torch.int32)
        half = x.half()
        buf = torch.zeros(256, device="cuda")
        with pytest.raises(TgoError, match="of the host"):
            ctx.rope(h, pos.cpu(), [(x, x)])
        with pytest.raises(TgoError, match="of the host"):
            ctx.rope(h, pos, [(x.cpu(), x)])
        with pytest.raises(TgoError, match="of the host"):
            ctx.packed_attention(plan, x, half, half.cpu(), torch.zeros_like(x), 0.1)
        with pytest.raises(TgoError, match="of the host"):
            ctx.packed_attention(plan, x, half, half, torch.zeros(2, 2, 1, 64, dtype=torch.float16), 0.1)
        y = torch.zeros(2, 32, device="cuda")
        for bad in (dict(x=x.cpu()), dict(y=y.cpu()), dict(base=y.cpu())):
            with pytest.raises(TgoError, match="of the host"):
                ctx.adapters(s, rows, **dict(dict(x=x, base=y, y=y), **bad))
        # fewer rows than the batch, another type than said
        for bad in (dict(x=x[:1]), dict(y=y[:1]), dict(base=y[:1]), dict(x=half), dict(y=y.half()), dict(x=half, x_dtype=tgo_amd.F16X2),
                    dict(base=y.half(), y_dtype=tgo_amd.F32)):
            with pytest.raises(TgoError, match="2 rows of \\[64, 32\\]"):
                ctx.adapters(s, rows, **dict(dict(x=x, base=y, y=y), **bad))
        g = (tgo_amd.RopeHeads * 1)(tgo_amd.RopeHeads(x.data_ptr(), buf.data_ptr(), 64, 64, 64, 64, 1, 0, 0, 1))
        assert L.tgohip_rope(ctx.h, h, buf.data_ptr() + 4 * 127, 2, g, 1) == tgo_amd.EINVAL
        assert "meets positions" in tgo_amd.last_error()
        assert L.tgohip_rope(ctx.h, h, buf.data_ptr() + 2, 2, g, 1) == tgo_amd.EINVAL
        assert "device buffer of int32" in tgo_amd.last_error()
        assert L.tgohip_rope(ctx.h, h, buf.data_ptr() + 4 * 128, 2, g, 1) == 0
        torch.cuda.synchronize()
    finally:
        for f, a in ((ctx.rope_free, h), (ctx.adapters_free, s), (ctx.adapter_rows_free, rows), (ctx.packed_free, plan)):
            f(a)


def test_handles_are_not_made_or_changed_under_capture(ctx, torch_gpu):
    """Every call that makes, changes or frees a handle is refused while the stream is captured, and the
    capture goes on: the graph holds the calls made between the refusals."""
    torch = torch_gpu
    h = ctx.rope_new(64, 1e4)
    s, rows, plan = ctx.adapters_new(64, 32, 1), ctx.adapter_rows([2], [0]), ctx.packed_plan([2], [2], 1, 1, head_dim=64)
    down, up = np.ones((4, 64), np.float32), np.ones((32, 4), np.float32)
    ctx.adapters_put(s, 0, down, up, 1.0)
    x, pos = torch.randn(2, 1, 64, device="cuda"), torch.arange(2, device="cuda", dtype=torch.int32)
    y, base, out = torch.empty_like(x), torch.randn(2, 32, device="cuda"), torch.empty(2, 32, device="cuda")

    def run():
        ctx.rope(h, pos, [(x, y)])
        ctx.adapters(s, rows, x, base, out)
    try:
        run()
        torch.cuda.synchronize()
        ey, eo = y.clone(), out.clone()
        calls = [lambda: ctx.rope_new(64, 1e4), lambda: ctx.rope_free(h), lambda: ctx.packed_plan([2], [2], 1, 1, head_dim=64),
                 lambda: ctx.packed_plan([2], [2], 1, 1, head_dim=64, plan=plan), lambda: ctx.packed_free(plan),
                 lambda: ctx.adapters_new(64, 32, 1), lambda: ctx.adapters_put(s, 0, down, up, 2.0),
                 lambda: ctx.adapters_drop(s, 0), lambda: ctx.adapters_free(s), lambda: ctx.adapter_rows([2], [0]),
                 lambda: ctx.adapter_rows([1], [0], rows=rows), lambda: ctx.adapter_rows_free(rows)]
        graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        ctx.set_stream(side.cuda_stream)
        try:
            with torch.cuda.graph(graph, stream=side):
                for c in calls[:6]:
                    with pytest.raises(TgoError, match="being captured"):
                        c()
                run()
                for c in calls[6:]:
                    with pytest.raises(TgoError, match="being captured"):
                        c()
        finally:
            ctx.set_stream(torch.cuda.current_stream().cuda_stream)
        for _ in range(3):
            y.fill_(float("nan"))
            out.fill_(float("nan"))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, ey) and torch.equal(out, eo)
    finally:
        for f, a in ((ctx.rope_free, h), (ctx.adapters_free, s), (ctx.adapter_rows_free, rows), (ctx.packed_free, plan)):
            f(a)


# ---------------------------------------------------------------------------
# scores past the steps of f32
# ---------------------------------------------------------------------------

def exact_scores(torch, nq, nk, H, Hkv, d, f16, bases, seed=1):
    """q, k, v whose products are whole numbers below 2^24, exact in f32 in every order: a key's first dim
    (`bases`, of the position in its sequence) sets the size, a small second one the order of the keys, with
    many ties. f32 queries have a lo part."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = torch.zeros(sum(nq), H, d, device="cuda")
    q[..., 0] = 2048 if f16 else 2049
    q[..., 1] = torch.randint(-3, 4, (sum(nq), H), device="cuda", generator=g).float()
    k = torch.zeros(sum(nk), Hkv, d, device="cuda")
    k[..., 0] = torch.cat([bases(m) for m in nk])[:, None]
    k[..., 1] = torch.randint(0, 40, (sum(nk), Hkv), device="cuda", generator=g).float()
    v = torch.randn(sum(nk), Hkv, d, device="cuda", generator=g).half()
    return (q.half() if f16 else q), k.half(), v


def check_exact_scores(torch, got, q, k, v, nq, nk, scale, causal):
    H, d = q.shape[1:]
    G, f16 = H // k.shape[1], q.dtype == torch.float16
    tq = tk = 0
    for n, m in zip(nq, nk):
        for h in range(H):
            s = scale * (q[tq:tq + n, h].double() @ k[tk:tk + m, h // G].double().t())
            seen = torch.ones_like(s, dtype=torch.bool)
            if causal:
                seen = torch.arange(m, device="cuda")[None] <= torch.arange(m - n, m, device="cuda")[:, None]
            s = s.masked_fill(~seen, -math.inf)
            live, top = seen.any(1, keepdim=True), s.amax(1, keepdim=True)
            gap = torch.where(seen, top - s, 0.0)
            p = torch.where(seen, (-gap).exp(), 0.0)
            l = p.sum(1, keepdim=True).clamp_min(1e-300)
            vh = v[tk:tk + m, h // G].double()
            want = torch.where(live, p @ vh / l, 0.0)
            # An exponent is the exact score less the reference: log2(e) scale is rounded twice (2 U of the gap),
            # the difference and its rest once each (U of themselves, the rest at most U |top|), as often as the
            # reference moves or parts are merged; past 2^32 two scores are equal or 2^9 apart and more, and the
            # rest is the same for equal ones. exp2 and few more steps: 64 U.
            rest = torch.where(top.abs() < 2.0 ** 32, 16 * U * U * 1.45 * top.abs(), 0.0)
            e = p * (8 * U * gap.clamp_max(200.0) + torch.where(live, rest, 0.0) + 64 * U + (HALF if f16 else 2.0 ** -22)
                     + 4 * math.sqrt(m) * U) + seen * (p < 1) * 2.0 ** -25
            tol = (e @ vh.abs() + (e.sum(1, keepdim=True) / l) * (p @ vh.abs())) / l
            out = got[tq:tq + n, h].double()
            tol = tol + (f16_step(want) if got.dtype == torch.float16 else U * want.abs())
            err = (out - want).abs()
            assert bool((err <= torch.where(live, tol, 0.0)).all()), (n, m, h, scale, int((~(err <= tol)).any(1).sum()),
                                                                      int(out.isnan().any(1).sum()), int((out == 0).all(1).sum()))
        tq, tk = tq + n, tk + m


LARGE = {"few": ([1, 1, 2], [64, 700, 131]), "tiles": ([200, 64, 33], [200, 300, 33]), "merged": ([1, 3], [30000, 9000]),
         "cut": ([100], [12000])}


@pytest.mark.parametrize("form", sorted(LARGE))
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("f16", [False, True])
def test_packed_attention_with_scores_past_f32_steps(ctx, torch_gpu, f16, d, form):
    """Scores of 2^20 to 2^54 in log2 units, where neighbouring f32 are up to 2^31 apart: the largest key,
    and the keys that tie with it, take all there is. Constant size, rising and falling along the context,
    and far below 0."""
    torch = torch_gpu
    nq, nk = LARGE[form]
    flat = lambda m: torch.full((m,), 2048.0, device="cuda")
    steps = lambda m: (torch.arange(m, device="cuda") * 8 // m).float() * 256
    for bases in (flat, lambda m: -flat(m), steps, lambda m: steps(m).flip(0), lambda m: steps(m) - 2048):
        q, k, v = exact_scores(torch, nq, nk, 4, 2, d, f16, bases)
        for bits in (20, 23, 25, 27, 28, 29, 31, 36, 46, 54):
            scale = float(np.float32(2.0 ** (bits - 22) / 1.44))
            out = attend(ctx, torch, q, k, v, nq, nk, True, out=torch.full(q.shape, float("nan"), device="cuda"), scale=scale)
            check_exact_scores(torch, out, q, k, v, nq, nk, scale, True)


@pytest.mark.parametrize("form", sorted(LARGE))
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("size,scale", [(1.0, 2.0 ** 24), (1.0, 2.0 ** 28), (60000.0, 128 ** -0.5), (60000.0, 2.0 ** 32)])
def test_packed_attention_over_the_whole_range_of_scores(ctx, torch_gpu, size, scale, f16, form):
    """Whatever the size of finite queries, keys and scale, a row is the value of its leading key where that
    leads by more than the products' own error, and lies among its values where it does not."""
    torch = torch_gpu
    nq, nk = LARGE[form]
    d, H, Hkv = 128, 4, 2
    g = torch.Generator(device="cuda").manual_seed(9)
    make = (lambda *s: torch.randn(*s, device="cuda", generator=g)) if size == 1 else (
        lambda *s: (torch.rand(*s, device="cuda", generator=g) * 2 - 1) * size)
    q, k, v = make(sum(nq), H, d), make(sum(nk), Hkv, d).half(), torch.randn(sum(nk), Hkv, d, device="cuda", generator=g).half()
    q = q.half() if f16 else q
    out = attend(ctx, torch, q, k, v, nq, nk, True, out=torch.full(q.shape, float("nan"), device="cuda"), scale=scale)
    led = tq = tk = 0
    for n, m in zip(nq, nk):
        seen = torch.arange(m, device="cuda")[None] <= torch.arange(m - n, m, device="cuda")[:, None]
        for h in range(H):
            qh, kh, vh = q[tq:tq + n, h].double(), k[tk:tk + m, h // 2].double(), v[tk:tk + m, h // 2].double()
            s = (qh @ kh.t()).masked_fill(~seen, -math.inf)
            off = (2.0 ** -22 + 4 * math.sqrt(d) * U) * (qh.abs() @ kh.abs().t()).amax(1)
            two = s.topk(min(2, m), 1).values
            got = out[tq:tq + n, h].double()
            lead = (two[:, 0] - two[:, -1] > 2 * off + 60 / scale) | (seen.sum(1) == 1)
            want = vh[s.argmax(1)]
            # the probability and its sum as pairs, or as the same f16, and the division
            assert bool(((got - want).abs() <= 2.0 ** -20 * want.abs() + 2.0 ** -30)[lead].all()), (n, m, h)
            lo = torch.where(seen[:, :, None], vh[None], math.inf).amin(1) if n * m < 1 << 16 else vh.amin(0)
            hi = torch.where(seen[:, :, None], vh[None], -math.inf).amax(1) if n * m < 1 << 16 else vh.amax(0)
            assert bool(((got >= lo - 2.0 ** -8) & (got <= hi + 2.0 ** -8)).all()), (n, m, h)
            led += int(lead.sum())
        tq, tk = tq + n, tk + m
    assert led > 0.8 * sum(nq) * H


@pytest.mark.parametrize("form", sorted(LARGE))
@pytest.mark.parametrize("f16", [False, True])
def test_rows_whose_keys_all_score_minus_infinity(ctx, torch_gpu, f16, form):
    """The softmax of scores that are all -inf is NaN, that of no scores is a row of zeros, and some of -inf
    count nothing beside finite ones."""
    torch = torch_gpu
    nq, nk = LARGE[form]
    nq, nk = nq + [5], nk + [3]  # two queries that see no key
    q, k, v = inputs(torch, nq, nk, 4, 2, 64, f16)
    q[..., 0] = 1 if f16 else 1 + 2.0 ** -12  # the lo part is not 0: 0 times -inf would be NaN
    part, rest = k.clone(), torch.ones(len(k), dtype=torch.bool, device="cuda")
    at = 0
    for m in nk:
        part[at + m // 3:at + m, :, 0] = float("-inf")
        rest[at + m // 3:at + m] = False
        at += m
    whole = k.clone()
    whole[..., 0] = float("-inf")
    out = attend(ctx, torch, q, whole, v, nq, nk)
    none = torch.zeros(len(q), dtype=torch.bool, device="cuda")
    none[sum(nq) - 5:sum(nq) - 3] = True
    assert bool((out[none] == 0).all()) and bool(out[~none].isnan().all())
    # the same rows over the keys that are left: as many as each query sees of them
    out = attend(ctx, torch, q, part, v, nq, nk, False)
    want = [m // 3 for m in nk]
    short = attend(ctx, torch, q, k[rest].contiguous(), v[rest].contiguous(), nq, want, False)
    live = torch.cat([torch.full((n,), m > 0, device="cuda") for n, m in zip(nq, want)])
    both = 2.0 ** -9 if f16 else 2.0 ** -18  # other tiles and cuts: a few roundings of probabilities and sums each
    assert bool(((out - short).abs()[live] <= both * v.abs().max()).all())


@pytest.mark.parametrize("form", sorted(LARGE))
@pytest.mark.parametrize("f16", [False, True])
def test_rows_of_large_scores_leave_the_rows_beside_them_alone(ctx, torch_gpu, f16, form):
    """Every other row's scores are of 2^30, those of the rows between are ordinary, and keep their bits; so do
    all of them beside a value that is not finite and that they do not see."""
    torch = torch_gpu
    nq, nk = LARGE[form]
    q, k, v = inputs(torch, nq, nk, 6, 2, 128, f16)
    q[..., 0] = 0
    k[:, :, 0] = torch.randint(1, 9, k.shape[:2], device="cuda").half() * 4096
    large = q.clone()
    large[:, ::2, 0] = 32768.0
    small = attend(ctx, torch, q, k, v, nq, nk)
    mixed = attend(ctx, torch, large, k, v, nq, nk)
    torch.cuda.synchronize()
    assert torch.equal(mixed[:, 1::2], small[:, 1::2])
    assert not bool(mixed.isnan().any())
    # the first sequence's last key, which its last query sees, and the last one's first, which all of it see
    for at, first, last in ((nk[0] - 1, nq[0] - 1, nq[0]), (sum(nk) - nk[-1], sum(nq) - nq[-1], sum(nq))):
        bad = v.clone()
        bad[at] = float("inf")
        out = attend(ctx, torch, large, k, bad, nq, nk)
        torch.cuda.synchronize()
        assert torch.equal(out[:first], mixed[:first]) and torch.equal(out[last:], mixed[last:])


@pytest.mark.parametrize("q_f16", [False, True])
@pytest.mark.parametrize("d", [64, 128])
def test_few_rows_again_over_every_number_of_tiles(ctx, torch_gpu, q_f16, d):
    """The few-row kernel's repeats for values that are not finite, over contexts of one to eight tiles a wave:
    each run over the keys starts in the buffer that the one before may have ended in."""
    torch = torch_gpu
    nk = [5, 32, 33, 64, 65, 96, 97, 130, 161, 200, 260, 330, 420, 500]
    nq = [5] * len(nk)
    q, k, v = inputs(torch, nq, nk, 4, 1, d, q_f16)
    clean = attend(ctx, torch, q, k, v, nq, nk)
    last = torch.tensor(nk, device="cuda").cumsum(0) - 1
    sees = (torch.arange(1, len(nk) + 1, device="cuda") * 5) - 1
    for value in (float("nan"), float("inf"), float("-inf")):
        bad = v.clone()
        bad[last, :, 7] = value
        for _ in range(3):
            out = attend(ctx, torch, q, k, bad, nq, nk)
            torch.cuda.synchronize()
            keep = torch.ones(len(q), dtype=torch.bool, device="cuda")
            keep[sees] = False
            assert torch.equal(out[keep], clean[keep])
            rest = [j for j in range(d) if j != 7]
            assert torch.equal(out[sees][..., rest], clean[sees][..., rest])
            assert not bool(out[sees][..., 7].isfinite().any())


def test_a_set_is_what_it_holds(ctx, torch_gpu):
    """An adapter of a large rank that was dropped or replaced leaves no trace: the bits of a set that never
    held it, and a call that is captured then is captured for the ranks loaded then."""
    torch = torch_gpu
    K, N, extents, who = 4096, 256, [600, 70, 3], [0, 1, 0]
    x, base = torch.randn(sum(extents), K, device="cuda").half(), torch.randn(sum(extents), N, device="cuda")
    fresh, used, rows = ctx.adapters_new(K, N, 3), ctx.adapters_new(K, N, 3), ctx.adapter_rows(extents, who)
    try:
        def put(h, i, r, seed):
            down, up = make_adapter(torch, K, N, r, seed)
            ctx.adapters_put(h, i, down.cpu().numpy(), up.cpu().numpy(), 1.0)

        def run(h):
            y = torch.full_like(base, float("nan"))
            ctx.adapters(h, rows, x, base, y, x_dtype=tgo_amd.F16)
            torch.cuda.synchronize()
            return y
        put(used, 2, 128, 9)
        put(used, 1, 100, 8)
        for h in (fresh, used):
            put(h, 0, 16, 1)
            put(h, 1, 8, 2)
        ctx.adapters_drop(used, 2)
        assert torch.equal(run(used), run(fresh))
        graph, side, y = torch.cuda.CUDAGraph(), torch.cuda.Stream(), torch.zeros_like(base)
        ctx.set_stream(side.cuda_stream)
        try:
            with torch.cuda.graph(graph, stream=side):
                ctx.adapters(used, rows, x, base, y, x_dtype=tgo_amd.F16)
        finally:
            ctx.set_stream(torch.cuda.current_stream().cuda_stream)
        put(used, 1, 33, 3)
        for _ in range(3):
            graph.replay()
            torch.cuda.synchronize()
            assert bool(y[600:670].isnan().all())
            assert torch.equal(y[:600], run(fresh)[:600]) and torch.equal(y[670:], run(fresh)[670:])
    finally:
        for f, a in ((ctx.adapters_free, fresh), (ctx.adapters_free, used), (ctx.adapter_rows_free, rows)):
            f(a)


@pytest.mark.parametrize("extents", [[1, 5, 9], [300, 1, 280]])
def test_adapters_of_small_activations(ctx, torch_gpu, extents):
    """f32 rows of 1, 1e-3, 1e-4 and 1e-6, and of all of them mixed: each x is carried as hi + lo, to 2^-22 of
    itself or to half of f16's smallest step, 2^-25."""
    torch = torch_gpu
    K, N, who = 1024, 192, [0, 1, 0]
    T = sum(extents)
    g = torch.Generator(device="cuda").manual_seed(12)
    sizes = torch.tensor([1.0, 1e-3, 1e-4, 1e-6], device="cuda")
    x = torch.randn(T, K, device="cuda", generator=g)
    row = torch.arange(T, device="cuda") % 5
    mixed = sizes[torch.randint(0, 4, (T, K), device="cuda", generator=g)]
    x *= torch.where(row[:, None] < 4, sizes[row.clamp_max(3)][:, None], mixed)
    s, rows = ctx.adapters_new(K, N, 2), ctx.adapter_rows(extents, who)
    try:
        loaded = {}
        for i, r in enumerate((16, 40)):
            down, up = make_adapter(torch, K, N, r, i)
            ctx.adapters_put(s, i, down.cpu().numpy(), up.cpu().numpy(), 1.0)
            loaded[i] = (down.double(), up.double(), 1.0)
        y = torch.full((T, N), float("nan"), device="cuda")
        ctx.adapters(s, rows, x, None, y)
        torch.cuda.synchronize()
        want, tol = adapters64(torch, x.double(), None, extents, who, loaded, K, N, True)
        at = 0
        for n, a in zip(extents, who):  # the floor of every x through both products
            down, up, _ = loaded[a]
            tol[at:at + n] += (2.0 ** -25 * down.abs().sum(1)) @ up.abs().t() * (1 + 2.0 ** -20)
            at += n
        assert bool(((y.double() - want).abs() <= tol).all())
    finally:
        ctx.adapter_rows_free(rows)
        ctx.adapters_free(s)


@pytest.mark.parametrize("nq,nk", [([1, 2], [900, 64]), ([150, 40], [150, 300])])
def test_packed_attention_of_small_queries(ctx, torch_gpu, nq, nk):
    """f32 queries of 1e-4 over keys of some hundreds: each q is carried to 2^-25 at worst."""
    torch = torch_gpu
    q, k, v = inputs(torch, nq, nk, 4, 2, 128, False, seed=6)
    q, k = q * 1e-4, (k * 200).half()
    out = attend(ctx, torch, q, k, v, nq, nk, scale=0.25)
    torch.cuda.synchronize()
    want, tol = attention64(torch, q, k, v, nq, nk, 0.25, True)
    # a score is off by that of every dim; a probability and its sum by e^ds - 1 < 1.1 ds each
    ds = 0.25 * 2.0 ** -25 * float(k.abs().double().sum(-1).max())
    assert ds < 0.01
    assert bool(((out.double() - want).abs() <= tol + 2.2 * ds * float(v.abs().max()) + U * want.abs()).all())


def test_tensors_of_other_ranks_are_refused(ctx, torch_gpu):
    """Operands without the axes that the call needs, with the binding's own error."""
    torch = torch_gpu
    h, plan = ctx.rope_new(64, 1e4), ctx.packed_plan([2], [2], 1, 1, head_dim=64)
    try:
        x, pos = torch.zeros(2, 1, 64, device="cuda"), torch.zeros(2, device="cuda", dtype=torch.int32)
        for shape in ((2, 64), (128,), (2, 1, 64, 1), ()):
            flat = torch.zeros(shape, device="cuda")
            with pytest.raises(TgoError, match="tensor 0 is"):
                ctx.rope(h, pos, [(flat, flat)])
            with pytest.raises(TgoError, match="\\[rows, heads, head_dim\\]"):
                ctx.packed_attention(plan, flat, x.half(), x.half(), torch.zeros_like(x), 0.1)
        with pytest.raises(TgoError, match="tensors of heads"):
            ctx.rope(h, pos, [])
        with pytest.raises(TgoError, match="tensors of heads"):
            ctx.rope(h, pos, [(x, torch.zeros_like(x))] * 4)
    finally:
        ctx.rope_free(h)
        ctx.packed_free(plan)
