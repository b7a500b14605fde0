"""The 8-bit paged cache (store, read, move, attention) against plain float64 forms.

Tolerances count roundings, as in test_operators_gpu: u = 2^-24 for an f32 operation, 2^-22 for an
operand carried as an f16 hi + lo pair, half an ulp of f16 (2^-11 of the value, 2^-25 below its normal
range) for an f16 result; a sum of n terms in f32 is off by 4 sqrt(n) u of their magnitudes. A code is
off by half a step: 1/2 of an int8 row's scale, 2^-4 of an e4m3 value or 2^-10 of its scale."""
import itertools
import math

import numpy as np
import pytest

import tgo_amd
from tgo_amd import TgoError

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
HALF = 2.0 ** -11
FORMS = ("i8", "f8")
TOP = {"i8": 127.0, "f8": 448.0}


def f16_step(y):
    return HALF * y.abs() + 2.0 ** -25


class Pool:
    """Codes and scales with the values of anything a test wrote before; NaN everywhere at first."""

    def __init__(self, torch, layers, pages, kv, block, d, form):
        shape = (layers, pages, kv, block, d)
        self.torch, self.form, self.block, self.capacity = torch, form, block, pages * block
        t = torch.int8 if form == "i8" else torch.float8_e4m3fn
        self.k, self.v = (torch.full(shape, 85, device="cuda", dtype=torch.uint8).view(t) for _ in "kv")
        self.ks, self.vs = (torch.full(shape[:4], float("nan"), device="cuda") for _ in "kv")
        self.cache = tgo_amd.Cache(self.k, self.v, self.ks, self.vs)

    def fill(self, seed=1, spread=0.7):
        torch = self.torch
        g = torch.Generator(device="cuda").manual_seed(seed)
        for c, s in ((self.k, self.ks), (self.v, self.vs)):
            x = torch.randn(c.shape, device="cuda", generator=g)
            c.copy_((x * 42).round().clamp(-127, 127).to(torch.int8) if self.form == "i8" else
                    (x * 150).clamp(-448, 448).to(torch.float8_e4m3fn))
            s.copy_((torch.randn(s.shape, device="cuda", generator=g) * spread).exp() * (3 / TOP[self.form]))
        return self

    def values(self, slots, layer=0):
        """K's and V's rows of slots (host or device ints) in float64, [n, kv, d]."""
        at = self.torch.as_tensor(slots, device="cuda").long()
        out = []
        for c, s in ((self.k, self.ks), (self.v, self.vs)):
            page, off = at // self.block, at % self.block
            codes = c[layer].view(self.torch.uint8)[page, :, off].view(c.dtype)
            out.append(codes.double() * s[layer][page, :, off].double()[..., None])
        return out

    def bytes(self):
        return [t.view(self.torch.uint8).clone() for t in (self.k, self.v, self.ks, self.vs)]


def same_bytes(torch, a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


# ---------------------------------------------------------------------------
# store
# ---------------------------------------------------------------------------

def turned64(torch, x, gain, eps, pos, rd, layout, w, m):
    """Normed and rotated in float64, and the error an f32 result may have.

    Norm: a sum of d squares (8 in a row, then 4 pairs: 12 u), halved by the root, a quotient, root, and
    two products: 11 u. Rotation: 2^-21 of the pair's magnitudes (test_operators_gpu's), and the norm's of both."""
    x = x.double()
    err = torch.zeros_like(x)
    if gain is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * gain.double()
        err = 11 * U * x.abs()
    if rd:
        ang = pos.double().cpu()[:, None] * torch.from_numpy(w)[None, :]
        c, s = (m * ang.cos()).to(x.device)[:, None], (m * ang.sin()).to(x.device)[:, None]
        ia = torch.arange(rd // 2, device=x.device)
        ia, ib = (ia, ia + rd // 2) if layout == tgo_amd.ROPE_HALF else (2 * ia, 2 * ia + 1)
        y, e = x.clone(), err.clone()
        a, b = x[..., ia], x[..., ib]
        y[..., ia], y[..., ib] = a * c - b * s, a * s + b * c
        mag = m * (a.abs() + b.abs())
        e[..., ia] = e[..., ib] = (2.0 ** -21 + (11 * U if gain is not None else 0)) * mag
        x, err = y, e
    return x, err


def check_rows(torch, pool, form, got, y, err):
    """Values read back against the float64 row, and the scales that they were taken with."""
    scale = (y.abs().amax(-1, keepdim=True) / TOP[form]).clamp_min(2.0 ** -40)
    off = err.amax(-1, keepdim=True) / TOP[form] + 2 * U * scale  # of the scale
    if form == "i8":
        step = 0.5 * scale + 0.5 * off
    else:
        step = torch.maximum(2.0 ** -4 * y.abs(), 2.0 ** -10 * scale) + 0.07 * (err + off * TOP[form])
    # the quotient (three roundings of up to `top` steps) decides near a border
    tol = step + err + 4 * U * y.abs() + off * TOP[form] * 2
    bad = (got - y).abs() > tol
    assert not bool(bad.any()), (float(((got - y).abs() / tol).max()), int(bad.sum()))


def store(ctx, torch, pool, layer, slots, q, k, v, **kw):
    q_out = kw.pop("q_out", None)
    if q is not None and q_out is None:
        q_out = torch.full(q.shape, float("nan"), device="cuda", dtype=q.dtype)
    ctx.cache_store(pool.cache, layer, slots, k, v, q, q_out, **kw)
    return q_out


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("layout", [tgo_amd.ROPE_INTERLEAVED, tgo_amd.ROPE_HALF])
@pytest.mark.parametrize("d,rd,T,H,Hkv,block,norm", [
    (128, 128, 1, 32, 8, 32, True), (128, 64, 37, 5, 3, 16, True), (64, 64, 300, 2, 1, 8, True), (128, 96, 65, 28, 4, 64, False),
    (64, 20, 9, 3, 1, 1, True), (128, 6, 130, 4, 2, 1024, True), (128, 0, 33, 7, 7, 16, True), (64, 0, 5, 1, 1, 4, False),
    (128, 128, 1153, 16, 8, 16, True), (64, 32, 5000, 1, 1, 32, True), (128, 128, 2, 300, 100, 2, True)])
def test_store_over_a_fused_row(ctx, torch_gpu, d, rd, T, H, Hkv, block, norm, layout, f16, form):
    torch = torch_gpu
    g = torch.Generator(device="cuda").manual_seed(d * T + rd)
    row = torch.randn(T, H + 2 * Hkv, d, device="cuda", generator=g) * 3
    row = row.half() if f16 else row
    pos = torch.randint(-70000, 200000, (T,), device="cuda", generator=g, dtype=torch.int32)
    gains = [1 + 0.3 * torch.randn(d, device="cuda", generator=g) for _ in "qk"] if norm else [None, None]
    pages = (T + block - 1) // block + 2
    pool = Pool(torch, 2, pages, Hkv, block, d, form)
    slots = torch.randperm(pool.capacity, device="cuda", generator=g)[:T].int()
    before = pool.bytes()
    h = ctx.rope_new(d, 1e6, rotary_dim=rd, layout=layout) if rd else 0
    try:
        w, m = tgo_amd.rope_freqs(d, 1e6, rotary_dim=rd, layout=layout) if rd else (None, 1.0)
        q, k, v = row[:, :H], row[:, H:H + Hkv], row[:, H + Hkv:]
        kw = dict(positions=pos if rd else None, rope=h, q_gain=gains[0], k_gain=gains[1], eps=1e-5)
        q_out = store(ctx, torch, pool, 1, slots, q, k, v, **kw)
        torch.cuda.synchronize()
        want, err = turned64(torch, q, gains[0], 1e-5, pos, rd, layout, w, m)
        err = err + (f16_step(want) if f16 else U * want.abs())
        assert bool(((q_out.double() - want).abs() <= err).all()), float(((q_out.double() - want).abs() / err).max())
        gk, gv = pool.values(slots, 1)
        check_rows(torch, pool, form, gk, *turned64(torch, k, gains[1], 1e-5, pos, rd, layout, w, m))
        check_rows(torch, pool, form, gv, v.double(), torch.zeros_like(v, dtype=torch.float64))
        # scales are the rows' own, codes reach the top
        at = slots.long()
        vs = pool.vs[1][at // block, :, at % block].double()
        assert bool(((vs - v.double().abs().amax(-1) / TOP[form]).abs() <= 2 * U * vs).all())
        # the other layer and the slots that no row names stay as they were
        after = pool.bytes()
        for b, a in zip(before, after):
            assert torch.equal(b[0], a[0])
            rest = torch.ones(pool.capacity, dtype=torch.bool, device="cuda")
            rest[at] = False
            rest = rest.view(pages, block)
            shape = (pages, Hkv, block, -1)
            assert torch.equal(b[1].reshape(shape).transpose(1, 2)[rest], a[1].reshape(shape).transpose(1, 2)[rest])
        # f16 queries of f32 rows and the other way round, in place, and without queries: the same keys and values
        other = torch.full(q.shape, float("nan"), device="cuda", dtype=torch.float32 if f16 else torch.float16)
        store(ctx, torch, pool, 1, slots, q, k, v, q_out=other, **kw)
        assert torch.equal(other.half() if f16 else other, q_out if f16 else q_out.half())
        store(ctx, torch, pool, 1, slots, None, k, v, **kw)
        flat = row.clone()
        store(ctx, torch, pool, 1, slots, flat[:, :H], flat[:, H:H + Hkv], flat[:, H + Hkv:], q_out=flat[:, :H], **kw)
        torch.cuda.synchronize()
        assert torch.equal(flat[:, :H], q_out) and torch.equal(flat[:, H:], row[:, H:])
        assert same_bytes(torch, after, pool.bytes())
    finally:
        if h:
            ctx.rope_free(h)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("layout", [tgo_amd.ROPE_INTERLEAVED, tgo_amd.ROPE_HALF])
def test_store_strides_orders_and_alignments(ctx, torch_gpu, layout, form):
    """Heads-major order, rows and heads apart by odd distances, starts off 16 bytes, one row or head read by
    all: without a norm the codes, scales and queries of the dense call, to the bit (the norm's sum has
    another order there)."""
    torch = torch_gpu
    T, H, Hkv, d, rd = 33, 6, 2, 64, 48
    h = ctx.rope_new(d, 1e4, rotary_dim=rd, layout=layout)
    pos = torch.arange(T, device="cuda", dtype=torch.int32) * 977
    slots = torch.randperm(48, device="cuda")[:T].int()
    pool, other = (Pool(torch, 1, 3, Hkv, 16, d, form) for _ in range(2))
    try:
        for xt in (torch.float32, torch.float16):
            x = [torch.randn(T, n, d, device="cuda").to(xt) for n in (H, Hkv, Hkv)]
            dense = store(ctx, torch, pool, 0, slots, *x, positions=pos, rope=h)
            for off, pad, order in ((0, 0, "hm"), (1, 3, "rm"), (2, 6, "rm"), (5, 1, "hm"), (4, 8, "rm")):
                def strided(t):
                    n = t.shape[1]
                    shape = (T, n, d + pad) if order == "rm" else (n, T, d + pad)
                    buf = torch.full((off + math.prod(shape),), -7.0, device="cuda", dtype=t.dtype)
                    y = buf[off:].view(shape)[..., :d]
                    y = y if order == "rm" else y.transpose(0, 1)
                    y.copy_(t)
                    return buf, y
                xs = [strided(t)[1] for t in x]
                buf, ys = strided(torch.zeros_like(x[0]))
                store(ctx, torch, other, 0, slots, *xs, q_out=ys, positions=pos, rope=h)
                torch.cuda.synchronize()
                assert torch.equal(ys, dense), (xt, off, pad, order)
                ys.fill_(-7.0)
                assert bool((buf == -7.0).all())
                assert same_bytes(torch, pool.bytes(), other.bytes()), (xt, off, pad, order)
        k = torch.randn(1, 1, d, device="cuda").expand(T, Hkv, d)
        store(ctx, torch, pool, 0, slots, None, k, k, positions=pos, rope=h)
        store(ctx, torch, other, 0, slots, None, k.contiguous(), k.contiguous(), positions=pos, rope=h)
        assert same_bytes(torch, pool.bytes(), other.bytes())
    finally:
        ctx.rope_free(h)


@pytest.mark.parametrize("form", FORMS)
def test_store_rows_of_every_size(ctx, torch_gpu, form):
    """Rows of zeros, of one value, from 2^-140 to 2^37, past 2^40, infinite and NaN: what the format says they
    stand for; no code is a NaN's."""
    torch = torch_gpu
    d = 64
    sizes = [0.0] + [2.0 ** e for e in (-140, -60, -48, -41, -40, -30, -14, 0, 15, 17, 30, 37)]
    rows = [s * torch.randn(d, device="cuda") for s in sizes] + [s * torch.ones(d, device="cuda") for s in sizes]
    for bad in (float("nan"), float("inf"), -float("inf"), 2.0 ** 41):
        r = torch.randn(d, device="cuda")
        r[17] = bad
        rows.append(r)
    edge = torch.zeros(d, device="cuda")
    edge[3] = -2.0 ** 40
    x = torch.stack(rows + [edge]).view(-1, 1, d)
    T = len(x)
    pool = Pool(torch, 1, T, 1, 1, d, form)
    slots = torch.arange(T, device="cuda", dtype=torch.int32)
    store(ctx, torch, pool, 0, slots, None, x, x.flip(0))
    torch.cuda.synchronize()
    k, v = pool.values(slots)
    n = 2 * len(sizes)
    for got, y in ((k[:, 0], x[:, 0].double()), (v.flip(0)[:, 0], x[:, 0].double())):
        assert bool(got[n:n + 4].isnan().all())
        fine = torch.cat([torch.arange(n), torch.tensor([n + 4])]).cuda()
        # f32 subnormal rows round to 0 at the least scale anyway
        check_rows(torch, pool, form, got[fine], y[fine], torch.zeros_like(y[fine]))
    for c in (pool.k, pool.v):
        assert not bool((c.view(torch.uint8) & 0x7f == 0x7f).any()) or form == "i8"
        assert bool((c.view(torch.uint8)[0][n:n + 4] == 0).all()) or c is pool.v
    if form == "i8":
        assert int(pool.k.min()) >= -127


@pytest.mark.parametrize("form", FORMS)
def test_store_drops_what_lies_outside_the_pool(ctx, torch_gpu, form):
    torch = torch_gpu
    T, H, Hkv, d = 9, 3, 2, 128
    pool = Pool(torch, 1, 2, Hkv, 8, d, form)
    q, k, v = (torch.randn(T, n, d, device="cuda") for n in (H, Hkv, Hkv))
    slots = torch.tensor([0, 16, 15, -1, 2 ** 31 - 1, -2 ** 31, 7, 17, 8], device="cuda", dtype=torch.int32)
    before = pool.bytes()
    ones = torch.ones(d, device="cuda")
    out = store(ctx, torch, pool, 0, slots, q, k, v, q_gain=ones, k_gain=ones)
    torch.cuda.synchronize()
    want, err = turned64(torch, q, ones, 1e-6, None, 0, 0, None, 1.0)
    assert bool(((out.double() - want).abs() <= err + U * want.abs()).all())
    kept = [0, 2, 6, 8]
    gk, gv = pool.values(slots[kept])
    check_rows(torch, pool, form, gk, *turned64(torch, k[kept], ones, 1e-6, None, 0, 0, None, 1.0))
    check_rows(torch, pool, form, gv, v[kept].double(), torch.zeros(4, Hkv, d, device="cuda", dtype=torch.float64))
    rest = [s for s in range(16) if s not in (0, 15, 7, 8)]
    for b, a in zip(before, pool.bytes()):
        s = (2, Hkv, 8, -1)
        b, a = (t[0].reshape(s).transpose(1, 2).reshape(16, Hkv, -1)[rest] for t in (b, a))
        assert torch.equal(a, b)
    store(ctx, torch, pool, 0, slots[:0], q[:0], k[:0], v[:0])  # no rows


# ---------------------------------------------------------------------------
# read, move
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("Hkv,block,d", [(1, 1, 64), (8, 16, 128), (3, 32, 128), (5, 64, 64)])
@pytest.mark.parametrize("n", [1, 7, 300])
def test_read(ctx, torch_gpu, n, Hkv, block, d, form):
    torch = torch_gpu
    pages = 300 // block + 1
    pool = Pool(torch, 3, pages, Hkv, block, d, form).fill(seed=n)
    g = torch.Generator(device="cuda").manual_seed(n)
    slots = torch.randint(-3, pool.capacity + 3, (n,), device="cuda", generator=g, dtype=torch.int32)  # twice, outside
    inside = ((slots >= 0) & (slots < pool.capacity))[:, None, None]
    k64, v64 = (torch.where(inside, x, 0.0) for x in pool.values(slots.clamp(0, pool.capacity - 1), 2))
    for dt in (torch.float32, torch.float16):
        for off, pad in ((0, 0), (0, 8), (1, 3)):
            bufs = [torch.full((off + n * Hkv * (d + pad),), -7.0, device="cuda", dtype=dt) for _ in "kv"]
            k, v = (b[off:].view(n, Hkv, d + pad)[..., :d] for b in bufs)
            ctx.cache_read(pool.cache, 2, slots, k, v)
            for got, want in ((k, k64), (v, v64)):
                tol = U * want.abs() + (f16_step(want) if dt == torch.float16 else 0)
                assert bool(((got.double() - want).abs() <= tol).all())
            both = [k.clone(), v.clone()]
            for y, b in ((k, bufs[0]), (v, bufs[1])):
                y.fill_(-7.0)
                assert bool((b == -7.0).all())
            ctx.cache_read(pool.cache, 2, slots, k)
            ctx.cache_read(pool.cache, 2, slots, v_out=v)
            assert torch.equal(k, both[0]) and torch.equal(v, both[1])
    ctx.cache_read(pool.cache, 0, slots[:0], k[:0], v[:0])
    ctx.cache_read(pool.cache, 0, slots)


def test_read_of_rows_that_stand_for_nan(ctx, torch_gpu):
    torch = torch_gpu
    pool = Pool(torch, 1, 4, 2, 4, 64, "i8").fill()
    pool.ks[0, 1, 0, 2] = float("nan")
    pool.vs[0, 3, 1, 0] = 0.0
    slots = torch.arange(16, device="cuda", dtype=torch.int32)
    k, v = (torch.empty(16, 2, 64, device="cuda", dtype=torch.float16) for _ in "kv")
    ctx.cache_read(pool.cache, 0, slots, k, v)
    nan = k.isnan()
    assert bool(nan[6, 0].all()) and int(nan.sum()) == 64
    assert bool((v[12, 1] == 0).all()) and bool(v.isfinite().all())


def moved(torch, pool, src, dst):
    out = []
    for t in pool.bytes():
        t = t.view(t.shape[0], t.shape[1], t.shape[2], pool.block, -1)
        new = t.clone()
        for s, e in zip(src, dst):
            new[:, e // pool.block, :, e % pool.block] = t[:, s // pool.block, :, s % pool.block]
        out.append(new)
    return out


def moves(kind, n, r):
    """(src, dst, slots)"""
    if kind == "apart":
        p = r.permutation(2 * n)
        return p[:n], p[n:], 2 * n
    if kind == "down":      # n rows one place down: a chain of any length
        return np.arange(1, n + 1), np.arange(n), n + 1
    if kind == "up":
        return np.arange(n), np.arange(1, n + 1), n + 1
    if kind == "paths":     # accepted paths in regions of 8: places 0, 1, ... from places at or past them
        src, dst = [], []
        for s in range(n):
            path = sorted(r.choice(8, r.integers(1, 6), replace=False))
            src += [8 * s + int(p) for p in path]
            dst += [8 * s + i for i in range(len(path))]
        return np.array(src), np.array(dst), 8 * n
    if kind == "swaps":     # cycles of two
        p = r.permutation(2 * n)
        return p, np.concatenate([p[n:], p[:n]]), 2 * n
    if kind == "spread":    # one row to many places, itself replaced
        return np.concatenate([np.zeros(n, int), [n + 1]]), np.concatenate([np.arange(1, n + 1), [0]]), n + 2
    if kind == "cycles":    # of 64, and chains into them
        src = np.concatenate([64 * s + np.arange(64) for s in range(n)])
        dst = np.concatenate([64 * s + (np.arange(64) + 1) % 64 for s in range(n)])
        extra = 64 * n + np.arange(5 * n)  # five copies out of each cycle
        return np.concatenate([src, np.repeat(64 * np.arange(n) + 3, 5)]), np.concatenate([dst, extra]), 69 * n
    if kind == "cycle_behind_a_chain":
        # 100 rows, each onto the next's source, whose last reads what the cycle of 40 writes over
        chain_src, chain_dst = 40 + np.arange(100), 41 + np.arange(100)
        return (np.concatenate([np.arange(40), chain_src[::-1], [5]]),
                np.concatenate([(np.arange(40) + 1) % 40, chain_dst[::-1], [40]]), 141)
    if kind == "random":
        src, dst = r.integers(0, 3 * n, n), r.permutation(3 * n)[:n]
        return src, dst, 3 * n
    raise ValueError(kind)


@pytest.mark.parametrize("form,d", [("i8", 128), ("f8", 64)])
@pytest.mark.parametrize("kind,n", [("apart", 1), ("apart", 333), ("apart", 480), ("apart", 481), ("down", 5), ("down", 64), ("down", 65), ("down", 1000),
                                    ("up", 1000), ("up", 64), ("up", 65), ("paths", 1), ("paths", 64), ("paths", 200), ("swaps", 100), ("spread", 200),
                                    ("cycles", 3), ("cycle_behind_a_chain", 0), ("random", 40), ("random", 900)])
def test_move(ctx, torch_gpu, kind, n, form, d):
    torch = torch_gpu
    r = np.random.default_rng(n)
    src, dst, slots = moves(kind, n, r)
    order = r.permutation(len(src))
    if kind == "random":  # its random functions may hold cycles of more than 64: none is this long here
        assert longest_cycle(src, dst) <= 64
    block = 16
    pool = Pool(torch, 3, (slots + block - 1) // block, 3, block, d, form).fill(seed=n)
    want = moved(torch, pool, src, dst)
    ctx.cache_move(pool.cache, src[order], dst[order])
    torch.cuda.synchronize()
    for got, w in zip(pool.bytes(), want):
        assert torch.equal(got.view(w.shape), w)


def longest_cycle(src, dst):
    to = {int(d): int(s) for s, d in zip(src, dst) if s != d}
    best = 0
    for d in to:
        at, n = to[d], 1
        while at != d and at in to and n <= len(to):
            at, n = to[at], n + 1
        best = max(best, n if at == d else 0)
    return best


@pytest.mark.parametrize("n", [7, 400, 700])
def test_moves_follow_each_other(ctx, torch_gpu, n):
    """Moves of other rows without a wait between them: each acts on what the one before left."""
    torch = torch_gpu
    r = np.random.default_rng(n)
    pool = Pool(torch, 2, (3 * n + 15) // 16, 2, 16, 64, "i8").fill(seed=n)
    before = pool.bytes()
    steps = []
    for _ in range(6):
        p = r.permutation(3 * n)
        steps.append((p[:n], p[n:2 * n]))
    host = [t.cpu().view(2, pool.k.shape[1], 2, 16, -1) for t in before]
    for src, dst in steps:
        ctx.cache_move(pool.cache, [int(x) for x in src], dst)
    for i, t in enumerate(host):
        for src, dst in steps:
            t[:, dst // 16, :, dst % 16] = t[:, src // 16, :, src % 16].clone()
    torch.cuda.synchronize()
    for got, want in zip(pool.bytes(), host):
        assert torch.equal(got.cpu().view(want.shape), want)


def test_move_refusals(ctx, torch_gpu):
    torch = torch_gpu
    pool = Pool(torch, 2, 5, 2, 16, 64, "i8").fill()
    before = pool.bytes()
    ring = np.arange(65)
    for src, dst, word in (([0], [80], "slot 80 of a pool of 80"), ([-1], [0], "slot -1"), ([0, 1], [2, 2], "two rows go to slot 2"),
                           (ring, (ring + 1) % 65, "cycle of 65 slots; up to 64"), ([0, 1], [0], "2 slots to 1")):
        with pytest.raises(TgoError, match=word):
            ctx.cache_move(pool.cache, src, dst)
    ctx.cache_move(pool.cache, [], [])
    ctx.cache_move(pool.cache, [3, 4], [3, 4])
    torch.cuda.synchronize()
    assert same_bytes(torch, before, pool.bytes())


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------

def ancestors(parents):
    n = len(parents)
    seen = np.zeros((n, n), bool)
    for i in range(n):
        a = i
        while a >= 0:
            seen[i, a] = True
            a = parents[a]
    return seen


def attention64(torch, q, kv, vs, extents, lengths, parents, scale):
    """(output, tolerance of an f32 result before its own rounding) in float64. kv: each sequence's keys and values
    [length, kv, d] in float64; vs: the values' scales [length, kv]."""
    H, d = q.shape[1:]
    f16 = q.dtype == torch.float16
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    t = 0
    for (k, v), sv, n, m, up in zip(kv, vs, extents, lengths, parents):
        G = H // k.shape[1] if m else 1
        for i0 in range(0, n, 1024):
            i1 = min(n, i0 + 1024)
            if up is None:
                seen = torch.arange(m, device=q.device)[None] <= torch.arange(m - n + i0, m - n + i1, device=q.device)[:, None]
            else:
                seen = torch.ones(i1 - i0, m, dtype=torch.bool, device=q.device)
                seen[:, m - n:] = torch.from_numpy(ancestors(up)[i0:i1]).to(q.device)
            for h in range(H):
                qh, kh, vh = q[t + i0:t + i1, h].double(), k[:, h // G], v[:, h // G]
                w = sv[:, h // G].double().clamp(2.0 ** -40, 2.0 ** 40)
                s = (scale * (qh @ kh.t().contiguous())).masked_fill(~seen, -math.inf)
                top = s.max(1, keepdim=True)[0]
                p = (s - top).exp()
                l = p.sum(1, keepdim=True)
                out[t + i0:t + i1, h] = p @ vh / l
                # relative error of a term: its score's (the operands' pairs, d terms summed, two products and
                # the multiply-add), log2 of the value's scale (an ulp), the subtraction in log2 units, the
                # exponential's 2^-23, the f32 sums
                mag = scale * (qh.abs() @ kh.abs().t().contiguous())
                b = w.log2().abs().max()
                size = 1.45 * torch.where(seen, s.abs(), 0.0) + 1.45 * top.abs() + 2 * b + 8
                ds = ((0 if f16 else 2.0 ** -22) + 4 * math.sqrt(d) * U) * mag + 3 * U * torch.where(seen, s.abs(), 0.0)
                ds = ds + (0 if f16 else 2.0 ** -25 * scale) * kh.abs().sum(1) + 3 * U * size + 2 * U * b
                e = torch.where(seen, p * (ds + 2.0 ** -22 + 4 * math.sqrt(m) * U), 0.0)
                # what the second product takes besides: the rounding to f16 (or a pair), and its absolute floor,
                # 2^-32 of the largest probability times value scale
                f = e + p * (HALF if f16 else 2.0 ** -22) + seen * (2.0 ** -32 * (p * w).max(1, keepdim=True)[0] / w)
                tol[t + i0:t + i1, h] = (f @ vh.abs() + (e.sum(1, keepdim=True) / l) * (p @ vh.abs())) / l
        t += n
    return out, tol


class Batch:
    def __init__(self, torch, extents, lengths, H, Hkv, d, form, f16, block=16, trees=None, seed=1, spread=0.7, layers=2,
                 size=1.0):
        self.torch, self.extents, self.lengths, self.H, self.block = torch, extents, lengths, H, block
        need = [(l + block - 1) // block for l in lengths]
        self.pool = Pool(torch, layers, sum(need) + 3, Hkv, block, d, form).fill(seed, spread)
        r = np.random.default_rng(seed)
        order = r.permutation(sum(need) + 3)
        self.pages = np.zeros((len(lengths), max(need + [1]) + 1), np.uint32)
        at = 0
        for s, m in enumerate(need):
            self.pages[s, :m] = order[at:at + m]
            at += m
        self.parents = trees or [None] * len(extents)
        g = torch.Generator(device="cuda").manual_seed(seed)
        q = torch.randn(sum(extents), H, d, device="cuda", generator=g) * size
        self.q = q.half() if f16 else q
        self.scale = 1 / math.sqrt(d)
        self.layer = layers - 1

    def slots(self, s):
        p = np.arange(self.lengths[s])
        return self.pages[s, p // self.block].astype(np.int64) * self.block + p % self.block

    def plan(self, ctx, plan=0):
        up = None
        if any(p is not None for p in self.parents):
            up = sum([list(range(-1, n - 1)) if p is None else list(p) for n, p in zip(self.extents, self.parents)], [])
        return ctx.cache_plan(self.pool.cache, self.extents, self.lengths, self.pages, self.H, parents=up,
                              q_dtype=tgo_amd.F16 if self.q.dtype == self.torch.float16 else tgo_amd.F32, plan=plan)

    def run(self, ctx, out=None, plan=0):
        h = plan or self.plan(ctx)
        if out is None:
            out = self.torch.full(self.q.shape, float("nan"), device="cuda", dtype=self.q.dtype)
        ctx.cache_attention(h, self.pool.cache, self.layer, self.q, out, self.scale)
        if not plan:
            ctx.cache_plan_free(h)
        return out

    def exact(self):
        torch, kv, vs = self.torch, [], []
        for s in range(len(self.lengths)):
            at = torch.from_numpy(self.slots(s)).cuda()
            kv.append(self.pool.values(at, self.layer))
            vs.append(self.pool.vs[self.layer][at // self.block, :, at % self.block])
        return attention64(torch, self.q, kv, vs, self.extents, self.lengths, self.parents, self.scale)

    def check(self, got):
        want, tol = self.exact()
        tol = tol + (f16_step(want) if got.dtype == self.torch.float16 else U * want.abs())
        err = (got.double() - want).abs()
        assert bool((err <= tol).all()), (float((err / (tol + 1e-30)).max()), int((~(err <= tol)).sum()))


BATCHES = {
    "one": ([1], [1]), "tiny": ([3, 1, 2], [3, 1, 2]), "edges": ([31, 32, 33, 63, 64, 65], [31, 32, 33, 63, 64, 65]),
    "idle": ([0, 5, 0, 7, 1], [40, 5, 0, 7, 300]), "decode": ([1] * 9, [1, 2, 63, 64, 65, 700, 127, 129, 2049]),
    "few": ([2, 5, 8, 1, 7], [500, 5, 1025, 33, 1000]), "chunks": ([100, 17, 257], [1000, 17, 700]),
    "prompt": ([777], [777]), "mixed": ([1, 300, 1, 40], [3000, 300, 64, 2000]),
}


@pytest.mark.parametrize("batch", sorted(BATCHES))
@pytest.mark.parametrize("H,Hkv,d,block", [(8, 2, 128, 16), (4, 4, 64, 32), (7, 1, 128, 1), (64, 1, 64, 8), (6, 2, 128, 64),
                                           (10, 2, 64, 1024)])
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("form", FORMS)
def test_attention(ctx, torch_gpu, batch, H, Hkv, d, block, f16, form):
    b = Batch(torch_gpu, *BATCHES[batch], H, Hkv, d, form, f16, block)
    b.check(b.run(ctx))


def random_tree(r, n, wide):
    return [-1 if i == 0 or r.random() < 0.1 else int(r.integers(max(0, i - wide), i)) for i in range(n)]


@pytest.mark.parametrize("ctx_len", [0, 1, 30, 64, 1000, 9000])
@pytest.mark.parametrize("n,wide", [(1, 1), (2, 2), (5, 4), (16, 16), (33, 4), (63, 8), (64, 64)])
@pytest.mark.parametrize("H,Hkv,d,form,f16", [(8, 2, 128, "i8", False), (5, 1, 64, "f8", True), (4, 4, 128, "f8", False),
                                              (64, 2, 128, "i8", True)])
def test_trees_of_drafted_tokens(ctx, torch_gpu, n, wide, ctx_len, H, Hkv, d, form, f16):
    r = np.random.default_rng(n + ctx_len)
    b = Batch(torch_gpu, [n, 1, n], [ctx_len + n, 77, n + 3], H, Hkv, d, form, f16,
              trees=[random_tree(r, n, wide), None, [-1] * n])
    b.check(b.run(ctx))


@pytest.mark.parametrize("f16,d,form", [(False, 128, "i8"), (True, 128, "f8"), (False, 64, "f8"), (True, 64, "i8")])
def test_last_rows_of_every_kind(ctx, torch_gpu, f16, d, form):
    """Chunks that end in items of 128, 32 or fewer rows, beside single tokens and a tree; for f16 queries of many
    rows, items of 256 with others behind them."""
    sizes = [1, 16, 17, 96, 97, 127, 128, 129, 144, 160, 161, 191, 192, 193, 255, 256, 257, 1, 40]
    r = np.random.default_rng(3)
    lengths = [n + int(r.integers(0, 900)) for n in sizes]
    trees = [None] * (len(sizes) - 1) + [random_tree(r, 40, 8)]
    b = Batch(torch_gpu, sizes, lengths, 3, 3, d, form, f16, trees=trees)
    b.check(b.run(ctx))
    for extents, lengths, H, Hkv in (([2580, 1, 5, 0], [3080, 3000, 70, 9], 2, 1), ([2048, 700], [2048, 1900], 2, 1),
                                     ([2048, 1, 3], [27000, 700, 33], 8, 2)):
        b = Batch(torch_gpu, extents, lengths, H, Hkv, d, form, f16)
        b.check(b.run(ctx))


def test_a_chain_of_parents_is_a_causal_chunk(ctx, torch_gpu):
    """Parents -1, 0, 1, ... say nothing new, whatever the extent: the same bits."""
    b = Batch(torch_gpu, [300, 1, 20], [900, 40, 20], 8, 2, 128, "i8", False)
    plain = b.run(ctx)
    b.parents = [list(range(-1, n - 1)) for n in b.extents]
    assert torch_gpu.equal(plain, b.run(ctx))


@pytest.mark.parametrize("extents,lengths,H,Hkv,d,f16,form", [
    ([1, 1], [40000, 9000], 32, 8, 128, False, "i8"),   # long contexts of single tokens, cut and merged
    ([4], [30011], 16, 2, 64, True, "f8"),
    ([300], [20000], 8, 1, 128, True, "i8"),            # a chunk far behind its keys
    ([64], [16001], 4, 2, 128, False, "f8"),
    ([3000, 1100, 2047], [3000, 1100, 2047], 16, 8, 128, True, "i8"),
    ([2500], [2500], 28, 4, 128, False, "f8"),
    ([1500, 700], [1500, 9700], 16, 16, 64, False, "i8"),
])
def test_attention_over_long_contexts(ctx, torch_gpu, extents, lengths, H, Hkv, d, f16, form):
    b = Batch(torch_gpu, extents, lengths, H, Hkv, d, form, f16, seed=3)
    out = b.run(ctx)
    b.check(out)
    assert torch_gpu.equal(out, b.run(ctx))


@pytest.mark.parametrize("seed", range(12))
def test_attention_over_random_batches(ctx, torch_gpu, seed):
    """Single tokens, trees and chunks in one call, cut, merged and whole."""
    r = np.random.default_rng(seed)
    n = int(r.integers(2, 14))
    lengths = [int(x) for x in np.exp(r.uniform(0, math.log(9000), n))]
    extents = [int(r.choice([0, 1, 1, 2, r.integers(1, min(64, l) + 1), r.integers(1, min(600, l) + 1)])) for l in lengths]
    extents = [min(e, l) for e, l in zip(extents, lengths)]
    trees = [random_tree(r, e, int(r.integers(1, 9))) if 0 < e <= 64 and r.random() < 0.5 else None for e in extents]
    H, Hkv = [(32, 8), (16, 8), (28, 4), (64, 8), (5, 5)][seed % 5]
    b = Batch(torch_gpu, extents, lengths, H, Hkv, [128, 64][seed % 2], FORMS[seed // 2 % 2], bool(seed // 4 % 2),
              block=[16, 32, 4][seed % 3], trees=trees, seed=seed)
    b.check(b.run(ctx))


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("spread", [0.0, 8.0])
def test_scales_far_apart(ctx, torch_gpu, f16, spread):
    """Value rows of one size, or e^-24 to e^24: what the largest ones leave is right to their size, rows of
    zeros count in the sum, keys whose scores spread over hundreds."""
    torch = torch_gpu
    b = Batch(torch, [1, 40, 5], [700, 333, 5], 8, 2, 128, "i8", f16, spread=0.5)
    r = torch.Generator(device="cuda").manual_seed(5)
    b.pool.vs.copy_((torch.randn(b.pool.vs.shape, device="cuda", generator=r) * spread).exp().clamp(2.0 ** -38, 2.0 ** 38))
    b.pool.vs[..., ::3] = 2.0 ** -40
    b.pool.v[..., ::3, :] = 0
    b.check(b.run(ctx, out=torch.empty(b.q.shape, device="cuda")))  # past f16's range


@pytest.mark.parametrize("f16", [False, True])
def test_the_least_scale(ctx, torch_gpu, f16):
    """Scores of next to nothing, beside value rows of 2^-40 to 2^38: all that is seen weighs the same."""
    torch = torch_gpu
    b = Batch(torch, [1, 40, 300], [700, 333, 700], 8, 2, 128, "i8", f16)
    b.scale = 2.0 ** -64
    b.pool.ks.fill_(2.0 ** -40)
    b.pool.vs.copy_(torch.exp2(torch.randint(-40, 39, b.pool.vs.shape, device="cuda").float()))
    b.check(b.run(ctx, out=torch.empty(b.q.shape, device="cuda")))  # past f16's range


@pytest.mark.parametrize("size", [20.0, 400.0, 30000.0])
@pytest.mark.parametrize("f16", [False, True])
def test_peaked_scores(ctx, torch_gpu, size, f16):
    b = Batch(torch_gpu, [1, 40, 300], [700, 333, 300], 8, 2, 128, "i8", f16, size=min(size, 12000.0), spread=0.3)
    b.q.clamp_(-65000.0, 65000.0)  # |q| < 65504
    b.check(b.run(ctx))


@pytest.mark.parametrize("q_f16", [False, True])
def test_outputs_in_every_type(ctx, torch_gpu, q_f16):
    torch = torch_gpu
    for extents, lengths in (([1, 40, 3], [9000, 333, 3]), ([200], [500])):
        b = Batch(torch, extents, lengths, 8, 2, 128, "f8", q_f16)
        T = sum(extents)
        out = b.run(ctx, out=torch.empty(T, 8, 128, device="cuda"))
        half = b.run(ctx, out=torch.empty(T, 8, 128, device="cuda", dtype=torch.float16))
        pair = b.run(ctx, out=torch.empty(2, T, 8, 128, device="cuda", dtype=torch.float16))
        b.check(out)
        assert torch.equal(half, out.half())
        assert torch.equal(pair[0], out.half()) and torch.equal(pair[1], (out - out.half().float()).half())


@pytest.mark.parametrize("q_f16", [False, True])
def test_rows_of_wider_buffers(ctx, torch_gpu, q_f16):
    """q and out as columns of wider rows; nothing else of them is written, nor rows behind the last."""
    torch = torch_gpu
    b = Batch(torch, [1, 40, 3], [9000, 333, 3], 8, 2, 64, "i8", q_f16)
    T, w = 44, 8 * 64
    plain = b.run(ctx)
    wide = torch.full((T + 2, w + 64), -7.0, device="cuda", dtype=b.q.dtype)
    wide[:T, 32:32 + w] = b.q.view(T, w)
    out = torch.full((T + 2, w + 128), -7.0, device="cuda", dtype=b.q.dtype)
    h = b.plan(ctx)
    ctx.cache_attention(h, b.pool.cache, b.layer, wide[:T, 32:32 + w].unflatten(1, (8, 64)),
                        out[:T, 64:64 + w].unflatten(1, (8, 64)), b.scale)
    ctx.cache_plan_free(h)
    torch.cuda.synchronize()
    assert torch.equal(out[:T, 64:64 + w].reshape(T, 8, 64), plain)
    out[:T, 64:64 + w] = -7.0
    assert bool((out == -7.0).all())


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("f16", [False, True])
def test_nothing_unseen_reaches_a_row(ctx, torch_gpu, f16, form):
    """Rows standing for NaN at later tokens, other branches, other sequences, other heads, past the sequence in its
    last page, in pages that no table names: who does not see one keeps the bits, who does is NaN."""
    torch = torch_gpu
    r = np.random.default_rng(1)
    tree = random_tree(r, 40, 5)
    b = Batch(torch, [300, 40, 1, 5], [1000, 500, 2100, 90], 8, 2, 128, form, f16, trees=[None, tree, None, None])
    clean = b.run(ctx)
    b.check(clean)
    hit = torch.zeros(b.pool.capacity, dtype=torch.bool, device="cuda")
    for s in range(4):
        hit[torch.from_numpy(b.slots(s)).cuda()] = True
    at = (~hit).nonzero().flatten()
    for sc in (b.pool.ks, b.pool.vs):  # what nobody sees
        sc[b.layer][at // 16, :, at % 16] = float("nan")
    assert torch.equal(clean, b.run(ctx))

    def poison(seq, pos, head, scales):
        at = int(b.slots(seq)[pos])
        scales[b.layer, at // 16, head, at % 16] = float("nan")
    poison(0, 830, 0, b.pool.vs)   # token 130 of the chunk
    poison(0, 905, 0, b.pool.ks)
    poison(1, 460 + 7, 1, b.pool.vs)  # a drafted token
    poison(3, 3, 0, b.pool.ks)
    got = b.run(ctx)
    nan = torch.zeros_like(got, dtype=torch.bool)
    nan[130:300, :4] = True
    nan[300:340, 4:] = torch.from_numpy(ancestors(tree)[:, 7]).cuda()[:, None, None]
    nan[341:, :4] = True
    assert torch.equal(got.isnan(), nan)
    assert torch.equal(got[~nan], clean[~nan])


def test_rows_do_not_depend_on_each_other(ctx, torch_gpu):
    """A query that is infinite or NaN spoils its own row alone."""
    torch = torch_gpu
    b = Batch(torch, [1, 40, 300], [700, 333, 300], 8, 2, 128, "i8", False)
    clean = b.run(ctx)
    b.q[5, 3, 17] = float("nan")
    b.q[100, 0, 0] = float("inf")
    got = b.run(ctx)
    nan = torch.zeros_like(got, dtype=torch.bool)
    nan[5, 3] = nan[100, 0] = True
    assert torch.equal(got.isnan(), nan) and torch.equal(got[~nan], clean[~nan])


def test_shared_pages(ctx, torch_gpu):
    """Two sequences whose tables begin with the same pages, and one whose table names a page twice."""
    torch = torch_gpu
    b = Batch(torch, [1, 5, 1], [600, 640, 64], 8, 2, 128, "i8", False)
    b.pages[1, :30] = b.pages[0, :30]
    b.pages[2, :4] = b.pages[2, 0]
    b.check(b.run(ctx))


def test_offsets_past_32_bits(ctx, torch_gpu):
    """A layer of more than 2^32 bytes of codes, and a layer behind it: its last pages are stored, read, attended
    to and moved."""
    torch = torch_gpu
    Hkv, d, block, pages = 8, 128, 64, 2 ** 16 + 100  # 4.3 GB a layer
    shape = (2, pages, Hkv, block, d)
    k, v = (torch.zeros(shape, device="cuda", dtype=torch.int8) for _ in "kv")
    ks, vs = (torch.zeros(shape[:4], device="cuda") for _ in "kv")
    cache = tgo_amd.Cache(k, v, ks, vs)
    n = 130
    table = np.array([[pages - 1, 3, pages - 7]], np.uint32)
    pos = np.arange(n)
    at = table[0, pos // block].astype(np.int64) * block + pos % block
    slots = torch.from_numpy(at).int().cuda()
    x = [torch.randn(n, h, d, device="cuda") for h in (16, Hkv, Hkv)]
    q = torch.empty_like(x[0])
    ctx.cache_store(cache, 1, slots, x[1], x[2], x[0], q)
    gk, gv = (torch.empty(n, Hkv, d, device="cuda") for _ in "kv")
    ctx.cache_read(cache, 1, slots, gk, gv)
    for got, want in ((gk, x[1]), (gv, x[2])):
        check_rows(torch, None, "i8", got.double(), want.double(), torch.zeros_like(want, dtype=torch.float64))
    assert not bool(ks[0].any()) and int((ks[1] != 0).sum()) == n * Hkv
    h = ctx.cache_plan(cache, [n], [n], table, 16)
    out = torch.empty_like(q)
    ctx.cache_attention(h, cache, 1, q, out, d ** -0.5)
    ctx.cache_plan_free(h)
    off = torch.from_numpy(at).cuda()
    want, tol = attention64(torch, q, [(gk.double(), gv.double())], [vs[1][off // block, :, off % block]], [n], [n], [None], d ** -0.5)
    assert bool(((out.double() - want).abs() <= tol + 4 * U * want.abs()).all())
    ctx.cache_move(cache, at[:50], at[:50] - 1000 * block)
    mk = torch.empty_like(gk)
    ctx.cache_read(cache, 1, slots - 1000 * block, mk)
    assert torch.equal(mk[:50], gk[:50]) and not bool(mk[50:64].any())


def test_plans_are_replaced_and_shared_by_layers(ctx, torch_gpu):
    torch = torch_gpu
    a = Batch(torch, [1, 40], [9000, 333], 8, 2, 128, "i8", False)
    b = Batch(torch, [500, 1], [700, 3], 8, 2, 128, "i8", False, seed=2)
    h = a.plan(ctx)
    try:
        first = a.run(ctx, plan=h)
        a.check(first)
        a.layer = 0
        a.check(a.run(ctx, plan=h))
        a.layer = 1
        assert b.plan(ctx, plan=h) == h
        b.check(b.run(ctx, plan=h))
        a.plan(ctx, plan=h)
        assert torch.equal(first, a.run(ctx, plan=h))
    finally:
        ctx.cache_plan_free(h)


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("form", FORMS)
def test_a_layer_that_verifies_drafted_tokens(ctx, torch_gpu, form):
    """A prompt, then drafted trees verified, their accepted paths moved, then the next token: projection, store,
    attention, each stage against float64 of what the stage before left; the result of the last token equals that
    of a cache into which the accepted tokens went in order. Captured and replayed: the eager bits."""
    torch = torch_gpu
    K, H, Hkv, d, block = 256, 8, 2, 128, 16
    N = (H + 2 * Hkv) * d
    g = torch.Generator(device="cuda").manual_seed(4)
    w = (torch.randn(K, N, device="cuda", generator=g) / 16).half()
    gains = [1 + 0.2 * torch.randn(d, device="cuda", generator=g) for _ in "qk"]
    kw = dict(layout=tgo_amd.ROPE_HALF)
    wh, rope = ctx.weight_upload(tgo_amd.FORM_F16, K, N, w.cpu()), ctx.rope_new(d, 1e6, **kw)
    fr, m = tgo_amd.rope_freqs(d, 1e6, **kw)
    pool, plain = (Pool(torch, 1, 20, Hkv, block, d, form) for _ in range(2))
    table = np.random.default_rng(2).permutation(20).astype(np.uint32).reshape(2, 10)
    plans = []

    def slot(s, p):
        return int(table[s, p // block]) * block + p % block

    def forward(pool, x, extents, lengths, depth, parents=None, plan=0):
        """depth: each new token's position behind its sequence's old ones"""
        T = sum(extents)
        qkv = torch.empty(T, H + 2 * Hkv, d, device="cuda")
        old = [l - n for l, n in zip(lengths, extents)]
        slots, pos, t = [], [], 0
        for s, n in enumerate(extents):
            slots += [slot(s, old[s] + i) for i in range(n)]
            pos += [old[s] + depth[t + i] for i in range(n)]
            t += n
        slots, pos = (torch.tensor(a, device="cuda", dtype=torch.int32) for a in (slots, pos))
        q, out = torch.empty(T, H, d, device="cuda"), torch.empty(T, H, d, device="cuda")
        h = ctx.cache_plan(pool.cache, extents, lengths, table, H, parents=parents, plan=plan)
        plans.append(h)
        state = dict(x=x, qkv=qkv, slots=slots, pos=pos, q=q, out=out, plan=h, pool=pool)
        layer(state)
        torch.cuda.synchronize()
        up, t = [], 0
        for n in extents:
            up.append(None if parents is None else parents[t:t + n])
            t += n
        want, err = turned64(torch, qkv[:, :H], gains[0], 1e-6, pos, d, kw["layout"], fr, m)
        assert bool(((q.double() - want).abs() <= err + U * want.abs()).all())
        gk, gv = pool.values(slots)
        check_rows(torch, pool, form, gk, *turned64(torch, qkv[:, H:H + Hkv], gains[1], 1e-6, pos, d, kw["layout"], fr, m))
        check_rows(torch, pool, form, gv, qkv[:, H + Hkv:].double(), torch.zeros_like(gv))
        kv, vs = [], []
        for s, l in enumerate(lengths):
            at = torch.tensor([slot(s, p) for p in range(l)], device="cuda")
            kv.append(pool.values(at))
            vs.append(pool.vs[0][at // block, :, at % block])
        want, tol = attention64(torch, q, kv, vs, extents, lengths, up, d ** -0.5)
        assert bool(((out.double() - want).abs() <= tol + U * want.abs()).all())
        return state

    def layer(s):
        ctx.linear(wh, s["x"], s["x"].shape[0], s["qkv"])
        attend(s)

    def attend(s):
        ctx.cache_store(s["pool"].cache, 0, s["slots"], s["qkv"][:, H:H + Hkv], s["qkv"][:, H + Hkv:], s["qkv"][:, :H], s["q"],
                        positions=s["pos"], rope=rope, q_gain=gains[0], k_gain=gains[1])
        ctx.cache_attention(s["plan"], s["pool"].cache, 0, s["q"], s["out"], d ** -0.5)
    try:
        prompts = torch.randn(33 + 70, K, device="cuda", generator=g)
        for p in (pool, plain):
            forward(p, prompts, [33, 70], [33, 70], list(range(33)) + list(range(70)))
        trees = [[-1, 0, 0, 1, 2, 4, -1], [-1, 0, 1, 1, 3]]
        depth = []
        for t in trees:
            at = len(depth)
            for p in t:
                depth.append(0 if p < 0 else depth[at + p] + 1)
        drafted = torch.randn(12, K, device="cuda", generator=g)
        state = forward(pool, drafted, [7, 5], [40, 75], depth, parents=sum(trees, []))
        eager, rows = state["out"].clone(), pool.bytes()
        graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        ctx.set_stream(side.cuda_stream)
        try:
            torch.cuda.synchronize()
            with torch.cuda.graph(graph, stream=side):
                attend(state)
                for call in (lambda: ctx.cache_move(pool.cache, [0], [1]), lambda: ctx.cache_plan_free(state["plan"]),
                             lambda: ctx.cache_plan(pool.cache, [1], [1], [[0]], H)):
                    with pytest.raises(TgoError, match="being captured"):
                        call()
        finally:
            ctx.set_stream(torch.cuda.current_stream().cuda_stream)
        for _ in range(4):
            state["out"].fill_(float("nan"))
            state["q"].fill_(float("nan"))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(state["out"], eager) and same_bytes(torch, rows, pool.bytes())
            layer(state)
            torch.cuda.synchronize()
        # the paths 0, 2, 4 and 0, 1, 3, 4 are accepted
        paths = [[0, 2, 4], [0, 1, 3, 4]]
        ctx.cache_move(pool.cache, [slot(s, o + a) for s, o in ((0, 33), (1, 70)) for a in paths[s]],
                       [slot(s, o + i) for s, o in ((0, 33), (1, 70)) for i in range(len(paths[s]))])
        kept = drafted[[0, 2, 4, 7, 8, 10, 11]]
        forward(plain, kept, [3, 4], [36, 74], [0, 1, 2, 0, 1, 2, 3])
        for s, l in enumerate((36, 74)):
            at = torch.tensor([slot(s, p) for p in range(l)], device="cuda")
            for a, b in zip(pool.values(at), plain.values(at)):
                assert torch.equal(a, b)
        last = torch.randn(2, K, device="cuda", generator=g)
        a, b = (forward(p, last, [1, 1], [37, 75], [0, 0])["out"] for p in (pool, plain))
        assert torch.equal(a, b)
    finally:
        ctx.weight_free(wh)
        ctx.rope_free(rope)
        for h in plans:
            ctx.cache_plan_free(h)


def test_refusals(ctx, torch_gpu):
    """What the binding refuses before the call, and operands that meet in memory."""
    torch = torch_gpu
    pool = Pool(torch, 2, 4, 2, 16, 64, "i8").fill()
    c = pool.cache
    q, k, v, out = (torch.zeros(3, n, 64, device="cuda") for n in (4, 2, 2, 4))
    slots = torch.zeros(3, device="cuda", dtype=torch.int32)
    before = pool.bytes()
    h = ctx.cache_plan(c, [2, 1], [2, 60], np.zeros((2, 4), np.uint32), 4)
    r, r128 = ctx.rope_new(64, 1e4), ctx.rope_new(128, 1e4)
    inside = pool.ks.view(-1)[:64].expand(3, 2, 64)
    cases = [
        ("k and v are", lambda: ctx.cache_store(c, 0, slots, k[:2], v, q, out)),
        ("k and v are", lambda: ctx.cache_store(c, 0, slots, k[..., :32], v, q, out)),
        ("q and q_out", lambda: ctx.cache_store(c, 0, slots, k, v, q)),
        ("of one type", lambda: ctx.cache_store(c, 0, slots, k.half(), v, q, out)),
        ("float32 or float16", lambda: ctx.cache_store(c, 0, slots, k.bfloat16(), v.bfloat16())),
        ("slots is int32", lambda: ctx.cache_store(c, 0, slots.long(), k, v)),
        ("positions is int32 \\[3\\]", lambda: ctx.cache_store(c, 0, slots, k, v, rope=r)),
        ("q_gain is float32", lambda: ctx.cache_store(c, 0, slots, k, v, q, out, q_gain=torch.ones(32, device="cuda"))),
        ("tensor of the host", lambda: ctx.cache_store(c, 0, slots, k.cpu(), v)),
        ("tensor of the host", lambda: ctx.cache_store(c, 0, slots.cpu(), k, v)),
        ("layer 2 of 2", lambda: ctx.cache_store(c, 2, slots, k, v)),
        ("layer -1 of 2", lambda: ctx.cache_read(c, -1, slots, k)),
        ("no handle 9999", lambda: ctx.cache_store(c, 0, slots, k, v, positions=slots, rope=9999)),
        ("heads of 128, the cache of 64", lambda: ctx.cache_store(c, 0, slots, k, v, positions=slots, rope=r128)),
        ("eps is nan", lambda: ctx.cache_store(c, 0, slots, k, v, q, out, q_gain=torch.ones(64, device="cuda"), eps=float("nan"))),
        ("q_out meets k", lambda: ctx.cache_store(c, 0, slots, k, v, k, k)),
        ("q_out meets q in", lambda: ctx.cache_store(c, 0, slots, k, v, out.view(-1)[64:].as_strided((3, 2, 64), (128, 64, 1)),
                                                    out.view(-1).as_strided((3, 2, 64), (128, 64, 1)))),
        ("heads of q_out overlap", lambda: ctx.cache_store(c, 0, slots, k, v, q, out[:1].expand(3, 4, 64))),
        ("k meets the cache's k_scale", lambda: ctx.cache_store(c, 0, slots, inside, v)),
        ("k_out is", lambda: ctx.cache_read(c, 0, slots, q)),
        ("both of one type", lambda: ctx.cache_read(c, 0, slots, k, v.half())),
        ("k_out and v_out meet", lambda: ctx.cache_read(c, 0, slots, k, k)),
        ("heads of k_out overlap", lambda: ctx.cache_read(c, 0, slots, k[:1].expand(3, 2, 64))),
        ("q is \\[3, 4, 64\\]", lambda: ctx.cache_attention(h, c, 0, q[:2], out, 1.0)),
        ("q is float32", lambda: ctx.cache_attention(h, c, 0, q.half(), out, 1.0)),
        ("scale is 0", lambda: ctx.cache_attention(h, c, 0, q, out, 0.0)),
        ("scale is nan", lambda: ctx.cache_attention(h, c, 0, q, out, float("nan"))),
        ("out meets q", lambda: ctx.cache_attention(h, c, 0, q, q, 1.0)),
        ("16-byte boundaries", lambda: ctx.cache_attention(h, c, 0, torch.zeros(3 * 258 + 1, device="cuda")[1:].as_strided((3, 4, 64), (258, 64, 1)), out, 1.0)),
        ("the plan is of 4 pages", lambda: ctx.cache_attention(h, Pool(torch, 2, 8, 2, 8, 64, "i8").cache, 0, q, out, 1.0)),
        ("no handle 9999", lambda: ctx.cache_plan_free(9999)),
        ("page 3 is 4 of a pool of 4", lambda: ctx.cache_plan(c, [1], [60], np.full((1, 4), [0, 1, 2, 4], np.uint32), 4)),
        ("3 parents for 2", lambda: ctx.cache_plan(c, [2], [2], [[0]], 4, parents=[-1, 0, 1])),
        ("both int8", lambda: tgo_amd.Cache(pool.k.view(torch.uint8), pool.v, pool.ks, pool.vs)),
        ("k and v are", lambda: tgo_amd.Cache(pool.k[0], pool.v[0], pool.ks[0], pool.vs[0])),
        ("is not contiguous", lambda: tgo_amd.Cache(pool.k[:, :, :, ::2], pool.v[:, :, :, ::2], pool.ks, pool.vs)),
        ("v_scale is", lambda: tgo_amd.Cache(pool.k, pool.v, pool.ks, pool.vs[:1])),
        ("another device", lambda: tgo_amd.Cache(pool.k, pool.v, pool.ks, pool.vs.cpu())),
        ("k and v meet", lambda: ctx.cache_read(tgo_amd.Cache(pool.k, pool.k, pool.ks, pool.vs), 0, slots, k)),
    ]
    try:
        for word, call in cases:
            with pytest.raises(TgoError, match=word):
                call()
        torch.cuda.synchronize()
        assert same_bytes(torch, before, pool.bytes()) and not bool(out.any())
    finally:
        ctx.cache_plan_free(h)
        ctx.rope_free(r)
        ctx.rope_free(r128)
    with pytest.raises(TgoError, match="no handle"):
        ctx.cache_attention(h, c, 0, q[:0, :1], out[:0, :1], 1.0)


def test_another_stream_and_the_device_of_the_context(ctx, torch_gpu):
    """Calls on a stream of the caller's choice, ordered by it alone."""
    torch = torch_gpu
    b = Batch(torch, [1, 40], [9000, 333], 8, 2, 128, "f8", False)
    want = b.run(ctx)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    ctx.set_stream(side.cuda_stream)
    try:
        got = torch.empty_like(want)
        h = b.plan(ctx)
        ctx.cache_attention(h, b.pool.cache, b.layer, b.q, got, b.scale)
        side.synchronize()
        ctx.cache_plan_free(h)
    finally:
        ctx.set_stream(torch.cuda.current_stream().cuda_stream)
    assert torch.equal(got, want)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("off", [0, 1])
def test_codes_are_rounded_quotients(ctx, torch_gpu, off, f16, form):
    """Rows neither normed nor rotated, in units of eight elements and of two: each code is value / scale as f32 gives
    it, to the nearest, ties to even, and the scale the row's largest over 127 or 448, bit for bit. Half of the rows
    consist of exact half steps."""
    torch = torch_gpu
    T, Hkv, d = 1024, 4, 128
    r = np.random.default_rng(5)
    x = r.standard_normal((T, Hkv, d)).astype(np.float32)
    # a scale of few bits, times which the top and every half step are exact in the type
    bits = 3 if f16 else 16
    s = (2.0 ** (bits - 1) + r.integers(0, 2 ** (bits - 1), (T, Hkv, 1))) * 2.0 ** (1 - bits)
    if form == "i8":
        steps = np.arange(127) + 0.5
    else:
        grid = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).float().numpy()
        steps = (grid[1:] + grid[:-1]) / 2
    halves = r.choice(steps, (T, Hkv, d)) * r.choice([-1.0, 1.0], (T, Hkv, d))
    halves[..., 77] = TOP[form]
    x[::2] = (halves * s)[::2]
    x = x.astype(np.float16 if f16 else np.float32)
    y = x.astype(np.float32)
    scale = np.maximum(np.abs(y).max(-1) / np.float32(TOP[form]), np.float32(2.0 ** -40))
    q = y / scale[..., None]
    want = np.rint(q) if form == "i8" else torch.from_numpy(q).to(torch.float8_e4m3fn).float().numpy()
    buf = torch.zeros(off + x.size, device="cuda", dtype=torch.float16 if f16 else torch.float32)
    buf[off:] = torch.from_numpy(x).cuda().flatten()
    x = buf[off:].view(T, Hkv, d)
    pool = Pool(torch, 1, T // 16, Hkv, 16, d, form)
    store(ctx, torch, pool, 0, torch.arange(T, device="cuda", dtype=torch.int32), None, x, x)
    torch.cuda.synchronize()
    for codes, scales in ((pool.k, pool.ks), (pool.v, pool.vs)):
        assert np.array_equal(scales[0].transpose(1, 2).reshape(T, Hkv).cpu().numpy(), scale)
        got = codes[0].float().transpose(1, 2).reshape(T, Hkv, d).cpu().numpy()
        assert np.array_equal(got, want), (float(np.abs(got - want).max()), int((got != want).sum()))


def log2_units(b):
    """Makes a key's score q . code * k_scale in log2 units, to the bit."""
    b.scale = next(float(x) for x in np.float32(math.log(2)) * (1 + np.arange(-8, 9, dtype=np.float32) * np.float32(2.0 ** -24))
                   if np.float32(x) * np.float32(1.4426950408889634) == 1)


# rows of one kv head that go as an item of up to 16, 32, 128 rows, and of 256 where queries are f16
ITEMS = [5, 20, 100, 256]


@pytest.mark.parametrize("n", ITEMS)
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("e", [10, 21, 23, 24, 25, 27])
def test_a_key_sixteen_above_the_ones_before(ctx, torch_gpu, e, f16, n):
    """Scores of 2^e, and in a later tile one of 16 more: every term is a power of two, so results are exact but for
    the sums' roundings (4 sqrt(n) u and a quotient)."""
    torch = torch_gpu
    b = Batch(torch, [n], [700], 1, 1, 128, "i8", f16)
    log2_units(b)
    b.pool.k.zero_()
    b.pool.k[..., 0] = 64
    b.pool.ks.fill_(2.0 ** (e - 21))
    b.pool.vs.fill_(1.0)
    late = int(b.slots(0)[200])
    b.pool.k[b.layer, late // 16, 0, late % 16, 1] = 16
    b.q.zero_()
    b.q[..., 0] = 2.0 ** 15
    b.q[..., 1] = 2.0 ** (21 - e)
    got = b.run(ctx)
    v = b.pool.values(b.slots(0), b.layer)[1][:, 0]
    w = torch.ones(700, device="cuda", dtype=torch.float64)
    w[200] = 2.0 ** 16
    for i in range(n):
        m = 700 - n + i + 1
        want = (w[:m] @ v[:m]) / w[:m].sum()
        err = (got[i, 0].double() - want).abs()
        tol = (4 * math.sqrt(700) + 2) * U * 127 + (f16_step(want) if f16 else 0)
        assert bool((err <= tol).all()), (i, float(err.max()))


@pytest.mark.parametrize("n", ITEMS)
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("e", [16, 22, 26, 29, 33, 60])
@pytest.mark.parametrize("form,d", [("i8", 128), ("f8", 64)])
def test_keys_alike_far_from_zero(ctx, torch_gpu, form, d, e, f16, n):
    """Keys that are all the same weigh the same, whatever their score (up to 2^e in size, of either sign): the mean
    of the values seen, where the first row of a prompt sees one and a long context is cut and merged."""
    torch = torch_gpu
    for m in (n, 700, 9000):
        b = Batch(torch, [n], [m], 1, 1, d, form, f16, size=1000.0)
        b.pool.k.copy_(b.pool.k[0, 0, 0, 0].clone().expand_as(b.pool.k))
        top = float(b.pool.k[0, 0, 0, 0].float().abs().sum()) * 5000 * b.scale * 1.4427
        b.pool.ks.fill_(2.0 ** e / top)
        b.pool.vs.fill_(0.37)
        got = b.run(ctx).double()[:, 0]
        v = b.pool.values(b.slots(0), b.layer)[1][:, 0]
        want = (v.cumsum(0) / torch.arange(1, m + 1, device="cuda")[:, None])[m - n:]
        # sums of m terms, 1 / v_scale, a quotient; f16 queries' terms, all alike, are rounded to f16
        tol = (4 * math.sqrt(m) + 4) * U * v.abs().max() + (2 * f16_step(want) if f16 else 0)
        assert bool(((got - want).abs() <= tol).all()), (m, float(((got - want).abs() / tol).max()))


@pytest.mark.parametrize("n", ITEMS)
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("sign", [-1.0, 1.0])
def test_the_largest_scores(ctx, torch_gpu, sign, f16, n):
    """Queries, rows and the scale at the ends of their ranges: scores of 2^104 in size, where keys that are alike
    weigh the same."""
    torch = torch_gpu
    for m in (n, 700, 9000):
        b = Batch(torch, [n], [m], 1, 1, 128, "f8", f16)
        b.scale = 2.0 ** 32
        b.pool.k.copy_(torch.full(b.pool.k.shape, 448.0, device="cuda").to(b.pool.k.dtype))
        b.pool.ks.fill_(2.0 ** 40)
        b.pool.vs.fill_(0.37)
        b.q.fill_(sign * 65472.0)
        got = b.run(ctx).double()[:, 0]
        v = b.pool.values(b.slots(0), b.layer)[1][:, 0]
        want = (v.cumsum(0) / torch.arange(1, m + 1, device="cuda")[:, None])[m - n:]
        tol = (4 * math.sqrt(m) + 4) * U * v.abs().max() + (f16_step(want) if f16 else 0)
        assert bool(((got - want).abs() <= tol).all()), (m, float(((got - want).abs() / tol).max()))


@pytest.mark.parametrize("n", ITEMS)
@pytest.mark.parametrize("value", [math.inf, -math.inf])
def test_f16_queries_that_are_infinite(ctx, torch_gpu, value, n):
    """Scores that are all infinite, of either sign or both, make their row NaN in every kind of item, whole or cut, a
    tree's too, and no other row."""
    torch = torch_gpu
    for m, tree, signs in itertools.product((n, 700, 9000), (False, True), (1, 2)):
        # a tree behind it keeps 256 rows out of one item
        b = Batch(torch, [n] + tree * [4], [m] + tree * [m + 4], 1, 1, 128, "i8", True, trees=tree * [None, [-1, -1, 0, 1]])
        b.pool.k[..., 3] = 5 if signs == 1 else torch.where(b.pool.k[..., 3] < 0, -7, 7).to(torch.int8)
        clean = b.run(ctx)
        assert bool(clean.isfinite().all())
        rows = [0, n - 1] + tree * [n, n + 2]
        b.q[rows, 0, 3] = value
        got = b.run(ctx)
        nan = torch.zeros_like(got, dtype=torch.bool)
        nan[rows] = True
        assert torch.equal(got.isnan(), nan), (m, tree, signs, int((got.isnan() != nan).sum()))
        assert torch.equal(got[~nan], clean[~nan])


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("size,eps", [(1e-30, 0.0), (1e-21, 1e-40), (1e-10, 0.0), (1e18, 1e-6), (1e25, 1e-6), (1e37, 1e30)])
def test_norms_of_rows_of_every_size(ctx, torch_gpu, size, eps, form):
    """f32 rows whose squares leave f32's range are normed like others, beside rows of ordinary size."""
    torch = torch_gpu
    T, H, Hkv, d = 37, 3, 2, 128
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(T, H + 2 * Hkv, d, device="cuda", generator=g)
    x[::2, :H + Hkv] *= size
    gains = [1 + 0.3 * torch.randn(d, device="cuda", generator=g) for _ in "qk"]
    pool = Pool(torch, 1, 3, Hkv, 16, d, form)
    slots = torch.arange(T, device="cuda", dtype=torch.int32)
    q = store(ctx, torch, pool, 0, slots, x[:, :H], x[:, H:H + Hkv], x[:, H + Hkv:], q_gain=gains[0], k_gain=gains[1], eps=eps)
    eps = float(np.float32(eps))
    want, err = turned64(torch, x[:, :H], gains[0], eps, None, 0, 0, None, 1.0)
    # a product below f32's normal range is off by up to 2^-126
    assert bool(((q.double() - want).abs() <= err + U * want.abs() + 2.0 ** -126).all())
    gk, _ = pool.values(slots)
    check_rows(torch, pool, form, gk, *turned64(torch, x[:, H:H + Hkv], gains[1], eps, None, 0, 0, None, 1.0))


@pytest.mark.parametrize("H,Hkv,d,form", [(8, 2, 128, "i8"), (32, 1, 64, "f8"), (16, 16, 128, "f8")])
def test_f16_queries_of_few_rows_to_f32(ctx, torch_gpu, H, Hkv, d, form):
    """Single tokens, small trees and chunks of f16 queries are as near as f32 ones that hold the same values: the
    tolerance without an f16 term."""
    r = np.random.default_rng(2)
    most = 64 * Hkv // H
    extents = [1, 1, most, min(most, 12), 1, 2]
    lengths = [1, 9000, most + 300, 1500, 64, 700]
    b = Batch(torch_gpu, extents, lengths, H, Hkv, d, form, True, trees=[None, None, None, random_tree(r, extents[3], 4), None, None])
    got = b.run(ctx, out=torch_gpu.empty(b.q.shape, device="cuda"))
    b.q = b.q.float()
    b.check(got)
