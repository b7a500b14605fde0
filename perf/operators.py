"""Three operators beside the projections and paged attention, as cases that can be timed.

  rope       Context.rope: rotary positions over strided heads, interleaved or half
             layout, part of the head, frequencies scaled for long contexts.
  attention  Context.packed_attention: attention over packed sequences of different
             lengths whose K and V are plain f16 rows, causal or full, grouped heads;
             whole prompts, chunks of new tokens and single tokens.
  adapters   Context.adapters: the low-rank adapters of many requests added to a
             shared projection's output.

own = False computes them in their plain form, with elementary torch operations in
32 bits; own = True makes the calls of the library's Python API. listed() names the
cases, draw(rng) gives more of the same ranges, prepare() makes what a program holds
before the call, run() makes one call, work() counts the bytes and flops it cannot do
without, exact() restates it in 64 bits.
"""
import math
import random

import torch

own = False

# Query heads and kv heads: those of the 0.6B, 8B and 32B configurations in bench.py,
# then one head of keys for each of queries, and groups that are no power of two.
HEADS = [(16, 8), (32, 8), (64, 8), (16, 16), (24, 8), (28, 4)]
# Projections [K, N] as a layer of those configurations runs them (QKV and gate/up fused).
SHAPES = [(1024, 4096), (2048, 1024), (1024, 6144), (4096, 6144), (4096, 4096), (4096, 24576), (12288, 4096),
          (5120, 10240), (8192, 5120)]
LARGEST_PAIRS = 32 * 16384 * 16384 // 2   # query head x visible key pairs of the longest prompt listed
LARGEST_ADAPTED = 1152 * 24576 * 4        # output elements of the largest adapted projection drawn


def listed():
    return [
        # one sequence decoding: q, k rotated and v narrowed out of the fused QKV row
        dict(name="rope_decode_1", kind="rope", t=1, heads=32, kv_heads=8, d=128, rd=128, layout="interleaved",
             scaling="none", io="qkv", far=40960),
        # a mixed step of 128 decode rows and two 512-token chunks, a 131072-position context by parts
        dict(name="rope_step_1152", kind="rope", t=1152, heads=32, kv_heads=8, d=128, rd=128, layout="half",
             scaling="yarn", io="qkv", far=131072),
        # a prompt of 16384 tokens, f16 heads, half of each head rotated, frequencies scaled by bands
        dict(name="rope_prompt_16384", kind="rope", t=16384, heads=64, kv_heads=8, d=128, rd=64, layout="half",
             scaling="bands", io="f16", far=131072),
        # a batch of 64 decoding sequences over their own rows of keys
        dict(name="attn_decode_64", kind="attention", form="decode", n=64, lo=16, hi=8192, heads=32, kv_heads=8,
             d=128, causal=True, q="f32", lens=21),
        # chunks of new tokens behind long contexts
        dict(name="attn_chunk_4", kind="attention", form="chunk", n=4, lo=2048, hi=8192, heads=32, kv_heads=8,
             d=128, causal=True, q="f32", lens=22),
        # a batch of prompts of different lengths, packed
        dict(name="attn_prompts_16", kind="attention", form="prompt", n=16, lo=1, hi=2048, heads=32, kv_heads=8,
             d=128, causal=True, q="f16", lens=23),
        # texts embedded without a mask, heads of 64
        dict(name="attn_full_32", kind="attention", form="prompt", n=32, lo=16, hi=768, heads=16, kv_heads=16,
             d=64, causal=False, q="f32", lens=24),
        # one long prompt
        dict(name="attn_long_16384", kind="attention", form="prompt", n=1, lo=16384, hi=16384, heads=32, kv_heads=8,
             d=128, causal=True, q="f16", lens=25),
        # one request decoding beside the attention output projection
        dict(name="adapters_decode_1", kind="adapters", k=4096, n=4096, decodes=1, chunks=0, chunk=0, adapters=1,
             rank=16, x="f32", y="f32", lens=31),
        # 128 requests decoding with 32 adapters between them, fused QKV
        dict(name="adapters_decode_128", kind="adapters", k=4096, n=6144, decodes=128, chunks=0, chunk=0,
             adapters=32, rank=16, x="f32", y="f32", lens=32),
        # 128 decode rows beside two 512-token chunks, gate/up, activations as hi + lo pairs
        dict(name="adapters_step_1152", kind="adapters", k=4096, n=24576, decodes=128, chunks=2, chunk=512,
             adapters=32, rank=64, x="x2", y="f32", lens=33),
        # prompts alone in f16, the down projection, a rank that is no power of two
        dict(name="adapters_prompt_f16", kind="adapters", k=12288, n=4096, decodes=0, chunks=8, chunk=1000,
             adapters=5, rank=24, x="f16", y="f16", lens=34),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["rope", "attention", "attention", "adapters"])
    if kind == "rope":
        heads, kv = rng.choice(HEADS)
        d = rng.choice([64, 80, 96, 128, 128, 256])
        rd = rng.choice([d, d, d // 2, d // 4])
        t = _log_int(rng, 1, 16384)
        t = max(1, min(t, 16384 * 72 * 128 // (heads + 2 * kv) // d // 2))
        return dict(kind="rope", t=t, heads=heads, kv_heads=kv, d=d, rd=rd,
                    layout=rng.choice(["interleaved", "half"]),
                    scaling=rng.choice(["none", "linear", "yarn", "bands"]), io=rng.choice(["qkv", "f16"]),
                    far=_log_int(rng, 512, 1 << 20))
    if kind == "attention":
        heads, kv = rng.choice(HEADS)
        form = rng.choice(["decode", "chunk", "prompt", "prompt"])
        n = _log_int(rng, 1, 128 if form == "decode" else 24)
        hi = _log_int(rng, 64, 32768 if form == "decode" else 12288)
        lo = rng.randint(1, hi)
        case = dict(kind="attention", form=form, n=n, lo=lo, hi=hi, heads=heads, kv_heads=kv,
                    d=rng.choice([64, 128, 128]), causal=rng.random() < 0.75, q=rng.choice(["f32", "f16"]),
                    lens=rng.randint(0, 1 << 20))
        while (_attention_pairs(case) * heads * case["d"] > LARGEST_PAIRS * 128
               or sum(_lengths(case)[1]) * kv > 4194304):
            case["n"], case["hi"] = max(1, case["n"] * 2 // 3), max(64, case["hi"] * 3 // 4)
            case["lo"] = min(case["lo"], case["hi"])
        return case
    k, n = rng.choice(SHAPES)
    if rng.random() < 0.25:  # other widths a checkpoint may have
        k, n = 64 * _log_int(rng, 8, 160), 32 * _log_int(rng, 8, 320)
    decodes, chunks = rng.choice([(1, 0), (1, 0), (0, 1), (1, 1)])
    decodes *= _log_int(rng, 1, 256)
    chunks *= rng.randint(1, 6)
    chunk = _log_int(rng, 4, 2048) if chunks else 0
    while (decodes + chunks * chunk) * n > LARGEST_ADAPTED:
        chunk = chunk * 2 // 3
    x = rng.choice(["f32", "x2", "f16"])
    return dict(kind="adapters", k=k, n=n, decodes=decodes, chunks=chunks, chunk=chunk,
                adapters=min(decodes + chunks, _log_int(rng, 1, 64)), rank=rng.choice([1, 4, 8, 8, 16, 16, 20, 32, 64, 128]),
                x=x, y="f16" if x == "f16" else "f32", lens=rng.randint(0, 1 << 20))


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


_ctx = None


def _context():
    """The library's context: one per process, on torch's stream, as a program keeps it."""
    global _ctx
    import tgo_amd
    if _ctx is None:
        _ctx = tgo_amd.Context(0)
        _ctx.set_stream(torch.cuda.current_stream().cuda_stream)
    return _ctx


# The scaling of each kind: (factor, original context, fast, slow)
SCALINGS = {"none": (1.0, 0.0, 0.0, 0.0), "linear": (4.0, 0.0, 0.0, 0.0), "yarn": (4.0, 32768.0, 32.0, 1.0),
            "bands": (8.0, 8192.0, 4.0, 1.0)}
THETA = 1e6


def _positions(case, g):
    """One sequence's consecutive rows from a far start on, or decode rows anywhere."""
    t, far = case["t"], case["far"]
    if t <= 256:
        return torch.randint(0, far, (t,), device="cuda", generator=g, dtype=torch.int32)
    start = torch.randint(0, max(1, far - t), (1,), device="cuda", generator=g, dtype=torch.int32)
    return torch.arange(t, device="cuda", dtype=torch.int32) + start


class Rope:
    def __init__(self, case, seed):
        self.case = case
        g = _gen(seed)
        t, h, kv, d = case["t"], case["heads"], case["kv_heads"], case["d"]
        self.positions = _positions(case, g)
        if case["io"] == "qkv":
            # the fused projection's rows: q and k rotated (k into f16, as a cache holds it), v narrowed
            row = _randn(g, t, h + 2 * kv, d)
            self.x = [row[:, :h], row[:, h:h + kv], row[:, h + kv:]]
            self.turn = [True, True, False]
            types = [torch.float32, torch.float16, torch.float16]
        else:
            self.x = [_randn(g, t, h, d).half(), _randn(g, t, kv, d).half()]
            self.turn = [True, True]
            types = [torch.float16, torch.float16]
        if own:
            import tgo_amd
            self.ctx = _context()
            factor, original, fast, slow = SCALINGS[case["scaling"]]
            self.handle = self.ctx.rope_new(
                d, THETA, rotary_dim=case["rd"],
                layout=tgo_amd.ROPE_HALF if case["layout"] == "half" else tgo_amd.ROPE_INTERLEAVED,
                scaling={"none": tgo_amd.ROPE_UNSCALED, "linear": tgo_amd.ROPE_LINEAR, "yarn": tgo_amd.ROPE_YARN,
                         "bands": tgo_amd.ROPE_BANDS}[case["scaling"]],
                factor=factor, original=original, fast=fast, slow=slow)
        self.y = [torch.empty(x.shape, device="cuda", dtype=ty) for x, ty in zip(self.x, types)]

    def run(self):
        if own:
            self.ctx.rope(self.handle, self.positions, list(zip(self.x, self.y, self.turn)))
            return self.y
        return [self.plain(x, y.dtype) if turn else x.to(y.dtype) for x, y, turn in zip(self.x, self.y, self.turn)]

    def plain(self, x, dtype):
        c = self.case
        d, rd = c["d"], c["rd"]
        i = torch.arange(rd // 2, device="cuda", dtype=torch.float64)
        freq = THETA ** (-2 * i / rd)
        factor, original, fast, slow = SCALINGS[c["scaling"]]
        m = 1.0
        if c["scaling"] == "linear":
            freq = freq / factor
        elif c["scaling"] == "yarn":
            # the pairs that turn more than `fast` times over the original context keep their
            # frequency, those below `slow` turns are divided by factor, a ramp over the index between
            edge = lambda turns: rd * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(THETA))
            lo, hi = max(math.floor(edge(fast)), 0), min(math.ceil(edge(slow)), rd - 1)
            ramp = ((i - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
            freq = freq * (1 - ramp) + freq / factor * ramp
            m = 0.1 * math.log(factor) + 1.0
        elif c["scaling"] == "bands":
            # the same ends, and between them a ramp over the turns themselves
            turns = original * freq / (2 * math.pi)
            keep = ((turns - slow) / (fast - slow)).clamp(0, 1)
            freq = freq * keep + freq / factor * (1 - keep)
        angle = self.positions.double()[:, None] * freq[None, :]
        cos, sin = (angle.cos() * m).float()[:, None, :], (angle.sin() * m).float()[:, None, :]
        xf = x.float()
        head, rest = xf[..., :rd], xf[..., rd:]
        if c["layout"] == "half":
            a, b = head[..., :rd // 2], head[..., rd // 2:]
            turned = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
        else:
            a, b = head[..., 0::2], head[..., 1::2]
            turned = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
        return torch.cat([turned, rest], -1).to(dtype)

    def exact(self):
        c = self.case
        rd = c["rd"]
        w = []
        factor, original, fast, slow = SCALINGS[c["scaling"]]
        size = 1.0
        if c["scaling"] == "yarn":
            size = 1.0 + math.log(factor) / 10
            first = max(0, math.floor(math.log(original / fast / math.tau) * rd / math.log(THETA) / 2))
            last = min(rd - 1, math.ceil(math.log(original / slow / math.tau) * rd / math.log(THETA) / 2))
        for j in range(rd // 2):
            f = math.exp(-math.log(THETA) * 2 * j / rd)
            if c["scaling"] == "linear":
                f /= factor
            elif c["scaling"] == "yarn":
                share = min(1.0, max(0.0, (j - first) / max(last - first, 1e-3)))
                f = share * f / factor + (1 - share) * f
            elif c["scaling"] == "bands":
                wave = math.tau / f
                if wave > original / slow:
                    f /= factor
                elif wave > original / fast:
                    mix = (original / wave - slow) / (fast - slow)
                    f = (1 - mix) * f / factor + mix * f
            w.append(f)
        w = torch.tensor(w, device="cuda", dtype=torch.float64)
        turn = torch.polar(torch.full((1,), size, device="cuda", dtype=torch.float64),
                           torch.outer(self.positions.double(), w))[:, None, :]
        outs = []
        for x, rotated in zip(self.x, self.turn):
            x = x.double()
            if rotated:
                pairs = x[..., :rd].unflatten(-1, (2, rd // 2) if c["layout"] == "half" else (rd // 2, 2))
                axis = -2 if c["layout"] == "half" else -1
                z = torch.complex(pairs.select(axis, 0).contiguous(), pairs.select(axis, 1).contiguous()) * turn
                x = torch.cat([torch.stack([z.real, z.imag], axis).flatten(-2), x[..., rd:]], -1)
            outs.append(x)
        return outs

    def __del__(self):
        if getattr(self, "handle", None) is not None and self.ctx.h:
            self.ctx.rope_free(self.handle)


def _lengths(case):
    """(new tokens, keys) of each sequence."""
    r = random.Random(case["lens"])
    keys = [max(1, int(round(math.exp(r.uniform(math.log(case["lo"]), math.log(case["hi"]))))))
            for _ in range(case["n"])]
    if case["form"] == "decode":
        return [1] * len(keys), keys
    if case["form"] == "prompt":
        return list(keys), keys
    return [r.randint(1, max(1, min(512, l // 2))) for l in keys], keys


def _attention_pairs(case):
    """Visible (query, key) pairs."""
    q, k = _lengths(case)
    if not case["causal"]:
        return float(sum(n * m for n, m in zip(q, k)))
    return float(sum(n * (m - n) + n * (n + 1) // 2 for n, m in zip(q, k)))


class Attention:
    def __init__(self, case, seed):
        self.case = case
        g = _gen(seed)
        self.nq, self.nk = _lengths(case)
        h, kv, d = case["heads"], case["kv_heads"], case["d"]
        q = _randn(g, sum(self.nq), h, d)
        self.q = q.half() if case["q"] == "f16" else q
        self.k = _randn(g, sum(self.nk), kv, d).half()
        self.v = _randn(g, sum(self.nk), kv, d).half()
        self.scale = 1 / math.sqrt(d)
        if own:
            import tgo_amd
            self.ctx = _context()
            self.plan = self.ctx.packed_plan(self.nq, self.nk, h, kv, head_dim=d, causal=case["causal"],
                                             q_dtype=tgo_amd.F16 if case["q"] == "f16" else tgo_amd.F32)
            self.out = torch.empty_like(self.q)

    def run(self):
        if own:
            self.ctx.packed_attention(self.plan, self.q, self.k, self.v, self.out, self.scale)
            return self.out
        out = torch.empty_like(self.q)
        h, kv, d = self.case["heads"], self.case["kv_heads"], self.case["d"]
        group = h // kv
        tq = tk = 0
        for n, m in zip(self.nq, self.nk):
            k = self.k[tk:tk + m].float().permute(1, 2, 0).contiguous()  # [kv, d, m]
            v = self.v[tk:tk + m].float().transpose(0, 1).contiguous()   # [kv, m, d]
            rows = max(1, min(n, (1 << 28) // (h * m)))
            for i in range(0, n, rows):
                j = min(n, i + rows)
                q = self.q[tq + i:tq + j].float().reshape(j - i, kv, group, d).permute(1, 2, 0, 3)
                s = torch.matmul(q.reshape(kv, group * (j - i), d), k).mul_(self.scale).view(kv, group, j - i, m)
                if self.case["causal"]:
                    at = torch.arange(m - n + i, m - n + j, device="cuda")
                    s.masked_fill_(torch.arange(m, device="cuda")[None, :] > at[:, None], float("-inf"))
                s = s.sub_(s.amax(-1, keepdim=True)).exp_()
                total = s.sum(-1, keepdim=True)
                o = torch.matmul(s.view(kv, group * (j - i), m), v).view(kv, group, j - i, d) / total
                out[tq + i:tq + j] = o.permute(2, 0, 1, 3).reshape(j - i, h, d)
            tq, tk = tq + n, tk + m
        return out

    def exact(self):
        h, kv, d = self.case["heads"], self.case["kv_heads"], self.case["d"]
        group = h // kv
        out = torch.empty(self.q.shape, device="cuda", dtype=torch.float64)
        tq = tk = 0
        for n, m in zip(self.nq, self.nk):
            for head in range(kv):
                k = self.k[tk:tk + m, head].double()
                v = self.v[tk:tk + m, head].double()
                for i in range(0, n, 2048):
                    j = min(n, i + 2048)
                    last = m - n + j if self.case["causal"] else m
                    for sub in range(head * group, (head + 1) * group):
                        e = (self.q[tq + i:tq + j, sub].double() * self.scale) @ k[:last].t()
                        if self.case["causal"]:
                            e = e.masked_fill(torch.ones_like(e, dtype=torch.bool).triu(m - n + i + 1), -math.inf)
                        p = torch.exp(e - e.max(1, keepdim=True)[0])
                        out[tq + i:tq + j, sub] = (p @ v[:last]) / p.sum(1, keepdim=True)
            tq, tk = tq + n, tk + m
        return out

    def __del__(self):
        if getattr(self, "plan", None) is not None and self.ctx.h:
            self.ctx.packed_free(self.plan)


def _requests(case):
    """Each request's rows and adapter; one in eight carries none."""
    r = random.Random(case["lens"])
    extents = [1] * case["decodes"] + [case["chunk"]] * case["chunks"]
    some = list(range(case["adapters"]))
    who = [some[i] if i < len(some) else (-1 if r.random() < 0.125 else r.choice(some)) for i in range(len(extents))]
    r.shuffle(who)
    return extents, who


class Adapters:
    def __init__(self, case, seed):
        self.case = case
        g = _gen(seed)
        self.extents, self.who = _requests(case)
        m, k, n, r = sum(self.extents), case["k"], case["n"], case["rank"]
        x = _randn(g, m, k)
        if case["x"] == "x2":  # the pair a step's producers write
            hi = x.half()
            self.x = torch.stack([hi, (x - hi.float()).half()])
        else:
            self.x = x.half() if case["x"] == "f16" else x
        self.base = _randn(g, m, n)
        if case["y"] == "f16":
            self.base = self.base.half()
        # trained adapters: rows of down of about unit length, up small; scales of 2, a little apart
        self.down = (_randn(g, case["adapters"], r, k) / math.sqrt(k)).half()
        self.up = (_randn(g, case["adapters"], n, r) * 0.02).half()
        self.scales = [2.0 + 0.125 * (a % 5) for a in range(case["adapters"])]
        rows = torch.tensor(self.who).repeat_interleave(torch.tensor(self.extents))
        self.rows = [(rows == a).nonzero().flatten().cuda() for a in range(case["adapters"])]
        if own:
            import tgo_amd
            self.ctx = _context()
            self.set = self.ctx.adapters_new(k, n, case["adapters"])
            down, up = self.down.cpu().numpy(), self.up.cpu().numpy()
            for a in range(case["adapters"]):
                self.ctx.adapters_put(self.set, a, down[a], up[a], self.scales[a])
            self.plan = self.ctx.adapter_rows(self.extents, self.who)
            self.y = torch.empty_like(self.base)
            self.x_dtype = {"f32": tgo_amd.F32, "f16": tgo_amd.F16, "x2": tgo_amd.F16X2}[case["x"]]
            self.y_dtype = tgo_amd.F16 if case["y"] == "f16" else tgo_amd.F32

    def run(self):
        if own:
            self.ctx.adapters(self.set, self.plan, self.x, self.base, self.y, x_dtype=self.x_dtype,
                              y_dtype=self.y_dtype)
            return self.y
        y = self.base.float() if self.case["y"] == "f16" else self.base.clone()
        for a, rows in enumerate(self.rows):
            x = self.x[0, rows].float() + self.x[1, rows].float() if self.case["x"] == "x2" else self.x[rows].float()
            u = torch.matmul(x, self.down[a].float().t().contiguous())
            y.index_add_(0, rows, torch.matmul(u, self.up[a].float().t().contiguous()), alpha=self.scales[a])
        return y.to(self.base.dtype)

    def exact(self):
        x = self.x.double()
        if self.case["x"] == "x2":
            x = x[0] + x[1]
        y = self.base.double()
        at = 0
        for extent, a in zip(self.extents, self.who):
            if a >= 0:
                u = x[at:at + extent] @ self.down[a].double().t()
                y[at:at + extent] += self.scales[a] * (u @ self.up[a].double().t())
            at += extent
        return y

    def __del__(self):
        if getattr(self, "plan", None) is not None and self.ctx.h:
            self.ctx.adapter_rows_free(self.plan)
        if getattr(self, "set", None) is not None and self.ctx.h:
            self.ctx.adapters_free(self.set)


KINDS = {"rope": Rope, "attention": Attention, "adapters": Adapters}


def prepare(case, seed):
    return KINDS[case["kind"]](case, seed)


def run(state):
    return state.run()


def exact(case, seed):
    return KINDS[case["kind"]](case, seed).exact()


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    if case["kind"] == "rope":
        t, d, h, kv = case["t"], case["d"], case["heads"], case["kv_heads"]
        if case["io"] == "qkv":
            by = t * d * (h * 8.0 + 2 * kv * 6.0)
        else:
            by = t * d * (h + kv) * 4.0
        return dict(bytes=by + 4.0 * t, flops=3.0 * t * (h + kv) * case["rd"])
    if case["kind"] == "attention":
        q, k = _lengths(case)
        size = 2 if case["q"] == "f16" else 4
        return dict(bytes=2.0 * sum(q) * case["heads"] * case["d"] * size + 4.0 * sum(k) * case["kv_heads"] * case["d"],
                    flops=4.0 * case["d"] * case["heads"] * _attention_pairs(case))
    extents, who = _requests(case)
    m, used = sum(extents), len({a for a in who if a >= 0})
    adapted = sum(n for n, a in zip(extents, who) if a >= 0)
    k, n, r = case["k"], case["n"], case["rank"]
    return dict(bytes=adapted * k * (2.0 if case["x"] == "f16" else 4.0) + 2 * m * n * (2.0 if case["y"] == "f16" else 4.0) +
                used * r * (k + n) * 2.0, flops=2.0 * adapted * r * (k + n))
