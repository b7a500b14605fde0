"""Four operators of an 8-bit paged cache, as cases that can be timed.

  store      Context.cache_store: queries and keys normed per head and rotated, keys and values
             quantised to 8 bits and written to their slots of the cache, in one pass; then
             Context.cache_read of the rows written.
  attention  Context.cache_attention: attention over that cache by page table: single tokens,
             chunks of new tokens, trees of drafted tokens.
  read       Context.cache_read: slots of the cache back as rows.
  move       Context.cache_move: the accepted tokens' rows to their places, in every layer.

A cache holds int8 or e4m3 codes [layers, pages, kv_heads, block, head_dim] and a float32 scale
per row [layers, pages, kv_heads, block]: a row's scale is its largest magnitude over 127 or 448
(at least 2^-40), its codes the nearest to value / scale.

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

# Query heads and kv heads: those of the 0.6B, 8B and 32B configurations in bench.py, then one
# head of keys for each of queries, and groups that are no power of two.
HEADS = [(16, 8), (32, 8), (64, 8), (16, 16), (24, 8), (28, 4)]
EPS = 1e-6
THETA = 1e6
TOP = {"i8": 127.0, "f8": 448.0}
MOST_PAIRS = 32 * 2048 * 32768       # query heads x padded pairs of the largest attention listed
MOST_KEYS = 128 * 8192 * 8 * 128     # padded key elements of the largest decoding batch listed


def listed():
    return [
        # one sequence decoding: q, k, v of the fused QKV row into its cache slot
        dict(name="store_decode_1", kind="store", t=1, heads=32, kv_heads=8, d=128, rd=128, layout="interleaved",
             io="f32", form="i8", norm=True, block=32, far=40960, dropped=0),
        # a mixed step of 128 decode rows and two 512-token chunks
        dict(name="store_step_1152", kind="store", t=1152, heads=32, kv_heads=8, d=128, rd=128, layout="half",
             io="f32", form="f8", norm=True, block=16, far=131072, dropped=0),
        # a prompt of 16384 tokens in f16, half of each head rotated
        dict(name="store_prompt_16384", kind="store", t=16384, heads=64, kv_heads=8, d=128, rd=64, layout="half",
             io="f16", form="i8", norm=True, block=32, far=131072, dropped=0),
        # one long conversation decoding: latency
        dict(name="attend_decode_1", kind="attention", form="decode", n=1, lo=8192, hi=8192, new=1, heads=32,
             kv_heads=8, d=128, cache="i8", q="f32", block=32, lens=41),
        # a batch of 128 decoding sequences of all lengths
        dict(name="attend_decode_128", kind="attention", form="decode", n=128, lo=16, hi=8192, new=1, heads=32,
             kv_heads=8, d=128, cache="i8", q="f32", block=16, lens=42),
        # 32 sequences verifying trees of up to 64 drafted tokens
        dict(name="attend_tree_32", kind="attention", form="tree", n=32, lo=256, hi=4096, new=64, heads=32,
             kv_heads=8, d=128, cache="i8", q="f32", block=32, lens=43),
        # chunks of new tokens behind long contexts, e4m3
        dict(name="attend_chunk_4", kind="attention", form="chunk", n=4, lo=2048, hi=8192, new=512, heads=32,
             kv_heads=8, d=128, cache="f8", q="f32", block=16, lens=44),
        # the last chunk of a long prompt, f16 queries
        dict(name="attend_chunk_32768", kind="attention", form="chunk", n=1, lo=32768, hi=32768, new=2048, heads=32,
             kv_heads=8, d=128, cache="i8", q="f16", block=32, lens=45),
        # a shared prefix read back for a kernel that wants f16 rows
        dict(name="read_prefix_2048", kind="read", n=2048, kv_heads=8, d=128, form="i8", y="f16", block=32),
        # a whole context
        dict(name="read_context_131072", kind="read", n=131072, kv_heads=8, d=128, form="f8", y="f16", block=16),
        # one sequence's accepted path of a tree, every layer of the 8B configuration
        dict(name="move_1", kind="move", layers=36, n=1, new=16, kv_heads=8, d=128, form="i8", block=32, lens=51),
        # a batch's
        dict(name="move_64", kind="move", layers=36, n=64, new=64, kv_heads=8, d=128, form="i8", block=16, lens=52),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["store", "store", "attention", "attention", "attention", "read", "move"])
    heads, kv = rng.choice(HEADS)
    form, block, d = rng.choice(["i8", "f8"]), rng.choice([16, 32, 64]), rng.choice([64, 128, 128])
    if kind == "store":
        t = _log_int(rng, 1, 16384)
        t = max(1, min(t, 16384 * 80 * 128 // (heads + 2 * kv) // d // 2))
        return dict(kind="store", t=t, heads=heads, kv_heads=kv, d=d, rd=rng.choice([d, d, d // 2, d // 4, 3 * d // 4]),
                    layout=rng.choice(["interleaved", "half"]), io=rng.choice(["f32", "f16"]), form=form,
                    norm=rng.random() < 0.75, block=block, far=_log_int(rng, 512, 1 << 20),
                    dropped=rng.choice([0, 0, t // 3]))
    if kind == "read":
        return dict(kind="read", n=min(_log_int(rng, 1, 131072), 131072 * 1024 // (kv * d)), kv_heads=kv, d=d, form=form,
                    y=rng.choice(["f32", "f16"]) if kv * d <= 512 else "f16", block=block)
    if kind == "move":
        return dict(kind="move", layers=rng.choice([28, 36]), n=_log_int(rng, 1, 64), new=_log_int(rng, 4, 64),
                    kv_heads=min(kv, 8), d=d, form=form, block=block, lens=rng.randint(0, 1 << 20))
    f = rng.choice(["decode", "tree", "chunk"])
    n = _log_int(rng, 1, {"decode": 128, "tree": 48, "chunk": 12}[f])
    hi = _log_int(rng, 64, 32768)
    new = 1 if f == "decode" else _log_int(rng, 2, 64) if f == "tree" else _log_int(rng, 16, 2048)
    while n * new * hi * heads > MOST_PAIRS or n * hi * kv * d > MOST_KEYS:
        if n > 1:
            n = n * 2 // 3
        else:
            new, hi = max(1, new * 2 // 3), max(64, hi * 3 // 4)
    return dict(kind="attention", form=f, n=n, lo=rng.randint(1, hi), hi=hi, new=new, heads=heads, kv_heads=kv, d=d,
                cache=form, q=rng.choice(["f32", "f16"]), block=block, lens=rng.randint(0, 1 << 20))


# ---------------------------------------------------------------------------
# the cache
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


def _code_type(form):
    return torch.int8 if form == "i8" else torch.float8_e4m3fn


class Pool:
    """k, v codes and their rows' scales."""

    def __init__(self, layers, pages, kv, block, d, form):
        self.form, self.block, self.capacity = form, block, pages * block
        shape = (layers, pages, kv, block, d)
        self.k, self.v = (torch.zeros(shape, device="cuda", dtype=torch.uint8).view(_code_type(form)) for _ in range(2))
        self.k_scale, self.v_scale = (torch.zeros(shape[:4], device="cuda") for _ in range(2))

    def fill(self, g, spread):
        """What an earlier store left: rows of about unit size, some far larger than others."""
        for codes, scale, s in ((self.k, self.k_scale, spread / 2), (self.v, self.v_scale, spread)):
            for layer in range(codes.shape[0]):
                x = _randn(g, *codes.shape[1:])
                codes[layer] = (x * 42).round_().clamp_(-127, 127).to(torch.int8) if self.form == "i8" else \
                    (x * 150).clamp_(-448, 448).to(torch.float8_e4m3fn)
            scale.copy_((_randn(g, *scale.shape) * s).exp_() * (3 / TOP[self.form]))
        return self

    def handle(self):
        import tgo_amd
        return tgo_amd.Cache(self.k, self.v, self.k_scale, self.v_scale)

    def rows(self, codes, scale, slots, dtype):
        """The values of slots (any shape) of layer 0: [..., kv_heads, d]; none outside the pool."""
        inside = (slots >= 0) & (slots < self.capacity)
        at = torch.where(inside, slots, 0).long()
        page, off = at // self.block, at % self.block
        c = codes[0].view(torch.uint8)[page, :, off].view(codes.dtype)
        return torch.where(inside[..., None, None], c.to(dtype) * scale[0][page, :, off][..., None].to(dtype), 0.0)


# ---------------------------------------------------------------------------
# norm, rotate, quantise, write; read back
# ---------------------------------------------------------------------------

class Store:
    def __init__(self, case, seed):
        self.case = case
        g = _gen(seed)
        t, h, kv, d, block = case["t"], case["heads"], case["kv_heads"], case["d"], case["block"]
        row = _randn(g, t, h + 2 * kv, d) * 1.5
        self.row = row.half() if case["io"] == "f16" else row
        self.q, self.k, self.v = self.row[:, :h], self.row[:, h:h + kv], self.row[:, h + kv:]
        self.q_gain, self.k_gain = (1 + 0.2 * _randn(g, d) for _ in range(2))
        if t <= 256:  # decode rows anywhere
            self.positions = torch.randint(0, case["far"], (t,), device="cuda", generator=g, dtype=torch.int32)
        else:
            self.positions = torch.arange(t, device="cuda", dtype=torch.int32) + int(seed) % case["far"]
        pages = (t + block - 1) // block + 3
        self.pool = Pool(1, pages, kv, block, d, case["form"])
        order = torch.randperm(pages, device="cuda", generator=g)
        i = torch.arange(t, device="cuda")
        self.slots = (order[i // block] * block + i % block).int()
        if case["dropped"]:  # a bucket's padding rows
            self.slots[t - case["dropped"]:] = self.pool.capacity
        self.q_out = torch.empty(t, h, d, device="cuda", dtype=self.row.dtype)
        self.k_out, self.v_out = (torch.empty(t, kv, d, device="cuda", dtype=torch.float16) for _ in range(2))
        if own:
            import tgo_amd
            self.ctx = _context()
            self.cache = self.pool.handle()
            self.rope = self.ctx.rope_new(d, THETA, rotary_dim=case["rd"], layout=tgo_amd.ROPE_HALF
                                          if case["layout"] == "half" else tgo_amd.ROPE_INTERLEAVED)

    def run(self):
        gains = (self.q_gain, self.k_gain) if self.case["norm"] else (None, None)
        if own:
            self.ctx.cache_store(self.cache, 0, self.slots, self.k, self.v, self.q, self.q_out, positions=self.positions,
                                 rope=self.rope, q_gain=gains[0], k_gain=gains[1], eps=EPS)
            self.ctx.cache_read(self.cache, 0, self.slots, self.k_out, self.v_out)
            return self.q_out, self.k_out, self.v_out
        q, k = self.turned(self.q, gains[0]), self.turned(self.k, gains[1])
        self.write(self.pool.k, self.pool.k_scale, k)
        self.write(self.pool.v, self.pool.v_scale, self.v.float())
        p = self.pool
        return (q.to(self.row.dtype), p.rows(p.k, p.k_scale, self.slots, torch.float32).half(),
                p.rows(p.v, p.v_scale, self.slots, torch.float32).half())

    def turned(self, x, gain):
        c = self.case
        x = x.float()
        if gain is not None:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * gain
        rd = c["rd"]
        freq = THETA ** (-2 * torch.arange(rd // 2, device="cuda", dtype=torch.float64) / rd)
        angle = self.positions.double()[:, None] * freq
        cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
        head, rest = x[..., :rd], x[..., rd:]
        if c["layout"] == "half":
            a, b = head[..., :rd // 2], head[..., rd // 2:]
            head = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
        else:
            a, b = head[..., 0::2], head[..., 1::2]
            head = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
        return torch.cat([head, rest], -1)

    def write(self, codes, scale, y):
        keep = self.slots < self.pool.capacity
        at = self.slots[keep].long()
        y = y[keep]
        s = (y.abs().amax(-1) / TOP[self.case["form"]]).clamp_min_(2.0 ** -40)
        c = y / s[..., None]
        c = c.round_().to(torch.int8) if self.case["form"] == "i8" else c.to(torch.float8_e4m3fn)
        page, off = at // self.case["block"], at % self.case["block"]
        codes[0].view(torch.uint8)[page, :, off] = c.view(torch.uint8)
        scale[0][page, :, off] = s

    def exact(self):
        c = self.case
        rd = c["rd"]
        turn = torch.polar(torch.ones(1, device="cuda", dtype=torch.float64), torch.outer(
            self.positions.double(), torch.tensor([math.exp(-2 * j / rd * math.log(THETA)) for j in range(rd // 2)],
                                                  device="cuda", dtype=torch.float64)))[:, None]
        outs = []
        for x, gain in ((self.q, self.q_gain), (self.k, self.k_gain), (self.v, None)):
            x = x.double()
            if gain is not None:
                if c["norm"]:
                    x = gain.double() * x / (x.square().sum(-1, keepdim=True) / c["d"] + EPS).sqrt()
                pairs = x[..., :rd].unflatten(-1, (2, rd // 2) if c["layout"] == "half" else (rd // 2, 2))
                axis = -2 if c["layout"] == "half" else -1
                z = torch.complex(pairs.select(axis, 0).contiguous(), pairs.select(axis, 1).contiguous()) * turn
                x = torch.cat([torch.stack([z.real, z.imag], axis).flatten(-2), x[..., rd:]], -1)
            outs.append(x)
        for i in (1, 2):
            scale = torch.maximum(outs[i].abs().max(-1, keepdim=True)[0] / TOP[c["form"]],
                                  torch.tensor(2.0 ** -40, device="cuda", dtype=torch.float64))
            y = outs[i] / scale
            if c["form"] == "i8":
                y = torch.round(y)
            else:  # three bits behind the leading one, down to 2^-9
                step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)
                y = torch.round(y / step) * step
            outs[i] = y * scale * (self.slots < self.pool.capacity)[:, None, None]
        return outs

    def __del__(self):
        if getattr(self, "rope", None) is not None and self.ctx.h:
            self.ctx.rope_free(self.rope)


class Read:
    def __init__(self, case, seed):
        self.case = case
        g = _gen(seed)
        n, kv, d, block = case["n"], case["kv_heads"], case["d"], case["block"]
        pages = (n + block - 1) // block + 2
        self.pool = Pool(1, pages, kv, block, d, case["form"]).fill(g, 0.7)
        order = torch.randperm(pages, device="cuda", generator=g)
        i = torch.arange(n, device="cuda")
        self.slots = (order[i // block] * block + i % block).int()
        y = torch.float16 if case["y"] == "f16" else torch.float32
        self.k_out, self.v_out = (torch.empty(n, kv, d, device="cuda", dtype=y) for _ in range(2))
        if own:
            self.ctx = _context()
            self.cache = self.pool.handle()

    def run(self):
        if own:
            self.ctx.cache_read(self.cache, 0, self.slots, self.k_out, self.v_out)
            return self.k_out, self.v_out
        p = self.pool
        return tuple(p.rows(c, s, self.slots, torch.float32).to(self.k_out.dtype)
                     for c, s in ((p.k, p.k_scale), (p.v, p.v_scale)))

    def exact(self):
        at = self.slots.long()
        outs = []
        for codes, scale in ((self.pool.k, self.pool.k_scale), (self.pool.v, self.pool.v_scale)):
            flat = codes[0].double().transpose(1, 2).flatten(0, 1)
            outs.append(flat[at] * scale[0].double().transpose(1, 2).flatten(0, 1)[at][..., None])
        return outs


def _tree(r, n, wide):
    """Parents of n drafted tokens (-1: the context), children of the last few."""
    return [-1 if i == 0 or r.random() < 0.08 else r.randint(max(0, i - wide), i - 1) for i in range(n)]


class Move:
    def __init__(self, case, seed):
        self.case = case
        g = _gen(seed)
        n, new, block = case["n"], case["new"], case["block"]
        per = (new + 2 * block - 2) // block
        self.pool = Pool(case["layers"], n * per + 1, case["kv_heads"], block, case["d"], case["form"]).fill(g, 0.7)
        order = torch.randperm(n * per + 1, generator=torch.Generator().manual_seed(int(seed))).tolist()
        self.src, self.dst = [], []
        for s, (first, path) in enumerate(_accepted(case)):
            slot = lambda p: order[s * per + p // block] * block + p % block  # noqa: E731
            self.src += [slot(first + p) for p in path]
            self.dst += [slot(first + i) for i in range(len(path))]
        if own:
            self.ctx = _context()
            self.cache = self.pool.handle()

    def run(self):
        p = self.pool
        if own:
            self.ctx.cache_move(self.cache, self.src, self.dst)
        else:
            src, dst = (torch.tensor(x, device="cuda") for x in (self.src, self.dst))
            b = p.block
            for codes, scale in ((p.k.view(torch.uint8), p.k_scale), (p.v.view(torch.uint8), p.v_scale)):
                codes[:, dst // b, :, dst % b] = codes[:, src // b, :, src % b]
                scale[:, dst // b, :, dst % b] = scale[:, src // b, :, src % b]
        return p.k.view(torch.int8), p.v.view(torch.int8), p.k_scale, p.v_scale

    def exact(self):
        outs = []
        b = self.pool.block
        for t in (self.pool.k.view(torch.int8), self.pool.v.view(torch.int8), self.pool.k_scale, self.pool.v_scale):
            new = t.clone()
            for s, e in zip(self.src, self.dst):
                new[:, e // b, :, e % b] = t[:, s // b, :, s % b]
            outs.append(new.double() if new.is_floating_point() else None)
        return outs


def _accepted(case):
    """Each sequence's first drafted position within its page, and the accepted path of its tree."""
    r = random.Random(case["lens"])
    out = []
    for _ in range(case["n"]):
        n = r.randint(max(2, case["new"] // 2), case["new"])
        parents = _tree(r, n, 4)
        at, path = r.randrange(n), []
        while at >= 0:
            path.append(at)
            at = parents[at]
        out.append((r.randrange(case["block"]), path[::-1]))
    return out


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------

def _batch(case):
    """(new tokens, positions, parents) of each sequence."""
    r = random.Random(case["lens"])
    extents, lengths, parents = [], [], []
    for _ in range(case["n"]):
        l = max(1, int(round(math.exp(r.uniform(math.log(case["lo"]), math.log(case["hi"]))))))
        n = 1 if case["form"] == "decode" else min(l, r.randint(max(1, case["new"] // 4), case["new"]))
        if case["form"] == "chunk" and case["n"] == 1:
            n = min(l, case["new"])
        extents.append(n)
        lengths.append(l)
        parents.append(_tree(r, n, 6) if case["form"] == "tree" else list(range(-1, n - 1)))
    return extents, lengths, parents


def _seen(parents):
    """Ancestors of each token, itself among them: [n, n] truth values."""
    n = len(parents)
    seen = torch.zeros(n, n, dtype=torch.bool)
    for i, p in enumerate(parents):
        if p >= 0:
            seen[i] = seen[p]
        seen[i, i] = True
    return seen


class Attention:
    def __init__(self, case, seed):
        self.case = case
        g = _gen(seed)
        self.extents, self.lengths, self.parents = _batch(case)
        h, kv, d, block = case["heads"], case["kv_heads"], case["d"], case["block"]
        need = [(l + block - 1) // block for l in self.lengths]
        pages = sum(need) + 2
        self.pool = Pool(1, pages, kv, block, d, case["cache"]).fill(g, 0.7)
        order = torch.randperm(pages, generator=torch.Generator().manual_seed(int(seed)))
        self.pages = torch.zeros(case["n"], max(need), dtype=torch.int32)
        at = 0
        for s, m in enumerate(need):
            self.pages[s, :m] = order[at:at + m]
            at += m
        q = _randn(g, sum(self.extents), h, d)
        self.q = q.half() if case["q"] == "f16" else q
        self.scale = 1 / math.sqrt(d)
        if own:
            import tgo_amd
            self.ctx = _context()
            self.cache = self.pool.handle()
            self.plan = self.ctx.cache_plan(self.cache, self.extents, self.lengths, self.pages.numpy(), h,
                                            parents=sum(self.parents, []) if case["form"] == "tree" else None,
                                            q_dtype=tgo_amd.F16 if case["q"] == "f16" else tgo_amd.F32)
            self.out = torch.empty_like(self.q)
            return
        # the plain form's plan: the page table, each token's place in a batch padded to the longest
        # sequence, which tokens see which of the new ones
        most = max(self.extents)
        self.table = self.pages.cuda().long()
        self.base = (torch.tensor(self.lengths) - torch.tensor(self.extents)).cuda()
        self.place = torch.cat([torch.arange(n) + s * most for s, n in enumerate(self.extents)]).cuda()
        self.new = None
        if case["form"] == "tree":
            seen = torch.zeros(case["n"], most, most, dtype=torch.bool)
            for s, p in enumerate(self.parents):
                seen[s, :len(p), :len(p)] = _seen(p)
            self.new = seen.cuda()

    def run(self):
        if own:
            self.ctx.cache_attention(self.plan, self.cache, 0, self.q, self.out, self.scale)
            return self.out
        c, p = self.case, self.pool
        h, kv, d, n = c["heads"], c["kv_heads"], c["d"], c["n"]
        most, longest, group = max(self.extents), max(self.lengths), h // kv
        pos = torch.arange(longest, device="cuda")
        slots = self.table[:, pos // c["block"]] * c["block"] + pos % c["block"]
        k = p.rows(p.k, p.k_scale, slots, torch.float32).permute(0, 2, 3, 1).contiguous()
        v = p.rows(p.v, p.v_scale, slots, torch.float32).transpose(1, 2).contiguous()
        q = torch.zeros(n * most, h, d, device="cuda")
        q[self.place] = self.q.float()
        q = q.view(n, most, kv, group, d).permute(0, 2, 3, 1, 4).reshape(n, kv, group * most, d)
        s = torch.matmul(q, k).mul_(self.scale).view(n, kv, group, most, longest)
        rel = pos - self.base[:, None]                                      # [n, longest]
        token = torch.arange(most, device="cuda")
        if self.new is None:
            visible = rel[:, None] <= token[None, :, None]
        else:
            at = rel.clamp(0, most - 1)[:, None].expand(n, most, longest)
            visible = (rel < 0)[:, None] | (self.new.gather(2, at) & (rel < most)[:, None])
        s.masked_fill_(~visible[:, None, None], float("-inf"))
        s = s.sub_(s.amax(-1, keepdim=True)).exp_()
        total = s.sum(-1, keepdim=True)
        o = torch.matmul(s.view(n, kv, group * most, longest), v).view(n, kv, group, most, d) / total
        return o.permute(0, 3, 1, 2, 4).reshape(n * most, h, d)[self.place].to(self.q.dtype)

    def exact(self):
        h, kv, d, block = self.case["heads"], self.case["kv_heads"], self.case["d"], self.case["block"]
        group = h // kv
        out = torch.empty(self.q.shape, device="cuda", dtype=torch.float64)
        t = 0
        for s, (n, m) in enumerate(zip(self.extents, self.lengths)):
            page = self.pages[s, :(m + block - 1) // block].cuda().long()
            hidden = torch.zeros(n, m, dtype=torch.bool)
            if self.case["form"] == "tree":
                hidden[:, m - n:] = True
                for i in range(n):
                    a = i
                    while a >= 0:
                        hidden[i, m - n + a] = False
                        a = self.parents[s][a]
            else:
                hidden = torch.ones(n, m, dtype=torch.bool, device="cuda").triu(m - n + 1)
            hidden = hidden.cuda()
            for head in range(kv):
                k, v = (self._rows64(codes, scale, page, head)[:m] for codes, scale in
                        ((self.pool.k, self.pool.k_scale), (self.pool.v, self.pool.v_scale)))
                for sub in range(head * group, (head + 1) * group):
                    e = (self.q[t:t + n, sub].double() @ k.t().contiguous()) * self.scale
                    e = e.masked_fill(hidden, -math.inf)
                    w = torch.exp(e - e.max(1, keepdim=True)[0])
                    out[t:t + n, sub] = (w / w.sum(1, keepdim=True)) @ v
            t += n
        return out

    def _rows64(self, codes, scale, page, head):
        c = codes[0, :, head].contiguous().view(torch.uint8)[page].view(codes.dtype)
        return (c.double() * scale[0, :, head][page].double()[..., None]).flatten(0, 1)

    def __del__(self):
        if getattr(self, "plan", None) is not None and self.ctx.h:
            self.ctx.cache_plan_free(self.plan)


KINDS = {"store": Store, "read": Read, "move": Move, "attention": Attention}


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
    kv, d = case["kv_heads"], case["d"]
    if case["kind"] == "store":
        t, h, size = case["t"], case["heads"], 4.0 if case["io"] == "f32" else 2.0
        # rows in, queries out, codes and scales written and read back, f16 rows out
        by = t * d * ((h + 2 * kv) * size + h * size) + (t - case["dropped"]) * 2 * kv * 2.0 * (d + 4) + t * 2 * kv * d * 2.0
        return dict(bytes=by + 8.0 * t, flops=t * (h + kv) * (3.0 * case["rd"] + 4.0 * d))
    if case["kind"] == "read":
        return dict(bytes=case["n"] * (2.0 * kv * (d + 4 + d * (2 if case["y"] == "f16" else 4)) + 4), flops=2.0 * case["n"] * kv * d)
    if case["kind"] == "move":
        moved = sum(sum(i != a for i, a in enumerate(path)) for _, path in _accepted(case))
        return dict(bytes=case["layers"] * max(1, moved) * 2.0 * kv * 2 * (d + 4), flops=0.0)
    extents, lengths, parents = _batch(case)
    size = 2 if case["q"] == "f16" else 4
    pairs = 0.0
    for n, m, p in zip(extents, lengths, parents):
        pairs += n * (m - n) + (int(_seen(p).sum()) if case["form"] == "tree" else n * (n + 1) // 2)
    return dict(bytes=2.0 * sum(extents) * case["heads"] * d * size + sum(lengths) * 2.0 * kv * (d + 4),
                flops=4.0 * d * case["heads"] * pairs)
