"""Rotary frequencies (tgohip_rope_freqs) against their definitions, and the refusals of the
rotary, packed-attention and adapter entry points that need no GPU: every argument a handle is
made from is checked before the context is touched."""
import ctypes
import math

import numpy as np
import pytest

import tgo_amd
from tgo_amd import TgoError

NAN = float("nan")
YARN = dict(scaling=tgo_amd.ROPE_YARN, factor=4.0, original=32768.0, fast=32.0, slow=1.0)
BANDS = dict(scaling=tgo_amd.ROPE_BANDS, factor=8.0, original=8192.0, fast=4.0, slow=1.0)


def by_hand(rd, base, scaling, factor, original, fast, slow):
    w = []
    for i in range(rd // 2):
        f = base ** (-2 * i / rd)
        wave = 2 * math.pi / f  # positions per turn
        if scaling == tgo_amd.ROPE_LINEAR:
            f /= factor
        elif scaling == tgo_amd.ROPE_YARN:
            at = lambda turns: rd / 2 * math.log(original / (2 * math.pi * turns), base)  # the pair with `turns` turns
            lo, hi = max(0, math.floor(at(fast))), min(rd - 1, math.ceil(at(slow)))
            t = min(1, max(0, (i - lo) / max(hi - lo, 1e-3)))
            f = (1 - t) * f + t * f / factor
        elif scaling == tgo_amd.ROPE_BANDS:
            if wave > original / slow:
                f /= factor
            elif wave > original / fast:
                t = (original / wave - slow) / (fast - slow)
                f = t * f + (1 - t) * f / factor
        w.append(f)
    return np.array(w)


@pytest.mark.parametrize("rd", [2, 32, 96, 128, 256])
@pytest.mark.parametrize("kw", [dict(), dict(scaling=tgo_amd.ROPE_LINEAR, factor=2.5), YARN, BANDS,
                                dict(YARN, original=64.0), dict(BANDS, factor=1.0)])
def test_rope_frequencies(rd, kw):
    w, m = tgo_amd.rope_freqs(256, 1e6, rotary_dim=rd, **kw)
    full = dict(dict(scaling=tgo_amd.ROPE_UNSCALED, factor=1.0, original=0.0, fast=0.0, slow=0.0), **kw)
    # both sides are a few float64 operations on exp and log
    assert np.allclose(w, by_hand(rd, 1e6, **full), rtol=1e-13, atol=0)
    want = 0.1 * math.log(full["factor"]) + 1 if full["scaling"] == tgo_amd.ROPE_YARN else 1.0
    assert abs(m - want) < 1e-15
    assert tgo_amd.rope_freqs(256, 1e6, rotary_dim=rd, attention=1.25, **kw)[1] == 1.25


def test_scaled_frequencies_keep_the_fast_pairs_and_stretch_the_slow_ones():
    plain, _ = tgo_amd.rope_freqs(128, 1e6)
    for kw in (YARN, BANDS):
        w, _ = tgo_amd.rope_freqs(128, 1e6, **kw)
        assert w[0] == plain[0]
        assert abs(w[-1] * kw["factor"] / plain[-1] - 1) < 1e-14
        assert (np.diff(w) < 0).all()


@pytest.mark.parametrize("change,word", [
    (dict(head_dim=0), "head_dim is 0"), (dict(head_dim=7), "head_dim is 7"), (dict(head_dim=258), "head_dim is 258"),
    (dict(rotary_dim=0), "rotary_dim is 0"), (dict(rotary_dim=5), "rotary_dim is 5"),
    (dict(rotary_dim=130), "rotary_dim is 130 of head_dim 128"), (dict(layout=2), "layout is 2"),
    (dict(scaling=4), "scaling is 4"), (dict(scaling=-1), "scaling is -1"), (dict(base=1.0), "base is 1"),
    (dict(base=NAN), "base is nan"), (dict(base=math.inf), "base is inf"), (dict(attention=-1.0), "attention is -1"),
    (dict(attention=NAN), "attention is nan"), (dict(scaling=tgo_amd.ROPE_LINEAR, factor=0.5), "factor is 0.5"),
    (dict(YARN, factor=NAN), "factor is nan"), (dict(YARN, original=0.0), "original is 0"),
    (dict(BANDS, slow=0.0), "slow 0"), (dict(BANDS, fast=1.0), "fast is 1 and slow 1"),
    (dict(YARN, fast=math.inf), "fast is inf"), (dict(BANDS, slow=NAN), "slow nan"),
])
def test_rope_refusals(change, word):
    args = dict(dict(head_dim=128, base=1e6), **change)
    with pytest.raises(TgoError, match=word):
        tgo_amd.rope_freqs(**args)
    c, h = tgo_amd.rope_cfg(**args), ctypes.c_int(0)
    assert tgo_amd.lib().tgohip_rope_new(None, ctypes.byref(c), ctypes.byref(h)) == tgo_amd.EINVAL
    assert word in tgo_amd.last_error() and h.value == 0


def plan(nq, nk, H=8, Hkv=2, d=128, q=tgo_amd.F32, B=None):
    a, b, h = tgo_amd.i32(nq), tgo_amd.i32(nk), ctypes.c_int(0)
    rc = tgo_amd.lib().tgohip_packed_plan(None, len(nq) if B is None else B, tgo_amd.ptr(a) if len(nq) else None,
                                          tgo_amd.ptr(b) if len(nk) else None, H, Hkv, d, 1, q, ctypes.byref(h))
    assert h.value == 0
    return rc, tgo_amd.last_error()


@pytest.mark.parametrize("kw,word", [
    (dict(nq=[1], nk=[1], B=-1), "-1 sequences"), (dict(nq=[], nk=[], B=2), "q_lengths and kv_lengths"),
    (dict(nq=[1], nk=[1], d=96), "head_dim is 96"), (dict(nq=[1], nk=[1], H=6, Hkv=4), "6 query heads over 4"),
    (dict(nq=[1], nk=[1], H=0), "0 query heads"), (dict(nq=[1], nk=[1], Hkv=0), "over 0 kv heads"),
    (dict(nq=[1], nk=[1], q=tgo_amd.F16X2), "q_dtype is 2"), (dict(nq=[4, -1], nk=[4, 4]), "sequence 1 has -1 queries"),
    (dict(nq=[4, 1], nk=[-7, 4]), "and -7 keys"), (dict(nq=[1 << 28], nk=[4]), "below 2\\^30"),
    (dict(nq=[1] * 4, nk=[1 << 29] * 4), "below 2\\^30"), (dict(nq=[3], nk=[5]), "context is missing"),
    (dict(nq=[], nk=[]), "context is missing"), (dict(nq=[1], nk=[1], H=65538, Hkv=2), "65538 query heads; at most 65536"),
])
def test_packed_plan_refusals(kw, word):
    import re
    rc, msg = plan(**kw)
    assert rc == tgo_amd.EINVAL and re.search(word, msg), msg


@pytest.mark.parametrize("K,N,cap,word", [
    (0, 64, 1, "projection is"), (96, 64, 1, "K a multiple of 64"), (64, 48, 1, "N of 32|N a multiple of 32"),
    (-64, 64, 1, "projection is"), ((1 << 22) + 64, 64, 1, "up to 2\\^22"), (64, 1 << 23, 1, "up to 2\\^22"), (64, 64, 0, "capacity is 0"), (64, 64, 65537, "capacity is 65537"),
    (64, 64, 4, "context is missing"),
])
def test_adapter_set_refusals(K, N, cap, word):
    import re
    h = ctypes.c_int(0)
    assert tgo_amd.lib().tgohip_adapters_new(None, K, N, cap, ctypes.byref(h)) == tgo_amd.EINVAL
    assert re.search(word, tgo_amd.last_error())


@pytest.mark.parametrize("change,word", [
    (dict(rank=0), "rank is 0"), (dict(rank=129), "rank is 129"), (dict(dtype=2), "dtype is 2"),
    (dict(down=None), "host planes"), (dict(up=None), "host planes"), (dict(scale=math.inf), "scale is inf"),
    (dict(scale=NAN), "scale is nan"), (dict(), "context is missing"),
])
def test_adapter_put_refusals(change, word):
    plane = np.zeros(64 * 128, np.float32)
    a = dict(dict(rank=4, dtype=tgo_amd.F32, down=plane, up=plane, scale=1.0), **change)
    assert tgo_amd.lib().tgohip_adapters_put(None, 1, 0, a["rank"], a["dtype"], tgo_amd.ptr(a["down"]),
                                             tgo_amd.ptr(a["up"]), a["scale"]) == tgo_amd.EINVAL
    assert word in tgo_amd.last_error()


@pytest.mark.parametrize("extents,who,B,word", [
    ([1], [0], -1, "-1 requests"), ([], [], 1, "host arrays"), ([1, -2], [0, 0], 2, "request 1 has -2 rows"),
    ([1, 1], [0, -2], 2, "names adapter -2"), ([1], [65536], 1, "names adapter 65536"),
    ([1 << 19, 1 << 19], [0, 0], 2, "below 2\\^20"), ([3, 0], [0, -1], 2, "context is missing"),
])
def test_adapter_rows_refusals(extents, who, B, word):
    import re
    e, w, h = tgo_amd.i32(extents), tgo_amd.i32(who), ctypes.c_int(0)
    assert tgo_amd.lib().tgohip_adapter_rows(None, B, tgo_amd.ptr(e) if extents else None,
                                             tgo_amd.ptr(w) if who else None, ctypes.byref(h)) == tgo_amd.EINVAL
    assert re.search(word, tgo_amd.last_error())


def test_calls_without_a_context_are_refused():
    L, g = tgo_amd.lib(), (tgo_amd.RopeHeads * 1)()
    for rc in (L.tgohip_rope(None, 1, None, 1, g, 1), L.tgohip_rope_free(None, 1), L.tgohip_packed_free(None, 1),
               L.tgohip_packed_attention(None, 1, None, 0, None, 0, None, 0, 1.0, None, 0, 0),
               L.tgohip_adapters(None, 1, 1, None, 0, None, None, 0), L.tgohip_adapters_drop(None, 1, 0),
               L.tgohip_adapters_free(None, 1), L.tgohip_adapter_rows_free(None, 1)):
        assert rc == tgo_amd.EINVAL and "context is missing" in tgo_amd.last_error()


def describe(nq, nk, **kw):
    p = tgo_amd.packed_describe(nq, nk, kw.pop("H", 32), kw.pop("Hkv", 8), **kw)
    return p.tiles, p.few, p.longest_tile, p.longest_few, p.part_rows, p.merged_rows


def test_packed_batches_are_decomposed_by_their_sizes():
    # one short prompt: 40 tokens x 4 heads are two tiles of 128 rows for each of 8 kv heads
    assert describe([40], [40]) == (16, 0, 40, 0, 0, 0)
    # single tokens go to the few-row kernel, whole where they fill the chip evenly ...
    assert describe([1] * 64, [4096] * 64) == (0, 512, 0, 4096, 0, 0)
    # ... and cut where few of them would leave it idle: 8 items on 512 slots
    tiles, few, _, longest, parts, merged = describe([1], [32768])
    assert tiles == 0 and few > 400 and longest <= 640 and parts == 4 * few and merged == 32
    # beside prompts that hold most of the keys they take a tile each
    assert describe([1, 2000], [50, 2000])[1] == 0
    assert describe([1, 20], [5000, 20])[1] > 0
    # a long prompt's tiles are many and of every length: none is cut
    assert describe([16384], [16384], q_dtype=tgo_amd.F16) == (4096, 0, 16384, 0, 0, 0)
    # a chunk far behind its keys is cut: its partial rows hold every row at least twice
    tiles, _, longest, _, parts, merged = describe([128], [32768])
    assert tiles > 32 and longest < 32768 and merged == 128 * 32 and parts >= 2 * merged
    # queries that see no key still have an item, which writes zeros
    assert describe([7], [0]) == (8, 0, 0, 0, 0, 0)
    assert describe([0, 0], [3, 0]) == (0, 0, 0, 0, 0, 0)
    assert describe([], []) == (0, 0, 0, 0, 0, 0)


@pytest.mark.parametrize("seed", range(20))
def test_packed_parts_cover_every_key_once(seed):
    """Rows merged are whole items', and the keys of the parts of any batch are those of its items."""
    r = np.random.default_rng(seed)
    n = int(r.integers(1, 40))
    nk = r.integers(0, 6000, n)
    nq = np.where(r.random(n) < 0.5, r.integers(0, 5, n), r.integers(0, 900, n))
    H, Hkv = [(32, 8), (7, 1), (16, 16), (64, 4)][seed % 4]
    for causal in (True, False):
        p = tgo_amd.packed_describe(nq, nk, H, Hkv, causal=causal)
        assert p.part_rows >= 2 * p.merged_rows and (p.part_rows > 0) == (p.merged_rows > 0)
        assert p.merged_rows <= int(nq.sum()) * H
        assert max(p.longest_tile, p.longest_few) <= nk.max()
        # as on one compute unit, where nothing is cut
        one = tgo_amd.packed_describe(nq, nk, H, Hkv, causal=causal, ncu=1)
        assert one.tiles + one.few <= p.tiles + p.few


def test_a_batch_is_cut_where_that_ends_sooner():
    """On 256 compute units of two workgroups: a batch that fills them evenly stays whole, one that a few
    workgroups outlast is cut, and a short batch of long contexts goes over the whole chip."""
    def plan(nq, nk, **kw):
        return tgo_amd.packed_describe(nq, nk, 32, 8, **kw)
    p = plan([1] * 64, [4096] * 64)  # 512 workgroups of one length
    assert (p.few, p.longest_few, p.part_rows) == (512, 4096, 0)
    p = plan([1] * 66, [4096] * 66)  # 16 more than run at a time
    assert p.few > 528 and p.longest_few == 4096 and 0 < p.merged_rows < 66 * 32
    p = plan([1], [32768])  # 8 kv heads over every compute unit, in pieces of one size
    assert (p.few, p.longest_few, p.part_rows, p.merged_rows) == (512, 512, 2048, 32)
    p = plan([100, 20], [2300, 2700])
    assert p.tiles == 256 and p.longest_tile < 2300 / 4 and p.merged_rows == 120 * 32
    p = plan([2048], [2048], q_dtype=tgo_amd.F16)  # the long rows beside the short ones
    assert (p.tiles, p.part_rows) == (512, 0)


def test_packed_describe_refusals():
    for kw in (dict(head_dim=80), dict(ncu=0), dict(q_dtype=2)):
        with pytest.raises(TgoError):
            tgo_amd.packed_describe([1], [1], 8, 2, **kw)


def check_pieces(nq, nk, H, Hkv, causal, **kw):
    """Every row of every kv head is in one block of rows; a block's pieces hold its keys, each once; cut blocks
    have partial rows of their own and merges that join each row once."""
    pieces, merges = tgo_amd.packed_pieces(nq, nk, H, Hkv, causal=causal, **kw)
    p = tgo_amd.packed_describe(nq, nk, H, Hkv, causal=causal, **kw)
    assert len(pieces) == p.tiles + p.few
    G, q0, k0 = H // Hkv, np.concatenate([[0], np.cumsum(nq)]), np.concatenate([[0], np.cumsum(nk)])
    by = {}
    for i, t in enumerate(pieces):
        by.setdefault((int(t["q0"]), int(t["kv_head"]), int(t["row"]), int(t["rows"])), []).append((t, i >= p.tiles))
    blocks = {}
    for (at, head, row, rows) in by:
        blocks.setdefault((at, head), []).append((row, rows))
    used, joined = np.zeros(p.part_rows, np.int32), {}
    for m in merges:
        for i in range(m["rows"]):
            key = (int(m["q0"]), int(m["kv_head"]), int(m["row"]) + i)
            assert key not in joined
            joined[key] = (int(m["part"]) + i, int(m["parts"]), int(m["step"]))
        assert 1 <= m["rows"] <= 8
    for s, (n, k) in enumerate(zip(nq, nk)):
        for head in range(Hkv if n else 0):
            end = 0
            for row, rows in sorted(blocks.pop((int(q0[s]), head))):
                assert row == end and 1 <= rows <= 128
                end = row + rows
                cut = sorted(by[int(q0[s]), head, row, rows], key=lambda c: c[0]["kv_lo"])
                last = (end - 1) // G  # the block's last query, which sees the most
                hi = max(0, min(k, last + k - n + 1)) if causal else k
                at = 0
                for t, few in cut:
                    assert t["k0"] == k0[s] and t["kv_lo"] == at and (t["kv_hi"] > at or hi == 0)
                    assert t["kv_lo"] % 64 == 0 and (not few or n * G <= 32)
                    # queries see up to their own position, or everything
                    assert all(min(i + int(t["shift"]), k - 1) == (min(i + k - n, k - 1) if causal else k - 1)
                               for i in (row // G, last))
                    at = t["kv_hi"]
                assert at == hi and len({few for _, few in cut}) == 1
                if len(cut) == 1:
                    assert cut[0][0]["part"] == -1 and (int(q0[s]), head, row) not in joined
                    continue
                base = min(int(t["part"]) for t, _ in cut)
                for j, (t, _) in enumerate(cut):  # the merge adds them in the keys' order
                    assert t["part"] == base + j * rows
                    used[t["part"]:t["part"] + rows] += 1
                for i in range(rows):
                    assert joined.pop((int(q0[s]), head, row + i)) == (base + i, len(cut), rows)
            assert end == n * G
    assert not blocks and not joined and (used == 1).all()


@pytest.mark.parametrize("seed", range(40))
def test_packed_pieces_hold_every_row_and_key_once(seed):
    r = np.random.default_rng(1000 + seed)
    n = int(r.integers(1, 24))
    top = int(np.exp(r.uniform(0, math.log(40000))))
    nk = np.exp(r.uniform(0, math.log(top + 1), n)).astype(int) - (r.random(n) < 0.1)
    kind = r.integers(0, 4)
    nq = [np.ones(n, int), r.integers(0, 9, n), r.integers(0, 500, n), np.minimum(nk, 3000)][kind]
    H, Hkv = [(32, 8), (7, 1), (4, 4), (64, 4), (160, 1)][seed % 5]
    for causal in (True, False):
        for ncu in (256, 1, 40, 2048):
            check_pieces(nq.tolist(), nk.tolist(), H, Hkv, causal, ncu=ncu, head_dim=[64, 128][seed % 2],
                         q_dtype=[tgo_amd.F32, tgo_amd.F16][seed // 2 % 2])


def test_packed_pieces_of_batches_that_are_cut():
    for nq, nk in (([1], [32768]), ([1] * 66, [4096] * 66), ([100, 20], [2300, 2700]), ([128], [32768]), ([7], [0]),
                   ([0, 0], [3, 0]), ([], []), ([1, 20], [5000, 20]), ([1] * 300, list(range(1, 30001, 100)))):
        check_pieces(nq, nk, 32, 8, True)
        check_pieces(nq, nk, 32, 8, False)


def test_packed_pieces_refusals():
    with pytest.raises(TgoError, match="head_dim is 80"):
        tgo_amd.packed_pieces([1], [1], 8, 2, head_dim=80)
    with pytest.raises(TgoError, match="ncu"):
        tgo_amd.packed_pieces([1], [1], 8, 2, ncu=0)
    a, n, m = tgo_amd.i32([5]), ctypes.c_int(1), ctypes.c_int(0)
    one = np.zeros(1, tgo_amd.PIECE)
    assert tgo_amd.lib().tgohip_packed_pieces(1, tgo_amd.ptr(a), tgo_amd.ptr(a), 8, 2, 128, 1, 0, 256, tgo_amd.ptr(one),
                                              ctypes.byref(n), None, ctypes.byref(m)) == tgo_amd.EINVAL
    assert "hold 1 pieces" in tgo_amd.last_error() and (n.value, m.value) == (2, 0)


def test_batches_of_more_workgroups_than_a_launch_takes_are_refused():
    """Before anything is decomposed: these have 8.5 and 65 million blocks of rows, the last would fill the
    host's memory."""
    for B in (130, 1000, 16000):
        for call in (tgo_amd.packed_describe, tgo_amd.packed_pieces):
            with pytest.raises(TgoError, match="workgroups, more than one launch takes"):
                call([1] * B, [1] * B, 65536, 65536)
        rc, msg = plan([1] * B, [1] * B, H=65536, Hkv=65536)
        assert rc == tgo_amd.EINVAL and "more than one launch takes" in msg
    p = tgo_amd.packed_describe([1] * 100, [1] * 100, 65536, 8192, head_dim=64)
    assert p.tiles + p.few == 100 * 8192
    for ncu in (0, -1, 65537, 2 ** 31 - 1):
        for call in (tgo_amd.packed_describe, tgo_amd.packed_pieces):
            with pytest.raises(TgoError, match="ncu"):
                call([1], [9000], 8, 2, ncu=ncu)


@pytest.mark.parametrize("attention", [1e39, 3.5e38, 1e300])
def test_rope_factors_past_f32_are_refused(attention):
    """cos and sin are multiplied in f32: a factor past its range would make every output infinite or NaN."""
    with pytest.raises(TgoError, match="attention is"):
        tgo_amd.rope_freqs(128, 1e6, attention=attention)
    assert tgo_amd.rope_freqs(128, 1e6, attention=3.4e38)[1] == 3.4e38
