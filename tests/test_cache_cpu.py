"""What the 8-bit cache's entry points refuse before they touch a context: every argument is checked first, so
these calls need no GPU."""
import ctypes
import re

import numpy as np
import pytest

import tgo_amd

NAN = float("nan")
BASE = 1 << 40  # addresses that nothing reads


def cache(**kw):
    """A cache of 2 layers, 8 pages of 16 positions, 4 heads of 64: 32768 bytes of codes a layer, 2048 of scales."""
    a = dict(k=BASE, v=BASE + (1 << 20), k_scale=BASE + (2 << 20), v_scale=BASE + (3 << 20), form=tgo_amd.CACHE_I8, layers=2,
             pages=8, kv_heads=4, block=16, head_dim=64)
    a.update(kw)
    return tgo_amd.CacheC(*(a[n] for n, _ in tgo_amd.CacheC._fields_))


GEOMETRY = [
    (dict(form=2), "form is 2"), (dict(head_dim=96), "head_dim is 96"), (dict(head_dim=0), "head_dim is 0"),
    (dict(block=0), "block is 0"), (dict(block=24), "block is 24; a power of two"), (dict(block=2048), "block is 2048"),
    (dict(kv_heads=0), "0 kv heads"), (dict(kv_heads=4097), "4097 kv heads"), (dict(layers=0), "0 layers"),
    (dict(layers=1 << 14), "16384 layers of 4 kv heads"), (dict(pages=0), "0 pages"), (dict(pages=-1), "-1 pages"),
    (dict(pages=1 << 25), "below 2\\^31"),
]
BUFFERS = [
    (dict(k=None), "device buffers"), (dict(v_scale=None), "device buffers"), (dict(k=BASE + 8), "16-byte boundaries"),
    (dict(v=BASE + (1 << 20) + 4), "16-byte boundaries"), (dict(k_scale=BASE + (2 << 20) + 2), "4-byte ones"),
    (dict(v=BASE + 65520), "k and v meet"), (dict(v_scale=BASE + (2 << 20) + 4092), "k_scale and v_scale meet"),
    (dict(k_scale=BASE + 65532), "k and k_scale meet"),
]


def calls(c):
    """Every entry point over a cache, on arguments that it would take."""
    L, at, h = tgo_amd.lib(), ctypes.byref(c), ctypes.c_int(0)
    one, page = tgo_amd.i32([1]), tgo_amd.u32([0])
    return [lambda: L.tgohip_cache_store(None, at, 0, 0, None, BASE + (9 << 20), 1, rows()),
            lambda: L.tgohip_cache_read(None, at, 0, BASE + (9 << 20), 1, BASE + (10 << 20), 256, 64, None, 0, 0, 0),
            lambda: L.tgohip_cache_move(None, at, tgo_amd.ptr(one), tgo_amd.ptr(one), 1),
            lambda: L.tgohip_cache_attention(None, 1, at, 0, BASE + (9 << 20), 256, 1.0, BASE + (10 << 20), 256, 0),
            lambda: L.tgohip_cache_plan(None, at, 1, tgo_amd.ptr(one), tgo_amd.ptr(one), tgo_amd.ptr(page), 1, None, 4, 0,
                                        ctypes.byref(h))]


def rows(**kw):
    a = dict(q=BASE + (10 << 20), k=BASE + (11 << 20), v=BASE + (12 << 20), q_out=BASE + (13 << 20), q_row=512, q_head=64,
             k_row=256, k_head=64, v_row=256, v_head=64, out_row=512, out_head=64, q_gain=None, k_gain=None, eps=1e-6, heads=8,
             x_dtype=tgo_amd.F32, out_dtype=tgo_amd.F32)
    a.update(kw)
    return ctypes.byref(tgo_amd.CacheRows(*(a[n] for n, _ in tgo_amd.CacheRows._fields_)))


@pytest.mark.parametrize("change,word", GEOMETRY + BUFFERS)
def test_caches_that_are_refused(change, word):
    for i, call in enumerate(calls(cache(**change))):
        if i == 4 and (change, word) in BUFFERS:
            continue  # a plan needs the geometry alone
        assert call() == tgo_amd.EINVAL
        assert re.search(word, tgo_amd.last_error()), (i, tgo_amd.last_error())


def test_calls_without_a_context_are_refused():
    L = tgo_amd.lib()
    for call in calls(cache()) + [lambda: L.tgohip_cache_plan_free(None, 1)]:
        assert call() == tgo_amd.EINVAL and "context is missing" in tgo_amd.last_error()
    L.tgohip_cache_store(None, None, 0, 0, None, None, 0, None)
    assert "the cache is missing" in tgo_amd.last_error()


SLOTS = BASE + (9 << 20)


@pytest.mark.parametrize("call,row,word", [
    (dict(layer=2), {}, "layer 2 of 2"), (dict(layer=-1), {}, "layer -1 of 2"), (dict(T=-1), {}, "-1 rows"),
    (dict(T=1 << 24), {}, "0 to 2\\^24 - 1"), (dict(rows=None), {}, "rows are missing"), (dict(slots=None), {}, "device buffers"),
    (dict(slots=SLOTS + 2), {}, "not aligned"), (dict(rope=1), {}, "positions is a device buffer"), ({}, dict(heads=-1), "-1 query heads"),
    ({}, dict(heads=4097), "4097 query heads"), ({}, dict(x_dtype=2), "f32 or f16"), ({}, dict(out_dtype=2), "f32 or f16"),
    ({}, dict(k=None), "device buffers"), ({}, dict(q=None), "device buffers"), ({}, dict(q_out=None), "device buffers"),
    ({}, dict(q_gain=BASE + (14 << 20), eps=-1.0), "eps is -1"), ({}, dict(k_gain=BASE + (14 << 20), eps=NAN), "eps is nan"),
    ({}, dict(k_gain=BASE + (14 << 20) + 2), "not aligned"), ({}, dict(v=BASE + 2), "not aligned"),
    ({}, dict(k_row=-1), "strides are not negative"), ({}, dict(v_head=1 << 37), "strides are not negative"),
    ({}, dict(out_head=63), "heads of q_out overlap"), ({}, dict(out_row=511), "heads of q_out overlap"),
    ({}, dict(out_row=0), "heads of q_out overlap"),
])
def test_store_refusals(call, row, word):
    a = dict(layer=0, rope=0, positions=None, slots=SLOTS, T=3, rows=rows(**row))
    a.update(call)
    c = cache()
    assert tgo_amd.lib().tgohip_cache_store(None, ctypes.byref(c), a["layer"], a["rope"], a["positions"], a["slots"], a["T"],
                                            a["rows"]) == tgo_amd.EINVAL
    assert re.search(word, tgo_amd.last_error()), tgo_amd.last_error()


@pytest.mark.parametrize("change,word", [
    (dict(layer=3), "layer 3 of 2"), (dict(T=-1), "-1 rows"), (dict(T=1 << 29), "below 2\\^29"), (dict(dtype=2), "out_dtype is 2"),
    (dict(slots=None), "slots is a device buffer"), (dict(k=BASE + (10 << 20) + 2), "k_out is not aligned"),
    (dict(k_row=-4), "strides are not negative"), (dict(k_head=32), "heads of k_out overlap"), (dict(k=BASE + 64), "k_out meets the cache's k "),
    (dict(k=BASE + (3 << 20)), "k_out meets the cache's v_scale"), (dict(k=SLOTS), "k_out meets slots"),
    (dict(v=BASE + (10 << 20) + 64), "k_out and v_out meet"), (dict(v_row=0), "heads of v_out overlap"),
])
def test_read_refusals(change, word):
    a = dict(layer=0, slots=SLOTS, T=3, k=BASE + (10 << 20), k_row=256, k_head=64, v=BASE + (11 << 20), v_row=256, v_head=64, dtype=0)
    a.update(change)
    c = cache()
    assert tgo_amd.lib().tgohip_cache_read(None, ctypes.byref(c), a["layer"], a["slots"], a["T"], a["k"], a["k_row"], a["k_head"],
                                           a["v"], a["v_row"], a["v_head"], a["dtype"]) == tgo_amd.EINVAL
    assert re.search(word, tgo_amd.last_error()), tgo_amd.last_error()


RING = list(range(65))


@pytest.mark.parametrize("src,dst,word", [
    ([0], [128], "from slot 0 to slot 128 of a pool of 128"), ([-1], [0], "slot -1"), ([128], [0], "slot 128"),
    ([0, 1], [5, 5], "two rows go to slot 5"), ([3, 1], [3, 3], "two rows go to slot 3"),
    (RING, RING[1:] + RING[:1], "a cycle of 65 slots; up to 64"), (RING[:64], RING[1:64] + RING[:1], "context is missing"),
    (list(range(127)), list(range(1, 128)), "context is missing"), ([], [], "context is missing"),
])
def test_move_refusals(src, dst, word):
    a, b, c = tgo_amd.i32(src + [0]), tgo_amd.i32(dst + [0]), cache()
    assert tgo_amd.lib().tgohip_cache_move(None, ctypes.byref(c), tgo_amd.ptr(a), tgo_amd.ptr(b), len(src)) == tgo_amd.EINVAL
    assert re.search(word, tgo_amd.last_error()), tgo_amd.last_error()


@pytest.mark.parametrize("change,word", [
    (dict(B=-1), "-1 sequences"), (dict(extents=None), "host arrays"), (dict(max_pages=-1), "-1 pages a sequence"),
    (dict(H=6), "6 query heads over 4"), (dict(H=0), "0 query heads"), (dict(H=65540), "H at most 65536"), (dict(q=2), "q_dtype is 2"),
    (dict(extents=[1, -1]), "sequence 1 has -1 new tokens"), (dict(extents=[1, 21]), "sequence 1 has 21 new tokens of 20"),
    (dict(lengths=[33, 20]), "sequence 0 has 33 positions and 2 pages of 16"), (dict(pages=[0, 1, 8, 0]), "sequence 1: page 0 is 8 of a pool of 8"),
    (dict(pages=[0, 1, 0, 1 << 31]), "sequence 1: page 1 is"), (dict(extents=[0, 0], pages=[9, 9, 9, 9]), "context is missing"),
    (dict(parents=[-2, -1, 0]), "token 0 has parent -2"), (dict(parents=[0, -1, 0]), "token 0 has parent 0"),
    (dict(parents=[-1, -1, 1]), "sequence 1: token 1 has parent 1"), (dict(parents=[-1, -1, -1]), "context is missing"),
    (dict(), "context is missing"),
])
def test_plan_refusals(change, word):
    a = dict(B=2, extents=[1, 2], lengths=[5, 20], pages=[3, 0, 7, 2], max_pages=2, parents=None, H=8, q=0)
    a.update(change)
    arrays = [None if a[n] is None else f(a[n]) for n, f in (("extents", tgo_amd.i32), ("lengths", tgo_amd.i32),
                                                             ("pages", tgo_amd.u32), ("parents", tgo_amd.i32))]
    e, l, p, up = (tgo_amd.ptr(x) for x in arrays)
    c, h = cache(), ctypes.c_int(0)
    assert tgo_amd.lib().tgohip_cache_plan(None, ctypes.byref(c), a["B"], e, l, p, a["max_pages"], up, a["H"], a["q"],
                                           ctypes.byref(h)) == tgo_amd.EINVAL and h.value == 0
    assert re.search(word, tgo_amd.last_error()), tgo_amd.last_error()


def test_trees_have_as_many_tokens_as_a_mask_has_bits():
    c, h = cache(pages=8, block=64), ctypes.c_int(0)
    for n, chain, word in ((65, False, "a tree of 65 tokens; up to 64"), (64, False, "context is missing"), (65, True, "context is missing")):
        up = tgo_amd.i32(list(range(-1, n - 1)) if chain else [-1] * n)
        e, t = tgo_amd.i32([n]), tgo_amd.u32([0, 1])
        assert tgo_amd.lib().tgohip_cache_plan(None, ctypes.byref(c), 1, tgo_amd.ptr(e), tgo_amd.ptr(e), tgo_amd.ptr(t), 2,
                                               tgo_amd.ptr(up), 4, 0, ctypes.byref(h)) == tgo_amd.EINVAL
        assert word in tgo_amd.last_error()


@pytest.mark.parametrize("change,word", [
    (dict(layer=2), "layer 2 of 2"), (dict(scale=0.0), "scale is 0"), (dict(scale=-1.0), "scale is -1"), (dict(scale=NAN), "scale is nan"),
    (dict(scale=2.0 ** 33), "at most 2\\^32"), (dict(scale=2.0 ** -65), "at least 2\\^-64"), (dict(dtype=3), "out_dtype is 3"), ({}, "context is missing"),
])
def test_attention_refusals(change, word):
    a = dict(layer=0, scale=1.0, dtype=0)
    a.update(change)
    c = cache()
    assert tgo_amd.lib().tgohip_cache_attention(None, 1, ctypes.byref(c), a["layer"], SLOTS, 512, a["scale"], BASE + (10 << 20), 512,
                                                a["dtype"]) == tgo_amd.EINVAL
    assert re.search(word, tgo_amd.last_error()), tgo_amd.last_error()


def host_context():
    """A context that never was, and a cache of tensors of the host: its calls end where the library asks for it."""
    import torch
    tgo_amd.lib()
    c = object.__new__(tgo_amd.Context)
    c.h, c.device, c._plans = None, -1, {}
    codes = [torch.zeros(1, 8, 2, 16, 64, dtype=torch.int8) for _ in "kv"]
    return c, tgo_amd.Cache(*codes, *(torch.zeros(1, 8, 2, 16) for _ in "kv"))


@pytest.mark.parametrize("good", [[5], (5,), np.array([5]), np.array([5], np.int32), np.array([5], np.uint8), [np.int64(5)]])
@pytest.mark.parametrize("bad", [np.array([2 ** 32 + 5]), [2 ** 32 + 5], [-2 ** 31 - 1], [2 ** 70], [1.7], np.array([5.0]), ["5"],
                                 np.array([2 ** 31], np.uint32), (2 ** 40,)])
def test_host_arrays_of_other_numbers_are_refused(good, bad):
    """Slots, extents, lengths, pages and parents that are no whole numbers of 32 bits are not made into some."""
    ctx, c = host_context()
    table = [[0, 1, 2, 3]]
    for src, dst in ((good, bad), (bad, good)):
        with pytest.raises(tgo_amd.TgoError, match="slots are whole numbers of 32 bits"):
            ctx.cache_move(c, src, dst)
    with pytest.raises(tgo_amd.TgoError, match="context is missing"):
        ctx.cache_move(c, good, [7])
    with pytest.raises(tgo_amd.TgoError, match="extents are whole numbers"):
        ctx.cache_plan(c, bad, good, table, 4)
    with pytest.raises(tgo_amd.TgoError, match="lengths are whole numbers"):
        ctx.cache_plan(c, good, bad, table, 4)
    with pytest.raises(tgo_amd.TgoError, match="parents are whole numbers"):
        ctx.cache_plan(c, [1], good, table, 4, parents=bad)
    with pytest.raises(tgo_amd.TgoError, match="context is missing"):
        ctx.cache_plan(c, good, [60], table, 4, parents=list(range(-1, 4)))


@pytest.mark.parametrize("pages,word", [
    ([[2 ** 32 + 1]], "pages are whole numbers"), (np.array([[2 ** 32 + 1]]), "pages are whole numbers"), ([[1.5]], "pages are whole numbers"),
    ([[-1]], "page 0 is 4294967295 of a pool of 8"), (np.array([[-1]], np.int32), "page 0 is 4294967295 of a pool of 8"),
    ([[3, -1]], "context is missing"), (np.array([[3, -1]]), "context is missing"), (np.array([[3]], np.uint32), "context is missing"),
    ([3], "a page table of \\(1,\\)"),
])
def test_page_tables(pages, word):
    ctx, c = host_context()
    with pytest.raises(tgo_amd.TgoError, match=word):
        ctx.cache_plan(c, [1], [9], pages, 4)


def test_lists_of_other_shapes_are_refused():
    ctx, c = host_context()
    for extents, lengths in (([[1, 1]], [9]), ([1], [[9]]), ([1, 1], [9])):
        with pytest.raises(tgo_amd.TgoError, match="cache_plan: extents of"):
            ctx.cache_plan(c, extents, lengths, [[0]], 4)
    with pytest.raises(tgo_amd.TgoError, match="slots are a list"):
        ctx.cache_move(c, np.array([[1]]), [1])


@pytest.mark.parametrize("T,row,word", [
    (1 << 28, 1 << 36, "k_out's 268435456 rows are 68719476736 elements apart"), (1 << 28, (1 << 32) + 1, "at most 2\\^60"),
    (1 << 28, 1 << 32, "context is missing"), ((1 << 29) - 1, 1 << 31, "context is missing"),
    ((1 << 29) - 1, 1 << 34, "v_out's 536870911 rows"), (3, 1 << 36, "context is missing"),
])
def test_reads_of_rows_far_apart(T, row, word):
    """What is computed of operands' places stays in 64 bits, whatever rows and strides are asked for."""
    c = cache(kv_heads=1)
    out = [BASE + (1 << 40), None]
    if "v_out" in word:
        out.reverse()
    assert tgo_amd.lib().tgohip_cache_read(None, ctypes.byref(c), 0, SLOTS, T, out[0], row, 64, out[1], row, 64,
                                           0) == tgo_amd.EINVAL
    assert re.search(word, tgo_amd.last_error()), tgo_amd.last_error()
