"""A cache in pages, on the GPU: appended rows against the single calls bit for bit (and, behind norms, against float64),
attention against its plain float64 form (tests/paged_util.py, the bounds derived there), index checks, host buffers, captured
calls, and the two operators together as a server uses them."""
import os
import subprocess
import sys
import threading

import numpy as np
import pytest

import llama_hip as lh
from tests import hip_util as hu
from tests import paged_util as pu
from tests import requests_util as ru

pytestmark = pytest.mark.gpu
F = np.float32


@pytest.fixture
def L():
    lib = lh.load()
    assert lib.llhip_init() == 0, lh.last_error()
    lh.record_failures()
    layout = lib.kernels_kv_layout_name().decode()
    yield lib
    lib.kernels_kv_layout_select(layout.encode())
    lib.llhip_synchronize()
    lib.llhip_clear_error()
    lib.llhip_set_fail_mode(lh.LLHIP_FAIL_EXIT)


def quiet(L):
    L.llhip_synchronize()
    assert not lh.last_error(), lh.last_error()


def fails(L, words):
    L.llhip_synchronize()
    message = lh.last_error()
    L.llhip_clear_error()
    assert words in message, message


def within(got, want, bound, what=""):
    off = np.abs(got.astype(np.float64) - want)
    assert np.isfinite(got).all(), what
    worst = np.unravel_index(np.argmax(off - bound), off.shape)
    assert (off <= bound).all(), (what, worst, got[worst], want[worst], off[worst], bound[worst])


def cache_dev(a):
    """A device copy of a cache; BF16 bits as int16, which torch copies."""
    return hu.dev(a.view(np.int16) if a.dtype == np.uint16 else a)


def cache_host(x):
    a = hu.host(x)
    return a.view(np.uint16) if a.dtype == np.int16 else a


def shifted(a, floats=1):
    """A device copy of `a` whose address is 4 * floats bytes off the allocation's 16-byte alignment."""
    t = hu.torch()
    flat = hu.empty(a.size + floats, t.float32)
    view = flat[floats:].reshape(a.shape)
    view.copy_(t.from_numpy(a))
    t.cuda.synchronize()
    return view


def rope_table(L, rows, hd):
    cfg = lh.Config(head_dim=hd, rope_theta=500000.0)
    table = np.zeros((rows, 2 * hd), F)
    for p in range(rows):
        L.k_rope_table(ru.byref(cfg), p, lh.ptr(table[p]))
    return table


# ---- appended rows ------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("layout", ["head", "rows"])
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("heads,kv,hd", [(4, 2, 64), (3, 1, 128), (5, 5, 6), (8, 2, 80), (2, 1, 256), (2, 2, 2), (3, 1, 130)])
@pytest.mark.parametrize("form", ["apart", "packed", "shifted"])
def test_appended_rows_equal_the_single_calls_bit_for_bit(L, layout, bf16, heads, kv, hd, form):
    """Against k_rope_apply of each row alone: ragged requests (none, one and many rows, over a page's end), rows before the
    first and behind the last request, in place on packed QKV rows, into a buffer of another stride, off 16-byte alignment."""
    L.kernels_kv_layout_select(layout.encode())
    rng = np.random.default_rng(hd + heads)
    b = pu.Pages(hu.dev, [3, 0, 1, 40, 2], [0, 99, 7, 11, 30], page=9 if heads == 3 else 16, bf16=bf16, first=2, spare=3)
    dq, dkv = heads * hd, kv * hd
    table = rope_table(L, b.seq_len, hd)
    caches = [b.cache(rng, layout, kv, hd) for _ in range(2)]
    wide = rng.standard_normal((b.rows, dq + 2 * dkv + 4), dtype=F)
    q, k, v = wide[:, :dq], wide[:, dq:dq + dkv], wide[:, dq + dkv:dq + 2 * dkv]
    kd, vd, td = cache_dev(caches[0]), cache_dev(caches[1]), hu.dev(table)
    put = shifted if form == "shifted" else hu.dev
    if form == "packed":
        rows = hu.dev(wide)
        qd, kr, vr = rows, rows[:, dq:], rows[:, dq + dkv:]
        out, o_stride, stride, kv_stride = rows, wide.shape[1], wide.shape[1], wide.shape[1]
    else:
        qd, kr, vr = (put(np.ascontiguousarray(x)) for x in (q, k, v))
        out, o_stride, stride, kv_stride = put(np.full((b.rows, dq + 8), 7.0, F)), dq + 8, dq, dkv
    L.llhip_rope_kv_append_paged(lh.ptr(out), o_stride, lh.ptr(qd), stride, lh.ptr(kr), lh.ptr(vr), kv_stride, lh.ptr(td),
                                 None, None, 0.0, b.struct, heads, kv, hd, lh.ptr(kd), lh.ptr(vd))
    quiet(L)
    got = hu.host(out)
    want = wide.copy() if form == "packed" else np.full((b.rows, dq + 8), 7.0, F)
    for r, rows_, length in b.requests():
        for j, i in enumerate(range(rows_.start, rows_.stop)):
            qi, ki, vi = q[i].copy(), k[i].copy(), v[i].copy()
            L.k_rope_apply(lh.ptr(qi), lh.ptr(ki), lh.ptr(table[length + j]), heads, kv, hd)
            want[i, :dq] = qi
            for c, x in ((caches[0], ki), (caches[1], vi)):
                b.row(c, layout, r, length + j)[:] = (pu.to_bf16(x) if bf16 else x).reshape(kv, hd)
    assert np.array_equal(hu.bits(got), hu.bits(want))
    assert np.array_equal(cache_host(kd).view(np.uint8), caches[0].view(np.uint8))
    assert np.array_equal(cache_host(vd).view(np.uint8), caches[1].view(np.uint8))


@pytest.mark.parametrize("heads,kv,hd", [(4, 2, 64), (5, 5, 6), (3, 1, 130)])
def test_appended_values_of_every_kind_round_as_bf16_does(L, heads, kv, hd):
    """Ties both ways, denormals, the largest floats (which round to infinity), zeros of both signs, infinities and NaN."""
    L.kernels_kv_layout_select(b"head")
    rng = np.random.default_rng(hd)
    b = pu.Pages(hu.dev, [3, 40], [5, 0], bf16=True)
    bits = rng.integers(0, 1 << 32, (b.rows, kv * hd), dtype=np.uint64).astype(np.uint32)  # any float at all
    kinds = np.array([0x3F808000, 0x3F818000, 0x3F817FFF, 0x3F818001, 1, 0x8000, 0x18000, 0x807FFFFF, 0x007F8000, 0x7F7FFFFF,
                      0x7F7F7FFF, 0xFF7FFFFF, 0, 0x80000000, 0x7F800000, 0xFF800000, 0x7FC00000, 0xFF800001], np.uint32)
    bits[:, :len(kinds)] = kinds[:kv * hd]
    bits[::2, :len(kinds)] = kinds[::-1][:kv * hd]
    v = bits.view(F)
    table = rope_table(L, b.seq_len, hd)
    q, k = (rng.standard_normal((b.rows, n * hd), dtype=F) for n in (heads, kv))
    caches = [b.cache(rng, "head", kv, hd) for _ in range(2)]
    kd, vd, out = cache_dev(caches[0]), cache_dev(caches[1]), hu.dev(np.zeros_like(q))
    ins = [hu.dev(x) for x in (q, k, v, table)]
    L.llhip_rope_kv_append_paged(lh.ptr(out), heads * hd, lh.ptr(ins[0]), heads * hd, lh.ptr(ins[1]), lh.ptr(ins[2]), kv * hd,
                                 lh.ptr(ins[3]), None, None, 0.0, b.struct, heads, kv, hd, lh.ptr(kd), lh.ptr(vd))
    quiet(L)
    got = cache_host(vd)
    for r, rows, length in b.requests():
        for j, i in enumerate(range(rows.start, rows.stop)):
            mine, want = b.row(got, "head", r, length + j).reshape(-1), pu.to_bf16(v[i])
            nan = np.isnan(v[i])
            assert np.isnan(pu.values(mine)[nan]).all() and np.array_equal(mine[~nan], want[~nan])


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("heads,kv,hd", [(4, 2, 64), (3, 1, 128), (5, 5, 6), (8, 2, 80), (2, 1, 256), (3, 1, 130)])
@pytest.mark.parametrize("which", ["both", "q", "k"])
def test_appended_rows_behind_norms(L, bf16, heads, kv, hd, which):
    """Norms of queries and keys against float64; a row of zeros, of tiny and of large values among them."""
    L.kernels_kv_layout_select(b"head")
    rng = np.random.default_rng(hd)
    b = pu.Pages(hu.dev, [1, 20, 1], [5, 0, 31], page=16, bf16=bf16, first=1, spare=1)
    table = rope_table(L, b.seq_len, hd)
    q, k, v = (rng.standard_normal((b.rows, n * hd), dtype=F) for n in (heads, kv, kv))
    q[2], k[3], q[4], k[4], q[5], k[6] = 0.0, 0.0, q[4] * F(1e-12), k[4] * F(1e-6), q[5] * F(1e6), k[6] * F(1e15)
    weights = [rng.uniform(0.5, 1.5, hd).astype(F) for _ in range(2)]
    caches = [b.cache(rng, "head", kv, hd) for _ in range(2)]
    qn, kn = hu.dev(weights[0]), hu.dev(weights[1])
    out, kd, vd = hu.dev(np.zeros_like(q)), cache_dev(caches[0]), cache_dev(caches[1])
    ins = [hu.dev(x) for x in (q, k, v, table)]
    L.llhip_rope_kv_append_paged(lh.ptr(out), heads * hd, lh.ptr(ins[0]), heads * hd, lh.ptr(ins[1]), lh.ptr(ins[2]),
                                 kv * hd, lh.ptr(ins[3]), lh.ptr(qn) if which != "k" else None,
                                 lh.ptr(kn) if which != "q" else None, 1e-5, b.struct, heads, kv, hd, lh.ptr(kd), lh.ptr(vd))
    quiet(L)
    got, keys = hu.host(out), cache_host(kd)
    assert not got[0].any() and not got[-1].any()
    for r, rows_, length in b.requests():
        for j, i in enumerate(range(rows_.start, rows_.stop)):
            t = table[length + j]
            qi, ki = q[i].copy(), k[i].copy()
            L.k_rope_apply(lh.ptr(qi), lh.ptr(ki), lh.ptr(t), heads, kv, hd)
            if which != "k":
                want, bound = pu.normed_rope(q[i], weights[0], 1e-5, t, hd)
                within(got[i].reshape(heads, hd), want, bound, ("q", i))
            else:
                assert np.array_equal(hu.bits(got[i]), hu.bits(qi))
            row = pu.values(np.ascontiguousarray(b.row(keys, "head", r, length + j)))
            if which != "q":
                want, bound = pu.normed_rope(k[i], weights[1], 1e-5, t, hd)
                if bf16:  # half a step of BF16, and of its subnormals
                    bound = bound + (np.abs(want) + bound) * 2.0 ** -8 + 2.0 ** -134
                within(row, want, bound, ("k", i))
            else:
                want = pu.values(pu.to_bf16(ki)) if bf16 else ki
                assert np.array_equal(hu.bits(row), hu.bits(want.reshape(kv, hd)))


@pytest.mark.parametrize("count", [1, 255, 256, 257, 1024])
def test_append_many_requests(L, count):
    """As many requests as a call takes, some without rows; pages of one position and of more."""
    L.kernels_kv_layout_select(b"head")
    rng = np.random.default_rng(count)
    rows_of = rng.choice([0, 1, 1, 1, 3], count)
    rows_of[0] = 1
    for page in (1, 32):
        b = pu.Pages(hu.dev, rows_of, rng.integers(0, 60, count), page=page, first=1, spare=2, seed=count)
        heads, kv, hd = 2, 1, 16
        table = np.concatenate((np.ones((b.seq_len, hd), F), np.zeros((b.seq_len, hd), F)), 1)  # no rotation
        q, k, v = (rng.standard_normal((b.rows, n * hd), dtype=F) for n in (heads, kv, kv))
        caches = [b.cache(rng, "head", kv, hd) for _ in range(2)]
        out, kd, vd = hu.dev(np.zeros_like(q)), hu.dev(caches[0]), hu.dev(caches[1])
        ins = [hu.dev(x) for x in (q, k, v, table)]
        L.llhip_rope_kv_append_paged(lh.ptr(out), heads * hd, lh.ptr(ins[0]), heads * hd, lh.ptr(ins[1]), lh.ptr(ins[2]),
                                     kv * hd, lh.ptr(ins[3]), None, None, 0.0, b.struct, heads, kv, hd, lh.ptr(kd),
                                     lh.ptr(vd))
        quiet(L)
        want = np.zeros_like(q)
        for r, rows_, length in b.requests():
            want[rows_] = q[rows_]
            for j, i in enumerate(range(rows_.start, rows_.stop)):
                b.row(caches[0], "head", r, length + j)[:] = k[i]
                b.row(caches[1], "head", r, length + j)[:] = v[i]
        assert np.array_equal(hu.host(out), want)
        assert np.array_equal(hu.host(kd), caches[0]) and np.array_equal(hu.host(vd), caches[1])


def test_append_refuses_what_lies_outside(L):
    """A request outside the buffers stores nothing and fails at the wait, the others are done; a row whose page lies outside
    the caches is not stored; two requests that append to one page fail."""
    heads, kv, hd = 2, 1, 8
    L.kernels_kv_layout_select(b"head")

    def call(change, seq_len=None):
        b = pu.Pages(lambda x: x, [2, 2], [0, 30], page=16, seq_len=seq_len)
        change(b)
        keep = [hu.dev(a) for a in (b.start, b.length, b.table)]
        b.struct.start, b.struct.length, b.struct.pages = (lh.ptr(a) for a in keep)
        kd, vd = (hu.dev(np.zeros(b.shape("head", kv, hd), F)) for _ in range(2))
        table = np.concatenate((np.ones((b.seq_len, hd), F), np.zeros((b.seq_len, hd), F)), 1)
        q, k, t = hu.dev(np.ones((4, heads * hd), F)), hu.dev(np.ones((4, kv * hd), F)), hu.dev(table)
        out = hu.dev(np.zeros((4, heads * hd), F))
        L.llhip_rope_kv_append_paged(lh.ptr(out), heads * hd, lh.ptr(q), heads * hd, lh.ptr(k), lh.ptr(k), kv * hd,
                                     lh.ptr(t), None, None, 0.0, b.struct, heads, kv, hd, lh.ptr(kd), lh.ptr(vd))
        L.llhip_synchronize()
        return hu.host(out), hu.host(kd)

    def set_(name, i, value):
        def change(b):
            getattr(b, name).reshape(-1)[i] = value
        return change

    for change, seq_len in ((set_("start", 2, 5), None), (set_("start", 1, 5), None), (set_("start", 0, -1), None),
                            (set_("length", 1, -1), None), (set_("length", 1, 63), None), (set_("length", 1, 2 ** 31 - 1), None),
                            (set_("length", 1, 34), 35)):
        call(change, seq_len)
        message = lh.last_error()
        L.llhip_clear_error()
        assert "lie outside the batch's buffers" in message, message
    got, _ = call(set_("length", 1, 63))
    L.llhip_clear_error()
    assert got[:2].all() and not got[2:].any()
    for bad in (-1, 6, 2 ** 31 - 1, -2 ** 31):
        def second(b):
            assert b.pool == 6
            b.table[1, 1] = bad
        got, keys = call(second)  # positions 30 and 31 of request 1
        message = lh.last_error()
        L.llhip_clear_error()
        assert "a page of a request lies outside the caches" in message, message
        assert got.all() and keys.sum() == 2 * hd

    def same(b):
        b.table[0, 0] = b.table[1, 1]
    call(same)
    message = lh.last_error()
    L.llhip_clear_error()
    assert "two requests of one call append to the same page" in message, message
    got, keys = call(lambda b: None)
    assert not lh.last_error() and keys.sum() == 4 * hd


# ---- attention -----------------------------------------------------------------------------------------------------------


def attention_case(L, seed, heads, kv, hd, layout, b, *, caches=None, q=None, stride=0, form="dev", tolerance=1.0):
    L.kernels_kv_layout_select(layout.encode())
    rng = np.random.default_rng(seed)
    dq = heads * hd
    wide = rng.standard_normal((b.rows, dq + stride), dtype=F)
    if q is not None:
        wide[:, :dq] = q
    q = np.ascontiguousarray(wide[:, :dq])
    key, value = caches or (b.cache(rng, layout, kv, hd), b.cache(rng, layout, kv, hd))
    want, bound = pu.attention(b, q, key, value, heads, kv, hd, layout)
    put = shifted if form == "shifted" else hu.dev
    qd, kd, vd = put(wide), cache_dev(key), cache_dev(value)
    out = put(np.full((b.rows, dq), 7.0, F))
    L.llhip_attention_paged(lh.ptr(out), lh.ptr(qd), dq + stride, lh.ptr(kd), lh.ptr(vd), b.struct, heads, kv, hd)
    quiet(L)
    got = hu.host(out)
    mine = np.zeros(b.rows, bool)
    for _, rows, _ in b.requests():
        mine[rows] = True
    assert (got[~mine] == 7.0).all()
    if mine.any():
        within(got[mine], want[mine], bound[mine] * tolerance, (heads, kv, hd, layout, b.page))
    return got


@pytest.mark.parametrize("layout", ["head", "rows"])
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("heads,kv,hd", [(8, 2, 64), (32, 8, 128), (4, 4, 128), (16, 1, 64), (6, 2, 80), (10, 2, 96),
                                         (4, 2, 256), (5, 1, 8), (3, 1, 30), (4, 2, 7), (8, 1, 200), (2, 1, 160)])
@pytest.mark.parametrize("page", [1, 16, 24, 64])
def test_attention_of_single_rows(L, layout, bf16, heads, kv, hd, page):
    """One new token a request: lengths of none, one, around a step's and a page's ends, and longer; requests without a row,
    rows of nobody."""
    lengths = [0, 1, 14, 15, 16, 30, 31, 32, 47, 63, 64, 65, 5, 127, 200, 331]
    rows_of = [0 if i == 12 else 1 for i in range(len(lengths))]
    b = pu.Pages(hu.dev, rows_of, lengths, page=page, bf16=bf16, first=1, spare=2, seed=page)
    attention_case(L, hd, heads, kv, hd, layout, b, stride=4 if page == 16 else 0)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("heads,kv,hd", [(8, 2, 64), (32, 8, 128), (6, 2, 80), (4, 4, 96), (16, 1, 128), (4, 2, 256), (6, 2, 36)])
@pytest.mark.parametrize("page", [8, 16, 32, 128])
def test_attention_of_drafts_and_prompts(L, bf16, heads, kv, hd, page):
    """Requests of one row, drafts and prompts in one batch, in sizes around the tiles' (16 to 128 query vectors), behind
    nothing and behind longer parts; the first pages shared."""
    rows_of = [1, 2, 0, 7, 33, 1, 129, 64, 5, 17]
    lengths = [256, 300, 256, 257, 400, 511, 256, 290, 700, 256]
    b = pu.Pages(hu.dev, rows_of, lengths, page=page, bf16=bf16, shared=256, first=3, spare=1, seed=page)
    attention_case(L, hd, heads, kv, hd, "head", b)
    b = pu.Pages(hu.dev, [20, 1, 150, 3], [0, 0, 0, 1], page=page, bf16=bf16, seed=page)
    attention_case(L, hd, heads, kv, hd, "rows" if page == 16 else "head", b)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("heads,kv,hd,length", [(32, 8, 128, 9000), (8, 2, 64, 20011), (16, 1, 128, 5000), (6, 2, 96, 3333)])
def test_attention_split_over_a_long_cache(L, bf16, heads, kv, hd, length):
    """One request's positions over many blocks, with a short one beside it."""
    b = pu.Pages(hu.dev, [1, 1], [length, 3], page=16, bf16=bf16)
    attention_case(L, length, heads, kv, hd, "head", b)
    b = pu.Pages(hu.dev, [6], [length - 777], page=64, bf16=bf16)
    attention_case(L, length, heads, kv, hd, "rows", b)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("rows_of", [[1], [6], [12], [40], [1, 30, 2]])
@pytest.mark.parametrize("heads,kv,hd,length,page", [(256, 128, 8, 19000, 16), (256, 128, 8, 19000, 48), (600, 600, 8, 6000, 64),
                                                     (600, 600, 8, 2000, 20)])
def test_attention_of_many_kv_heads(L, bf16, rows_of, heads, kv, hd, length, page):
    """So many KV heads that one or four blocks take all positions of one: thousands of positions a wave, past those whose pages
    it looks up at once."""
    b = pu.Pages(hu.dev, rows_of, [length, 40, 700][:len(rows_of)], page=page, bf16=bf16)
    attention_case(L, length, heads, kv, hd, "head", b)


@pytest.mark.parametrize("kv,hd", [(4096, 8), (4097, 8)])
@pytest.mark.parametrize("bf16", [False, True])
def test_attention_of_the_most_kv_heads(L, bf16, kv, hd):
    """On both sides of the matrix-core form's limit."""
    b = pu.Pages(hu.dev, [1, 5], [70, 3], page=16, bf16=bf16)
    attention_case(L, kv, kv, kv, hd, "rows", b)


@pytest.mark.parametrize("count", [64, 255, 257, 1024])
def test_attention_many_requests(L, count):
    rng = np.random.default_rng(count)
    rows_of = rng.choice([0, 1, 1, 1, 4, 9], count)
    b = pu.Pages(hu.dev, rows_of, rng.integers(0, 90, count), page=16, bf16=count % 2 == 0, first=1, spare=2)
    attention_case(L, count, 4, 2, 64, "head", b)


def test_attention_without_rows(L):
    b = pu.Pages(hu.dev, [0, 0, 0], [0, 5, 9], first=2, spare=5)
    attention_case(L, 1, 4, 2, 64, "head", b)


@pytest.mark.parametrize("hd,kv,layout,form", [(64, 2, "head", "shifted"), (128, 1, "rows", "shifted"), (128, 3, "rows", "dev")])
@pytest.mark.parametrize("bf16", [False, True])
def test_attention_off_alignment(L, bf16, hd, kv, layout, form):
    """q and out off 16-byte boundaries, a q stride that is no multiple of 4."""
    b = pu.Pages(hu.dev, [1, 5, 40], [100, 37, 3], page=16, bf16=bf16)
    attention_case(L, 3, 4 * kv, kv, hd, layout, b, form=form, stride=3)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("rows_of", [[1, 1, 1], [6, 70, 1]])
def test_attention_over_caches_off_alignment(L, bf16, rows_of):
    """Caches on the alignment of one value."""
    heads, kv, hd = 8, 2, 64
    L.kernels_kv_layout_select(b"head")
    b = pu.Pages(hu.dev, rows_of, [100, 37, 3], page=16, bf16=bf16)
    rng = np.random.default_rng(4)
    caches = [b.cache(rng, "head", kv, hd) for _ in range(2)]
    q = rng.standard_normal((b.rows, heads * hd), dtype=F)
    want, bound = pu.attention(b, q, *caches, heads, kv, hd, "head")
    T = hu.torch()
    views = []
    for c in caches:
        flat = hu.empty(c.size + 1, T.int16 if bf16 else T.float32)
        flat[1:].copy_(T.from_numpy((c.view(np.int16) if bf16 else c).reshape(-1)))
        views.append(flat[1:])
    qd, out = hu.dev(q), hu.dev(np.zeros_like(q))
    T.cuda.synchronize()
    L.llhip_attention_paged(lh.ptr(out), lh.ptr(qd), heads * hd, lh.ptr(views[0]), lh.ptr(views[1]), b.struct, heads, kv, hd)
    quiet(L)
    within(hu.host(out), want, bound)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("rows_of", [[1, 1], [1, 40]])
def test_attention_of_scores_far_below_zero(L, bf16, rows_of):
    """Scores of -1e38, the same for all positions: their weights are equal, as for any others."""
    heads, kv, hd = 8, 2, 8
    b = pu.Pages(hu.dev, rows_of, [100, 30], page=16, bf16=bf16)
    rng = np.random.default_rng(5)
    q = np.full((b.rows, heads * hd), 2.0 ** 60, F)
    key = np.full(b.shape("head", kv, hd), -(2.0 ** 63), F)  # a dot of -8 * 2^123, a score of -3e37 * sqrt(8)
    value = b.cache(rng, "head", kv, hd)
    got = attention_case_equal_scores(L, b, q, pu.to_bf16(key) if bf16 else key, value, heads, kv, hd)
    for r, rows, length in b.requests():
        seen = length + rows.stop - rows.start
        vals = b.gather(value, "head", r, seen)
        for j, i in enumerate(range(rows.start, rows.stop)):
            n = length + j + 1
            mean = np.repeat(vals[:, :n].mean(1), heads // kv, 0)
            size = np.repeat(np.abs(vals[:, :n]).mean(1), heads // kv, 0)
            assert (np.abs(got[i].reshape(heads, hd) - mean) <= (3 * n + 72) * ru.U * size).all()


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("rows_of", [[1, 1], [7], [1, 40]])
@pytest.mark.parametrize("hd", [64, 128, 50])
def test_attention_over_denormal_keys(L, bf16, rows_of, hd):
    """Keys below 2^-126 under queries of 2^124: scores as any others."""
    heads, kv = 8, 2
    b = pu.Pages(hu.dev, rows_of, [100, 30][:len(rows_of)], page=16, bf16=bf16)
    rng = np.random.default_rng(6)
    key = (rng.integers(-15, 16, b.shape("head", kv, hd)) * 2.0 ** -132).astype(F)
    assert (np.abs(key) < 2.0 ** -126).all()
    q = (rng.standard_normal((b.rows, heads * hd)) * 2.0 ** 124).astype(F)
    caches = [pu.to_bf16(key) if bf16 else key, b.cache(rng, "head", kv, hd)]
    attention_case(L, 3, heads, kv, hd, "head", b, caches=caches, q=q)


def attention_case_equal_scores(L, b, q, key, value, heads, kv, hd):
    L.kernels_kv_layout_select(b"head")
    qd, kd, vd, out = hu.dev(q), cache_dev(key), cache_dev(value), hu.dev(np.zeros_like(q))
    L.llhip_attention_paged(lh.ptr(out), lh.ptr(qd), heads * hd, lh.ptr(kd), lh.ptr(vd), b.struct, heads, kv, hd)
    quiet(L)
    return hu.host(out)


@pytest.mark.parametrize("bf16", [False, True])
def test_pages_past_32_bits(L, bf16):
    """Caches of more than 2^32 bytes and 2^31 values, their last pages in use: appended rows and attention, single rows and a
    prompt's."""
    T = hu.torch()
    L.kernels_kv_layout_select(b"head")
    heads, kv, hd, page = 8, 2, 128, 64
    pages = (1 << 31) // (kv * page * hd) + 40
    dtype = T.int16 if bf16 else T.float32
    big = [T.empty((pages, kv, page, hd), dtype=dtype, device="cuda") for _ in range(2)]
    rng = np.random.default_rng(6)
    b = pu.Pages(lambda x: x, [1, 70, 1], [150, 30, 0], page=page, bf16=bf16)
    shift = pages - b.pool  # the pool lies at the caches' end
    keep = [hu.dev(a) for a in (b.start, b.length, np.where(b.table < 0, -1, b.table + shift).astype(np.int32))]
    b.struct.start, b.struct.length, b.struct.pages = (lh.ptr(a) for a in keep)
    b.struct.num_pages = pages
    caches = [b.cache(rng, "head", kv, hd) for _ in range(2)]
    for x, c in zip(big, caches):
        x[shift:].copy_(T.from_numpy(c.view(np.int16) if bf16 else c))
    table = rope_table(L, b.seq_len, hd)
    q, k, v = (rng.standard_normal((b.rows, n * hd), dtype=F) for n in (heads, kv, kv))
    dev = [hu.dev(x) for x in (q, k, v, table)]
    rot, out = hu.dev(np.zeros_like(q)), hu.dev(np.zeros_like(q))
    T.cuda.synchronize()
    L.llhip_rope_kv_append_paged(lh.ptr(rot), heads * hd, lh.ptr(dev[0]), heads * hd, lh.ptr(dev[1]), lh.ptr(dev[2]), kv * hd,
                                 lh.ptr(dev[3]), None, None, 0.0, b.struct, heads, kv, hd, lh.ptr(big[0]), lh.ptr(big[1]))
    L.llhip_attention_paged(lh.ptr(out), lh.ptr(rot), heads * hd, lh.ptr(big[0]), lh.ptr(big[1]), b.struct, heads, kv, hd)
    quiet(L)
    for r, rows, length in b.requests():
        for j, i in enumerate(range(rows.start, rows.stop)):
            qi, ki = q[i].copy(), k[i].copy()
            L.k_rope_apply(lh.ptr(qi), lh.ptr(ki), lh.ptr(table[length + j]), heads, kv, hd)
            for c, x in ((caches[0], ki), (caches[1], v[i])):
                b.row(c, "head", r, length + j)[:] = (pu.to_bf16(x) if bf16 else x).reshape(kv, hd)
    for x, c in zip(big, caches):
        got = hu.host(x[shift:])
        assert np.array_equal(got.view(np.uint8), c.view(np.uint8))
    want, bound = pu.attention(b, hu.host(rot), *caches, heads, kv, hd, "head")
    within(hu.host(out), want, bound)


def test_calls_from_two_threads(L):
    """Attention over pages and scoring from two threads at once, whose kernels share one workspace."""
    import threading
    L.kernels_kv_layout_select(b"head")
    rng = np.random.default_rng(7)
    heads, kv, hd = 8, 2, 64
    b = pu.Pages(hu.dev, [1, 3] * 8, rng.integers(0, 2000, 16), page=16)
    caches = [b.cache(rng, "head", kv, hd) for _ in range(2)]
    q = rng.standard_normal((b.rows, heads * hd), dtype=F)
    want, bound = pu.attention(b, q, *caches, heads, kv, hd, "head")
    qd, kd, vd, out = hu.dev(q), hu.dev(caches[0]), hu.dev(caches[1]), hu.dev(np.zeros_like(q))
    logits, tokens = rng.standard_normal((40, 5000)).astype(F), rng.integers(0, 5000, 40).astype(np.int32)
    ld, td, lp = hu.dev(logits), hu.dev(tokens), hu.dev(np.zeros(40, F))

    def attend():
        for _ in range(200):
            L.llhip_attention_paged(lh.ptr(out), lh.ptr(qd), heads * hd, lh.ptr(kd), lh.ptr(vd), b.struct, heads, kv, hd)

    def score():
        for _ in range(200):
            L.llhip_token_logprobs(lh.ptr(lp), None, None, None, 0, lh.ptr(ld), 5000, lh.ptr(td), 40, 5000, 1.0)

    attend(), score()
    quiet(L)
    alone = hu.host(lp).copy()
    team = [threading.Thread(target=f) for f in (attend, score)]
    for t in team:
        t.start()
    for t in team:
        t.join()
    quiet(L)
    within(hu.host(out), want, bound)
    assert np.array_equal(hu.host(lp), alone)


@pytest.mark.parametrize("rows_of,lengths", [([1], [30000]), ([1, 200, 3], [700, 900, 4000])])
def test_a_call_repeats_itself_bit_for_bit(L, rows_of, lengths):
    """The parts of a walk are joined in their order, whichever block comes last."""
    heads, kv, hd = 32, 8, 128
    L.kernels_kv_layout_select(b"head")
    for bf16 in (False, True):
        b = pu.Pages(hu.dev, rows_of, lengths, page=16, bf16=bf16)
        rng = np.random.default_rng(8)
        qd = hu.dev(rng.standard_normal((b.rows, heads * hd), dtype=F))
        caches = [cache_dev(b.cache(rng, "head", kv, hd)) for _ in range(2)]
        first = None
        for _ in range(20):
            out = hu.dev(np.zeros((b.rows, heads * hd), F))
            L.llhip_attention_paged(lh.ptr(out), lh.ptr(qd), heads * hd, lh.ptr(caches[0]), lh.ptr(caches[1]), b.struct, heads,
                                    kv, hd)
            quiet(L)
            got = hu.host(out)
            assert first is None or np.array_equal(got, first)
            first = got


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("rows_of,lengths", [([1, 1], [33, 200]), ([3, 40], [61, 100])])
@pytest.mark.parametrize("hd", [64, 128, 72])
@pytest.mark.parametrize("page", [64, 20, 27])
def test_attention_leaves_the_pages_rest_alone(L, bf16, rows_of, lengths, hd, page):
    """NaN and infinities in pages that no request names, and behind the last position of a request's last page."""
    heads, kv = 8, 2
    b = pu.Pages(hu.dev, rows_of, lengths, page=page, bf16=bf16)
    rng = np.random.default_rng(8)
    caches = [b.cache(rng, "head", kv, hd) for _ in range(2)]
    bad = np.array([np.nan, np.inf, -np.inf, 3e38], F)
    for c in caches:
        odd = pu.to_bf16(bad) if bf16 else bad
        for free in b.free:
            c[free] = rng.choice(odd, c[free].shape)
        for r, rows, length in b.requests():
            seen = length + rows.stop - rows.start
            if seen % page:
                c[b.table[r, seen // page]][:, seen % page:] = rng.choice(odd, (kv, page - seen % page, hd))
    attention_case(L, 9, heads, kv, hd, "head", b, caches=caches)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("hd", [64, 128, 256, 50])
@pytest.mark.parametrize("what", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("page", [16, 12])
def test_a_value_that_is_not_finite_reaches_the_rows_that_see_it(L, bf16, hd, what, page):
    """One V value of a prompt's own rows: the rows before it keep their results, in every dimension; the rows that see it
    have it in its dimension alone, and other requests nothing of it."""
    heads, kv, layout = 8, 2, "head"
    L.kernels_kv_layout_select(layout.encode())
    b = pu.Pages(hu.dev, [50, 1, 6], [20, 90, 30], page=page, bf16=bf16)
    rng = np.random.default_rng(4)
    key, value = b.cache(rng, layout, kv, hd), b.cache(rng, layout, kv, hd)
    q = rng.standard_normal((b.rows, heads * hd), dtype=F)
    want, bound = pu.attention(b, q, key, value, heads, kv, hd, layout)
    hit = {0: (33, 1, 3), 2: (33, 0, 1)}  # request: position, KV head, dimension
    for r, (t, g, d) in hit.items():
        b.row(value, layout, r, t)[g, d] = pu.to_bf16(np.array([what], F))[0] if bf16 else what
    qd, kd, vd, out = hu.dev(q), cache_dev(key), cache_dev(value), hu.dev(np.zeros_like(q))
    L.llhip_attention_paged(lh.ptr(out), lh.ptr(qd), heads * hd, lh.ptr(kd), lh.ptr(vd), b.struct, heads, kv, hd)
    quiet(L)
    got = hu.host(out).reshape(b.rows, heads, hd)
    odd = np.zeros(got.shape, bool)
    for r, rows, length in b.requests():
        if r in hit:
            t, g, d = hit[r]
            odd[rows.start + max(t - length, 0):rows.stop, g * 4:(g + 1) * 4, d] = True
    assert (~np.isfinite(got[odd])).all()
    if np.isnan(what):
        assert np.isnan(got[odd]).all()
    fine = ~odd
    within(got[fine], want.reshape(got.shape)[fine], bound.reshape(got.shape)[fine], (hd, what))


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("heads,kv,hd", [(8, 2, 64), (8, 2, 128), (4, 2, 256), (6, 2, 80), (8, 2, 50)])
@pytest.mark.parametrize("rows_of,lengths", [([1], [70]), ([3, 1], [40, 200]), ([50, 1, 6], [20, 90, 30]), ([1], [9000]),
                                             ([2, 40], [5000, 3000])])
@pytest.mark.parametrize("page", [16, 12])
def test_a_seen_infinity_gives_infinity(L, bf16, heads, kv, hd, rows_of, lengths, page):
    """V values that are not finite, wherever a row sees them and whatever their weight: infinity gives infinity, both signs or
    a NaN give NaN, in their dimension alone. One lies at the position of the largest score of some row (a weight of 1, whose
    lower parts are zero), others where weights are far below the smallest float (scores some hundreds apart), at the first
    position, in the middle and in the prompts' own rows."""
    L.kernels_kv_layout_select(b"head")
    b = pu.Pages(hu.dev, rows_of, lengths, page=page, bf16=bf16)
    rng = np.random.default_rng(hd + len(rows_of))
    key, value = b.cache(rng, "head", kv, hd), b.cache(rng, "head", kv, hd)
    q = rng.standard_normal((b.rows, heads * hd), dtype=F)
    q[::2] *= F(60.0)
    clean = value.copy()
    for r, rows, length in b.requests():
        seen, n = length + rows.stop - rows.start, rows.stop - rows.start
        scores = b.gather(key, "head", r, length + 1)[1] @ q[rows.start].reshape(heads, hd)[heads // kv]
        places = [(0, 0, 1, np.inf), (int(scores.argmax()), 1, 2, np.inf), (int(scores.argmin()), 1, 3, -np.inf),
                  (length // 2, 0, 4, np.inf), (length // 2 + 1, 0, 4, -np.inf), (length // 3, 1, 5, np.nan),
                  (length + n // 2, 0, hd - 1, np.inf), (seen - 1, 1, hd - 2, -np.inf)]
        for t, g, d, x in places:
            b.row(value, "head", r, t)[g, d] = pu.to_bf16(np.array([x], F))[0] if bf16 else x
    want, bound = pu.attention(b, q, key, clean, heads, kv, hd, "head")
    want, bound = want.reshape(b.rows, heads, hd), bound.reshape(b.rows, heads, hd)
    for r, rows, length in b.requests():
        vals = b.gather(value, "head", r, length + rows.stop - rows.start)
        for j, i in enumerate(range(rows.start, rows.stop)):
            with np.errstate(invalid="ignore"):
                odd = np.repeat(np.where(np.isfinite(vals), 0.0, vals)[:, :length + j + 1].sum(1), heads // kv, 0)
            want[i] = np.where(odd == 0.0, want[i], odd)
    got = attention_case_equal_scores(L, b, q, key, value, heads, kv, hd).reshape(want.shape)
    odd = ~np.isfinite(want)
    assert odd.any() and np.array_equal(got[odd], want[odd], equal_nan=True)
    within(got[~odd], want[~odd], bound[~odd], (heads, kv, hd, page))


STAIRS = [([1], [400], (3, 131, 259)), ([6], [400], (3, 131, 259)), ([60], [400], (3, 131, 259)),
          ([1], [9000], (3, 131, 8900)), ([40], [5000], (3, 131, 4900))]
# beside long requests, which make the parts of 8 KV heads' walks longer
LONG_STAIRS = [([1] * 11, [400] + [4000] * 10, (3, 131, 259)), ([60] + [1] * 12, [400] + [6000] * 12, (3, 35, 67))]


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("heads,kv,hd,rows_of,lengths,places",
                         [(*shape, *c) for shape in [(8, 2, 64), (8, 2, 128), (4, 2, 256), (6, 2, 50)] for c in STAIRS] +
                         [(16, 8, 64, *c) for c in STAIRS + LONG_STAIRS])
def test_weights_near_the_smallest_float(L, bf16, heads, kv, hd, rows_of, lengths, places):
    """Scores, in powers of two, of 0, 7.9 and 126.5, in steps of one wave that follow each other and in two parts of a walk:
    the second's weight is 2^-118.6 of the largest, and with a V of 1e30 there it is all that the row has."""
    L.kernels_kv_layout_select(b"head")
    b = pu.Pages(hu.dev, rows_of, lengths, page=16, bf16=bf16)
    key, value = (np.zeros(b.shape("head", kv, hd), F) for _ in range(2))
    q = np.zeros((b.rows, heads, hd), F)
    q[:, :, 0] = np.sqrt(hd) * np.log(2.0)
    key[..., 0] = -100.0
    for t, score in zip(places, (0.0, 7.90625, 126.5)):
        b.row(key, "head", 0, t)[:, 0] = score
    b.row(value, "head", 0, places[1])[:] = 1e30
    caches = [pu.to_bf16(x) if bf16 else x for x in (key, value)]
    attention_case(L, 1, heads, kv, hd, "head", b, caches=caches, q=q.reshape(b.rows, -1))


def test_attention_fails_for_scores_that_are_not_finite(L):
    L.kernels_kv_layout_select(b"head")
    for hd, rows_of, lengths in ((64, [1], [40]), (128, [20], [10]), (40, [1], [13]), (18, [2], [9])):
        for bf16 in (False, True):
            b = pu.Pages(hu.dev, rows_of, lengths, bf16=bf16)
            rng = np.random.default_rng(1)
            for what in (np.nan, np.inf):
                key, value = b.cache(rng, "head", 1, hd), b.cache(rng, "head", 1, hd)
                b.row(key, "head", 0, 5)[0, 2] = pu.to_bf16(np.array([what], F))[0] if bf16 else what
                q = hu.dev(rng.standard_normal((b.rows, 2 * hd), dtype=F))
                kd, vd, out = cache_dev(key), cache_dev(value), hu.dev(np.zeros((b.rows, 2 * hd), F))
                L.llhip_attention_paged(lh.ptr(out), lh.ptr(q), 2 * hd, lh.ptr(kd), lh.ptr(vd), b.struct, 2, 1, hd)
                fails(L, "nonfinite value in softmax")


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("rows_of", [[1, 1, 1], [1, 40, 1]])
def test_attention_of_extreme_values(L, bf16, rows_of):
    """Queries so large that one position takes all the weight, of zeros, and values of very different sizes."""
    heads, kv, hd = 8, 2, 128
    b = pu.Pages(hu.dev, rows_of, [100, 300, 700], page=32, bf16=bf16)
    rng = np.random.default_rng(2)
    q = rng.standard_normal((b.rows, heads * hd), dtype=F)
    q[0] *= F(100.0)
    q[-1] = 0.0
    key, value = (rng.standard_normal(b.shape("head", kv, hd), dtype=F) for _ in range(2))
    value *= (10.0 ** rng.uniform(-20, 20, value.shape[:3] + (1,))).astype(F)
    caches = [pu.to_bf16(x) if bf16 else x for x in (key, value)]
    attention_case(L, 3, heads, kv, hd, "head", b, caches=caches, q=q)


def test_attention_fails_for_pages_outside_the_caches(L):
    """The request with such a page fails at the wait; the other requests' rows are right. A page behind the last position
    is not looked at."""
    heads, kv, hd = 8, 2, 64
    L.kernels_kv_layout_select(b"head")
    rng = np.random.default_rng(6)
    for rows_of in ([1, 1, 1], [1, 30, 1]):
        for page in (16, 12):
            b = pu.Pages(hu.dev, rows_of, [40, 70, 200], page=page)
            key, value = b.cache(rng, "head", kv, hd), b.cache(rng, "head", kv, hd)
            q = rng.standard_normal((b.rows, heads * hd), dtype=F)
            want, bound = pu.attention(b, q, key, value, heads, kv, hd, "head")
            qd, kd, vd, out = hu.dev(q), hu.dev(key), hu.dev(value), hu.dev(np.zeros_like(q))
            for bad in (-1, b.pool, 2 ** 31 - 1, -2 ** 31):
                table = b.table.copy()
                table[1, 2] = bad
                table[0, -1] = 2 ** 30  # behind its last position
                b.keep[2].copy_(hu.torch().from_numpy(table))
                hu.torch().cuda.synchronize()
                out.zero_()
                hu.torch().cuda.synchronize()
                L.llhip_attention_paged(lh.ptr(out), lh.ptr(qd), heads * hd, lh.ptr(kd), lh.ptr(vd), b.struct, heads, kv, hd)
                fails(L, "a page of a request lies outside the caches")
                got = hu.host(out)
                for r, rows, _ in b.requests():
                    if r != 1:
                        within(got[rows], want[rows], bound[rows], (r, bad))


def test_attention_fails_for_requests_outside_the_buffers(L):
    """Such a request's rows are left as they are, the others are right."""
    heads, kv, hd = 4, 2, 64
    L.kernels_kv_layout_select(b"head")
    rng = np.random.default_rng(7)
    b = pu.Pages(hu.dev, [1, 2, 1], [40, 70, 90], seq_len=91)
    key, value = b.cache(rng, "head", kv, hd), b.cache(rng, "head", kv, hd)
    q = rng.standard_normal((b.rows, heads * hd), dtype=F)
    want, bound = pu.attention(b, q, key, value, heads, kv, hd, "head")
    qd, kd, vd = hu.dev(q), hu.dev(key), hu.dev(value)
    T = hu.torch()
    for name, array, lost in (("length", [40, -1, 90], {1}), ("length", [40, 90, 90], {1}), ("length", [40, 2 ** 31 - 1, 90], {1}),
                              ("start", [0, 1, 3, 5], {2}), ("start", [0, 1, 0, 4], {1, 2}), ("start", [-2 ** 31, 1, 3, 4], {0})):
        for x, y in ((b.keep[0], b.start), (b.keep[1], b.length)):
            x.copy_(T.from_numpy(y))
        b.keep[0 if name == "start" else 1].copy_(T.from_numpy(np.array(array, np.int64).astype(np.int32)))
        out = hu.dev(np.full(q.shape, 7.0, F))
        L.llhip_attention_paged(lh.ptr(out), lh.ptr(qd), heads * hd, lh.ptr(kd), lh.ptr(vd), b.struct, heads, kv, hd)
        fails(L, "lie outside the batch's buffers")
        got = hu.host(out)
        for r, rows, _ in b.requests():
            if r not in lost:
                within(got[rows], want[rows], bound[rows], (name, array, r))
            elif name == "length":
                assert (got[rows] == 7.0).all()


# ---- host buffers, graphs, both together -----------------------------------------------------------------------------------


def test_host_buffers(L):
    """Arrays, rows and caches in host memory: the calls copy them in and out and wait."""
    heads, kv, hd = 8, 2, 64
    L.kernels_kv_layout_select(b"head")
    rng = np.random.default_rng(10)
    for bf16 in (False, True):
        b = pu.Pages(lambda x: x, [1, 3], [37, 5], bf16=bf16, first=1, spare=1)
        caches = [b.cache(rng, "head", kv, hd) for _ in range(2)]
        table = rope_table(L, b.seq_len, hd)
        q, k, v = (rng.standard_normal((b.rows, n * hd), dtype=F) for n in (heads, kv, kv))
        rot = np.full_like(q, 7.0)
        L.llhip_rope_kv_append_paged(lh.ptr(rot), heads * hd, lh.ptr(q), heads * hd, lh.ptr(k), lh.ptr(v), kv * hd,
                                     lh.ptr(table), None, None, 0.0, b.struct, heads, kv, hd, lh.ptr(caches[0]),
                                     lh.ptr(caches[1]))
        assert not lh.last_error(), lh.last_error()
        assert (rot[0] == 7.0).all() and (rot[-1] == 7.0).all()
        for r, rows, length in b.requests():
            for j, i in enumerate(range(rows.start, rows.stop)):
                qi, ki = q[i].copy(), k[i].copy()
                L.k_rope_apply(lh.ptr(qi), lh.ptr(ki), lh.ptr(table[length + j]), heads, kv, hd)
                assert np.array_equal(rot[i], qi)
                assert np.array_equal(b.row(caches[0], "head", r, length + j).reshape(-1), pu.to_bf16(ki) if bf16 else ki)
        out = np.full_like(q, 7.0)
        L.llhip_attention_paged(lh.ptr(out), lh.ptr(rot), heads * hd, lh.ptr(caches[0]), lh.ptr(caches[1]), b.struct, heads,
                                kv, hd)
        assert not lh.last_error(), lh.last_error()
        want, bound = pu.attention(b, rot, *caches, heads, kv, hd, "head")
        assert (out[0] == 7.0).all() and (out[-1] == 7.0).all()
        within(out[1:-1], want[1:-1], bound[1:-1])


@pytest.mark.parametrize("rows_of", [[1, 1, 1], [1, 40, 6]])
def test_a_captured_step_follows_the_arrays(L, rows_of):
    """A served step (append, attention) captured once and replayed with other lengths, page tables and starts, each replay
    against the eager calls; eager calls on other operands, which take a larger workspace, between them."""
    T = hu.torch()
    L.kernels_kv_layout_select(b"head")
    rng = np.random.default_rng(12)
    heads, kv, hd = 8, 2, 128
    b = pu.Pages(hu.dev, rows_of, [300, 290, 310], page=16, bf16=True)
    caches = [cache_dev(b.cache(rng, "head", kv, hd)) for _ in range(2)]
    table = hu.dev(rope_table(L, b.seq_len, hd))
    q, k, v = (hu.dev(rng.standard_normal((b.rows, n * hd), dtype=F)) for n in (heads, kv, kv))
    rot, out = hu.dev(np.zeros((b.rows, heads * hd), F)), hu.dev(np.zeros((b.rows, heads * hd), F))
    other = pu.Pages(hu.dev, [1] * 40, rng.integers(100, 4000, 40), page=16, bf16=True)
    other_cache = [cache_dev(other.cache(rng, "head", kv, hd)) for _ in range(2)]
    other_q = hu.dev(rng.standard_normal((40, heads * hd), dtype=F))
    other_out = hu.dev(np.zeros((40, heads * hd), F))

    def calls():
        L.llhip_rope_kv_append_paged(lh.ptr(rot), heads * hd, lh.ptr(q), heads * hd, lh.ptr(k), lh.ptr(v), kv * hd,
                                     lh.ptr(table), None, None, 0.0, b.struct, heads, kv, hd, lh.ptr(caches[0]),
                                     lh.ptr(caches[1]))
        L.llhip_attention_paged(lh.ptr(out), lh.ptr(rot), heads * hd, lh.ptr(caches[0]), lh.ptr(caches[1]), b.struct, heads,
                                kv, hd)

    calls()  # the workspace grows outside of the capture
    quiet(L)
    assert L.llhip_graph_begin() == 0, lh.last_error()
    calls()
    graph = L.llhip_graph_end()
    assert graph, lh.last_error()
    for lengths in ([3, 200, 100], [310, 0, 5], [100, 290, 0]):
        order = rng.permutation(b.pool)
        need = -(-(np.array(lengths) + rows_of) // 16)
        tab = np.full_like(b.table, -1)
        at = 0
        for r, n in enumerate(need):
            tab[r, :n] = order[at:at + n]
            at += n
        b.keep[1].copy_(T.from_numpy(np.asarray(lengths, np.int32)))
        b.keep[2].copy_(T.from_numpy(tab))
        b.length[:], b.table[:] = lengths, tab
        T.cuda.synchronize()
        start = [c.clone() for c in caches]
        T.cuda.synchronize()
        calls()
        quiet(L)
        want = [x.clone() for x in (rot, out, *caches)]
        for c, s in zip(caches, start):
            c.copy_(s)
        rot.zero_(), out.zero_()
        T.cuda.synchronize()
        L.llhip_attention_paged(lh.ptr(other_out), lh.ptr(other_q), heads * hd, lh.ptr(other_cache[0]),
                                lh.ptr(other_cache[1]), other.struct, heads, kv, hd)
        assert L.llhip_graph_launch(graph) == 0
        quiet(L)
        for g, w in zip((rot, out, *caches), want):
            assert T.equal(g, w)
        plain, bound = pu.attention(b, hu.host(rot), cache_host(caches[0]), cache_host(caches[1]), heads, kv, hd, "head")
        within(hu.host(out), plain, bound, lengths)
    L.llhip_graph_destroy(graph)


GROWING = r'''
import sys
sys.path[:0] = [sys.argv[1], sys.argv[1] + "/llama3.x.c_amd"]
import numpy as np
import llama_hip as lh
from tests import hip_util as hu, paged_util as pu
L = lh.load()
assert L.llhip_init() == 0
lh.record_failures()
L.kernels_kv_layout_select(b"head")
T = hu.torch()
rng = np.random.default_rng(1)

def make(rows_of, lengths, heads, kv, hd):
    b = pu.Pages(hu.dev, rows_of, lengths, page=16, bf16=True)
    caches = [b.cache(rng, "head", kv, hd) for _ in range(2)]
    q = rng.standard_normal((b.rows, heads * hd), dtype=np.float32)
    want, bound = pu.attention(b, q, *caches, heads, kv, hd, "head")
    dev = [hu.dev(q)] + [hu.dev(c.view(np.int16)) for c in caches]
    return dict(b=b, dev=dev, out=hu.dev(np.zeros_like(q)), want=want, bound=bound, shape=(heads, kv, hd))

def call(m):
    q, k, v = (lh.ptr(x) for x in m["dev"])
    heads, kv, hd = m["shape"]
    L.llhip_attention_paged(lh.ptr(m["out"]), q, heads * hd, k, v, m["b"].struct, heads, kv, hd)

def right(m):
    got = hu.host(m["out"]).astype(np.float64)
    assert not lh.last_error(), lh.last_error()
    assert (np.abs(got - m["want"]) <= m["bound"]).all()
    m["out"].zero_()
    T.cuda.synchronize()

small, large = make([1, 1, 1], [3000, 2500, 40], 8, 2, 64), make([1, 40, 6], [900, 2900, 310], 8, 2, 128)
start = L.llhip_hbm_claimed()
call(small)
right(small)
one = L.llhip_hbm_claimed() - start
assert one > 0
assert L.llhip_graph_begin() == 0, lh.last_error()
call(small)
assert not lh.last_error(), lh.last_error()
graph = L.llhip_graph_end()
assert graph, lh.last_error()
# a capture that would need more is refused, and nothing of it is kept
assert L.llhip_graph_begin() == 0, lh.last_error()
call(large)
message = lh.last_error()
L.llhip_clear_error()
empty = L.llhip_graph_end()
if empty:
    L.llhip_graph_destroy(empty)
L.llhip_clear_error()
assert "workspace during graph capture" in message, message
assert L.llhip_hbm_claimed() - start == one
for turn in range(3):
    assert L.llhip_graph_launch(graph) == 0
    right(small)
    call(large)
    right(large)
    assert L.llhip_hbm_claimed() - start > 2.25 * one, (one, L.llhip_hbm_claimed())  # another buffer, beside the captured one
    other = T.full((64 << 20,), float("nan"), device="cuda")
    T.cuda.synchronize()
    assert L.llhip_graph_launch(graph) == 0
    call(large)
    right(small)
    right(large)
    assert T.isnan(other).all()
L.llhip_graph_destroy(graph)
print("workspace ok", flush=True)
'''


def test_a_captured_call_keeps_its_workspace():
    """In a process of its own, whose workspace no other test has grown: a graph captured on the first workspace replays right
    behind eager calls that take a larger one, which comes beside it; a capture that would need more than there is is refused."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", GROWING, root], capture_output=True, text=True, timeout=110)
    assert r.returncode == 0 and "workspace ok" in r.stdout, (r.stdout[-2000:], r.stderr[-4000:])


def test_calls_from_threads_that_share_a_workspace(L):
    """Two batches' attention over pages at once, which share the pages' workspace and counters, beside scoring and attention
    behind a shared prefix, which share the requests'."""
    L.kernels_kv_layout_select(b"head")
    rng = np.random.default_rng(17)
    heads, kv, hd = 8, 2, 64
    jobs = []
    for rows_of, lengths, bf16 in (([1, 3] * 8, rng.integers(0, 2000, 16), False), ([2, 70, 1], [4000, 300, 2500], True)):
        b = pu.Pages(hu.dev, rows_of, lengths, page=16, bf16=bf16)
        caches = [b.cache(rng, "head", kv, hd) for _ in range(2)]
        q = rng.standard_normal((b.rows, heads * hd), dtype=F)
        want, bound = pu.attention(b, q, *caches, heads, kv, hd, "head")
        dev, out = [hu.dev(q)] + [cache_dev(c) for c in caches], hu.dev(np.zeros_like(q))

        def attend(b=b, dev=dev, out=out):
            L.llhip_attention_paged(lh.ptr(out), lh.ptr(dev[0]), heads * hd, lh.ptr(dev[1]), lh.ptr(dev[2]), b.struct, heads, kv,
                                    hd)

        jobs.append((attend, lambda out=out, want=want, bound=bound: within(hu.host(out), want, bound)))
    logits, tokens = rng.standard_normal((40, 5000)).astype(F), rng.integers(0, 5000, 40).astype(np.int32)
    ld, td, lp = hu.dev(logits), hu.dev(tokens), hu.dev(np.zeros(40, F))
    scored = pu.scores(logits, tokens, 1.0, 0)[0]

    def score():
        L.llhip_token_logprobs(lh.ptr(lp), None, None, None, 0, lh.ptr(ld), 5000, lh.ptr(td), 40, 5000, 1.0)

    # z of at most 10: the sum is off by (2 * 10 + 28) U of itself, a log probability of at most 16 by U of its own, together
    # below 4e-6
    jobs.append((score, lambda: within(hu.host(lp), scored, np.full(40, 1e-5))))
    r = ru.Batch(hu.dev, [1] * 20, rng.integers(0, 100, 20), prefix=300, prefix_seq_len=300, seq_len=128)
    a = [rng.standard_normal(n, dtype=F) for n in ((r.rows, heads * hd), (kv, 300, hd), (kv, 300, hd), (r.slots, kv, 128, hd),
                                                   (r.slots, kv, 128, hd))]
    behind, behind_bound = ru.attention(r, *a, heads, kv, hd, "head")
    rdev, rout = [hu.dev(x) for x in a], hu.dev(np.zeros_like(a[0]))
    jobs.append((lambda: L.llhip_attention_requests(lh.ptr(rout), *[lh.ptr(x) for x in rdev], r.struct, heads, kv, hd),
                 lambda: within(hu.host(rout), behind, behind_bound)))
    for run, _ in jobs:
        run()
    quiet(L)

    def many(run):
        for _ in range(150):
            run()

    team = [threading.Thread(target=many, args=(run,)) for run, _ in jobs]
    for t in team:
        t.start()
    for t in team:
        t.join()
    quiet(L)
    for _, check in jobs:
        check()


@pytest.mark.parametrize("bf16", [False, True])
def test_a_prompt_and_its_answer_over_pages(L, bf16):
    """A served sequence: its prompt in two chunks, then tokens one by one beside another request's, each step's rows appended
    and attended; against float64 over the keys and values in order, and, for F32 pages, against the single sequence's own
    calls."""
    L.kernels_kv_layout_select(b"head")
    rng = np.random.default_rng(13)
    heads, kv, hd, page = 8, 2, 64, 16
    total = [75, 40]
    steps = [([30, 0], [0, 0]), ([35, 38], [30, 0])] + [([1, 1 if i < 2 else 0], [65 + i, 38 + i]) for i in range(10)]
    pool = 12
    order = rng.permutation(pool).astype(np.int32)
    tables = np.stack((order[:6], np.concatenate((order[6:9], [-1, -1, -1])))).astype(np.int32)
    dtype = np.uint16 if bf16 else F
    caches = [cache_dev(np.zeros((pool, kv, page, hd), dtype)) for _ in range(2)]
    table = rope_table(L, 96, hd)
    td, pages = hu.dev(table), hu.dev(tables)
    full = [[rng.standard_normal((n, m * hd), dtype=F) for m in (heads, kv, kv)] for n in total]
    weights = [rng.uniform(0.8, 1.2, hd).astype(F) for _ in range(2)]
    wd = [hu.dev(w) for w in weights]
    outs = [np.zeros((n, heads * hd), F) for n in total]
    for rows_of, lengths in steps:
        start = np.concatenate(([0], np.cumsum(rows_of))).astype(np.int32)
        sd, ld = hu.dev(start), hu.dev(np.asarray(lengths, np.int32))
        struct = lh.PagedBatch(lh.ptr(sd), lh.ptr(ld), lh.ptr(pages), 2, int(start[-1]), 6, page, pool, 96,
                               lh.PAGE_BF16 if bf16 else lh.PAGE_F32)
        q, k, v = (hu.dev(np.concatenate([full[r][i][lengths[r]:lengths[r] + rows_of[r]] for r in range(2)]))
                   for i in range(3))
        out = hu.dev(np.zeros(tuple(q.shape), F))
        L.llhip_rope_kv_append_paged(lh.ptr(q), heads * hd, lh.ptr(q), heads * hd, lh.ptr(k), lh.ptr(v), kv * hd, lh.ptr(td),
                                     lh.ptr(wd[0]), lh.ptr(wd[1]), 1e-6, struct, heads, kv, hd, lh.ptr(caches[0]),
                                     lh.ptr(caches[1]))
        L.llhip_attention_paged(lh.ptr(out), lh.ptr(q), heads * hd, lh.ptr(caches[0]), lh.ptr(caches[1]), struct, heads, kv,
                                hd)
        quiet(L)
        got = hu.host(out)
        for r in range(2):
            outs[r][lengths[r]:lengths[r] + rows_of[r]] = got[start[r]:start[r + 1]]
    for r in range(2):
        n, mul = total[r], heads // kv
        turned = [np.stack([pu.normed_rope(full[r][i][t], weights[i], 1e-6, table[t], hd)[0] for t in range(n)])
                  for i in range(2)]
        q, k, v = turned[0], turned[1].astype(F), full[r][2].reshape(n, kv, hd)
        if bf16:
            k, v = pu.values(pu.to_bf16(k)), pu.values(pu.to_bf16(v))
        for t in range(n):
            for h in range(heads):
                s = k[:t + 1, h // mul].astype(np.float64) @ q[t, h] / np.sqrt(hd)
                p = np.exp(s - s.max())
                want = (p / p.sum()) @ v[:t + 1, h // mul]
                # a key that rounds to the other neighbour in BF16 (its float32 norm is off by a few U) moves its score by a
                # step of one of hd products; the norms' own error moves scores by (hd + 24) U of sum|q k|
                spread = (np.abs(k[:t + 1, h // mul]) @ np.abs(q[t, h])).max() / np.sqrt(hd)
                step = (np.abs(k[:t + 1, h // mul]).max() * np.abs(q[t, h]).max() / np.sqrt(hd)) * 2.0 ** -7 if bf16 else 0.0
                off = 2 * (spread * (4 * hd + 40) * ru.U + 4 * step) + (3 * t + 80) * ru.U
                assert np.abs(outs[r][t].reshape(heads, hd)[h] - want).max() <= off * np.abs(v[:t + 1, h // mul]).max()
