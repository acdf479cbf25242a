"""Many requests on one model, on the GPU: each operator against its plain float64 form (tests/requests_util.py, the bounds
derived there), its index checks, host buffers and captured calls; and a small model served by all of them together."""
import ctypes
import mmap
import os

import numpy as np
import pytest

import llama_hip as lh
from llama_hip import checkpoint as ck
from tests import hip_util as hu
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


def shifted(a, floats=1):
    """A device copy of `a` whose address is 4 * floats bytes off the allocation's 16-byte alignment."""
    t = hu.torch()
    flat = hu.empty(a.size + floats, t.float32)
    view = flat[floats:].reshape(a.shape)
    view.copy_(t.from_numpy(a))
    t.cuda.synchronize()
    return view


# ---- RoPE and cache rows ------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("layout", ["head", "rows"])
@pytest.mark.parametrize("heads,kv,hd", [(4, 2, 64), (3, 1, 128), (5, 5, 6), (8, 2, 80), (2, 1, 256)])
@pytest.mark.parametrize("packed", [False, True])
def test_rope_rows_equal_the_single_calls_bit_for_bit(L, layout, heads, kv, hd, packed):
    """Against k_rope_apply and k_kv_store of each row alone: ragged requests (none, one and many rows), permuted slots,
    rows before the first and behind the last request, in place on packed QKV rows or into another buffer."""
    L.kernels_kv_layout_select(layout.encode())
    rng = np.random.default_rng(hd + heads)
    b = ru.Batch(hu.dev, [3, 0, 1, 40, 2], [0, 99, 7, 11, 30], slot=[4, 77, 0, 5, 2], slots=7, prefix=9, seq_len=53, first=2,
                 spare=3)
    dq, dkv = heads * hd, kv * hd
    cfg = lh.Config(head_dim=hd, rope_theta=500000.0)
    table = np.zeros((9 + 53, 2 * hd), F)
    for p in range(len(table)):
        L.k_rope_table(ru.byref(cfg), p, lh.ptr(table[p]))
    caches = [rng.standard_normal((7,) + ru.cache_shape(layout, 53, kv, hd), dtype=F) for _ in range(2)]
    wide = rng.standard_normal((b.rows, dq + 2 * dkv + 4), dtype=F)
    q, k, v = wide[:, :dq], wide[:, dq:dq + dkv], wide[:, dq + dkv:dq + 2 * dkv]
    kd, vd, td = hu.dev(caches[0]), hu.dev(caches[1]), hu.dev(table)
    if packed:
        rows = hu.dev(wide)
        qd, kr, vr = rows, rows[:, dq:], rows[:, dq + dkv:]
        out, stride, kv_stride = rows, wide.shape[1], wide.shape[1]
    else:
        qd, kr, vr = (hu.dev(np.ascontiguousarray(x)) for x in (q, k, v))
        out, stride, kv_stride = hu.dev(np.full((b.rows, dq), 7.0, F)), dq, dkv
    L.llhip_rope_kv_store_requests(lh.ptr(out), lh.ptr(qd), stride, lh.ptr(kr), lh.ptr(vr), kv_stride, lh.ptr(td),
                                   b.struct, heads, kv, hd, lh.ptr(kd), lh.ptr(vd))
    quiet(L)
    got = hu.host(out)[:, :dq]
    want = q.copy() if packed else np.full((b.rows, dq), 7.0, F)
    for _, rows_, length, slot in b.requests():
        for j, i in enumerate(range(rows_.start, rows_.stop)):
            qi, ki, vi = q[i].copy(), k[i].copy(), v[i].copy()
            L.k_rope_apply(lh.ptr(qi), lh.ptr(ki), lh.ptr(table[9 + length + j]), heads, kv, hd)
            want[i] = qi
            for c, x in ((caches[0], ki), (caches[1], vi)):
                ru.by_head(c[slot], layout)[:, length + j] = x.reshape(kv, hd)
    assert np.array_equal(hu.bits(got), hu.bits(want))
    assert np.array_equal(hu.bits(hu.host(kd)), hu.bits(caches[0]))
    assert np.array_equal(hu.bits(hu.host(vd)), hu.bits(caches[1]))
    if packed:
        assert np.array_equal(hu.host(rows)[:, dq:], wide[:, dq:])


def test_rope_rows_refuse_what_lies_outside(L):
    """A request outside the buffers stores nothing and fails at the wait, the others are done; two requests in one slot
    fail."""
    heads, kv, hd, seq = 2, 1, 8, 10
    L.kernels_kv_layout_select(b"head")
    table = hu.dev(np.ones((seq, 2 * hd), F))
    q, k = hu.dev(np.ones((4, heads * hd), F)), hu.dev(np.ones((4, kv * hd), F))

    def call(**over):
        args = {"rows_of": [2, 2], "length": [0, 3], "slot": [0, 1], "slots": 2, "seq_len": seq}
        args.update(over)
        b = ru.Batch(hu.dev, **args)
        out = hu.dev(np.zeros((4, heads * hd), F))
        caches = [hu.dev(np.zeros((2, kv, seq, hd), F)) for _ in range(2)]
        L.llhip_rope_kv_store_requests(lh.ptr(out), lh.ptr(q), heads * hd, lh.ptr(k), lh.ptr(k), kv * hd, lh.ptr(table),
                                       b.struct, heads, kv, hd, lh.ptr(caches[0]), lh.ptr(caches[1]))
        return out, caches

    call()
    quiet(L)
    for over in ({"length": [0, 9]}, {"length": [0, -1]}, {"slot": [0, 2]}, {"slot": [0, -1]},
                 {"length": [0, 2 ** 31 - 1]}):
        out, caches = call(**over)
        fails(L, "outside the batch's buffers")
        got, cache = hu.host(out), hu.host(caches[1])  # (1, 1) turned by (1, 1) is (0, 2): the values are counted
        assert (got[2:] == 0).all() and (got[:2] != 0).any()
        assert np.count_nonzero(cache[0]) == 2 * hd and not cache[1].any()
    call(slot=[1, 1])
    fails(L, "into the same slot")
    # a request without rows may hold any length and slot
    call(rows_of=[4, 0], length=[0, -7], slot=[0, 99])
    quiet(L)


# ---- attention --------------------------------------------------------------------------------------------------------


def attention_case(L, seed, heads, kv, hd, layout, b, offset=0, scale=1.0, nan_spare=True):
    """Random operands of a batch, the call's output and the float64 one; the spare rows' q is NaN and their out kept."""
    L.kernels_kv_layout_select(layout.encode())
    rng = np.random.default_rng(seed)
    q = scale * rng.standard_normal((b.rows, heads * hd), dtype=F)
    pk, pv = (rng.standard_normal(ru.cache_shape(layout, max(b.prefix_seq_len, 1), kv, hd), dtype=F) for _ in range(2))
    k, v = (rng.standard_normal((b.slots,) + ru.cache_shape(layout, b.seq_len, kv, hd), dtype=F) for _ in range(2))
    live = np.zeros(b.rows, bool)
    for _, rows, length, slot in b.requests():
        live[rows] = True
    if nan_spare:  # what no row may see: idle rows, cache places behind every request's last row
        q[~live] = np.nan
        end = np.zeros(b.slots, int)
        for _, rows, length, slot in b.requests():
            end[slot] = max(end[slot], length + rows.stop - rows.start)
        for c in (k, v):
            for s in range(b.slots):
                ru.by_head(c[s], layout)[:, end[s]:] = np.nan
        for c in (pk, pv):
            ru.by_head(c, layout)[:, b.prefix:] = np.nan
    put = (lambda a: shifted(a, offset)) if offset else hu.dev
    out = put(np.full((b.rows, heads * hd), 5.0, F))
    args = [put(a) for a in (q, pk, pv, k, v)]
    L.llhip_attention_requests(lh.ptr(out), *[lh.ptr(a) for a in args], b.struct, heads, kv, hd)
    quiet(L)
    got = hu.host(out)
    clean = [np.nan_to_num(a) for a in (q, pk, pv, k, v)]
    want, bound = ru.attention(b, clean[0], clean[1], clean[2], clean[3], clean[4], heads, kv, hd, layout)
    want[~live] = 5.0
    within(got, want, bound)
    return got


SHAPES = [(4, 2, 64), (8, 2, 128), (32, 8, 64), (3, 3, 128), (6, 1, 64), (16, 1, 128), (4, 2, 80), (2, 1, 256), (3, 1, 7),
          (5, 1, 96), (12, 4, 48)]


@pytest.mark.parametrize("layout", ["head", "rows"])
@pytest.mark.parametrize("heads,kv,hd", SHAPES)
def test_attention_decode(L, layout, heads, kv, hd):
    """One row a request (and requests without rows) at ragged lengths from the first own position on, permuted slots."""
    b = ru.Batch(hu.dev, [1, 1, 0, 1, 1, 1], [0, 63, 5, 64, 200, 1], slot=[3, 1, 0, 6, 2, 4], slots=7, prefix=131,
                 prefix_seq_len=140, seq_len=202, first=1, spare=2)
    attention_case(L, hd, heads, kv, hd, layout, b)


@pytest.mark.parametrize("prefix", [0, 1, 31, 32, 33, 64, 255, 700])
@pytest.mark.parametrize("heads,kv,hd", [(8, 2, 128), (4, 2, 64), (4, 4, 96)])
def test_attention_prefix_lengths(L, prefix, heads, kv, hd):
    b = ru.Batch(hu.dev, [1, 3, 1], [0, 0, 32], prefix=prefix, prefix_seq_len=prefix + 3, seq_len=40)
    attention_case(L, prefix, heads, kv, hd, "head", b)


@pytest.mark.parametrize("rows_of,length", [([2, 7, 1, 5], [10, 0, 64, 31]), ([1], [0]), ([33], [0]), ([130, 1, 65], [0, 90, 3]),
                                            ([16, 17, 32, 31], [1, 2, 3, 4]), ([1] * 70, list(range(70)))])
@pytest.mark.parametrize("heads,kv,hd", [(8, 2, 128), (4, 4, 64), (10, 2, 64), (6, 2, 80)])
def test_attention_drafts_and_prompts(L, rows_of, length, heads, kv, hd):
    """Several rows a request, causal among themselves, over tile edges; more vectors than a tile holds."""
    b = ru.Batch(hu.dev, rows_of, length, prefix=77, prefix_seq_len=80, seq_len=160, spare=1)
    attention_case(L, len(rows_of), heads, kv, hd, "head", b)


@pytest.mark.parametrize("heads,kv,hd", [(8, 2, 128), (4, 2, 64)])
def test_attention_shared_slots_and_long_own(L, heads, kv, hd):
    """Requests that read one slot, and lengths far apart: one of 3000 own positions beside short ones."""
    b = ru.Batch(hu.dev, [1, 1, 2, 1], [2999, 3, 40, 0], slot=[1, 0, 1, 2], prefix=2000, prefix_seq_len=2000, seq_len=3001)
    attention_case(L, 5, heads, kv, hd, "head", b)


@pytest.mark.parametrize("offset", [1, 2])
def test_attention_unaligned(L, offset):
    b = ru.Batch(hu.dev, [1, 4], [20, 0], prefix=50, prefix_seq_len=51, seq_len=30)
    attention_case(L, 9, 4, 2, 64, "head", b, offset=offset)


def test_attention_sharp_scores(L):
    """Scores of some hundred units: one position takes nearly the whole weight, in the prefix or behind it."""
    b = ru.Batch(hu.dev, [1, 2, 1], [100, 40, 0], prefix=300, prefix_seq_len=300, seq_len=128)
    attention_case(L, 10, 8, 2, 128, "head", b, scale=30.0)


@pytest.mark.parametrize("rows_of", [[1, 3], [40, 20]])
def test_attention_spread_values(L, rows_of):
    """Keys and values of very different sizes from position to position and dimension to dimension."""
    L.kernels_kv_layout_select(b"head")
    heads, kv, hd = 8, 2, 128
    b = ru.Batch(hu.dev, rows_of, [90 - rows_of[0], 0], prefix=200, prefix_seq_len=200, seq_len=100)
    rng = np.random.default_rng(11)
    spread = lambda shape: (rng.standard_normal(shape) * 10.0 ** rng.uniform(-6, 4, shape)).astype(F)  # noqa: E731
    q = (1e-3 * rng.standard_normal((b.rows, heads * hd))).astype(F)
    pk, k = (1e-2 * spread((kv, 200, hd))).astype(F), (1e-2 * spread((2, kv, 100, hd))).astype(F)
    pv, v = spread((kv, 200, hd)), spread((2, kv, 100, hd))
    out = hu.dev(np.zeros_like(q))
    args = [hu.dev(a) for a in (q, pk, pv, k, v)]
    L.llhip_attention_requests(lh.ptr(out), *[lh.ptr(a) for a in args], b.struct, heads, kv, hd)
    quiet(L)
    want, bound = ru.attention(b, q, pk, pv, k, v, heads, kv, hd, "head")
    within(hu.host(out), want, bound)


@pytest.mark.parametrize("rows_of", [[1, 3], [40, 20]])
@pytest.mark.parametrize("sizes", [(1e35,), (1e-20,), (1e24, 1.0, 0.0), (1e10, 1e-15, 0.0), (0.0,)])
def test_attention_value_sizes(L, rows_of, sizes):
    """V rows of extreme sizes, position by position, and of zeros; keys and queries whose scores stay ordinary. (The sums
    are divided by the weights' at the end, so the values of n positions with weights near the largest must stay below
    3.4e38 / n, here 3.4e38 / 290 = 1.2e36; 1e38 overflows, in k_attention too.)"""
    L.kernels_kv_layout_select(b"head")
    heads, kv, hd = 8, 2, 128
    b = ru.Batch(hu.dev, rows_of, [90 - rows_of[0], 0], prefix=200, prefix_seq_len=200, seq_len=100)
    rng = np.random.default_rng(12)
    size = lambda n: np.asarray(sizes, F)[np.arange(n) // 8 % len(sizes)][:, None]  # noqa: E731
    q = (1e-30 * rng.standard_normal((b.rows, heads * hd))).astype(F)
    pk, k = ((1e30 * rng.standard_normal(s)).astype(F) for s in ((kv, 200, hd), (2, kv, 100, hd)))
    pv, v = (size(s[-2]) * rng.uniform(0.5, 1.5, s).astype(F) for s in ((kv, 200, hd), (2, kv, 100, hd)))
    out = hu.dev(np.zeros_like(q))
    args = [hu.dev(a) for a in (q, pk, pv, k, v)]
    L.llhip_attention_requests(lh.ptr(out), *[lh.ptr(a) for a in args], b.struct, heads, kv, hd)
    quiet(L)
    want, bound = ru.attention(b, q, pk, pv, k, v, heads, kv, hd, "head")
    within(hu.host(out), want, bound)


@pytest.mark.parametrize("heads,kv,hd", [(8, 2, 128), (4, 2, 64), (10, 2, 80)])
@pytest.mark.parametrize("form", ["element", "half", "own"])
@pytest.mark.parametrize("raised", [1e2, 1e4, 1e7, 1e12, 1e30])
def test_attention_large_value_elements(L, heads, kv, hd, form, raised):
    """Tiles of a block over V rows of which some elements are far larger than the rest: one element of a prefix row, half
    the dimensions of eight rows, one element of an own row that only the later rows see. The other dimensions' sums keep
    their own accuracy."""
    L.kernels_kv_layout_select(b"head")
    rng = np.random.default_rng(13)
    b = ru.Batch(hu.dev, [40, 30], [37, 5], prefix=256, prefix_seq_len=256, seq_len=96)
    q = rng.standard_normal((b.rows, heads * hd), dtype=F)
    pk, pv = (rng.standard_normal((kv, 256, hd), dtype=F) for _ in range(2))
    k, v = (rng.standard_normal((2, kv, 96, hd), dtype=F) for _ in range(2))
    if form == "element":
        pv[:, 100, 3] = raised
    elif form == "half":
        pv[:, rng.choice(256, 8, replace=False), hd // 2:] *= F(raised)
    else:
        v[0, :, 50, hd - 1] = raised
    out = hu.dev(np.zeros_like(q))
    dev = [hu.dev(a) for a in (q, pk, pv, k, v)]
    L.llhip_attention_requests(lh.ptr(out), *[lh.ptr(a) for a in dev], b.struct, heads, kv, hd)
    quiet(L)
    want, bound = ru.attention(b, q, pk, pv, k, v, heads, kv, hd, "head")
    within(hu.host(out), want, bound)


@pytest.mark.parametrize("layout", ["head", "rows"])
@pytest.mark.parametrize("heads,kv,hd", [(16, 1, 128), (6, 2, 64), (8, 2, 128)])
def test_attention_large_elements_in_some_slices(L, layout, heads, kv, hd):
    """A prefix cut into slices of which one holds a large element, an own walk that holds another beside a V value that is
    not finite and only the last row sees; the parts with and without meet in the same rows."""
    L.kernels_kv_layout_select(layout.encode())
    rng = np.random.default_rng(heads)
    b = ru.Batch(hu.dev, [45, 1, 20], [700, 3, 0], prefix=3000, prefix_seq_len=3001, seq_len=760)
    q = rng.standard_normal((b.rows, heads * hd), dtype=F)
    pk, pv = (rng.standard_normal(ru.cache_shape(layout, 3001, kv, hd), dtype=F) for _ in range(2))
    k, v = (rng.standard_normal((3,) + ru.cache_shape(layout, 760, kv, hd), dtype=F) for _ in range(2))
    ru.by_head(pv, layout)[0, 1700, 5] = 1e12
    ru.by_head(v[0], layout)[:, 650, hd - 2] = -1e9
    want, bound = ru.attention(b, q, pk, pv, k, v, heads, kv, hd, layout)
    ru.by_head(v[0], layout)[0, 744, 9] = np.inf  # request 0's last row's own position
    out = hu.dev(np.zeros_like(q))
    dev = [hu.dev(a) for a in (q, pk, pv, k, v)]
    L.llhip_attention_requests(lh.ptr(out), *[lh.ptr(a) for a in dev], b.struct, heads, kv, hd)
    quiet(L)
    got = hu.host(out).reshape(b.rows, heads, hd)
    hit = np.zeros(got.shape, bool)
    hit[44, :heads // kv, 9] = True
    assert (got[hit] == np.inf).all()
    within(got[~hit], want.reshape(got.shape)[~hit], bound.reshape(got.shape)[~hit])


@pytest.mark.parametrize("sizes", [(1e-17, 1e-19), (1e-28,), (1e-28, 1.0), (1.0, 100.0, 0.0, 0.01)])
def test_attention_small_values(L, sizes):
    """Tiles of a block over V rows below what the FP16 parts' exponents take, and around the border; rows of zeros between
    others; the first rows larger or smaller than the rest."""
    L.kernels_kv_layout_select(b"head")
    heads, kv, hd = 8, 2, 128
    b = ru.Batch(hu.dev, [40, 30], [50, 0], prefix=200, prefix_seq_len=200, seq_len=100)
    rng = np.random.default_rng(15)
    size = lambda n: np.asarray(sizes, F)[np.arange(n) // 8 % len(sizes)][:, None]  # noqa: E731
    q = rng.standard_normal((b.rows, heads * hd), dtype=F)
    pk, k = (rng.standard_normal(s, dtype=F) for s in ((kv, 200, hd), (2, kv, 100, hd)))
    pv, v = (size(s[-2]) * rng.uniform(0.5, 1.5, s).astype(F) for s in ((kv, 200, hd), (2, kv, 100, hd)))
    out = hu.dev(np.zeros_like(q))
    args = [hu.dev(a) for a in (q, pk, pv, k, v)]
    L.llhip_attention_requests(lh.ptr(out), *[lh.ptr(a) for a in args], b.struct, heads, kv, hd)
    quiet(L)
    want, bound = ru.attention(b, q, pk, pv, k, v, heads, kv, hd, "head")
    within(hu.host(out), want, bound)


@pytest.mark.parametrize("heads,kv,hd", [(8, 2, 128), (4, 2, 64)])
@pytest.mark.parametrize("gap", [5.0, 12.0, 18.0])
def test_attention_one_position_without_values(L, heads, kv, hd, gap):
    """Nearly the whole weight, all but exp(-gap) or less, on a position whose V row is zero among ordinary ones, so that
    the outputs are the small weights' sums. A weight is held to 2^-36 of the row's largest over V rows of one size, and the
    exponents of four normal rows' largest differ by two at most: 2^-34 of each value beside the plain bound."""
    L.kernels_kv_layout_select(b"head")
    rng = np.random.default_rng(14)
    b = ru.Batch(hu.dev, [40, 30], [37, 5], prefix=256, prefix_seq_len=256, seq_len=96)
    q = (0.5 * rng.standard_normal((b.rows, heads * hd))).astype(F)
    pk, pv = (rng.standard_normal((kv, 256, hd), dtype=F) for _ in range(2))
    k, v = (rng.standard_normal((2, kv, 96, hd), dtype=F) for _ in range(2))
    q.reshape(b.rows, heads, hd)[:, :, 0] = 1.0
    pk[:, :, 0], k[..., 0] = 0.0, 0.0
    pk[:, 33] = 0.0
    pk[:, 33, 0] = (gap + 3.0) * np.sqrt(hd)  # the other scores are below 3
    pv[:, 33] = 0.0
    out = hu.dev(np.zeros_like(q))
    dev = [hu.dev(a) for a in (q, pk, pv, k, v)]
    L.llhip_attention_requests(lh.ptr(out), *[lh.ptr(a) for a in dev], b.struct, heads, kv, hd)
    quiet(L)
    want, bound = ru.attention(b, q, pk, pv, k, v, heads, kv, hd, "head")
    sums = np.abs(pv).sum(1)[None, :, None] + np.abs(v).sum(2).max(0)[None, :, None]
    extra = np.broadcast_to(2.0 ** -34 * sums, (b.rows, kv, heads // kv, hd)).reshape(bound.shape)
    within(hu.host(out), want, bound + extra)


@pytest.mark.parametrize("rows", [3, 20, 45])
@pytest.mark.parametrize("value", [np.inf, -np.inf, np.nan])
def test_attention_nonfinite_values_reach_only_the_rows_that_see_them(L, rows, value):
    """V of an own position that only the last row sees, V of a prefix position in one dimension, K behind the diagonal: the
    other rows and dimensions are as without them (one tile of a wave, and tiles of a block)."""
    L.kernels_kv_layout_select(b"head")
    heads, kv, hd = 8, 2, 128
    rng = np.random.default_rng(rows)
    b = ru.Batch(hu.dev, [rows, 1], [30, 2], prefix=90, prefix_seq_len=90, seq_len=100)
    q = rng.standard_normal((b.rows, heads * hd), dtype=F)
    pk, pv = (rng.standard_normal((kv, 90, hd), dtype=F) for _ in range(2))
    k, v = (rng.standard_normal((2, kv, 100, hd), dtype=F) for _ in range(2))
    want, bound = ru.attention(b, q, pk, pv, k, v, heads, kv, hd, "head")
    pv[1, 40, 7] = value
    v[0, 0, 30 + rows - 1, 64:] = value
    k[0, :, 30 + rows:] = value
    out = hu.dev(np.zeros_like(q))
    dev = [hu.dev(a) for a in (q, pk, pv, k, v)]
    L.llhip_attention_requests(lh.ptr(out), *[lh.ptr(a) for a in dev], b.struct, heads, kv, hd)
    quiet(L)
    got = hu.host(out).reshape(b.rows, heads, hd)
    hit = np.zeros(got.shape, bool)
    hit[:, heads // 2:, 7] = True
    hit[rows - 1, :heads // 2, 64:] = True
    same = np.isnan(got[hit]) if np.isnan(value) else got[hit] == value
    assert same.all()
    rest = ~hit
    within(got[rest], want.reshape(got.shape)[rest], bound.reshape(got.shape)[rest])


def test_attention_refuses_what_lies_outside(L):
    """The rows of a request outside the buffers are left, the others are done, and the wait reports it; a non-finite
    score is reported as k_attention reports it."""
    heads, kv, hd, seq = 4, 2, 64, 40
    L.kernels_kv_layout_select(b"head")
    rng = np.random.default_rng(3)
    q = rng.standard_normal((4, heads * hd), dtype=F)
    pk, pv = (rng.standard_normal((kv, 50, hd), dtype=F) for _ in range(2))
    k, v = (rng.standard_normal((2, kv, seq, hd), dtype=F) for _ in range(2))

    def call(q=q, start=None, **over):
        args = {"rows_of": [2, 2], "length": [0, 3], "slot": [0, 1], "slots": 2, "seq_len": seq, "prefix": 50}
        args.update(over)
        b = ru.Batch(hu.dev, **args)
        if start is not None:
            b.rows = b.struct.rows = 4
            b.keep += (hu.dev(np.asarray(start, np.int32)),)
            b.struct.start = lh.ptr(b.keep[-1])
        out = hu.dev(np.zeros_like(q))
        dev = [hu.dev(a) for a in (q, pk, pv, k, v)]
        L.llhip_attention_requests(lh.ptr(out), *[lh.ptr(a) for a in dev], b.struct, heads, kv, hd)
        return out

    want = hu.host(call())
    quiet(L)
    for over in ({"length": [0, seq - 1]}, {"length": [0, -1]}, {"slot": [0, 2]}, {"slot": [0, -5]}, {"start": [0, 2, 5]},
                 {"start": [0, 2, 1]}, {"start": [0, 2, 2 ** 31 - 1]}):
        out = call(**over)
        fails(L, "outside the batch's buffers")
        got = hu.host(out)
        assert np.array_equal(got[:2], want[:2]) and (got[2:] == 0).all(), over
    out = call(start=[-1, 2, 4])
    fails(L, "outside the batch's buffers")
    assert np.array_equal(hu.host(out)[2:], want[2:]) and (hu.host(out)[:2] == 0).all()
    # requests over each other's rows, each whole in itself: nothing is done
    out = call(rows_of=[1] * 9, length=[0] * 9, slot=[0] * 9, start=[0, 4, 0, 4, 0, 4, 0, 4, 0, 4])
    fails(L, "outside the batch's buffers")
    assert (hu.host(out) == 0).all()
    # rows of a whole request behind start[count]
    out = call(rows_of=[1] * 3, length=[0, 0, 3], slot=[0, 0, 1], start=[0, 0, 2, 0])
    fails(L, "outside the batch's buffers")
    assert np.array_equal(hu.host(out)[:2], want[:2]) and (hu.host(out)[2:] == 0).all()
    worse = q.copy()
    worse[3, 5] = np.inf
    call(q=worse)
    fails(L, "nonfinite value in softmax")


def test_attention_from_host_memory(L):
    """Plain host buffers and arrays: copied in and out, rows without a request kept."""
    heads, kv, hd = 4, 2, 64
    L.kernels_kv_layout_select(b"rows")
    rng = np.random.default_rng(4)
    b = ru.Batch(lambda a: a, [1, 2], [4, 0], prefix=20, prefix_seq_len=24, seq_len=8, spare=1)
    q = rng.standard_normal((b.rows, heads * hd), dtype=F)
    pk, pv = (rng.standard_normal((24, kv, hd), dtype=F) for _ in range(2))
    k, v = (rng.standard_normal((2, 8, kv, hd), dtype=F) for _ in range(2))
    out = np.full_like(q, 3.0)
    L.llhip_attention_requests(*[lh.ptr(a) for a in (out, q, pk, pv, k, v)], b.struct, heads, kv, hd)
    assert not lh.last_error(), lh.last_error()
    want, bound = ru.attention(b, q, pk, pv, k, v, heads, kv, hd, "rows")
    within(out[:3], want[:3], bound[:3])
    assert (out[3] == 3.0).all()


def test_attention_repeats_itself_and_does_not_depend_on_neighbours_order(L):
    """Bit for bit the same on every call."""
    b = ru.Batch(hu.dev, [1] * 9 + [5, 40], [17 * i for i in range(9)] + [500, 0], prefix=1000, prefix_seq_len=1000,
                 seq_len=600)
    first = attention_case(L, 12, 8, 2, 128, "head", b)
    for _ in range(3):
        assert np.array_equal(hu.bits(first), hu.bits(attention_case(L, 12, 8, 2, 128, "head", b)))


# ---- adapters ---------------------------------------------------------------------------------------------------------


def bf16(a):
    """`a` rounded to BF16: its bits, and the values they stand for."""
    bits = hu.bits(a)
    up = ((bits.astype(np.uint64) + 0x7FFF + ((bits >> 16) & 1)) >> 16).astype(np.uint16)
    return up, (up.astype(np.uint32) << 16).view(F).reshape(a.shape)


class Adapters:
    """One segment's operands on the device, and what the call should give."""

    def __init__(self, rng, m, k, n, rank, adapters, is_bf16, swiglu, ldc=None, in_place=False, offset=0, scaled=True):
        self.n, self.rank, self.ldc, self.swiglu, self.is_bf16 = n, rank, ldc or n, swiglu, is_bf16
        self.m = m
        put = (lambda a: shifted(a, offset)) if offset else hu.dev
        self.base = [rng.standard_normal((m, self.ldc), dtype=F) for _ in range(1 + swiglu)]
        self.scale = rng.uniform(0.5, 2.0, adapters).astype(F) if scaled else None
        self.pairs, dev = [], []
        for _ in range(1 + swiglu):
            a = (rng.standard_normal((adapters, rank, k)) / np.sqrt(k)).astype(F)
            b = (rng.standard_normal((adapters, n, rank)) / np.sqrt(rank)).astype(F)
            if is_bf16:
                (abits, a), (bbits, b) = bf16(a), bf16(b)
                if offset:
                    t = hu.torch()
                    pads = []
                    for x in (abits, bbits):
                        flat = hu.dev(np.concatenate((np.zeros(offset, np.uint16), x.reshape(-1))).view(np.int16))
                        pads.append(flat[offset:])
                    dev.append(pads)
                else:
                    dev.append([hu.dev(abits.view(np.int16)), hu.dev(bbits.view(np.int16))])
            else:
                dev.append([put(a), put(b)])
            self.pairs.append((a, b))
        self.c = hu.dev(self.base[0]) if in_place else put(np.full((m, self.ldc), 9.0, F))
        base_dev = [self.c if in_place else put(self.base[0])] + [put(x) for x in self.base[1:]]
        self.in_place = in_place
        scale_dev = None if self.scale is None else hu.dev(self.scale)
        self.keep = (dev, base_dev, scale_dev)
        third = {"base3": base_dev[1], "a3": dev[1][0], "b3": dev[1][1]} if swiglu else {}
        self.struct = ru.lora_segment(is_bf16, self.c, self.ldc, base_dev[0], dev[0][0], dev[0][1], scale_dev, n, rank,
                                      **third)

    def check(self, x, ids):
        scale = np.ones(len(self.pairs[0][0])) if self.scale is None else self.scale.astype(np.float64)
        n = self.n
        want, bound = ru.adapters(x, ids, self.base[0][:, :n], *self.pairs[0], scale)
        if self.swiglu:
            want, bound = ru.swiglu(want, bound, *ru.adapters(x, ids, self.base[1][:, :n], *self.pairs[1], scale))
        got = hu.host(self.c)
        within(got[:, :n], want, bound + 2 * ru.U * np.abs(want), (self.m, n, self.rank))
        pad = self.base[0][:, n:] if self.in_place else np.full((self.m, self.ldc - n), 9.0, F)
        assert np.array_equal(got[:, n:], pad)
        return got


def run_lora(L, x, ldx, k, ids, adapters, segs, is_bf16):
    xd, idd = x if hasattr(x, "data_ptr") else hu.dev(x), hu.dev(np.asarray(ids, np.int32))
    fn = L.llhip_lora_bf16 if is_bf16 else L.llhip_lora_f32
    fn(lh.ptr(xd), ldx, len(ids), k, lh.ptr(idd), adapters, ru.array([s.struct for s in segs]), len(segs))
    return xd, idd


def ids_of(rng, m, adapters, form):
    if form == "each":
        return rng.integers(-1, adapters, m)
    if form == "runs":
        return np.repeat(rng.integers(-1, adapters, m // 7 + 1), 7)[:m]
    return np.full(m, {"one": adapters - 1, "none": -1}[form])


@pytest.mark.parametrize("is_bf16", [False, True])
@pytest.mark.parametrize("form", ["each", "runs", "one", "none"])
@pytest.mark.parametrize("m", [1, 2, 5, 16, 17, 33, 64, 65, 130])
def test_lora_rows(L, is_bf16, form, m):
    """Rows from one to more than a tile, their adapters mixed, in runs, all one, and none at all; three segments."""
    rng = np.random.default_rng(m)
    k, adapters = 320, 6
    x = rng.standard_normal((m, k), dtype=F)
    ids = ids_of(rng, m, adapters, form)
    segs = [Adapters(rng, m, k, n, rank, adapters, is_bf16, False) for n, rank in ((192, 16), (64, 8), (40, 32))]
    keep = run_lora(L, x, k, k, ids, adapters, segs, is_bf16)
    quiet(L)
    for s in segs:
        s.check(x, ids)
    del keep


@pytest.mark.parametrize("is_bf16", [False, True])
@pytest.mark.parametrize("k,n,rank", [(8, 1, 1), (257, 33, 3), (1000, 130, 12), (64, 16, 4), (96, 50, 256), (2048, 257, 64),
                                      (4096, 48, 100), (40, 4000, 24)])
@pytest.mark.parametrize("m", [3, 90])
def test_lora_sizes(L, is_bf16, k, n, rank, m):
    """Odd sizes, ranks to the largest, strided rows and outputs, no scale array."""
    rng = np.random.default_rng(k + n)
    ldx, adapters = k + 5, 3
    wide = rng.standard_normal((m, ldx), dtype=F)
    ids = ids_of(rng, m, adapters, "each")
    s = Adapters(rng, m, k, n, rank, adapters, is_bf16, False, ldc=n + 3, scaled=False)
    keep = run_lora(L, wide, ldx, k, ids, adapters, [s], is_bf16)
    quiet(L)
    s.check(wide[:, :k], ids)
    del keep


@pytest.mark.parametrize("is_bf16", [False, True])
@pytest.mark.parametrize("m", [1, 20, 200])
@pytest.mark.parametrize("in_place", [False, True])
def test_lora_swiglu(L, is_bf16, m, in_place):
    rng = np.random.default_rng(m + 1)
    k, n, rank, adapters = 256, 352, 16, 4
    x = rng.standard_normal((m, k), dtype=F)
    ids = ids_of(rng, m, adapters, "runs")
    segs = [Adapters(rng, m, k, n, rank, adapters, is_bf16, True, in_place=in_place),
            Adapters(rng, m, k, 64, 8, adapters, is_bf16, False, in_place=in_place)]
    keep = run_lora(L, x, k, k, ids, adapters, segs, is_bf16)
    quiet(L)
    for s in segs:
        s.check(x, ids)
    del keep


@pytest.mark.parametrize("is_bf16", [False, True])
@pytest.mark.parametrize("m", [4, 100])
def test_lora_unaligned(L, is_bf16, m):
    rng = np.random.default_rng(77)
    k, adapters = 128, 3
    x = rng.standard_normal((m, k), dtype=F)
    ids = ids_of(rng, m, adapters, "each")
    s = Adapters(rng, m, k, 96, 16, adapters, is_bf16, False, offset=1)
    keep = run_lora(L, shifted(x), k, k, ids, adapters, [s], is_bf16)
    quiet(L)
    s.check(x, ids)
    del keep


@pytest.mark.parametrize("m", [6, 90])
def test_lora_refuses_unknown_adapters(L, m):
    """An id outside the table is never followed: its row is left, the others are done, the wait reports it."""
    rng = np.random.default_rng(5)
    k, adapters = 64, 2
    x = rng.standard_normal((m, k), dtype=F)
    for wrong in (2, -2, 2 ** 31 - 1, -2 ** 31):
        ids = np.array([0, 1, -1] * (m // 3))
        ids[3] = wrong
        s = Adapters(rng, m, k, 48, 8, adapters, True, False)
        keep = run_lora(L, x, k, k, ids, adapters, [s], True)
        fails(L, "adapter id outside the table")
        got = hu.host(s.c)
        assert (got[3] == 9.0).all()
        ids[3] = -1
        want, bound = ru.adapters(x, ids, s.base[0], *s.pairs[0], s.scale)
        rest = np.arange(m) != 3
        within(got[rest], want[rest], bound[rest])
        del keep


def test_lora_rows_do_not_mix(L):
    """A row of infinities (or another adapter's) does not reach its neighbours."""
    rng = np.random.default_rng(6)
    for m in (9, 80):
        k, adapters = 96, 2
        x = rng.standard_normal((m, k), dtype=F)
        ids = np.zeros(m, int)
        s = Adapters(rng, m, k, 32, 16, adapters, True, False)
        bad = x.copy()
        bad[4] = np.inf
        keep = run_lora(L, bad, k, k, ids, adapters, [s], True)
        quiet(L)
        got = hu.host(s.c)
        want, bound = ru.adapters(x, ids, s.base[0], *s.pairs[0], s.scale)
        rest = np.arange(m) != 4
        within(got[rest], want[rest], bound[rest])
        del keep


def test_lora_from_host_memory(L):
    rng = np.random.default_rng(8)
    m, k, n, rank, adapters = 3, 40, 24, 4, 2
    x, base = rng.standard_normal((m, k), dtype=F), rng.standard_normal((m, n), dtype=F)
    a, b = rng.standard_normal((adapters, rank, k), dtype=F), rng.standard_normal((adapters, n, rank), dtype=F)
    base3, a3, b3 = base[::-1].copy(), a[::-1].copy(), b[::-1].copy()
    scale, ids = np.array([1.5, 0.5], F), np.array([1, -1, 0], np.int32)
    outs, segs = [np.zeros((m, n), F) for _ in range(3)], []
    for c in outs:
        segs.append(ru.lora_segment(False, c, n, base, a, b, scale, n, rank, base3, a3, b3))
    L.llhip_lora_f32(lh.ptr(x), k, m, k, lh.ptr(ids), adapters, ru.array(segs), 3)
    assert not lh.last_error(), lh.last_error()
    want, bound = ru.swiglu(*ru.adapters(x, ids, base, a, b, scale), *ru.adapters(x, ids, base3, a3, b3, scale))
    for c in outs:
        within(c, want, bound + 2 * ru.U * np.abs(want))


# ---- verification -----------------------------------------------------------------------------------------------------


def verify_inputs(rng, rows_of, vocab, temperature, model, masked=0.0, first=0, ld=None, spread=2.0):
    start = np.concatenate(([first], first + np.cumsum(rows_of))).astype(np.int32)
    rows = int(start[-1])
    logits = (spread * rng.standard_normal((rows, ld or vocab))).astype(F)
    if masked:
        logits[rng.random(logits.shape) < masked] = -np.inf
        logits[:, vocab // 2] = 0.5
    draft = (logits + 0.5 * rng.standard_normal(logits.shape)).astype(F)
    tokens = np.zeros(rows, np.int32)
    for i in range(rows - 1):
        p = ru.softmax(draft[i, :vocab].astype(np.float64) / max(temperature, 0.2))
        tokens[i + 1] = rng.choice(vocab, p=p) if temperature else int(logits[i, :vocab].argmax())
        if temperature == 0.0 and rng.random() < 0.3:
            tokens[i + 1] = rng.integers(vocab)
    return start, logits, draft if model else None, tokens, rng.random((rows, 2)).astype(F)


def run_verify(L, start, logits, draft, tokens, uniform, vocab, temperature, keep_value=-9):
    count = len(start) - 1
    accepted, following = (hu.dev(np.full(count, keep_value, np.int32)) for _ in range(2))
    dev = [None if a is None else hu.dev(a) for a in (logits, draft, tokens, uniform, start)]
    L.llhip_verify_drafts(lh.ptr(accepted), lh.ptr(following), lh.ptr(dev[0]), logits.shape[1], lh.ptr(dev[1]),
                          0 if draft is None else draft.shape[1], lh.ptr(dev[2]), lh.ptr(dev[3]), lh.ptr(dev[4]), count,
                          len(logits), vocab, temperature)
    L.llhip_synchronize()
    return list(zip(hu.host(accepted).tolist(), hu.host(following).tolist()))


@pytest.mark.parametrize("temperature", [0.0, 0.3, 1.0, 1.7])
@pytest.mark.parametrize("model", [False, True])
@pytest.mark.parametrize("vocab,ld", [(1, None), (2, 3), (31, None), (1000, 1001), (5003, None), (32000, 32768)])
def test_verify(L, temperature, model, vocab, ld):
    """Requests of no row, one row (a plain draw) and drafts up to eight; rows before the first request."""
    rng = np.random.default_rng(vocab)
    inputs = verify_inputs(rng, [3, 1, 0, 9, 2, 1, 5], vocab, temperature, model, first=2, ld=ld)
    got = run_verify(L, *inputs, vocab, temperature)
    assert not lh.last_error(), lh.last_error()
    start, logits, draft, tokens, uniform = inputs
    want = ru.verify(start, logits[:, :vocab], None if draft is None else draft[:, :vocab], tokens, uniform, temperature)
    assert got == [(-9, -9) if w is None else w for w in want]


def test_verify_full_vocabulary(L):
    """128256 tokens, many borders: three hundred draws and the drafts before them."""
    rng = np.random.default_rng(1)
    for model in (True, False):
        inputs = verify_inputs(rng, [1] * 60 + [2, 4, 3, 5, 2], 128256, 0.9, model, spread=3.0)
        got = run_verify(L, *inputs, 128256, 0.9)
        assert not lh.last_error(), lh.last_error()
        assert got == ru.verify(*inputs, 0.9)


@pytest.mark.parametrize("temperature", [0.0, 0.8])
def test_verify_masked_and_extreme_rows(L, temperature):
    """Tokens masked out by -infinity or the type's lowest value, single tokens left, logits of 1e30, equal logits (the
    lowest token wins a tie), a draft that its own model or the target gives no weight, uniforms of 0 and just below 1."""
    rng = np.random.default_rng(2)
    vocab = 700
    start, logits, draft, tokens, uniform = verify_inputs(rng, [2] * 12, vocab, temperature, True, masked=0.6)
    low = np.finfo(F).min
    logits[0] = -np.inf
    logits[0, 699] = -3.0
    tokens[1] = 699
    logits[2] = low
    logits[2, 5] = low / 2
    logits[4] = 1e30 * np.sign(rng.standard_normal(vocab))
    logits[6] = 0.25
    logits[6, :9] = 0.2
    tokens[7] = 9
    logits[8, tokens[9]] = -np.inf
    draft[10, tokens[11]] = -np.inf
    logits[10, tokens[11]] = 1.0
    uniform[12:14] = 0.0
    uniform[14:18] = np.float32(1.0) - np.float32(2.0 ** -24)
    draft[18] = logits[18]
    draft[20] = -np.inf
    draft[20, tokens[21]] = 0.0
    got = run_verify(L, start, logits, draft, tokens, uniform, vocab, temperature)
    assert not lh.last_error(), lh.last_error()
    assert got == ru.verify(start, logits, draft, tokens, uniform, temperature)
    one_hot = run_verify(L, start, logits, None, tokens, uniform, vocab, temperature)
    assert one_hot == ru.verify(start, logits, None, tokens, uniform, temperature)


@pytest.mark.parametrize("temperature", [0.0, 1.0])
def test_verify_refuses_rows_that_decide_nothing(L, temperature):
    """NaN, +infinity or nothing left in a row that decides: -1 and a failure at the wait; behind the row that stopped
    the request they do not matter. A draft or rows outside: likewise."""
    rng = np.random.default_rng(3)
    vocab = 300

    def inputs():
        start, logits, draft, tokens, uniform = verify_inputs(rng, [2, 2, 1], vocab, temperature, True)
        tokens[1] = int(logits[0].argmax())
        uniform[0, 0] = 0.0  # accepted
        return start, logits, draft, tokens, uniform

    for value in (np.nan, np.inf):
        for row in (0, 1):
            start, logits, draft, tokens, uniform = inputs()
            logits[row, 17] = value
            got = run_verify(L, start, logits, draft, tokens, uniform, vocab, temperature)
            fails(L, "leave no token")
            logits[row] = 0.0
            want = ru.verify(start, logits, draft, tokens, uniform, temperature)
            assert got == [(-1, -1)] + want[1:]
    start, logits, draft, tokens, uniform = inputs()
    logits[0] = -np.inf
    assert run_verify(L, start, logits, draft, tokens, uniform, vocab, temperature)[0] == (-1, -1)
    fails(L, "leave no token")
    start, logits, draft, tokens, uniform = inputs()
    logits[0] = -np.inf
    logits[0, 3], tokens[1] = 0.0, 4  # refused for certain: row 1 is not reached
    logits[1] = np.nan
    draft[0] = 0.0
    got = run_verify(L, start, logits, draft, tokens, uniform, vocab, temperature)
    assert got[0] == (0, 3) and not lh.last_error()
    for wrong in (-1, vocab, 2 ** 31 - 1):
        start, logits, draft, tokens, uniform = inputs()
        tokens[1] = wrong
        got = run_verify(L, start, logits, draft, tokens, uniform, vocab, temperature)
        fails(L, "outside the vocabulary")
        tokens[1] = 0
        assert got == [(-1, -1)] + ru.verify(start, logits, draft, tokens, uniform, temperature)[1:]
    start, logits, draft, tokens, uniform = inputs()
    got = run_verify(L, np.array([0, 2, 6], np.int32), logits, draft, tokens, uniform, vocab, temperature)
    fails(L, "outside the batch's buffers")
    assert got[1] == (-9, -9) and got[0] == ru.verify(start[:2], logits, draft, tokens, uniform, temperature)[0]


def at_a_mappings_end(a):
    """A host copy of `a` whose last byte is its mapping's: the page behind cannot be read."""
    page = mmap.PAGESIZE
    room = (a.nbytes + page - 1) // page * page
    m = mmap.mmap(-1, room + page)
    libc = ctypes.CDLL(None, use_errno=True)
    libc.mprotect.argtypes = [ctypes.c_void_p, ctypes.c_size_t, ctypes.c_int]
    view = np.frombuffer(m, a.dtype, a.size, room - a.nbytes).reshape(a.shape)
    view[...] = a
    assert libc.mprotect(view.ctypes.data + a.nbytes, page, 0) == 0, ctypes.get_errno()
    return view


@pytest.mark.parametrize("ld", [5000, 5008])
@pytest.mark.parametrize("rows_of,spare", [([1], 0), ([4], 0), ([3, 1, 2], 0), ([3, 2], 2)])
def test_verify_reads_no_draft_row_behind_the_last(L, rows_of, spare, ld):
    """draft_logits of rows - 1 rows: on the device an allocation that ends with them, on the host a mapping."""
    vocab, rng = 5000, np.random.default_rng(ld + sum(rows_of))
    start, logits, draft, tokens, uniform = verify_inputs(rng, rows_of + [spare], vocab, 0.9, True, ld=ld)
    start, rows, count = start[:-1].copy(), len(logits), len(rows_of)
    want = ru.verify(start, logits[:, :vocab], draft[:, :vocab], tokens, uniform, 0.9)
    exact = at_a_mappings_end(draft[:-1].reshape(-1)[:max((rows - 2) * ld + vocab, 0)])
    device = L.llhip_malloc(exact.nbytes) if exact.nbytes else None
    try:
        if exact.nbytes:
            L.llhip_memcpy_h2d(device, lh.ptr(exact), exact.nbytes)
        for place in ("host", "device"):
            accepted, following = np.full(count, -9, np.int32), np.full(count, -9, np.int32)
            L.llhip_verify_drafts(lh.ptr(accepted), lh.ptr(following), lh.ptr(logits), ld,
                                  exact.ctypes.data if place == "host" else device, ld, lh.ptr(tokens), lh.ptr(uniform),
                                  lh.ptr(start), count, rows, vocab, 0.9)
            assert not lh.last_error(), lh.last_error()
            assert list(zip(accepted.tolist(), following.tolist())) == want
    finally:
        if device:
            L.llhip_free(device)


def test_verify_emits_the_targets_distribution(L):
    """20000 requests' worth of draws over six tokens: the emitted first tokens' frequencies are the target's within five
    standard deviations, whatever the draft's distribution."""
    rng = np.random.default_rng(9)
    vocab, count, t = 6, 1000, 1.0
    target, other = np.array([0.1, 1.0, -0.5, 0.7, -2.0, 0.3], F), np.array([1.0, -1.0, 0.5, 0.0, 0.5, -0.7], F)
    p, q = ru.softmax(target.astype(np.float64)), ru.softmax(other.astype(np.float64))
    seen = np.zeros(vocab)
    start = np.arange(0, 2 * count + 1, 2).astype(np.int32)
    logits, draft = np.tile(target, (2 * count, 1)), np.tile(other, (2 * count, 1))
    for _ in range(20):
        tokens = np.zeros(2 * count, np.int32)
        tokens[1::2] = rng.choice(vocab, count, p=q)
        got = run_verify(L, start, logits, draft, tokens, rng.random((2 * count, 2)).astype(F), vocab, t)
        first = [tokens[2 * i + 1] if a else n for i, (a, n) in enumerate(got)]
        seen += np.bincount(first, minlength=vocab)
    n = 20 * count
    assert (np.abs(seen - n * p) < 5 * np.sqrt(n * p * (1 - p))).all(), (seen / n, p)


# ---- captured calls ---------------------------------------------------------------------------------------------------


def test_captured_calls_follow_their_arrays(L):
    """All four captured in one graph and replayed while the arrays, lengths and logits change, with eager work between the
    replays; every replay equals the eager calls."""
    T = hu.torch()
    L.kernels_kv_layout_select(b"head")
    rng = np.random.default_rng(21)
    heads, kv, hd, vocab, k = 8, 2, 64, 4000, 512
    b = ru.Batch(hu.dev, [1, 3, 1], [5, 0, 60], prefix=100, prefix_seq_len=100, seq_len=80, slot=[2, 0, 1], slots=3)
    q, kn, vn = (rng.standard_normal((b.rows, n * hd), dtype=F) for n in (heads, kv, kv))
    table = rng.standard_normal((180, 2 * hd), dtype=F)
    pk, pv = (rng.standard_normal((kv, 100, hd), dtype=F) for _ in range(2))
    kc, vc = (rng.standard_normal((3, kv, 80, hd), dtype=F) for _ in range(2))
    dev = {n: hu.dev(a) for n, a in (("q", q), ("k", kn), ("v", vn), ("t", table), ("pk", pk), ("pv", pv))}
    cache = [hu.dev(kc), hu.dev(vc)]
    rot, out = hu.dev(np.zeros_like(q)), hu.dev(np.zeros_like(q))
    lora = Adapters(rng, b.rows, k, 96, 16, 4, True, False)
    x, ids = hu.dev(rng.standard_normal((b.rows, k), dtype=F)), hu.dev(np.array([0, 1, 1, 3, -1], np.int32))
    seg = ru.array([lora.struct])
    start, logits, draft, tokens, uniform = verify_inputs(rng, [1, 3, 1], vocab, 0.7, True)
    vdev = [hu.dev(a) for a in (logits, draft, tokens, uniform)]
    acc, nxt = hu.dev(np.zeros(3, np.int32)), hu.dev(np.zeros(3, np.int32))

    def calls():
        L.llhip_rope_kv_store_requests(lh.ptr(rot), lh.ptr(dev["q"]), heads * hd, lh.ptr(dev["k"]), lh.ptr(dev["v"]),
                                       kv * hd, lh.ptr(dev["t"]), b.struct, heads, kv, hd, lh.ptr(cache[0]),
                                       lh.ptr(cache[1]))
        L.llhip_attention_requests(lh.ptr(out), lh.ptr(rot), lh.ptr(dev["pk"]), lh.ptr(dev["pv"]), lh.ptr(cache[0]),
                                   lh.ptr(cache[1]), b.struct, heads, kv, hd)
        L.llhip_lora_bf16(lh.ptr(x), k, b.rows, k, lh.ptr(ids), 4, seg, 1)
        L.llhip_verify_drafts(lh.ptr(acc), lh.ptr(nxt), lh.ptr(vdev[0]), vocab, lh.ptr(vdev[1]), vocab, lh.ptr(vdev[2]),
                              lh.ptr(vdev[3]), lh.ptr(b.keep[0]), 3, b.rows, vocab, 0.7)

    def results():
        return [hu.host(a).copy() for a in (rot, out, lora.c, acc, nxt, cache[0], cache[1])]

    calls()  # workspaces grow outside of the capture
    quiet(L)
    assert L.llhip_graph_begin() == 0, lh.last_error()
    calls()
    graph = L.llhip_graph_end()
    assert graph, lh.last_error()
    for step, length in enumerate(([6, 3, 61], [70, 10, 0], [1, 77, 79])):
        b.keep[1].copy_(T.from_numpy(np.asarray(length, np.int32)))
        ids.copy_(T.from_numpy(np.roll(np.array([0, 1, 1, 3, -1], np.int32), step)))
        vdev[3].copy_(T.from_numpy(rng.random((b.rows, 2)).astype(F)))
        T.cuda.synchronize()
        calls()
        quiet(L)
        want = results()
        for a in (rot, out, lora.c, acc, nxt):
            a.zero_()
        T.cuda.synchronize()
        assert L.llhip_graph_launch(graph) == 0
        quiet(L)
        for g, w in zip(results(), want):
            assert np.array_equal(g, w)
    L.llhip_graph_destroy(graph)


def test_two_graphs_share_the_workspace(L):
    """Two graphs of the same operators over other operands, replayed in turn with a larger eager call between, which takes
    another workspace; a call that would need a larger one while it is captured is refused."""
    T = hu.torch()
    L.kernels_kv_layout_select(b"head")
    rng = np.random.default_rng(5)
    heads, kv, hd = 8, 2, 128

    def make(rows_of, length, prefix):
        b = ru.Batch(hu.dev, rows_of, length, prefix=prefix, prefix_seq_len=prefix, seq_len=200)
        a = [rng.standard_normal(n, dtype=F) for n in ((b.rows, heads * hd), (kv, prefix, hd), (kv, prefix, hd),
                                                       (b.slots, kv, 200, hd), (b.slots, kv, 200, hd))]
        want, bound = ru.attention(b, *a, heads, kv, hd, "head")
        return b, [hu.dev(x) for x in a], hu.dev(np.zeros_like(a[0])), want, bound

    def call(m):
        L.llhip_attention_requests(lh.ptr(m[2]), *[lh.ptr(x) for x in m[1]], m[0].struct, heads, kv, hd)

    one, two = make([1] * 9, rng.integers(0, 199, 9), 700), make([30, 1, 5], [100, 5, 190], 90)
    graphs = []
    for m in (one, two):
        call(m)
        quiet(L)
        assert L.llhip_graph_begin() == 0
        call(m)
        graphs.append(L.llhip_graph_end())
        assert graphs[-1], lh.last_error()
    m, k, n, rank = 60000, 64, 16, 256
    x = hu.dev(rng.standard_normal((m, k), dtype=F))
    big = Adapters(rng, 1, k, n, rank, 1, True, False)
    c = hu.dev(np.zeros((m, n), F))
    seg = ru.array([ru.lora_segment(True, c, n, c, big.keep[0][0][0], big.keep[0][0][1], None, n, rank)] * 1)
    ids = hu.dev(np.zeros(m, np.int32))
    assert L.llhip_graph_begin() == 0
    L.llhip_lora_bf16(lh.ptr(x), k, m, k, lh.ptr(ids), 1, seg, 1)
    message = lh.last_error()
    refused = "during graph capture" in message
    L.llhip_clear_error()
    empty = L.llhip_graph_end()
    if empty:
        L.llhip_graph_destroy(empty)
    L.llhip_clear_error()
    assert refused, message
    for turn in range(3):
        if turn == 1:
            L.llhip_lora_bf16(lh.ptr(x), k, m, k, lh.ptr(ids), 1, seg, 1)
        for a in (one, two):
            a[2].zero_()
        T.cuda.synchronize()
        for g in graphs + graphs[::-1]:
            assert L.llhip_graph_launch(g) == 0
        quiet(L)
        for a in (one, two):
            within(hu.host(a[2]), a[3], a[4], turn)
    for g in graphs:
        L.llhip_graph_destroy(g)


def test_calls_from_two_threads(L):
    """Attention and verification from two threads at once, whose kernels share one workspace."""
    import threading
    L.kernels_kv_layout_select(b"head")
    rng = np.random.default_rng(6)
    heads, kv, hd = 8, 2, 64
    b = ru.Batch(hu.dev, [1] * 20, rng.integers(0, 100, 20), prefix=300, prefix_seq_len=300, seq_len=128)
    a = [rng.standard_normal(n, dtype=F) for n in ((b.rows, heads * hd), (kv, 300, hd), (kv, 300, hd),
                                                   (b.slots, kv, 128, hd), (b.slots, kv, 128, hd))]
    want, bound = ru.attention(b, *a, heads, kv, hd, "head")
    dev, out = [hu.dev(x) for x in a], hu.dev(np.zeros_like(a[0]))
    start, logits, draft, tokens, uniform = verify_inputs(rng, [3] * 20, 4000, 0.7, True)
    vdev = [hu.dev(x) for x in (logits, draft, tokens, uniform, start)]
    acc, nxt = hu.dev(np.zeros(20, np.int32)), hu.dev(np.zeros(20, np.int32))

    def attend():
        for _ in range(200):
            L.llhip_attention_requests(lh.ptr(out), *[lh.ptr(x) for x in dev], b.struct, heads, kv, hd)

    def judge():
        for _ in range(200):
            L.llhip_verify_drafts(lh.ptr(acc), lh.ptr(nxt), lh.ptr(vdev[0]), 4000, lh.ptr(vdev[1]), 4000, lh.ptr(vdev[2]),
                                  lh.ptr(vdev[3]), lh.ptr(vdev[4]), 20, 60, 4000, 0.7)

    attend(), judge()
    quiet(L)
    team = [threading.Thread(target=f) for f in (attend, judge)]
    for t in team:
        t.start()
    for t in team:
        t.join()
    quiet(L)
    within(hu.host(out), want, bound)
    assert list(zip(hu.host(acc).tolist(), hu.host(nxt).tolist())) == ru.verify(start, logits, draft, tokens, uniform, 0.7)


# ---- the largest numbers ----------------------------------------------------------------------------------------------


@pytest.mark.parametrize("count", [64, 65, 128, 129, 300, 1024])
def test_attention_many_requests(L, count):
    """As many requests as a call takes, some without rows, behind a prefix and without one; vectors of one row, drafts."""
    rng = np.random.default_rng(count)
    rows_of = rng.choice([0, 1, 1, 1, 4, 9], count)
    for prefix in (0, 70):
        b = ru.Batch(hu.dev, rows_of, rng.integers(0, 40, count), slot=rng.permutation(count), prefix=prefix, seq_len=49,
                     first=1, spare=2)
        attention_case(L, count, 4, 2, 64, "head", b)


def test_attention_without_rows(L):
    b = ru.Batch(hu.dev, [0, 0, 0], [0, 5, 9], prefix=9, seq_len=16, first=2, spare=5)
    attention_case(L, 1, 4, 2, 64, "head", b)


@pytest.mark.parametrize("count", [257, 1024])
def test_rope_many_requests(L, count):
    L.kernels_kv_layout_select(b"rows")
    rng = np.random.default_rng(count)
    heads, kv, hd = 3, 1, 8
    rows_of = rng.choice([0, 1, 1, 3], count)
    b = ru.Batch(hu.dev, rows_of, rng.integers(0, 20, count), slot=rng.permutation(count), prefix=3, seq_len=24)
    q, k, v = (rng.standard_normal((b.rows, n * hd), dtype=F) for n in (heads, kv, kv))
    angle = rng.standard_normal((27, hd // 2))
    cos, sin = np.cos(angle).astype(F), np.sin(angle).astype(F)
    table = np.concatenate((np.repeat(cos, 2, 1), np.stack((-sin, sin), 2).reshape(27, -1)), 1)
    out, kc, vc = hu.dev(np.zeros_like(q)), hu.dev(np.zeros((count, 24, hd), F)), hu.dev(np.zeros((count, 24, hd), F))
    keep = [hu.dev(x) for x in (q, k, v, table)]
    L.llhip_rope_kv_store_requests(lh.ptr(out), lh.ptr(keep[0]), heads * hd, lh.ptr(keep[1]), lh.ptr(keep[2]), hd,
                                   lh.ptr(keep[3]), b.struct, heads, kv, hd, lh.ptr(kc), lh.ptr(vc))
    quiet(L)
    at = np.zeros(b.rows, int)
    want_k, want_v = np.zeros((count, 24, hd), F), np.zeros((count, 24, hd), F)

    def turn(x, at):
        x = x.reshape(len(x), -1, hd // 2, 2)
        c, s = cos[at][:, None], sin[at][:, None]
        return np.stack((x[..., 0] * c - x[..., 1] * s, x[..., 0] * s + x[..., 1] * c), -1).reshape(len(x), -1)

    for _, rows, length, _ in b.requests():
        at[rows] = 3 + length + np.arange(rows.stop - rows.start)
    turned = turn(k, at)
    for _, rows, length, slot in b.requests():
        n = rows.stop - rows.start
        want_k[slot, length:length + n], want_v[slot, length:length + n] = turned[rows], v[rows]
    assert np.array_equal(hu.host(out), turn(q, at))
    assert np.array_equal(hu.host(kc), want_k) and np.array_equal(hu.host(vc), want_v)


def test_verify_1024_requests(L):
    rng = np.random.default_rng(4)
    inputs = verify_inputs(rng, rng.integers(0, 4, 1024), 50, 0.9, True)
    got = run_verify(L, *inputs, 50, 0.9)
    assert not lh.last_error(), lh.last_error()
    assert got == [(-9, -9) if w is None else w for w in ru.verify(*inputs, 0.9)]


@pytest.mark.parametrize("m", [1, 40, 300])
def test_lora_many_adapters(L, m):
    """More adapters than the tiles' search takes, and as many."""
    for adapters in (4096, 4097):
        rng = np.random.default_rng(m)
        k, n, rank = 16, 24, 4
        x = rng.standard_normal((m, k), dtype=F)
        ids = rng.integers(-1, adapters, m)
        ids[-1] = adapters - 1
        s = Adapters(rng, m, k, n, rank, adapters, False, False)
        keep = run_lora(L, x, k, k, ids, adapters, [s], False)
        quiet(L)
        s.check(x, ids)
        del keep


def test_caches_past_32_bits(L):
    """Slots that begin past 2^32 values and bytes, stored into and read."""
    T = hu.torch()
    L.kernels_kv_layout_select(b"head")
    rng = np.random.default_rng(7)
    heads, kv, hd, seq_len, slots = 4, 1, 64, 1 << 20, 66
    key, value = (T.empty(slots, kv, seq_len, hd, device="cuda") for _ in range(2))
    lengths, slot, rows_of = [300, seq_len - 3, 7], [65, 64, 0], [2, 3, 1]
    b = ru.Batch(hu.dev, rows_of, lengths, slot=slot, slots=slots, prefix=0, seq_len=seq_len)
    q, k, v = (rng.standard_normal((b.rows, n * hd), dtype=F) for n in (heads, kv, kv))
    table = T.zeros(seq_len, 2 * hd, device="cuda")
    table[:, :hd] = 1.0  # no turn
    old = {s: rng.standard_normal((2, 300, hd), dtype=F) for s in (65, 0)}
    for s, x in old.items():
        key[s, 0, :300].copy_(T.from_numpy(x[0]))
        value[s, 0, :300].copy_(T.from_numpy(x[1]))
    key[64].zero_()
    value[64].zero_()
    # the last own rows of slot 64 take all of the weight
    q[2:5] = 1.0
    k[2:5] = 60.0 / 8.0
    T.cuda.synchronize()
    rot, out = hu.dev(np.zeros_like(q)), hu.dev(np.zeros_like(q))
    keep = [hu.dev(x) for x in (q, k, v)]
    L.llhip_rope_kv_store_requests(lh.ptr(rot), lh.ptr(keep[0]), heads * hd, lh.ptr(keep[1]), lh.ptr(keep[2]),
                                   kv * hd, lh.ptr(table), b.struct, heads, kv, hd, lh.ptr(key), lh.ptr(value))
    L.llhip_attention_requests(lh.ptr(out), lh.ptr(rot), None, None, lh.ptr(key), lh.ptr(value), b.struct, heads, kv, hd)
    quiet(L)
    got = hu.host(out)
    small = ru.Batch(hu.dev, [2, 1], [300, 7], seq_len=302)
    cache = np.zeros((2, 2, 1, 302, hd), F)
    for i, (s, rows) in enumerate(((65, slice(0, 2)), (0, slice(5, 6)))):
        cache[:, i, 0, :300] = old[s]
        at = lengths[slot.index(s)]
        cache[0, i, 0, at:at + rows.stop - rows.start], cache[1, i, 0, at:at + rows.stop - rows.start] = k[rows], v[rows]
    none = np.zeros((1, 0, hd), F)
    want, bound = ru.attention(small, q[[0, 1, 5]], none, none, cache[0], cache[1], heads, kv, hd, "head")
    within(got[[0, 1, 5]], want, bound)
    # equal scores of 60 over the positions stored: 2^20 others weigh exp(-60) each, below 1e-19 together; three sums' and a
    # division's roundings, and the weights' of scores near 60 (72 U of the score), stay below 5000 U
    for j in range(3):
        mean = v[2:3 + j].astype(np.float64).mean(0)
        assert np.abs(got[2 + j].reshape(heads, hd) - mean).max() < 5000 * ru.U * np.abs(v[2:5]).max()
    assert T.equal(key[65, 0, 300:302].cpu(), T.from_numpy(k[:2]))
    assert T.equal(value[64, 0, seq_len - 3:].cpu(), T.from_numpy(v[2:5]))


def test_attention_walk_past_2_gib(L):
    """Positions whose rows lie more than 2^31 bytes into a slot: the form for any shape."""
    T = hu.torch()
    L.kernels_kv_layout_select(b"head")
    rng = np.random.default_rng(8)
    hd, seq_len = 256, (1 << 21) + 64
    key, value = (T.zeros(1, 1, seq_len, hd, device="cuda") for _ in range(2))
    b = ru.Batch(hu.dev, [2], [seq_len - 2], seq_len=seq_len)
    q = np.ones((2, hd), F)
    v = rng.standard_normal((2, hd), dtype=F)
    key[0, 0, -2:] = 60.0 / 16.0
    value[0, 0, -2:].copy_(T.from_numpy(v))
    T.cuda.synchronize()
    out, qd = hu.dev(np.zeros((2, hd), F)), hu.dev(q)
    L.llhip_attention_requests(lh.ptr(out), lh.ptr(qd), None, None, lh.ptr(key), lh.ptr(value), b.struct, 1, 1, hd)
    quiet(L)
    got = hu.host(out)
    for j in range(2):  # as above
        assert np.abs(got[j] - v[:1 + j].astype(np.float64).mean(0)).max() < 5000 * ru.U * np.abs(v).max()


# ---- the engine's step over drafts ------------------------------------------------------------------------------------


ENGINE = dict(dim=128, hidden_dim=256, n_layers=2, n_heads=4, n_kv_heads=2, vocab_size=1500, seq_len=96, rope_theta=10000.0)


def engine_model(path, kind):
    gs = 64
    norms, t = ck.synthetic(ENGINE, gs, 17)
    if kind.startswith("q8"):
        ck.write_q8_v3(path, ENGINE, gs, norms, t)
    else:
        f32 = {n: q.astype(F) * np.repeat(s.reshape(-1), gs).reshape(q.shape).astype(F) for n, (q, s) in t.items()}
        ck.write_f32_v3(path, ENGINE, norms, f32)


@pytest.mark.parametrize("kind", ["q8", "q8_fp32_activations", "f32", "bf16", "q8_no_gemm"])
def test_engine_verify(L, tmp_path, monkeypatch, kind):
    """llhip_engine_verify's decisions are the plain form's on the logits that engine_forward_batch gives for the same rows
    at the same place, drawn and greedy, with a draft model and without, for one row and many; a model goes on from the
    accepted drafts; and its refusals, which leave the model usable."""
    if kind == "q8_fp32_activations":
        monkeypatch.setenv("LLAMA_Q8_ACTIVATIONS", "fp32")
    if kind == "bf16":
        monkeypatch.setenv("LLAMA_PRECISION", "bf16")
    if kind == "q8_no_gemm":
        monkeypatch.setenv("LLAMA_PREFILL_GEMM", "off")
    if kind in ("q8_fp32_activations", "q8_no_gemm"):  # rows run one at a time; a batch is one row unless asked for
        monkeypatch.setenv("LLAMA_PREFILL_BATCH", "24")
    L.kernels_kv_layout_select(b"head")
    path = os.path.join(tmp_path, "tiny.bin")
    engine_model(path, kind)
    vocab = ENGINE["vocab_size"]
    rng = np.random.default_rng(8)
    model, following = lh.Model(), ctypes.c_int(-7)
    at = ctypes.byref(model)

    def verify(tokens, pos, draft, uniform, temperature):
        return L.llhip_engine_verify(at, lh.ptr(tokens), len(tokens), pos, lh.ptr(draft), 0 if draft is None else vocab,
                                     lh.ptr(uniform), temperature, ctypes.byref(following))

    try:
        L.engine_load(at, path.encode())
        assert model.implementation, lh.last_error()
        prompt = rng.integers(0, vocab, 20).astype(np.int32)
        assert L.engine_forward_batch(at, lh.ptr(prompt), 20, 0, lh.LOGITS_LAST), lh.last_error()
        known, pos, accepted_any = int(prompt[0]), 20, 0
        for n, temperature, drawn in ((1, 0.0, False), (5, 0.0, False), (4, 0.8, True), (6, 1.3, False), (1, 0.7, False),
                                      (8, 0.5, True)):
            tokens = rng.integers(0, vocab, n).astype(np.int32)
            tokens[0] = known
            for i in range(1, n):  # the model's own choice, but for the last
                p = L.engine_forward_batch(at, lh.ptr(tokens[:i]), i, pos, lh.LOGITS_ALL)
                row = np.ctypeslib.as_array(ctypes.cast(p, ctypes.POINTER(ctypes.c_float)), (i, vocab))[i - 1]
                if i < n - 1:
                    tokens[i] = int(row.argmax())
            p = L.engine_forward_batch(at, lh.ptr(tokens), n, pos, lh.LOGITS_ALL)
            logits = np.ctypeslib.as_array(ctypes.cast(p, ctypes.POINTER(ctypes.c_float)), (n, vocab)).copy()
            draft = (logits + 0.3 * rng.standard_normal(logits.shape)).astype(F) if drawn else None
            uniform = rng.random((n, 2)).astype(F) if temperature else None
            want = ru.verify([0, n], logits, draft, tokens, uniform, temperature)[0]
            got = verify(tokens, pos, draft, uniform, temperature)
            assert not lh.last_error(), lh.last_error()
            assert (got, following.value) == want, (n, temperature)
            if drawn:  # from device memory
                keep = hu.dev(draft), hu.dev(uniform)
                assert verify(tokens, pos, keep[0], keep[1], temperature) == want[0] and following.value == want[1]
            pos, known, accepted_any = pos + got + 1, following.value, accepted_any + got
        assert accepted_any >= 3  # greedy accepts the model's own choices: 3 of its 4 at least
        u = np.zeros((2, 2), F)
        following.value = -7
        two = np.array([1, 2], np.int32)
        for call, words in ((lambda: verify(two, 95, None, u, 0.5), "batch input out of range"),
                            (lambda: verify(np.array([1, vocab], np.int32), 20, None, u, 0.5), "out of range: token="),
                            (lambda: verify(two, 20, None, None, 0.5), "null buffer"),
                            (lambda: verify(two, 20, None, u, -1.0), "not negative"),
                            (lambda: L.llhip_engine_verify(at, lh.ptr(two), 2, 20, lh.ptr(u), vocab - 1, lh.ptr(u), 0.5,
                                                           ctypes.byref(following)), "at a stride of"),
                            (lambda: L.llhip_engine_verify(at, lh.ptr(two), 0, 20, None, 0, None, 0.0,
                                                           ctypes.byref(following)), "batch input out of range"),
                            (lambda: L.llhip_engine_verify(at, None, 2, 20, None, 0, None, 0.0,
                                                           ctypes.byref(following)), "batch input out of range"),
                            (lambda: L.llhip_engine_verify(at, lh.ptr(two), 2, 20, None, 0, None, 0.0, None), "null buffer")):
            assert call() == -1 and following.value == -7
            assert words in lh.last_error(), lh.last_error()
        assert verify(two, 20, None, None, 0.0) >= 0 and not lh.last_error()
    finally:
        L.engine_free(at)


def test_engine_verify_reads_a_draft_row_for_each_draft(L, tmp_path):
    """count - 1 rows of draft_logits, at the end of a mapping and of a device allocation; none for one row."""
    L.kernels_kv_layout_select(b"head")
    path = os.path.join(tmp_path, "tiny.bin")
    engine_model(path, "q8")
    vocab, rng = ENGINE["vocab_size"], np.random.default_rng(12)
    model, following, device = lh.Model(), ctypes.c_int(-7), None
    at = ctypes.byref(model)
    try:
        L.engine_load(at, path.encode())
        for n in (5, 2, 1):
            tokens, uniform = rng.integers(0, vocab, n).astype(np.int32), rng.random((n, 2)).astype(F)
            p = L.engine_forward_batch(at, lh.ptr(tokens), n, 0, lh.LOGITS_ALL)
            logits = np.ctypeslib.as_array(ctypes.cast(p, ctypes.POINTER(ctypes.c_float)), (n, vocab)).copy()
            draft = (logits + rng.standard_normal(logits.shape)).astype(F)
            want = ru.verify([0, n], logits, draft, tokens, uniform, 0.9)[0]
            exact = at_a_mappings_end(draft[:-1])
            device = L.llhip_malloc(max(exact.nbytes, 4))
            if exact.nbytes:
                L.llhip_memcpy_h2d(device, lh.ptr(exact), exact.nbytes)
            for place in (exact.ctypes.data, device):
                got = L.llhip_engine_verify(at, lh.ptr(tokens), n, 0, place, vocab, lh.ptr(uniform), 0.9,
                                            ctypes.byref(following))
                assert not lh.last_error(), lh.last_error()
                assert (got, following.value) == want
            L.llhip_free(device)
            device = None
    finally:
        if device:
            L.llhip_free(device)
        L.engine_free(at)


def reconfigured(L, tmp_path, monkeypatch, kind, gemm):
    """A q8 or f32 model loaded for batches of 4, with its GEMM `gemm`, verified once, then configured for batches of 24 with
    the GEMM on: (the model, the tokens of 24 rows, uniforms for them, and the logits of a model loaded for 24)."""
    L.kernels_kv_layout_select(b"head")
    path = os.path.join(tmp_path, "tiny.bin")
    engine_model(path, kind)
    vocab, rng = ENGINE["vocab_size"], np.random.default_rng(31)
    tokens, uniform = rng.integers(0, vocab, 24).astype(np.int32), rng.random((24, 2)).astype(F)
    monkeypatch.setenv("LLAMA_PREFILL_BATCH", "24")
    fresh, model, following = lh.Model(), lh.Model(), ctypes.c_int(-7)
    L.engine_load(ctypes.byref(fresh), path.encode())
    p = L.engine_forward_batch(ctypes.byref(fresh), lh.ptr(tokens), 24, 0, lh.LOGITS_ALL)
    assert p, lh.last_error()
    logits = np.ctypeslib.as_array(ctypes.cast(p, ctypes.POINTER(ctypes.c_float)), (24, vocab)).copy()
    L.engine_free(ctypes.byref(fresh))
    monkeypatch.setenv("LLAMA_PREFILL_BATCH", "4")
    monkeypatch.setenv("LLAMA_PREFILL_GEMM", gemm)
    L.engine_load(ctypes.byref(model), path.encode())
    at = ctypes.byref(model)
    assert L.llhip_engine_verify(at, lh.ptr(tokens), 4, 0, None, 0, None, 0.0, ctypes.byref(following)) >= 0, lh.last_error()
    monkeypatch.setenv("LLAMA_PREFILL_BATCH", "24")
    monkeypatch.setenv("LLAMA_PREFILL_GEMM", "on")
    L.prefill_configure_engine(at, 24, kind == "q8")
    assert not lh.last_error() and L.engine_max_batch(at) == 24
    return model, tokens, uniform, logits


@pytest.mark.parametrize("kind", ["q8", "f32"])
def test_engine_verify_holds_the_logits_of_a_larger_batch(L, tmp_path, monkeypatch, kind):
    """Rows one at a time with room for 4 rows' logits, then the GEMM with 24: the logits' buffer grows by both paths."""
    model, tokens, uniform, logits = reconfigured(L, tmp_path, monkeypatch, kind, "off")
    at, vocab, following = ctypes.byref(model), ENGINE["vocab_size"], ctypes.c_int(-7)
    try:
        claimed = L.llhip_hbm_claimed()
        got = L.llhip_engine_verify(at, lh.ptr(tokens), 24, 0, None, 0, lh.ptr(uniform), 0.8, ctypes.byref(following))
        assert not lh.last_error(), lh.last_error()
        assert (got, following.value) == ru.verify([0, 24], logits, None, tokens, uniform, 0.8)[0]
        # the 24 rows of the GEMMs and 20 rows of logits more
        assert L.llhip_hbm_claimed() - claimed >= 4 * (20 * vocab + 24 * 3 * ENGINE["dim"])
        p = L.engine_forward_batch(at, lh.ptr(tokens), 24, 0, lh.LOGITS_ALL)
        assert (np.ctypeslib.as_array(ctypes.cast(p, ctypes.POINTER(ctypes.c_float)), (24, vocab)) == logits).all()
        monkeypatch.setenv("LLAMA_PREFILL_BATCH", "40")  # and by rows one at a time
        monkeypatch.setenv("LLAMA_PREFILL_GEMM", "off")
        L.prefill_configure_engine(at, 40, kind == "q8")
        forty = np.resize(tokens, 40)
        claimed = L.llhip_hbm_claimed()
        assert L.llhip_engine_verify(at, lh.ptr(forty), 40, 0, None, 0, None, 0.0, ctypes.byref(following)) >= 0
        assert not lh.last_error() and L.llhip_hbm_claimed() - claimed == 4 * 16 * vocab
    finally:
        L.engine_free(at)


@pytest.mark.parametrize("kind", ["q8", "f32", "bf16"])
def test_engine_verify_holds_the_rows_of_a_larger_batch(L, tmp_path, monkeypatch, kind):
    """The GEMM's rows allocated for batches of 4 grow for a batch of 24, and stay for one of 3."""
    if kind == "bf16":
        monkeypatch.setenv("LLAMA_PRECISION", "bf16")
    model, tokens, uniform, logits = reconfigured(L, tmp_path, monkeypatch, kind, "on")
    at, vocab, following = ctypes.byref(model), ENGINE["vocab_size"], ctypes.c_int(-7)
    try:
        claimed = L.llhip_hbm_claimed()
        got = L.llhip_engine_verify(at, lh.ptr(tokens), 24, 0, None, 0, lh.ptr(uniform), 0.8, ctypes.byref(following))
        assert not lh.last_error(), lh.last_error()
        assert (got, following.value) == ru.verify([0, 24], logits, None, tokens, uniform, 0.8)[0]
        claimed = L.llhip_hbm_claimed() - claimed
        assert claimed >= 4 * 20 * (vocab + 3 * ENGINE["dim"] + ENGINE["hidden_dim"])
        p = L.engine_forward_batch(at, lh.ptr(tokens), 24, 0, lh.LOGITS_ALL)
        assert (np.ctypeslib.as_array(ctypes.cast(p, ctypes.POINTER(ctypes.c_float)), (24, vocab)) == logits).all()
        monkeypatch.setenv("LLAMA_PREFILL_BATCH", "3")
        L.prefill_configure_engine(at, 3, kind == "q8")
        claimed = L.llhip_hbm_claimed()
        assert L.llhip_engine_verify(at, lh.ptr(tokens), 3, 0, None, 0, None, 0.0, ctypes.byref(following)) >= 0
        assert not lh.last_error() and L.llhip_hbm_claimed() == claimed
    finally:
        L.engine_free(at)


# ---- a small model served by all of them ------------------------------------------------------------------------------


class Served:
    """Two layers with their adapters: the float64 forward of one request's whole sequence, and the operands on the
    device."""
    dim, heads, kv, hd, hidden, vocab, layers, rank, adapters = 256, 4, 2, 64, 352, 700, 2, 8, 3

    def __init__(self, rng):
        kvl = self.kv * self.hd
        shapes = {"q": (self.dim, self.dim), "k": (kvl, self.dim), "v": (kvl, self.dim), "o": (self.dim, self.dim),
                  "1": (self.hidden, self.dim), "3": (self.hidden, self.dim), "2": (self.dim, self.hidden)}
        normal = lambda *s: (rng.standard_normal(s) / np.sqrt(s[-1])).astype(F)
        self.embed, self.cls = rng.standard_normal((self.vocab, self.dim), dtype=F), 4 * normal(self.vocab, self.dim)
        self.norm = np.ones(self.dim, F)
        self.w, self.a, self.b, self.scale = [], [], [], rng.uniform(0.5, 1.5, self.adapters).astype(F)
        for _ in range(self.layers):
            self.w.append({n: normal(*s) for n, s in shapes.items()})
            self.a.append({n: normal(self.adapters, self.rank, s[1]) for n, s in shapes.items()})
            self.b.append({n: normal(self.adapters, s[0], self.rank) for n, s in shapes.items()})
        self.dev = [{n: tuple(hu.dev(x) for x in (w[n], a[n], b[n])) for n in shapes}
                    for w, a, b in zip(self.w, self.a, self.b)]
        self.head = hu.dev(self.norm), hu.dev(self.cls), hu.dev(self.scale)

    def tables(self, positions):
        freq = 10000.0 ** (-np.arange(0, self.hd, 2) / self.hd)
        angle = np.arange(positions)[:, None] * freq
        return np.cos(angle).astype(F), np.sin(angle).astype(F)

    def plain(self, prefix, own, adapter):
        """The own tokens' logits in float64; the prefix has no adapter."""
        n, total = len(prefix), len(prefix) + len(own)
        x = self.embed[np.concatenate((prefix, own)).astype(int)].astype(np.float64)
        ids = np.array([-1] * n + [adapter] * len(own))
        cos, sin = (t.astype(np.float64) for t in self.tables(total))

        def project(l, name, x):
            y = x @ self.w[l][name].T.astype(np.float64)
            if adapter >= 0:
                low = x[n:] @ self.a[l][name][adapter].T.astype(np.float64)
                y[n:] += float(self.scale[adapter]) * (low @ self.b[l][name][adapter].T.astype(np.float64))
            return y

        def turn(y):
            y = y.reshape(total, -1, self.hd // 2, 2)
            c, s = cos[:, None], sin[:, None]
            return np.stack((y[..., 0] * c - y[..., 1] * s, y[..., 0] * s + y[..., 1] * c), -1).reshape(total, -1, self.hd)

        norm = lambda x: x / np.sqrt((x * x).mean(1, keepdims=True) + 1e-5)
        mul = self.heads // self.kv
        for l in range(self.layers):
            y = norm(x)
            q, k = turn(project(l, "q", y)), np.repeat(turn(project(l, "k", y)), mul, 1)
            v = np.repeat(project(l, "v", y).reshape(total, self.kv, self.hd), mul, 1)
            s = np.einsum("ihd,jhd->hij", q, k) / np.sqrt(self.hd)
            s[:, np.triu_indices(total, 1)[0], np.triu_indices(total, 1)[1]] = -np.inf
            p = np.exp(s - s.max(2, keepdims=True))
            p /= p.sum(2, keepdims=True)
            x = x + project(l, "o", np.einsum("hij,jhd->ihd", p, v).reshape(total, -1))
            y = norm(x)
            gate = project(l, "1", y)
            x = x + project(l, "2", gate / (1.0 + np.exp(-gate)) * project(l, "3", y))
        return (norm(x) @ self.cls.T.astype(np.float64))[n:]

    def run(self, L, tokens, b, ids, caches, prefix_caches, table, rows_of_logits=None):
        """The batch's logits on the device, by the library alone; caches [layer][key, value]."""
        T, m, kvl = hu.torch(), b.rows, self.kv * self.hd
        x = hu.dev(self.embed[np.asarray(tokens)])
        buf = {n: hu.dev(np.zeros((m, w), F)) for n, w in (("y", self.dim), ("q", self.dim), ("k", kvl), ("v", kvl),
                                                            ("at", self.dim), ("1", self.hidden), ("3", self.hidden))}
        idd = hu.dev(np.asarray(ids, np.int32))
        norm, cls, scale = self.head

        def gemm(x, k, *segments):
            L.k_gemm_f32(lh.ptr(x), k, m, k, ru.array([lh.GemmSegment(lh.ptr(c), w.shape[0], lh.ptr(w), None, k, w.shape[0],
                                                                      kind) for c, w, kind in segments]), len(segments))

        def lora(x, k, *segments):
            if b.count:
                L.llhip_lora_f32(lh.ptr(x), k, m, k, lh.ptr(idd), self.adapters, ru.array(segments), len(segments))

        def beside(l, name, c, **third):
            w, a, bb = self.dev[l][name]
            return ru.lora_segment(False, c, w.shape[0], c, a, bb, scale, w.shape[0], self.rank, **third)

        for l in range(self.layers):
            d = self.dev[l]
            L.k_rmsnorm_rows(lh.ptr(buf["y"]), lh.ptr(x), lh.ptr(norm), m, self.dim, 1e-5)
            gemm(buf["y"], self.dim, *[(buf[n], d[n][0], lh.GEMM_STORE) for n in "qkv"])
            lora(buf["y"], self.dim, *[beside(l, n, buf[n]) for n in "qkv"])
            L.llhip_rope_kv_store_requests(lh.ptr(buf["q"]), lh.ptr(buf["q"]), self.dim, lh.ptr(buf["k"]),
                                           lh.ptr(buf["v"]), kvl, lh.ptr(table), b.struct, self.heads, self.kv, self.hd,
                                           lh.ptr(caches[l][0]), lh.ptr(caches[l][1]))
            pk, pv = prefix_caches[l] if prefix_caches else (None, None)
            L.llhip_attention_requests(lh.ptr(buf["at"]), lh.ptr(buf["q"]), lh.ptr(pk), lh.ptr(pv), lh.ptr(caches[l][0]),
                                       lh.ptr(caches[l][1]), b.struct, self.heads, self.kv, self.hd)
            gemm(buf["at"], self.dim, (x, d["o"][0], lh.GEMM_ADD))
            lora(buf["at"], self.dim, beside(l, "o", x))
            L.k_rmsnorm_rows(lh.ptr(buf["y"]), lh.ptr(x), lh.ptr(norm), m, self.dim, 1e-5)
            gemm(buf["y"], self.dim, (buf["1"], d["1"][0], lh.GEMM_STORE), (buf["3"], d["3"][0], lh.GEMM_STORE))
            lora(buf["y"], self.dim, beside(l, "1", buf["1"], base3=buf["3"], a3=d["3"][1], b3=d["3"][2]))
            gemm(buf["1"], self.hidden, (x, d["2"][0], lh.GEMM_ADD))
            lora(buf["1"], self.hidden, beside(l, "2", x))
        L.k_rmsnorm_rows(lh.ptr(buf["y"]), lh.ptr(x), lh.ptr(norm), m, self.dim, 1e-5)
        quiet(L)
        last = buf["y"] if rows_of_logits is None else buf["y"][T.as_tensor(rows_of_logits, device="cuda")].contiguous()
        T.cuda.synchronize()
        m = len(last)
        logits = hu.dev(np.zeros((m, self.vocab), F))
        gemm(last, self.dim, (logits, cls, lh.GEMM_STORE))
        quiet(L)
        return logits


@pytest.mark.parametrize("layout", ["head", "rows"])
def test_a_model_served_by_all_of_them(L, layout):
    """A prefix computed once, then three requests with adapters 2, none and 0: their prompts, a step with drafts, and one
    more from where the drafts were left, whose cache rows replace the refused ones'. Logits against the whole sequences in
    float64, the decisions against those logits.

    Tolerance: each of the 2 * 9 products, sums and norms adds at most (dim / 32 + 48) U = 56 U of the sum of its terms'
    magnitudes, which here are at most 8 times the result's size; normed rows of size 1 carry it on unchanged, so that the
    logits, of size 4, are off by less than 18 * 56 * 8 * 4 U = 2e-3."""
    L.kernels_kv_layout_select(layout.encode())
    rng = np.random.default_rng(31)
    s = Served(rng)
    prefix, seq_len, slots, adapter, slot = rng.integers(0, s.vocab, 37), 40, 5, [2, -1, 0], [3, 0, 4]
    cos, sin = s.tables(len(prefix) + seq_len)
    table = hu.dev(np.concatenate((np.repeat(cos, 2, 1), np.stack((-sin, sin), 2).reshape(len(cos), -1)), 1).astype(F))
    made = lambda n, lead: [[hu.dev(np.full(lead + ru.cache_shape(layout, n, s.kv, s.hd), np.nan, F)) for _ in range(2)]
                            for _ in range(s.layers)]
    shared, caches = made(len(prefix), (1,)), made(seq_len, (slots,))
    alone = ru.Batch(hu.dev, [len(prefix)], [0], seq_len=len(prefix), slots=1)
    got = hu.host(s.run(L, prefix, alone, [-1] * len(prefix), shared, None, table))
    assert np.abs(got - s.plain([], prefix, -1)).max() < 2e-3
    own = [list(rng.integers(0, s.vocab, n)) for n in (7, 1, 12)]
    start = np.array([0, 7, 8, 20], np.int32)

    def batch(rows_of, length):
        return ru.Batch(hu.dev, rows_of, length, slot=slot, slots=slots, prefix=len(prefix), seq_len=seq_len)

    ids = lambda rows_of: np.repeat(adapter, rows_of)
    prompts = [len(o) for o in own]
    logits = s.run(L, sum(own, []), batch(prompts, [0, 0, 0]), ids(prompts), caches, shared, table, start[1:] - 1)
    got = hu.host(logits)
    want = [s.plain(prefix, o, a) for o, a in zip(own, adapter)]
    for r in range(3):
        assert np.abs(got[r] - want[r][-1]).max() < 2e-3, r
    decided = run_verify(L, np.arange(4, dtype=np.int32), got, None, np.zeros(3, np.int32), None, s.vocab, 0.0)
    assert decided == [(0, int(w.argmax())) for w in got]
    known = [n for _, n in decided]
    for rows_of, temperature in (([4, 1, 3], 0.0), ([2, 5, 3], 0.9), ([1, 2, 1], 0.0)):
        tokens, full = [], []
        for r in range(3):
            mine = [known[r]]
            while len(mine) < rows_of[r]:  # the model's own next token, but a wrong one last in the third request
                z = s.plain(prefix, own[r] + mine, adapter[r])[-1]
                mine.append(int(z.argmin() if r == 2 and len(mine) == rows_of[r] - 1 else z.argmax()))
            tokens += mine
            full.append(mine)
        b = batch(rows_of, [len(o) for o in own])
        got = hu.host(s.run(L, tokens, b, ids(rows_of), caches, shared, table))
        for r in range(3):
            want = s.plain(prefix, own[r] + full[r], adapter[r])[len(own[r]):]
            assert np.abs(got[b.start[r]:b.start[r + 1]] - want).max() < 2e-3, (r, rows_of)
        uniform = rng.random((b.rows, 2)).astype(F) if temperature else None
        tokens = np.asarray(tokens, np.int32)
        decided = run_verify(L, b.start, got, None, tokens, uniform, s.vocab, temperature)
        assert decided == ru.verify(b.start, got, None, tokens, uniform, temperature)
        for r, (n, following) in enumerate(decided):
            own[r] += full[r][:n + 1]
            known[r] = following
    quiet(L)
