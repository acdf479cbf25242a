"""Log probabilities of given tokens, entropies and the likeliest tokens, on the GPU, against float64 (tests/paged_util.py)."""
import ctypes
import os

import numpy as np
import pytest

import llama_hip as lh
from llama_hip import checkpoint as ck
from tests import hip_util as hu
from tests import paged_util as pu
from tests.requests_util import U

pytestmark = pytest.mark.gpu
F = np.float32


@pytest.fixture
def L():
    lib = lh.load()
    assert lib.llhip_init() == 0, lh.last_error()
    lh.record_failures()
    yield lib
    lib.llhip_synchronize()
    lib.llhip_clear_error()
    lib.llhip_set_fail_mode(lh.LLHIP_FAIL_EXIT)


def call(L, logits, tokens, temperature=1.0, top=0, entropy=True, ld=None, dev=hu.dev):
    rows, vocab = logits.shape
    wide = logits
    if ld:
        wide = np.full((rows, ld), np.nan, F)
        wide[:, :vocab] = logits
    ld = ld or vocab
    ins = [dev(wide), None if tokens is None else dev(np.asarray(tokens, np.int32))]
    outs = [None if tokens is None else dev(np.full(rows, 7.0, F)), dev(np.full(rows, 7.0, F)) if entropy else None,
            dev(np.full((rows, top), 7, np.int32)) if top else None, dev(np.full((rows, top), 7.0, F)) if top else None]
    L.llhip_token_logprobs(*[lh.ptr(x) for x in outs], top, lh.ptr(ins[0]), ld, lh.ptr(ins[1]), rows, vocab, temperature)
    return [None if x is None else x if isinstance(x, np.ndarray) else hu.host(x) for x in outs]


def check(L, logits, tokens, temperature=1.0, top=0, **kw):
    """The bound: with z = (l - max) / T, an exponential is off by (|z| + 4) 2 U of itself (the difference's rounding, the
    scale's and the exponential's), so the rest of the sum, r = S - 1, by E = U sum over the others of e^z (2 |z| + 8) + 20 U r
    (16 values a lane, the lanes) and log1p(r) by E / (1 + r) at most; a log probability by that and its own rounding. The
    entropy log S + sum(-z e^z) / S: its second sum by U sum e^z |z| (2 |z| + 30), both relative to S, and by its own rounding."""
    got = call(L, logits, tokens, temperature, top, **kw)
    L.llhip_synchronize()
    assert not lh.last_error(), lh.last_error()
    logprob, entropy, tops, top_logprob = pu.scores(logits, tokens, temperature, top)
    z = logits.astype(np.float64) / float(F(temperature))
    z = z - z.max(1, keepdims=True)
    e = np.exp(z)
    size = np.where(e > 0, -z, 0.0)
    other = np.where(z < 0, e, 0.0)
    whole = e.sum(1)
    off = U * ((other * (2 * size + 8)).sum(1) + 20 * other.sum(1)) / whole
    if tokens is not None:
        want = logprob
        fine = np.isfinite(want)
        assert np.array_equal(got[0][~fine], want[~fine].astype(F))
        assert (np.abs(got[0] - want)[fine] <= (off + U * np.abs(want))[fine] + 1e-38).all()
    if got[1] is not None:
        second = (e * size).sum(1) / whole
        bound = off * (1 + second) + U * (e * size * (2 * size + 30)).sum(1) / whole + U * np.abs(entropy) + 1e-38
        assert (np.abs(got[1] - entropy) <= bound).all(), np.abs(got[1] - entropy) / bound
    if top:
        assert np.array_equal(got[2], tops)
        there = tops >= 0
        assert (got[3][~there] == -np.inf).all()
        with np.errstate(invalid="ignore"):
            wrong = np.abs(got[3] - top_logprob)
        assert (wrong[there] <= (off[:, None] + U * np.abs(top_logprob))[there] + 1e-38).all()
    return got


@pytest.mark.parametrize("vocab", [1, 2, 63, 64, 65, 300, 1023, 1024, 1025, 5000, 32000, 128256])
@pytest.mark.parametrize("top", [0, 1, 5, 20, 32])
@pytest.mark.parametrize("temperature", [1.0, 0.3])
def test_scores(L, vocab, top, temperature):
    rng = np.random.default_rng(vocab + top)
    rows = 5
    logits = (3.0 * rng.standard_normal((rows, vocab))).astype(F)
    tokens = rng.integers(0, vocab, rows)
    tokens[1] = -1
    tokens[2] = logits[2].argmax()
    check(L, logits, tokens, temperature, top)
    check(L, logits, None, temperature, top, ld=vocab + 3)
    check(L, logits, tokens, temperature, top, entropy=False, ld=vocab + 4)


@pytest.mark.parametrize("vocab", [70, 1024, 3000, 40000])
def test_equal_logits_and_masked_ones(L, vocab):
    """Rows of one value, of few values (ties go to the lower token), of zeros of both signs, with all but some tokens masked
    out, and peaked rows."""
    rng = np.random.default_rng(vocab)
    logits = np.zeros((9, vocab), F)
    logits[1] = rng.integers(0, 3, vocab)
    logits[2] = rng.choice(np.array([0.0, -0.0], F), vocab)
    logits[3] = -np.inf
    logits[3, [5, vocab - 1]] = 2.0
    logits[4] = np.where(rng.random(vocab) < 0.9, -np.inf, rng.standard_normal(vocab))
    logits[4, 7] = 0.0
    logits[5] = rng.standard_normal(vocab)
    logits[5, 3] = 80.0
    logits[6] = -1e30
    logits[6, vocab // 2] = 1e30
    logits[7] = np.linspace(9, -9, vocab)
    logits[8] = np.linspace(-9, 9, vocab) * F(1e-3)
    tokens = [vocab - 1, 3, 0, 6, 7, 3, vocab // 2, 0, vocab - 1]
    for top in (0, 1, 7, 32):
        got = check(L, logits, tokens, 1.0, top)
        assert got[0][3] == -np.inf
    check(L, logits, [5, 0, vocab - 1, 5, 7, 0, 0, 1, 2], 0.01, 32)


def test_rows_that_decide_nothing(L):
    """NaN, +infinity or nothing left: NaN in all places and tokens -1, a failure at the wait, and the rows beside them right."""
    rng = np.random.default_rng(1)
    for what in (np.nan, np.inf, None):
        logits = rng.standard_normal((3, 2000)).astype(F)
        if what is None:
            logits[1] = -np.inf
        else:
            logits[1, 1500] = what
        got = call(L, logits, [1, 2, 3], top=4)
        L.llhip_synchronize()
        assert "leave no token" in lh.last_error()
        L.llhip_clear_error()
        assert np.isnan(got[0][1]) and np.isnan(got[1][1]) and np.isnan(got[3][1]).all() and (got[2][1] == -1).all()
        rest = [0, 2]
        want = check(L, logits[rest], [1, 3], top=4)
        for g, w in zip(got, want):
            assert np.array_equal(g[rest], w)


def test_tokens_outside_the_vocabulary(L):
    rng = np.random.default_rng(2)
    logits = rng.standard_normal((4, 100)).astype(F)
    for bad in (100, -2, 2 ** 31 - 1, -2 ** 31):
        got = call(L, logits, [5, bad, -1, 99])
        L.llhip_synchronize()
        assert "scored token outside the vocabulary" in lh.last_error()
        L.llhip_clear_error()
        assert np.isnan(got[0][1]) and got[0][2] == 0.0 and np.isfinite(got[0]).sum() == 3


@pytest.mark.parametrize("temperature", [1e-40, 1e-20, 1e-3, 100.0, 3e38])
def test_temperatures(L, temperature):
    """Very cold and very hot ones: finite entropies, alternatives in the same order."""
    rng = np.random.default_rng(3)
    logits = rng.standard_normal((3, 5000)).astype(F)
    got = call(L, logits, logits.argmax(1), temperature, top=6)
    L.llhip_synchronize()
    assert not lh.last_error()
    if 1e-30 < temperature:
        check(L, logits, logits.argmax(1), temperature, top=6)
    assert np.isfinite(got[1]).all() and (got[0] <= 0.0).all()
    assert np.array_equal(got[2], np.argsort(-logits, 1, kind="stable")[:, :6])


@pytest.mark.parametrize("rows", [5, 8, 9, 16, 17, 64])
@pytest.mark.parametrize("vocab,top", [(1, 1), (65, 32), (1025, 5), (5000, 20), (32000, 0), (128256, 20), (128256, 32)])
@pytest.mark.parametrize("temperature", [1.0, 0.3])
def test_scores_of_few_and_many_rows(L, rows, vocab, top, temperature):
    """Both forms, one launch and two, over one chunk and many."""
    rng = np.random.default_rng(vocab + top + rows)
    logits = (3.0 * rng.standard_normal((rows, vocab))).astype(F)
    tokens = rng.integers(0, vocab, rows)
    tokens[1] = -1
    tokens[2] = logits[2].argmax()
    check(L, logits, tokens, temperature, top)
    check(L, logits, None, temperature, top, ld=vocab + 3)
    check(L, logits, tokens, temperature, top, entropy=False, ld=vocab + 4)


@pytest.mark.parametrize("rows", [5, 16, 17])
def test_vocabularies_past_the_groups_maxima(L, rows):
    """More than 262144 tokens: chunks' maxima in the groups' place; random rows, sorted ones, few values, masked ones."""
    rng = np.random.default_rng(rows)
    vocab = 300001
    logits = rng.standard_normal((rows, vocab)).astype(F)
    logits[1] = np.sort(logits[1])
    logits[2] = rng.integers(0, 3, vocab)
    logits[3] = np.where(rng.random(vocab) < 0.9999, -np.inf, logits[3])
    logits[3, 7] = 0.0
    logits[4] = np.sort(logits[4])[::-1]
    for top in (1, 32):
        check(L, logits, rng.integers(0, vocab, rows), 0.8, top)


@pytest.mark.parametrize("rows", [9, 17, 40])
@pytest.mark.parametrize("vocab", [70, 1024, 3000, 40000, 128256])
def test_equal_logits_and_masked_ones_of_many_rows(L, rows, vocab):
    """As test_equal_logits_and_masked_ones, each kind of row again and again; 32 alternatives of rows of one value, where more
    than 512 candidates meet."""
    rng = np.random.default_rng(vocab + rows)
    logits, tokens = np.zeros((rows, vocab), F), np.zeros(rows, np.int64)
    for i in range(rows):
        x, kind = logits[i], i % 8
        tokens[i] = rng.integers(0, vocab)
        if kind == 1:
            x[:] = rng.integers(0, 3, vocab)
        elif kind == 2:
            x[:] = rng.choice(np.array([0.0, -0.0], F), vocab)
        elif kind == 3:
            x[:] = -np.inf
            x[[5, vocab - 1]] = 2.0
        elif kind == 4:
            x[:] = np.where(rng.random(vocab) < 0.9, -np.inf, rng.standard_normal(vocab))
            x[7] = 0.0
        elif kind == 5:
            x[:] = rng.standard_normal(vocab)
            x[3] = 80.0
        elif kind == 6:
            x[:] = -1e30
            x[vocab // 2] = 1e30
        elif kind == 7:
            x[:] = np.linspace(9, -9, vocab)
    for top in (0, 1, 7, 32):
        check(L, logits, tokens, 1.0, top)


@pytest.mark.parametrize("vocab", [2000, 128256, 270000])
def test_rows_that_decide_nothing_among_many(L, vocab):
    """As test_rows_that_decide_nothing, in two launches; the other rows' results are those of the rows without them."""
    rng = np.random.default_rng(vocab)
    rows = 20
    for what in (np.nan, np.inf, None):
        logits = rng.standard_normal((rows, vocab)).astype(F)
        tokens = rng.integers(0, vocab, rows)
        bad = [0, 7, 19]
        for i in bad:
            if what is None:
                logits[i] = -np.inf
            else:
                logits[i, rng.integers(0, vocab)] = what
        got = call(L, logits, tokens, top=20)
        L.llhip_synchronize()
        assert "leave no token" in lh.last_error()
        L.llhip_clear_error()
        for i in bad:
            assert np.isnan(got[0][i]) and np.isnan(got[1][i]) and np.isnan(got[3][i]).all() and (got[2][i] == -1).all()
        rest = [i for i in range(rows) if i not in bad]
        want = check(L, logits[rest], tokens[rest], top=20)
        for g, w in zip(got, want):
            assert np.array_equal(g[rest], w)


def test_tokens_outside_the_vocabulary_among_many(L):
    rng = np.random.default_rng(2)
    rows, vocab = 33, 5000
    logits = rng.standard_normal((rows, vocab)).astype(F)
    good = rng.integers(0, vocab, rows)
    want = check(L, logits, good, top=3)
    for bad in (vocab, -2, 2 ** 31 - 1, -2 ** 31):
        tokens = good.copy()
        tokens[20] = bad
        got = call(L, logits, tokens, top=3)
        L.llhip_synchronize()
        assert "scored token outside the vocabulary" in lh.last_error()
        L.llhip_clear_error()
        assert np.isnan(got[0][20])
        assert np.array_equal(np.delete(got[0], 20), np.delete(want[0], 20))
        for g, w in zip(got[1:], want[1:]):
            assert np.array_equal(g, w)


@pytest.mark.parametrize("vocab", [700, 5000, 128256, 300001])
def test_a_row_scores_the_same_beside_any_others(L, vocab):
    """Bit for bit, in one launch and in two."""
    rng = np.random.default_rng(vocab)
    logits = (2.0 * rng.standard_normal((17, vocab))).astype(F)
    logits[3] = rng.integers(0, 3, vocab)
    tokens = rng.integers(0, vocab, 17)
    many = call(L, logits, tokens, 0.7, 32)
    for rows in ([3], [0, 3, 5, 16, 9], list(range(8)), list(range(9))):
        few = call(L, logits[rows], tokens[rows], 0.7, 32)
        for m, f in zip(many, few):
            assert np.array_equal(m[rows], f)
    L.llhip_synchronize()
    assert not lh.last_error()


def test_large_vocabularies_and_many_rows(L):
    rng = np.random.default_rng(4)
    logits = rng.standard_normal((2, 1 << 22)).astype(F)
    logits[1] = np.sort(logits[1])
    check(L, logits, [0, (1 << 22) - 1], top=32)
    logits = rng.standard_normal((33000, 70)).astype(F)
    check(L, logits, rng.integers(0, 70, 33000), top=3)


def test_host_buffers_and_graphs(L):
    rng = np.random.default_rng(5)
    logits = rng.standard_normal((6, 3000)).astype(F)
    tokens = rng.integers(0, 3000, 6).astype(np.int32)
    want = check(L, logits, tokens, top=5)
    got = call(L, logits, tokens, top=5, dev=lambda x: x)
    assert not lh.last_error()
    for g, w in zip(got, want):
        assert np.array_equal(g, w)
    T = hu.torch()
    ld, td = hu.dev(logits), hu.dev(tokens)
    outs = [hu.dev(np.zeros(6, F)), hu.dev(np.zeros(6, F)), hu.dev(np.zeros((6, 5), np.int32)), hu.dev(np.zeros((6, 5), F))]
    args = [lh.ptr(x) for x in outs] + [5, lh.ptr(ld), 3000, lh.ptr(td), 6, 3000, 0.7]
    L.llhip_token_logprobs(*args)
    L.llhip_synchronize()
    assert L.llhip_graph_begin() == 0
    L.llhip_token_logprobs(*args)
    graph = L.llhip_graph_end()
    assert graph, lh.last_error()
    for _ in range(3):
        logits = rng.standard_normal((6, 3000)).astype(F)
        ld.copy_(T.from_numpy(logits))
        td.copy_(T.from_numpy(rng.integers(0, 3000, 6).astype(np.int32)))
        T.cuda.synchronize()
        L.llhip_token_logprobs(*args)
        L.llhip_synchronize()
        eager = [hu.host(x).copy() for x in outs]
        for x in outs:
            x.zero_()
        T.cuda.synchronize()
        assert L.llhip_graph_launch(graph) == 0
        L.llhip_synchronize()
        for g, w in zip(outs, eager):
            assert np.array_equal(hu.host(g), w)
    L.llhip_graph_destroy(graph)


ENGINE = dict(dim=128, hidden_dim=192, n_layers=2, n_heads=4, n_kv_heads=2, vocab_size=1100, seq_len=96, head_dim=32)


def engine_model(path, kind):
    gs = 64
    norms, t = ck.synthetic(ENGINE, gs, 19)
    if kind == "q8":
        ck.write_q8_v3(path, ENGINE, gs, norms, t)
    else:
        f32 = {n: q.astype(F) * np.repeat(s.reshape(-1), gs).reshape(q.shape).astype(F) for n, (q, s) in t.items()}
        ck.write_f32_v3(path, ENGINE, norms, f32)


@pytest.mark.parametrize("kind", ["q8", "f32", "bf16", "q8_no_gemm"])
def test_engine_scores_a_text(L, tmp_path, monkeypatch, kind):
    """llhip_engine_logprobs against float64 on the logits that engine_forward_batch gives for the same rows at the same
    place: whole texts and one token, behind a prefix, into host and device memory; the model goes on as after
    engine_forward_batch; refusals leave it usable."""
    if kind == "bf16":
        monkeypatch.setenv("LLAMA_PRECISION", "bf16")
    if kind == "q8_no_gemm":
        monkeypatch.setenv("LLAMA_PREFILL_GEMM", "off")
        monkeypatch.setenv("LLAMA_PREFILL_BATCH", "24")
    L.kernels_kv_layout_select(b"head")
    path = os.path.join(tmp_path, "tiny.bin")
    engine_model(path, kind.split("_")[0])
    vocab = ENGINE["vocab_size"]
    rng = np.random.default_rng(3)
    model = lh.Model()
    at = ctypes.byref(model)
    try:
        L.engine_load(at, path.encode())
        assert model.implementation, lh.last_error()
        pos = 0
        for n, top, t in ((20, 5, 1.0), (1, 0, 1.0), (7, 32, 0.5), (24, 1, 1.7)):
            tokens = rng.integers(0, vocab, n).astype(np.int32)
            p = L.engine_forward_batch(at, lh.ptr(tokens), n, pos, lh.LOGITS_ALL)
            assert p, lh.last_error()
            logits = np.ctypeslib.as_array(ctypes.cast(p, ctypes.POINTER(ctypes.c_float)), (n, vocab)).copy()
            want = call(L, logits, np.append(tokens[1:], -1), t, top)
            L.llhip_synchronize()
            for dev in (lambda x: x, hu.dev):
                out = [dev(np.full(n, 7.0, F)), dev(np.full(n, 7.0, F)), dev(np.full((n, top), 7, np.int32)) if top else None,
                       dev(np.full((n, top), 7.0, F)) if top else None]
                assert L.llhip_engine_logprobs(at, lh.ptr(tokens), n, pos, t, top, *[lh.ptr(x) for x in out]) == 0, lh.last_error()
                got = [x if x is None or isinstance(x, np.ndarray) else hu.host(x) for x in out]
                for g, w in zip(got, want):
                    assert g is w is None or np.array_equal(g, w)
            plain = pu.scores(logits, np.append(tokens[1:], -1), t, top)
            assert np.allclose(got[0], plain[0], atol=1e-5) and (top == 0 or np.array_equal(got[2], plain[2]))
            pos += n
        out = np.full(2, 7.0, F)
        two, ints = np.array([1, 2], np.int32), np.zeros(8, np.int32)
        for args, words in (((lh.ptr(two), 2, 95, 1.0, 0, lh.ptr(out), None, None, None), "batch input out of range"),
                            ((lh.ptr(np.array([1, vocab], np.int32)), 2, 0, 1.0, 0, lh.ptr(out), None, None, None), "token="),
                            ((None, 2, 0, 1.0, 0, lh.ptr(out), None, None, None), "batch input out of range"),
                            ((lh.ptr(two), 0, 0, 1.0, 0, lh.ptr(out), None, None, None), "batch input out of range"),
                            ((lh.ptr(two), 2, 0, 0.0, 0, lh.ptr(out), None, None, None), "finite and positive"),
                            ((lh.ptr(two), 2, 0, 1.0, 33, lh.ptr(out), None, lh.ptr(ints), lh.ptr(ints)), "0 to 32"),
                            ((lh.ptr(two), 2, 0, 1.0, 1, lh.ptr(out), None, None, None), "null buffer"),
                            ((lh.ptr(two), 2, 0, 1.0, 0, None, None, None, None), "null buffer")):
            assert L.llhip_engine_logprobs(at, *args) == -1 and (out == 7.0).all()
            assert words in lh.last_error(), (words, lh.last_error())
        assert L.llhip_engine_logprobs(at, lh.ptr(two), 2, 0, 1.0, 0, lh.ptr(out), None, None, None) == 0
        assert out[1] == 0.0 and out[0] < 0.0
    finally:
        L.engine_free(at)
        L.llhip_clear_error()


def test_engine_scores_a_long_text_in_several_calls(L, tmp_path, monkeypatch):
    """Each call begins with the last token of the call before: bit for bit the text in one call, where rows run one at a time."""
    monkeypatch.setenv("LLAMA_PREFILL_GEMM", "off")
    monkeypatch.setenv("LLAMA_PREFILL_BATCH", "24")
    L.kernels_kv_layout_select(b"head")
    path = os.path.join(tmp_path, "tiny.bin")
    engine_model(path, "q8")
    tokens = np.random.default_rng(4).integers(0, ENGINE["vocab_size"], 24).astype(np.int32)
    model = lh.Model()
    at = ctypes.byref(model)

    def score(a, b, top=3):
        n = b - a
        out = [np.zeros(n, F), np.zeros(n, F), np.zeros((n, top), np.int32), np.zeros((n, top), F)]
        mine = np.ascontiguousarray(tokens[a:b])
        assert L.llhip_engine_logprobs(at, lh.ptr(mine), n, a, 0.8, top, *[lh.ptr(x) for x in out]) == 0, lh.last_error()
        return out

    try:
        L.engine_load(at, path.encode())
        assert model.implementation, lh.last_error()
        whole = score(0, 24)
        for cuts in ((0, 9, 24), (0, 1, 2, 16, 24)):
            parts = []
            for i, (a, b) in enumerate(zip(cuts, cuts[1:])):
                got = score(a - 1 if i else a, b)
                parts.append([x if b == 24 else x[:-1] for x in got])
            for w, *p in zip(whole, *parts):
                assert np.array_equal(np.concatenate(p), w), cuts
    finally:
        L.engine_free(at)
        L.llhip_clear_error()
