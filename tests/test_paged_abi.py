"""The entry points over pages and of the scoring without a GPU: struct layouts as a C compiler sees them, and every refusal
that the host decides, each before anything is launched. CPU only."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

import llama_hip as lh
from tests import paged_util as pu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
F = np.float32


@pytest.fixture
def L():
    lib = lh.load()
    lh.record_failures()
    yield lib
    lib.llhip_set_fail_mode(lh.LLHIP_FAIL_EXIT)
    lib.llhip_clear_error()


def refused(L, words):
    message = lh.last_error()
    L.llhip_clear_error()
    assert words in message, message


def test_struct_layouts(tmp_path):
    src = r'''
#include <stdio.h>
#include "llama_hip_paged.h"
int main(void) {
  printf("%zu %zu %zu %d %d %d\n", sizeof(PagedBatch), offsetof(PagedBatch, max_pages), offsetof(PagedBatch, type),
         (int)PAGE_F32, (int)PAGE_BF16, (int)LLHIP_MAX_TOP);
  return 0;
}
'''
    (tmp_path / "probe.c").write_text(src)
    exe = str(tmp_path / "probe")
    subprocess.run(["gcc", "-std=c11", f"-I{ROOT}/include", str(tmp_path / "probe.c"), "-o", exe], check=True)
    got = [int(v) for v in subprocess.run([exe], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [ctypes.sizeof(lh.PagedBatch), lh.PagedBatch.max_pages.offset, lh.PagedBatch.type.offset, lh.PAGE_F32,
                   lh.PAGE_BF16, lh.LLHIP_MAX_TOP]


def make(**over):
    args = {"rows_of": [2, 1], "length": [0, 30], "page": 16}
    args.update(over)
    return pu.Pages(lambda x: x, **args)


BATCH_FAULTS = (("start", None, "index array"), ("length", None, "index array"), ("pages", None, "index array"),
                ("type", 2, "type 2"), ("type", -1, "type -1"), ("count", lh.LLHIP_MAX_REQUESTS + 1, "at most 1024"),
                ("page_size", 0, "pages of 0"), ("page_size", -16, "pages of -16"), ("max_pages", 0, "at most 0 pages"),
                ("num_pages", 0, "0 pages in all"), ("seq_len", 0, "0 positions"), ("seq_len", 65, "65 positions"))


def attention_call(L, batch, heads=4, kv=2, hd=8, rows=3, q_stride=None, pool=6, **over):
    a = {"out": np.zeros((rows, heads * hd), F), "q": np.zeros((rows, heads * hd), F),
         "k": np.zeros((pool, kv, 16, hd), F), "v": np.zeros((pool, kv, 16, hd), F)}
    a.update(over)
    L.llhip_attention_paged(lh.ptr(a["out"]), lh.ptr(a["q"]), q_stride or heads * hd, lh.ptr(a["k"]), lh.ptr(a["v"]), batch,
                            heads, kv, hd)


def test_attention_refusals(L):
    attention_call(L, None)
    refused(L, "null batch")
    for field, value, words in BATCH_FAULTS:
        b = make()
        assert b.seq_len == 64 and b.pool == 6
        setattr(b.struct, field, value)
        attention_call(L, b.struct)
        refused(L, words)
    b = make()
    attention_call(L, b.struct, heads=5)
    refused(L, "5 heads over 2 KV heads")
    attention_call(L, b.struct, heads=34)
    refused(L, "at most 16 per KV head")
    attention_call(L, b.struct, hd=257)
    refused(L, "head_dim <= 256")
    attention_call(L, b.struct, q_stride=31)
    refused(L, "shorter than its row")
    for name in ("out", "q", "k", "v"):
        attention_call(L, b.struct, **{name: None})
        refused(L, "null buffer")
    both = np.zeros((4, 32), F)
    attention_call(L, b.struct, q=both, out=both[1:])
    refused(L, "must not overlap")
    wide = np.zeros((3, 80), F)
    attention_call(L, b.struct, q=wide, q_stride=80, out=wide.reshape(-1)[100:])
    refused(L, "must not overlap")
    for name in ("k", "v"):
        cache = np.zeros((6, 2, 16, 8), F)
        attention_call(L, b.struct, **{name: cache, "out": cache.reshape(-1, 32)[40:]})
        refused(L, "must not overlap")
    for array in b.keep:
        attention_call(L, b.struct, out=array)
        refused(L, "must not overlap")
    # nothing to do is no failure, whatever the rest holds
    for field in ("count", "rows"):
        b = make()
        setattr(b.struct, field, 0)
        attention_call(L, b.struct, q=None)
        assert not lh.last_error()


def test_attention_of_no_heads_is_refused(L):
    """No head, or fewer: the tiles' rows would be a quotient by the heads of a KV head."""
    b, rows, cache = make(), np.zeros((3, 32), F), np.zeros((2, 6, 2, 16, 8), F)
    for heads in (0, -2, -2 ** 31):
        L.llhip_attention_paged(lh.ptr(rows), lh.ptr(rows.copy()), 32, lh.ptr(cache[0]), lh.ptr(cache[1]), b.struct, heads, 2, 8)
        refused(L, f"{heads} heads over 2 KV heads")


def append_call(L, batch, heads=4, kv=2, hd=8, rows=3, o_stride=None, q_stride=None, kv_stride=None, **over):
    a = {"o": np.zeros((rows, heads * hd), F), "q": np.zeros((rows, heads * hd), F), "k": np.zeros((rows, kv * hd), F),
         "v": np.zeros((rows, kv * hd), F), "t": np.zeros((64, 2 * hd), F), "qn": np.zeros(hd, F), "kn": np.zeros(hd, F),
         "kc": np.zeros((6, kv, 16, hd), F), "vc": np.zeros((6, kv, 16, hd), F)}
    a.update(over)
    L.llhip_rope_kv_append_paged(lh.ptr(a["o"]), o_stride or heads * hd, lh.ptr(a["q"]), q_stride or heads * hd,
                                 lh.ptr(a["k"]), lh.ptr(a["v"]), kv_stride or kv * hd, lh.ptr(a["t"]), lh.ptr(a["qn"]),
                                 lh.ptr(a["kn"]), 1e-5, batch, heads, kv, hd, lh.ptr(a["kc"]), lh.ptr(a["vc"]))


def test_append_refusals(L):
    append_call(L, None)
    refused(L, "null batch")
    for field, value, words in BATCH_FAULTS:
        b = make()
        setattr(b.struct, field, value)
        append_call(L, b.struct)
        refused(L, words)
    b = make()
    append_call(L, b.struct, hd=7)
    refused(L, "head_dim even")
    append_call(L, b.struct, heads=34)
    refused(L, "at most 16 per KV head")
    for stride in ({"q_stride": 31}, {"o_stride": 31}, {"kv_stride": 15}):
        append_call(L, b.struct, **stride)
        refused(L, "shorter than its row")
    for name in ("o", "q", "k", "v", "t", "kc", "vc"):
        append_call(L, b.struct, **{name: None})
        refused(L, "null buffer")
    rows = np.zeros((4, 32), F)
    append_call(L, b.struct, o=rows, q=rows, o_stride=40)
    refused(L, "at another stride")
    append_call(L, b.struct, o=rows[1:], q=rows)
    refused(L, "must not overlap")
    cache = np.zeros((6, 2, 16, 8), F)
    for over in ({"kc": cache, "vc": cache}, {"kc": cache, "q": cache}, {"vc": cache, "k": cache}, {"kc": cache, "v": cache},
                 {"vc": cache, "t": cache}, {"kc": cache, "qn": cache}, {"kc": cache, "kn": cache}, {"vc": cache, "o": cache}):
        append_call(L, b.struct, **over)
        refused(L, "must not overlap")
    # rows of one buffer: q's columns and k's must differ
    packed = np.zeros((4, 64), F)
    flat = packed.reshape(-1)
    for at in (16, 31, 64 - 15):
        append_call(L, b.struct, o=flat, q=flat, o_stride=64, q_stride=64, kv_stride=64, k=flat[at:])
        refused(L, "must not overlap")
    table, norm = np.zeros((64, 16), F), np.zeros(8, F)
    for over in ({"o": table, "t": table}, {"o": norm, "qn": norm}, {"o": norm, "kn": norm}):
        append_call(L, b.struct, **over)
        refused(L, "must not overlap")
    for array in b.keep:
        for name in ("o", "kc", "vc"):
            append_call(L, b.struct, **{name: array})
            refused(L, "must not overlap")


def score_call(L, rows=3, vocab=10, top=2, ld=None, temperature=1.0, **over):
    a = {"p": np.zeros(rows, F), "e": np.zeros(rows, F), "tt": np.zeros((rows, 2), np.int32), "tp": np.zeros((rows, 2), F),
         "l": np.zeros((rows, vocab), F), "t": np.zeros(rows, np.int32)}
    a.update(over)
    L.llhip_token_logprobs(lh.ptr(a["p"]), lh.ptr(a["e"]), lh.ptr(a["tt"]), lh.ptr(a["tp"]), top, lh.ptr(a["l"]),
                           vocab if ld is None else ld, lh.ptr(a["t"]), rows, vocab, temperature)


def test_score_refusals(L):
    for t in (0.0, -1.0, float("inf"), float("nan")):
        score_call(L, temperature=t)
        refused(L, "finite and positive")
    for top in (-1, lh.LLHIP_MAX_TOP + 1):
        score_call(L, top=top)
        refused(L, "0 to 32 are given")
    score_call(L, ld=9)
    refused(L, "at a stride of 9")
    score_call(L, vocab=0, l=np.zeros(4, F))
    refused(L, "rows of 0 logits")
    one = np.zeros(1, F)
    score_call(L, rows=(1 << 20) + 1, p=one, e=one, t=one, l=one)
    refused(L, "at most 2^20 rows")
    score_call(L, vocab=(1 << 22) + 1, l=one)
    refused(L, "2^22 tokens")
    for name in ("l", "t", "p", "tt", "tp"):
        score_call(L, **{name: None})
        refused(L, "null buffer")
    both, ints = np.zeros((4, 10), F), np.zeros(8, np.int32)
    for over in ({"p": both, "e": both}, {"p": both, "tp": both[0, 2:]}, {"e": both, "tp": both}, {"p": both, "l": both},
                 {"e": both[2:], "l": both}, {"tp": both, "l": both}, {"tt": ints, "t": ints}, {"p": ints, "t": ints[2:]}):
        score_call(L, **over)
        refused(L, "must not overlap")
    score_call(L, rows=0, l=None)  # nothing to do
    score_call(L, top=0, p=None, t=None, e=None, tt=None, tp=None)
    assert not lh.last_error()


def test_sizes_that_no_memory_holds(L):
    """Products of sizes past 64 bits, some of them 0 modulo 2^64: refused before an address is formed of them."""
    for stride in (1 << 61, 1 << 62, (1 << 62) + 32, (1 << 63) - 1, (1 << 64) - 1, 1 << 56):
        attention_call(L, make().struct, q_stride=stride)
        refused(L, "more than 2^56 bytes")
        for name in ("o_stride", "q_stride", "kv_stride"):
            append_call(L, make().struct, **{name: stride})
            refused(L, "more than 2^56 bytes")
        score_call(L, ld=stride)
        refused(L, "more than 2^56 bytes")
    for pages, page in ((2 ** 31 - 1, 2 ** 31 - 1), (2 ** 30, 2 ** 30), (2 ** 27, 2 ** 30)):
        for call, kv in ((attention_call, 2), (append_call, 2), (attention_call, 4)):
            b = make()
            b.struct.num_pages, b.struct.page_size = pages, page
            call(L, b.struct, kv=kv)
            refused(L, "more than 2^56 bytes")


def test_engine_logprobs_without_a_model(L):
    model, out = lh.Model(), np.full(2, 7.0, F)
    for m in (None, ctypes.byref(model)):
        got = L.llhip_engine_logprobs(m, lh.ptr(np.zeros(2, np.int32)), 2, 0, 1.0, 0, lh.ptr(out), None, None, None)
        assert got == -1 and (out == 7.0).all()
        refused(L, "no model loaded")
