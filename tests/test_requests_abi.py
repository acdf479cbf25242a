"""The entry points for many requests without a GPU: struct layouts as a C compiler sees them, and every refusal that the
host decides, each before anything is launched. CPU only."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

import llama_hip as lh
from tests import requests_util as ru

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


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
#include "llama_hip_requests.h"
int main(void) {
  printf("%zu %zu %zu %zu %zu %zu %zu %d %d\n", sizeof(RequestBatch), offsetof(RequestBatch, slots), sizeof(LoraSegment),
         offsetof(LoraSegment, scale), offsetof(LoraSegment, kind), sizeof(LoraBf16Segment),
         offsetof(LoraBf16Segment, kind), (int)LLHIP_MAX_REQUESTS, (int)LLHIP_MAX_LORA_RANK);
  return 0;
}
'''
    (tmp_path / "probe.c").write_text(src)
    exe = str(tmp_path / "probe")
    subprocess.run(["gcc", "-std=c11", f"-I{ROOT}/include", str(tmp_path / "probe.c"), "-o", exe], check=True)
    got = [int(v) for v in subprocess.run([exe], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [ctypes.sizeof(lh.RequestBatch), lh.RequestBatch.slots.offset, ctypes.sizeof(lh.LoraSegment),
                   lh.LoraSegment.scale.offset, lh.LoraSegment.kind.offset, ctypes.sizeof(lh.LoraBf16Segment),
                   lh.LoraBf16Segment.kind.offset, lh.LLHIP_MAX_REQUESTS, lh.LLHIP_MAX_LORA_RANK]


def attention_call(L, batch, heads=4, kv=2, hd=8, rows=3, **over):
    a = {"out": np.zeros((rows, heads * hd), np.float32), "q": np.zeros((rows, heads * hd), np.float32),
         "pk": np.zeros((kv, 8, hd), np.float32), "pv": np.zeros((kv, 8, hd), np.float32),
         "k": np.zeros((2, kv, 16, hd), np.float32), "v": np.zeros((2, kv, 16, hd), np.float32)}
    a.update(over)
    L.llhip_attention_requests(*[lh.ptr(a[n]) for n in ("out", "q", "pk", "pv", "k", "v")], batch, heads, kv, hd)
    return a


def make(**over):
    args = {"rows_of": [2, 1], "length": [0, 3], "prefix": 5, "prefix_seq_len": 8, "seq_len": 16, "slots": 2}
    args.update(over)
    return ru.Batch(lambda x: x, **args)


def test_attention_refusals(L):
    attention_call(L, None)
    refused(L, "null batch")
    for field, value, words in (("seq_len", 0, "slots of"), ("slots", 0, "slots of"), ("prefix", -1, "a prefix of"),
                                ("prefix", 9, "a prefix of"), ("seq_len", 2 ** 31 - 2, "a prefix of"),
                                ("count", lh.LLHIP_MAX_REQUESTS + 1, "at most 1024"), ("start", None, "index array"),
                                ("length", None, "index array")):
        b = make()
        setattr(b.struct, field, value)
        attention_call(L, b.struct)
        refused(L, words)
    b = make()
    attention_call(L, b.struct, heads=5)
    refused(L, "5 heads over 2 KV heads")
    attention_call(L, b.struct, heads=34, kv=2)
    refused(L, "at most 16 per KV head")
    attention_call(L, b.struct, hd=257)
    refused(L, "head_dim <= 256")
    attention_call(L, b.struct, pk=None)
    refused(L, "null buffer")
    attention_call(L, b.struct, q=None)
    refused(L, "null buffer")
    both = np.zeros((4, 32), np.float32)
    attention_call(L, b.struct, q=both, out=both[1:])
    refused(L, "must not overlap")
    k = np.zeros((2, 2, 16, 8), np.float32)
    attention_call(L, b.struct, k=k, out=k.reshape(-1, 32))
    refused(L, "must not overlap")
    # nothing to do is no failure, whatever the rest holds
    b.struct.count = 0
    attention_call(L, b.struct, q=None)
    assert not lh.last_error()


def rope_call(L, batch, heads=4, kv=2, hd=8, rows=3, q_stride=None, kv_stride=None, **over):
    a = {"o": np.zeros((rows, heads * hd), np.float32), "q": np.zeros((rows, heads * hd), np.float32),
         "k": np.zeros((rows, kv * hd), np.float32), "v": np.zeros((rows, kv * hd), np.float32),
         "t": np.zeros((21, 2 * hd), np.float32), "kc": np.zeros((2, kv, 16, hd), np.float32),
         "vc": np.zeros((2, kv, 16, hd), np.float32)}
    a.update(over)
    L.llhip_rope_kv_store_requests(lh.ptr(a["o"]), lh.ptr(a["q"]), q_stride or heads * hd, lh.ptr(a["k"]),
                                   lh.ptr(a["v"]), kv_stride or kv * hd, lh.ptr(a["t"]), batch, heads, kv, hd,
                                   lh.ptr(a["kc"]), lh.ptr(a["vc"]))


def test_rope_refusals(L):
    b = make()
    rope_call(L, None)
    refused(L, "null batch")
    rope_call(L, b.struct, hd=7)
    refused(L, "head_dim even")
    rope_call(L, b.struct, q_stride=31)
    refused(L, "shorter than its row")
    rope_call(L, b.struct, kv_stride=15)
    refused(L, "shorter than its row")
    for name in ("o", "q", "k", "v", "t", "kc", "vc"):
        rope_call(L, b.struct, **{name: None})
        refused(L, "null buffer")
    cache = np.zeros((2, 2, 16, 8), np.float32)
    rope_call(L, b.struct, kc=cache, vc=cache)
    refused(L, "must not overlap")
    rope_call(L, b.struct, kc=cache, k=cache.reshape(-1, 16))
    refused(L, "must not overlap")
    rows = np.zeros((4, 32), np.float32)
    rope_call(L, b.struct, o=rows[1:], q=rows)
    refused(L, "must not overlap")
    packed = np.zeros((3, 64), np.float32)  # k starting inside q's columns
    rope_call(L, b.struct, o=packed, q=packed, k=packed.reshape(-1)[31:], v=packed.reshape(-1)[48:], q_stride=64,
              kv_stride=64)
    refused(L, "must not overlap")


@pytest.mark.parametrize("array", [0, 1, 2])
def test_outputs_over_the_batchs_arrays_are_refused(L, array):
    """An output over the first or last entry of start, length or slot, of which a slot may be missing."""
    for entry, at in ((0, 0), (0, 95), (-1, 50)):
        b = make(slot=[1, 0])
        memory = np.zeros(4096, np.float32)
        field = ("start", "length", "slot")[array]
        ints = memory[1024:1024 + len(b.keep[array])].view(np.int32)
        ints[:] = b.keep[array]
        setattr(b.struct, field, lh.ptr(ints))
        begin = 1024 + entry % ints.size - at
        attention_call(L, b.struct, out=memory[begin:begin + 96].reshape(3, 32))
        refused(L, "must not overlap")
        rope_call(L, b.struct, o=memory[begin:begin + 96].reshape(3, 32))
        refused(L, "must not overlap")
        for cache in ("kc", "vc"):
            rope_call(L, b.struct, **{cache: memory[begin:begin + 512]})
            refused(L, "must not overlap")


def lora_call(L, m=3, k=8, ldx=8, adapters=2, count=1, bf16=False, x=True, ids=True, edit=None, segments=None, **over):
    kind = np.uint16 if bf16 else np.float32
    c, base = np.zeros((m, 6), np.float32), np.zeros((m, 6), np.float32)
    a, b, scale = np.zeros((adapters, 4, k), kind), np.zeros((adapters, 6, 4), kind), np.ones(adapters, np.float32)
    segs = segments or ru.array([ru.lora_segment(bf16, c, 6, base, a, b, scale, 6, 4) for _ in range(max(count, 1))])
    for field, value in (edit or {}).items():
        setattr(segs[0], field, value)
    xs, id_ = np.zeros((m, ldx), np.float32), np.zeros(m, np.int32)
    fn = L.llhip_lora_bf16 if bf16 else L.llhip_lora_f32
    fn(lh.ptr(xs) if x else None, over.get("ldx_", ldx), m, k, lh.ptr(id_) if ids else None, over.get("n_adapters", adapters),
       segs, over.get("n_segments", count))
    return (c, base, a, b, scale, xs, id_)


@pytest.mark.parametrize("bf16", [False, True])
def test_lora_refusals(L, bf16):
    lora_call(L, bf16=bf16, n_segments=4)
    refused(L, "4 segments")
    lora_call(L, bf16=bf16, ldx_=7)
    refused(L, "at stride 7")
    lora_call(L, bf16=bf16, n_adapters=0)
    refused(L, "0 adapters")
    lora_call(L, bf16=bf16, x=False)
    refused(L, "null buffer")
    lora_call(L, bf16=bf16, ids=False)
    refused(L, "null buffer")
    for edit, words in (({"kind": lh.GEMM_STORE}, "not GEMM_ADD"), ({"kind": 9}, "not GEMM_ADD"), ({"n": 0}, "0 columns"),
                        ({"ldc": 5}, "stride 5"), ({"rank": 0}, "rank 0"), ({"rank": 257}, "rank 257"),
                        ({"c": None}, "null buffer"), ({"base": None}, "null buffer"), ({"b": None}, "null buffer"),
                        ({"kind": lh.GEMM_SWIGLU}, "null buffer")):
        lora_call(L, bf16=bf16, edit=edit)
        refused(L, words)
    # two segments with one output, an output inside x, a shifted base
    shared = np.zeros((4, 6), np.float32)
    a, b = np.zeros((2, 4, 8), np.uint16 if bf16 else np.float32), np.zeros((2, 6, 4), np.uint16 if bf16 else np.float32)
    one = lambda c, base: ru.lora_segment(bf16, c, 6, base, a, b, None, 6, 4)  # noqa: E731
    lora_call(L, bf16=bf16, n_segments=2, segments=ru.array([one(shared, shared), one(shared, shared)]))
    refused(L, "overlaps")
    lora_call(L, bf16=bf16, segments=ru.array([one(shared[1:], shared)]))
    refused(L, "overlaps")
    lora_call(L, m=0, bf16=bf16, x=False)
    assert not lh.last_error()


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("own", [False, True])
def test_lora_refuses_outputs_over_any_segments_inputs(L, bf16, own):
    """An output over the adapters, the second adapters or the scales of its own segment or another, or over the ids."""
    kind = np.uint16 if bf16 else np.float32
    memory = np.zeros(4096, np.float32)
    c, base = memory[64:64 + 18].reshape(3, 6), np.zeros((3, 6), np.float32)
    a, b, scale = np.zeros((2, 4, 8), kind), np.zeros((2, 6, 4), kind), np.ones(2, np.float32)
    fn = L.llhip_lora_bf16 if bf16 else L.llhip_lora_f32
    x, ids = np.zeros((3, 8), np.float32), np.zeros(3, np.int32)

    def call(ids=ids, **over):
        t = {"a": a, "b": b, "a3": a, "b3": b, "scale": scale}
        t.update(over)
        target = ru.lora_segment(bf16, c if own else np.zeros((3, 6), np.float32), 6, base, t["a"], t["b"], t["scale"], 6, 4,
                                 base, t["a3"], t["b3"])
        first = ru.lora_segment(bf16, c, 6, base, a, b, None, 6, 4)
        segs = ru.array([target] if own else [first, target])
        fn(lh.ptr(x), 8, 3, 8, lh.ptr(ids), 2, segs, len(segs))

    units = memory.view(kind)
    per = units.size // memory.size
    for name, size in (("a", 64), ("b", 48), ("a3", 64), ("b3", 48)):
        for at in (64 * per - size + 1, 64 * per + 5, (64 + 18) * per - 1):
            call(**{name: units[at:at + size]})
            refused(L, "overlaps an input")
    for at in (63, 70, 81):
        call(scale=memory[at:at + 2])
        refused(L, "overlaps an input")
    for at in (62, 70, 81):
        call(ids=memory.view(np.int32)[at:at + 3])
        refused(L, "overlaps an input")


def verify_call(L, vocab=10, rows=4, count=2, temperature=1.0, ld=10, draft_ld=10, **over):
    a = {"accepted": np.zeros(2, np.int32), "next": np.zeros(2, np.int32), "logits": np.zeros((4, 10), np.float32),
         "draft": np.zeros((4, 10), np.float32), "tokens": np.zeros(4, np.int32), "uniform": np.zeros((4, 2), np.float32),
         "start": np.array([0, 2, 4], np.int32)}
    a.update(over)
    L.llhip_verify_drafts(lh.ptr(a["accepted"]), lh.ptr(a["next"]), lh.ptr(a["logits"]), ld, lh.ptr(a["draft"]), draft_ld,
                          lh.ptr(a["tokens"]), lh.ptr(a["uniform"]), lh.ptr(a["start"]), count, rows, vocab, temperature)


def test_verify_refusals(L):
    for t in (-0.5, float("nan"), float("inf")):
        verify_call(L, temperature=t)
        refused(L, "must be finite and not negative")
    verify_call(L, count=lh.LLHIP_MAX_REQUESTS + 1)
    refused(L, "at most 1024")
    verify_call(L, vocab=0)
    refused(L, "rows of 0 logits")
    verify_call(L, ld=9)
    refused(L, "at strides 9")
    verify_call(L, draft_ld=9)
    refused(L, "and 9")
    for name in ("accepted", "next", "logits", "tokens", "uniform", "start"):
        verify_call(L, **{name: None})
        refused(L, "null buffer")
    same = np.zeros(3, np.int32)
    verify_call(L, accepted=same, next=same[1:])
    refused(L, "must not overlap")
    for name in ("accepted", "next"):
        tokens, start, uniform = np.zeros(4, np.int32), np.array([0, 2, 4], np.int32), np.zeros((4, 2), np.float32)
        logits, draft = np.zeros((4, 10), np.float32), np.zeros((4, 10), np.float32)
        for over in ({"tokens": tokens, name: tokens[2:]}, {"start": start, name: start[1:]},
                     {"uniform": uniform, name: uniform.view(np.int32)[1:]}, {"logits": logits, name: logits[3, 8:]},
                     {"draft": draft, name: draft[3, 8:]}):
            verify_call(L, **over)
            refused(L, "must not overlap an input")
    verify_call(L, count=0, logits=None)
    assert not lh.last_error()


def test_engine_verify_without_a_model(L):
    following = ctypes.c_int(7)
    model = lh.Model()
    for m in (None, ctypes.byref(model)):
        got = L.llhip_engine_verify(m, lh.ptr(np.zeros(2, np.int32)), 2, 0, None, 0, None, 0.0, ctypes.byref(following))
        assert got == -1 and following.value == 7
        refused(L, "no model loaded")
