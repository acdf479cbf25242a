"""The operators of a batch of requests that one model serves, as cases that can be timed and checked one by one.

  attention  llhip_attention_requests: each request's rows attend to a prefix that all share, then to their own cache.
  rope       llhip_rope_kv_store_requests: RoPE of the rows at their requests' positions, and their cache rows.
  lora       llhip_lora_f32 / llhip_lora_bf16: each row's adapter beside a projection that all rows share.
  verify     llhip_verify_drafts: drafted tokens against the target's logits, from given random numbers.

run() computes them in elementary torch operations, or, where `own` is set, through the library's entry points. exact()
is written from the definitions, in float64.
"""
import math
import os
import random
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

# The attention heads of the Llama 3 sizes that the benchmark and the tests run.
HEADS_1B = {"heads": 32, "kv_heads": 8, "hd": 64}
HEADS_8B = {"heads": 32, "kv_heads": 8, "hd": 128}
VOCAB = 128256
DIM_8B, KV_8B, HIDDEN_8B, DIM_1B = 4096, 1024, 14336, 2048


def listed():
    return [
        # one chat request, its first own tokens behind a short system prompt: latency
        {"name": "attention_1b_first_tokens", "kind": "attention", **HEADS_1B, "requests": 1, "rows_min": 1,
         "rows_max": 1, "prefix": 200, "own": 5, "lens": 1},
        # a server's decode step: 32 chats behind one instruction prompt, each at its own length
        {"name": "attention_8b_decode_32", "kind": "attention", **HEADS_8B, "requests": 32, "rows_min": 1,
         "rows_max": 1, "prefix": 2048, "own": 700, "lens": 2},
        # the same with up to six drafted rows a request
        {"name": "attention_8b_drafts_16", "kind": "attention", **HEADS_8B, "requests": 16, "rows_min": 2,
         "rows_max": 7, "prefix": 4096, "own": 1500, "lens": 3},
        # new prompts read in one batch behind the prefix
        {"name": "attention_8b_prompts", "kind": "attention", **HEADS_8B, "requests": 5, "rows_min": 90,
         "rows_max": 600, "prefix": 1024, "own": 0, "lens": 4},
        # a full server behind a document that everybody asks about
        {"name": "attention_8b_decode_64_long", "kind": "attention", **HEADS_8B, "requests": 64, "rows_min": 1,
         "rows_max": 1, "prefix": 8192, "own": 1000, "lens": 5},
        # a decode step's rows, and the prompts' rows, into the requests' caches
        {"name": "rope_8b_decode_32", "kind": "rope", **HEADS_8B, "requests": 32, "rows_min": 1, "rows_max": 1,
         "prefix": 2048, "own": 700, "lens": 6},
        {"name": "rope_1b_prompts", "kind": "rope", **HEADS_1B, "requests": 7, "rows_min": 60, "rows_max": 500,
         "prefix": 1000, "own": 40, "lens": 7},
        # one request's adapter beside Wo of a small model
        {"name": "lora_1b_one_row", "kind": "lora", "dtype": "f32", "rows": 1, "runs": 1, "adapters": 4, "rank": 8,
         "k": DIM_1B, "n1": DIM_1B, "n2": 0, "n3": 0, "swiglu": False, "lens": 8},
        # a decode step of 32 requests beside the QKV projection, most with an adapter of their own
        {"name": "lora_8b_qkv_decode_32", "kind": "lora", "dtype": "bf16", "rows": 32, "runs": 32, "adapters": 24,
         "rank": 16, "k": DIM_8B, "n1": DIM_8B, "n2": KV_8B, "n3": KV_8B, "swiglu": False, "lens": 9},
        # prompts of several tenants beside W1 and W3
        {"name": "lora_8b_swiglu_prompts", "kind": "lora", "dtype": "bf16", "rows": 1100, "runs": 6, "adapters": 5,
         "rank": 64, "k": DIM_8B, "n1": HIDDEN_8B, "n2": 0, "n3": 0, "swiglu": True, "lens": 10},
        # one chat with four tokens drafted from its own text (no draft model)
        {"name": "verify_one_lookup", "kind": "verify", "requests": 1, "drafts_min": 4, "drafts_max": 4, "vocab": VOCAB,
         "temperature": 0.8, "model": False, "masked": 0.0, "lens": 11},
        # a server's step: 32 requests, up to seven drafts of a draft model
        {"name": "verify_32_model", "kind": "verify", "requests": 32, "drafts_min": 0, "drafts_max": 7, "vocab": VOCAB,
         "temperature": 0.7, "model": True, "masked": 0.02, "lens": 12},
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(low * (high / low) ** rng.random()))))


def draw(rng):
    kind = rng.choice(("attention", "attention", "attention", "rope", "lora", "lora", "verify", "verify"))
    lens = rng.randrange(1 << 30)
    if kind in ("attention", "rope"):
        heads = dict(rng.choice((HEADS_1B, HEADS_8B, HEADS_8B)))
        if rng.random() < 0.4:  # a generic decoder
            kv = rng.choice((1, 2, 4, 6))
            heads = {"heads": kv * rng.choice((1, 2, 3, 5, 8)), "kv_heads": kv,
                     "hd": rng.choice((64, 128, 128, 80, 96))}
        form = rng.choice(("decode", "decode", "drafts", "prompts"))
        requests = _log_int(rng, 1, {"decode": 64, "drafts": 24, "prompts": 6}[form])
        low, high = {"decode": (1, 1), "drafts": (1, rng.randint(2, 8)),
                     "prompts": (rng.randint(1, 60), rng.randint(60, 500))}[form]
        return {"kind": kind, **heads, "requests": requests, "rows_min": low, "rows_max": high,
                "prefix": rng.choice((0, _log_int(rng, 1, 1500), _log_int(rng, 16, 1500 if form == "prompts" else 8192))),
                "own": rng.choice((0, _log_int(rng, 1, 1000))), "lens": lens}
    if kind == "lora":
        rows = _log_int(rng, 1, 1100)
        return {"kind": kind, "dtype": rng.choice(("bf16", "bf16", "f32")), "rows": rows,
                "runs": rows if rows <= 64 and rng.random() < 0.7 else rng.randint(1, min(rows, 12)),
                "adapters": rng.randint(1, 32), "rank": rng.choice((4, 8, 12, 16, 16, 32, 64)),
                "k": 8 * _log_int(rng, 32, 512) if rng.random() < 0.8 else _log_int(rng, 200, 3000),
                "n1": 8 * _log_int(rng, 32, 1024), "n2": rng.choice((0, 0, _log_int(rng, 100, 1024))), "n3": 0,
                "swiglu": rng.random() < 0.3, "lens": lens}
    model = rng.random() < 0.6
    return {"kind": kind, "requests": _log_int(rng, 1, 32), "drafts_min": rng.randint(0, 2),
            "drafts_max": rng.randint(2, 7), "vocab": _log_int(rng, 300, VOCAB) if rng.random() < 0.5 else VOCAB,
            "temperature": rng.choice((0.0, 0.3, 0.7, 1.0, 1.5)), "model": model,
            "masked": rng.choice((0.0, 0.0, 0.3)), "lens": lens}


# ---- inputs ------------------------------------------------------------------------------------------------------


class State:
    pass


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(g, *shape, std=1.0):
    return torch.randn(*shape, generator=g, device="cuda").mul_(std)


def _ints(values):
    return torch.tensor(list(values), dtype=torch.int32, device="cuda")


def _requests(c):
    """The batch's first rows, own lengths and cache slots: the case's, whatever the seed of the values."""
    rng = random.Random(c["lens"])
    start, length = [0], []
    for _ in range(c["requests"]):
        start.append(start[-1] + rng.randint(c["rows_min"], c["rows_max"]))
        length.append(rng.randint(c["own"] // 4, c["own"]))
    slots = c["requests"] + 2  # a server's caches: some are free
    return start, length, rng.sample(range(slots), c["requests"]), slots, (c["own"] + c["rows_max"] + 63) // 64 * 64


def _caches(c, g, slots, seq):
    kv, hd = c["kv_heads"], c["hd"]
    return _randn(g, slots, kv, seq, hd), _randn(g, slots, kv, seq, hd)


def _prepare_requests(c, seed):
    g, st = _generator(seed), State()
    st.start, st.length, st.slot, st.slots, st.seq = _requests(c)
    rows, kv, hd = st.start[-1], c["kv_heads"], c["hd"]
    st.rows = rows
    st.start_dev, st.length_dev, st.slot_dev = _ints(st.start), _ints(st.length), _ints(st.slot)
    st.q = _randn(g, rows, c["heads"] * hd, std=1.3)
    st.key, st.value = _caches(c, g, st.slots, st.seq)
    st.prefix_seq = (c["prefix"] + 64) // 64 * 64
    if c["kind"] == "attention":
        st.prefix_key, st.prefix_value = _randn(g, kv, st.prefix_seq, hd), _randn(g, kv, st.prefix_seq, hd)
    else:
        st.k, st.v = _randn(g, rows, kv * hd), _randn(g, rows, kv * hd)
        freq = 1.0 / 500000.0 ** (torch.arange(0, hd, 2, dtype=torch.float64, device="cuda") / hd)
        angle = torch.arange(c["prefix"] + st.seq, dtype=torch.float64, device="cuda")[:, None] * freq
        cos, sin = torch.cos(angle), torch.sin(angle)
        st.table = torch.cat((cos.repeat_interleave(2, 1), torch.stack((-sin, sin), -1).reshape(-1, hd)), 1).float()
    st.out = torch.empty_like(st.q)
    return st


def _adapter_of_rows(c):
    """Rows in runs (a request's rows lie together), each run with one adapter or none."""
    rng = random.Random(c["lens"])
    cuts = sorted(rng.sample(range(1, c["rows"]), c["runs"] - 1)) if c["rows"] > 1 else []
    ids = []
    for first, last in zip([0] + cuts, cuts + [c["rows"]]):
        ids += [-1 if rng.random() < 0.1 and c["rows"] > 1 else rng.randrange(c["adapters"])] * (last - first)
    return ids


def _prepare_lora(c, seed):
    g, st = _generator(seed), State()
    m, k, rank, count = c["rows"], c["k"], c["rank"], c["adapters"]
    dtype = torch.bfloat16 if c["dtype"] == "bf16" else torch.float32
    st.ids = _ints(_adapter_of_rows(c))
    st.x = _randn(g, m, k)
    st.scale = torch.rand(count, generator=g, device="cuda") + 0.5

    def pair(n):
        return (_randn(g, count, rank, k, std=k ** -0.5).to(dtype), _randn(g, count, n, rank, std=rank ** -0.5).to(dtype))

    st.segments = []
    for n in (c["n1"], c["n2"], c["n3"]):
        if n:
            st.segments.append({"n": n, "base": _randn(g, m, n), "ab": pair(n), "c": torch.empty(m, n, device="cuda"),
                                "base3": _randn(g, m, n) if c["swiglu"] else None,
                                "ab3": pair(n) if c["swiglu"] else None})
    return st


def _drafts(c):
    rng = random.Random(c["lens"])
    start = [0]
    for _ in range(c["requests"]):
        start.append(start[-1] + 1 + rng.randint(min(c["drafts_min"], c["drafts_max"]), c["drafts_max"]))
    return start


def _prepare_verify(c, seed):
    g, st = _generator(seed), State()
    start, vocab = _drafts(c), c["vocab"]
    rows = start[-1]
    st.start, st.rows, st.start_dev = start, rows, _ints(start)
    st.logits = _randn(g, rows, vocab, std=3.0)
    if c["masked"]:  # tokens that a filter or a grammar took out
        st.logits.masked_fill_(torch.rand(rows, vocab, generator=g, device="cuda") < c["masked"], float("-inf"))
        st.logits[:, 0] = 1.0
    st.draft = st.logits + _randn(g, rows, vocab, std=0.7)
    # row i + 1's token: drawn from row i of the draft
    noise = torch.rand(rows, vocab, generator=g, device="cuda").clamp_(1e-9, 1 - 1e-7).log_().neg_().log_().neg_()
    drawn = (st.draft / max(c["temperature"], 0.3) + noise).argmax(1)
    st.tokens = torch.cat((drawn.new_zeros(1), drawn[:-1])).to(torch.int32)
    if not c["model"]:
        st.draft = None
    st.uniform = torch.rand(rows, 2, generator=g, device="cuda")
    st.accepted = torch.empty(c["requests"], dtype=torch.int32, device="cuda")
    st.next = torch.empty_like(st.accepted)
    return st


def prepare(case, seed):
    st = {"lora": _prepare_lora, "verify": _prepare_verify}.get(case["kind"], _prepare_requests)(case, seed)
    st.case = case
    if own:
        st.call = _OWN[case["kind"]](st, case)
    return st


# ---- the library's calls -----------------------------------------------------------------------------------------


def _library():
    pkg = os.path.join(ROOT, "llama3.x.c_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import llama_hip

    return llama_hip, llama_hip.load()


def _batch(lh, st, c):
    return lh.RequestBatch(lh.ptr(st.start_dev), lh.ptr(st.length_dev), lh.ptr(st.slot_dev), c["requests"], st.rows,
                           c["prefix"], st.prefix_seq, st.seq, st.slots)


def _own_attention(st, c):
    lh, lib = _library()
    batch = _batch(lh, st, c)
    args = (lh.ptr(st.out), lh.ptr(st.q), lh.ptr(st.prefix_key), lh.ptr(st.prefix_value), lh.ptr(st.key),
            lh.ptr(st.value), batch, c["heads"], c["kv_heads"], c["hd"])

    def call():
        lib.llhip_attention_requests(*args)
        return st.out

    return call


def _own_rope(st, c):
    lh, lib = _library()
    batch = _batch(lh, st, c)
    args = (lh.ptr(st.out), lh.ptr(st.q), c["heads"] * c["hd"], lh.ptr(st.k), lh.ptr(st.v), c["kv_heads"] * c["hd"],
            lh.ptr(st.table), batch, c["heads"], c["kv_heads"], c["hd"], lh.ptr(st.key), lh.ptr(st.value))

    def call():
        lib.llhip_rope_kv_store_requests(*args)
        return {"q": st.out, "key": st.key, "value": st.value}

    return call


def _own_lora(st, c):
    lh, lib = _library()
    kind = lh.GEMM_SWIGLU if c["swiglu"] else lh.GEMM_ADD
    struct, fn = ((lh.LoraBf16Segment, lib.llhip_lora_bf16) if c["dtype"] == "bf16"
                  else (lh.LoraSegment, lib.llhip_lora_f32))
    segments = (struct * len(st.segments))(*[
        struct(lh.ptr(s["c"]), s["n"], lh.ptr(s["base"]), lh.ptr(s["base3"]), lh.ptr(s["ab"][0]), lh.ptr(s["ab"][1]),
               lh.ptr(s["ab3"][0]) if s["ab3"] else None, lh.ptr(s["ab3"][1]) if s["ab3"] else None, lh.ptr(st.scale),
               s["n"], c["rank"], kind) for s in st.segments])
    args = (lh.ptr(st.x), c["k"], c["rows"], c["k"], lh.ptr(st.ids), c["adapters"], segments, len(st.segments))
    out = [s["c"] for s in st.segments]

    def call():
        fn(*args)
        return out

    return call


def _own_verify(st, c):
    lh, lib = _library()
    args = (lh.ptr(st.accepted), lh.ptr(st.next), lh.ptr(st.logits), c["vocab"],
            lh.ptr(st.draft) if st.draft is not None else None, c["vocab"], lh.ptr(st.tokens), lh.ptr(st.uniform),
            lh.ptr(st.start_dev), c["requests"], st.rows, c["vocab"], c["temperature"])

    def call():
        lib.llhip_verify_drafts(*args)
        return {"accepted": st.accepted, "next": st.next}

    return call


_OWN = {"attention": _own_attention, "rope": _own_rope, "lora": _own_lora, "verify": _own_verify}


# ---- the plain forms ---------------------------------------------------------------------------------------------


def _plain_attention(st, c):
    """The prefix scores of all rows at once; each request's own scores; one softmax over both."""
    nh, nkv, hd, prefix = c["heads"], c["kv_heads"], c["hd"], c["prefix"]
    mul, scale = nh // nkv, 1.0 / math.sqrt(hd)
    out = torch.empty_like(st.q)
    q = st.q.reshape(st.rows, nkv, mul, hd).transpose(0, 1)  # KV head, row, head of the group, dimension
    shared_k = st.prefix_key[:, :prefix].transpose(1, 2).contiguous()
    shared = torch.matmul(q.reshape(nkv, st.rows * mul, hd), shared_k).reshape(nkv, st.rows, mul, prefix) * scale
    for r in range(c["requests"]):
        a, b, before, slot = st.start[r], st.start[r + 1], st.length[r], st.slot[r]
        n = b - a
        if n == 0:
            continue
        seen = before + n
        own_k, own_v = st.key[slot, :, :seen], st.value[slot, :, :seen]
        mine = torch.matmul(q[:, a:b].reshape(nkv, n * mul, hd), own_k.transpose(1, 2).contiguous())
        mine = mine.reshape(nkv, n, mul, seen) * scale
        later = torch.arange(seen, device="cuda")[None, :] > before + torch.arange(n, device="cuda")[:, None]
        mine = mine.masked_fill(later[None, :, None, :], float("-inf"))
        far = shared[:, a:b]
        top = mine.amax(-1, keepdim=True)
        if prefix:
            top = torch.maximum(top, far.amax(-1, keepdim=True))
        mine, far = torch.exp(mine - top), torch.exp(far - top)
        total = mine.sum(-1, keepdim=True) + far.sum(-1, keepdim=True)
        o = torch.matmul(mine.reshape(nkv, n * mul, seen), own_v)
        if prefix:
            o = o + torch.matmul(far.reshape(nkv, n * mul, prefix), st.prefix_value[:, :prefix])
        o = o.reshape(nkv, n, mul, hd) / total
        out[a:b] = o.transpose(0, 1).reshape(n, nh * hd)
    return out


def _plain_rope(st, c):
    """All rows rotated by their positions' table rows, then each request's rows into its slot."""
    nh, nkv, hd, prefix = c["heads"], c["kv_heads"], c["hd"], c["prefix"]
    first = st.start_dev[:-1].long()
    count = st.start_dev[1:].long() - first
    request = torch.repeat_interleave(torch.arange(c["requests"], device="cuda"), count, output_size=st.rows)
    at = st.length_dev.long()[request] + torch.arange(st.rows, device="cuda") - first[request]
    t = st.table[prefix + at]
    cos, sin = t[:, None, 0:hd:2], t[:, None, hd + 1::2]

    def rotate(x, heads):
        x = x.reshape(st.rows, heads, hd // 2, 2)
        a, b = x[..., 0], x[..., 1]
        return torch.stack((a * cos - b * sin, a * sin + b * cos), -1).reshape(st.rows, heads, hd)

    slot = st.slot_dev.long()[request]
    st.key[slot, :, at] = rotate(st.k, nkv)
    st.value[slot, :, at] = st.v.reshape(st.rows, nkv, hd)
    return {"q": rotate(st.q, nh).reshape(st.rows, nh * hd), "key": st.key, "value": st.value}


def _plain_lora(st, c):
    def product(s, ab, base):
        got = base.clone()
        for a in range(c["adapters"]):
            rows = (st.ids == a).nonzero()[:, 0]
            if rows.numel():
                low = torch.matmul(st.x[rows], ab[0][a].float().t())
                got[rows] = base[rows] + st.scale[a] * torch.matmul(low, ab[1][a].float().t())
        return got

    out = []
    for s in st.segments:
        y = product(s, s["ab"], s["base"])
        if s["ab3"]:
            y = y / (1.0 + torch.exp(-y)) * product(s, s["ab3"], s["base3"])
        out.append(y)
    return out


def _softmax64(logits, temperature):
    z = logits.double()
    e = torch.exp((z - z.amax(1, keepdim=True)) / temperature)
    return e / e.sum(1, keepdim=True)


def _plain_verify(st, c):
    """The probabilities of every row in 64 bits (a border that moves turns a token), the first refusal by a running
    product, and the inverse of the stopping rows' running sums."""
    first, last = st.start_dev[:-1].long(), st.start_dev[1:].long() - 1
    count = last - first
    most = int(max(b - a - 1 for a, b in zip(st.start, st.start[1:])))
    step = torch.arange(max(most, 1), device="cuda")
    at = torch.minimum(first[:, None] + step, last[:, None])  # the judging rows, the last one repeated
    drafted = torch.cat((st.tokens[1:], st.tokens[:1])).long()  # row i judges row i + 1's token
    greedy = c["temperature"] == 0.0
    if greedy:
        best = st.logits.argmax(1)
        fine = best == drafted
    else:
        t = float(torch.tensor(c["temperature"], dtype=torch.float32))
        p = _softmax64(st.logits, t)
        px = p.gather(1, drafted[:, None])[:, 0]
        if st.draft is not None:
            q = _softmax64(st.draft, t)
            qx = q.gather(1, drafted[:, None])[:, 0]
        else:
            qx = torch.ones_like(px)
        fine = st.uniform[:, 0].double() * qx < px
    passed = fine[at] & (step < count[:, None])
    accepted = torch.cumprod(passed.long(), 1).sum(1)
    stop = first + accepted
    if greedy:
        return {"accepted": accepted.to(torch.int32), "next": best[stop].to(torch.int32)}
    w = p[stop]
    refused = accepted < count
    if st.draft is not None:
        less = q[stop]
    else:
        less = torch.zeros_like(w).scatter_(1, drafted[stop][:, None], 1.0)
    rest = torch.where(refused[:, None], (w - less).clamp(min=0.0), w)
    empty = rest.sum(1, keepdim=True) <= 0.0
    rest = torch.where(empty, w, rest)
    running = torch.cumsum(rest, 1)
    over = running > st.uniform[stop, 1].double()[:, None] * running[:, -1:]
    return {"accepted": accepted.to(torch.int32), "next": over.to(torch.int8).argmax(1).to(torch.int32)}


_PLAIN = {"attention": _plain_attention, "rope": _plain_rope, "lora": _plain_lora, "verify": _plain_verify}


def run(state):
    if own:
        return state.call()
    return _PLAIN[state.case["kind"]](state, state.case)


# ---- what a pass cannot do without -------------------------------------------------------------------------------


def work(case):
    c = case
    if c["kind"] in ("attention", "rope"):
        start, length, _, _, _ = _requests(c)
        rows, dq, dkv = start[-1], c["heads"] * c["hd"], c["kv_heads"] * c["hd"]
        if c["kind"] == "rope":
            return {"bytes": 4 * rows * (2 * dq + 4 * dkv + 2 * c["hd"]), "flops": 3 * rows * (dq + dkv)}
        pairs = own_positions = 0
        for r in range(c["requests"]):
            n = start[r + 1] - start[r]
            own_positions += length[r] + n if n else 0
            pairs += sum(c["prefix"] + length[r] + j + 1 for j in range(n))
        return {"bytes": 8 * dkv * (c["prefix"] + own_positions) + 8 * rows * dq, "flops": 4 * dq * pairs}
    if c["kind"] == "lora":
        ids = _adapter_of_rows(c)
        used, active = len(set(ids) - {-1}), sum(i >= 0 for i in ids)
        size, parts = 2 if c["dtype"] == "bf16" else 4, 2 if c["swiglu"] else 1
        nbytes, flops = 4 * c["rows"] * c["k"], 0
        for n in (c["n1"], c["n2"], c["n3"]):
            if n:
                nbytes += parts * (used * size * c["rank"] * (c["k"] + n) + 4 * c["rows"] * n) + 4 * c["rows"] * n
                flops += parts * 2 * active * c["rank"] * (c["k"] + n)
        return {"bytes": nbytes, "flops": flops}
    rows = _drafts(c)[-1]
    read = rows + (rows - c["requests"] if c["model"] and c["temperature"] else 0)
    return {"bytes": 4 * read * c["vocab"], "flops": 4 * read * c["vocab"]}


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------


def _exact_attention(st, c):
    nh, nkv, hd, prefix = c["heads"], c["kv_heads"], c["hd"], c["prefix"]
    mul = nh // nkv
    out = torch.zeros(st.rows, nh, hd, dtype=torch.float64, device="cuda")
    for r in range(c["requests"]):
        a, b, before = st.start[r], st.start[r + 1], st.length[r]
        seen = before + b - a
        for g in range(nkv):
            k = torch.cat((st.prefix_key[g, :prefix], st.key[st.slot[r], g, :seen])).double()
            v = torch.cat((st.prefix_value[g, :prefix], st.value[st.slot[r], g, :seen])).double()
            x = st.q[a:b].double().reshape(b - a, nh, hd)[:, g * mul:(g + 1) * mul]
            s = (x.reshape(-1, hd) @ k.t().contiguous() / hd ** 0.5).reshape(b - a, mul, prefix + seen)
            visible = prefix + before + torch.arange(b - a, device="cuda") + 1
            hidden = torch.arange(prefix + seen, device="cuda")[None, :] >= visible[:, None]
            w = torch.softmax(s.masked_fill(hidden[:, None, :], float("-inf")), -1)
            out[a:b, g * mul:(g + 1) * mul] = (w.reshape(-1, prefix + seen) @ v).reshape(b - a, mul, hd)
    return out.reshape(st.rows, nh * hd)


def _exact_rope(st, c):
    hd = c["hd"]
    key, value = st.key.double(), st.value.double()
    q = torch.empty(st.rows, c["heads"] * hd, dtype=torch.float64, device="cuda")
    for r in range(c["requests"]):
        rows, at = slice(st.start[r], st.start[r + 1]), st.length[r]
        n = st.start[r + 1] - st.start[r]
        t = st.table[c["prefix"] + at:c["prefix"] + at + n].double()

        def turn(x, heads):
            x = x[rows].double().reshape(n, heads, hd)
            pairs = x.reshape(n, heads, hd // 2, 2).flip(-1).reshape(n, heads, hd)
            return x * t[:, None, :hd] + pairs * t[:, None, hd:]

        q[rows] = turn(st.q, c["heads"]).reshape(n, -1)
        key[st.slot[r], :, at:at + n] = turn(st.k, c["kv_heads"]).transpose(0, 1)
        value[st.slot[r], :, at:at + n] = st.v[rows].double().reshape(n, -1, hd).transpose(0, 1)
    return {"q": q, "key": key, "value": value}


def _exact_lora(st, c):
    ids = _adapter_of_rows(c)
    cuts = [i for i in range(len(ids)) if i == 0 or ids[i] != ids[i - 1]] + [len(ids)]
    x = st.x.double()

    def with_adapters(base, ab):
        y = base.double()
        for first, last in zip(cuts, cuts[1:]):
            if ids[first] >= 0:
                a, b = ab[0][ids[first]].double(), ab[1][ids[first]].double()
                y[first:last] += st.scale[ids[first]].double() * (x[first:last] @ a.t().contiguous()) @ b.t().contiguous()
        return y

    out = []
    for s in st.segments:
        y = with_adapters(s["base"], s["ab"])
        if c["swiglu"]:
            y = y * torch.sigmoid(y) * with_adapters(s["base3"], s["ab3"])
        out.append(y)
    return out


def _exact_verify(st, c):
    """Request by request and draft by draft, as one would check them by hand."""
    t = float(torch.tensor(c["temperature"], dtype=torch.float32))

    def distribution(logits):
        return torch.softmax(logits.double() / t, 0)

    tokens, uniform = st.tokens.tolist(), st.uniform.double().tolist()
    accepted, following = [], []
    for a, b in zip(st.start, st.start[1:]):
        row = a
        if t == 0.0:
            best = st.logits[a:b].cpu().numpy().argmax(1)
            while row + 1 < b and best[row - a] == tokens[row + 1]:
                row += 1
            token = int(best[row - a])
        else:
            while True:
                p = distribution(st.logits[row])
                if row + 1 == b:
                    break
                x = tokens[row + 1]
                if st.draft is not None:
                    q = distribution(st.draft[row])
                else:
                    q = torch.zeros_like(p)
                    q[x] = 1.0
                if uniform[row][0] * float(q[x]) < float(p[x]):
                    row += 1
                    continue
                rest = torch.clamp(p - q, min=0.0)
                p = rest if float(rest.sum()) > 0.0 else p
                break
            running = torch.cumsum(p, 0)
            token = int((running <= uniform[row][1] * running[-1]).sum())
        accepted.append(row - a)
        following.append(token)
    return {"accepted": _ints(accepted), "next": _ints(following)}


def exact(case, seed):
    c = case
    if c["kind"] == "lora":
        return _exact_lora(_prepare_lora(c, seed), c)
    if c["kind"] == "verify":
        return _exact_verify(_prepare_verify(c, seed), c)
    st = _prepare_requests(c, seed)
    return (_exact_attention if c["kind"] == "attention" else _exact_rope)(st, c)
