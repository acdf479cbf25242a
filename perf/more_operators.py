"""The operators of a paged key-value cache and of scoring, as cases that can be timed and checked one by one.

  append     llhip_rope_kv_append_paged: RoPE of the rows at their requests' positions (behind a norm of each head where the
             model has one), and their keys and values into the requests' pages.
  attention  llhip_attention_paged: each request's rows attend to the positions that its pages hold.
  logprobs   llhip_token_logprobs: log probabilities of given tokens, the rows' entropies and their likeliest tokens.

run() computes them in elementary torch operations, or, where `own` is set, through the library's entry points: those are
queued on the library's own stream, so what run() returns is read behind llhip_synchronize or a synchronization of the
device. exact() is written from the definitions, in float64.
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
EPSILON = 1e-5


def listed():
    return [
        # one chat request, its first tokens: latency
        {"name": "attention_1b_first_tokens", "kind": "attention", **HEADS_1B, "type": "bf16", "page": 16, "requests": 1,
         "rows_min": 1, "rows_max": 1, "shared": 0, "own": 37, "lens": 1},
        # a server's decode step: 32 chats, each at its own length
        {"name": "attention_8b_decode_32", "kind": "attention", **HEADS_8B, "type": "bf16", "page": 16, "requests": 32,
         "rows_min": 1, "rows_max": 1, "shared": 0, "own": 3000, "lens": 2},
        # a full server of long chats
        {"name": "attention_8b_decode_64_long", "kind": "attention", **HEADS_8B, "type": "bf16", "page": 64, "requests": 64,
         "rows_min": 1, "rows_max": 1, "shared": 0, "own": 9000, "lens": 3},
        # one question about a book, in an F32 cache: the one row's positions are all the parallel work there is
        {"name": "attention_8b_one_long_f32", "kind": "attention", **HEADS_8B, "type": "f32", "page": 128, "requests": 1,
         "rows_min": 1, "rows_max": 1, "shared": 0, "own": 60000, "lens": 4},
        # up to six drafted rows a request, behind a system prompt whose pages all of them name
        {"name": "attention_8b_drafts_16", "kind": "attention", **HEADS_8B, "type": "f32", "page": 32, "requests": 16,
         "rows_min": 2, "rows_max": 7, "shared": 512, "own": 1500, "lens": 5},
        # chunks of prompts read in one batch, behind what their pages hold already
        {"name": "attention_8b_prompts", "kind": "attention", **HEADS_8B, "type": "bf16", "page": 64, "requests": 5,
         "rows_min": 90, "rows_max": 600, "shared": 0, "own": 2000, "lens": 6},
        # a decode step's rows into the pages
        {"name": "append_8b_decode_32", "kind": "append", **HEADS_8B, "type": "bf16", "page": 16, "requests": 32,
         "rows_min": 1, "rows_max": 1, "shared": 0, "own": 1000, "norm": False, "lens": 7},
        # prompts of a model that norms its heads
        {"name": "append_1b_norm_prompts", "kind": "append", **HEADS_1B, "type": "f32", "page": 32, "requests": 7,
         "rows_min": 60, "rows_max": 500, "shared": 256, "own": 200, "norm": True, "lens": 8},
        # the same into BF16 pages, larger
        {"name": "append_8b_norm_prompts", "kind": "append", **HEADS_8B, "type": "bf16", "page": 64, "requests": 6,
         "rows_min": 300, "rows_max": 900, "shared": 0, "own": 300, "norm": True, "lens": 9},
        # the token that one chat answered, with its five likeliest
        {"name": "logprobs_one_row", "kind": "logprobs", "rows": 1, "vocab": VOCAB, "top": 5, "entropy": False,
         "temperature": 1.0, "masked": 0.0, "lens": 10},
        # a server's step, twenty alternatives for everybody
        {"name": "logprobs_64_top_20", "kind": "logprobs", "rows": 64, "vocab": VOCAB, "top": 20, "entropy": True,
         "temperature": 0.7, "masked": 0.02, "lens": 11},
        # a prompt's tokens scored
        {"name": "logprobs_prompt_1000", "kind": "logprobs", "rows": 1000, "vocab": VOCAB, "top": 0, "entropy": True,
         "temperature": 1.0, "masked": 0.0, "lens": 12},
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(low * (high / low) ** rng.random()))))


def draw(rng):
    kind = rng.choice(("attention", "attention", "attention", "append", "append", "logprobs", "logprobs"))
    lens = rng.randrange(1 << 30)
    if kind == "logprobs":
        rows = _log_int(rng, 1, 1000)
        return {"kind": kind, "rows": rows, "vocab": _log_int(rng, 300, VOCAB) if rng.random() < 0.5 else VOCAB,
                "top": rng.choice((0, 1, 2, 5, 10, 20, 32)), "entropy": rng.random() < 0.6,
                "temperature": rng.choice((1.0, 1.0, 0.3, 0.7, 1.5)), "masked": rng.choice((0.0, 0.0, 0.3)), "lens": lens}
    heads = dict(rng.choice((HEADS_1B, HEADS_8B, HEADS_8B)))
    if rng.random() < 0.4:  # a generic decoder
        kv = rng.choice((1, 2, 4, 6))
        heads = {"heads": kv * rng.choice((1, 2, 3, 5, 8)), "kv_heads": kv, "hd": rng.choice((64, 128, 128, 80, 96, 256))}
    form = rng.choice(("decode", "decode", "drafts", "prompts"))
    requests = _log_int(rng, 1, {"decode": 64, "drafts": 24, "prompts": 6}[form])
    low, high = {"decode": (1, 1), "drafts": (1, rng.randint(2, 8)),
                 "prompts": (rng.randint(1, 60), rng.randint(60, 500))}[form]
    page = rng.choice((8, 16, 16, 32, 64, 128))
    c = {"kind": kind, **heads, "type": rng.choice(("bf16", "bf16", "f32")), "page": page, "requests": requests,
         "rows_min": low, "rows_max": high, "shared": page * rng.choice((0, 0, rng.randint(1, 512 // page + 1))),
         "own": rng.choice((0 if form == "prompts" else 3, _log_int(rng, 1, 1000),
                            _log_int(rng, 16, 1500 if form == "prompts" else 4000))), "lens": lens}
    if kind == "append":
        c["norm"] = rng.random() < 0.5
        c["own"] = min(c["own"], 1000)
    return c


# ---- inputs ------------------------------------------------------------------------------------------------------


class State:
    pass


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(g, *shape, std=1.0, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda", dtype=dtype).mul_(std)


def _ints(values):
    return torch.tensor(list(values), dtype=torch.int32, device="cuda")


def _requests(c):
    """The batch's first rows, the positions before them, and the pages of every request: the case's, whatever the seed of
    the values. The first pages of all requests are the shared prompt's; the others lie in the order that a server's
    allocator came to them, and some of the pool's are free."""
    rng = random.Random(c["lens"])
    start, length = [0], []
    for _ in range(c["requests"]):
        start.append(start[-1] + rng.randint(c["rows_min"], c["rows_max"]))
        length.append(c["shared"] + rng.randint(c["own"] // 4, c["own"]))
    page, common = c["page"], c["shared"] // c["page"]
    need = [(n + b - a + page - 1) // page for n, a, b in zip(length, start, start[1:])]
    most = max(need) + 2
    pool = common + sum(n - common for n in need) + 8
    order = list(range(pool))
    rng.shuffle(order)
    first, at, table = order[:common], common, []
    for n in need:
        mine = first + order[at:at + n - common]
        at += n - common
        table.append(mine + [-1] * (most - n))
    return start, length, table, pool


def _cache_type(c):
    return torch.bfloat16 if c["type"] == "bf16" else torch.float32


def _prepare_requests(c, seed):
    g, st = _generator(seed), State()
    st.start, st.length, st.table, st.pool = _requests(c)
    rows, heads, kv, hd = st.start[-1], c["heads"], c["kv_heads"], c["hd"]
    st.rows, st.max_pages = rows, len(st.table[0])
    st.seq = st.max_pages * c["page"]
    st.start_dev, st.length_dev = _ints(st.start), _ints(st.length)
    st.pages = torch.tensor(st.table, dtype=torch.int32, device="cuda")
    shape = (st.pool, kv, c["page"], hd)
    st.key, st.value = (_randn(g, *shape, dtype=_cache_type(c)) for _ in range(2))
    st.q = _randn(g, rows, heads * hd, std=1.3)
    if c["kind"] == "append":
        st.k, st.v = _randn(g, rows, kv * hd), _randn(g, rows, kv * hd)
        freq = 1.0 / 500000.0 ** (torch.arange(0, hd, 2, dtype=torch.float64, device="cuda") / hd)
        angle = torch.arange(st.seq, dtype=torch.float64, device="cuda")[:, None] * freq
        cos, sin = torch.cos(angle), torch.sin(angle)
        st.rope = torch.cat((cos.repeat_interleave(2, 1), torch.stack((-sin, sin), -1).reshape(-1, hd)), 1).float()
        st.q_norm = st.k_norm = None
        if c["norm"]:
            st.q_norm, st.k_norm = (torch.rand(hd, generator=g, device="cuda") + 0.5 for _ in range(2))
    st.out = torch.empty_like(st.q)
    return st


def _prepare_logprobs(c, seed):
    g, st = _generator(seed), State()
    rows, vocab = c["rows"], c["vocab"]
    st.logits = _randn(g, rows, vocab, std=3.0)
    if c["masked"]:  # tokens that a filter or a grammar took out
        st.logits.masked_fill_(torch.rand(rows, vocab, generator=g, device="cuda") < c["masked"], float("-inf"))
        st.logits[:, 0] = 1.0
    noise = torch.rand(rows, vocab, generator=g, device="cuda").clamp_(1e-9, 1 - 1e-7).log_().neg_().log_().neg_()
    st.tokens = (st.logits / c["temperature"] + noise).argmax(1).to(torch.int32)
    rng = random.Random(c["lens"])
    ends = [i for i in range(rows) if rows > 4 and rng.random() < 0.02]  # rows with no token behind them
    st.tokens[ends] = -1
    st.logprob = torch.empty(rows, device="cuda")
    st.entropy = torch.empty(rows, device="cuda") if c["entropy"] else None
    st.top_token = torch.empty(rows, c["top"], dtype=torch.int32, device="cuda")
    st.top_logprob = torch.empty(rows, c["top"], device="cuda")
    return st


def prepare(case, seed):
    st = (_prepare_logprobs if case["kind"] == "logprobs" else _prepare_requests)(case, seed)
    st.case = case
    if own:
        st.call = _OWN[case["kind"]](st, case)
        torch.cuda.synchronize()  # the inputs were made on torch's stream; the library has its own
    return st


# ---- the library's calls -----------------------------------------------------------------------------------------


def _library():
    pkg = os.path.join(ROOT, "llama3.x.c_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import llama_hip

    return llama_hip, llama_hip.load()


def _batch(lh, st, c):
    kind = lh.PAGE_BF16 if c["type"] == "bf16" else lh.PAGE_F32
    return lh.PagedBatch(lh.ptr(st.start_dev), lh.ptr(st.length_dev), lh.ptr(st.pages), c["requests"], st.rows,
                         st.max_pages, c["page"], st.pool, st.seq, kind)


def _own_attention(st, c):
    lh, lib = _library()
    batch = _batch(lh, st, c)
    args = (lh.ptr(st.out), lh.ptr(st.q), c["heads"] * c["hd"], lh.ptr(st.key), lh.ptr(st.value), batch, c["heads"],
            c["kv_heads"], c["hd"])

    def call():
        lib.llhip_attention_paged(*args)
        return st.out

    return call


def _own_append(st, c):
    lh, lib = _library()
    batch = _batch(lh, st, c)
    args = (lh.ptr(st.out), c["heads"] * c["hd"], lh.ptr(st.q), c["heads"] * c["hd"], lh.ptr(st.k), lh.ptr(st.v),
            c["kv_heads"] * c["hd"], lh.ptr(st.rope), lh.ptr(st.q_norm), lh.ptr(st.k_norm), EPSILON, batch, c["heads"],
            c["kv_heads"], c["hd"], lh.ptr(st.key), lh.ptr(st.value))

    def call():
        lib.llhip_rope_kv_append_paged(*args)
        return {"q": st.out, "key": st.key, "value": st.value}

    return call


def _scores(st):
    out = {"logprob": st.logprob}
    if st.entropy is not None:
        out["entropy"] = st.entropy
    if st.top_token.shape[1]:
        out["top_token"], out["top_logprob"] = st.top_token, st.top_logprob
    return out


def _own_logprobs(st, c):
    lh, lib = _library()
    top = c["top"]
    args = (lh.ptr(st.logprob), lh.ptr(st.entropy), lh.ptr(st.top_token) if top else None,
            lh.ptr(st.top_logprob) if top else None, top, lh.ptr(st.logits), c["vocab"], lh.ptr(st.tokens), c["rows"],
            c["vocab"], c["temperature"])
    out = _scores(st)

    def call():
        lib.llhip_token_logprobs(*args)
        return out

    return call


_OWN = {"attention": _own_attention, "append": _own_append, "logprobs": _own_logprobs}


# ---- the plain forms ---------------------------------------------------------------------------------------------


def _plain_attention(st, c):
    """Request by request: its pages gathered, all KV heads' scores in one product, the softmax, the values' product."""
    nh, kv, hd = c["heads"], c["kv_heads"], c["hd"]
    mul, scale = nh // kv, 1.0 / math.sqrt(hd)
    out = torch.empty_like(st.q)
    for r in range(c["requests"]):
        a, b, before = st.start[r], st.start[r + 1], st.length[r]
        n, seen = b - a, before + b - a
        mine = st.pages[r, :(seen + c["page"] - 1) // c["page"]].long()
        k = st.key[mine].float().transpose(0, 1).reshape(kv, -1, hd)[:, :seen]
        v = st.value[mine].float().transpose(0, 1).reshape(kv, -1, hd)[:, :seen]
        q = st.q[a:b].reshape(n, kv, mul, hd).transpose(0, 1).reshape(kv, n * mul, hd)
        s = (torch.matmul(q, k.transpose(1, 2).contiguous()) * scale).reshape(kv, n, mul, seen)
        if n > 1:
            later = torch.arange(seen, device="cuda")[None, :] > before + torch.arange(n, device="cuda")[:, None]
            s = s.masked_fill(later[None, :, None, :], float("-inf"))
        e = torch.exp(s - s.amax(-1, keepdim=True))
        o = torch.matmul(e.reshape(kv, n * mul, seen), v.contiguous()).reshape(kv, n, mul, hd)
        o = o / e.sum(-1, keepdim=True)
        out[a:b] = o.transpose(0, 1).reshape(n, nh * hd)
    return out


def _plain_append(st, c):
    """All rows normed and rotated by their positions' table rows, then keys and values into their pages."""
    nh, kv, hd, page = c["heads"], c["kv_heads"], c["hd"], c["page"]
    first = st.start_dev[:-1].long()
    count = st.start_dev[1:].long() - first
    request = torch.repeat_interleave(torch.arange(c["requests"], device="cuda"), count, output_size=st.rows)
    at = st.length_dev.long()[request] + torch.arange(st.rows, device="cuda") - first[request]
    t = st.rope[at]
    cos, sin = t[:, None, 0:hd:2], t[:, None, hd + 1::2]

    def rotate(x, heads, weight):
        x = x.reshape(st.rows, heads, hd)
        if weight is not None:
            x = weight * (x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPSILON))
        x = x.reshape(st.rows, heads, hd // 2, 2)
        a, b = x[..., 0], x[..., 1]
        return torch.stack((a * cos - b * sin, a * sin + b * cos), -1).reshape(st.rows, heads, hd)

    where = st.pages[request, at // page].long()
    st.key[where, :, at % page] = rotate(st.k, kv, st.k_norm).to(st.key.dtype)
    st.value[where, :, at % page] = st.v.reshape(st.rows, kv, hd).to(st.value.dtype)
    return {"q": rotate(st.q, nh, st.q_norm).reshape(st.rows, nh * hd), "key": st.key, "value": st.value}


def _plain_logprobs(st, c):
    """The rows' softmax statistics in passes over the logits; the likeliest tokens by keys that hold a logit's order in
    their upper bits and, for equal logits, the lower token's precedence in the lower ones."""
    t = float(torch.tensor(c["temperature"], dtype=torch.float32))
    z = (st.logits - st.logits.amax(1, keepdim=True)) / t
    e = torch.exp(z)
    whole = e.sum(1, keepdim=True)
    log = torch.log(whole)
    given = z.gather(1, st.tokens.clamp(min=0).long()[:, None]) - log
    out = {"logprob": torch.where(st.tokens < 0, torch.zeros_like(given[:, 0]), given[:, 0])}
    if c["entropy"]:
        out["entropy"] = (log - (z.clamp(min=-1e4) * e).sum(1, keepdim=True) / whole)[:, 0]
    if c["top"]:
        bits = st.logits.view(torch.int32).long()
        order = torch.where(bits < 0, -2147483648 - bits, bits)
        keys = order * (1 << 22) + (c["vocab"] - 1 - torch.arange(c["vocab"], device="cuda"))
        best = torch.topk(keys, c["top"], 1).values
        token = c["vocab"] - 1 - (best & ((1 << 22) - 1))
        out["top_token"] = token.to(torch.int32)
        out["top_logprob"] = z.gather(1, token) - log
    return out


_PLAIN = {"attention": _plain_attention, "append": _plain_append, "logprobs": _plain_logprobs}


def run(state):
    if own:
        return state.call()
    return _PLAIN[state.case["kind"]](state, state.case)


# ---- what a pass cannot do without -------------------------------------------------------------------------------


def work(case):
    c = case
    if c["kind"] == "logprobs":
        return {"bytes": 4 * c["rows"] * (c["vocab"] + 2 * c["top"] + 2), "flops": 4 * c["rows"] * c["vocab"]}
    start, length, _, _ = _requests(c)
    rows, dq, dkv = start[-1], c["heads"] * c["hd"], c["kv_heads"] * c["hd"]
    size = 2 if c["type"] == "bf16" else 4
    if c["kind"] == "append":
        return {"bytes": rows * (8 * dq + 2 * dkv * (4 + size) + 8 * c["hd"]),
                "flops": rows * (3 * (dq + dkv) + (4 * (dq + dkv) if c["norm"] else 0))}
    pairs, positions = 0, c["shared"]
    for r in range(c["requests"]):
        n = start[r + 1] - start[r]
        positions += length[r] - c["shared"] + n
        pairs += sum(length[r] + j + 1 for j in range(n))
    return {"bytes": 2 * size * dkv * positions + 8 * rows * dq, "flops": 4 * dq * pairs}


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------


def _exact_attention(st, c):
    nh, kv, hd, page = c["heads"], c["kv_heads"], c["hd"], c["page"]
    mul = nh // kv
    out = torch.zeros(st.rows, nh, hd, dtype=torch.float64, device="cuda")
    for r in range(c["requests"]):
        a, b, before = st.start[r], st.start[r + 1], st.length[r]
        seen = before + b - a
        position = torch.arange(seen, device="cuda")
        lies = st.pages[r].long()[position // page]
        visible = before + torch.arange(b - a, device="cuda") + 1
        hidden = position[None, :] >= visible[:, None]
        for g in range(kv):
            k = st.key[lies, g, position % page].double()
            v = st.value[lies, g, position % page].double()
            x = st.q[a:b].double().reshape(b - a, nh, hd)[:, g * mul:(g + 1) * mul]
            s = (x.reshape(-1, hd) @ k.t().contiguous() / hd ** 0.5).reshape(b - a, mul, seen)
            w = torch.softmax(s.masked_fill(hidden[:, None, :], float("-inf")), -1)
            out[a:b, g * mul:(g + 1) * mul] = (w.reshape(-1, seen) @ v).reshape(b - a, mul, hd)
    return out.reshape(st.rows, nh * hd)


def _exact_append(st, c):
    hd, page = c["hd"], c["page"]
    key, value = st.key.double(), st.value.double()
    q = torch.empty(st.rows, c["heads"] * hd, dtype=torch.float64, device="cuda")
    for r in range(c["requests"]):
        rows, at = slice(st.start[r], st.start[r + 1]), st.length[r]
        n = st.start[r + 1] - st.start[r]
        t = st.rope[at:at + n].double()

        def turn(x, heads, weight):
            x = x[rows].double().reshape(n, heads, hd)
            if weight is not None:
                x = x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + float(torch.tensor(EPSILON))) * weight.double()
            pairs = x.reshape(n, heads, hd // 2, 2).flip(-1).reshape(n, heads, hd)
            return x * t[:, None, :hd] + pairs * t[:, None, hd:]

        q[rows] = turn(st.q, c["heads"], st.q_norm).reshape(n, -1)
        k, v = turn(st.k, c["kv_heads"], st.k_norm), st.v[rows].double().reshape(n, -1, hd)
        done = 0
        while done < n:  # page by page
            p, within = st.table[r][(at + done) // page], (at + done) % page
            m = min(page - within, n - done)
            key[p, :, within:within + m] = k[done:done + m].transpose(0, 1)
            value[p, :, within:within + m] = v[done:done + m].transpose(0, 1)
            done += m
    return {"q": q, "key": key, "value": value}


def _exact_logprobs(st, c):
    t = float(torch.tensor(c["temperature"], dtype=torch.float32))
    tokens = st.tokens.long()
    logprob = torch.zeros(c["rows"], dtype=torch.float64, device="cuda")
    entropy = torch.zeros_like(logprob)
    top_token = torch.zeros(c["rows"], c["top"], dtype=torch.int32, device="cuda")
    top_logprob = torch.zeros(c["rows"], c["top"], dtype=torch.float64, device="cuda")
    for i in range(0, c["rows"], 64):
        rows = slice(i, min(i + 64, c["rows"]))
        log = torch.log_softmax(st.logits[rows].double() / t, 1)
        given = tokens[rows]
        logprob[rows] = torch.where(given < 0, 0.0, log.gather(1, given.clamp(min=0)[:, None])[:, 0])
        p = log.exp()
        entropy[rows] = -torch.where(p > 0.0, p * log, torch.zeros_like(p)).sum(1)
        if c["top"]:
            order = torch.sort(st.logits[rows], dim=1, descending=True, stable=True).indices[:, :c["top"]]
            top_token[rows], top_logprob[rows] = order.to(torch.int32), log.gather(1, order)
    out = {"logprob": logprob}
    if c["entropy"]:
        out["entropy"] = entropy
    if c["top"]:
        out["top_token"], out["top_logprob"] = top_token, top_logprob
    return out


def exact(case, seed):
    c = case
    if c["kind"] == "logprobs":
        return _exact_logprobs(_prepare_logprobs(c, seed), c)
    st = _prepare_requests(c, seed)
    return (_exact_attention if c["kind"] == "attention" else _exact_append)(st, c)
