"""Plain float64 forms of the operators over pages and of the scoring, and their error bounds, shared by their tests."""
import numpy as np

import llama_hip as lh
from tests.requests_util import U

F = np.float32


def to_bf16(x):
    """The BF16 bits nearest to float32 values, ties to even (finite values, infinities and NaN as they are)."""
    b = np.ascontiguousarray(x, F).view(np.uint32).astype(np.uint64)
    rounded = ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), rounded)


def values(cache):
    """A cache's values as float32: uint16 ones are BF16 bits."""
    return (cache.astype(np.uint32) << 16).view(F) if cache.dtype == np.uint16 else cache


class Pages:
    """A batch's index arrays on the device (or, with dev the identity, on the host), and the struct that names them. Each
    request's pages are its own, in a random order, but for the first `shared` positions' (a multiple of the page), which all
    requests name; entries behind its last position name no page."""

    def __init__(self, dev, rows_of, length, page=16, bf16=False, shared=0, first=0, spare=0, seed=0, extra=2, seq_len=None):
        rng = np.random.default_rng(seed)
        self.start = np.concatenate(([first], first + np.cumsum(rows_of))).astype(np.int32)
        self.length = np.asarray(length, np.int32)
        self.count, self.rows, self.page, self.bf16 = len(rows_of), int(self.start[-1]) + spare, page, bf16
        need = [-(-(int(n) + int(m)) // page) if m else 0 for n, m in zip(length, rows_of)]
        common = shared // page
        self.max_pages = max(need + [1]) + extra
        own = [max(n - common, 0) for n in need]
        self.pool = common + sum(own) + 3
        order = rng.permutation(self.pool).astype(np.int32)
        self.table = np.full((self.count, self.max_pages), -1, np.int32)
        at = common
        for r, n in enumerate(own):
            if need[r]:
                self.table[r, :common] = order[:common]
                self.table[r, common:common + n] = order[at:at + n]
                at += n
        self.free = order[at:]
        self.seq_len = self.max_pages * page if seq_len is None else seq_len
        self.keep = (dev(self.start), dev(self.length), dev(self.table))
        self.struct = lh.PagedBatch(*[lh.ptr(a) for a in self.keep], self.count, self.rows, self.max_pages, page, self.pool,
                                    self.seq_len, lh.PAGE_BF16 if bf16 else lh.PAGE_F32)

    def requests(self):
        """(request, its rows as a slice, the positions before them) of the requests that have rows."""
        for r in range(self.count):
            a, b = int(self.start[r]), int(self.start[r + 1])
            if b > a:
                yield r, slice(a, b), int(self.length[r])

    def shape(self, layout, kv, hd):
        return (self.pool, kv, self.page, hd) if layout == "head" else (self.pool, self.page, kv, hd)

    def cache(self, rng, layout, kv, hd):
        x = rng.standard_normal(self.shape(layout, kv, hd), dtype=F)
        return to_bf16(x) if self.bf16 else x

    def row(self, cache, layout, r, t):
        """Position t of request r in a cache as [KV head][dimension], a view."""
        page = cache[self.table[r, t // self.page]]
        return page[:, t % self.page] if layout == "head" else page[t % self.page]

    def gather(self, cache, layout, r, n):
        """The first n positions of request r as float64 [KV head][position][dimension]."""
        pages = values(cache[self.table[r, :-(-n // self.page)]])
        if layout != "head":
            pages = np.swapaxes(pages, 1, 2)
        return np.concatenate(list(pages), 1)[:, :n].astype(np.float64)


def attention(b, q, key, value, heads, kv, hd, layout):
    """Outputs in float64 and a bound of the kernels' error, rows without a request left zero.

    A factor meets the pages' values whole or as three parts that are exact, so a score sums at most 3 hd products: its error
    is at most (3 hd + 8) U sum|q k| / sqrt(hd) (with the division and the scale to base 2); a weight's twice the largest of
    the row's, relative, with 8 U for the exponential and the rescales; the value sums' (3 positions + 64) U of sum p|v|,
    every merge and the division included. A weight is a float32 relative to one that is at least 1: below 2^-126, the
    smallest normal number, the exponential (and the lower parts of a weight that is split) may be 0, so that each |v| adds up
    to 2^-125 of itself: proof enough for values 10^40 apart, where such weights' terms decide a row's sum."""
    mul = heads // kv
    out = np.zeros((b.rows, heads, hd))
    bound = np.zeros_like(out)
    for r, rows, length in b.requests():
        seen = length + rows.stop - rows.start
        keys, vals = b.gather(key, layout, r, seen), b.gather(value, layout, r, seen)
        for g in range(kv):
            for j, i in enumerate(range(rows.start, rows.stop)):
                n = length + j + 1
                k, v = keys[g, :n], vals[g, :n]
                x = q[i].reshape(heads, hd)[g * mul:(g + 1) * mul].astype(np.float64)
                s = x @ k.T / np.sqrt(hd)
                off = ((np.abs(x) @ np.abs(k).T) / np.sqrt(hd)).max(1) * (3 * hd + 8) * U
                p = np.exp(s - s.max(1, keepdims=True))
                p /= p.sum(1, keepdims=True)
                out[i, g * mul:(g + 1) * mul] = p @ v
                bound[i, g * mul:(g + 1) * mul] = ((p @ np.abs(v)) * (2 * off[:, None] + (3 * n + 72) * U) +
                                                   np.abs(v).sum(0) * 2.0 ** -125 + 2.0 ** -126)
    return out.reshape(b.rows, -1), bound.reshape(b.rows, -1)


def normed_rope(x, weight, epsilon, table, hd):
    """A row's heads normed by `weight` and rotated by its table row, in float64, and a bound of the float32 error: the sum
    of hd squares, the mean, the sum with epsilon, the root and the quotient are off by (hd / 2 + 6) U together, the two
    products by 2 U, each rotation's products and sum by 3 U of sum|terms|."""
    x = x.reshape(-1, hd).astype(np.float64)
    y = weight.astype(np.float64) * x / np.sqrt((x * x).mean(1, keepdims=True) + float(F(epsilon)))
    c, s = table[0:hd:2].astype(np.float64), table[hd + 1::2].astype(np.float64)
    a, b = y[:, 0::2], y[:, 1::2]
    out, size = np.empty_like(y), np.empty_like(y)
    out[:, 0::2], out[:, 1::2] = a * c - b * s, a * s + b * c
    size[:, 0::2], size[:, 1::2] = np.abs(a * c) + np.abs(b * s), np.abs(a * s) + np.abs(b * c)
    return out, size * (hd / 2 + 12) * U


def scores(logits, tokens, temperature, top):
    """Rows' log probabilities of the tokens, entropies, likeliest tokens and their log probabilities, in float64."""
    t = float(F(temperature))
    rows = len(logits)
    logprob, entropy = np.zeros(rows), np.zeros(rows)
    tops, top_logprob = np.full((rows, top), -1, np.int64), np.full((rows, top), -np.inf)
    for i in range(rows):
        z = logits[i].astype(np.float64) / t
        m = z.max()
        with np.errstate(invalid="ignore", divide="ignore"):
            e = np.exp(z - m)
            log = z - m - np.log1p(e[np.arange(len(z)) != z.argmax()].sum())
            entropy[i] = -np.where(e > 0, np.exp(log) * np.where(e > 0, log, 0.0), 0.0).sum()
        if tokens is not None and tokens[i] >= 0:
            logprob[i] = log[tokens[i]]
        order = np.lexsort((np.arange(len(z)), -logits[i]))
        order = order[np.isfinite(logits[i][order])][:top]
        tops[i, :len(order)], top_logprob[i, :len(order)] = order, log[order]
    return logprob, entropy, tops, top_logprob
