"""Plain float64 forms of the operators for many requests, and their error bounds, shared by their tests."""
import ctypes

import numpy as np

import llama_hip as lh

U = 2.0 ** -24  # half a step of float32, relative


class Batch:
    """A batch's index arrays on the device (or, with dev the identity, on the host), and the struct that names them."""

    def __init__(self, dev, rows_of, length, slot=None, slots=None, prefix=0, prefix_seq_len=None, seq_len=64, first=0,
                 spare=0):
        self.start = np.concatenate(([first], first + np.cumsum(rows_of))).astype(np.int32)
        self.length = np.asarray(length, np.int32)
        self.slot = np.arange(len(rows_of), dtype=np.int32) if slot is None else np.asarray(slot, np.int32)
        self.count, self.rows = len(rows_of), int(self.start[-1]) + spare
        self.prefix, self.seq_len = prefix, seq_len
        self.prefix_seq_len = prefix if prefix_seq_len is None else prefix_seq_len
        self.slots = int(self.slot.max()) + 1 if slots is None else slots
        self.keep = (dev(self.start), dev(self.length), None if slot is None else dev(self.slot))
        self.struct = lh.RequestBatch(*[lh.ptr(a) for a in self.keep], self.count, self.rows, prefix,
                                      self.prefix_seq_len, seq_len, self.slots)

    def requests(self):
        """(request, its rows as a slice, own length, slot) of the requests that have rows."""
        for r in range(self.count):
            a, b = int(self.start[r]), int(self.start[r + 1])
            if b > a:
                yield r, slice(a, b), int(self.length[r]), int(self.slot[r])


def cache_shape(layout, positions, kv, hd):
    return (kv, positions, hd) if layout == "head" else (positions, kv, hd)


def by_head(cache, layout):
    """A cache as [KV head][position][dimension], a view."""
    return cache if layout == "head" else np.swapaxes(cache, -3, -2)


def attention(b, q, prefix_key, prefix_value, key, value, heads, kv, hd, layout):
    """Outputs in float64 and a bound of the float32 kernels' error, rows without a request left zero.

    A score's error is at most (hd + 8) U sum|q k| / sqrt(hd) (hd products and sums, the division, the scale to base 2);
    a weight's twice the largest of the row's, relative, with 8 U for the exponential and the rescales; the value sums'
    (positions + 64) U of sum p|v|, every merge and the division included."""
    mul = heads // kv
    out = np.zeros((b.rows, heads, hd))
    bound = np.zeros_like(out)
    for _, rows, length, slot in b.requests():
        for g in range(kv):
            k = np.concatenate((by_head(prefix_key, layout)[g, :b.prefix], by_head(key[slot], layout)[g])).astype(np.float64)
            v = np.concatenate((by_head(prefix_value, layout)[g, :b.prefix], by_head(value[slot], layout)[g])).astype(np.float64)
            for j, i in enumerate(range(rows.start, rows.stop)):
                n = b.prefix + length + j + 1
                x = q[i].reshape(heads, hd)[g * mul:(g + 1) * mul].astype(np.float64)
                s = x @ k[:n].T / np.sqrt(hd)
                off = ((np.abs(x) @ np.abs(k[:n]).T) / np.sqrt(hd)).max(1) * (hd + 8) * U
                p = np.exp(s - s.max(1, keepdims=True))
                p /= p.sum(1, keepdims=True)
                out[i, g * mul:(g + 1) * mul] = p @ v[:n]
                bound[i, g * mul:(g + 1) * mul] = (p @ np.abs(v[:n])) * (2 * off[:, None] + (n + 72) * U)
    return out.reshape(b.rows, -1), bound.reshape(b.rows, -1)


def adapters(x, ids, base, a, b, scale):
    """base + scale B (A x) in float64 and a bound of the float32 kernels' error: A x over k values in partial sums of at
    most k / 32 + 40 terms in a row, B's product of rank + 8, the scale and the sum with the base."""
    y, bound = base.astype(np.float64), np.abs(base.astype(np.float64)) * 2 * U
    for i, at in enumerate(ids):
        if at < 0:
            continue
        aa, bb, xx = a[at].astype(np.float64), b[at].astype(np.float64), x[i].astype(np.float64)
        low = aa @ xx
        wrong = (np.abs(aa) @ np.abs(xx)) * (len(xx) / 32 + 40) * U
        y[i] += scale[at] * (bb @ low)
        bound[i] += abs(scale[at]) * (np.abs(bb) @ (wrong + (len(low) + 8) * U * np.abs(low))) + 2 * U * np.abs(y[i])
    return y, bound


def swiglu(gate, gate_bound, up, up_bound):
    """silu(gate) * up; silu's slope is at most 1.1, and its own evaluation is off by at most 8 U of it."""
    s = gate / (1.0 + np.exp(-gate))
    off = 1.1 * gate_bound + 8 * U * np.abs(s)
    return s * up, off * (np.abs(up) + up_bound) + np.abs(s) * up_bound + U * np.abs(s * up)


def softmax(z):
    e = np.exp(z - z.max())
    return e / e.sum()


def verify(start, logits, draft, tokens, uniform, temperature):
    """(accepted, next) of each request with rows, one draft at a time in float64; None for the others."""
    got = []
    t = float(np.float32(temperature))
    for a, b in zip(start, start[1:]):
        if a == b:
            got.append(None)
            continue
        row = int(a)
        while True:
            z = logits[row].astype(np.float64)
            x = int(tokens[row + 1]) if row + 1 < b else -1
            if t == 0.0:
                if x >= 0 and int(z.argmax()) == x:
                    row += 1
                    continue
                got.append((row - int(a), int(z.argmax())))
                break
            p = softmax(z / t)
            if x >= 0:
                if draft is not None:
                    q = softmax(draft[row].astype(np.float64) / t)
                else:
                    q = np.zeros_like(p)
                    q[x] = 1.0
                if float(uniform[row, 0]) * q[x] < p[x]:
                    row += 1
                    continue
                rest = np.maximum(p - q, 0.0)
                p = rest if rest.sum() > 0.0 else p
            running = np.cumsum(p)
            got.append((row - int(a), int((running <= float(uniform[row, 1]) * running[-1]).sum())))
            break
    return got


def lora_segment(bf16, c, ldc, base, a, b, scale, n, rank, base3=None, a3=None, b3=None):
    struct = lh.LoraBf16Segment if bf16 else lh.LoraSegment
    kind = lh.GEMM_ADD if base3 is None else lh.GEMM_SWIGLU
    return struct(*[lh.ptr(c), ldc] + [lh.ptr(x) for x in (base, base3, a, b, a3, b3, scale)] + [n, rank, kind])


def array(structs):
    return (type(structs[0]) * len(structs))(*structs)


def byref(x):
    return ctypes.byref(x)
