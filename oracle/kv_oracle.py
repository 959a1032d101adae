"""Plain 64-bit forms of the paged 8-bit K/V cache and its attention, in numpy (test infrastructure only).

No counterpart in the reference: pages of 64 tokens taken from one stack in a fixed order, e4m3
codes with a power-of-two scale per page and head, softmax attention over them and over packed
prompts, each written from its definition.
"""

from __future__ import annotations

import numpy as np

PAGE = 64


def pages_of(n: int) -> int:
    return -(-n // PAGE)


class Pages:
    """Block tables, lengths and free stack."""

    def __init__(self, requests: int, pages: int, max_blocks: int) -> None:
        self.tables = np.full((requests, max_blocks), -1, np.int64)
        self.lengths = np.zeros(requests, np.int64)
        self.free = list(range(pages))

    def resize(self, targets):
        """Move to ``targets``; (starts, slots, positions, pieces) of the new tokens."""
        targets = [int(t) for t in targets]
        freed = []
        for b, target in enumerate(targets):
            for block in range(pages_of(target), pages_of(int(self.lengths[b]))):
                freed.append(int(self.tables[b, block]))
                self.tables[b, block] = -1
        self.free.extend(reversed(freed))
        starts, slots, positions, pieces = [0], [], [], []
        for b, target in enumerate(targets):
            cur = int(self.lengths[b])
            for block in range(pages_of(cur), pages_of(target)):
                self.tables[b, block] = self.free.pop()
            for p in range(cur, target):
                slot = int(self.tables[b, p // PAGE]) * PAGE + p % PAGE
                if p == cur or p % PAGE == 0:
                    pieces.append([len(slots), 0, slot // PAGE, p % PAGE])
                pieces[-1][1] += 1
                slots.append(slot)
                positions.append(p)
            starts.append(len(slots))
            self.lengths[b] = target
        return starts, slots, positions, pieces


def e4m3(x: np.ndarray) -> np.ndarray:
    """Nearest e4m3 value, ties to even; beyond 448 the largest, NaN stays NaN."""
    x = np.asarray(x, np.float64)
    finite = np.where(np.isfinite(x), x, 0.0)
    _, exponent = np.frexp(finite)
    step = np.exp2(np.maximum(exponent, -5) - 4.0)  # four significant bits, least normal 2^-6
    near = np.clip(np.round(finite / step) * step, -448.0, 448.0)
    return np.where(np.isnan(x), np.nan, np.where(np.isinf(x), np.sign(x) * 448.0, near))


def scale_of(x: np.ndarray) -> float:
    """The smallest power of two s >= 2^-64 with |x| <= 448 s over the finite values."""
    finite = np.abs(x[np.isfinite(x)])
    most = float(finite.max()) if finite.size else 0.0
    e = -64
    while most > 448.0 * 2.0**e:
        e += 1
    return 2.0**e


class Store:
    """Codes (as the numbers they stand for, before the scale) and scales by page."""

    def __init__(self, heads: int, width: int) -> None:
        self.heads, self.width = heads, width
        self.codes: dict[int, np.ndarray] = {}
        self.scales: dict[int, np.ndarray] = {}

    def put(self, x: np.ndarray, pieces) -> None:
        for first, count, page, offset in pieces:
            new = np.asarray(x[first:first + count], np.float64)
            if offset == 0:
                self.codes[page] = np.zeros((PAGE, self.heads, self.width))
                self.scales[page] = np.zeros(self.heads)
            for h in range(self.heads):
                s = scale_of(new[:, h])
                if offset:
                    old = self.scales[page][h]
                    s = max(s, old)
                    self.codes[page][:offset, h] = e4m3(self.codes[page][:offset, h] * (old / s))
                self.codes[page][offset:offset + count, h] = e4m3(new[:, h] / s)
                self.scales[page][h] = s

    def rows(self, slots) -> np.ndarray:
        return np.stack([self.codes[s // PAGE][s % PAGE] * self.scales[s // PAGE][:, None] for s in slots]) if len(slots) \
            else np.zeros((0, self.heads, self.width))


def softmax_rows(q: np.ndarray, k: np.ndarray, v: np.ndarray, scale: float) -> np.ndarray:
    """q [n, width] against k, v [m, width], row i of q seeing the first m - n + i + 1."""
    n, m = q.shape[0], k.shape[0]
    out = np.zeros((n, v.shape[1]))
    for i in range(n):
        see = m - n + i + 1
        if see <= 0:
            continue
        with np.errstate(all="ignore"):
            s = scale * (k[:see] @ q[i])
            p = np.exp(s - s.max())
            out[i] = (p @ v[:see]) / p.sum()
    return out


def prompt(q, k, v, starts, scale=None) -> np.ndarray:
    """Causal attention over packed sequences; [tokens, heads, width] in 64 bits."""
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    scale = q.shape[2] ** -0.5 if scale is None else scale
    group = q.shape[1] // k.shape[1]
    out = np.full(q.shape, np.nan)
    for a, z in zip(starts[:-1], starts[1:]):
        for h in range(q.shape[1]):
            out[a:z, h] = softmax_rows(q[a:z, h], k[a:z, h // group], v[a:z, h // group], scale)
    return out


def attend(q, k_rows, v_rows, scale=None) -> np.ndarray:
    """q [requests, heads, width] over each request's rows [n, kv_heads, width]; zeros without rows."""
    q = np.asarray(q, np.float64)
    scale = q.shape[2] ** -0.5 if scale is None else scale
    out = np.zeros(q.shape)
    for b in range(q.shape[0]):
        if not len(k_rows[b]):
            continue
        group = q.shape[1] // k_rows[b].shape[1]
        for h in range(q.shape[1]):
            out[b, h] = softmax_rows(q[b, h][None], k_rows[b][:, h // group], v_rows[b][:, h // group], scale)[0]
    return out


def _row_with_bound(q, k, v, scale):
    """One query row against all of k, v [n, width], and how far float32 arithmetic may take each output, from the row's
    own sums: a score is off by u of |scale| * sum_d |q_d k_jd| and a weight p by that and u of itself, which moves the mean
    o = sum p v by p |v - o| of it; the mean's products and sum take u of sum p |v|.  u = 2^-20: eight roundings."""
    s = scale * (k @ q)
    p = np.exp(s - s.max())
    p /= p.sum()
    o = p @ v
    reach = abs(scale) * (np.abs(k) @ np.abs(q))
    return o, 2.0**-20 * ((p * (reach + 1)) @ np.abs(v - o) + p @ np.abs(v))


def prompt_with_bound(q, k, v, starts, scale=None):
    """``prompt`` and how far float32 arithmetic may take each of its outputs."""
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    scale = q.shape[2] ** -0.5 if scale is None else scale
    group = q.shape[1] // k.shape[1]
    out, bound = np.full(q.shape, np.nan), np.zeros(q.shape)
    for a, z in zip(starts[:-1], starts[1:]):
        for h in range(q.shape[1]):
            for i in range(a, z):
                out[i, h], bound[i, h] = _row_with_bound(q[i, h], k[a:i + 1, h // group], v[a:i + 1, h // group], scale)
    return out, bound


def attend_with_bound(q, k_rows, v_rows, scale=None):
    """``attend`` and how far float32 arithmetic may take each of its outputs."""
    q = np.asarray(q, np.float64)
    scale = q.shape[2] ** -0.5 if scale is None else scale
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    for b in range(q.shape[0]):
        for h in range(q.shape[1]) if len(k_rows[b]) else ():
            group = q.shape[1] // k_rows[b].shape[1]
            out[b, h], bound[b, h] = _row_with_bound(q[b, h], k_rows[b][:, h // group], v_rows[b][:, h // group], scale)
    return out, bound
