"""A plain model of the paged 4-bit cache for the tests, in 64 bits, from the layout and the formulas that include/cutb.h states."""
import numpy as np

SHIFT = (0, 16, 4, 20, 8, 24, 12, 28)


def pad(head):
    return (head + 63) // 64 * 64


def half(x):
    """float64 -> the fp16 number nearest to it, as float64 (numpy rounds float64 to float16 once)."""
    return np.asarray(x, dtype=np.float64).astype(np.float16).astype(np.float64)


def quantised(x):
    """The values that a head's elements x [..., head] (float32) stand for once they are held, and whether any was out of range."""
    x = np.asarray(x, dtype=np.float32)
    c = np.where(np.isnan(x), np.float32(0), np.clip(x, np.float32(-32768), np.float32(32768))).astype(np.float32)
    out = np.empty(x.shape, dtype=np.float64)
    for g in range(0, x.shape[-1], 32):
        part = c[..., g: g + 32]
        m = part.min(-1, keepdims=True).astype(np.float16)
        mf = m.astype(np.float32)
        d = np.maximum(((part.max(-1, keepdims=True) - mf) / np.float32(15)), 0).astype(np.float16)
        df = d.astype(np.float32)
        with np.errstate(divide="ignore", invalid="ignore"):
            q = np.where(df > 0, np.clip(np.rint((part - mf) / df), 0, 15), 0)
        out[..., g: g + 32] = half(q.astype(np.float64) * df + mf)
    return out, bool((c != x).any())


def turned(x, pos, cos, sin, rot, pairing):
    """x [heads, head] float32 turned at pos, products and sums rounded one by one."""
    y = x.astype(np.float32).copy()
    for i in range(rot // 2):
        a, b = (2 * i, 2 * i + 1) if pairing else (i, i + rot // 2)
        c, s = np.float32(cos[pos, i]), np.float32(sin[pos, i])
        u, w = x[:, a].astype(np.float32), x[:, b].astype(np.float32)
        y[:, a] = (u * c).astype(np.float32) - (w * s).astype(np.float32)
        y[:, b] = (u * s).astype(np.float32) + (w * c).astype(np.float32)
    return y


def tables_of(head, rot, n):
    f = 10000.0 ** (-np.arange(rot // 2) * 2 / max(rot, 1))
    a = np.arange(n)[:, None] * f[None, :]
    return np.cos(a).astype(np.float32), np.sin(a).astype(np.float32)


def unit_values(unit, head, which):
    """bytes of a unit -> float64 [16, head]"""
    dp = pad(head)
    groups, h = dp // 32, unit.view(np.float16).astype(np.float64)
    out = np.zeros((16, head))
    for t in range(16):
        for i in range(head):
            g = i // 32
            if which == "k":
                w = 4 if dp % 128 == 0 else 2
                word = t * dp // 8 + g // w * 4 * w + i % 32 // 8 * w + g % w
                at = SHIFT[i % 8]
                q = int(unit[4 * word + at // 8]) >> at % 8 & 15
                d, m = h[8 * dp + 2 * (t * groups + g)], h[8 * dp + 2 * (t * groups + g) + 1]
            else:
                r = i % 16
                word = i // 16 // 4 * 128 + (r % 8 * 4 + t // 4) * 4 + i // 16 % 4
                q = int(unit[8 * dp + 4 * word + (0, 2, 1, 3)[t % 4]]) >> (4 if r >= 8 else 0) & 15
                d, m = h[9 * dp + 8 * (g * 4 + t // 4) + t % 4], h[9 * dp + 8 * (g * 4 + t // 4) + 4 + t % 4]
            out[t, i] = half(q * d + m)
    return out


def attention(q, k, v, pos, scale, window):
    """One row: q [head], k and v [tokens, head] in float64, position pos -> (output, sum of p |v|, largest sum |q k| over the keys seen)."""
    lo = max(0, pos + 1 - window) if window else 0
    k, v = k[lo: pos + 1], v[lo: pos + 1]
    if not len(k):
        return np.zeros(v.shape[1]), np.zeros(v.shape[1]), 0.0
    s = k @ q * scale
    p = np.exp(s - s.max())
    p /= p.sum()
    return p @ v, p @ np.abs(v), float((np.abs(k) @ np.abs(q)).max())


def tolerance(y, spread, products, scale, kind):
    """How far an output may be from y.  Scores are sums of head products in fp32, tensor cores adding 16 at a time for two terms of a
    query: at most 32 additions, each off by at most 2^-23 of the sum of the products' magnitudes, and the second term leaves 2^-22 of
    them: 2^-18 in all.  A score's error moves a weight and the sum of the weights, and the exponentials and the sums are each within
    2^-20 of theirs.  16-bit types: weights as one fp16 number (2^-11 of each, and of the queries', 2^-11 of the products, for bf16
    none), and half a step of the output's type."""
    score = 2.0 ** -18 * products * abs(scale)
    tol = (2 * score + 2.0 ** -18) * spread
    if kind != "f32":
        tol = tol + 2.0 ** -11 * spread + np.abs(y) * {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}[kind]
    return tol + 1e-6


class Pool:
    """The bookkeeping as one would do it by hand."""

    def __init__(self, n_pages, n_slots, width, page):
        self.tables = -np.ones((n_slots, width), dtype=np.int64)
        self.lengths, self.refs, self.page = np.zeros(n_slots, dtype=np.int64), np.zeros(n_pages, dtype=np.int64), page
        self.bytes, self.wrong = None, set()

    def count(self, s):
        return -(-int(self.lengths[s]) // self.page)

    def reserve(self, slots, counts):
        free = [p for p in range(len(self.refs)) if not self.refs[p]]
        seen, refused, shed = set(), False, []
        for s, c in zip(slots, counts):
            if not 0 <= s < len(self.lengths) or s in seen or self.lengths[s] + c > self.tables.shape[1] * self.page:
                self.wrong.add("invalid")
                continue
            seen.add(s)
            have, want = self.count(s), -(-(int(self.lengths[s]) + c) // self.page)
            last = self.tables[s, have - 1] if c and self.lengths[s] % self.page else None
            copies = last is not None and self.refs[last] > 1
            need = want - have + copies
            if refused or need > len(free):
                refused = True
                self.wrong.add("pages")
                continue
            if copies:
                p = free.pop(0)
                self.refs[last] -= 1
                self.refs[p] = 1
                self.tables[s, have - 1] = p
                shed.append((last, p))
            for i in range(have, want):
                p = free.pop(0)
                self.tables[s, i], self.refs[p] = p, 1
            self.lengths[s] += c
        for a, b in shed:
            if self.bytes is not None:
                self.bytes[b] = self.bytes[a]

    def fork(self, src, dst):
        lengths, used = self.lengths.copy(), set()
        for a, b in zip(src, dst):
            if not (0 <= a < len(lengths) and 0 <= b < len(lengths)) or a == b or b in used or lengths[b]:
                self.wrong.add("invalid")
                used.add(b)
                continue
            used.add(b)
            n = -(-int(lengths[a]) // self.page)
            self.tables[b, :n] = self.tables[a, :n]
            self.refs[self.tables[a, :n]] += 1
            self.lengths[b] = lengths[a]

    def free(self, slots):
        for s in slots:
            if not 0 <= s < len(self.lengths):
                self.wrong.add("invalid")
                continue
            n = self.count(s)
            self.refs[self.tables[s, :n]] -= 1
            self.tables[s, :n] = -1
            self.lengths[s] = 0

    def compact(self):
        live = [p for p in range(len(self.refs)) if self.refs[p]]
        n = len(live)
        holes, late = [p for p in range(n) if not self.refs[p]], [p for p in live if p >= n]
        to = {a: b for a, b in zip(late, holes)}
        for a, b in to.items():
            self.refs[b], self.refs[a] = self.refs[a], 0
            if self.bytes is not None:
                self.bytes[b] = self.bytes[a]
        self.tables = np.array([[to.get(int(p), int(p)) for p in row] for row in self.tables])


def sampled(x, t, k, p, least, u):
    """(token, log of its share) of one row in float64; None where there is no choice."""
    x = np.where(np.isnan(x), -np.inf, np.asarray(x, dtype=np.float64))
    if x.max() == -np.inf:
        return None, -np.inf
    if t == 0:
        return int(np.argmax(x)), 0.0
    with np.errstate(invalid="ignore"):
        w_all = np.where(x == x.max(), 1.0, np.exp((x - x.max()) / t))
    order = np.argsort(-x, kind="stable")
    if 0 < k < len(x):
        order = order[:k]
    w = w_all[order]
    if p < 1:
        before = np.cumsum(w) - w
        n = max(1, int(np.count_nonzero(before < p * w.sum())))
        order, w = order[:n], w[:n]
    n = max(1, int(np.count_nonzero(w >= least)))
    kept = np.sort(order[:n])
    sums = np.cumsum(w_all[kept])
    i = min(int(np.searchsorted(sums, u * sums[-1], side="right")), len(sums) - 1)
    return int(kept[i]), float(np.log(w_all[kept[i]] / sums[-1]))
