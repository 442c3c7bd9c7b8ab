"""Plain statements of the cache operators for the tests: the codes in numpy's 32-bit arithmetic (they are defined by it), the
attention in 64 bits, one row and head at a time."""
import numpy as np
import torch

from deepx_amd import lib as dx

TT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
DT = {"f32": dx.F32, "f16": dx.F16, "bf16": dx.BF16}
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"f32": 2.0 ** -149, "f16": 2.0 ** -25, "bf16": 2.0 ** -133}
CODE = {"i8": dx.I8, "e4m3": dx.F8E4M3}
MAX = {"i8": np.float32(127), "e4m3": np.float32(448)}
INV = {"i8": np.float32(1) / np.float32(127), "e4m3": np.float32(1) / np.float32(448)}


def heads(t):
    return dx.Heads(t.data_ptr(), t.stride(0), t.stride(1))


def decode(raw, code):
    """int8 storage -> fp32 values of the codes"""
    if code == "i8":
        return raw.astype(np.float32)
    return torch.from_numpy(np.ascontiguousarray(raw)).view(torch.float8_e4m3fn).float().numpy()


def encode(x, f, code):
    with np.errstate(all="ignore"):
        y = (x.astype(np.float32) * np.float32(f)).astype(np.float32)
        y = np.where(np.isnan(y), y, np.clip(y, -MAX[code], MAX[code]))
        if code == "i8":
            return np.where(np.isnan(y), 0, np.rint(y)).astype(np.int8)
    return torch.from_numpy(np.ascontiguousarray(y)).to(torch.float8_e4m3fn).view(torch.int8).numpy()


class Cache:
    """A paged cache with random contents, on the host and on the GPU."""

    def __init__(self, code, page, heads, dim, batch, per_seq, seed, spare=2, paged=True, missing=()):
        rng = np.random.default_rng(seed)
        self.code, self.page, self.heads, self.dim, self.batch, self.per_seq = code, page, heads, dim, batch, per_seq
        self.pages = batch * per_seq + (spare if paged else 0)
        shape = (self.pages, heads)
        values = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
        self.k = encode(values(*shape, page, dim), MAX[code] / 4, code)
        self.v = encode(values(*shape, dim, page), MAX[code] / 4, code)
        self.ks, self.vs = ((0.5 + rng.random(shape)).astype(np.float32) / (MAX[code] / 4) for _ in range(2))
        self.table = rng.permutation(self.pages)[:batch * per_seq].reshape(batch, per_seq).astype(np.int32) if paged else None
        for b, i, p in missing:
            self.table[b, i] = p

    def upload(self):
        self.dev = [torch.from_numpy(t).cuda() for t in (self.k, self.v, self.ks, self.vs)]
        self.dev_table = torch.from_numpy(self.table).cuda() if self.table is not None else None
        return dx.KvCache(*[t.data_ptr() for t in self.dev], self.dev_table.data_ptr() if self.table is not None else None, self.pages, self.per_seq, self.page, self.heads, self.dim, CODE[self.code])

    def download(self):
        return [t.cpu().numpy() for t in self.dev]

    def page_of(self, b, slot):
        if not 0 <= slot < self.per_seq:
            return -1
        p = int(self.table[b, slot]) if self.table is not None else b * self.per_seq + slot
        return p if 0 <= p < self.pages else -1


class Rows:
    """Packed rows: counts of each sequence and its tokens in the cache; `extra` rows behind the last sequence."""

    def __init__(self, counts, lengths, extra=0, max_rows=None, uniform=False):
        self.counts, self.lengths, self.uniform = list(counts), list(lengths), uniform
        self.max_rows = max(counts) if max_rows is None else max_rows
        self.offsets = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        self.rows = int(self.offsets[-1]) + extra

    def upload(self):
        self.dev = [torch.from_numpy(np.asarray(x, dtype=np.int32)).cuda() for x in (self.offsets, self.lengths)]
        return dx.KvRows(None if self.uniform else self.dev[0].data_ptr(), self.dev[1].data_ptr(), self.rows, len(self.counts), self.max_rows)

    def each(self):
        """(sequence, packed row, token) of every row that a call processes"""
        for b, n in enumerate(self.counts):
            for i in range(min(n, self.max_rows)):
                yield b, int(self.offsets[b]) + i, max(0, int(self.lengths[b])) - n + i


def write(c, rows, k, v):
    """the definition of dxh_kvcache_write on c's host arrays; k, v: fp32 [rows, heads, dim]"""
    touched = {}
    for b, r, t in rows.each():
        if t >= 0 and c.page_of(b, t // c.page) >= 0:
            touched.setdefault((b, t // c.page), []).append((t % c.page, r))
    for (b, slot), new in touched.items():
        p, at, src = c.page_of(b, slot), [t for t, _ in new], [r for _, r in new]
        first = at[0]
        for x, codes, scales, across in ((k, c.k, c.ks, False), (v, c.v, c.vs, True)):
            for h in range(c.heads):
                val = x[src, h]
                with np.errstate(all="ignore"):
                    top = np.minimum(np.fmax.reduce(np.abs(val).ravel(), initial=np.float32(0)), np.finfo(np.float32).max)
                scale = np.maximum(np.float32(top) * INV[c.code], np.float32(2.0 ** -100))
                old = scales[p, h]
                if first > 0:
                    scale = np.fmax(scale, old)
                inv = np.float32(1) / scale
                view = codes[p, h].T if across else codes[p, h]
                if first > 0 and scale > old:
                    view[:first] = encode(decode(view[:first], c.code), old * inv, c.code)
                view[at] = encode(val, inv, c.code)
                scales[p, h] = scale


def read(c, rows, which):
    """fp32 values of the processed rows: {packed row: [heads, dim]}"""
    out = {}
    for b, r, t in rows.each():
        p = c.page_of(b, t // c.page) if t >= 0 else -1
        if p < 0:
            out[r] = np.zeros((c.heads, c.dim), np.float32)
        else:
            raw = c.v[p, :, :, t % c.page] if which else c.k[p, :, t % c.page]
            out[r] = decode(raw, c.code) * (c.vs if which else c.ks)[p][:, None]
    return out


def attention(c, rows, q, scale, causal, window):
    """64-bit values of the processed rows and, for the bars, per row and head: out, lse, sum p |v|, largest scale sum |q||k|, tokens seen.
    q: float64 [rows, q_heads, dim].  A token that a row does not see is not looked at."""
    G = q.shape[1] // c.heads
    res = {}
    for b, r, t in rows.each():
        n = max(0, min(int(rows.lengths[b]), c.per_seq * c.page))
        hi = (min(t + 1, n) if causal else n) if t >= 0 else 0
        lo = max(0, t - window + 1) if window else 0
        toks = [j for j in range(lo, hi) if c.page_of(b, j // c.page) >= 0]
        out, lse = np.zeros((q.shape[1], c.dim)), np.full(q.shape[1], -np.inf)
        mag, big, weight = np.zeros((q.shape[1], c.dim)), np.zeros(q.shape[1]), np.zeros(q.shape[1])
        if toks:
            pg, at = np.array([c.page_of(b, j // c.page) for j in toks]), np.array(toks) % c.page
            K = decode(c.k[pg, :, at], c.code).astype(np.float64) * c.ks[pg].astype(np.float64)[..., None]
            V = decode(c.v[pg, :, :, at], c.code).astype(np.float64) * c.vs[pg].astype(np.float64)[..., None]
            for h in range(q.shape[1]):
                s = K[:, h // G] @ q[r, h] * scale
                m = s.max()
                e = np.exp(s - m)
                out[h], lse[h] = e @ V[:, h // G] / e.sum(), m + np.log(e.sum())
                weight[h] = (e * np.abs(c.vs[pg, h // G])).max() / e.sum()
                mag[h], big[h] = e @ np.abs(V[:, h // G]) / e.sum(), (np.abs(K[:, h // G]) @ np.abs(q[r, h])).max() * abs(scale)
        res[r] = (out, lse, mag, big, len(toks), np.abs(V).max() if toks else 0.0, weight)
    return res


def attention_bar(name, c, entry, far=0.0):
    """How far a result may be from the 64-bit value.  With u = 2^-24:
      score: a product of D exact terms in an fp32 accumulator, each passing through at most D/32 chained and 32 inner additions, and three
      products with scales: (D/32 + 40) u of scale sum|q||k|; f32 rows add 2^-24 of it for the split of q.
      probability: that as a relative error, the rounding of s - m (2 u |s - m|, |s - m| under twice the largest score) and of 2^x (4 u).
      sums over N tokens: (N/32 + 64) u.  Both the sum and its normalisation carry these: twice.
      rounding of p * v_scale to f16, or to two f16 parts for f32 rows: 2^-11, 2^-22 of sum p|v|; p * v_scale is held relative to its largest, at least
      2^7 times as large for f16 and bf16 rows and 2^15 times for f32 rows, so that f16's smallest steps (half of 2^-24) add at most 2^-32, 2^-40 of
      the largest times a code for each token; of the result: half a step.
      underflow: the hardware's 2^x gives 0 below 2^-126, the smallest normal fp32 number; with l >= 1 (the largest term is 1) each of the N
      terms is off by at most 2^-126 max|v|.
      far: the largest |log2| of the value scales, where they are far from 1.  A scale enters as its logarithm (rounded, and one unit off at most: 3 u
      far in all) and the sum with the score is rounded (u far), in base 2: ln 2 * 4 u far < 4 u far of a probability and of its share of the sum."""
    out, lse, mag, big, n, top, weight = entry
    u = 2.0 ** -24
    s = ((c.dim / 32 + 42) * big + 4 * big + 4 + 4 * far) * u
    sums = (n / 32 + 64) * u
    part = {"bf16": 2.0 ** -11, "f16": 2.0 ** -11, "f32": 2.0 ** -22}[name]
    bar = (n * (2.0 ** -40 if name == "f32" else 2.0 ** -32) * float(MAX[c.code]) * weight)[:, None] + mag * (part + 2 * s + 2 * sums)[:, None] + np.abs(out) * HALF_STEP[name] * (1 + 2 ** -8) + TINY[name] + n * 2.0 ** -126 * top
    return bar, s + sums + np.abs(np.where(np.isfinite(lse), lse, 0)) * 2 * u
