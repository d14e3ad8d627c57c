"""Plain float64 implementation of the paged-cache operators (numpy, CPU), and batches for their
tests. Pool slots that hold no position are NaN, so that anything read from them shows."""
import numpy as np


def bf16(x):
    """float array -> the nearest bf16 values (ties to even), as float64."""
    u = np.ascontiguousarray(x, dtype=np.float32).view(np.uint32).astype(np.uint64)
    u = (u + 0x7FFF + ((u >> 16) & 1)) & 0xFFFF0000
    return u.astype(np.uint32).view(np.float32).astype(np.float64)


def normal(rng, *shape):
    return bf16(rng.standard_normal(shape))


def rotate(x, pos, theta):
    """x [n, H, D] at positions pos [n], split halves."""
    half = x.shape[-1] // 2
    ang = np.asarray(pos, np.float64)[:, None] * theta ** (-np.arange(half) / half)
    c, s = np.cos(ang)[:, None], np.sin(ang)[:, None]
    a, b = x[..., :half], x[..., half:]
    return np.concatenate([a * c - b * s, a * s + b * c], -1)


def norm(x, w, eps):
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w


def attend(q, k, v, last, scale):
    """q [n, Hq, D] over k, v [L, Hkv, D]; row i sees keys <= last[i]. Returns (out [n, Hq, D],
    sum of weight * |v|); rows that see nothing are zeros."""
    n, Hq, D = q.shape
    L, Hkv = k.shape[:2]
    G = Hq // Hkv
    out, mag = np.zeros((n, Hq, D)), np.zeros((n, Hq, D))
    if not L or not n:
        return out, mag
    seen = np.arange(L)[None] <= np.asarray(last)[:, None]
    some = seen.any(1)
    for h in range(Hq):
        s = q[:, h] @ k[:, h // G].T * scale
        s = np.where(seen, s, -np.inf)[some]
        p = np.exp(s - s.max(1, keepdims=True))
        p /= p.sum(1, keepdims=True)
        out[some, h] = p @ v[:, h // G]
        mag[some, h] = p @ np.abs(v[:, h // G])
    return out, mag


class Batch:
    """A ragged batch over a pool: new[b] query rows of sequence b, kv[b] positions held (rows
    included), pages in a shuffled order. holes: (b, page) pairs whose table entry is bad."""

    def __init__(self, new, kv, page, Hq, Hkv, seed, D=128, prefix=0, holes=(), spare=2, bad=(-1, 1 << 30)):
        rng = np.random.default_rng(seed)
        self.new, self.kv, self.page, self.Hq, self.Hkv, self.D, self.prefix = list(new), list(kv), page, Hq, Hkv, D, prefix
        counts = [-(-n // page) for n in kv]
        cols = max(max(counts), 1)
        npre = -(-prefix // page)
        self.n_pages = sum(counts) + npre + spare
        order = rng.permutation(self.n_pages)
        self.table = np.full((len(new), cols), -1, np.int32)
        self.k = np.full((self.n_pages, Hkv, page, D), np.nan)
        self.v = np.full((self.n_pages, Hkv, page, D), np.nan)
        self.held = []
        at = 0
        for b, (n, c) in enumerate(zip(kv, counts)):
            self.table[b, :c] = order[at:at + c]
            at += c
            k, v = normal(rng, n, Hkv, D), normal(rng, n, Hkv, D)
            self._put(self.table[b], k, v)
            self.held.append([k, v])
        self.prefix_table = order[at:at + npre].astype(np.int32)
        k, v = normal(rng, prefix, Hkv, D), normal(rng, prefix, Hkv, D)
        self._put(self.prefix_table, k, v)
        self.shared = [k, v]
        for i, (b, p) in enumerate(holes):  # positions of a bad entry read as zero rows
            self.table[b, p] = bad[i % len(bad)]
            for x in self.held[b]:
                x[p * page:(p + 1) * page] = 0.0
        self.starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        self.rows = int(self.starts[-1])
        self.q = normal(rng, self.rows, Hq, D)

    def _put(self, pages, k, v):
        P = self.page
        for p in range(-(-k.shape[0] // P)):
            n = min(P, k.shape[0] - p * P)
            self.k[pages[p], :, :n] = k[p * P:p * P + n].transpose(1, 0, 2)
            self.v[pages[p], :, :n] = v[p * P:p * P + n].transpose(1, 0, 2)

    def attention(self, scale=None, causal=True):
        scale = self.D ** -0.5 if scale is None else scale
        outs, mags = [], []
        for b, (n, L) in enumerate(zip(self.new, self.kv)):
            k, v = (np.concatenate([s, h]) for s, h in zip(self.shared, self.held[b]))
            # the last key of each row; a row before the first own position sees the prefix alone
            last = np.maximum(self.prefix - 1, self.prefix + L - n + np.arange(n)) if causal else np.full(n, self.prefix + L)
            o, m = attend(self.q[self.starts[b]:self.starts[b + 1]], k, v, last, scale)
            outs.append(o)
            mags.append(m)
        return (np.concatenate(x).reshape(-1, self.Hq * self.D) for x in (outs, mags))


def check_attention(got, ref, mag, what):
    """Elementwise bound. P is rounded to bf16 (half a step: 2^-8 of a weight) and the row sum is
    taken over the rounded P, so the weights are off by at most 2 * 2^-8 of themselves; the
    output is rounded once (2^-8 of it); scores and sums in 32 bits add less than 2^-14 of the
    weighted magnitudes at the tests' sizes."""
    assert np.isfinite(got).all(), f"{what}: not finite"
    bound = (2.0 ** -7 + 2.0 ** -14) * mag + 2.0 ** -8 * np.abs(ref)
    d = np.abs(got - ref)
    worst = float((d / np.maximum(bound, 1e-30)).max()) if d.size else 0.0
    print(f"  {what}: worst error / bound {worst:.3f}", flush=True)
    assert (d <= bound + 1e-30).all(), f"{what}: error {worst} of the bound at {np.unravel_index((d - bound).argmax(), d.shape)}"
