"""A paged cache and its plain model side by side, for the GPU tests.

`Pair` drives one backend cache and keeps, per sequence, the K and V rows (as
the cache's kind holds them) in 64 bits; `attend` is the definition of the
attention over them, with the bound its result is held to.

The bound, per output element, from the arithmetic.  Queries, weights and (f32)
keys and values are taken as two fp16 halves after a scaling by powers of two
(each rounding is off by at most 2^-11 of what it rounds, the second half's by
2^-22 of the value, and so is the product of two second halves that is left
out) or as three bf16 parts (better still), so a score is off by at most
3 * 2^-22 sum |q k| / sqrt(D) and, summed in f32 over D terms (tensor cores truncate:
2^-23 a term), by D 2^-23 of the same sum more; dx is its largest over the row's
keys.  A weight exp(x - max) is then off by the factor exp(dx), and so is the sum of
the weights; its argument is rounded in powers of two, by at most 2^-23 |x - max| /
ln 2, which times the weight is at most 2^-23; 2^-18 covers that, the exponential
(2^-22) and the rescales of a few hundred tiles' running maximum (2^-23 each,
only where the maximum grows).  Halves of weights and values cost 3 * 2^-22, the
tensor cores' sums over a tile of at most 256 keys in steps of 16 32 * 2^-23, and
n / 64 + 16 additions of tiles and pieces 2^-24 each.  All act on sum p |v|.
"""
import math

import numpy as np
import torch

import kernrt_b200


def rounded(x, kind):
    """f32 rows as the cache holds them, in 64 bits."""
    t = torch.from_numpy(np.ascontiguousarray(x, np.float32))
    if kind == kernrt_b200.BF16:
        t = t.to(torch.bfloat16)
    return t.double().numpy()


def attend(q, keys, vals, group, first, heads=None):
    """q [n, H, D] in 64 bits, keys and vals [L, HK, D]; row i sees keys 0 .. first + i.
    Returns out [n, H, D] and its bound (of some heads, if given)."""
    n, all_heads, d = q.shape
    heads = range(all_heads) if heads is None else heads
    out, bound = np.empty((n, len(heads), d)), np.empty((n, len(heads), d))
    with np.errstate(all="ignore"):
        for i in range(n):
            m = first + i + 1
            k, v = keys[:m], vals[:m]
            for z, h in enumerate(heads):
                kj, vj = k[:, h // group], v[:, h // group]
                x = kj @ q[i, h] / math.sqrt(d)
                dx = float((np.abs(kj) @ np.abs(q[i, h])).max()) / math.sqrt(d) * (3 * 2.0 ** -22 + d * 2.0 ** -23)
                p = np.exp(x - x.max())
                p /= p.sum()
                out[i, z] = p @ vj
                rel = 2 * math.expm1(min(dx, 50.0)) + 2.0 ** -18 + 3 * 2.0 ** -22 + 32 * 2.0 ** -23 + (m / 64 + 16) * 2.0 ** -24
                bound[i, z] = rel * (p @ np.abs(vj))
    return out, bound


class Pair:
    def __init__(self, b, kind, heads, kv_heads, head, page, n_pages, max_seqs, max_len, layers=1):
        self.b, self.kind, self.heads, self.kv_heads, self.head, self.page = b, kind, heads, kv_heads, head, page
        self.layers = layers
        self.p = b.pages_create(kind, layers, heads, kv_heads, head, page, n_pages, max_seqs, max_len)
        self.kv = {}    # sequence -> per layer (K rows, V rows), lists of [HK, D]
        self.bufs = []

    def close(self):
        self.b.pages_destroy(self.p)
        for h in self.bufs:
            self.b.free(h)

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    def up(self, a):
        h = self.b.upload(a)
        self.bufs.append(h)
        return h

    def open(self):
        s = self.b.seq_open(self.p)
        self.kv[s] = [([], []) for _ in range(self.layers)]
        return s

    def fork(self, s, length, n=1):
        got = self.b.seq_fork(self.p, s, length, n)
        for c in got:
            self.kv[c] = [(k[:length], v[:length]) for k, v in self.kv[s]]
        return got

    def copy(self, s, length):
        c = self.b.seq_copy(self.p, s, length)
        self.kv[c] = [(k[:length], v[:length]) for k, v in self.kv[s]]
        return c

    def trim(self, s, length):
        self.b.seq_trim(self.p, s, length)
        self.kv[s] = [(k[:length], v[:length]) for k, v in self.kv[s]]

    def end(self, seqs):
        self.b.seq_close(self.p, seqs)
        for s in seqs:
            del self.kv[s]

    def rows(self, rng, n, scale=1.0):
        """q, k, v of n rows."""
        return [(scale * rng.standard_normal((n, w))).astype(np.float32)
                for w in (self.heads * self.head, self.kv_heads * self.head, self.kv_heads * self.head)]

    def step(self, seqs, rows, data, check=True, check_rows=None, heads=None):
        """One step over all layers; data[layer] = (q, k, v).  Returns the outputs."""
        b = self.b
        b.pages_step(self.p, seqs, rows)
        outs = []
        total = sum(rows)
        for layer in range(self.layers):
            q, k, v = data[layer]
            out = self.up(np.full((total + 2, self.heads * self.head), 7.0, np.float32))
            b.pages_write(self.p, layer, self.up(k), self.up(v))
            b.pages_attention(self.p, layer, self.up(q), out)
            got = b.read(out, (total + 2) * self.heads * self.head).reshape(total + 2, -1)
            assert (got[total:] == 7.0).all(), "rows behind the step's last were written"
            outs.append(got[:total].reshape(total, self.heads, self.head))
        for layer in range(self.layers):
            q, k, v = data[layer]
            rk, rv = (rounded(x, self.kind).reshape(total, self.kv_heads, self.head) for x in (k, v))
            at = 0
            for s, n in zip(seqs, rows):
                ks, vs = self.kv[s][layer]
                first = len(ks)
                # new lists: forks keep theirs
                self.kv[s][layer] = (ks + list(rk[at:at + n]), vs + list(rv[at:at + n]))
                if check and n:
                    some = np.arange(n) if check_rows is None or n <= check_rows else np.unique(
                        np.concatenate([np.linspace(0, n - 1, check_rows).astype(int), [0, n - 1]]))
                    keys, vals = (np.stack(x) for x in self.kv[s][layer])
                    q64 = q[at:at + n].astype(np.float64).reshape(n, self.heads, self.head)
                    for i in some:
                        want, bound = attend(q64[i:i + 1], keys, vals, self.heads // self.kv_heads, first + i, heads)
                        got = outs[layer][at + i]
                        same(got if heads is None else got[heads], want[0], bound[0], f"layer {layer} sequence {s} row {i} of {n}, "
                                                                     f"{first} before")
                at += n
        return outs


def same(got, want, bound, what):
    got = got.astype(np.float64)
    nan = np.isnan(want)
    assert (np.isnan(got) == nan).all(), f"{what}: NaN at {np.argwhere(np.isnan(got) != nan)[:4].tolist()}"
    inf = np.isinf(want)
    assert (got[inf] == want[inf]).all(), f"{what}: infinities differ"
    fine = ~nan & ~inf
    err = np.abs(got[fine] - want[fine])
    over = err > bound[fine] + 1e-37
    if over.any():
        i = int(np.argmax(err / (bound[fine] + 1e-37)))
        raise AssertionError(f"{what}: {over.sum()} of {over.size} beyond the bound; worst {err[i]:.3g}, "
                             f"bound {bound[fine][i]:.3g}, value {want[fine][i]:.3g}")
