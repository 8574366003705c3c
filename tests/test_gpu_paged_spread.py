"""Attention of many query rows over keys, queries and values of very different
size: what is large, masked or infinite in one place leaves the rest of its tile
as it is by the definition.

The bound, per output element, with p_t the weights, v_t the values and o the
output in 64 bits.  A score of key t is off by at most dx_t = (3 * 2^-22 + D 2^-23)
sum |q k_t| / sqrt(D), as in tests/_paged.py but of its own key, and 2^-18 for what
16-bit halves lose far below a tile's or a row's largest element; that moves o by
at most sum p_t e_t |v_t - o| with e_t = exp(dx_t) - 1, doubled for the terms of
second order.  Everything else acts on sum p |v|: 2^-18 as there, once more for
values far below a tile's largest, 3 * 2^-22 and 32 * 2^-23 as there, and the
additions: n / 64 + 16 of tiles and pieces where the tensor cores take the tiles,
n one by one where the rows are attended in f32, 2^-24 each.
"""
import math

import numpy as np
import pytest

from kernrt_b200 import BF16, F32
from tests._paged import Pair, rounded, same

pytestmark = pytest.mark.gpu

KINDS = pytest.mark.parametrize("kind", [BF16, F32], ids=["bf16", "f32"])
D = 128


def check(c, data, out, rows, heads, by_one=True):
    """Some rows of a first step of one sequence."""
    q, k, v = data
    n = len(q)
    d = c.head
    q = q.astype(np.float64).reshape(n, c.heads, d)
    k, v = (rounded(x, c.kind).reshape(n, c.kv_heads, d) for x in (k, v))
    for r in rows:
        m = r + 1
        adds = (m if by_one else m / 64) + 16
        rest = 2 * 2.0 ** -18 + 3 * 2.0 ** -22 + 32 * 2.0 ** -23 + adds * 2.0 ** -24
        for h in heads:
            kj, vj = k[:m, h * c.kv_heads // c.heads], v[:m, h * c.kv_heads // c.heads]
            x = kj @ q[r, h] / math.sqrt(d)
            dx = np.abs(kj) @ np.abs(q[r, h]) / math.sqrt(d) * (3 * 2.0 ** -22 + d * 2.0 ** -23) + 2.0 ** -18
            p = np.exp(x - x.max())
            p /= p.sum()
            o = p @ vj
            bound = 2 * (p * np.expm1(np.minimum(dx, 50))) @ np.abs(vj - o) + rest * (p @ np.abs(vj))
            same(out[r, h], o, bound, f"row {r} head {h}")


def attend(gpu, kind, data, heads=16, kv_heads=8):
    n = len(data[0])
    with Pair(gpu, kind, heads, kv_heads, D, 64, n // 64 + 2, 1, n) as c:
        return c, c.step([c.open()], [n], [data], check=False)[0]


def normal(seed, n=1100, heads=16, kv_heads=8):
    rng = np.random.default_rng(seed)
    return [rng.standard_normal((n, w * D)).astype(np.float32) for w in (heads, kv_heads, kv_heads)]


@KINDS
def test_an_infinity_leaves_the_query_tiles_before_it_bit_for_bit(gpu, kind):
    """Rows whose tiles of keys all lie before an infinity (or a wide spread): 256
    rows of a head share their loads, in two tiles of 128."""
    clean = normal(1, heads=16, kv_heads=16)
    _, want = attend(gpu, kind, clean, 16, 16)
    for at, put in ((200, np.inf), (460, 1e30), (1000, -np.inf)):
        for which in (1, 2):
            data = [x.copy() for x in clean]
            data[which][at, 5::D] = put
            for _ in range(4):
                c, got = attend(gpu, kind, data, 16, 16)
                first = at // 128 * 128
                assert np.array_equal(got[:first], want[:first]), (at, put, which)


@KINDS
@pytest.mark.parametrize("scale", [1e6, 1e8, 1e12, 1e30], ids=str)
def test_a_large_key_leaves_the_rows_before_it(gpu, kind, scale):
    data = normal(2)
    data[1][400] *= scale
    c, out = attend(gpu, kind, data)
    check(c, data, out, [272, 300, 383, 384, 390, 399, 400, 401, 511, 900], [0, 3, 15])


@KINDS
@pytest.mark.parametrize("scale", [1e6, 1e12, 1e30], ids=str)
def test_a_large_key_across_the_query(gpu, kind, scale):
    """Large where every query is 0."""
    data = normal(3)
    data[0][:, 17::D] = 0
    data[1][400, 17::D] = scale
    data[1][700:, 17::D] = -scale
    c, out = attend(gpu, kind, data)
    check(c, data, out, [390, 399, 400, 401, 511, 699, 700, 1099], [0, 3, 15])


@KINDS
@pytest.mark.parametrize("scale", [1e6, 1e12, 1e30], ids=str)
def test_a_large_query_element_across_the_keys(gpu, kind, scale):
    """Large where every key is 0, in some rows."""
    data = normal(4)
    data[1][:, 17::D] = 0
    data[0][::3, 17::D] = scale
    c, out = attend(gpu, kind, data)
    check(c, data, out, [0, 1, 300, 301, 900, 901], [0, 3, 15])


@KINDS
def test_scales_whose_product_leaves_f32(gpu, kind):
    """Queries of 1e30 where keys are 0 and keys of 1e20 where queries are 0: the
    scores are ordinary.  And queries of 1e-36 before keys of 1e36."""
    data = normal(5)
    data[0][:, 0::D], data[1][:, 0::D] = 1e30, 0
    data[0][:, 1::D], data[1][:, 1::D] = 0, 1e20
    c, out = attend(gpu, kind, data)
    check(c, data, out, [0, 255, 256, 777, 1099], [0, 9, 15])
    data = normal(6)
    data[0] *= np.float32(1e-36)
    data[1] *= np.float32(1e36)
    c, out = attend(gpu, kind, data)
    check(c, data, out, [0, 255, 256, 777, 1099], [0, 9, 15], by_one=False)


@KINDS
@pytest.mark.parametrize("small", [1e-7, 1e-12, 1e-19, 1e-30], ids=str)
def test_small_values_beside_masked_ones(gpu, kind, small):
    data = normal(7)
    data[2][:700] *= np.float32(small)
    c, out = attend(gpu, kind, data)
    check(c, data, out, [0, 639, 640, 650, 699, 700, 1000], [0, 9, 15])


@KINDS
@pytest.mark.parametrize("scale", [1e5, 1e8, 1e12, 1e25], ids=str)
@pytest.mark.parametrize("columns", [(0,), (0, 1), (6, 7)], ids=str)
def test_large_columns_beside_ordinary_ones(gpu, kind, scale, columns):
    """Values that are large in one or two of every eight elements, in every row."""
    data = normal(8)
    for x in columns:
        data[2][:, x::8] *= np.float32(scale)
    c, out = attend(gpu, kind, data)
    check(c, data, out, [0, 100, 650, 1099], [0, 9, 15])


MANY = (64, 32)  # heads and kv heads of enough pieces that none is split: a split's parts have maxima of their own


def leveled(seed, levels, sizes):
    """Scores next to `levels` (per key, the same for every query), values of `sizes`."""
    q, k, v = normal(seed, len(levels), *MANY)
    q *= np.float32(0.3)
    k *= np.float32(0.3)
    q[:, 0::D] = math.sqrt(D)
    k[:, 0::D] = np.asarray(levels, np.float32)[:, None]
    v *= np.asarray(sizes, np.float32)[:, None]
    return [q, k, v]


@KINDS
@pytest.mark.parametrize("level,size", [(-14, 1e5), (-21, 1e8), (-26, 1e11), (-30, 1e12), (-60, 1e25)], ids=str)
def test_small_weights_of_large_values(gpu, kind, level, size):
    """One key holds nearly all the weight; a tile of others has weights of e^level
    on values so large that they count as much."""
    levels, sizes = np.full(1300, -80.0), np.ones(1300)
    levels[0] = 0
    levels[1024:1152], sizes[1024:1152] = level, size
    data = leveled(9, levels, sizes)
    c, out = attend(gpu, kind, data, *MANY)
    check(c, data, out, [1023, 1100, 1151, 1152, 1290], [0, 9, 63], by_one=False)
    # the same within a tile
    levels, sizes = np.full(1300, -80.0), np.ones(1300)
    levels[1030] = 0
    levels[1031:1150], sizes[1031:1150] = level, size
    data = leveled(10, levels, sizes)
    c, out = attend(gpu, kind, data, *MANY)
    check(c, data, out, [1029, 1030, 1100, 1151, 1290], [0, 9, 63])


@KINDS
@pytest.mark.parametrize("level", [-15, -25, -45], ids=str)
@pytest.mark.parametrize("size", [0.0, 1e-30], ids=["zero", "tiny"])
def test_a_key_of_most_weight_whose_value_is_zero(gpu, kind, level, size):
    """All of the output comes from keys of its tile with weights far below it."""
    levels, sizes = np.full(1300, -120.0), np.ones(1300)
    levels[1030], sizes[1030] = 0, size
    levels[1031:1150] = level
    data = leveled(11, levels, sizes)
    c, out = attend(gpu, kind, data, *MANY)
    check(c, data, out, [1031, 1100, 1149, 1151, 1290], [0, 9, 63])
    assert not np.isnan(out).any()


@KINDS
def test_values_of_zero(gpu, kind):
    data = normal(12)
    data[2][:] = 0
    c, out = attend(gpu, kind, data)
    assert (out == 0).all()
    data = normal(12)
    data[2][:, 3 * D:4 * D] = 0
    data[2][:, 7::D] = 0
    c, out = attend(gpu, kind, data)
    check(c, data, out, [0, 255, 256, 777, 1099], [0, 6, 7, 15], by_one=False)


@KINDS
@pytest.mark.parametrize("head", [64, 128])
def test_short_sequences_among_prompts(gpu, kind, head):
    """Sequences of a few keys packed with a prompt: large columns, large values in
    later rows, a large key; and ordinary ones, which no check sends the long way."""
    rng = np.random.default_rng(13)
    lens = [1500, 1, 2, 7, 9, 15, 17, 31, 32, 33, 40]
    starts = np.cumsum([0] + lens[:-1])
    total = sum(lens)
    q, k, v = (rng.standard_normal((total, w * head)).astype(np.float32) for w in (32, 8, 8))
    v[lens[0]:, 2::8] *= 1e12
    for a, n in zip(starts, lens):
        k[a + n // 2 + 1:a + n, 9::head] *= 1e12
    with Pair(gpu, kind, 32, 8, head, 16, total // 16 + 20, len(lens), 1500) as c:
        seqs = [c.open() for _ in lens]
        out = c.step(seqs, lens, [(q, k, v)], check=False)[0]
        for a, n in zip(starts, lens):
            check(c, [x[a:a + n] for x in (q, k, v)], out[a:a + n], sorted({0, n // 2, n - 1}), [0, 13, 31])
