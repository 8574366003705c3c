"""Attention over the paged cache where the tensor cores' kernel takes it: many
query rows with much work (few rows, or little work, go to the single tokens'
kernel, tests/test_gpu_paged.py).  Held to the same definition and bound
(tests/_paged.py), on some rows and heads of each call."""
import numpy as np
import pytest

from kernrt_b200 import BF16, F32
from tests._paged import Pair

pytestmark = pytest.mark.gpu

KINDS = pytest.mark.parametrize("kind", [BF16, F32], ids=["bf16", "f32"])

# the work below which the single tokens' kernel is taken (backend.cu): groups of
# 8 query rows of a kv head x keys x kv heads x head, x 2.5 for f32 pages
FEW_WORK = 36 << 20


def work(kind, heads, kv_heads, head, ctx, new):
    rows = new * heads // kv_heads
    return -(-rows // 8) * (ctx + new // 2 + 1) * kv_heads * head * (2.5 if kind == F32 else 1)


def some_heads(heads):
    return sorted({0, 1, heads // 2, heads - 1})


# heads, kv heads, head size, page, ctx, new: tiles of 256 query rows and of 128 or
# 64 keys cut short everywhere, groups that share tiles and straddle them
CASES = [(48, 16, 64, 16, 0, 1027), (32, 32, 64, 32, 0, 1151), (16, 8, 128, 64, 0, 1500), (20, 4, 128, 128, 37, 1111),
         (40, 1, 128, 16, 2000, 300), (24, 24, 80, 32, 5, 900), (32, 32, 8, 16, 0, 3001), (18, 6, 104, 64, 129, 1023),
         (32, 16, 64, 64, 6001, 130), (16, 16, 128, 128, 9000, 65), (64, 16, 32, 16, 3000, 129),
         (12, 12, 72, 16, 127, 1409), (32, 8, 128, 64, 12345, 33), (16, 16, 120, 32, 0, 1279)]


@KINDS
@pytest.mark.parametrize("heads,kv_heads,head,page,ctx,new", CASES)
def test_shapes(gpu, kind, heads, kv_heads, head, page, ctx, new):
    assert work(kind, heads, kv_heads, head, ctx, new) > FEW_WORK
    rng = np.random.default_rng(heads + ctx + new)
    n_pages = (ctx + new) // page + 4
    with Pair(gpu, kind, heads, kv_heads, head, page, n_pages, 2, ctx + new) as c:
        s = c.open()
        if ctx:
            c.step([s], [ctx], [c.rows(rng, ctx)], check=False)
        c.step([s], [new], [c.rows(rng, new)], check_rows=9, heads=some_heads(heads))


@KINDS
def test_mixed_step(gpu, kind):
    """Prompts, chunks, single tokens and idle sequences in one step: both
    kernels write their rows of one output."""
    rng = np.random.default_rng(3)
    with Pair(gpu, kind, 16, 8, 128, 32, 400, 8, 4000) as c:
        a, b, d, e, f, g = [c.open() for _ in range(6)]
        c.step([b, a, d], [700, 33, 1900], [c.rows(rng, 2633)], check_rows=4, heads=[0, 9, 15])
        rows = [1257, 1, 0, 31, 2, 600]
        c.step([e, d, a, f, b, g], rows, [c.rows(rng, sum(rows))], check_rows=6, heads=[0, 9, 15])


@KINDS
def test_few_long_pieces_are_split_and_joined(gpu, kind):
    rng = np.random.default_rng(4)
    with Pair(gpu, kind, 4, 2, 128, 64, 500, 3, 30000) as c:
        a, b = c.open(), c.open()
        c.step([a, b], [24000, 500], [c.rows(rng, 24500)], check=False)
        seen = set()
        q, k, v = c.rows(rng, 450)
        c.step([a, b], [150, 300], [(q, k, v)], check_rows=8)
        # the same call again, bit for bit
        gpu.pages_step(c.p, [a, b], [150, 300])
        gpu.pages_write(c.p, 0, c.up(k), c.up(v))
        hq, out = c.up(q), c.up(np.zeros_like(q))
        for _ in range(10):
            gpu.pages_attention(c.p, 0, hq, out)
            seen.add(gpu.read(out, q.size).tobytes())
        assert len(seen) == 1


@KINDS
def test_forked_prompts(gpu, kind):
    """Chunks behind a shared prefix, in pages the children share and their own."""
    rng = np.random.default_rng(5)
    with Pair(gpu, kind, 24, 8, 64, 16, 600, 6, 3000) as c:
        a = c.open()
        c.step([a], [1500], [c.rows(rng, 1500)], check_rows=4, heads=[0, 23])
        kids = c.fork(a, 1234, 3)
        rows = [400, 401, 399, 300]
        c.step(kids + [a], rows, [c.rows(rng, sum(rows))], check_rows=5, heads=[0, 11, 23])
        c.end([kids[0]])
        gpu.pages_compact(c.p)
        c.step(kids[1:], [300, 500], [c.rows(rng, 800)], check_rows=5, heads=[0, 11, 23])


@KINDS
def test_masked_places_do_not_reach_a_row(gpu, kind):
    """NaN, infinities and huge values in recycled pages and in later positions
    of the same prompt; a NaN and an infinite query row among others."""
    rng = np.random.default_rng(6)
    heads = [0, 5, 15]
    with Pair(gpu, kind, 16, 8, 128, 64, 40, 3, 2500) as c:
        dirty = c.open()
        q, k, v = c.rows(rng, 2000)
        k[:], v[:] = np.nan, np.inf
        c.step([dirty], [2000], [(q, k, v)], check=False)
        c.end([dirty])
        s = c.open()
        c.step([s], [1100], [c.rows(rng, 1100)], check_rows=6, heads=heads)
        q, k, v = c.rows(rng, 700)
        q[100], q[333, 7] = np.nan, np.inf
        c.step([s], [700], [(q, k, v)], check_rows=29, heads=heads)  # rows 100, 325 .. among them
        c.trim(s, 1100)
        for put in (lambda: v.__setitem__((690, 3), np.inf), lambda: v.__setitem__((650, 70), np.nan),
                    lambda: k.__setitem__(600, np.nan), lambda: v.__setitem__(500, 3e38), lambda: k.__setitem__(400, -np.inf)):
            q, k, v = c.rows(rng, 700)
            put()
            c.step([s], [700], [(q, k, v)], check_rows=29, heads=heads)
            c.trim(s, 1100)


@KINDS
@pytest.mark.parametrize("scale", [1e-30, 1e-6, 1.0, 1e4, 1e15], ids=str)
def test_magnitudes(gpu, kind, scale):
    """Keys, queries and values of any size: scores far out of exp's range and
    near 0, values next to the largest, dimensions of very different size."""
    rng = np.random.default_rng(7)
    with Pair(gpu, kind, 16, 8, 128, 32, 80, 2, 2200) as c:
        s = c.open()
        q, k, v = c.rows(rng, 1800)
        k *= scale
        q *= min(1.0 / scale, 1e30)
        v *= np.repeat(np.float32(10.0) ** np.arange(8), 128)  # per kv head
        v[:, 5::128] *= 1e-4                                   # a small dimension of each
        q[:, 128:256] *= 20                                    # peaked
        q[:, 256:384] = 0
        c.step([s], [1800], [(q, k, v)], check_rows=12, heads=[0, 1, 2, 15])


@KINDS
def test_tiles_that_spread_too_far_for_one_scale(gpu, kind):
    """Key rows from 1e-25 to 1e25 side by side, values alike."""
    rng = np.random.default_rng(8)
    with Pair(gpu, kind, 16, 8, 128, 32, 40, 2, 1200) as c:
        s = c.open()
        q, k, v = c.rows(rng, 1100)
        k *= (10.0 ** rng.uniform(-25, 0, (1100, 1))).astype(np.float32)
        v *= (10.0 ** rng.uniform(-25, 25, (1100, 1))).astype(np.float32)
        c.step([s], [1100], [(q, k, v)], check_rows=10, heads=[0, 7, 15])


def test_offsets_past_32_bits(gpu):
    """A cache of more than 2^32 elements, used in its last layer and pages."""
    rng = np.random.default_rng(9)
    layers, page, kv_heads, head = 40, 64, 8, 128
    n_pages = (1 << 32) // (2 * layers * kv_heads * page * head) + 900
    b = gpu
    p = b.pages_create(BF16, layers, 16, kv_heads, head, page, n_pages, 4, (n_pages + 1) * page)
    try:
        from kernrt_b200.interop import pages_as_torch

        filler, s = b.seq_open(p), b.seq_open(p)
        b.pages_step(p, [filler], [(n_pages - 40) * page])
        rows = 1300
        q, k, v = (rng.standard_normal((rows, w)).astype(np.float32) for w in (2048, 1024, 1024))
        hs = [b.upload(x) for x in (q, k, v)]
        out = b.alloc(q.size)
        b.pages_step(p, [s], [rows])
        b.pages_write(p, layers - 1, hs[1], hs[2])
        b.pages_attention(p, layers - 1, hs[0], out)
        got = b.read(out, q.size).reshape(rows, 16, head)
        table = b.seq_table(p, s)
        assert table[0] == n_pages - 40
        # the same rows in a small cache, bit for bit
        with Pair(b, BF16, 16, kv_heads, head, page, 60, 2, 2000) as c:
            want = c.step([c.open()], [rows], [(q, k, v)], check_rows=2, heads=[0, 15])[0]
        assert np.array_equal(got, want)
        b.pages_step(p, [s], [1])  # a single token reads it, too
        h1 = [b.upload(x[:1]) for x in (q, k, v)]
        b.pages_write(p, layers - 1, h1[1], h1[2])
        b.pages_attention(p, layers - 1, h1[0], out)
        one = b.read(out, 2048)
        keys = np.concatenate([k, k[:1]]).reshape(-1, kv_heads, head)
        import torch
        kk, vv = (torch.from_numpy(np.concatenate([x, x[:1]])).to(torch.bfloat16).double().numpy().reshape(keys.shape)
                  for x in (k, v))
        x = kk[:, 0] @ q[0, :head].astype(np.float64) / head ** 0.5
        w = np.exp(x - x.max())
        assert np.allclose(one[:head], (w / w.sum()) @ vv[:, 0], atol=1e-5)
        # a copy on write, and a move, of the last layer's data
        child = b.seq_fork(p, s, rows, 1)[0]
        b.pages_step(p, [child], [1])
        view = pages_as_torch(b, p)
        b.synchronize()
        src, dst = int(b.seq_table(p, s)[rows // page]), int(b.seq_table(p, child)[rows // page])
        assert src != dst and torch.equal(view[-1, :, src, :, :rows % page], view[-1, :, dst, :, :rows % page])
        before = view[-1, :, [int(t) for t in b.seq_table(p, s)]].clone()
        b.seq_close(p, [filler])
        assert b.pages_compact(p) > 0
        b.synchronize()
        assert torch.equal(view[-1, :, [int(t) for t in b.seq_table(p, s)]], before)
        for h in hs + h1 + [out]:
            b.free(h)
    finally:
        b.pages_destroy(p)
