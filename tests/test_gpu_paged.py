"""Attention over the paged key/value cache against its definition in 64 bits
(tests/_paged.py has the bound and where it comes from)."""
import numpy as np
import pytest

import kernrt_b200
from kernrt_b200 import BF16, F32, KernrtCudaError
from tests._paged import Pair, rounded

pytestmark = pytest.mark.gpu

KINDS = pytest.mark.parametrize("kind", [BF16, F32], ids=["bf16", "f32"])


# heads, kv heads, head size, page size
SHAPES = [(4, 4, 64, 16), (8, 2, 128, 64), (6, 2, 64, 32), (3, 1, 128, 128), (16, 2, 64, 16), (5, 5, 8, 16), (4, 2, 80, 32),
          (9, 3, 104, 64), (40, 2, 32, 16)]


@KINDS
@pytest.mark.parametrize("heads,kv_heads,head,page", SHAPES)
def test_prompts_then_single_tokens(gpu, kind, heads, kv_heads, head, page):
    """Packed prompts of odd lengths, then two steps of single tokens."""
    lens = [1, page - 1, page, page + 1, 3 * page + 5, 200]
    rng = np.random.default_rng(heads * 1000 + head)
    with Pair(gpu, kind, heads, kv_heads, head, page, 200, 8, 1000) as c:
        seqs = [c.open() for _ in lens]
        c.step(seqs, lens, [c.rows(rng, sum(lens))], check_rows=12)
        for _ in range(2):
            c.step(seqs, [1] * len(seqs), [c.rows(rng, len(seqs))])


@KINDS
@pytest.mark.parametrize("ctx,new", [(0, 127), (0, 128), (0, 129), (0, 255), (0, 257), (100, 60), (1000, 3), (1000, 130),
                                     (1023, 1), (1024, 1), (1025, 2), (0, 700), (3000, 1), (513, 9), (2047, 17)])
def test_context_and_new_rows(gpu, kind, ctx, new):
    """A chunk of new rows behind a context, around the tiles' edges."""
    rng = np.random.default_rng(ctx + new)
    with Pair(gpu, kind, 6, 3, 64, 16, 300, 2, 4096) as c:
        s = c.open()
        if ctx:
            c.step([s], [ctx], [c.rows(rng, ctx)], check=False)
        c.step([s], [new], [c.rows(rng, new)], check_rows=20)


@KINDS
def test_mixed_step(gpu, kind):
    """Single tokens, chunks, whole prompts and sequences without rows in one
    step, over three layers, in an order other than that of their places."""
    rng = np.random.default_rng(5)
    with Pair(gpu, kind, 8, 4, 128, 32, 200, 9, 2000, layers=3) as c:
        a, b, d, e, f = [c.open() for _ in range(5)]
        c.step([b, a, d], [400, 33, 129], [c.rows(rng, 562) for _ in range(3)], check_rows=6)
        c.step([e, d, a, f, b], [257, 1, 0, 31, 2], [c.rows(rng, 291) for _ in range(3)], check_rows=6)
        c.step([a, b], [1, 1], [c.rows(rng, 2) for _ in range(3)])
        c.step([], [], [c.rows(rng, 0) for _ in range(3)])
        c.step([a, f], [0, 0], [c.rows(rng, 0) for _ in range(3)])


@KINDS
@pytest.mark.parametrize("n", [1, 3, 40, 200])
def test_many_sequences(gpu, kind, n):
    rng = np.random.default_rng(n)
    lens = [int(x) for x in rng.integers(1, 300, n)]
    with Pair(gpu, kind, 4, 2, 64, 16, 20 * n + 10, n, 400) as c:
        seqs = [c.open() for _ in lens]
        c.step(seqs, lens, [c.rows(rng, sum(lens))], check=False)
        c.step(seqs, [1] * n, [c.rows(rng, n)])


@KINDS
def test_long_context_splits(gpu, kind):
    """One sequence whose length is split over many CTAs, and new rows of a
    chunk over the same length."""
    rng = np.random.default_rng(11)
    with Pair(gpu, kind, 4, 1, 64, 64, 700, 2, 40000) as c:
        s = c.open()
        c.step([s], [40], [c.rows(rng, 40)], check=False)
        c.step([s], [30011], [c.rows(rng, 30011)], check=False)
        c.step([s], [1], [c.rows(rng, 1)])
        c.step([s], [5], [c.rows(rng, 5)])
        c.step([s], [150], [c.rows(rng, 150)], check_rows=5)


@KINDS
def test_page_contents_and_rounding(gpu, kind):
    """The cache holds k and v rounded to nearest even, ties and specials among
    them, and nothing else changes."""
    import torch

    from kernrt_b200.interop import pages_as_torch

    rng = np.random.default_rng(12)
    with Pair(gpu, kind, 2, 2, 16, 16, 8, 2, 64) as c:
        view = pages_as_torch(gpu, c.p)
        s, other = c.open(), c.open()
        c.step([other], [20], [c.rows(rng, 20)], check=False)
        c.step([s], [18], [c.rows(rng, 18)], check=False)
        gpu.synchronize()
        before = view.clone()
        q, k, v = c.rows(rng, 5)
        k[0, :8] = [1.00390625, 1.01171875, -1.00390625, np.inf, -np.inf, np.nan, 3.4e38, 1e-45]  # 1 + 2^-8: a tie
        c.step([s], [5], [(q, k, v)], check=False)
        gpu.synchronize()
        t = gpu.seq_table(c.p, s).tolist()
        assert t == [2, 3]
        got = view.double().cpu().numpy()
        for i in range(5):
            pos = 18 + i
            for kv, x in ((0, k), (1, v)):
                want = rounded(x[i], kind).reshape(2, 16)
                assert np.array_equal(got[0, kv, t[pos // 16], :, pos % 16], want, equal_nan=True)
        after = view.clone()
        after[0, :, 3, :, 2:7] = before[0, :, 3, :, 2:7]
        raw = torch.int32 if kind == F32 else torch.int16
        assert torch.equal(after.view(raw), before.view(raw))


@KINDS
def test_forks_share_and_diverge(gpu, kind):
    """Forks of one prompt, of a fork, at lengths inside and at the end of
    pages; parents that go on; copies; trims; a closed parent; compaction."""
    rng = np.random.default_rng(21)

    def go(seqs, rows):
        c.step(seqs, rows, [c.rows(rng, sum(rows)) for _ in range(2)], check_rows=8)

    with Pair(gpu, kind, 4, 2, 64, 16, 60, 12, 300, layers=2) as c:
        a = c.open()
        go([a], [75])
        free = gpu.pages_ptr(c.p).available
        kids = c.fork(a, 75, 3) + c.fork(a, 64, 1) + c.fork(a, 7, 1)
        assert gpu.pages_ptr(c.p).available == free, "a fork takes no pages"
        go([a] + kids, [1, 2, 1, 30, 1, 1])
        grand = c.fork(kids[0], 70, 2)
        go(grand + [kids[0]], [1, 5, 1])
        d = c.copy(kids[2], 90)
        go([d, kids[2]], [3, 3])
        c.trim(a, 40)
        go([a], [25])
        c.end([kids[1], grand[0]])
        moved = gpu.pages_compact(c.p)
        assert moved > 0
        info = gpu.pages_ptr(c.p)
        used = {int(p) for s in c.kv for p in gpu.seq_table(c.p, s)}
        assert used == set(range(int(info.n_pages - info.available)))
        go(list(c.kv), [1] * len(c.kv))
        assert gpu.pages_compact(c.p) == 0
        go(list(c.kv), [1] * len(c.kv))


@KINDS
@pytest.mark.parametrize("new", [1, 4, 150], ids=["token", "tokens", "prompt"])
def test_masked_places_do_not_reach_a_row(gpu, kind, new):
    """NaN and infinities in recycled pages, behind a fork's length, and in
    later positions of the same prompt leave the rows that cannot see them as
    they would be without."""
    rng = np.random.default_rng(31 + new)
    with Pair(gpu, kind, 4, 2, 64, 64, 40, 6, 700) as c:
        dirty = c.open()
        q, k, v = c.rows(rng, 640)
        k[:], v[:] = np.nan, np.inf
        c.step([dirty], [640], [(q, k, v)], check=False)
        c.end([dirty])
        s = c.open()
        c.step([s], [70], [c.rows(rng, 70)])  # takes the dirty pages
        parent = c.fork(s, 70)[0]
        q, k, v = c.rows(rng, 5)
        v[2:] = np.nan
        c.step([parent], [5], [(q, k, v)])
        child = c.fork(parent, 72)[0]  # the parent's NaN rows lie behind it
        q, k, v = c.rows(rng, 2 * new)
        if new > 1:  # in the last rows of each sequence: seen by those alone
            for at in (new - 1, 2 * new - 1):
                v[at, 3], v[at, 70] = np.inf, np.nan
                k[at, 5] = np.nan if at > new else 1.0
        c.step([child, s], [new, new], [(q, k, v)], check_rows=24)


@KINDS
@pytest.mark.parametrize("new", [1, 200], ids=["token", "prompt"])
def test_scores_of_every_size(gpu, kind, new):
    """Scores far below and above exp's range, a run of keys that score -inf, a
    row where every key does (no distribution: NaN), values near the largest."""
    rng = np.random.default_rng(41 + new)
    with Pair(gpu, kind, 4, 4, 64, 16, 80, 3, 700) as c:
        s = c.open()
        q, k, v = c.rows(rng, 300)
        c.step([s], [300], [(q, 30 * k, v)], check_rows=10)
        q, k, v = c.rows(rng, new)
        q[:, 64:128] = 0.0         # head 1: uniform weights
        q[:, 128:192] *= 1e-30     # head 2: tiny scores
        v[:, 192:256] *= 1e37      # head 3: large values
        c.step([s], [new], [(8 * q, k, v)], check_rows=10)
        t = c.open()
        q, k, v = c.rows(rng, 40)
        q[:] = np.abs(q)
        k[:20] = -np.inf
        c.step([t], [40], [(q, k, v)])
        q, k, v = c.rows(rng, new)
        q[:] = np.abs(q)
        c.step([t], [new], [(q, k, v)], check_rows=10)


@KINDS
def test_step_by_step_equals_one_prompt(gpu, kind):
    """The same tokens as one prompt, in chunks, and one by one hold the same
    cache bit for bit and agree in their last row."""
    from kernrt_b200.interop import pages_as_torch

    rng = np.random.default_rng(51)
    with Pair(gpu, kind, 4, 2, 64, 16, 60, 4, 300) as c:
        q, k, v = c.rows(rng, 150)
        for chunks in ([150], [1] * 150, [64, 5, 81], [149, 1]):
            s = c.open()
            at = 0
            for n in chunks:
                out = c.step([s], [n], [(q[at:at + n], k[at:at + n], v[at:at + n])], check=at + n == 150, check_rows=3)
                at += n
            gpu.synchronize()
            pages = pages_as_torch(gpu, c.p)[0][:, gpu.seq_table(c.p, s).tolist()].float().cpu().numpy()
            rows = pages.transpose(0, 1, 3, 2, 4).reshape(2, -1, 2, 64)[:, :150]
            if len(chunks) == 1:
                first, last = rows, out[0][-1]
            assert np.array_equal(rows, first)
            assert np.allclose(out[0][-1], last, rtol=0, atol=1e-4)


def test_repeated_calls_give_the_same_bits(gpu):
    """Splits join in a fixed order: no result depends on which CTA came last."""
    rng = np.random.default_rng(61)
    with Pair(gpu, BF16, 8, 2, 128, 16, 700, 9, 3000) as c:
        seqs = [c.open() for _ in range(9)]
        lens = [2900, 1, 17, 900, 64, 1000, 5, 2000, 300]
        c.step(seqs, lens, [c.rows(rng, sum(lens))], check=False)
        rows = [1, 3, 40, 1, 1, 90, 1, 1, 1]
        q, k, v = c.rows(rng, sum(rows))
        gpu.pages_step(c.p, seqs, rows)
        gpu.pages_write(c.p, 0, c.up(k), c.up(v))
        hq, out = c.up(q), c.up(np.zeros_like(q))
        seen = set()
        for _ in range(20):
            gpu.pages_attention(c.p, 0, hq, out)
            seen.add(gpu.read(out, q.size).tobytes())
        assert len(seen) == 1


def test_two_caches_and_two_contexts_at_once(gpu):
    """A draft's and a model's cache interleaved in one context, and a second
    context whose stream runs beside it."""
    rng = np.random.default_rng(71)
    with kernrt_b200.CudaBackend(0) as other, Pair(gpu, BF16, 4, 2, 64, 16, 80, 2, 600) as a, \
            Pair(gpu, F32, 2, 2, 32, 32, 80, 2, 600) as b, Pair(other, BF16, 4, 2, 64, 16, 80, 2, 600) as d:
        todo = [(c, c.open(), c.rows(rng, 500)) for c in (a, b, d)]
        outs = []
        for c, s, (q, k, v) in todo:
            c.b.pages_step(c.p, [s], [500])
            outs.append([c.up(q), c.up(k), c.up(v), c.up(np.zeros_like(q))])
        for _ in range(5):
            for (c, s, _), (q, k, v, out) in zip(todo, outs):
                c.b.pages_write(c.p, 0, k, v)
                c.b.pages_attention(c.p, 0, q, out)
        got = [c.b.read(o[3], x[0].size).reshape(x[0].shape) for (c, s, x), o in zip(todo, outs)]
        for (c, s, x), g in zip(todo, got):
            t = c.open()
            assert np.array_equal(c.step([t], [500], [x], check_rows=4)[0].reshape(g.shape), g)


def test_refusals(gpu):
    b = gpu
    good = (BF16, 1, 4, 2, 64, 16, 8, 3, 60)
    for bad in [(2,) + good[1:], (BF16, 0) + good[2:], (BF16, 1, 4, 3) + good[4:], (BF16, 1, 4, 2, 60) + good[5:],
                (BF16, 1, 4, 2, 136) + good[5:], (BF16, 1, 4, 2, 64, 8) + good[6:], (BF16, 1, 4, 2, 64, 48) + good[6:],
                good[:6] + (0, 3, 60), good[:6] + (8, 0, 60), good[:6] + (8, 3, 0), good[:6] + (2 ** 40, 3, 60),
                good[:7] + (2 ** 20, 60), good[:8] + (2 ** 40,), (BF16, 2 ** 15, 4, 2, 64, 128, 2 ** 20, 3, 60)]:
        with pytest.raises(KernrtCudaError) as e:
            b.pages_create(*bad)
        assert e.value.code == kernrt_b200.E_INVALID, bad
    with Pair(b, *good[:1], *good[2:], layers=2) as c:
        s = c.open()
        q, k, v, out = (c.up(np.zeros((4, w), np.float32)) for w in (256, 128, 128, 256))
        small = c.up(np.zeros(300, np.float32))

        def refused(code, call):
            with pytest.raises(KernrtCudaError) as e:
                call()
            assert e.value.code == code, str(e.value)

        invalid, state = kernrt_b200.E_INVALID, kernrt_b200.E_STATE
        refused(state, lambda: b.pages_write(c.p, 0, k, v))
        refused(state, lambda: b.pages_attention(c.p, 0, q, out))
        refused(invalid, lambda: b.pages_step(c.p, [s, s], [1, 1]))
        refused(invalid, lambda: b.pages_step(c.p, [s], [61]))
        refused(invalid, lambda: b.pages_step(c.p, [s + 1], [1]))
        refused(invalid, lambda: b.pages_step(c.p, [s], [2 ** 63]))
        refused(invalid, lambda: b.pages_step(c.p + 99, [s], [1]))
        refused(invalid, lambda: b.seq_open(0))
        b.pages_step(c.p, [s], [4])
        refused(invalid, lambda: b.pages_write(c.p, 2, k, v))
        refused(invalid, lambda: b.pages_write(c.p, 0, k, small))
        refused(invalid, lambda: b.pages_attention(c.p, 0, q, q))
        refused(invalid, lambda: b.pages_attention(c.p, 0, q, small))
        refused(invalid, lambda: b.pages_attention(c.p, 0, small, out))
        refused(invalid, lambda: b.pages_attention(c.p, 0, q, 10 ** 9))
        b.pages_attention(c.p, 1, q, out)
        refused(invalid, lambda: b.seq_fork(c.p, s, 5))
        refused(state, lambda: b.seq_fork(c.p, s, 4, 3))
        b.pages_attention(c.p, 1, q, out)  # a refused fork leaves the step as it is
        b.seq_fork(c.p, s, 4, 1)
        refused(state, lambda: b.pages_attention(c.p, 1, q, out))
        b.pages_step(c.p, [s], [1])
        b.seq_trim(c.p, s, 4)
        refused(state, lambda: b.pages_write(c.p, 1, k, v))
        t = c.open()
        b.pages_step(c.p, [t, s], [56, 30])
        refused(state, lambda: b.pages_step(c.p, [s], [26]))  # eight pages in all
        b.seq_close(c.p, [s])
        refused(invalid, lambda: b.seq_close(c.p, [s]))
        refused(invalid, lambda: b.seq_trim(c.p, s, 0))
        refused(invalid, lambda: b.seq_table(c.p, s))
        refused(invalid, lambda: b.seq_copy(c.p, t, 57))
    with pytest.raises(KernrtCudaError):
        b.seq_open(c.p)  # destroyed


@KINDS
def test_layer_calls_replay_in_a_graph(gpu, kind):
    """A step's layer calls captured after its first attention call and replayed
    on new rows, two graphs over one cache's scratch, a prompt's and a token's
    pieces in both."""
    import torch

    from kernrt_b200.interop import as_torch

    rng = np.random.default_rng(81)
    with Pair(gpu, kind, 16, 8, 128, 32, 300, 4, 4000, layers=2) as c:
        a, b = c.open(), c.open()
        c.step([a, b], [1500, 900], [c.rows(rng, 2400) for _ in range(2)], check=False)
        lens = [700, 1]
        gpu.pages_step(c.p, [a, b], lens)
        rows = sum(lens)
        stream = torch.cuda.ExternalStream(gpu.stream())
        bufs, graphs = [], []
        for layer in range(2):
            hs = [c.up(x) for x in c.rows(rng, rows)] + [c.up(np.zeros((rows, 2048), np.float32))]
            bufs.append(hs)
            gpu.pages_write(c.p, layer, hs[1], hs[2])
            gpu.pages_attention(c.p, layer, hs[0], hs[3])
        gpu.synchronize()
        for layer, hs in enumerate(bufs):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=stream):
                gpu.pages_write(c.p, layer, hs[1], hs[2])
                gpu.pages_attention(c.p, layer, hs[0], hs[3])
            graphs.append(g)
        for _ in range(2):  # new rows through the graphs, then the plain calls
            want = []
            for hs in bufs:
                for h, x in zip(hs, c.rows(rng, rows)):
                    as_torch(gpu, h, x.shape).copy_(torch.from_numpy(x))
            torch.cuda.synchronize()
            for layer, hs in enumerate(bufs):
                gpu.pages_write(c.p, layer, hs[1], hs[2])
                gpu.pages_attention(c.p, layer, hs[0], hs[3])
                want.append(gpu.read(hs[3], rows * 2048))
                as_torch(gpu, hs[3], (rows * 2048,)).zero_()
            torch.cuda.synchronize()
            with torch.cuda.stream(stream):
                for g in graphs:
                    g.replay()
            torch.cuda.synchronize()
            for hs, w in zip(bufs, want):
                assert np.array_equal(gpu.read(hs[3], rows * 2048), w)


def test_calls_that_cannot_be_replayed_are_refused_in_a_capture(gpu):
    """They change nothing, and the capture goes on."""
    import torch

    from kernrt_b200.interop import as_torch

    rng = np.random.default_rng(83)
    with Pair(gpu, kernrt_b200.BF16, 4, 2, 64, 16, 60, 6, 300) as c:
        a, b = c.open(), c.open()
        c.step([a, b], [40, 20], [c.rows(rng, 60)])
        gpu.pages_step(c.p, [a, b], [1, 30])
        q, k, v = [c.up(x) for x in c.rows(rng, 31)]
        out, spare = c.up(np.zeros((31, 256), np.float32)), gpu.alloc(5)
        gpu.pages_write(c.p, 0, k, v)
        gpu.synchronize()
        free, stream = gpu.pages_ptr(c.p).available, torch.cuda.ExternalStream(gpu.stream())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            gpu.pages_write(c.p, 0, k, v)
            for call in (lambda: gpu.pages_attention(c.p, 0, q, out), lambda: gpu.pages_step(c.p, [a], [1]),
                         lambda: gpu.seq_copy(c.p, a, 10), lambda: gpu.pages_compact(c.p),
                         lambda: gpu.pages_destroy(c.p), lambda: gpu.free(spare),
                         lambda: gpu.pages_create(kernrt_b200.F32, 1, 1, 1, 8, 16, 2, 1, 16)):
                with pytest.raises(KernrtCudaError) as e:
                    call()
                assert e.value.code == kernrt_b200.E_STATE and "capture" in str(e.value)
        assert gpu.pages_ptr(c.p).available == free
        assert len(gpu.seq_table(c.p, a)) == 3 and len(gpu.seq_table(c.p, b)) == 4
        gpu.pages_attention(c.p, 0, q, out)  # the step stands
        want = gpu.read(out, 31 * 256)
        as_torch(gpu, out, (31 * 256,)).zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            g.replay()
        torch.cuda.synchronize()
        gpu.pages_attention(c.p, 0, q, out)
        assert np.array_equal(gpu.read(out, 31 * 256), want)
        gpu.free(spare)


def test_freed_memory_comes_back_zeroed(gpu):
    """A freed block serves the next allocation of its size, behind the work that
    still uses it."""
    for n in (10, 5000, 3 << 20):
        h = gpu.upload(np.full(n, 3.0, np.float32))
        other = gpu.upload(np.full(n, 2.0, np.float32))
        gpu.add_in_place(other, h, n)
        gpu.free(h)
        again = gpu.alloc(n)
        assert (gpu.read(again, n) == 0).all() and (gpu.read(other, n) == 5).all()
        gpu.free(again)
        gpu.free(other)
    # far more than is kept
    for _ in range(6):
        gpu.free(gpu.alloc_bytes(3 << 30))
    p = gpu.pages_create(BF16, 2, 4, 2, 64, 16, 100, 2, 1000)
    s = gpu.seq_open(p)
    gpu.pages_step(p, [s], [100])
    gpu.pages_destroy(p)
    q = gpu.pages_create(BF16, 2, 4, 2, 64, 16, 100, 2, 1000)
    from kernrt_b200.interop import pages_as_torch
    gpu.synchronize()
    assert not pages_as_torch(gpu, q).any()
    gpu.pages_destroy(q)


def test_free_waits_for_queued_work_and_ends_the_handle(gpu):
    a = np.arange(1000, dtype=np.float32)
    x, y = gpu.upload(a), gpu.upload(a)
    gpu.add_in_place(x, y, 1000)  # held back for fusion: free launches it first
    gpu.free(y)
    assert np.array_equal(gpu.read(x, 1000), 2 * a)
    for call in (lambda: gpu.read(y, 1), lambda: gpu.free(y), lambda: gpu.add_in_place(x, y, 1), lambda: gpu.free(0)):
        with pytest.raises(KernrtCudaError) as e:
            call()
        assert e.value.code == kernrt_b200.E_INVALID
    gpu.free(x)
