"""kernrt_cuda_logprobs against its definition in 64 bits.

The bound: x - m is exact to 2^-24 of itself; the sum of exponentials (each
within 2^-22 of its value, added in at most a few thousand f32 steps in a row: at
most 2^-24 * 4096 relative, far less in practice, taken as 2^-14) moves its
logarithm by that much; so a log probability is within 2^-14 + 2^-22 |value|.  The
entropy, sum p (L - x), is held to the same with (1 + entropy).
"""
import numpy as np
import pytest

import kernrt_b200
from kernrt_b200 import KernrtCudaError, TOP_MAX

pytestmark = pytest.mark.gpu


def plain(x, targets, top):
    x = x.astype(np.float64)
    with np.errstate(all="ignore"):
        m = x.max(1, keepdims=True)
        log_sum = np.log(np.exp(x - m).sum(1, keepdims=True))  # added to m it would vanish beside the largest logits
        logp = (x - m) - log_sum
        p = np.exp(logp)
        entropy = -np.where(p > 0, p * logp, 0.0).sum(1)
        entropy[np.isnan(logp).any(1)] = np.nan
        logp[np.isnan(log_sum[:, 0])] = np.nan
    order = np.argsort(np.where(np.isnan(x), -np.inf, -x) + 0.0, axis=1, kind="stable")[:, :top]
    return logp[np.arange(len(x)), targets], entropy, order, np.take_along_axis(logp, order, 1)


def call(b, x, targets, top, parts=("logprob", "entropy", "top")):
    rows, vocab = x.shape
    hx, ht = b.upload(x), b.upload_bytes(np.asarray(targets, np.int32))
    outs = [b.upload(np.full((rows + 1) * n, 7.0, np.float32)) for n in (1, 1, max(top, 1), max(top, 1))]
    top = top if "top" in parts else 0
    b.logprobs(hx, rows, vocab, ht if "logprob" in parts else 0, outs[0] if "logprob" in parts else 0,
               outs[1] if "entropy" in parts else 0, top, outs[2] if top else 0, outs[3] if top else 0)
    got = [b.read(outs[0], rows + 1), b.read(outs[1], rows + 1),
           b.read_bytes(outs[2], 4 * (rows + 1) * max(top, 1), np.int32), b.read(outs[3], (rows + 1) * max(top, 1))]
    seven = np.float32(7).view(np.int32)
    assert got[0][rows] == 7 and got[1][rows] == 7
    assert (got[2][rows * top:] == seven).all() and (got[3][rows * top:] == 7).all()
    for name, i in (("logprob", 0), ("entropy", 1)):
        if name not in parts:
            assert (got[i] == 7).all()
    for h in [hx, ht] + outs:
        b.free(h)
    return got[0][:rows], got[1][:rows], got[2][:rows * top].reshape(rows, top), got[3][:rows * top].reshape(rows, top)


def near(got, want, what):
    nan, inf = np.isnan(want), np.isinf(want)
    assert (np.isnan(got) == nan).all(), what
    assert (got[inf] == want[inf]).all(), what
    err = np.abs(got[~nan & ~inf] - want[~nan & ~inf])
    bound = 2.0 ** -14 + 2.0 ** -22 * np.abs(want[~nan & ~inf])
    assert (err <= bound).all(), f"{what}: {err.max():.3g}"


def check(b, x, targets, top):
    want = plain(x, targets, top)
    got = call(b, x, targets, top)
    near(got[0], want[0], "logprob")
    near(got[1], want[1], "entropy")
    assert np.array_equal(got[2], want[2]), "top ids"
    near(got[3], want[3], "top log probabilities")


@pytest.mark.parametrize("rows,vocab", [(1, 1), (1, 2), (3, 5), (2, 31), (7, 33), (1, 1000), (5, 1023), (2, 4097), (65, 8191),
                                        (1, 49152), (9, 65536), (1, 151936), (130, 3001), (2, 200003)])
@pytest.mark.parametrize("top", [0, 1, 20, TOP_MAX])
def test_rows_and_vocabularies(gpu, rows, vocab, top):
    rng = np.random.default_rng(rows * 7 + vocab)
    x = (3 * rng.standard_normal((rows, vocab))).astype(np.float32)
    check(gpu, x, rng.integers(0, vocab, rows), min(top, vocab))


@pytest.mark.parametrize("vocab", [100, 6000, 151936])
def test_ties_take_the_lowest_ids(gpu, vocab):
    """Logits of few distinct values (a quantised head): equal ones by id, -0 as +0."""
    rng = np.random.default_rng(vocab)
    x = rng.integers(-3, 3, (6, vocab)).astype(np.float32)
    x[1] = 0.0
    x[2] = np.where(rng.random(vocab) < 0.5, 0.0, -0.0)
    x[3] = -1.5
    x[3, vocab - 3:] = 2.0
    x[4] = np.arange(vocab) % 7
    x[5] = -np.arange(vocab)
    check(gpu, x, rng.integers(0, vocab, 6), min(vocab, TOP_MAX))


@pytest.mark.parametrize("vocab", [70, 5000, 151936])
def test_sorted_rows(gpu, vocab):
    """Ascending, descending, and the largest all in one place."""
    x = np.stack([np.linspace(-9, 9, vocab), np.linspace(9, -9, vocab), np.zeros(vocab)]).astype(np.float32)
    at = vocab // 2 - 8
    x[2, at:at + 40] = np.arange(40)[::-1] + 1
    check(gpu, x, [0, vocab - 1, at], 64)


def test_large_entries_spread_evenly_over_a_row(gpu):
    """Every stretch of the row holds one entry less than `top` of the largest, so
    that no stretch's list says much about the others'."""
    rng = np.random.default_rng(12)
    for vocab, every in ((151936, 1024), (600000, 1024), (600001, 2048)):
        x = rng.standard_normal((1, vocab)).astype(np.float32)
        at = np.arange(0, vocab - 64, every)[:, None] + np.arange(63)
        x[0, at.ravel()] = 100 + rng.permutation(at.size).astype(np.float32) / 64
        check(gpu, x, [5], 64)


@pytest.mark.parametrize("vocab", [49152, 600000, 2000001])
def test_many_candidates_every_time_alike(gpu, vocab):
    """Ascending rows (more entries reach the first bound than there is room for)
    and lists of many stretches (more than one batch of them in the join), over and
    over: threads that disagree about how many entries there are would show."""
    rng = np.random.default_rng(vocab)
    x = np.stack([np.arange(vocab) / 1024, rng.permutation(vocab) / 1024]).astype(np.float32)
    want = plain(x, [0, vocab - 1], 64)
    first = None
    for _ in range(20):
        got = call(gpu, x, [0, vocab - 1], 64)
        assert np.array_equal(got[2], want[2])
        first = first or got
        assert all(np.array_equal(a, b) for a, b in zip(got, first))
    near(first[0], want[0], "logprob")
    near(first[1], want[1], "entropy")
    near(first[3], want[3], "top log probabilities")


def test_masked_rows_and_rows_without_a_distribution(gpu):
    rng = np.random.default_rng(3)
    x = (3 * rng.standard_normal((9, 3001))).astype(np.float32)
    x[0, 5:] = -np.inf                # five tokens left
    x[1] = -np.inf
    x[1, 77] = -1e30                  # one
    x[2] = -np.inf                    # none
    x[3, 100] = np.nan
    x[4, [7, 2000]] = np.inf
    x[5, 9] = -np.nan
    x[6] = np.finfo(np.float32).min   # the type's lowest value everywhere: uniform
    x[7] = 3e38
    x[7, 1500:] = -3e38
    x[8, ::2] = -np.inf
    targets = [2, 77, 3, 4, 7, 9, 0, 1400, 8]
    got = call(gpu, x, targets, 40)
    want = plain(x, targets, 40)
    for r in range(9):
        for g, w, what in zip(got, want, ("logprob", "entropy", "ids", "tops")):
            if what == "ids":
                assert np.array_equal(g[r], w[r]), (r, what)
            else:
                near(np.atleast_1d(g[r]), np.atleast_1d(w[r]), (r, what))
    # a masked target has no probability
    assert call(gpu, x[:1], [9], 0, ("logprob",))[0][0] == -np.inf


@pytest.mark.parametrize("parts", [("logprob",), ("entropy",), ("top",), ("logprob", "top"), ("entropy", "top"), ()])
def test_parts_alone(gpu, parts):
    rng = np.random.default_rng(8)
    x = (3 * rng.standard_normal((3, 9999))).astype(np.float32)
    t = rng.integers(0, 9999, 3)
    whole = call(gpu, x, t, 10)
    got = call(gpu, x, t, 10, parts)
    for i, name in enumerate(("logprob", "entropy", "top", "top")):
        if name in parts:
            assert np.array_equal(got[i], whole[i])


def test_same_bits_every_time_and_wherever_the_row_stands(gpu):
    rng = np.random.default_rng(9)
    x = (3 * rng.standard_normal((1, 151936))).astype(np.float32)
    once = call(gpu, x, [5], 20)
    for _ in range(5):
        for a, b in zip(call(gpu, x, [5], 20), once):
            assert np.array_equal(a, b)


def test_target_outside_the_vocabulary(gpu):
    rng = np.random.default_rng(10)
    x = rng.standard_normal((4, 100)).astype(np.float32)
    hx, out = gpu.upload(x), gpu.alloc(4)
    gpu.logprobs(hx, 4, 100, gpu.upload_bytes(np.array([3, 100, -1, 99], np.int32)), out)
    with pytest.raises(KernrtCudaError) as e:
        gpu.synchronize()
    assert e.value.code == kernrt_b200.E_DEVICE
    got = gpu.read(out, 4)
    assert np.isnan(got[1:3]).all()
    near(got[[0, 3]], plain(x, [3, 0, 0, 99], 0)[0][[0, 3]], "the others")


def test_refusals(gpu):
    x, t = gpu.alloc(1000), gpu.alloc_bytes(40)
    o = [gpu.alloc(1000) for _ in range(4)]
    for args in [(x, 10, 101, t, o[0]), (x, 11, 100, t, o[0]), (x, 10, 0), (x, 10, 100, t, 0), (x, 10, 100, 0, o[0]),
                 (x, 10, 100, t, x), (x, 10, 100, t, o[0], o[0]), (x, 10, 100, t, t), (x, 10, 100, 0, 0, 0, 5),
                 (x, 10, 100, 0, 0, 0, 5, o[0], o[0]), (x, 10, 100, 0, 0, 0, 0, o[0], o[1]),
                 (x, 10, 100, 0, 0, 0, TOP_MAX + 1, o[0], o[1]), (x, 100, 10, 0, 0, 0, 11, o[0], o[1]),
                 (x, 10, 100, t, o[0], t), (99999, 1, 1, t, o[0]), (x, 2 ** 62, 100, t, o[0]), (x, 1, 2 ** 62, t, o[0]),
                 (x, 20, 50, t, o[0]), (x, 20, 50, 0, 0, 0, 50, gpu.alloc(999), o[1])]:
        with pytest.raises(KernrtCudaError) as e:
            gpu.logprobs(*args)
        assert e.value.code == kernrt_b200.E_INVALID, args
    gpu.logprobs(x, 0, 100, t, o[0], o[1], 3, o[2], o[3])  # no rows: nothing
    gpu.logprobs(x, 10, 100)                               # no outputs: nothing


def test_graphs_keep_their_scratch(gpu):
    """Captured calls of several sizes replay after larger calls have made larger
    scratch; a capture that would have to make some is refused."""
    import torch

    from kernrt_b200.interop import as_torch

    rng = np.random.default_rng(17)
    with kernrt_b200.CudaBackend(0) as b:
        stream = torch.cuda.ExternalStream(b.stream())

        def case(rows, vocab, top):
            x = (3 * rng.standard_normal((rows, vocab))).astype(np.float32)
            t = rng.integers(0, vocab, rows)
            hs = [b.upload(x), b.upload_bytes(t.astype(np.int32)), b.alloc(rows), b.alloc(rows), b.alloc(rows * top),
                  b.alloc(rows * top)]
            return hs, (rows, vocab, top), plain(x, t, top)

        def go(hs, size):
            b.logprobs(hs[0], size[0], size[1], hs[1], hs[2], hs[3], size[2], hs[4], hs[5])

        def held(hs, size, want):
            rows, _, top = size
            near(b.read(hs[2], rows), want[0], "logprob")
            near(b.read(hs[3], rows), want[1], "entropy")
            assert np.array_equal(b.read_bytes(hs[4], 4 * rows * top, np.int32).reshape(rows, top), want[2])

        cases = [case(1, 20000, 3), case(3, 49152, 20), case(5, 300001, 64)]
        graphs = []
        for hs, size, want in cases:
            go(hs, size)
            held(hs, size, want)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=stream):
                go(hs, size)
            graphs.append(g)
        big = case(40, 151936, 64)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            go(*cases[2][:2])
            with pytest.raises(KernrtCudaError) as e:
                go(*big[:2])
        assert e.value.code == kernrt_b200.E_STATE
        for _ in range(3):
            go(*big[:2])
            held(*big)
            spare = [b.alloc(n) for n in (4, 64, 1024, 16384)]  # where given-back scratch would go
            for hs, size, _ in cases:
                for h, n in zip(hs[2:], (size[0], size[0], size[0] * size[2], size[0] * size[2])):
                    as_torch(b, h, (n,)).zero_()
            torch.cuda.synchronize()
            with torch.cuda.stream(stream):
                for g in graphs:
                    g.replay()
            torch.cuda.synchronize()
            for c in cases:
                held(*c)
            for h, n in zip(spare, (4, 64, 1024, 16384)):
                assert not b.read(h, n).any()
                b.free(h)
