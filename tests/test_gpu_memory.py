"""A device without memory left: what the context keeps of freed blocks goes back
first, and a call that still finds none fails and changes nothing.

KERNRT_CUDA_FAIL_MALLOC=n (read once when a context is created; unset, nothing is
injected) makes that context's n-th request for device memory find the device
exhausted the first time it asks.  No GPU fault is involved: the request is refused
on the host."""
import os

import numpy as np
import pytest

import kernrt_b200
from kernrt_b200 import BF16, F32, KernrtCudaError

pytestmark = pytest.mark.gpu


def context(n):
    os.environ["KERNRT_CUDA_FAIL_MALLOC"] = str(n)
    try:
        return kernrt_b200.CudaBackend(0)
    finally:
        del os.environ["KERNRT_CUDA_FAIL_MALLOC"]


def test_kept_memory_goes_back_to_the_device_when_asked():
    import torch

    with kernrt_b200.CudaBackend(0) as b:
        b.release_freed()  # nothing kept
        x = b.upload(np.ones(1000, np.float32))
        h = b.alloc_bytes(6 << 30)
        b.synchronize()
        held = torch.cuda.mem_get_info(0)[0]
        b.free(h)
        assert torch.cuda.mem_get_info(0)[0] < held + (1 << 30)  # kept
        b.release_freed()
        assert torch.cuda.mem_get_info(0)[0] > held + (5 << 30)
        assert (b.read(x, 1000) == 1).all()
        stream, g = torch.cuda.ExternalStream(b.stream()), torch.cuda.CUDAGraph()
        y = b.alloc(1000)
        b.synchronize()
        with torch.cuda.graph(g, stream=stream):
            b.copy(x, 0, y, 0, 1000)
            with pytest.raises(KernrtCudaError) as e:
                b.release_freed()
        assert e.value.code == kernrt_b200.E_STATE


MATRIX = np.arange(64 * 32, dtype=np.float32).reshape(64, 32)
CALLS = {
    "alloc": lambda b: b.alloc(5000),
    "kv_prepare, keys": lambda b: b.kv_prepare(2, 64, 128),
    "kv_prepare, values": lambda b: b.kv_prepare(2, 64, 128),
    "prepare_matrix": lambda b: b.prepare_matrix(F32, MATRIX, None, 64, 32),
    "prepare_embedding": lambda b: b.prepare_embedding(F32, MATRIX, None, 64, 32),
    "pages_create": lambda b: b.pages_create(BF16, 1, 2, 1, 64, 16, 100, 4, 400),
}


@pytest.mark.parametrize("name", CALLS)
def test_kept_blocks_go_back_before_a_call_fails(name):
    at = 3 if "values" in name else 2
    with context(at) as b:
        b.free(b.alloc(1 << 20))  # request 1; the block is kept
        CALLS[name](b)
        b.synchronize()
    with context(at - 1) as b:  # nothing kept
        with pytest.raises(KernrtCudaError) as e:
            CALLS[name](b)
        assert e.value.code == kernrt_b200.E_CUDA and "memory" in str(e.value)
        CALLS[name](b)  # there is some again
        b.synchronize()


@pytest.mark.parametrize("part", [0, 1], ids=["keys", "values"])
def test_a_key_value_cache_whose_allocation_fails_is_not_there(part):
    """Nor the one before it, whose memory is gone."""
    rows = np.random.default_rng(1).standard_normal((3, 64)).astype(np.float32)
    with context(4 + part) as b:
        hk, hv = b.upload(rows), b.upload(-rows)  # requests 1 and 2
        hs = hk, hv, b.alloc(3 * 64)              # 3
        q, out, att = hs[0], hs[2], None
        with pytest.raises(KernrtCudaError) as e:
            b.kv_prepare(1, 64, 8)
        assert e.value.code == kernrt_b200.E_CUDA
        att = b.alloc(3 * 8)

        def write():
            b.kv_write(0, [0, 1, 2], hk, hv, 3)

        def attend():
            b.attention(q, out, att, 0, [(0, i, 0, 0) for i in range(3)], 1, 1, 64, 64, 8)

        for call in (write, attend):
            with pytest.raises(KernrtCudaError) as e:
                call()
            assert e.value.code == kernrt_b200.E_STATE
        b.kv_prepare(1, 64, 8)
        write()
        attend()
        assert np.array_equal(b.read(out, 64), -rows[0])  # one key: its value


@pytest.mark.parametrize("part", [0, 1], ids=["codes", "scales"])
def test_an_embedding_whose_allocation_fails_is_not_there(part):
    """Nor the one before it, whose memory is gone."""
    table = np.random.default_rng(2).standard_normal((8, 32)).astype(np.float32)
    codes, scales = np.arange(8 * 32, dtype=np.int8), np.ones(8, np.float32)
    with context(3 + part) as b:
        x = b.alloc(32)                                     # request 1
        b.prepare_embedding(F32, table, None, 8, 32)        # 2
        b.embed(5, x, 0)
        assert np.array_equal(b.read(x, 32), table[5])
        with pytest.raises(KernrtCudaError) as e:
            b.prepare_embedding(kernrt_b200.Q8_0, codes, scales, 8, 32)
        assert e.value.code == kernrt_b200.E_CUDA
        with pytest.raises(KernrtCudaError) as e:
            b.embed(5, x, 0)
        assert e.value.code == kernrt_b200.E_STATE
        b.prepare_embedding(kernrt_b200.Q8_0, codes, scales, 8, 32)
        b.embed(5, x, 0)
        assert np.array_equal(b.read(x, 32), codes.reshape(8, 32)[5].astype(np.float32))


def test_staging_that_cannot_grow_stays_as_it_was():
    """More rows' tokens in one call than the staging ring takes: it grows; a call
    that finds no memory for that fails, and smaller ones go on as before."""
    rows, dim, seq = 60000, 4, 60000
    k = np.random.default_rng(3).standard_normal((rows, dim)).astype(np.float32)
    with context(6) as b:
        hk, hv = b.upload(k), b.upload(-k)     # requests 1 and 2
        out = b.alloc(dim)                      # 3
        b.kv_prepare(1, dim, seq)               # 4 and 5
        with pytest.raises(KernrtCudaError) as e:
            b.kv_write(0, np.arange(rows), hk, hv, rows)
        assert e.value.code == kernrt_b200.E_CUDA
        att = b.alloc(seq)
        for n in (3, 1000, rows):
            for _ in range(20):  # around the ring
                b.kv_write(0, np.arange(rows - n, rows), hk, hv, n)
                b.synchronize()
            b.attention(hk, out, att, 0, [(rows - n, rows - n, 0, 0)], 1, 1, dim, dim, seq)
            assert np.array_equal(b.read(out, dim), -k[0])


def pages(b, n_pages, max_seqs, page=16, max_len=400000):
    from kernrt_b200.interop import pages_as_torch

    p = b.pages_create(F32, 1, 1, 1, 8, page, n_pages, max_seqs, max_len)  # requests 1 to 3
    b.synchronize()
    return p, pages_as_torch(b, p)[0, :, :, 0]  # [K or V, page, position, 8]


def write(b, p, rows, start):
    """Rows start, start + 1 .. of K (and their negatives of V) into the step."""
    k = np.repeat(np.arange(start, start + rows, dtype=np.float32), 8)
    hk, hv = b.upload(k), b.upload(-k)
    b.pages_write(p, 0, hk, hv)
    b.synchronize()


def content(view, table, length):
    k, v = view[:, table.tolist()].reshape(2, -1, 8)[:, :length].cpu().numpy()
    assert np.array_equal(k, -v) and (k == k[:, :1]).all()
    return k[:, 0].astype(int).tolist()


def fails(call):
    with pytest.raises(KernrtCudaError) as e:
        call()
    assert e.value.code == kernrt_b200.E_CUDA and "staging" in str(e.value)


def test_a_step_that_cannot_be_enqueued_changes_nothing():
    """4,000 forks of five positions take a copy each of their shared page: more than
    a segment of the staging ring, which finds no memory to grow."""
    n = 4000
    with context(6) as b:
        p, view = pages(b, n + 10, n + 2)
        s = b.seq_open(p)
        b.pages_step(p, [s], [5])
        write(b, p, 5, 100)  # requests 4 and 5
        kids = b.seq_fork(p, s, 5, n)
        free, table = b.pages_ptr(p).available, b.seq_table(p, s).tolist()
        fails(lambda: b.pages_step(p, kids, [1] * n))
        assert b.pages_ptr(p).available == free
        for q in [s, kids[0], kids[1], kids[-1]]:
            assert b.seq_length(p, q) == 5 and b.seq_table(p, q).tolist() == table
        b.pages_step(p, kids, [1] * n)  # there is memory again
        write(b, p, n, 1000)
        for i in (0, 1, 777, n - 1):
            assert content(view, b.seq_table(p, kids[i]), 6) == [100, 101, 102, 103, 104, 1000 + i]
        assert content(view, b.seq_table(p, s), 5) == [100, 101, 102, 103, 104]
        assert len({int(b.seq_table(p, q)[0]) for q in kids + [s]}) == n + 1


def test_a_step_that_cannot_be_enqueued_leaves_the_one_before_it():
    n = 4000
    with context(6) as b:
        p, view = pages(b, n + 10, n + 2)
        s, t = b.seq_open(p), b.seq_open(p)
        b.pages_step(p, [s], [5])
        write(b, p, 5, 100)  # requests 4 and 5
        kids = b.seq_fork(p, s, 5, n)
        b.pages_step(p, [t], [3])
        fails(lambda: b.pages_step(p, kids, [1] * n))
        write(b, p, 3, 7)  # t's rows
        assert content(view, b.seq_table(p, t), 3) == [7, 8, 9]
        assert content(view, b.seq_table(p, kids[5]), 5) == [100, 101, 102, 103, 104]


def test_a_copy_that_cannot_be_enqueued_opens_no_sequence():
    length = 16 * 11000 + 3  # as many page copies do not fit the ring
    with context(6) as b:
        p, view = pages(b, 22010, 3)
        s = b.seq_open(p)
        b.pages_step(p, [s], [length])
        write(b, p, length, 0)  # requests 4 and 5
        free = b.pages_ptr(p).available
        fails(lambda: b.seq_copy(p, s, length))
        assert b.pages_ptr(p).available == free
        write(b, p, length, 1)  # the step stands
        others = [b.seq_copy(p, s, length), b.seq_open(p)]  # both places are free
        b.synchronize()
        assert content(view, b.seq_table(p, others[0]), length) == list(range(1, length + 1))
        with pytest.raises(KernrtCudaError):
            b.seq_open(p)


def test_a_compaction_that_cannot_be_enqueued_moves_nothing():
    length = 16 * 11000 + 3
    with context(6) as b:
        p, view = pages(b, 22010, 3)
        gone, s = b.seq_open(p), b.seq_open(p)
        b.pages_step(p, [gone, s], [length, 3])
        b.seq_close(p, [])
        b.pages_step(p, [s], [length - 3])
        write(b, p, length - 3, 3)  # requests 4 and 5
        b.seq_close(p, [gone])
        free, table = b.pages_ptr(p).available, b.seq_table(p, s).tolist()
        fails(lambda: b.pages_compact(p))
        assert b.pages_ptr(p).available == free and b.seq_table(p, s).tolist() == table
        assert content(view, b.seq_table(p, s), length)[3:] == list(range(3, length))
        assert b.pages_compact(p) == 11001
        b.synchronize()
        assert sorted(b.seq_table(p, s).tolist()) == list(range(11001))
        assert content(view, b.seq_table(p, s), length)[3:] == list(range(3, length))
