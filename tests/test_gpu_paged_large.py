"""A paged cache of more than 2^31 rows (small heads: 34 GB of them), used in its last
layer and pages."""
import numpy as np
import pytest

from kernrt_b200 import BF16

pytestmark = pytest.mark.gpu


def test_more_than_2_to_the_31_rows(gpu):
    layers, page, head, rows = 64, 128, 8, 9000
    n_pages = (1 << 31) // (2 * layers * page) + 200
    rng = np.random.default_rng(1)
    q, k, v = (gpu.upload(rng.standard_normal((rows, head)).astype(np.float32)) for _ in range(3))
    got = []
    for pages, fill, layer in ((n_pages, n_pages - 80, layers - 1), (80, 0, 0)):
        p = gpu.pages_create(BF16, layers if fill else 1, 1, 1, head, page, pages, 2, pages * page)
        try:
            filler, s = gpu.seq_open(p), gpu.seq_open(p)
            gpu.pages_step(p, [filler], [fill * page])
            out = gpu.alloc(rows * head)
            for n in (rows, 1):  # a prompt, a token
                gpu.pages_step(p, [s], [n])
                gpu.pages_write(p, layer, k, v)
                gpu.pages_attention(p, layer, q, out)
                got.append(gpu.read(out, n * head))
            if fill:
                assert gpu.seq_table(p, s)[0] == fill
            gpu.free(out)
        finally:
            gpu.pages_destroy(p)
    assert np.isfinite(got[0]).all() and np.array_equal(got[0], got[2])
    assert np.isfinite(got[1]).all() and np.array_equal(got[1], got[3])
    for h in (q, k, v):
        gpu.free(h)
