"""Attention of many query rows over keys, queries and values of very different
size: what is large, masked or infinite in one place leaves the rest of its tile
as it is by the definition.
"""
import numpy as np
import pytest

from kernrt_b200 import BF16, F32
from tests._paged import Pair

pytestmark = pytest.mark.gpu

KINDS = pytest.mark.parametrize("kind", [BF16, F32], ids=["bf16", "f32"])
D = 128


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
