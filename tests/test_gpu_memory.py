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
