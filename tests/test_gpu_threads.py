"""A thread's first call of the library, on tensors that another thread made."""
import threading

import pytest
import torch

import block_scaled_cases as K
from vllm_gcu_b200.ops import cuda as C

pytestmark = pytest.mark.gpu


def _in_a_thread(call):
    got = []

    def work():
        try:
            got.append(call())
        except Exception as e:                            # (an exception of a thread alone would be lost)
            got.append(e)
    t = threading.Thread(target=work)
    t.start()
    t.join()
    assert not isinstance(got[0], Exception), got[0]
    return got[0]


@pytest.mark.parametrize("D", [64, 128])
def test_a_thread_that_begins_with_attention(D):
    cache = K.Cache(K.FP8, 2, D, 16, [300, 40]).to("cuda")
    q = torch.randn(2, 8, D, device="cuda", dtype=K.BF16)
    out = torch.empty_like(q)
    args = (q, *cache.parts(), cache.tables, cache.seq_lens, 0.1)
    want = C.block_scaled_decode(*args, num_splits=1)
    got = _in_a_thread(lambda: C.block_scaled_decode(*args, num_splits=1, out=out))
    assert torch.equal(got, want)


@pytest.mark.parametrize("M", [1, 64, 512])
def test_a_thread_that_begins_with_a_matrix_product(M):
    x, w = (torch.randn(n, 512, device="cuda", dtype=K.BF16) for n in (M, 1024))
    want = C.gemm_bf16(x, w)
    assert torch.equal(_in_a_thread(lambda: C.gemm_bf16(x, w)), want)
