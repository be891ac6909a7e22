"""MXFP4 operators at the ends of their ranges: rows of more values than 32 bits
count."""
import pytest
import torch

from tests.test_gpu_mxfp4 import DEV
from wisp.integrations.vllm import fused_moe_mxfp4 as mx

pytestmark = pytest.mark.gpu


def test_rows_longer_than_32_bits():
    """One row of 2^32 + 32 values: quantised and read back whole.  (Of each
    value's buffers the first stand in memory that held other bytes.)"""
    n = 2 ** 32 + 32
    for size in (n // 2, n // 32):
        torch.full((size,), 255, dtype=torch.uint8, device=DEV)
    w = torch.zeros(n, dtype=torch.bfloat16, device=DEV)
    for at, v in ((0, 3.0), (31, -0.5), (2 ** 31 - 1, 6.0), (2 ** 31, -1.5), (2 ** 32 - 1, 2.0),
                  (2 ** 32, -4.0), (n - 1, 1.0)):
        w[at] = v
    q, s = mx.quantize_mxfp4(w)
    assert q.shape == (n // 2,) and s.shape == (n // 32,)
    assert int((q != 0).sum()) == 7 and int((s != 0).sum()) == 5
    assert torch.equal(mx.dequantize_mxfp4(q, s), w)
