"""Edges of the gated recurrence, the norms around a block and 8-bit activations on CUDA: what a
call does with rows of the largest width, with values that are not finite, with outside
writes to its tensors and with arguments that it has to refuse."""
import pytest
import torch

pytestmark = pytest.mark.gpu
F32 = 5e-6  # relative, fp32 results against 64 bits: derived in test_gpu_gated.py


@pytest.mark.parametrize("H", [(1 << 31) - 1, (1 << 31) - 4, (1 << 31) - 40])
def test_codes_of_the_longest_rows(H):
    """Up to 2^31 - 1 values a row, the last group partly filled: both ends equal the same values alone."""
    from starry_unigraph.ops.checkpoint8 import Packed8, quantize8

    x = torch.randn(1 << 24, device="cuda", dtype=torch.bfloat16).repeat(1 << 7)[:H]
    q = quantize8(x)
    tail = H % 32
    want = quantize8(x[-tail:])
    assert q.codes.shape == (1, H) and q.scales.shape == (1, H // 32 + 1)
    assert torch.equal(q.codes[0, -tail:], want.codes[0]) and q.scales[0, -1] == want.scales[0, 0]
    n = 1 << 24  # the values repeat, and so do their codes
    for k in (0, 63, 126):
        assert torch.equal(q.codes[0, k * n:k * n + n].view(-1, 4096), quantize8(x[:n].view(-1, 4096)).codes)
    back = q.dequantize()
    assert torch.equal(back[-tail:], want.dequantize()) and torch.equal(back[:n], back[126 * n:127 * n])
    del x, back
    two = Packed8(q.codes.expand(2, H).contiguous(), q.scales.expand(2, -1).contiguous(), torch.Size((2, H)), torch.bfloat16)
    del q
    both = two.dequantize()
    assert torch.equal(both[0, -n:], both[1, -n:]) and torch.equal(both[0, :n], both[1, :n])
