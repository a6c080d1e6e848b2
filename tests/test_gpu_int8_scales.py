"""8-bit products whose scales are as far apart as 32 bits allow."""

import pytest
import torch

from conftest import device
from plain_int8 import check_product, product
from test_gpu_int8 import operands, run
from test_gpu_kernels import K

pytestmark = [pytest.mark.gpu, pytest.mark.needs_cuda]


# tiles of 16 to 128 tokens, alone and shared, pairs, and rows anywhere
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,N,k,pad", [(5, 300, 400, 0), (16, 1000, 4096, 0), (30, 2000, 8208, 0), (33, 384, 1040, 0), (125, 6100, 2064, 0),
                                       (300, 4090, 2064, 0), (513, 6200, 1040, 0), (33, 65, 77, 1)])
def test_results_that_32_bits_hold_of_sums_that_they_do_not(M, N, k, pad, dtype):
    """Tokens of every size beside channels that bring them back: the sum times the token's scale alone would be infinite."""
    x, xs, w, ws = operands(M * N + k, M, N, k, (pad, pad))
    sizes = torch.tensor([0.0, 60.0, 95.0, 97.0, 115.0, 120.0, 127.0, -60.0, -100.0], device=device())
    xs = torch.exp2(sizes[torch.arange(M, device=device()) % 9]) * (1 + torch.rand(M, device=device()) * 0.5)
    ws = ws * torch.exp2(torch.tensor([-60.0, -30.0, -20.0, -14.0], device=device())[torch.arange(N, device=device()) % 4])
    ref, size = product(x, xs, w, ws)
    holds = ref.abs() < 3.3e38
    got = run(x, xs, w, ws, dtype)
    assert holds.float().mean() > 0.9
    check_product(got[holds], ref[holds], size[holds])
