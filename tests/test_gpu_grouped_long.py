"""Expert products whose sums or tiles are many."""
from __future__ import annotations

import pytest
import torch

import spmm_b200 as S

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def stream():
    return torch.cuda.current_stream()


def test_weights_gradient_of_a_group_that_takes_longer_than_a_wait(cuda):
    """One block sums 64 million rows, which takes about a second. Values are -1, 0 and 1, so every sum is a whole number far
    below 2^24 and exact in whatever order."""
    rows = 64 << 20
    g = torch.Generator(device="cuda").manual_seed(1)
    dy, x = (torch.randint(-1, 2, (rows, 1), generator=g, device="cuda", dtype=torch.int8).to(BF16) for _ in range(2))
    dw = torch.full((2, 1, 1), float("nan"), device="cuda")
    offsets = torch.tensor([0, rows - 3, rows], dtype=torch.int32, device="cuda")
    S.grouped_mm_dw(offsets, dy, x, dw, stream=stream())
    torch.cuda.synchronize()
    assert S.device_error(0)[0] == 0
    prod = dy.flatten() * x.flatten()
    assert float(dw[0]) == float(prod[:rows - 3].double().sum()) and float(dw[1]) == float(prod[rows - 3:].double().sum())
