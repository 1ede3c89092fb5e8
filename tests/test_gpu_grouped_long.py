"""Expert products whose sums or tiles are many, and offsets that are wrong where tiles are taken over."""
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


@pytest.mark.parametrize("form", ["forward", "dx"])
@pytest.mark.parametrize("bad", [[0, 6000, 2000], [-1, 100, 6000], [6000, 5000, 0], [0, 10, 1 << 30]])
def test_bad_offsets_are_recorded_where_tiles_are_taken_over(cuda, form, bad):
    """More tiles than twice the SMs and rows of w across 128-byte lines, on an idle GPU and beside another stream's kernels."""
    rows, groups, wide, narrow = 6000, 60, 1000, 200  # the two columns that lie across lines: 400 and 2000 bytes
    N, K = (wide, narrow) if form == "forward" else (narrow, wide)
    x = torch.randn((rows, narrow), device="cuda").to(F16)
    w = torch.randn((groups, N, K), device="cuda").to(F16)
    guard = torch.full((rows + 40, wide), 5.0, dtype=F16, device="cuda")
    y = guard[20:20 + rows]
    good = torch.arange(0, rows + 1, rows // groups, dtype=torch.int32)
    call = S.grouped_mm if form == "forward" else S.grouped_mm_dx
    call(good.cuda(), x, w, y, stream=stream())
    torch.cuda.synchronize()
    assert S.device_error(0)[0] == 0
    other, m = torch.cuda.Stream(), torch.randn((4096, 4096), device="cuda").to(BF16)
    for busy in (False, True):
        off = good.clone()
        off[20:23] = torch.tensor(bad, dtype=torch.int32)
        off = off.cuda()
        torch.cuda.synchronize()
        if busy:
            with torch.cuda.stream(other):
                for _ in range(4):
                    m = (m @ m).clamp(-1, 1)
        call(off, x, w, y, stream=stream())
        torch.cuda.synchronize()
        assert S.device_error(0)[0] == -8
        assert (guard[:20] == 5).all() and (guard[20 + rows:] == 5).all()
