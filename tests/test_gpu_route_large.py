"""Routing of large batches (its streamed gradient, sums of few pairs) against 64-bit forms on the GPU."""
from __future__ import annotations

import pytest
import torch

import _rows as R
import spmm_b200 as S

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
SIZE = {F16: 2, BF16: 2, F32: 4}


def stream():
    return torch.cuda.current_stream()


def clean():
    torch.cuda.synchronize()
    code, detail = S.device_error(0)
    assert code == 0, f"device error {code} ({detail})"


def normal(g, shape, dtype, pad=0):
    n, c = shape
    return torch.full((n, c + pad), float("nan"), dtype=dtype, device="cuda")[:, :c].copy_(torch.randn(shape, generator=g, device="cuda"))


def routed(g, tokens, topk, drop):
    ids = torch.randint(0, 40, (tokens, topk), generator=g, device="cuda", dtype=torch.int32)
    ids = torch.where(torch.rand((tokens, topk), generator=g, device="cuda") < drop, -1, ids).to(torch.int32)
    off, pos = torch.zeros(41, dtype=torch.int32, device="cuda"), torch.zeros_like(ids)
    S.route_build(ids, 40, off, None, pos, stream=stream())
    return int(off[-1]), pos


def bytes_of(tokens, topk, H, dtype):
    return tokens * topk * H * SIZE[dtype]


# Rows of one piece of 4096 bytes and less, of two and three, with a last one of 16 bytes and more; 64 MB and a little.
WIDTHS = {1: 2056, 2: 5128, 3: 1032, 4: 512, 5: 1024, 7: 3000, 8: 2048}


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("topk", sorted(WIDTHS))
def test_combine_grad_of_large_batches(cuda, topk, dtype):
    H = WIDTHS[topk]
    tokens = -(-(64 << 20) // bytes_of(1, topk, H, dtype)) + topk % 3
    g = torch.Generator(device="cuda").manual_seed(topk)
    n, pos = routed(g, tokens, topk, 0.2)
    pad = 16 if topk % 2 else 0
    dy, ys = normal(g, (tokens, H), dtype, pad), normal(g, (tokens * topk, H), dtype, pad)
    ys[n:] = float("nan")  # rows that no pair has are not read
    w = torch.randn((tokens, topk), generator=g, device="cuda")
    at = pos.long().clamp(min=0)
    has = pos >= 0

    def run(ys_, w_, want_ys, want_w):
        dys = torch.full((tokens * topk, H + pad), 7.0, dtype=dtype, device="cuda")[:, :H] if want_ys else None
        dw = torch.full((tokens, topk), float("nan"), device="cuda") if want_w else None
        S.route_combine_grad(pos, dy, ys_, w_, dys, dw, stream=stream())
        clean()
        return dys, dw

    dys, dw = run(ys, w, True, True)
    for weight, got in ((w, dys), (None, run(ys, None, True, True)[0])):
        want = torch.full_like(got, 7.0)
        for j in range(topk):
            rows = dy.float() * weight[:, j:j + 1] if weight is not None else dy.float()
            want[at[has[:, j], j]] = rows.to(dtype)[has[:, j]]  # one product in 32 bits, one rounding
        assert torch.equal(got, want)
    for j in range(topk):
        prod = torch.where(has[:, j:j + 1], ys[at[:, j]].double(), 0.0) * dy.double()
        bound = (H + 1) * 2.0**-23 * prod.abs().sum(1)
        assert ((dw[:, j].double() - prod.sum(1)).abs() <= bound).all()
    assert (dw[~has] == 0).all()
    # Each alone, and all again: the same bits.
    assert torch.equal(run(None, w, True, False)[0], dys) and torch.equal(run(ys, None, False, True)[1], dw)
    again = run(ys, w, True, True)
    assert torch.equal(again[0], dys) and torch.equal(again[1], dw)


@pytest.mark.parametrize("tokens", [2047, 2048])
def test_combine_grad_on_either_side_of_the_limit(cuda, tokens):
    """The two kernels sum in orders of their own; their products with one weight are the same."""
    H, topk = 2048, 8
    g = torch.Generator(device="cuda").manual_seed(5)
    n, pos = routed(g, tokens, topk, 0.0)
    dy, ys = normal(g, (tokens, H), BF16), normal(g, (tokens * topk, H), BF16)
    w = torch.randn((tokens, topk), generator=g, device="cuda")
    dys, dw = torch.zeros_like(ys), torch.zeros_like(w)
    S.route_combine_grad(pos, dy, ys, w, dys, dw, stream=stream())
    clean()
    flat = pos.flatten().long()
    token = torch.arange(tokens, device="cuda").repeat_interleave(topk)
    assert torch.equal(dys[flat], (dy.float()[token] * w.flatten()[:, None]).to(BF16))
    prod = dy.double()[token] * ys.double()[flat]
    assert ((dw.double().flatten() - prod.sum(1)).abs() <= (H + 1) * 2.0**-23 * prod.abs().sum(1)).all()


def test_bad_positions_of_a_large_batch_are_recorded_and_skipped(cuda):
    H, topk, tokens = 2048, 8, 2100
    g = torch.Generator(device="cuda").manual_seed(6)
    n, pos = routed(g, tokens, topk, 0.1)
    dy, ys = normal(g, (tokens, H), BF16), normal(g, (tokens * topk, H), BF16)
    for t, bad in ((3, tokens * topk), (200, -2), (2099, 1 << 30)):
        now = pos.clone()
        lost = int(now[t, 4])
        now[t, 4] = bad
        dys, dw = torch.full_like(ys, 7.0), torch.full((tokens, topk), float("nan"), device="cuda")
        S.route_combine_grad(now, dy, ys, None, dys, dw, stream=stream())
        torch.cuda.synchronize()
        assert S.device_error(0) == (-8, t * topk + 4)
        assert float(dw[t, 4]) == 0.0 and not torch.isnan(dw).any()
        if lost >= 0:
            assert (dys[lost] == 7).all()
        rows = now[t][(now[t] >= 0) & (now[t] < tokens * topk)].long()
        assert torch.equal(dys[rows], dy[t].expand(len(rows), H))


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("topk,H", [(1, 1024), (1, 3001), (2, 1000), (2, 333), (2, 4104), (3, 520), (3, 2050), (4, 2048), (4, 1001), (4, 72)])
def test_combine_of_large_batches(cuda, topk, H, dtype):
    """At most four pairs, several vectors a thread, of every vector width."""
    row = H * SIZE[dtype]
    width = 16 if row % 16 == 0 else (4 if row % 4 == 0 else 2)
    tokens = (512 * 1024) // (row // width) + 37
    g = torch.Generator(device="cuda").manual_seed(topk + H)
    n, pos = routed(g, tokens, topk, 0.2)
    ys = normal(g, (tokens * topk, H), dtype)
    ys[n:] = float("nan")
    w = torch.randn((tokens, topk), generator=g, device="cuda")
    at, has = pos.long().clamp(min=0), pos >= 0
    for weight in (w, None):
        y = torch.full((tokens, H), float("nan"), dtype=dtype, device="cuda")
        S.route_combine(pos, ys, y, weight, stream=stream())
        clean()
        want, mag = torch.zeros((2, tokens, H), dtype=torch.float64, device="cuda")
        for j in range(topk):
            v = torch.where(has[:, j:j + 1], ys[at[:, j]].double(), 0.0) * (weight[:, j:j + 1].double() if weight is not None else 1.0)
            want += v
            mag += v.abs()
        sums = topk * 2.0**-23 * mag
        assert ((y.double() - want).abs() <= sums + R.STEP[dtype] * (want.abs() + sums) + R.TINY[dtype]).all()
        again = torch.empty_like(y)
        S.route_combine(pos, ys, again, weight, stream=stream())
        clean()
        assert torch.equal(y, again)
