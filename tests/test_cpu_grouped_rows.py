"""Refusals of the operators over grouped rows, on the host: sizes, types, pointers, strides and capacities are checked
before the device is looked at, so every one of them shows without a GPU; good arguments then report that there is none."""
from __future__ import annotations

import ctypes

import pytest
import torch

import spmm_b200 as S

INVALID, MISALIGNED, UNSUPPORTED, TOO_LARGE = -1, -2, -6, -10
P = 0x10000  # a pointer that is never followed
BIG = (1 << 31) - 1


def route(tokens=4, topk=2, rows=8, pos=P):
    return ctypes.byref(S.RouteView(tokens, topk, rows, pos))


def build(ids=P, tokens=4, topk=2, groups=3, offsets=P, order=P, pos=P, ws=0, n=0):
    return S.lib().spmm_route_build(ids, tokens, topk, groups, offsets, order, pos, ws, n, 0)


def gather(r=None, x=P, ldx=8, xs=P, ldxs=8, H=8, dt=1):
    return S.lib().spmm_route_gather(r or route(), x, ldx, xs, ldxs, H, dt, 0)


def combine(r=None, ys=P, ldys=8, w=P, y=P, ldy=8, H=8, dt=1):
    return S.lib().spmm_route_combine(r or route(), ys, ldys, w, y, ldy, H, dt, 0)


def combine_grad(r=None, dy=P, lddy=8, ys=P, ldys=8, w=P, dys=P, lddys=8, dw=P, H=8, dt=1):
    return S.lib().spmm_route_combine_grad(r or route(), dy, lddy, ys, ldys, w, dys, lddys, dw, H, dt, 0)


def mm(fn="spmm_grouped_mm", offsets=P, groups=2, rows=5, x=P, ldx=16, w=P, y=P, ldy=16, N=16, K=16, dt=1, odt=1):
    return getattr(S.lib(), fn)(offsets, groups, rows, x, ldx, w, y, ldy, N, K, dt, odt, 0)


def dw(offsets=P, groups=2, rows=5, dy=P, lddy=16, x=P, ldx=16, out=P, N=16, K=16, dt=1, odt=1):
    return S.lib().spmm_grouped_mm_dw(offsets, groups, rows, dy, lddy, x, ldx, out, N, K, dt, odt, 0)


def lora(adapters=2, rank=8, N=16, K=16, dt=1, a=P, b=P, scale=P, offsets=P, adapter=P, requests=3, rows=5, x=P, ldx=16, base=P, ldb=16,
         out=P * 2, ldo=16, ws=P, n=1 << 30):
    v = S.LoraView(adapters, rank, N, K, dt, a, b, scale)
    return S.lib().spmm_lora(ctypes.byref(v), offsets, adapter, requests, rows, x, ldx, base, ldb, out, ldo, ws, n, 0)


@pytest.mark.parametrize("call,args,want", [
    (build, dict(ids=0), INVALID), (build, dict(offsets=0), INVALID), (build, dict(pos=0), INVALID),
    (build, dict(tokens=-1), INVALID), (build, dict(topk=0), INVALID), (build, dict(groups=0), INVALID),
    (build, dict(groups=4097), TOO_LARGE), (build, dict(tokens=1 << 30, topk=2), TOO_LARGE), (build, dict(tokens=BIG, topk=BIG), TOO_LARGE),
    (build, dict(tokens=100000, topk=8), INVALID),  # needs a workspace
    (build, dict(tokens=100000, topk=8, ws=P, n=16), INVALID), (build, dict(tokens=100000, topk=8, ws=P + 1, n=1 << 30), MISALIGNED),
    (gather, dict(x=0), INVALID), (gather, dict(xs=0), INVALID), (gather, dict(ldx=7), INVALID), (gather, dict(ldxs=7), INVALID),
    (gather, dict(H=-1), INVALID), (gather, dict(dt=3), INVALID), (gather, dict(x=P + 1), MISALIGNED), (gather, dict(xs=P + 2, dt=2), MISALIGNED),
    (gather, dict(r=route(pos=0)), INVALID), (gather, dict(r=route(rows=-1)), INVALID), (gather, dict(r=route(tokens=1 << 30)), TOO_LARGE),
    (combine, dict(ys=0), INVALID), (combine, dict(y=0), INVALID), (combine, dict(w=P + 2), MISALIGNED), (combine, dict(ldy=7), INVALID),
    (combine_grad, dict(dys=0, dw=0), INVALID), (combine_grad, dict(ys=0), INVALID), (combine_grad, dict(dy=0), INVALID),
    (combine_grad, dict(lddys=7), INVALID), (combine_grad, dict(dw=P + 2), MISALIGNED),
    (mm, dict(offsets=0), INVALID), (mm, dict(groups=0), INVALID), (mm, dict(rows=-1), INVALID), (mm, dict(N=-1), INVALID), (mm, dict(K=-1), INVALID),
    (mm, dict(dt=2, odt=2), INVALID), (mm, dict(odt=0), INVALID), (mm, dict(x=0), INVALID), (mm, dict(w=0), INVALID), (mm, dict(y=0), INVALID),
    (mm, dict(ldx=15), INVALID), (mm, dict(ldy=15), INVALID), (mm, dict(x=P + 1), MISALIGNED), (mm, dict(y=P + 2, odt=2), MISALIGNED),
    (mm, dict(groups=4097), TOO_LARGE), (mm, dict(rows=BIG), TOO_LARGE), (mm, dict(N=1 << 25), TOO_LARGE), (mm, dict(K=1 << 25), TOO_LARGE),
    (mm, dict(fn="spmm_grouped_mm_dx", w=0), INVALID), (mm, dict(fn="spmm_grouped_mm_dx", ldx=15), INVALID),
    (dw, dict(dy=0), INVALID), (dw, dict(x=0), INVALID), (dw, dict(out=0), INVALID), (dw, dict(rows=0, out=0), INVALID), (dw, dict(ldx=15), INVALID),
    (lora, dict(rank=-1), INVALID), (lora, dict(rank=257), TOO_LARGE), (lora, dict(requests=4097), TOO_LARGE), (lora, dict(dt=2), INVALID),
    (lora, dict(a=0), INVALID), (lora, dict(b=0), INVALID), (lora, dict(x=0), INVALID), (lora, dict(out=0), INVALID), (lora, dict(adapter=0), INVALID),
    (lora, dict(offsets=0), INVALID),  # single tokens: a request for every row
    (lora, dict(ws=0), INVALID), (lora, dict(n=8), INVALID), (lora, dict(ws=P + 16), MISALIGNED), (lora, dict(scale=P + 2), MISALIGNED),
    (lora, dict(out=P, ldo=32), INVALID),  # in place with another stride
    (lora, dict(ldb=15), INVALID), (lora, dict(ldo=15), INVALID), (lora, dict(ldx=15), INVALID),
])
def test_refused(call, args, want):
    assert call(**args) == want


def test_good_arguments_report_the_missing_gpu():
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    for call in (build, gather, combine, combine_grad, mm, dw, lora):
        assert call() == UNSUPPORTED
    assert mm(fn="spmm_grouped_mm_dx") == UNSUPPORTED


def test_workspace_sizes():
    assert S.route_workspace_size(0, 1, 1) == 0
    assert S.route_workspace_size(512, 8, 256) == 0  # one block
    big = S.route_workspace_size(16384, 8, 256)
    assert big > 0 and big % (4 * 256) == 0
    # The largest input still fits its blocks: a histogram for each.
    assert S.route_workspace_size(BIG - 4095, 1, 4096) <= 128 * 4096 * 4
    n = ctypes.c_size_t()
    assert S.lib().spmm_route_workspace_size(1, 1, 1, None) == INVALID
    v = S.LoraView(2, 8, 16, 16, 1, 0, 0, 0)
    assert S.lib().spmm_lora_workspace_size(ctypes.byref(v), 3, 5, ctypes.byref(n)) == 0 and n.value >= 5 * 8 * 4
    assert S.lib().spmm_lora_workspace_size(ctypes.byref(v), 3, 5, None) == INVALID


def test_binding_refuses_tensors_off_the_gpu():
    ids = torch.zeros((4, 2), dtype=torch.int32)
    with pytest.raises(ValueError):
        S.route_build(ids, 3, torch.zeros(4, dtype=torch.int32), None, torch.zeros_like(ids))
    x = torch.zeros((4, 8), dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        S.route_gather(ids, x, torch.zeros((8, 8), dtype=torch.bfloat16))
    with pytest.raises(ValueError):
        S.grouped_mm(torch.zeros(2, dtype=torch.int32), x, torch.zeros((1, 8, 8), dtype=torch.bfloat16), x)
    with pytest.raises(ValueError):
        S.grouped_mm(torch.zeros(2, dtype=torch.int32), x.double(), torch.zeros((1, 8, 8)), x)


@pytest.mark.parametrize("call", [lambda **k: gather(ldx=1 << 26, ldxs=1 << 26, **k), lambda **k: combine(ldys=1 << 26, ldy=1 << 26, **k),
                                  lambda **k: combine_grad(lddy=1 << 26, ldys=1 << 26, lddys=1 << 26, **k)])
def test_rows_too_long_to_count_are_refused(call):
    assert call(H=(1 << 24) + 1) == TOO_LARGE
    assert call(H=1 << 24) != TOO_LARGE
