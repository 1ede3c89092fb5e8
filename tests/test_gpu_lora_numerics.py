"""What the adapters' intermediate u = a x keeps: FP16 values of any size, small terms behind a large base, long batches;
and the adapters that are recorded.

Bound: u is a sum of K terms in 32 bits (K * 2^-23 of the sum of their magnitudes). In bf16 it enters the product with b as it is. In
fp16 it may be two terms, half a step of a half step of itself (2^-22), with a power of two taken out of each row so that its largest
element lies in [2^14, 2^15): elements far below that one keep 2^-25 of the smallest step, 2^-39 of the largest. The product
with b is at most 3 * rank additions in 32 bits more, scale and base one rounding each."""
from __future__ import annotations

import pytest
import torch

import _rows as R
import spmm_b200 as S

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def stream():
    return torch.cuda.current_stream()


def offsets(sizes):
    return torch.tensor([0] + sizes, dtype=torch.int64).cumsum(0).to(torch.int32)


def normal(shape, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed))


def exact(sizes, adapter, x, a, b, base, scale):
    """out in 64 bits and a bound on its error before the last rounding (sizes None: a request a row)."""
    at = offsets(sizes if sizes is not None else [1] * x.shape[0]).tolist()
    out = torch.zeros((x.shape[0], b.shape[1]), dtype=torch.float64) if base is None else R.d(base)
    err = torch.zeros_like(out)
    K, rank = x.shape[1], a.shape[1]
    for e, i, j in zip(adapter.tolist(), at, at[1:]):
        if e < 0 or i == j:
            continue
        s = 1.0 if scale is None else float(scale[e])
        u, um = R.d(x[i:j]) @ R.d(a[e]).T, R.d(x[i:j]).abs() @ R.d(a[e]).abs().T
        kept = K * 2.0**-23 * um
        if x.dtype == F16:
            kept = kept + 2.0**-22 * u.abs() + 2.0**-39 * u.abs().amax(1, keepdim=True)
        bm, delta = R.d(b[e]).abs().T, s * (u @ R.d(b[e]).T)
        err[i:j] = abs(s) * (kept @ bm + 3 * rank * 2.0**-23 * (um @ bm)) + 2.0**-22 * (out[i:j].abs() + delta.abs())
        out[i:j] += delta
    return out, err


def check(sizes, adapter, x, a, b, base=None, scale=None, want_finite=True):
    """Both ways to say it: packed requests, and (where every request is a row) single tokens."""
    adapter = torch.tensor(adapter, dtype=torch.int32)
    out = torch.full((x.shape[0], b.shape[1]), 7.0, dtype=x.dtype, device="cuda")
    S.lora(None if sizes is None else offsets(sizes).cuda(), adapter.cuda(), x, a, b, out, base=base, scale=scale, stream=stream())
    torch.cuda.synchronize()
    code, detail = S.device_error(0)
    assert code == 0, f"device error {code} ({detail})"
    want, err = exact(sizes, adapter, x, a, b, base, scale)
    assert not want_finite or want.abs().max() < 65504
    bound = err + R.STEP[x.dtype] * (want.abs() + err) + R.TINY[x.dtype]
    off = (R.d(out) - want).abs()
    bad = ~(off <= bound)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {float((off / bound)[bad].max()):.3g} times the bound"
    return out


SIZES = [None, [1] * 64, [64], [1, 40, 0, 22, 1]]  # single tokens, short requests, tensor-core tiles, both in a batch


def ads(sizes):
    return [0] * (64 if sizes is None else len(sizes))


@pytest.mark.parametrize("rank", [8, 48, 72, 256])
@pytest.mark.parametrize("sizes", SIZES)
def test_large_intermediates_in_fp16(cuda, sizes, rank):
    """|u| around 2^22, which the scale brings back: finite in every form, whatever batch the row is in."""
    x = (normal((64, 64), 1) * 500 + 1000).to(F16).cuda()
    a = (normal((1, rank, 64), 2) * 20 + 60).to(F16).cuda()
    b = (normal((1, 72, rank), 3) * 2.0**-8).to(F16).cuda()
    b[:, :, 1::3] = 0
    assert (R.d(x) @ R.d(a[0]).T).abs().min() > 131008
    check(sizes, ads(sizes), x, a, b, scale=torch.full((1,), 2.0**-10, device="cuda"))


@pytest.mark.parametrize("rank", [8, 48, 72, 256])
@pytest.mark.parametrize("sizes", SIZES)
def test_small_intermediates_in_fp16(cuda, sizes, rank):
    """|u| around 2^-20, which b and the scale bring back."""
    x = (normal((64, 64), 1) * 2.0**-10).to(F16).cuda()
    a = (normal((1, rank, 64), 2) * 2.0**-13).to(F16).cuda()
    b = (normal((1, 72, rank), 3) * 64).to(F16).cuda()
    assert (R.d(x) @ R.d(a[0]).T).abs().max() < 2.0**-14
    check(sizes, ads(sizes), x, a, b, scale=torch.full((1,), 4096.0, device="cuda"))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("sizes", SIZES)
def test_rows_and_ranks_of_unlike_sizes(cuda, sizes, dtype):
    """Neighbouring rows, and elements of one row, that are powers of two apart; a row of zeros; one of the largest values."""
    x = normal((64, 96), 1) * torch.exp2(torch.arange(64) % 23 - 11.0)[:, None]
    x[7], x[9] = 0, 65504 * x[9].sign()
    a = normal((1, 48, 96), 2) * torch.exp2(-(torch.arange(48) % 13.0))[None, :, None]
    x, a, b = x.to(dtype).cuda(), a.to(dtype).cuda(), (normal((1, 136, 48), 3) * 2.0**-11).to(dtype).cuda()
    check(sizes, ads(sizes), x, a, b)
    assert (check(sizes, ads(sizes), x, a, b)[7] == 0).all()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("sizes", SIZES)
def test_base_that_cancels(cuda, sizes, dtype):
    """base = -delta to 16 bits: what is left shows the intermediate's own error, which no rounding hides."""
    x, a, b = (normal(s, k).to(dtype).cuda() for k, s in ((1, (64, 256)), (2, (1, 32, 256)), (3, (1, 136, 32))))
    want, _ = exact([64], torch.zeros(1, dtype=torch.int32), x, a, b, None, None)
    check(sizes, ads(sizes), x, a, b, base=(-want).to(dtype).cuda())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rank", [8, 16, 56, 72, 128, 200, 256])
@pytest.mark.parametrize("sizes", SIZES)
def test_ranks_that_cancel_exactly(cuda, sizes, rank, dtype):
    """Whole numbers: elements of u of 21 bits, pairs of which b subtracts to a value of x. Every sum is exact in 32 bits, so the
    result is too; any bit that u lost shows."""
    g = torch.Generator().manual_seed(rank)
    x, a = torch.randint(100, 201, (64, 64), generator=g), torch.randint(100, 201, (1, rank, 64), generator=g)
    a[0, 1::2] = a[0, ::2]
    at = torch.randint(0, 64, (rank // 2,), generator=g)
    a[0, torch.arange(0, rank, 2), at] += 1
    b = torch.zeros((1, 72, rank))
    pair = torch.arange(72) % (rank // 2)
    b[0, torch.arange(72), 2 * pair], b[0, torch.arange(72), 2 * pair + 1] = 1.0, -1.0
    out = check(sizes, ads(sizes), x.to(dtype).cuda(), a.to(dtype).cuda(), b.to(dtype).cuda())
    assert torch.equal(out.cpu(), x[:, at[pair]].to(dtype))


@pytest.mark.parametrize("dtype,rank", [(F16, 16), (BF16, 64), (F16, 96), (BF16, 256), (F16, 256)])
@pytest.mark.parametrize("N", [8, 200])
def test_many_row_tiles_a_block(cuda, dtype, rank, N):
    """Long enough that a block makes u for several row tiles, with and without an adapter between them, into the same memory."""
    sizes = [30000, 1, 0, 129, 41000, 128, 1, 17000, 640, 1]
    adapter = [0, 2, 1, -1, 1, 2, 0, -1, 2, -1]
    rows = sum(sizes)
    x = (normal((rows, 64), 1) * torch.exp2(torch.arange(rows) % 5 - 2.0)[:, None]).to(dtype).cuda()
    a, b = normal((3, rank, 64), 2).to(dtype).cuda(), (normal((3, N, rank), 3) / 16).to(dtype).cuda()
    base = normal((rows, N), 4).to(dtype).cuda()
    scale = torch.tensor([0.5, 2.0, -1.0], device="cuda")
    first = check(sizes, adapter, x, a, b, base=base, scale=scale)
    again = base.clone()
    S.lora(offsets(sizes).cuda(), torch.tensor(adapter, dtype=torch.int32).cuda(), x, a, b, again, base=again, scale=scale, stream=stream())
    torch.cuda.synchronize()
    assert torch.equal(first, again)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("sizes,rank,width", [(None, 16, 4096), (None, 64, 4096), ([1] * 256, 64, 4096), ([380] + [1] * 128, 64, 2048), ([380] + [1] * 128, 8, 1024),
                                              ([2] * 200, 128, 1024), ([2] * 200, 8, 1024), ([0] * 90 + [1, 2, 30] * 10, 128, 2048)])
def test_few_rows_a_request_in_either_form(cuda, sizes, rank, width, dtype):
    """At most four rows a request on average: the rank and the widths choose between rows and tiles."""
    n = 256 if sizes is None else sum(sizes)
    adapter = [(3 * r) % 5 - (r % 11 == 0) for r in range(n if sizes is None else len(sizes))]
    x, a, b = normal((n, width), 1).to(dtype).cuda(), (normal((5, rank, width), 2) * width**-0.5).to(dtype).cuda(), normal((5, width, rank), 3).to(dtype).cuda()
    check(sizes, adapter, x, a, b, base=normal((n, width), 4).to(dtype).cuda(), scale=torch.linspace(0.5, 2, 5, device="cuda"))


@pytest.mark.parametrize("adapters,rank,N,sizes,adapter,detail", [
    (2, 0, 64, [4, 2], [0, 2], 1),        # nothing to add
    (0, 8, 64, [4, 2], [-1, 0], 1),       # no adapters at all
    (2, 8, 64, [1, 0, 1], [0, 5, 1], 1),  # a request without rows: few rows a request
    (2, 8, 65, [1, 0, 1], [0, 5, 1], 1),  # off 16-byte boundaries
    (2, 8, 64, [40, 0, 1], [0, 5, 1], 1),  # tensor-core tiles
])
def test_adapters_past_the_last_are_recorded(cuda, adapters, rank, N, sizes, adapter, detail):
    rows = sum(sizes)
    x, a, b = (normal(s, k).to(BF16).cuda() for k, s in ((1, (rows, 64)), (2, (adapters, rank, 64)), (3, (adapters, N, rank))))
    base = normal((rows, N), 4).to(BF16).cuda()
    out = torch.zeros_like(base)
    S.lora(offsets(sizes).cuda(), torch.tensor(adapter, dtype=torch.int32).cuda(), x, a, b, out, base=base, stream=stream())
    torch.cuda.synchronize()
    assert S.device_error(0) == (-8, detail)
    if rank == 0 or adapters == 0:
        assert torch.equal(out, base)
