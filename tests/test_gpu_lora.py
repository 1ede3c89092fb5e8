"""Low-rank adapters of many requests on the GPU, against the plain 64-bit form."""
from __future__ import annotations

import pytest
import torch

import _rows as R
import spmm_b200 as S

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def stream():
    return torch.cuda.current_stream()


def clean():
    torch.cuda.synchronize()
    code, detail = S.device_error(0)
    assert code == 0, f"device error {code} ({detail})"


def offsets(sizes, first=0):
    return torch.tensor([first] + sizes, dtype=torch.int64).cumsum(0).to(torch.int32)


def values(shape, dtype, seed, pad=0, shift=0):
    v = torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype)
    if not pad and not shift:
        return v.cuda()
    n, c = shape
    buf = torch.zeros(n * (c + pad) + shift + 16, dtype=dtype, device="cuda")
    t = buf[shift:shift + n * (c + pad)].view(n, c + pad)[:, :c]
    t.copy_(v)
    return t


def close(got, want, real, err, dtype, mark):
    bound = err + R.STEP[dtype] * (want.abs() + err) + R.TINY[dtype]
    off = (R.d(got) - want).abs()
    bad = real[:, None] & ~(off <= bound)
    assert not bad.any(), f"{int(bad.sum())} off, worst {float((off / bound)[bad].max()):.3g} times the bound"
    assert (got[~real.cuda()] == mark).all()


def check(sizes, adapters, rank, N, K, dtype, base=True, scale=True, first=0, tail=0, pad=0, shift=0, none=(), single=False, in_place=False, seed=0):
    off = offsets(sizes, first)
    rows = int(off[-1]) + tail
    g = torch.Generator().manual_seed(seed)
    adapter = torch.randint(0, max(adapters, 1), (len(sizes),), generator=g, dtype=torch.int32)
    for r in none:
        adapter[r] = -1
    x = values((rows, K), dtype, seed + 1, pad, shift)
    x[:first], x[int(off[-1]):] = float("nan"), float("inf")
    a, b = values((adapters, rank, K), dtype, seed + 2), values((adapters, N, rank), dtype, seed + 3)
    bs = values((rows, N), dtype, seed + 4, pad, shift) if base else None
    sc = (torch.rand(adapters, generator=g) + 0.5).cuda() if scale else None
    want, real, err = R.lora(None if single else off, adapter, x, a, b, bs, sc)
    mark = 7.0
    if in_place:
        bs[~real.cuda()] = mark
        out = bs
    else:
        out = values((rows, N), dtype, 9, pad, shift).fill_(mark)
    S.lora(None if single else off.cuda(), adapter.cuda(), x, a, b, out, base=bs, scale=sc, stream=stream())
    clean()
    close(out, want, real, err, dtype, mark)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("sizes", [[1], [1] * 9, [0, 3, 0, 1], [128], [129, 1, 1, 63, 64, 65], [500, 0, 1, 1, 1, 260]])
def test_request_lengths(cuda, sizes, dtype):
    check(sizes, 3, 16, 136, 264, dtype)


@pytest.mark.parametrize("rank", [8, 16, 24, 32, 40, 64, 72, 128, 136, 256])
@pytest.mark.parametrize("sizes", [[1] * 5, [140, 2, 30]])
def test_ranks(cuda, rank, sizes):
    check(sizes, 4, rank, 328, 520, BF16)


@pytest.mark.parametrize("N,K", [(8, 8), (64, 4096), (4096, 64), (2056, 1032), (24, 72)])
def test_widths(cuda, N, K):
    check([1, 40, 1, 131], 2, 16, N, K, F16)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rank,N,K,pad,shift", [(1, 7, 9, 0, 0), (4, 64, 64, 0, 0), (13, 65, 33, 0, 0), (8, 64, 64, 1, 0), (8, 64, 64, 0, 3), (16, 100, 24, 4, 0)])
def test_operands_off_16_byte_boundaries(cuda, rank, N, K, pad, shift, dtype):
    check([1, 30, 0, 2], 3, rank, N, K, dtype, pad=pad, shift=shift, tail=1, none=(1,))


@pytest.mark.parametrize("base", [True, False])
@pytest.mark.parametrize("scale", [True, False])
def test_requests_without_an_adapter(cuda, base, scale):
    check([5, 200, 1, 1, 0, 70], 2, 32, 264, 136, BF16, base=base, scale=scale, none=(1, 2))
    check([5, 200, 1], 2, 32, 264, 136, BF16, base=base, scale=scale, none=(0, 1, 2))


def test_strides_rows_in_no_request_and_in_place(cuda):
    check([40, 1, 170], 3, 16, 192, 96, BF16, pad=24, shift=8, first=9, tail=140, none=(1,))
    check([40, 1, 170], 3, 16, 192, 96, BF16, pad=24, shift=8, first=9, tail=140, none=(1,), in_place=True)


@pytest.mark.parametrize("n", [1, 2, 64, 300])
def test_single_tokens(cuda, n):
    check([1] * n, 8, 16, 520, 1032, BF16, single=True, none=(0,) if n > 1 else ())
    check([1] * n, 8, 16, 520, 1032, F16, single=True, base=False)


def test_many_requests(cuda):
    check([1] * 4096, 16, 8, 64, 64, BF16, single=True)
    check([0, 1] * 2048, 16, 8, 64, 64, BF16)


def test_nothing_to_do(cuda):
    check([], 2, 8, 64, 64, BF16, tail=3)
    check([0, 0], 2, 8, 64, 64, BF16, tail=3)
    check([4], 0, 8, 64, 64, BF16, none=(0,))
    check([4, 2], 2, 0, 64, 64, BF16)
    check([4, 2], 2, 8, 64, 0, BF16)


def test_bad_adapters_and_offsets_are_recorded_and_stay_inside(cuda):
    x, a, b = values((20, 64), BF16, 1), values((2, 16, 64), BF16, 2), values((2, 72, 16), BF16, 3)
    base = values((20, 72), BF16, 4)
    guard = torch.full((60, 72), 5.0, dtype=BF16, device="cuda")
    out = guard[20:40]
    ad = torch.tensor([0, 2, 1], dtype=torch.int32, device="cuda")
    S.lora(offsets([6, 6, 8]).cuda(), ad, x, a, b, out, base=base, stream=stream())
    torch.cuda.synchronize()
    assert S.device_error(0)[0] == -8
    assert torch.equal(out[6:12], base[6:12])
    for bad in ([0, 30, 10, 20], [-5, 4, 8, 1 << 30], [20, 10, 0, -1]):
        S.lora(torch.tensor(bad, dtype=torch.int32, device="cuda"), ad.clamp(max=1), x, a, b, out, base=base, stream=stream())
        torch.cuda.synchronize()
        assert S.device_error(0)[0] == -8
        assert (guard[:20] == 5).all() and (guard[40:] == 5).all()


def test_not_a_number_stays_in_its_request(cuda):
    """A row of NaN, and an adapter that holds infinities, reach no other request's rows, though tiles hold both."""
    sizes = [3, 5, 130]
    x, a, b = values((138, 96), BF16, 1), values((2, 16, 96), BF16, 2), values((2, 136, 16), BF16, 3)
    a[1], x[1] = float("inf"), float("nan")
    out = torch.zeros((138, 136), dtype=BF16, device="cuda")
    S.lora(offsets(sizes).cuda(), torch.tensor([0, 1, 0], dtype=torch.int32, device="cuda"), x, a, b, out, stream=stream())
    clean()
    assert torch.isnan(out[1]).all() and not torch.isfinite(out[3:8]).any()
    rest = torch.ones(138, dtype=torch.bool, device="cuda")
    rest[1], rest[3:8] = False, False
    assert torch.isfinite(out[rest]).all()


def test_same_bits_on_another_stream_and_in_graphs_with_workspaces_of_their_own(cuda):
    sizes = [1] * 20 + [300, 150]
    x, a, b = values((470, 512), BF16, 1), values((4, 32, 512), BF16, 2), values((4, 264, 32), BF16, 3)
    o = offsets(sizes).cuda()
    ad = (torch.arange(22, dtype=torch.int32) % 4).cuda()
    outs = [torch.zeros((470, 264), dtype=BF16, device="cuda") for _ in range(4)]
    S.lora(o, ad, x, a, b, outs[0], stream=stream())
    side = torch.cuda.Stream()
    side.wait_stream(stream())
    S.lora(o, ad, x, a, b, outs[1], stream=side)
    side.synchronize()
    need = S.lora_workspace_size(a, b, 22, 470)
    graphs = []
    for out in outs[2:]:
        ws = torch.empty(need, dtype=torch.uint8, device="cuda")
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            S.lora(o, ad, x, a, b, out, ws=ws, stream=stream())
        graphs.append((graph, ws))
    with torch.cuda.stream(side):
        graphs[0][0].replay()
    graphs[1][0].replay()
    clean()
    assert all(torch.equal(outs[0], t) for t in outs[1:])


def test_sorted_requests_of_one_adapter_give_the_same_rows(cuda):
    """Requests grouped by route_build (a request is a token, its adapter the group) and run in sorted order."""
    n, adapters = 70, 5
    g = torch.Generator().manual_seed(2)
    ad = torch.randint(-1, adapters, (n, 1), generator=g, dtype=torch.int32)
    x, a, b = values((n, 264), BF16, 1), values((adapters, 16, 264), BF16, 2), values((adapters, 136, 16), BF16, 3)
    one = torch.zeros((n, 136), dtype=BF16, device="cuda")
    S.lora(None, ad.flatten().cuda(), x, a, b, one, stream=stream())
    i32 = dict(dtype=torch.int32, device="cuda")
    off, pos = torch.zeros(adapters + 1, **i32), torch.zeros((n, 1), **i32)
    xs, ys, two = torch.zeros_like(x), torch.zeros_like(one), torch.zeros_like(one)
    S.route_build(ad.cuda(), adapters, off, None, pos, stream=stream())
    S.route_gather(pos, x, xs, stream=stream())
    S.lora(off, torch.arange(adapters, **i32), xs, a, b, ys, stream=stream())
    S.route_combine(pos, ys, two, stream=stream())
    clean()
    want, real, err = R.lora(None, ad.flatten(), x, a, b, None, None)
    close(one, want, real, err, BF16, 0.0)
    close(two, want, real, err, BF16, 0.0)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("sizes", [[1, 1], [40, 1]])
def test_infinite_intermediates_give_infinities_not_nan(cuda, sizes, dtype):
    rows = sum(sizes)
    x, a, b = values((rows, 64), dtype, 1), values((2, 16, 64), dtype, 2).abs() + 1, values((2, 72, 16), dtype, 3).abs() + 1
    b[:, ::2] = -b[:, ::2]
    x[0, 5] = float("inf")
    out = torch.zeros((rows, 72), dtype=dtype, device="cuda")
    S.lora(offsets(sizes).cuda(), torch.zeros(2, dtype=torch.int32, device="cuda"), x, a, b, out, stream=stream())
    clean()
    want, _, _ = R.lora(offsets(sizes), torch.zeros(2, dtype=torch.int32), x, a, b, None, None)
    assert torch.isinf(want[0]).all() and torch.equal(R.d(out[0]), want[0])
    assert torch.isfinite(out[1:]).all()


@pytest.mark.parametrize("sizes", [[1, 1], [40, 1]])
def test_intermediates_past_the_range_of_fp16(cuda, sizes):
    """|u| is 64 * 64 or 80 times 16 and a little: kept to 2^-13 of itself, beside the bounds of the others."""
    rows = sum(sizes)
    x, b = torch.full((rows, 64), 16.0, dtype=F16, device="cuda"), values((2, 72, 16), F16, 3) * 2.0**-10
    x += torch.arange(64, device="cuda").to(F16) / 64
    a = torch.full((2, 16, 64), 64.0, dtype=F16, device="cuda")
    a[:, 1::2] = -80.0
    out = torch.zeros((rows, 72), dtype=F16, device="cuda")
    S.lora(offsets(sizes).cuda(), torch.zeros(2, dtype=torch.int32, device="cuda"), x, a, b, out, stream=stream())
    clean()
    want, real, err = R.lora(offsets(sizes), torch.zeros(2, dtype=torch.int32), x, a, b, None, None)
    u = R.d(x) @ R.d(a[0]).T
    assert (u.abs() > 65520).all() and (u.abs() < 131008).all() and want.abs().max() < 60000
    close(out, want, real, err + 2.0**-13 * (u.abs() @ R.d(b[0]).abs().T), F16, 0.0)
