"""Products of row groups with their own matrices on the GPU, and their gradients, against plain 64-bit forms."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import _rows as R
import spmm_b200 as S

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def stream():
    return torch.cuda.current_stream()


def clean():
    torch.cuda.synchronize()
    code, detail = S.device_error(0)
    assert code == 0, f"device error {code} ({detail})"


def offsets(sizes, first=0):
    return torch.tensor([first] + sizes, dtype=torch.int64).cumsum(0).to(torch.int32)


def values(shape, dtype, seed, pad=0, shift=0):
    """A contiguous tensor of the given shape, or rows at a stride of columns + pad, `shift` elements in."""
    v = torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype)
    if not pad and not shift:
        return v.cuda()
    n, c = shape
    buf = torch.zeros(n * (c + pad) + shift + 16, dtype=dtype, device="cuda")
    t = buf[shift:shift + n * (c + pad)].view(n, c + pad)[:, :c]
    t.copy_(v)
    return t


def check_all(sizes, N, K, dtype, out=None, pad=0, shift=0, first=0, tail=0, seed=0):
    """Forward, dx and dw of one set of operands; rows in no group hold NaN in the inputs and keep what they held."""
    out = out or dtype
    off = offsets(sizes, first)
    rows, n = int(off[-1]) + tail, int(off[-1])
    x, dy = values((rows, K), dtype, seed + 1, pad, shift), values((rows, N), dtype, seed + 2, pad, shift)
    for t in (x, dy):
        t[:first] = float("nan")
        t[n:] = float("inf")
    w = values((len(sizes), N, K), dtype, seed + 3)
    mark = 7.0
    y = values((rows, N), out, 4, pad, shift).fill_(mark)
    dx = values((rows, K), out, 5, pad, shift).fill_(mark)
    dw = torch.full((len(sizes), N, K), float("nan"), dtype=out, device="cuda")
    o = off.cuda()
    S.grouped_mm(o, x, w, y, stream=stream())
    S.grouped_mm_dx(o, dy, w, dx, stream=stream())
    S.grouped_mm_dw(o, dy, x, dw, stream=stream())
    clean()
    for got, (want, mag), terms in ((y, R.grouped(off, x, w), K), (dx, R.grouped_dx(off, dy, w), N)):
        R.close(got[first:n], want[first:n], mag[first:n], terms, out, "rows")
        assert (got[:first] == mark).all() and (got[n:] == mark).all()
    want, mag = R.grouped_dw(off, dy, x)
    R.close(dw, want, mag, max(sizes), out, "dw")
    for g, size in enumerate(sizes):
        if size == 0:
            assert (dw[g] == 0).all()
    return off, x, w, y


SIZES = [[1], [0, 1, 0], [5], [16, 15, 17], [64], [127, 1, 129], [128, 0, 256, 3], [130, 63, 64, 65], [300, 2, 0, 0, 41, 1]]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("sizes", SIZES)
def test_group_sizes(cuda, sizes, dtype):
    check_all(sizes, 136, 200, dtype)


@pytest.mark.parametrize("N,K", [(8, 8), (16, 64), (64, 16), (72, 8), (256, 64), (264, 72), (520, 328), (128, 1032), (1032, 128), (40, 2000)])
def test_widths(cuda, N, K):
    check_all([37, 0, 150, 5], N, K, BF16, out=F32)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("N,K,pad,shift", [(1, 1, 0, 0), (7, 13, 0, 0), (65, 130, 0, 0), (9, 300, 0, 0), (64, 64, 1, 0), (64, 64, 0, 1), (72, 40, 3, 5), (515, 1001, 0, 0)])
def test_operands_off_16_byte_boundaries(cuda, N, K, pad, shift, dtype):
    check_all([3, 70, 0, 1], N, K, dtype, pad=pad, shift=shift, tail=2)


@pytest.mark.parametrize("out", [BF16, F32])
def test_strides_and_rows_in_no_group(cuda, out):
    check_all([40, 0, 200, 9], 192, 96, BF16, out=out, pad=24, shift=8, first=11, tail=150)


@pytest.mark.parametrize("sizes,first,tail,dtype,out", [
    ([4000, 130], 0, 0, BF16, BF16), ([1, 4199], 3, 40, F16, F32), ([2304, 2305], 0, 5, F16, F16), ([4096], 0, 0, BF16, F32),
    ([257, 100, 0, 511, 256, 255, 400, 2, 1900, 300], 0, 1, BF16, BF16)])
@pytest.mark.parametrize("wide,narrow", [(5120, 72), (5000, 200)])
def test_long_groups(cuda, sizes, first, tail, dtype, out, wide, narrow):
    """Groups long enough for a pair of blocks a tile, with ragged ends, columns that end inside a tile, and sums that end
    inside a step: wide outputs of the forward product, then of dx."""
    off = offsets(sizes, first)
    n = int(off[-1])
    o = off.cuda()
    for forward in (True, False):
        rows_in = values((n + tail, narrow), dtype, 1)
        rows_in[:first], rows_in[n:] = float("nan"), float("inf")
        w = values((len(sizes), wide, narrow) if forward else (len(sizes), narrow, wide), dtype, 2)
        got = torch.full((n + tail, wide), 7.0, dtype=out, device="cuda")
        (S.grouped_mm if forward else S.grouped_mm_dx)(o, rows_in, w, got, stream=stream())
        clean()
        want, mag = (R.grouped if forward else R.grouped_dx)(off, rows_in, w)
        R.close(got[first:n], want[first:n], mag[first:n], narrow, out, "forward" if forward else "dx")
        assert (got[:first] == 7).all() and (got[n:] == 7).all()


@pytest.mark.parametrize("sizes,first,tail,dtype,out", [
    ([4000, 137], 0, 0, BF16, BF16), ([1, 4198], 3, 40, F16, F32), ([2304, 2320], 0, 5, F16, F16), ([0, 6200, 0], 1, 1, BF16, F32),
    ([2049, 2063, 2050, 2034, 2048], 0, 0, BF16, F32)])
@pytest.mark.parametrize("N,K", [(4608, 4352), (264, 38400), (4360, 4424)])
def test_long_groups_dw(cuda, sizes, first, tail, dtype, out, N, K):
    """The weights' gradient of long groups (pairs of blocks a tile): sums that end anywhere in a step, empty groups, edges.
    Checked on some rows and columns of every group and all of its corners."""
    off = offsets(sizes, first)
    n = int(off[-1])
    dy, x = values((n + tail, N), dtype, 1), values((n + tail, K), dtype, 2)
    for t in (dy, x):
        t[:first], t[n:] = float("nan"), float("inf")
    dw = torch.full((len(sizes), N, K), float("nan"), dtype=out, device="cuda")
    S.grouped_mm_dw(off.cuda(), dy, x, dw, stream=stream())
    clean()
    assert not torch.isnan(dw).any()
    g = torch.Generator().manual_seed(7)
    ns = torch.cat([torch.randint(0, N, (40,), generator=g), torch.tensor([0, 127, 128, 255, 256, N - 1])]).cuda()
    ks = torch.cat([torch.randint(0, K, (60,), generator=g), torch.tensor([0, 127, 128, 255, 256, K - 1])]).cuda()
    want, mag = R.grouped_dw(off, dy[:, ns], x[:, ks])
    R.close(dw[:, ns][:, :, ks], want, mag, max(sizes), out, "dw")


def test_long_groups_in_a_graph_between_other_kernels(cuda):
    """The clusters' launches captured, behind and before kernels of single blocks, give the eager bits again and again."""
    off = offsets([2500, 0, 3647]).cuda()
    x, dy, w = values((6147, 2048), BF16, 1), values((6147, 2304), BF16, 2), values((3, 2304, 2048), BF16, 3)

    def run():
        y, dx, dw = torch.zeros_like(dy), torch.zeros_like(x), torch.zeros(w.shape, device="cuda")
        small = torch.zeros((40, 2304), dtype=BF16, device="cuda")
        s = stream()
        S.grouped_mm(off, x, w, y, stream=s)
        S.grouped_mm_dx(off, y, w, dx, stream=s)
        S.grouped_mm_dw(off, y, x, dw, stream=s)
        S.grouped_mm(few, x[:40], w, small, stream=s)
        S.grouped_mm_dw(off, dy, dx, dw, stream=s)
        return y, dx, dw, small

    few = offsets([40, 0, 0]).cuda()
    eager = run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = run()
    for _ in range(3):
        graph.replay()
    clean()
    assert all(torch.equal(a, b) for a, b in zip(eager, captured))


def test_no_rows_and_empty_sums(cuda):
    check_all([0, 0], 64, 64, BF16, tail=5)
    x, w = torch.zeros((4, 0), dtype=BF16, device="cuda"), torch.zeros((1, 16, 0), dtype=BF16, device="cuda")
    y = torch.full((4, 16), 3.0, dtype=BF16, device="cuda")
    S.grouped_mm(offsets([3]).cuda(), x, w, y, stream=stream())
    dw = torch.full((2, 8, 8), 3.0, dtype=F32, device="cuda")
    e = torch.zeros((0, 8), dtype=BF16, device="cuda")
    S.grouped_mm_dw(offsets([0, 0]).cuda(), e, e, dw, stream=stream())
    clean()
    assert (y[:3] == 0).all() and (y[3:] == 3).all() and (dw == 0).all()


def test_many_groups(cuda):
    g = torch.Generator().manual_seed(5)
    check_all(torch.randint(0, 3, (1000,), generator=g).tolist(), 24, 16, BF16)
    check_all(([0] * 4095) + [9], 8, 8, F16)


def test_large_values_overflow_to_infinity_only_where_the_formula_does(cuda):
    x = torch.full((2, 64), 200.0, dtype=F16, device="cuda")
    x[1] = 1.0
    w = torch.full((1, 16, 64), 100.0, dtype=F16, device="cuda")
    y, y32 = torch.empty((2, 16), dtype=F16, device="cuda"), torch.empty((2, 16), device="cuda")
    S.grouped_mm(offsets([2]).cuda(), x, w, y, stream=stream())
    S.grouped_mm(offsets([2]).cuda(), x, w, y32, stream=stream())
    clean()
    assert torch.isinf(y[0]).all() and (y[1] == 6400).all() and (y32[0] == 64 * 200 * 100).all()


def test_equals_the_block_sparse_product_of_the_block_diagonal(cuda):
    """blockdiag(w) times the groups' rows, as a BSR matrix of dense 32 x 48 diagonal blocks."""
    groups, N, K, cols = 4, 32, 48, 24
    w = values((groups, N, K), F16, 1)
    x = values((groups * cols, K), F16, 2)
    y = torch.empty((groups * cols, N), device="cuda")
    S.grouped_mm(offsets([cols] * groups).cuda(), x, w, y, stream=stream())
    r, c = np.meshgrid(np.arange(N), np.arange(K), indexing="ij")
    coo = [(g * N + r.ravel(), g * K + c.ravel(), w[g].float().cpu().numpy().ravel()) for g in range(groups)]
    A = S.csr_from_coo(groups * N, groups * K, *(np.concatenate(v) for v in zip(*coo)))
    Hb = S.csr_to_bsr16(A, S.DTYPE_F16)
    dev = [torch.from_numpy(v).cuda() for v in (Hb.row_ptr, Hb.col_idx, Hb.values.view(np.int16))]
    view = Hb.view()
    view.row_ptr, view.col_idx, view.values = (S.ptr(v) for v in dev)
    B = x.view(groups, cols, K).transpose(1, 2).reshape(groups * K, cols).contiguous()
    C = torch.empty((groups * N, cols), device="cuda")
    S.bsr16(view, B, C, cols, 0, stream())
    clean()
    want, mag = R.grouped(offsets([cols] * groups), x, w)
    R.close(y, want, mag, K, F32)
    R.close(C.view(groups, N, cols).transpose(1, 2).reshape(groups * cols, N).contiguous(), want, mag, K, F32)


def test_gradients_against_differences(cuda):
    """Small whole numbers: every product and sum is exact, so a step of 1 changes <y, dy> by exactly the gradient."""
    g = torch.Generator().manual_seed(1)
    sizes, N, K = [5, 0, 20], 24, 40
    off = offsets(sizes).cuda()
    x, dy = (torch.randint(-4, 5, (25, c), generator=g).to(BF16).cuda() for c in (K, N))
    w = torch.randint(-4, 5, (3, N, K), generator=g).to(BF16).cuda()
    dx, dw = torch.empty((25, K), device="cuda"), torch.empty((3, N, K), device="cuda")
    S.grouped_mm_dx(off, dy, w, dx, stream=stream())
    S.grouped_mm_dw(off, dy, x, dw, stream=stream())

    def loss(x, w):
        y = torch.empty((25, N), device="cuda")
        S.grouped_mm(off, x, w, y, stream=stream())
        return float((y.double() * dy.double()).sum())

    at = loss(x, w)
    for p, k in ((0, 0), (4, 39), (24, 17)):
        v = x.clone()
        v[p, k] += 1
        assert loss(v, w) - at == float(dx[p, k])
    for e, n, k in ((0, 0, 0), (1, 3, 3), (2, 23, 39)):
        v = w.clone()
        v[e, n, k] += 1
        assert loss(x, v) - at == float(dw[e, n, k])
    clean()


def test_bad_offsets_stay_inside_and_are_recorded(cuda):
    x, w = values((20, 64), BF16, 1), values((3, 64, 64), BF16, 2)
    guard = torch.full((60, 64), 5.0, dtype=F32, device="cuda")
    y, dw = guard[20:40], torch.zeros((3, 64, 64), device="cuda")
    for bad in ([0, 30, 10, 20], [-5, 4, 8, 1 << 30], [20, 10, 0, -1]):
        o = torch.tensor(bad, dtype=torch.int32, device="cuda")
        S.grouped_mm(o, x, w, y, stream=stream())
        torch.cuda.synchronize()
        assert S.device_error(0)[0] == -8
        S.grouped_mm_dw(o, x, x, dw, stream=stream())
        torch.cuda.synchronize()
        assert S.device_error(0)[0] == -8
        assert (guard[:20] == 5).all() and (guard[40:] == 5).all()


def test_same_bits_again_on_another_stream_and_in_a_graph(cuda):
    sizes = [700, 3, 0, 450]
    off, x, w, y = check_all(sizes, 512, 256, BF16, seed=20)
    o = off.cuda()
    side = torch.cuda.Stream()
    side.wait_stream(stream())
    z = torch.zeros_like(y)
    S.grouped_mm(o, x, w, z, stream=side)
    side.synchronize()
    assert torch.equal(y, z)
    graph = torch.cuda.CUDAGraph()
    dw1, dw2 = torch.zeros((4, 256, 256), device="cuda"), torch.zeros((4, 256, 256), device="cuda")
    with torch.cuda.graph(graph):
        S.grouped_mm(o, x, w, z, stream=stream())
        S.grouped_mm_dw(o, x, x, dw1, stream=stream())
    z.zero_()
    graph.replay()
    S.grouped_mm_dw(o, x, x, dw2, stream=stream())
    clean()
    assert torch.equal(y, z) and torch.equal(dw1, dw2)


@pytest.mark.parametrize("captured", [False, True])
def test_experts_of_a_routed_batch_forward_and_backward(cuda, captured):
    """route, gather, two products with a relu between, combine, and back: the whole run against 64 bits."""
    tokens, topk, groups, H, I = 150, 3, 7, 96, 136
    g = torch.Generator().manual_seed(3)
    ids = torch.stack([torch.randperm(groups, generator=g)[:topk] for _ in range(tokens)]).to(torch.int32)
    ids[5], ids[9, 1] = -1, -1  # a token without an expert, a pair without one
    x, dy = values((tokens, H), F16, 1), values((tokens, H), F16, 2)
    w1 = (values((groups, I, H), F32, 3) * H**-0.5).to(F16)
    w2 = (values((groups, H, I), F32, 4) * I**-0.5).to(F16)
    wt = torch.rand((tokens, topk), generator=g).cuda()
    i32 = dict(dtype=torch.int32, device="cuda")
    d_ids, off, pos = ids.cuda(), torch.zeros(groups + 1, **i32), torch.zeros((tokens, topk), **i32)
    rows = tokens * topk

    def e(c, dtype=F16, n=rows):
        return torch.zeros((n, c), dtype=dtype, device="cuda")

    xs, h, ys, y = e(H), e(I), e(H), e(H, n=tokens)
    dys, dh, dxs, dx, dwt = e(H), e(I), e(H), e(H, n=tokens), torch.zeros_like(wt)
    dw1, dw2 = torch.zeros(w1.shape, device="cuda"), torch.zeros(w2.shape, device="cuda")
    kept = {}

    def run():
        s = stream()
        S.route_build(d_ids, groups, off, None, pos, stream=s)
        S.route_gather(pos, x, xs, stream=s)
        S.grouped_mm(off, xs, w1, h, stream=s)
        a = torch.relu(h)
        S.grouped_mm(off, a, w2, ys, stream=s)
        S.route_combine(pos, ys, y, wt, stream=s)
        S.route_combine_grad(pos, dy, ys, wt, dys, dwt, stream=s)
        S.grouped_mm_dw(off, dys, a, dw2, stream=s)
        S.grouped_mm_dx(off, dys, w2, dh, stream=s)
        da = torch.where(h > 0, dh, 0)
        S.grouped_mm_dw(off, da, xs, dw1, stream=s)
        S.grouped_mm_dx(off, da, w1, dxs, stream=s)
        S.route_combine(pos, dxs, dx, stream=s)
        kept["da"] = da

    run()
    if captured:
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            run()
        for t in (xs, h, ys, y, dys, dh, dxs, dx, dwt, dw1, dw2):
            t.zero_()
        graph.replay()
    clean()
    X, W1, W2, WT = (R.d(t).requires_grad_() for t in (x, w1, w2, wt))
    rowsum = []
    for t in range(tokens):
        out = torch.zeros(H, dtype=torch.float64)
        for j in range(topk):
            v = int(ids[t, j])
            if v >= 0:
                out = out + WT[t, j] * (W2[v] @ torch.relu(W1[v] @ X[t]))
        rowsum.append(out)
    Y = torch.stack(rowsum)
    Y.backward(R.d(dy))
    # Five roundings to 16 bits lie on the longest path (h, ys or dys, dh, dxs, dx), each at most 2^-11 of a row whose
    # values are of one size, and relu may flip where |h| is below its rounding: 8 * 2^-11 of the 2-norm covers both.
    for name, got, want in (("y", y, Y), ("dx", dx, X.grad), ("dw1", dw1, W1.grad), ("dw2", dw2, W2.grad), ("dwt", dwt, WT.grad)):
        off_by = (R.d(got) - want.detach()).norm() / want.norm()
        assert off_by < 8 * 2.0**-11, (name, float(off_by))
    assert (y[5] == 0).all() and (dx[5] == 0).all() and (dwt[5] == 0).all()


def test_binding_refuses_other_shapes_and_types(cuda):
    o, x, w, y = offsets([4, 4]).cuda(), values((8, 16), BF16, 1), values((2, 24, 16), BF16, 2), values((8, 24), BF16, 3)
    for bad in (dict(x=x[:, :8]), dict(x=x.half()), dict(w=w.half()), dict(w=w.transpose(1, 2)), dict(y=y[:7]), dict(offsets=o[:2]), dict(offsets=o.long())):
        with pytest.raises(ValueError):
            S.grouped_mm(**{**dict(offsets=o, x=x, w=w, y=y), **bad})
    with pytest.raises(S.SpmmError):
        S.grouped_mm(o, x, w, y.half())  # out is neither x's type nor float32


def test_offsets_that_count_rows_thousands_of_times(cuda):
    """4096 groups that alternate between all 2^27 rows and none (out of order): 2^31 row tiles if each were taken."""
    rows, i32 = 1 << 27, dict(dtype=torch.int32, device="cuda")
    x, w = torch.zeros((rows, 8), dtype=BF16, device="cuda"), torch.zeros((4096, 8, 8), dtype=BF16, device="cuda")
    guard = torch.full((rows + 64, 8), 5.0, dtype=BF16, device="cuda")
    off = torch.tensor([0, rows] * 2048 + [0], **i32)
    for run in (lambda y: S.grouped_mm(off, x, w, y, stream=stream()), lambda y: S.grouped_mm_dx(off, x, w, y, stream=stream()),
                lambda y: S.lora(off, torch.zeros(4096, **i32), x, w, w, y, stream=stream())):
        run(guard[32:32 + rows])
        torch.cuda.synchronize()
        assert S.device_error(0)[0] == -8
        assert (guard[:32] == 5).all() and (guard[-32:] == 5).all()


@pytest.mark.parametrize("out", [F16, F32])
@pytest.mark.parametrize("sizes", [[700] + [3] * 30 + [0, 0, 350, 64, 1, 129], [0] * 60 + [200, 15, 33] + [1] * 70, [5, 0, 90] * 60, [40] * 128])
def test_weights_gradients_of_many_tiles(cuda, sizes, out):
    """More tiles than blocks, of up to 128 groups (sorted) and of more: each computed once, whoever takes it."""
    off = offsets(sizes, 4)
    rows = int(off[-1]) + 70
    dy, x = values((rows, 520), F16, 1), values((rows, 328), F16, 2)
    dy[:4], x[int(off[-1]):] = float("nan"), float("inf")
    want, mag = R.grouped_dw(off, dy, x)
    runs = []
    for _ in range(3):
        dw = torch.full((len(sizes), 520, 328), float("nan"), dtype=out, device="cuda")
        S.grouped_mm_dw(off.cuda(), dy, x, dw, stream=stream())
        runs.append(dw)
    clean()
    R.close(runs[0], want, mag, max(sizes), out, "dw")
    assert all(torch.equal(runs[0], t) for t in runs[1:])


def test_weights_gradients_on_two_streams_at_once_and_replayed(cuda):
    """Kernels that take each other's place on the GPU keep to their own tiles."""
    sizes = [900, 0] + [60] * 38
    off = offsets(sizes).cuda()
    n = sum(sizes)
    ops = [(values((n, 520), BF16, 10 * i), values((n, 776), BF16, 10 * i + 1)) for i in range(2)]
    wants = []
    for dy, x in ops:
        wants.append(torch.zeros((40, 520, 776), device="cuda"))
        S.grouped_mm_dw(off, dy, x, wants[-1], stream=stream())
    torch.cuda.synchronize()
    gots, graphs, streams = [torch.zeros_like(w) for w in wants], [], [torch.cuda.Stream() for _ in wants]
    for (dy, x), got in zip(ops, gots):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            for _ in range(10):
                S.grouped_mm_dw(off, dy, x, got, stream=stream())
        graphs.append(graph)
    for _ in range(3):
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
    clean()
    assert all(torch.equal(w, g) for w, g in zip(wants, gots))


@pytest.mark.parametrize("out", [F16, F32])
@pytest.mark.parametrize("sizes", [[0] * 150 + [200, 30] + [1] * 60, [3] * 100 + [0, 600, 129], [64] * 200, [1, 128] * 50])
def test_products_of_many_tiles(cuda, sizes, out):
    """More tiles than blocks, fewer than the groups could have, rows of 464 and of 1040 bytes."""
    check_all(sizes, 520, 232, F16, out=out, first=5, tail=77)
    check_all(sizes, 232, 520, F16, out=out)
