"""Tokens routed to groups and back on the GPU, against plain 64-bit forms."""
from __future__ import annotations

import threading

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


def make_ids(tokens, topk, groups, drop=0.0, seed=0):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, groups, (tokens, topk), generator=g, dtype=torch.int32)
    return torch.where(torch.rand((tokens, topk), generator=g) < drop, -1, ids).to(torch.int32)


def build(ids, groups, with_order=True):
    tokens, topk = ids.shape
    off = torch.full((groups + 1,), -7, dtype=torch.int32, device="cuda")
    order = torch.full((tokens * topk,), -7, dtype=torch.int32, device="cuda") if with_order else None
    pos = torch.full((tokens, topk), -7, dtype=torch.int32, device="cuda")
    S.route_build(ids.cuda(), groups, off, order, pos, stream=stream())
    return off, order, pos


def rows(n, H, dtype, pad=0, shift=0, seed=1):
    """n x H values at a row stride of H + pad, `shift` elements off the allocation's start."""
    g = torch.Generator().manual_seed(seed)
    buf = torch.full((n * (H + pad) + shift + 16,), float("nan"), dtype=dtype, device="cuda")
    t = buf[shift:shift + n * (H + pad)].view(n, H + pad)[:, :H]
    t.copy_(torch.randn((n, H), generator=g).to(dtype))
    return t


@pytest.mark.parametrize("tokens,topk,groups,drop", [
    (0, 2, 4, 0.0), (1, 1, 1, 0.0), (1, 8, 8, 0.0), (7, 3, 5, 0.3), (31, 1, 300, 0.0), (33, 2, 2, 1.0), (512, 8, 256, 0.1),
    (513, 8, 64, 0.0), (2049, 2, 3, 0.0), (5000, 3, 1025, 0.2), (4097, 1, 2048, 0.0), (3000, 4, 4096, 0.5), (70001, 8, 33, 0.05)])
def test_build_is_a_stable_sort(cuda, tokens, topk, groups, drop):
    ids = make_ids(tokens, topk, groups, drop, seed=tokens)
    off, order, pos = build(ids, groups)
    clean()
    want = R.sort_pairs(ids, groups)
    assert torch.equal(off.cpu(), want[0]) and torch.equal(order.cpu(), want[1]) and torch.equal(pos.cpu(), want[2])
    off2, _, pos2 = build(ids, groups, with_order=False)
    clean()
    assert torch.equal(off2, off) and torch.equal(pos2, pos)


def test_build_many_blocks_grow(cuda):
    """More pairs than 128 blocks of the usual size: one group of all, and groups that are runs of tokens."""
    tokens = 128 * 4096 + 77
    ids = (torch.arange(tokens, dtype=torch.int32) // 1000)[:, None].contiguous()
    groups = int(ids.max()) + 1
    off, order, pos = build(ids, groups)
    clean()
    assert torch.equal(pos.cpu().flatten(), torch.arange(tokens, dtype=torch.int32))
    assert torch.equal(order.cpu(), torch.arange(tokens, dtype=torch.int32))
    assert torch.equal(off.cpu()[:-1], torch.arange(0, groups * 1000, 1000, dtype=torch.int32)) and int(off[-1]) == tokens


@pytest.mark.parametrize("tokens", [40, 9000])
def test_build_records_an_id_past_the_groups(cuda, tokens):
    ids = make_ids(tokens, 1, 4, seed=3)
    ids[17] = 4
    off, order, pos = build(ids, 4)
    torch.cuda.synchronize()
    code, detail = S.device_error(0)
    assert code == -8 and detail == 17
    ids[17] = -1
    want = R.sort_pairs(ids, 4)
    assert torch.equal(off.cpu(), want[0]) and torch.equal(pos.cpu(), want[2]) and torch.equal(order.cpu(), want[1])


CASES = [(1, 1, 64, 0, 0), (1, 8, 4096, 0, 0), (5, 2, 1, 0, 0), (13, 3, 7, 0, 0), (9, 2, 130, 2, 0), (21, 4, 1001, 0, 0), (6, 9, 520, 24, 8),
         (33, 17, 96, 0, 1), (3, 2, 5000, 0, 0), (130, 1, 256, 0, 0)]


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("tokens,topk,H,pad,shift", CASES)
def test_gather_and_combine(cuda, tokens, topk, H, pad, shift, dtype):
    ids = make_ids(tokens, topk, 5, 0.25, seed=H)
    off, _, pos = build(ids, 5)
    x = rows(tokens, H, dtype, pad, shift)
    xs = rows(tokens * topk, H, dtype, pad, shift, seed=2)
    before = xs.clone()
    S.route_gather(pos, x, xs, stream=stream())
    clean()
    want = before.clone()
    for t in range(tokens):
        for j in range(topk):
            if int(pos[t, j]) >= 0:
                want[int(pos[t, j])] = x[t]
    assert torch.equal(xs, want)

    ys = rows(tokens * topk, H, dtype, pad, shift, seed=3)
    ys[int(off[-1]):] = float("nan")  # rows that no pair has are not read
    w = torch.randn((tokens, topk), generator=torch.Generator().manual_seed(4)).cuda()
    for weight in (w, None):
        y = rows(tokens, H, dtype, pad, shift, seed=5)
        S.route_combine(pos, ys, y, weight, stream=stream())
        clean()
        ref, mag = R.combine(pos, ys, weight)
        R.close(y, ref, mag, topk, dtype, "combine")


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("tokens,topk,H,pad,shift", CASES)
def test_combine_grad(cuda, tokens, topk, H, pad, shift, dtype):
    ids = make_ids(tokens, topk, 5, 0.25, seed=H)
    off, _, pos = build(ids, 5)
    dy = rows(tokens, H, dtype, pad, shift)
    ys = rows(tokens * topk, H, dtype, pad, shift, seed=3)
    ys[int(off[-1]):] = float("inf")
    w = torch.randn((tokens, topk), generator=torch.Generator().manual_seed(4)).cuda()
    outs = []
    for want_ys, want_w in ((True, True), (True, False), (False, True)):
        dys = rows(tokens * topk, H, dtype, pad, shift, seed=6)
        dw = torch.full((tokens, topk), float("nan"), device="cuda")
        S.route_combine_grad(pos, dy, ys if want_w else None, w, dys if want_ys else None, dw if want_w else None, stream=stream())
        clean()
        outs.append((dys, dw))
    fresh = rows(tokens * topk, H, dtype, pad, shift, seed=6)
    assert torch.equal(outs[1][0], outs[0][0]) and torch.equal(outs[2][1], outs[0][1]) and torch.equal(outs[2][0], fresh)
    dys, dw = outs[0]
    for t in range(tokens):
        for j in range(topk):
            p = int(pos[t, j])
            if p < 0:
                assert float(dw[t, j]) == 0.0
                continue
            exact = float(w[t, j]) * R.d(dy[t])
            R.close(dys[p], exact, exact.abs(), 1, dtype, "dys")
            prod = R.d(dy[t]) * R.d(ys[p])
            R.close(dw[t, j], prod.sum(), prod.abs().sum(), H, F32, "dw")
    n = int(off[-1])
    assert torch.equal(dys[n:], fresh[n:])


def test_combine_is_the_csr_product_of_the_routing_matrix(cuda):
    """With 32-bit rows the way back is spmm_csr_f32 on (tokens x rows, topk nonzeros a row), bit for bit."""
    tokens, topk, H = 300, 4, 128
    off, _, pos = build(make_ids(tokens, topk, 16), 16)
    ys = rows(tokens * topk, H, F32)
    w = torch.randn((tokens, topk), device="cuda")
    y, c = torch.empty((tokens, H), device="cuda"), torch.empty((tokens, H), device="cuda")
    S.route_combine(pos, ys, y, w, stream=stream())
    ptr = torch.arange(0, tokens * topk + 1, topk, dtype=torch.int32, device="cuda")
    S.csr_f32(S.device_view(tokens, tokens * topk, ptr, pos.flatten(), w.flatten()), ys, c, H, S.CSR_ROWWARP, stream())
    clean()
    assert torch.equal(y, c)


def test_gradients_against_differences(cuda):
    """combine is linear in ys and in w: a step along an element changes <y, dy> by the step times its gradient."""
    tokens, topk, H = 6, 3, 24
    _, _, pos = build(make_ids(tokens, topk, 4, 0.2), 4)
    ys, dy = rows(tokens * topk, H, F32), rows(tokens, H, F32, seed=8)
    w = torch.randn((tokens, topk), device="cuda")
    dys, dw = torch.zeros_like(ys), torch.empty_like(w)
    S.route_combine_grad(pos, dy, ys, w, dys, dw, stream=stream())
    dx = torch.empty((tokens, H), device="cuda")
    S.route_combine(pos, dys, dx, stream=stream())  # the gather's gradient

    def loss(ys, w):
        y = torch.empty((tokens, H), device="cuda")
        S.route_combine(pos, ys, y, w, stream=stream())
        return float((y.double() * dy.double()).sum())

    def there_and_back(x):
        xs = torch.zeros_like(ys)
        S.route_gather(pos, x, xs, stream=stream())
        return float((xs.double() * dys.double()).sum())

    at = loss(ys, w)
    # y is off by at most 3 * 2^-23 of magnitudes below 20, times |dy| summed: under 1e-3 of a step of 1.
    for t, j in ((0, 0), (2, 1), (5, 2)):
        v = w.clone()
        v[t, j] += 1.0
        assert abs(loss(ys, v) - at - float(dw[t, j])) < 1e-3
    for p, h in ((0, 0), (4, 23), (9, 5)):
        v = ys.clone()
        v[p, h] += 1.0
        assert abs(loss(v, w) - at - float(dys[p, h])) < 1e-3
    x = rows(tokens, H, F32, seed=9)
    at = there_and_back(x)
    for t, h in ((0, 3), (5, 11)):
        v = x.clone()
        v[t, h] += 1.0
        assert abs(there_and_back(v) - at - float(dx[t, h])) < 1e-3
    clean()


def test_bad_positions_are_recorded_and_skipped(cuda):
    pos = torch.tensor([[0, 5], [-2, 1]], dtype=torch.int32, device="cuda")  # 5 and -2 are no rows of 4
    x = rows(2, 16, BF16)
    xs = torch.zeros((4, 16), dtype=BF16, device="cuda")
    S.route_gather(pos, x, xs, stream=stream())
    torch.cuda.synchronize()
    assert S.device_error(0)[0] == -8
    assert torch.equal(xs, torch.stack([x[0], x[1], xs[2] * 0, xs[3] * 0]))
    y = torch.empty_like(x)
    S.route_combine(pos, xs, y, stream=stream())
    torch.cuda.synchronize()
    assert S.device_error(0)[0] == -8
    assert torch.equal(y, x)


def test_infinities_and_nan_stay_in_their_rows(cuda):
    pos = torch.tensor([[0], [1], [-1]], dtype=torch.int32, device="cuda")
    ys = torch.ones((3, 8), device="cuda")
    ys[0], ys[2] = float("inf"), float("nan")
    y = torch.empty((3, 8), device="cuda")
    S.route_combine(pos, ys, y, torch.zeros((3, 1), device="cuda"), stream=stream())
    clean()
    assert torch.isnan(y[0]).all() and (y[1:] == 0).all()  # 0 * inf is the formula's NaN; the rest are clean zeros


def test_another_stream_and_a_graph(cuda):
    tokens, topk, groups, H = 3000, 4, 32, 256
    ids = make_ids(tokens, topk, groups).cuda()
    x = rows(tokens, H, BF16)
    off = torch.zeros(groups + 1, dtype=torch.int32, device="cuda")
    order, pos = torch.zeros(tokens * topk, dtype=torch.int32, device="cuda"), torch.zeros_like(ids)
    xs, y = torch.zeros((tokens * topk, H), dtype=BF16, device="cuda"), torch.zeros_like(x)

    def work(s):
        S.route_build(ids, groups, off, order, pos, stream=s)
        S.route_gather(pos, x, xs, stream=s)
        S.route_combine(pos, xs, y, stream=s)

    side = torch.cuda.Stream()
    side.wait_stream(stream())
    work(side)  # with torch's current stream another one
    side.synchronize()
    eager = [t.clone() for t in (off, order, pos, xs, y)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        work(stream())
    ids.copy_(make_ids(tokens, topk, groups, 0.1, seed=9).cuda())
    graph.replay()
    torch.cuda.synchronize()
    want = R.sort_pairs(ids.cpu(), groups)
    assert torch.equal(off.cpu(), want[0]) and torch.equal(pos.cpu(), want[2])
    ids.copy_(make_ids(tokens, topk, groups).cuda())
    xs.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(eager, (off, order, pos, xs, y)))
    clean()


def test_offsets_past_32_bits(cuda):
    """Rows whose byte and element offsets need 64 bits: a wide stride in place of many rows."""
    tokens, H, ld = 5, 64, (1 << 30) + 8
    buf = torch.empty((tokens - 1) * ld + H, dtype=BF16, device="cuda")
    xs = buf.as_strided((tokens, H), (ld, 1))
    x = rows(tokens, H, BF16)
    pos = torch.tensor([[4], [3], [2], [1], [0]], dtype=torch.int32, device="cuda")
    S.route_gather(pos, x, xs, stream=stream())
    y = torch.empty_like(x)
    S.route_combine(pos, xs, y, stream=stream())
    clean()
    assert torch.equal(xs, x.flip(0)) and torch.equal(y, x)


def test_binding_refuses_other_shapes_types_and_strides(cuda):
    pos = torch.zeros((4, 2), dtype=torch.int32, device="cuda")
    x, xs = torch.zeros((4, 16), dtype=BF16, device="cuda"), torch.zeros((8, 16), dtype=BF16, device="cuda")
    for bad in (x[:3], x[:, :8], x.half(), x.t()):
        with pytest.raises(ValueError):
            S.route_gather(pos, bad, xs)
    with pytest.raises(ValueError):
        S.route_gather(pos.long(), x, xs)
    with pytest.raises(ValueError):
        S.route_gather(pos, x.t().contiguous().t(), xs)  # elements of a row apart
    with pytest.raises(ValueError):
        S.route_gather(pos, x[:1].expand(4, 16), xs)  # rows that overlap
    with pytest.raises(ValueError):
        S.route_combine(pos, xs, x, torch.zeros((4, 1), device="cuda"))
    with pytest.raises(ValueError):
        S.route_combine_grad(pos, x, xs, None, None, None)


def test_builds_of_different_sizes_from_two_threads(cuda):
    """Each on its own stream, with numbers of groups that take different amounts of shared memory."""
    wants, errors = {}, []

    def work(groups):
        try:
            ids = make_ids(600, 2, groups, 0.1, seed=groups)
            want = R.sort_pairs(ids, groups)[2]
            with torch.cuda.stream(torch.cuda.Stream()):
                on_gpu = ids.cuda()
                off = torch.zeros(groups + 1, dtype=torch.int32, device="cuda")
                pos = [torch.zeros((600, 2), dtype=torch.int32, device="cuda") for _ in range(300)]
                for p in pos:
                    S.route_build(on_gpu, groups, off, None, p, stream=stream())
                stream().synchronize()
                wants[groups] = all(torch.equal(p.cpu(), want) for p in pos)
        except Exception as e:  # noqa: BLE001 - shown below
            errors.append(e)

    threads = [threading.Thread(target=work, args=(groups,)) for groups in (4096, 2500, 1500)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    clean()
    assert not errors and wants == {4096: True, 2500: True, 1500: True}, errors
