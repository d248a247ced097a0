"""Grouped matrix products (pf_gmm_*, pf_gmm_wgrad_*), through the C ABI,
against 64-bit products group by group.

Tolerances: products of 16-bit values are exact in fp32; a reduction of c terms
in fp32, each addition within one unit 2^-23 (a matrix unit may truncate), is
within (c + 4) 2^-23 of the sum of the terms' sizes; the result is rounded once
to its type.
"""
import math

import pytest
import torch

from dense_cases import DT, SENTINEL, TINY, UNIT, Buffer, pointers, within

pytestmark = pytest.mark.gpu


def stack(groups, rows, cols, dt, offset, pad, gap, data=None):
    """(groups, rows, cols) inside a sentinel-filled buffer."""
    ld = cols + pad
    step = rows * ld + gap
    flat = torch.full((offset + groups * step + 64,), SENTINEL, dtype=dt, device="cuda")
    view = torch.as_strided(flat, (groups, rows, cols), (step, ld, 1), offset)
    if data is not None:
        view.copy_(data)
    return flat, view


def stack_untouched(flat, view):
    keep = flat.clone()
    torch.as_strided(keep, view.shape, view.stride(), view.storage_offset()).fill_(SENTINEL)
    return bool((keep == SENTINEL).all())


def check(pf, lengths, n, k, mode, dtype="bf16", alpha=1.0, beta=0.0, idx=torch.int32, start=0,
          after=0, offset=0, pads=(0, 0, 0), gap=0, out="same", seed=0, X=None):
    """mode: fwd (X W^T), dx (X W) or dw (dY^T X), n and k as in the C call."""
    dt = DT[dtype]
    ot = torch.float32 if out == "f32" else dt
    groups, rows = len(lengths), start + sum(lengths) + after
    g = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *s: torch.randn(*s, generator=g, device="cuda").to(dt)  # noqa: E731
    ptr = pointers(lengths, start, idx)
    bounds = ptr.tolist()
    X = normal(rows, k) if X is None else X
    xb = Buffer(rows, k, dt, offset, pads[0], X)
    h = pf.Handle()
    if mode == "dw":
        dY = normal(rows, n)
        yb = Buffer(rows, n, dt, offset, pads[1], dY)
        d0 = torch.randn(groups, n, k, generator=g, device="cuda").to(ot)
        flat, dW = stack(groups, n, k, ot, offset, pads[2], gap, d0 if beta else None)
        pf.grouped_wgrad(h, ptr, yb.view, xb.view, dW, alpha, beta)
    else:
        shape = (n, k) if mode == "fwd" else (k, n)
        W = normal(groups, *shape)
        flat, w = stack(groups, *shape, dt, offset, pads[1], gap, W)
        Y0 = normal(rows, n)
        yb = Buffer(rows, n, dt, offset, pads[2], Y0 if beta else None)
        pf.grouped_mm(h, ptr, xb.view, w, yb.view, mode == "fwd", alpha, beta)
    torch.cuda.synchronize()
    assert h.device_error() == 0
    h.close()
    assert xb.outside_untouched() and yb.outside_untouched()
    if mode == "dw":
        assert stack_untouched(flat, dW)
    for i in range(groups):
        a, b = bounds[i], bounds[i + 1]
        x = X[a:b].double()
        if mode == "dw":
            y, got, before, count = dY[a:b].double(), dW[i], d0[i], b - a
            want, size = alpha * (y.t() @ x), abs(alpha) * (y.t().abs() @ x.abs())
        else:
            m = W[i].double().t() if mode == "fwd" else W[i].double()
            got, before, count = yb.view[a:b], Y0[a:b], k
            want, size = alpha * (x @ m), abs(alpha) * (x.abs() @ m.abs())
        if beta:
            want, size = want + beta * before.double(), size + abs(beta) * before.double().abs()
        unit = UNIT["f32"] if out == "f32" else UNIT[dtype]
        within(got, want, unit * want.abs() + (count + 4) * 2.0 ** -23 * size + TINY[dtype])
    if mode != "dw" and (start or after):  # rows of no group
        keep = (Y0 if beta else torch.full_like(Y0, SENTINEL))
        for part in (slice(0, start), slice(rows - after, rows)):
            assert torch.equal(yb.view[part], keep[part])


MODES = ["fwd", "dx", "dw"]


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("n,k", [(1, 1), (8, 8), (64, 64), (40, 136), (200, 72), (7, 33),
                                 (129, 257), (256, 128), (512, 520), (1000, 96)])
def test_sizes(pf, mode, dtype, n, k):
    check(pf, [5, 0, 130, 1, 64, 17], n, k, mode, dtype, seed=n)


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("lengths", [[0], [1], [0, 0, 0], [300], [1] * 70, [0, 0, 513, 0],
                                     [15, 16, 17, 31, 32, 33], [63, 64, 65, 127, 128, 129],
                                     [255, 256, 257], [2000, 1, 0, 900], [3] * 40 + [0] * 40 + [9]])
@pytest.mark.parametrize("n,k", [(136, 72), (45, 27)])
def test_group_lengths(pf, mode, lengths, n, k):
    check(pf, lengths, n, k, mode, seed=len(lengths))


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("idx", [torch.int32, torch.int64])
@pytest.mark.parametrize("offset,pads,gap", [(0, (0, 0, 0), 0), (8, (8, 16, 24), 64),
                                             (1, (0, 0, 0), 0), (0, (1, 0, 0), 0),
                                             (0, (0, 1, 0), 0), (0, (0, 0, 1), 0),
                                             (0, (4, 4, 4), 4), (0, (0, 0, 0), 3)])
def test_strides_alpha_beta_other_rows(pf, mode, idx, offset, pads, gap):
    """Leading dimensions, offsets, gaps between matrices, alpha and beta, rows
    before the first group and after the last."""
    check(pf, [30, 0, 7, 150], 72, 104, mode, "f16", -0.5, 1.5, idx, start=13, after=21,
          offset=offset, pads=pads, gap=gap, seed=7)


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("n,k", [(512, 2048), (2048, 512)])
@pytest.mark.parametrize("lengths", [[1, 2, 0, 1], [20], [3] * 9])
def test_few_rows(pf, mode, n, k, lengths):
    """Few rows to a group: the shapes of a decoding step."""
    check(pf, lengths, n, k, mode, seed=2)


@pytest.mark.parametrize("mode", MODES)
def test_many_tiles(pf, mode):
    """More tiles than the GPU holds at once, several to a CTA."""
    check(pf, [700, 0, 1300, 333, 2048, 64, 1], 1096, 776, mode, seed=3)


def test_long_reduction_few_outputs(pf):
    check(pf, [9000, 5000], 64, 72, "dw", seed=4)
    check(pf, [12], 64, 16384, "fwd", seed=4)


def test_wgrad_in_32_bits_accumulates(pf):
    check(pf, [40, 0, 500], 72, 200, "dw", out="f32", seed=5)
    check(pf, [40, 0, 500], 72, 200, "dw", "f16", 2.0, 1.0, out="f32", seed=5, pads=(0, 0, 4))
    check(pf, [40, 0, 500], 33, 21, "dw", "f16", 2.0, 1.0, out="f32", seed=5)


@pytest.mark.parametrize("n,k", [(72, 64), (33, 21)])
def test_nothing_leaks_between_groups(pf, n, k):
    """NaN in one group's rows, and in rows of no group, reaches no other
    group's results, in every direction."""
    lengths, start = [20, 33, 70, 5], 3
    rows = start + sum(lengths) + 4
    dt = torch.bfloat16
    ptr = pointers(lengths, start)
    bad = slice(start + 20, start + 53)  # group 1
    X, dY = torch.ones(rows, k, dtype=dt, device="cuda"), torch.ones(rows, n, dtype=dt, device="cuda")
    for t in (X, dY):
        t[bad] = math.nan
        t[:start] = math.nan
        t[-4:] = math.inf
    W = torch.ones(4, n, k, dtype=dt, device="cuda")
    h = pf.Handle()
    Y, dX = torch.zeros_like(dY), torch.zeros_like(X)
    dW = torch.zeros(4, n, k, dtype=dt, device="cuda")
    pf.grouped_mm(h, ptr, X, W, Y, True)
    pf.grouped_mm(h, ptr, dY, W, dX, False)
    pf.grouped_wgrad(h, ptr, dY, X, dW)
    good = torch.ones(rows, dtype=torch.bool)
    good[bad] = good[:start] = good[-4:] = False
    assert bool((Y[good] == k).all()) and bool((dX[good] == n).all())
    assert bool(Y[bad].isnan().all()) and bool(dX[bad].isnan().all())
    assert bool((Y[:start] == 0).all()) and bool((Y[-4:] == 0).all())
    for i, c in enumerate(lengths):
        assert bool(dW[i].isnan().all()) if i == 1 else bool((dW[i] == c).all())
    # NaN in one group's matrix stays in that group's rows
    W[2] = math.nan
    X[:] = 1
    pf.grouped_mm(h, ptr, X, W, Y, True)
    assert bool((Y[start:start + 53] == k).all()) and bool((Y[start + 123:-4] == k).all())
    assert h.device_error() == 0
    h.close()


def test_nan_output_is_not_read_without_beta(pf):
    X, W = torch.ones(40, 64, dtype=torch.bfloat16, device="cuda"), \
        torch.ones(2, 64, 64, dtype=torch.bfloat16, device="cuda")
    Y = torch.full((40, 64), math.nan, dtype=torch.bfloat16, device="cuda")
    dW = torch.full((2, 64, 64), math.nan, device="cuda")
    h = pf.Handle()
    pf.grouped_mm(h, pointers([17, 23]), X, W, Y)
    pf.grouped_wgrad(h, pointers([40, 0]), X, X, dW)
    assert bool((Y == 64).all()) and bool((dW[0] == 40).all()) and bool((dW[1] == 0).all())
    h.close()


@pytest.mark.parametrize("n,k", [(64, 128), (30, 50)])
def test_same_bits_every_call(pf, n, k):
    g = torch.Generator(device="cuda").manual_seed(1)
    X = torch.randn(5000, k, generator=g, device="cuda").bfloat16()
    dY = torch.randn(5000, n, generator=g, device="cuda").bfloat16()
    W = torch.randn(3, n, k, generator=g, device="cuda").bfloat16()
    ptr = pointers([4000, 11, 989])
    h = pf.Handle()
    got = []
    for _ in range(3):
        Y, dX, dW = torch.empty_like(dY), torch.empty_like(X), torch.empty_like(W)
        pf.grouped_mm(h, ptr, X, W, Y)
        pf.grouped_mm(h, ptr, dY, W, dX, False)
        pf.grouped_wgrad(h, ptr, dY, X, dW)
        got.append((Y, dX, dW))
    for other in got[1:]:
        assert all(torch.equal(a, b) for a, b in zip(got[0], other))
    h.close()


def test_gradients_against_differences(pf):
    """Y is linear in X and in W: with f = <dY, Y>, f(X + E) - f(X) is f(E)
    exactly, and <dX, E> has to equal it; likewise <dW, F> for a change F of W.
    Both sides carry their outputs' rounding."""
    dt, n, k, rows = torch.float16, 72, 104, 90
    g = torch.Generator(device="cuda").manual_seed(9)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda").to(dt)  # noqa: E731
    X, E, dY, W, F = r(rows, k), r(rows, k), r(rows, n), r(3, n, k), r(3, n, k)
    ptr = pointers([50, 0, 40])
    h = pf.Handle()
    YE, YF, dX, dW = torch.empty_like(dY), torch.empty_like(dY), torch.empty_like(X), torch.empty_like(W)
    pf.grouped_mm(h, ptr, E, W, YE)
    pf.grouped_mm(h, ptr, X, F, YF)
    pf.grouped_mm(h, ptr, dY, W, dX, False)
    pf.grouped_wgrad(h, ptr, dY, X, dW)
    for Y, d, way in ((YE, dX, E), (YF, dW, F)):
        a, b = dY.double() * Y.double(), d.double() * way.double()
        tol = 2 * UNIT["f16"] * (a.abs().sum() + b.abs().sum())
        within((a.sum() - b.sum())[None], torch.zeros(1), tol[None])
    h.close()


def test_bad_pointers_are_flagged(pf):
    h = pf.Handle()
    dt = torch.bfloat16
    for n, k in ((64, 64), (33, 21)):
        X, W = torch.ones(20, k, dtype=dt, device="cuda"), torch.ones(3, n, k, dtype=dt, device="cuda")
        Y, dW = torch.zeros(20, n, dtype=dt, device="cuda"), torch.full_like(W, 5.0)
        for bad in ([0, 8, 4, 20], [-3, 8, 8, 20], [0, 8, 8, 21]):
            ptr = torch.tensor(bad, dtype=torch.int32, device="cuda")
            Y.zero_()
            pf.grouped_mm(h, ptr, X, W, Y)
            assert h.device_error() == 4
            dW.fill_(5.0)
            pf.grouped_wgrad(h, ptr, torch.ones_like(Y), X, dW)
            assert h.device_error() == 4
            for i in range(3):
                a, b = bad[i], bad[i + 1]
                if a < 0 or b < a or b > 20:
                    assert bool((dW[i] == 0).all())
                else:
                    assert bool((Y[a:b] == k).all()) and bool((dW[i] == b - a).all())
    h.close()


def test_nothing_to_do(pf):
    h = pf.Handle()
    dt = torch.bfloat16
    X, W = torch.ones(0, 64, dtype=dt, device="cuda"), torch.ones(2, 64, 64, dtype=dt, device="cuda")
    pf.grouped_mm(h, pointers([0, 0]), X, W, X.clone())
    dW = torch.ones_like(W)
    pf.grouped_wgrad(h, pointers([0, 0]), X, X, dW, beta=2.0)
    assert bool((dW == 2).all())
    none = torch.empty(0, 64, 64, dtype=dt, device="cuda")
    Y = torch.full((5, 64), 3.0, dtype=dt, device="cuda")
    pf.grouped_mm(h, pointers([]), Y, none, Y.clone())
    # an empty reduction: Y = beta * Y
    X0, W0 = torch.ones(5, 0, dtype=dt, device="cuda"), torch.ones(1, 64, 0, dtype=dt, device="cuda")
    pf.grouped_mm(h, pointers([5]), X0, W0, Y, beta=2.0)
    assert bool((Y == 6).all()) and h.device_error() == 0
    h.close()


def test_capture(pf):
    """No call waits for the host or allocates after the first of its size."""
    h = pf.Handle()
    dt = torch.bfloat16
    X, W = torch.ones(50, 256, dtype=dt, device="cuda"), torch.ones(2, 128, 256, dtype=dt, device="cuda")
    Y, dW = torch.zeros(50, 128, dtype=dt, device="cuda"), torch.zeros_like(W)
    ptr = pointers([20, 30])

    def step():
        pf.grouped_mm(h, ptr, X, W, Y)
        pf.grouped_wgrad(h, ptr, Y, X, dW)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    Y.zero_()
    dW.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert bool((Y == 256).all()) and bool((dW[1] == 30 * 256).all())
    h.close()


def test_refusals(pf):
    h = pf.Handle()
    dt = torch.bfloat16
    X, W = torch.ones(50, 64, dtype=dt, device="cuda"), torch.ones(2, 32, 64, dtype=dt, device="cuda")
    Y, ptr = torch.zeros(50, 32, dtype=dt, device="cuda"), pointers([20, 30])
    pf.grouped_mm(h, ptr, X, W, Y)

    def refused(f, *a):
        with pytest.raises(pf.PfError) as e:
            f(h, *a)
        assert e.value.status == 1

    mm, wg = pf.grouped_mm, pf.grouped_wgrad
    refused(mm, ptr, X, W, Y, False)             # shapes of the other direction
    refused(mm, ptr, X.float(), W.float(), Y.float())
    refused(mm, ptr, X, W.half(), Y)
    refused(mm, ptr, X, W, Y.half())
    refused(mm, ptr[:2], X, W, Y)                # one group, two matrices
    refused(mm, ptr.float(), X, W, Y)
    refused(mm, ptr.cpu(), X, W, Y)
    refused(mm, ptr, X.cpu(), W, Y)
    refused(mm, ptr, X.t().contiguous().t(), W, Y)
    refused(mm, ptr, X, W.transpose(1, 2).contiguous().transpose(1, 2), Y)
    refused(mm, ptr, X, W, Y[:40])
    refused(mm, ptr, X, W[:1].expand(2, 32, 64)[:, :, :32], Y)
    refused(wg, ptr, Y, X, W.double())
    refused(wg, ptr, Y, X, W[:, :, :32])
    refused(wg, ptr, Y.half(), X, W)
    refused(wg, ptr, Y, X, W[:1].expand(2, 32, 64))  # one place for two results
    p = lambda t: t.data_ptr()  # noqa: E731
    args = [h.ptr, 2, 50, 32, 64, p(ptr), p(X), 64, p(W), 64, 2048, 1, 1.0, 0.0, p(Y), 32, None]
    assert pf.lib.pf_gmm_bf16_i32(*args) == 0
    for at, bad in ((0, None), (1, -1), (2, -1), (3, -1), (4, -1), (5, None), (6, None), (7, 63),
                    (8, None), (9, 63), (10, 2047), (14, None), (15, 31), (6, p(X) + 1),
                    (5, p(ptr) + 2), (1, 2 ** 31)):
        a = list(args)
        a[at] = bad
        assert pf.lib.pf_gmm_bf16_i32(*a) == 1, at
    args = [h.ptr, 2, 50, 32, 64, p(ptr), p(Y), 32, p(X), 64, 1.0, 0.0, p(W), 2, 64, 2048, None]
    assert pf.lib.pf_gmm_wgrad_bf16_i32(*args) == 0
    for at, bad in ((0, None), (1, -1), (5, None), (6, None), (7, 31), (8, None), (9, 63),
                    (12, None), (13, 8), (14, 63), (15, 2047), (12, p(W) + 1)):
        a = list(args)
        a[at] = bad
        assert pf.lib.pf_gmm_wgrad_bf16_i32(*a) == 1, at
    assert h.device_error() == 0
    h.close()


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("lengths,n,k", [([17], 512, 2048), ([3, 0, 300, 1], 264, 1000),
                                         ([2100], 136, 72), ([1500, 0, 33, 1000], 128, 264)])
def test_split_sums(pf, mode, lengths, n, k):
    """Few tiles: their sums are cut into parts and joined, with alpha and beta,
    uneven last parts, and rows before and after the groups."""
    check(pf, lengths, n, k, mode, "bf16", 0.5, -1.0, start=2, after=3, seed=11)
    check(pf, lengths, n, k, mode, "f16", out="f32" if mode == "dw" else "same", seed=12)


def test_split_sums_leave_no_trace(pf):
    """The joins' counters are back at zero after every call: calls of other
    shapes through the same handle, in any order, give the same bits."""
    g = torch.Generator(device="cuda").manual_seed(2)
    h = pf.Handle()
    r = lambda *s: torch.randn(*s, generator=g, device="cuda").bfloat16()  # noqa: E731
    cases = [(pointers([17]), r(17, 2048), r(1, 512, 2048)),
             (pointers([5, 90, 0, 1]), r(96, 512), r(4, 256, 512)),
             (pointers([400]), r(400, 1024), r(1, 128, 1024))]
    outs = []
    for _ in range(3):
        for ptr, X, W in cases:
            Y = torch.empty(X.shape[0], W.shape[1], dtype=X.dtype, device="cuda")
            dW = torch.empty_like(W)
            pf.grouped_mm(h, ptr, X, W, Y)
            pf.grouped_wgrad(h, ptr, Y, X, dW)
            outs.append((Y, dW))
    for i, (Y, dW) in enumerate(outs):
        assert torch.equal(Y, outs[i % 3][0]) and torch.equal(dW, outs[i % 3][1])
    assert h.device_error() == 0
    h.close()


def test_overlapping_groups_are_flagged(pf):
    """Pointers that go back and forth name more rows than there are: flagged,
    and nothing is written outside of the scratch made for valid ones."""
    h = pf.Handle()
    dt = torch.bfloat16
    ptr = torch.tensor([0, 20] * 40 + [0], dtype=torch.int32, device="cuda")
    X, W = torch.ones(20, 512, dtype=dt, device="cuda"), torch.ones(80, 64, 512, dtype=dt, device="cuda")
    Y = torch.zeros(20, 64, dtype=dt, device="cuda")
    pf.grouped_mm(h, ptr, X, W, Y)
    assert h.device_error() == 4
    pf.grouped_mm(h, pointers([20] + [0] * 79), X, W, Y)
    assert h.device_error() == 0 and bool((Y == 512).all())
    h.close()


def test_one_matrix_for_all_groups(pf):
    """W expanded to all groups (distance 0 between matrices)."""
    g = torch.Generator(device="cuda").manual_seed(3)
    X, W = (torch.randn(*s, generator=g, device="cuda").bfloat16() for s in ((90, 72), (1, 40, 72)))
    ptr = pointers([30, 0, 60])
    h = pf.Handle()
    for w in (W, W[:, :, :71]):
        k = w.shape[2]
        Y, Z = torch.empty(90, 40, dtype=X.dtype, device="cuda"), torch.empty(90, 40, dtype=X.dtype, device="cuda")
        pf.grouped_mm(h, ptr, X[:, :k], w.expand(3, 40, k), Y)
        pf.grouped_mm(h, ptr, X[:, :k], w.repeat(3, 1, 1), Z)
        # (another leading dimension may take the other kernel: another order of sums)
        within(Y, Z.double(), 2 * UNIT["bf16"] * Z.double().abs() + 1e-4)
    assert h.device_error() == 0
    h.close()


def test_captured_split_sums_outlive_larger_calls(pf):
    """A graph of split products (17 rows: 4 tiles of 32 blocks; a gradient
    over 5000 rows) replayed after larger split calls on the same handle, between
    other calls that use the same scratch."""
    g = torch.Generator(device="cuda").manual_seed(4)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda").bfloat16()  # noqa: E731
    h = pf.Handle()
    X, W, ptr = r(17, 2048), r(1, 512, 2048), pointers([17])
    A, B, ptr2 = r(5000, 64), r(5000, 72), pointers([5000])
    Y, dW = torch.empty(17, 512, dtype=X.dtype, device="cuda"), torch.empty(1, 64, 72, device="cuda")

    def step():
        pf.grouped_mm(h, ptr, X, W, Y)
        pf.grouped_wgrad(h, ptr2, A, B, dW)

    step()
    want = Y.clone(), dW.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    more = [(pointers([3, 0, 300, 1]), r(304, 1000), r(4, 264, 1000)),
            (pointers([60]), r(60, 4096), r(1, 4096, 4096)),
            (pointers([1] * 30), r(30, 2048), r(30, 128, 2048))]
    for p, x, w in more:
        Z, first = (torch.empty(x.shape[0], w.shape[1], dtype=x.dtype, device="cuda")
                    for _ in range(2))
        pf.grouped_mm(h, p, x, w, first)
        Y.fill_(math.nan)
        dW.fill_(math.nan)
        graph.replay()
        pf.grouped_mm(h, p, x, w, Z)
        assert torch.equal(Y, want[0]) and torch.equal(dW, want[1]) and torch.equal(Z, first)
    assert h.device_error() == 0
    del graph
    h.close()


def test_first_split_call_in_a_capture_is_refused(pf):
    h = pf.Handle()
    X = torch.ones(17, 2048, dtype=torch.bfloat16, device="cuda")
    W, Y = torch.ones(1, 512, 2048, dtype=X.dtype, device="cuda"), torch.zeros(17, 512, dtype=X.dtype,
                                                                              device="cuda")
    ptr, graph, other = pointers([17]), torch.cuda.CUDAGraph(), torch.zeros(4, device="cuda")
    with torch.cuda.graph(graph):
        with pytest.raises(pf.PfError) as e:
            pf.grouped_mm(h, ptr, X, W, Y)
        other += 1.0
    assert e.value.status == 4
    graph.replay()  # the capture goes on without it
    assert other.tolist() == [1.0] * 4 and float(Y.abs().sum()) == 0.0
    pf.grouped_mm(h, ptr, X, W, Y)
    assert bool((Y == 2048).all()) and h.device_error() == 0
    del graph
    h.close()
