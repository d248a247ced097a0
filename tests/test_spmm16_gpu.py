"""16-bit SpMM over wide rows (pf_spmm_f16/bf16_*) and the gradient of its
values (pf_sddmm_*), through the C ABI, against 64-bit sums on the CPU.

Tolerances: products of 16-bit values are exact in fp32, so a sum of c terms
is within (c + 4) 2^-24 of the sum of the terms' sizes (the + 4: alpha, beta and
their sum), and the result is rounded once to its type.
"""
import pytest
import torch

from dense_cases import DT, SENTINEL, TINY, UNIT, Buffer, pointers, within

pytestmark = pytest.mark.gpu


def matrix(lengths, n, seed):
    g = torch.Generator().manual_seed(seed)
    nnz = sum(lengths)
    return (torch.randint(0, max(n, 1), (nnz,), generator=g, dtype=torch.int32),
            torch.randn(nnz, generator=g))


def rows_of(lengths):
    return torch.repeat_interleave(torch.arange(len(lengths)), torch.tensor(lengths))


def check_spmm(pf, lengths, n, k, dtype, alpha=1.0, beta=0.0, idx=torch.int32, offset=0, padx=0,
               pady=0, start=0, seed=0):
    dt = DT[dtype]
    m, nnz = len(lengths), sum(lengths)
    col, val = matrix(lengths, n, seed)
    val = val.to(dt)
    g = torch.Generator().manual_seed(seed + 1)
    X, Y0 = torch.randn(n, k, generator=g).to(dt), torch.randn(m, k, generator=g).to(dt)
    xb = Buffer(n, k, dt, offset, padx, X)
    yb = Buffer(m, k, dt, offset, pady, Y0 if beta else None)
    lead = torch.zeros(start)
    h = pf.Handle()
    pf.spmm(h, m, n, nnz, pointers(lengths, start, idx), torch.cat([lead.int(), col]).cuda(),
            torch.cat([lead.to(dt), val]).cuda(), xb.view, yb.view, alpha, beta)
    torch.cuda.synchronize()
    assert h.device_error() == 0
    h.close()
    assert xb.outside_untouched() and yb.outside_untouched()
    row = rows_of(lengths)
    terms = val.double()[:, None] * X.double()[col.long()]
    want = alpha * torch.zeros(m, k, dtype=torch.float64).index_add_(0, row, terms)
    size = abs(alpha) * torch.zeros(m, k, dtype=torch.float64).index_add_(0, row, terms.abs())
    if beta:
        want += beta * Y0.double()
        size += abs(beta) * Y0.double().abs()
    count = torch.tensor(lengths, dtype=torch.float64)[:, None] + 4
    within(yb.view, want, UNIT[dtype] * want.abs() + count * 2.0 ** -24 * size + TINY[dtype])


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("k", [1, 2, 3, 8, 31, 64, 257, 1000, 1531, 2048, 4100])
def test_widths(pf, dtype, k):
    check_spmm(pf, [3, 0, 1, 8, 2, 5, 0, 17], 29, k, dtype, seed=k)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("idx", [torch.int32, torch.int64])
@pytest.mark.parametrize("offset,padx,pady", [(0, 0, 0), (1, 0, 0), (0, 1, 0), (0, 0, 1),
                                              (2, 2, 4), (3, 5, 6), (8, 8, 16)])
def test_alignment_strides_alpha_beta(pf, dtype, idx, offset, padx, pady):
    check_spmm(pf, [4, 1, 0, 2, 9], 12, 200, dtype, -0.5, 1.5, idx, offset, padx, pady, seed=3)


@pytest.mark.parametrize("lengths", [[0], [1], [5000], [1] * 3000, [0] * 40, [0, 300, 0, 7]])
@pytest.mark.parametrize("k", [40, 515])
def test_row_lengths(pf, lengths, k):
    check_spmm(pf, lengths, 1000, k, "bf16", seed=4)


def test_slice_of_a_larger_matrix(pf):
    check_spmm(pf, [2, 0, 3], 9, 72, "f16", start=5, seed=5)


@pytest.mark.parametrize("lengths", [[3, 0, 1, 8, 2, 5, 0, 17, 0], [1, 0, 1, 1, 0], [0, 40], [7],
                                     [5, 0, 0, 0, 0, 0, 0, 0, 0, 0]])
@pytest.mark.parametrize("k", [64, 51])
def test_pointers_that_end_at_the_largest_index(pf, lengths, k):
    """A slice whose 32-bit pointers end at 2^31 - 1 (col and val are addressed
    absolutely: only the slice's part of them is there) gives what the same rows
    give at 0, for the product and for the values' gradient."""
    dt, m, n, nnz = torch.bfloat16, len(lengths), 12, sum(lengths)
    start = 2 ** 31 - 1 - nnz
    col, val = matrix(lengths, n, 14)
    g = torch.Generator().manual_seed(15)
    X, dY = torch.randn(n, k, generator=g).to(dt).cuda(), torch.randn(m, k, generator=g).to(dt).cuda()
    col, val = col.cuda(), val.to(dt).cuda()
    h = pf.Handle()
    Y, Z = torch.zeros_like(dY), torch.ones_like(dY)
    d, e = torch.zeros_like(val), torch.ones_like(val)
    ptr, at0 = pointers(lengths, start), pointers(lengths)
    p = lambda t: t.data_ptr()  # noqa: E731
    pf.spmm(h, m, n, nnz, at0, col, val, X, Y)
    pf.sddmm(h, m, n, nnz, at0, col, dY, X, d)
    assert pf.lib.pf_spmm_bf16_i32(h.ptr, m, n, nnz, p(ptr), p(col) - 4 * start, p(val) - 2 * start,
                                   k, 1.0, p(X), k, 0.0, p(Z), k, None) == 0
    assert pf.lib.pf_sddmm_bf16_i32(h.ptr, m, n, nnz, p(ptr), p(col) - 4 * start, k, 1.0, p(dY), k,
                                    p(X), k, 0.0, p(e) - 2 * start, None) == 0
    assert h.device_error() == 0 and torch.equal(Y, Z) and torch.equal(d, e)
    h.close()


def test_column_agrees_with_spmv(pf):
    lengths = [3, 0, 4, 1]
    col, val = matrix(lengths, 10, 6)
    X = torch.randn(10, 1).to(torch.bfloat16).cuda()
    ptr, col, val = pointers(lengths), col.cuda(), val.to(torch.bfloat16).cuda()
    Y, y = (torch.zeros(4, 1, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    h = pf.Handle()
    pf.spmm(h, 4, 10, 8, ptr, col, val, X, Y)
    pf.spmv(h, 4, 10, 8, ptr, col, val, X.view(-1), y.view(-1))
    within(Y, y.double(), UNIT["bf16"] * 2 * y.double().abs() + 2.0 ** -20)
    h.close()


def test_infinities_and_nan_stay_in_their_rows(pf):
    """A value of inf or NaN reaches the rows that use it and no others, nor
    does it cross from the columns beside it."""
    n, k = 6, 130
    X = torch.ones(n, k, dtype=torch.bfloat16)
    X[2, 7], X[3, 64] = float("inf"), float("nan")
    lengths = [2, 2, 2]
    col = torch.tensor([0, 1, 2, 0, 3, 4], dtype=torch.int32)
    Y = torch.zeros(3, k, dtype=torch.bfloat16, device="cuda")
    h = pf.Handle()
    pf.spmm(h, 3, n, 6, pointers(lengths), col.cuda(),
            torch.ones(6, dtype=torch.bfloat16, device="cuda"), X.cuda(), Y)
    want = torch.full((3, k), 2.0)
    want[1, 7], want[2, 64] = float("inf"), float("nan")
    within(Y, want, torch.zeros_like(want))
    h.close()


def check_sddmm(pf, lengths, n, k, dtype, alpha=1.0, beta=0.0, idx=torch.int32, offset=0, padx=0,
                pady=0, start=0, seed=0):
    dt = DT[dtype]
    m, nnz = len(lengths), sum(lengths)
    col, d0 = matrix(lengths, n, seed)
    d0 = d0.to(dt)
    g = torch.Generator().manual_seed(seed + 1)
    X, dY = torch.randn(n, k, generator=g).to(dt), torch.randn(m, k, generator=g).to(dt)
    xb, yb = Buffer(n, k, dt, offset, padx, X), Buffer(m, k, dt, offset, pady, dY)
    out = torch.full((start + nnz + 9,), SENTINEL, dtype=dt, device="cuda")
    if beta:
        out[start:start + nnz] = d0.cuda()
    h = pf.Handle()
    pf.sddmm(h, m, n, nnz, pointers(lengths, start, idx),
             torch.cat([torch.zeros(start, dtype=torch.int32), col]).cuda(), yb.view, xb.view, out,
             alpha, beta)
    torch.cuda.synchronize()
    assert h.device_error() == 0
    h.close()
    assert xb.outside_untouched() and yb.outside_untouched()
    assert bool((out[:start] == SENTINEL).all()) and bool((out[start + nnz:] == SENTINEL).all())
    terms = dY.double()[rows_of(lengths)] * X.double()[col.long()]
    want, size = alpha * terms.sum(1), abs(alpha) * terms.abs().sum(1)
    if beta:
        want += beta * d0.double()
        size += abs(beta) * d0.double().abs()
    within(out[start:start + nnz], want,
           UNIT[dtype] * want.abs() + (k + 4) * 2.0 ** -24 * size + TINY[dtype])


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("k", [1, 2, 3, 8, 31, 64, 257, 1000, 1531, 2048, 4100])
def test_sddmm_widths(pf, dtype, k):
    check_sddmm(pf, [3, 0, 1, 8, 2, 5, 0, 17], 29, k, dtype, seed=k)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("idx", [torch.int32, torch.int64])
@pytest.mark.parametrize("offset,padx,pady", [(0, 0, 0), (1, 0, 0), (0, 1, 0), (0, 0, 1),
                                              (2, 2, 4), (3, 5, 6), (8, 8, 16)])
def test_sddmm_alignment_strides_alpha_beta(pf, dtype, idx, offset, padx, pady):
    check_sddmm(pf, [4, 1, 0, 2, 9], 12, 200, dtype, -0.5, 1.5, idx, offset, padx, pady, seed=3)


@pytest.mark.parametrize("lengths", [[0], [1], [900], [1] * 3000, [0] * 40, [0, 300, 0, 7]])
@pytest.mark.parametrize("k", [40, 515])
def test_sddmm_row_lengths(pf, lengths, k):
    check_sddmm(pf, lengths, 1000, k, "bf16", seed=4, start=3)


def test_gradients_against_differences(pf):
    """Y is linear in the values: with f(a) = <dY, A(a) X>, the difference
    f(a + e) - f(a) is f(e) exactly, and <dval, e> has to equal it; likewise
    for X with the transposed matrix. Both sides carry their outputs' rounding."""
    dt, lengths, n, k = torch.float16, [3, 0, 2, 4], 9, 96
    g = torch.Generator().manual_seed(8)
    col = torch.randperm(9, generator=g).int()
    row = rows_of(lengths)
    val, X = torch.randn(9, generator=g).to(dt).cuda(), torch.randn(n, k, generator=g).to(dt).cuda()
    dY, E = (torch.randn(s, k, generator=g).to(dt).cuda() for s in (4, n))
    e = torch.randn(9, generator=g).to(dt).cuda()
    ptr, dcol = pointers(lengths), col.cuda()
    h = pf.Handle()
    dval, dX = torch.empty_like(val), torch.empty_like(X)
    pf.sddmm(h, 4, n, 9, ptr, dcol, dY, X, dval)
    to, gate = torch.empty(9, dtype=torch.int32), torch.empty(9, dtype=dt)
    to[col.long()], gate[col.long()] = row.int(), val.cpu()
    pf.spmm(h, n, 4, 9, pointers([1] * 9), to.cuda(), gate.cuda(), dY, dX)
    Ye, YE = torch.empty_like(dY), torch.empty_like(dY)
    pf.spmm(h, 4, n, 9, ptr, dcol, e, X, Ye)
    pf.spmm(h, 4, n, 9, ptr, dcol, val, E, YE)
    for Y, d, way in ((Ye, dval, e), (YE, dX, E)):
        a, b = dY.double() * Y.double(), d.double() * way.double()
        tol = 2 * UNIT["f16"] * (a.abs().sum() + b.abs().sum())
        within((a.sum() - b.sum())[None], torch.zeros(1), tol[None])
    h.close()


def test_no_columns(pf):
    """Rows of length 0: nothing to write for the product, dval = beta * dval."""
    h = pf.Handle()
    dt, dev = torch.bfloat16, "cuda"
    X, Y = torch.ones(5, 0, dtype=dt, device=dev), torch.zeros(3, 0, dtype=dt, device=dev)
    ptr, col = pointers([2, 0, 1]), torch.zeros(3, dtype=torch.int32, device=dev)
    d = torch.full((3,), 2.0, dtype=dt, device=dev)
    pf.spmm(h, 3, 5, 3, ptr, col, d, X, Y)
    pf.sddmm(h, 3, 5, 3, ptr, col, Y, X, d, beta=1.5)
    assert d.tolist() == [3.0, 3.0, 3.0] and h.device_error() == 0
    # the same through pointers that are not null: they are not read
    some = torch.zeros(64, dtype=dt, device=dev)
    p = some.data_ptr() + 2
    assert pf.lib.pf_sddmm_bf16_i32(h.ptr, 3, 5, 3, ptr.data_ptr(), col.data_ptr(), 0, 1.0, p, 0, p,
                                    0, 2.0, d.data_ptr(), None) == 0
    assert d.tolist() == [6.0, 6.0, 6.0] and h.device_error() == 0
    h.close()


def test_bad_columns_and_pointers_are_flagged(pf):
    h = pf.Handle()
    dt, dev = torch.bfloat16, "cuda"
    X, Y = torch.ones(5, 64, dtype=dt, device=dev), torch.zeros(3, 64, dtype=dt, device=dev)
    val = torch.ones(6, dtype=dt, device=dev)
    col = torch.tensor([0, 5, 1, -1, 2, 3], dtype=torch.int32, device=dev)
    pf.spmm(h, 3, 5, 6, pointers([2, 2, 2]), col, val, X, Y)
    assert h.device_error() == 2 and Y[:, 0].tolist() == [1.0, 1.0, 2.0]
    d = torch.full((6,), SENTINEL, dtype=dt, device=dev)
    pf.sddmm(h, 3, 5, 6, pointers([2, 2, 2]), col, Y, X, d)
    assert h.device_error() == 2
    assert d.float().tolist() == [64.0, float(torch.tensor(SENTINEL).to(dt)), 64.0,
                                  float(torch.tensor(SENTINEL).to(dt)), 128.0, 128.0]
    ptr = torch.tensor([0, 9, 4, 6], dtype=torch.int32, device=dev)
    good = torch.zeros(6, dtype=torch.int32, device=dev)
    pf.spmm(h, 3, 5, 6, ptr, good, val, X, Y)
    assert h.device_error() == 4 and Y[:, 0].tolist() == [0.0, 0.0, 2.0]
    pf.sddmm(h, 3, 5, 6, ptr, good, Y, X, d)
    assert h.device_error() == 4
    h.close()


def test_refusals(pf):
    h = pf.Handle()
    dt, dev = torch.bfloat16, "cuda"
    X, Y = torch.ones(5, 64, dtype=dt, device=dev), torch.zeros(3, 64, dtype=dt, device=dev)
    ptr, col = pointers([2, 2, 2]), torch.zeros(6, dtype=torch.int32, device=dev)
    val, d = torch.ones(6, dtype=dt, device=dev), torch.zeros(6, dtype=dt, device=dev)
    good = (h, 3, 5, 6, ptr, col, Y, X, d)
    pf.sddmm(*good)

    def refused(at, what):
        a = list(good)
        a[at] = what
        with pytest.raises(pf.PfError) as e:
            pf.sddmm(*a)
        assert e.value.status == 1

    refused(1, 4)
    refused(2, 6)
    refused(3, 7)
    refused(4, ptr.float())
    refused(5, col.long())
    refused(6, Y.half())
    refused(6, Y.t().contiguous().t())
    refused(7, X[:, :32])
    refused(7, X.cpu())
    refused(8, d.float())
    p = lambda t: t.data_ptr()  # noqa: E731
    args = [h.ptr, 3, 5, 6, p(ptr), p(col), 64, 1.0, p(Y), 64, p(X), 64, 0.0, p(d), None]
    for at, bad in ((0, None), (1, -1), (4, None), (5, None), (8, None), (9, 63), (10, p(X) + 1),
                    (13, None), (2, 0)):
        a = list(args)
        a[at] = bad
        assert pf.lib.pf_sddmm_bf16_i32(*a) == 1, at
    args = [h.ptr, 3, 5, 6, p(ptr), p(col), p(val), 64, 1.0, p(X), 64, 0.0, p(Y), 64, None]
    assert pf.lib.pf_spmm_bf16_i32(*args) == 0
    for at, bad in ((0, None), (1, -1), (4, None), (5, None), (6, None), (7, -1), (9, None),
                    (10, 63), (12, p(Y) + 1), (13, 63), (2, 0)):
        a = list(args)
        a[at] = bad
        assert pf.lib.pf_spmm_bf16_i32(*a) == 1, at
    assert h.device_error() == 0
    h.close()
