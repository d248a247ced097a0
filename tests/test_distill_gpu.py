"""Distillation from a teacher's kept logits (pf_distill_*), through the C ABI,
against the formulas in 64 bits on the CPU.

Tolerances. Each softmax sum is of fp32 exponentials, each within 2^-21 of its
value (two units of the exponential, and the argument's rounding), added in
chains of at most a few hundred terms of 2^-24 each: EPS = 2e-5 bounds a sum's,
a probability's and a logarithm's error. The loss adds two logarithms and
sum p (t - z) / tau; the gradient is w / tau (q - p), rounded to its type.
"""
import math

import pytest
import torch

from dense_cases import DT, TINY, UNIT, Buffer, pointers, within

pytestmark = pytest.mark.gpu
EPS = 2e-5


def formulas(lengths, col, val, z, weight, tau):
    """loss, dz and their tolerances' parts, in 64 bits on the CPU."""
    m, n = z.shape
    z, val = z.double().cpu(), val.double().cpu()
    w = torch.ones(m, dtype=torch.float64) if weight is None else weight.double().cpu()
    col = col.long().cpu()
    loss = torch.zeros(m, dtype=torch.float64)
    dz = torch.zeros(m, n, dtype=torch.float64)
    loss_part = torch.zeros(m, dtype=torch.float64)
    dz_part = torch.zeros(m, n, dtype=torch.float64)
    at = 0
    for r, count in enumerate(lengths):
        c, t = col[at:at + count], val[at:at + count] / tau
        at += count
        ok = (c >= 0) & (c < n)
        c, t = c[ok], t[ok]
        if float(w[r]) == 0.0 or not bool((t != -math.inf).any()):
            continue
        p = torch.softmax(t, 0)
        if bool((z[r] == -math.inf).all()):
            q = torch.zeros(n, dtype=torch.float64)
            loss[r] = w[r] * math.inf
        else:
            lz = torch.logsumexp(z[r] / tau, 0)
            q = torch.exp(z[r] / tau - lz)
            lq = z[r][c] / tau - lz
            lp = t - torch.logsumexp(t, 0)
            use = p != 0
            loss[r] = w[r] * (p[use] * (lp - lq)[use]).sum()
            loss_part[r] = abs(w[r]) * (2 + (p[use] * (t - z[r][c] / tau)[use].abs()).sum())
        pc = torch.zeros(n, dtype=torch.float64).index_add_(0, c, p)
        dz[r] = w[r] / tau * (q - pc)
        dz_part[r] = (w[r] / tau).abs() * (q + pc)
    return loss, dz, loss_part.nan_to_num(0, 0), dz_part.nan_to_num(0, 0)


def run(pf, lengths, col, val, z, dtype, weight=None, tau=1.0, idx=torch.int32, start=0,
        offset=0, pad=0, want=("loss", "dz"), in_place=False, pad_out=None):
    dt = DT[dtype]
    m, n = z.shape
    nnz = sum(lengths)
    ptr = pointers(lengths, start, idx)
    fill = torch.zeros(start, dtype=torch.int32)
    dcol = torch.cat([fill, col.to(torch.int32).cpu()]).cuda()
    dval = torch.cat([fill.to(dt), val.to(dt).cpu()]).cuda()
    zb = Buffer(m, n, dt, offset, pad, z)
    ob = zb if in_place else Buffer(m, n, dt, offset, pad if pad_out is None else pad_out)
    loss = torch.full((m,), math.nan, device="cuda") if "loss" in want else None
    wt = None if weight is None else weight.cuda()
    h = pf.Handle()
    # the C entry takes nnz of the slice; the wrapper checks the whole arrays
    pf.distill(h, m, n, nnz, ptr, dcol, dval, zb.view, loss, ob.view if "dz" in want else None,
               wt, tau)
    torch.cuda.synchronize()
    bits = h.device_error()
    h.close()
    assert zb.outside_untouched() and ob.outside_untouched()
    return loss, ob.view if "dz" in want else None, bits


def check(pf, lengths, col, val, z, dtype, weight=None, tau=1.0, bits=0, **kw):
    dt = DT[dtype]
    z, val = z.to(dt), val.to(dt)
    loss, dz, err = run(pf, lengths, col, val, z, dtype, weight, tau, **kw)
    assert err == bits
    rl, rd, pl, pd = formulas(lengths, col, val, z, weight, tau)
    if loss is not None:
        within(loss, rl, EPS * pl + 2.0 ** -23 * rl.abs().nan_to_num(0, 0, 0) + 1e-37)
    if dz is not None:
        within(dz, rd, UNIT[dtype] * rd.abs().nan_to_num(0) + EPS * pd + TINY[dtype])
    return loss, dz


def inputs(m, n, lengths, seed, distinct=True):
    g = torch.Generator().manual_seed(seed)
    z = 3.0 * torch.randn(m, n, generator=g)
    cols = [torch.randperm(n, generator=g)[:c] if distinct else
            torch.randint(0, n, (c,), generator=g) for c in lengths]
    col = torch.cat(cols) if cols else torch.zeros(0, dtype=torch.int64)
    val = 4.0 + 3.0 * torch.randn(sum(lengths), generator=g)
    return col, val, z


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("n", [1, 2, 7, 33, 1000, 4099, 16385, 40001])
def test_sizes(pf, dtype, n):
    lengths = [min(n, k) for k in (5, 0, 1, 40, 3)]
    col, val, z = inputs(5, n, lengths, n)
    check(pf, lengths, col, val, z, dtype, tau=1.5)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("n", [65537, 131072, 131073, 300001])
def test_large_vocabularies(pf, dtype, n):
    lengths = [64, 3]
    col, val, z = inputs(2, n, lengths, n)
    check(pf, lengths, col, val, z, dtype)
    check(pf, lengths, col, val, z, dtype, in_place=True)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("idx", [torch.int32, torch.int64])
@pytest.mark.parametrize("offset,pad,pad_out", [(0, 0, 0), (1, 0, 0), (3, 5, 5), (0, 8, 3),
                                                (5, 1, 0)])
def test_alignment_strides_types(pf, dtype, idx, offset, pad, pad_out):
    lengths = [3, 17, 0, 9, 33, 1, 64]
    col, val, z = inputs(7, 777, lengths, 5)
    w = torch.tensor([0.5, 1.0, 2.0, 0.0, -1.0, 0.25, 3.0])
    check(pf, lengths, col, val, z, dtype, w, 0.7, idx=idx, offset=offset, pad=pad,
          pad_out=pad_out)


@pytest.mark.parametrize("want", [("loss",), ("dz",)])
@pytest.mark.parametrize("rows", [1, 2, 40, 700])
def test_one_output_alone(pf, want, rows):
    lengths = [(7 * r) % 23 for r in range(rows)]
    col, val, z = inputs(rows, 2050, lengths, rows)
    check(pf, lengths, col, val, z, "bf16", tau=2.0, want=want)


@pytest.mark.parametrize("n", [100, 5000, 40001])
def test_in_place_equals_out_of_place(pf, n):
    lengths = [60, 2, 0, 31]
    col, val, z = inputs(4, n, lengths, n)
    l0, d0 = check(pf, lengths, col, val, z, "bf16")
    l1, d1 = check(pf, lengths, col, val, z, "bf16", in_place=True)
    assert torch.equal(l0, l1) and torch.equal(d0, d1)


def test_no_rows_and_no_entries(pf):
    col, val, z = inputs(3, 50, [0, 0, 0], 1)
    loss, dz = check(pf, [0, 0, 0], col, val, z, "bf16")
    assert float(loss.abs().sum()) == 0.0 and float(dz.abs().sum()) == 0.0
    h = pf.Handle()
    empty = torch.zeros(0, 50, dtype=torch.bfloat16, device="cuda")
    pf.distill(h, 0, 50, 0, pointers([]), torch.zeros(0, dtype=torch.int32, device="cuda"),
               torch.zeros(0, dtype=torch.bfloat16, device="cuda"), empty,
               torch.zeros(0, device="cuda"))
    assert h.device_error() == 0


def test_no_columns(pf):
    """A vocabulary of nothing: losses of 0, and no read through any pointer."""
    h = pf.Handle()
    loss = torch.full((3,), math.nan, device="cuda")
    ptr, some = pointers([0, 0, 0]), torch.zeros(8, device="cuda")
    f = pf.lib.pf_distill_f32_i32
    for z in (None, some.data_ptr() + 4):
        assert f(h.ptr, 3, 0, 0, ptr.data_ptr(), None, None, 1.0, z, 5, None, loss.data_ptr(), None,
                 0, None) == 0
        torch.cuda.synchronize()
        assert loss.tolist() == [0.0, 0.0, 0.0]
        loss.fill_(math.nan)
    assert h.device_error() == 0
    h.close()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_no_columns_many_rows(pf, dtype):
    """Far more rows than clusters, so that each would take hundreds."""
    m = 200000
    z = torch.empty(m, 0, dtype=DT[dtype], device="cuda")
    loss, w = torch.full((m,), math.nan, device="cuda"), torch.rand(m, device="cuda")
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    h = pf.Handle()
    for weight, dz in ((None, None), (w, None), (w, torch.empty_like(z))):
        loss.fill_(math.nan)
        pf.distill(h, m, 0, 0, torch.zeros(m + 1, dtype=torch.int32, device="cuda"), none,
                   none.to(z.dtype), z, loss, dz, weight)
        assert bool((loss == 0).all()) and h.device_error() == 0
    h.close()


@pytest.mark.parametrize("keep", [64, 65, 200])
@pytest.mark.parametrize("n", [700, 20000])
def test_kept_around_the_listed_number(pf, keep, n):
    """Rows of up to 64 entries are listed by one warp, longer ones are not;
    repeated columns in both, beside rows of weight 0 and rows without entries."""
    lengths = [keep, 0, keep, 3, keep]
    col, val, z = inputs(5, n, lengths, keep, distinct=False)
    col[1] = col[0]
    col[keep - 1] = col[0]
    col[keep + 40] = col[keep + 2]
    w = torch.tensor([1.0, 1.0, 0.0, 2.0, -0.5])
    check(pf, lengths, col, val, z, "f32", w)
    check(pf, lengths, col, val, z, "bf16", w, in_place=True)


@pytest.mark.parametrize("rows", [300, 2500])
def test_more_rows_than_clusters(pf, rows):
    """Every cluster takes several rows, some of weight 0, some empty."""
    g = torch.Generator().manual_seed(rows)
    lengths = torch.randint(0, 70, (rows,), generator=g).tolist()
    col, val, z = inputs(rows, 1025, lengths, rows)
    w = torch.rand(rows, generator=g)
    w[::7] = 0.0
    check(pf, lengths, col, val, z, "f16", w, 1.1)
    check(pf, lengths, col, val, z, "f16", w, 1.1, want=("loss",))


@pytest.mark.parametrize("n,rows", [(150, 30000), (5000, 3000)])
def test_long_rows_among_many_short_ones(pf, n, rows):
    """Clusters take tens of rows each, of which now and then one has more
    entries than are listed: the first such row of a cluster can be any of them.
    The rows repeat a few, so that 64-bit results are computed for those alone."""
    kinds = 53
    lengths = [100 if r % 17 == 5 else r % 4 for r in range(kinds)]
    col, val, z = inputs(kinds, n, lengths, n)
    w = torch.ones(kinds)
    w[7] = 0.0
    z, val = z.bfloat16(), val.bfloat16()
    rl, rd, pl, pd = formulas(lengths, col, val, z, w, 1.0)
    start = [0]
    for c in lengths:
        start.append(start[-1] + c)
    kind = torch.randint(0, kinds, (rows,), generator=torch.Generator().manual_seed(rows))
    at = torch.cat([torch.arange(start[k], start[k + 1]) for k in kind.tolist()])
    loss, dz, err = run(pf, [lengths[k] for k in kind.tolist()], col[at], val[at], z[kind], "bf16",
                        w[kind])
    assert err == 0
    within(loss, rl[kind], (EPS * pl + 2.0 ** -23 * rl.abs() + 1e-37)[kind])
    within(dz, rd[kind], (UNIT["bf16"] * rd.abs() + EPS * pd + TINY["bf16"])[kind])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("n", [64, 9000])
def test_infinities_and_masks(pf, dtype, n):
    """-inf and the type's lowest value among the student's logits, -inf teacher
    logits on them, rows with nothing left on either side, +inf and NaN."""
    lengths = [4] * 8
    col, val, z = inputs(8, n, lengths, 3)
    c = col.view(8, 4)
    v = val.view(8, 4)
    low = float(torch.finfo(DT[dtype]).min)
    z[0, :] = -math.inf                       # nothing left, and teacher mass: loss inf
    z[1, : n // 2] = -math.inf                # masked half, teacher on live columns
    c[1] = torch.arange(n - 4, n)
    z[2, 1:] = low
    c[2] = torch.tensor([0, 1, 2, 3])
    v[3, 1:] = -math.inf                      # one teacher logit left
    z[3, c[3, 1:]] = -math.inf                # p = 0 where q = 0: adds nothing
    v[4, :] = -math.inf                       # no teacher mass
    z[5, c[5, 0]] = -math.inf                 # p > 0 where q = 0: loss inf
    z[6, 5] = math.nan
    z[7, :] = -math.inf                       # nothing on either side
    v[7, :] = -math.inf
    loss, dz = check(pf, lengths, col, val, z, dtype)
    assert loss[0] == math.inf and loss[5] == math.inf and loss[4] == 0 and loss[7] == 0
    assert bool(loss[6].isnan()) and bool(dz[6].isnan().all())
    assert float(dz[4].abs().sum()) == 0.0


@pytest.mark.parametrize("dtype,sizes", [
    ("bf16", (1e6, 1e8, 3e9, 1e10, 1e12, 1e15, 1e20, 1e30)),
    ("f32", (1e6, 1e8, 3e9, 1e10, 1e12, 1e15, 1e20, 1e30)), ("f16", (6e4,) * 8)])
@pytest.mark.parametrize("tau", [0.1, 1.0, 2.0])
@pytest.mark.parametrize("kind", ["half", "most", "high"])
@pytest.mark.parametrize("n", [700, 40001, 300001])
def test_finite_masks_of_any_size(pf, dtype, sizes, tau, kind, n):
    """Finite logits far below all others, as masks are written, on half of the
    columns or on all but five (threads, and CTAs of a row that several take,
    hold nothing else), and one logit far above: their exponentials are 0, so
    the results are those of -inf there, bit for bit. (f16 has no such values:
    there the temperature is low.)"""
    if dtype == "f16":
        tau *= 1e-5
    lengths = [4] * 8
    col, val, z = inputs(8, n, lengths, 21)
    val, z, c = val.to(DT[dtype]), z.to(DT[dtype]), col.view(8, 4)
    same = z.clone()
    for r, size in enumerate(sizes):
        if kind == "high":
            same[r, :] = -math.inf
            z[r, 3] = same[r, 3] = size
            c[r] = torch.tensor([3, 5, 1, n - 1])
        else:
            first = n // 2 if kind == "half" else n - 5
            z[r, :first], same[r, :first] = -size, -math.inf
            c[r] = torch.arange(n - 4, n)
    w = torch.full((8,), tau)
    loss, dz, err = run(pf, lengths, col, val, z, dtype, w, tau)
    want_loss, want, _ = run(pf, lengths, col, val, same, dtype, w, tau)
    assert err == 0 and torch.equal(dz, want) and bool(dz.isfinite().all())
    assert bool(loss.isfinite().all())
    if kind != "high":
        assert torch.equal(loss, want_loss)
    alone, _, _ = run(pf, lengths, col, val, z, dtype, w, tau, want=("loss",))
    assert torch.equal(alone, loss)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("n", [700, 40001, 300001])
def test_rows_of_one_large_value(pf, dtype, n):
    """Every logit of a row the same finite mask, up to the size at which the
    formulas in 64 bits still tell log n from 0."""
    col, val, z = inputs(8, n, [4] * 8, 22)
    for r, size in enumerate((1e6, 1e7, 3e7, 1e8, 1e9, 3e9, 6e9, 1e10)):
        z[r, :] = -size
    check(pf, [4] * 8, col, val, z, dtype)
    check(pf, [4] * 8, col, val, z, dtype, want=("loss",))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("tau", [0.7, 2.0])
@pytest.mark.parametrize("side", ["student", "teacher", "both"])
@pytest.mark.parametrize("n,keep", [(64, 4), (700, 64), (700, 200), (40001, 64), (300001, 300)])
def test_only_differences_count(pf, dtype, tau, side, n, keep):
    """Rows far from 0: rows of one large finite value (nothing left by a mask),
    and rows of multiples of a step, large enough that they are exact, moved by
    a multiple of it. Loss and gradient are those of the rows moved back, where
    the formulas are evaluated. The loss's error: EPS of the two logarithms and
    of the sums of p (max z - z) and p (max t - t) over tau, which do not change
    with the move."""
    steps = [0.0] * 4 + [2.0 ** -4, 2.0 ** -2, 2.0 ** 7, 2.0 ** 7]
    moves = [1e6, 1e10, 1e20, 3e38, 2.0 ** 3, 2.0 ** 5, 2.0 ** 14, -2.0 ** 14]
    g = torch.Generator().manual_seed(n + keep)
    lengths = [keep] * 8
    col = torch.cat([torch.randperm(n, generator=g)[:keep] for _ in lengths])
    z = torch.randint(-12, 13, (8, n), generator=g) * torch.tensor(steps)[:, None]
    t = torch.randint(-12, 13, (8, keep), generator=g) * torch.tensor(steps)[:, None]
    move = torch.tensor(moves)[:, None]
    move[:4] = -move[:4]
    zm, tm = (z - move, t) if side == "student" else (z, t - move) if side == "teacher" else \
        (z - move, t - move)
    zm, tm = zm.to(DT[dtype]), tm.to(DT[dtype])
    for moved, still, by in ((zm, z, side != "teacher"), (tm, t, side != "student")):
        back = moved[4:].double() + (move[4:].double() if by else 0.0)
        assert torch.equal(back, still[4:].double())  # nothing was rounded
    loss, dz, err = run(pf, lengths, col, tm.flatten(), zm, dtype, None, tau)
    rl, rd, _, pd = formulas(lengths, col, t.flatten(), z, None, tau)
    p = torch.softmax(t.double() / tau, 1)
    far = (p * (z.double().amax(1, keepdim=True) - z.double().gather(1, col.view(8, keep)))).sum(1) + \
        (p * (t.double().amax(1, keepdim=True) - t.double())).sum(1)
    assert err == 0
    within(loss, rl, EPS * (2 + far / tau) + 2.0 ** -23 * rl.abs())
    within(dz, rd, UNIT[dtype] * rd.abs() + EPS * pd + TINY[dtype])
    alone, _, _ = run(pf, lengths, col, tm.flatten(), zm, dtype, None, tau, want=("loss",))
    assert torch.equal(alone, loss)


def test_plus_infinity_is_nan(pf):
    col, val, z = inputs(2, 300, [3, 3], 4)
    z[0, 7] = math.inf
    val[4] = math.inf
    loss, dz, err = run(pf, [3, 3], col, val, z, "f32")
    assert err == 0 and bool(loss.isnan().all()) and bool(dz[0].isnan().any())


def test_extreme_logits_do_not_overflow(pf):
    """Logits of +-60000 at a low temperature: only differences count."""
    col, val, z = inputs(3, 500, [5, 5, 5], 6)
    z[0] += 60000.0
    z[1] -= 60000.0
    val[:5] += 60000.0
    val[5:10] -= 60000.0
    z[2] *= 1000.0
    check(pf, [5, 5, 5], col, val, z, "f32", tau=0.7)


def test_repeated_columns_add_up(pf):
    lengths = [50, 7, 200]
    col, val, z = inputs(3, 20, lengths, 7, distinct=False)
    l0, d0 = check(pf, lengths, col, val, z, "f32")
    l1, d1 = check(pf, lengths, col, val, z, "f32")
    assert torch.equal(l0, l1) and torch.equal(d0, d1)


@pytest.mark.parametrize("n", [3000, 20000])
def test_dense_teacher(pf, n):
    """Every column kept: the full divergence; equal logits give loss and gradient 0."""
    col, val, z = inputs(2, n, [n, n], 8)
    check(pf, [n, n], col, val, z, "f32", tau=3.0)
    c = col.view(2, n)
    val = z.gather(1, c).flatten()
    loss, dz, _ = run(pf, [n, n], col, val, z, "f32")
    assert float(loss.abs().max()) <= 2 * EPS and float(dz.abs().max()) <= EPS


def test_weight_zero_rows_are_not_read(pf):
    lengths = [4, 4, 4]
    col, val, z = inputs(3, 700, lengths, 9)
    z[1, :] = math.nan
    w = torch.tensor([1.0, 0.0, 2.0])
    loss, dz = check(pf, lengths, col, val, z, "f32", w)
    assert float(loss[1]) == 0.0 and float(dz[1].abs().sum()) == 0.0


def test_slice_of_a_larger_matrix(pf):
    """row_ptr[0] > 0: col and val are addressed with absolute positions."""
    lengths = [3, 0, 8, 5]
    col, val, z = inputs(4, 90, lengths, 10)
    check(pf, lengths, col, val, z, "f16", start=11)


def test_bad_columns_and_pointers_are_flagged(pf):
    lengths = [3, 2, 4]
    col, val, z = inputs(3, 60, lengths, 11)
    col[1], col[4], col[6] = 60, -1, 2 ** 31 - 1
    check(pf, lengths, col, val, z, "f32", bits=2)
    h = pf.Handle()
    ptr = torch.tensor([0, 5, 3, 9], dtype=torch.int32, device="cuda")  # row 1 decreases
    loss = torch.empty(3, device="cuda")
    pf.distill(h, 3, 60, 9, ptr, torch.zeros(9, dtype=torch.int32, device="cuda"),
               val.cuda(), z.cuda(), loss)
    assert h.device_error() == 4 and float(loss[1]) == 0.0
    h.close()


def test_gradient_against_differences(pf):
    """The loss along a direction against the gradient. Central differences of
    step h: the fp32 losses' errors over 2h, and h^2 / 6 times a third
    derivative of at most 1 / tau^3 (the direction's entries are +-1)."""
    g = torch.Generator().manual_seed(12)
    lengths = [6] * 16
    col, val, z = inputs(16, 200, lengths, 13)
    tau, h = 1.3, 0.05
    w = torch.rand(16, generator=g) + 0.5
    d = torch.randint(0, 2, (16, 200), generator=g) * 2.0 - 1.0
    _, dz, _ = run(pf, lengths, col, val, z, "f32", w, tau)
    up, _, _ = run(pf, lengths, col, val, z + h * d, "f32", w, tau)
    down, _, _ = run(pf, lengths, col, val, z - h * d, "f32", w, tau)
    _, _, part, _ = formulas(lengths, col, val, z + h * d, w, tau)
    slope = (up.double() - down.double()).cpu() / (2 * h)
    within(slope, (dz.double().cpu() * d).sum(1),
           (EPS * part + 2.0 ** -22 * up.double().abs().cpu()) / h + w * h * h / 6 / tau ** 3 + 1e-4)


def test_backward_call_of_its_own(pf):
    """loss = None with the upstream gradient in the weights: the fused gradient scaled."""
    lengths = [5, 9, 0, 2]
    col, val, z = inputs(4, 1234, lengths, 14)
    up = torch.tensor([0.5, -2.0, 1.0, 4.0])
    _, d1, _ = run(pf, lengths, col, val, z, "f32", up, 1.0, want=("dz",))
    _, d2, _ = run(pf, lengths, col, val, z, "f32", None, 1.0)
    assert torch.equal(d1, d2 * up[:, None].cuda())


def test_another_stream_and_capture(pf):
    lengths = [8] * 32
    col, val, z = inputs(32, 3001, lengths, 15)
    l0, d0, _ = run(pf, lengths, col, val, z, "bf16")
    ptr, dcol, dval = pointers(lengths), col.int().cuda(), val.to(torch.bfloat16).cuda()
    zz = z.to(torch.bfloat16).cuda()
    loss, dz = torch.zeros(32, device="cuda"), torch.zeros_like(zz)
    h = pf.Handle()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        pf.distill(h, 32, 3001, 256, ptr, dcol, dval, zz, loss, dz)
    side.synchronize()
    assert torch.equal(loss, l0) and torch.equal(dz, d0)
    loss.zero_()
    with torch.cuda.graph(graph, stream=side):
        pf.distill(h, 32, 3001, 256, ptr, dcol, dval, zz, loss, dz)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(loss, l0)
    h.close()


@pytest.mark.parametrize("n", [333, 40001])
def test_a_replay_writes_loss_and_gradient(pf, n):
    """A captured call writes both outputs anew at every replay, from the inputs
    of that time, and flags nothing."""
    lengths = [8, 0, 70, 1]
    col, val, z = inputs(4, n, lengths, 16)
    want = [run(pf, lengths, col, val, x, "bf16")[:2] for x in (z, -z)]
    ptr, dcol, dval = pointers(lengths), col.int().cuda(), val.to(torch.bfloat16).cuda()
    zz = z.to(torch.bfloat16).cuda()
    loss, dz = torch.zeros(4, device="cuda"), torch.zeros_like(zz)
    h, graph = pf.Handle(), torch.cuda.CUDAGraph()
    pf.distill(h, 4, n, 79, ptr, dcol, dval, zz, loss, dz)
    with torch.cuda.graph(graph):
        pf.distill(h, 4, n, 79, ptr, dcol, dval, zz, loss, dz)
    for x, (l, d) in zip((z, -z), want):
        zz.copy_(x)
        loss.fill_(math.nan)
        dz.fill_(math.nan)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(loss, l) and torch.equal(dz, d) and h.device_error() == 0
    del graph
    h.close()


def test_refusals(pf):
    h = pf.Handle()
    ptr = pointers([2, 2])
    col = torch.zeros(4, dtype=torch.int32, device="cuda")
    z = torch.zeros(2, 10, dtype=torch.bfloat16, device="cuda")
    val = torch.zeros(4, dtype=torch.bfloat16, device="cuda")
    loss = torch.zeros(2, device="cuda")
    good = (h, 2, 10, 4, ptr, col, val, z)
    pf.distill(*good, loss)

    def refused(*a, **kw):
        with pytest.raises(pf.PfError) as e:
            pf.distill(*a, **kw)
        assert e.value.status == 1

    refused(*good)                                              # nothing asked for
    refused(*good, loss, temperature=0.0)
    refused(*good, loss, temperature=-1.0)
    refused(*good, loss, temperature=math.nan)
    refused(*good, loss.double())
    refused(*good, loss, z.float())
    refused(*good, loss, weight=torch.zeros(3, device="cuda"))
    refused(h, 2, 10, 4, ptr, col, val.float(), z, loss)
    refused(h, 2, 10, 5, ptr, col, val, z, loss)                # fewer entries than nnz
    refused(h, 3, 10, 4, ptr, col, val, z, loss)
    refused(h, 2, 10, 4, ptr.float(), col, val, z, loss)
    refused(h, 2, 10, 4, ptr, col.long(), val, z, loss)
    refused(h, 2, 10, 4, ptr, col, val, z.t().contiguous().t(), loss)
    refused(h, 2, 10, 4, ptr.cpu(), col, val, z, loss)
    refused(h, 2, 10, 4, ptr, col, val, z.cpu(), loss)
    lib = pf.lib
    p = lambda t: t.data_ptr()  # noqa: E731
    f = lib.pf_distill_bf16_i32
    args = [h.ptr, 2, 10, 4, p(ptr), p(col), p(val), 1.0, p(z), 10, None, p(loss), None, 0, None]
    for at, bad in ((0, None), (1, -1), (4, None), (5, None), (8, None), (9, 9), (8, p(z) + 1),
                    (11, p(loss) + 2)):
        a = list(args)
        a[at] = bad
        assert f(*a) == 1, at
    a = list(args)
    a[12], a[13] = p(z), 12                                     # in place, other stride
    assert f(*a) == 1
    assert h.device_error() == 0
    h.close()
