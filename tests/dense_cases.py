"""Shared pieces of the tests of the operators with dense 16-bit arrays:
row-major tensors inside larger, sentinel-filled buffers, and rounding units."""
import torch

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
# unit roundoff of a value rounded to nearest, and half the smallest step near 0
UNIT = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f32": 2.0 ** -24}
TINY = {"bf16": 2.0 ** -126, "f16": 2.0 ** -25, "f32": 2.0 ** -126}
SENTINEL = 777.0  # exact in every type


class Buffer:
    """A rows x cols row-major view, `offset` elements into a buffer that holds
    SENTINEL everywhere else, with leading dimension cols + pad."""

    def __init__(self, rows, cols, dtype, offset=0, pad=0, data=None):
        self.ld = cols + pad
        self.flat = torch.full((offset + rows * self.ld + 64,), SENTINEL, dtype=dtype,
                               device="cuda")
        self.view = torch.as_strided(self.flat, (rows, cols), (self.ld, 1), offset)
        if data is not None:
            self.view.copy_(data)

    def outside_untouched(self):
        """Whether every element around the view still holds the sentinel."""
        keep = self.flat.clone()
        torch.as_strided(keep, self.view.shape, (self.ld, 1),
                         self.view.storage_offset()).fill_(SENTINEL)
        return bool((keep == SENTINEL).all())


def pointers(lengths, start=0, dtype=torch.int32):
    p = torch.zeros(len(lengths) + 1, dtype=torch.int64)
    p[1:] = torch.tensor(lengths, dtype=torch.int64).cumsum(0)
    return (p + start).to(dtype).cuda()


def within(got, want, tol):
    """got and want agree to tol, infinities and NaN in the same places."""
    got, want, tol = got.double().cpu(), want.double().cpu(), tol.double().cpu()
    special = ~torch.isfinite(want)
    same = (got == want) | (got.isnan() & want.isnan())
    assert bool(same[special].all()), "infinities or NaN differ"
    err = (got - want).abs()
    bad = ~special & ~(err <= tol)
    if bool(bad.any()):
        i = int(torch.where(bad.flatten(), (err / tol).flatten(), -1.0).argmax())
        raise AssertionError(f"{int(bad.sum())} values out of tolerance, worst at {i}: "
                             f"{float(got.flatten()[i])!r} for {float(want.flatten()[i])!r}, "
                             f"tolerance {float(tol.flatten()[i]):.3g}")
