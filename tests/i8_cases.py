"""Shared by the tests of the 8-bit operators: matrices with a pitch, an offset and a guard behind them."""
import numpy as np
import torch

TORCH = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16, "int8": torch.int8}
HALF_STEP = {"fp32": 2.0 ** -24, "fp16": 2.0 ** -11, "bf16": 2.0 ** -8}     # finfo.eps / 2: relative error of one rounding
SMALLEST = {"fp32": 2.0 ** -149, "fp16": 2.0 ** -24, "bf16": 2.0 ** -133}   # spacing of the subnormal numbers
CODES = {"fp32": 0, "fp16": 1, "bf16": 2}


class Buffer:
    """[rows, cols] with row pitch `ld`, starting `offset` elements into an allocation that is filled with a known pattern: what
    lies before, between and behind the rows can be checked to be untouched."""

    def __init__(self, rows, cols, kind, ld=None, offset=0, values=None, device="cuda"):
        self.rows, self.cols, self.ld, self.offset = rows, cols, ld or max(cols, 1), offset
        count = offset + max(rows, 1) * self.ld + 64
        self.flat = torch.full((count,), 77, dtype=TORCH[kind], device=device)
        self.view = self.flat[offset:offset + rows * self.ld].view(rows, self.ld)[:, :cols]
        if values is not None:
            self.view.copy_(torch.as_tensor(np.ascontiguousarray(values)).to(device=device, dtype=TORCH[kind]))

    @property
    def address(self):
        return self.flat.data_ptr() + self.offset * self.flat.element_size()

    def numpy(self):
        v = self.view
        return (v.cpu() if v.dtype == torch.int8 else v.double().cpu()).numpy()

    def untouched(self):
        """Everything outside the matrix still holds the pattern."""
        mask = torch.ones_like(self.flat, dtype=torch.bool)
        mask[self.offset:self.offset + self.rows * self.ld].view(self.rows, self.ld)[:, :self.cols] = False
        return bool((self.flat[mask] == 77).all())


def activations(rng, rows, cols, kind, spread=1.0):
    """Normal values with a few large features and rows of different size, rounded to `kind`."""
    x = rng.standard_normal((rows, cols)) * np.exp(spread * rng.standard_normal((rows, 1)))
    x *= np.where(rng.random(cols) < 0.02, 15.0, 1.0)
    return torch.from_numpy(x).to(TORCH[kind]).double().numpy()


def check_rounded(got, want, kind, relative, what=""):
    """|got - want| within `relative` * |want| before the rounding plus half a step of `kind` for it (NaN where NaN is due)."""
    want = np.asarray(want, dtype=np.float64)
    assert np.array_equal(np.isnan(got), np.isnan(want)), what
    fine = np.isfinite(want)
    bound = (relative + HALF_STEP[kind] * (1 + relative)) * np.abs(want[fine]) + SMALLEST[kind]
    with np.errstate(invalid="ignore"):
        worst = np.max(np.abs(got[fine] - want[fine]) / bound) if fine.any() else 0.0
    assert worst <= 1.0, f"{what}: {worst} of the bound"
