"""The norm with an 8-bit result on rows whose squares, or whose mean square plus eps, leave FP32.

Bounds are those of the ordinary range (test_gpu_i8_rows.py): sums of squares scaled by a power of two round as the plain ones do
as long as they stay in the normal numbers, which for rows beyond FP32 they do: with a sum of plain squares above 2^128 over at most 2^17
elements, squares that matter to 2^-24 of it are above 2^(128 - 17 - 24) = 2^87.  Scaling by a power of two is exact."""
import numpy as np
import pytest
import torch

from i8_cases import TORCH, check_rounded
from oracle import i8_model as model
from test_gpu_i8_rows import check_norm, r, rmsnorm  # noqa: F401

pytestmark = pytest.mark.gpu

# how the rows lie, and with it the kernel: aligned vectors, vectors shifted against the rows, rows that share no alignment
FORMS = {"aligned": dict(pad=16, offset=0, roffset=0), "shifted": dict(pad=1, offset=3, roffset=3), "anyhow": dict(pad=1, offset=3, roffset=2)}


def rounded(x, kind):
    return torch.from_numpy(np.asarray(x, dtype=np.float64)).to(TORCH[kind]).double().numpy()


def call(runner, x, g, kind, eps, form, residual=True):
    k = x.shape[1]
    ld = (k + 15) // 16 * 16 + (FORMS[form]["pad"] if FORMS[form]["pad"] < 16 else 0)
    return rmsnorm(runner, x, g, kind, np.zeros_like(x) if residual else None, eps, ld=ld, ldq=(k + 15) // 16 * 16, offset=FORMS[form]["offset"],
                   roffset=FORMS[form]["roffset"])


@pytest.mark.parametrize("kind", ["fp32", "bf16"])
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("k", [1, 200, 4096, 70001])
def test_rows_of_any_magnitude_that_is_served(r, kind, form, k):   # noqa: F811
    """Every size from where squares begin to leave FP32 to the largest peak there is a scale for; gamma about 1, small (so that only the
    row itself is large), and large."""
    rng = np.random.default_rng(k)
    sizes = [50, 55, 58, 61, 63, 64, 65, 90, 112, 116, 120, 122, 125, 127]
    x = rounded(rng.choice([-1, 1], (len(sizes) + 2, k)) * rng.uniform(0.5, 0.99, (len(sizes) + 2, k)) * 2.0 ** np.array(sizes + [40, 0])[:, None], kind)
    x[-2:, k // 2] = 2.0 ** 126       # one element decides
    gamma = rounded(rng.uniform(0.5, 1.0, k), kind)
    for power in (0, -20, -120):
        g = gamma * 2.0 ** power
        got = call(r, x, g, kind, 1e-6, form)
        check_norm(got, x, g, kind, np.zeros_like(x), passes=1 + k // 8192)
        assert (got[1] > 0).all() or power == -120
    low = x[:7] * 2.0 ** -2
    g = gamma * 2.0 ** 60
    got = call(r, low, g, kind, 1e-6, form)
    check_norm(got, low, g, kind, np.zeros_like(low), passes=1 + k // 8192)


@pytest.mark.parametrize("kind", ["fp32", "bf16"])
@pytest.mark.parametrize("form", FORMS)
def test_large_eps_and_large_rows(r, kind, form):   # noqa: F811
    """The mean and eps are FP32 numbers and their sum is not; eps beside a mean beyond FP32's squares counts too."""
    rng = np.random.default_rng(1)
    x = rounded(rng.uniform(0.5, 0.99, (6, 512)) * 2.0 ** np.array([0, 62, 63, 64, 64, 70])[:, None], kind)
    g = rounded(rng.uniform(0.5, 1.0, 512), kind)
    for eps in (2.0 ** 120, 2.0 ** 127, float(np.float32(3e38))):
        check_norm(call(r, x, g, kind, eps, form), x, g, kind, np.zeros_like(x), eps=eps)


@pytest.mark.parametrize("kind", ["fp32", "bf16"])
def test_a_full_prompt_of_large_rows(r, kind):   # noqa: F811
    """Many rows: 32 elements a thread, and the scale of the definition, 1 / 127, for rows of one value."""
    x = np.full((2000, 4096), 2.0 ** 125)
    x[::2] *= -1
    got = rmsnorm(r, x, np.ones(4096), kind)
    assert (np.abs(got[0]) == 127).all()
    check_rounded(got[1], np.full(2000, 1.0 / 127.0), "fp32", 66 * 2.0 ** -24)
    assert np.array_equal(got[2], model.round_to(x, kind))


# Rows whose squares vanish in FP32: exponents of their magnitudes.
SMALL = {"fp32": [0, -30, -44, -46, -60, -63, -70, -75, -80, -100], "bf16": [0, -30, -44, -46, -60, -63, -70, -75, -80, -100], "fp16": [0, -10, -14, -20, -22]}
EPS = [0.0, 2.0 ** -149, 2.0 ** -130, 2.0 ** -91, 2.0 ** -89, 1e-20, 1e-6]


def small_rows(k, kind, sizes):
    """Rows of zeros, of the given magnitudes, and (the third) one of a single number among zeros."""
    rng = np.random.default_rng(k)
    x = rounded(rng.choice([-1, 1], (len(sizes) + 1, k)) * rng.uniform(0.5, 0.99, (len(sizes) + 1, k)) * 2.0 ** np.array([0] + sizes)[:, None], kind)
    x[0] = 0.0
    x[2, 1:] = 0.0
    return x, rounded(rng.uniform(0.5, 1.0, k), kind)


@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("k", [1, 300, 4096, 40000])
@pytest.mark.parametrize("eps", EPS)
def test_small_rows_and_small_eps(r, kind, form, k, eps):   # noqa: F811
    """A row of zeros has scale 0 for every eps, one that is not has the definition's scale.  (Squares below the normal
    numbers are summed again from values times 2^92.  The root of K in place of 1 / K, one more product: within the bound, which had
    6 * 2^-24 to spare.)"""
    x, gamma = small_rows(k, kind, SMALL[kind])
    eps = float(np.float32(eps))
    for power in (0, -10):
        g = rounded(gamma * 2.0 ** power, kind)
        got = call(r, x, g, kind, eps, form)
        check_norm(got, x, g, kind, np.zeros_like(x), eps=eps, passes=1 + k // 8192)
        assert got[1][0] == 0 and (got[0][0] == 0).all()


@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
def test_a_padding_row_of_zeros_without_eps(r, kind):   # noqa: F811
    rng = np.random.default_rng(2)
    x = rounded(rng.standard_normal((12, 300)), kind)
    x[4] = 0.0
    g = rounded(rng.standard_normal(300), kind)
    got = rmsnorm(r, x, g, kind, eps=0.0, want_sum=False)
    check_norm(got, x, g, kind, eps=0.0)
    assert got[1][4] == 0 and (got[0][4] == 0).all()


@pytest.mark.parametrize("kind", ["fp32", "bf16"])
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("k", [1, 300, 4096, 40000])
@pytest.mark.parametrize("eps", EPS)
def test_peaks_whose_127th_is_below_the_normal_numbers(r, kind, form, k, eps):   # noqa: F811
    """Small rows, small gamma or both: the scale is one rounding away from the definition however small max |h * gamma| / 127 is."""
    x, gamma = small_rows(k, kind, [0, -10, -100, -110, -120, -126, -131] + [-140, -147] * (kind == "fp32"))
    eps = float(np.float32(eps))
    for power in (0, -30, -110, -120):
        g = rounded(gamma * 2.0 ** power, kind)
        got = call(r, x, g, kind, eps, form)
        check_norm(got, x, g, kind, np.zeros_like(x), eps=eps, passes=1 + k // 8192)
        assert got[1][0] == 0 and (got[0][0] == 0).all()
