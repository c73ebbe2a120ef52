"""8-bit rows on the device: quantize, restore and the norm with an 8-bit result, against the 64-bit definitions.

q has to equal the definition's integers.  Scales: max|x| is exact, so max|x| / 127 is one rounding (2^-24); a power of two
is exact.  The norm's scale has the rounding of P / 127, of the mean (a sum of K squares: each addition rounds to 2^-24 of a
partial sum that is no larger than the total; a thread adds at most 32 squares of a pass, then a pass's sum to the others', a warp 5 and a
block 5 more sums), of the product with 1 / K (2^-23) and the addition of eps, all halved by the root, then of rsqrtf (2 last places:
2^-22) and of the product: (32 + 16 passes + 10 + 3) / 2 + 4 + 2 times 2^-24, below the (50 + 16 passes) * 2^-24 the tests allow."""
import numpy as np
import pytest
import torch

from i8_cases import TORCH, Buffer, activations, check_rounded
from oracle import i8_model as model
from runner import api

pytestmark = pytest.mark.gpu

KINDS = ["fp32", "fp16", "bf16"]
# one element, less than a vector, vectors with a tail, whole warps, several vectors per thread, a block per row, rows read twice
LENGTHS = [1, 3, 8, 31, 64, 250, 256, 1001, 2048, 4100, 8192, 33000, 70001]


@pytest.fixture(scope="module")
def r(built):
    with api.SgemmRunner(*built.ensure(built.DEFAULT_I8)) as runner:
        yield runner


def quantize(r, x, kind, pow2, ld=None, ldq=None, offset=0, qoffset=0):
    rows, k = x.shape
    src = Buffer(rows, k, kind, ld, offset, x)
    q, s = Buffer(rows, k, "int8", ldq, qoffset), Buffer(1, rows, "fp32")
    r.i8_quantize(src.address, q.address, s.address, k, rows, pow2=pow2, ldx=src.ld, ldq=q.ld, x_type=KINDS.index(kind))
    torch.cuda.synchronize()
    assert q.untouched() and s.untouched() and src.untouched()
    return q.numpy(), s.numpy()[0]


def check_quantize(got, x, pow2):
    q, s = model.quantize(x, pow2)
    assert np.array_equal(got[0], q)
    check_rounded(got[1], s, "fp32", 0.0)
    if pow2:
        assert np.array_equal(got[1], s, equal_nan=True)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("pow2", [False, True])
@pytest.mark.parametrize("k", LENGTHS)
def test_quantize(r, kind, pow2, k):
    rows = 5 if k > 20000 else 37
    x = activations(np.random.default_rng(k), rows, k, kind)
    check_quantize(quantize(r, x, kind, pow2), x, pow2)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("k,ld,ldq,offset,qoffset", [(64, 80, 96, 0, 0), (100, 103, 101, 0, 0), (100, 104, 112, 3, 0), (1000, 1008, 1000, 8, 5),
                                                     (4096, 4099, 4112, 1, 16), (33, 64, 34, 0, 2)])
def test_quantize_pitches_and_unaligned_bases(r, kind, k, ld, ldq, offset, qoffset):
    x = activations(np.random.default_rng(ld), 19, k, kind)
    check_quantize(quantize(r, x, kind, False, ld, ldq, offset, qoffset), x, False)
    check_quantize(quantize(r, x, kind, True, ld, ldq, offset, qoffset), x, True)


@pytest.mark.parametrize("rows", [1, 2, 7, 8, 9, 300, 5000])
def test_quantize_row_counts(r, rows):
    x = activations(np.random.default_rng(rows), rows, 96, "bf16")
    check_quantize(quantize(r, x, "bf16", True), x, True)


@pytest.mark.parametrize("pow2", [False, True])
@pytest.mark.parametrize("kind", KINDS)
def test_quantize_halves_go_to_the_even_integer(r, kind, pow2):
    """A peak of 127 (times a power of two) makes every half-integer an exact tie; neighbours of ties one FP32 step away are not."""
    ties = np.concatenate([np.arange(-126.5, 127.0, 1.0), [127.0]])
    rows = [ties, ties * 2.0 ** -7, np.append(ties[:-1], -127.0)]
    if kind == "fp32":
        for toward in (-1e9, 1e9):
            rows.append(np.append(np.nextafter(ties[:-1].astype(np.float32), np.float32(toward)).astype(np.float64), 127.0))
        # a peak that is no multiple of 127: quotients as close to a half as FP32 values get
        peak = np.float32(1.2345678)
        near = ((np.arange(0, 127) + 0.5) * np.float64(peak) / 127.0).astype(np.float32)
        for step in (-1, 0, 1):
            v = near if step == 0 else np.nextafter(near, np.float32(step * 9))
            rows.append(np.concatenate([v.astype(np.float64), -v.astype(np.float64)])[:len(ties) - 1].tolist() + [float(peak)])
    x = np.array(rows)
    x = torch.from_numpy(x).to(TORCH[kind]).double().numpy()
    check_quantize(quantize(r, x, kind, pow2), x, pow2)


@pytest.mark.parametrize("pow2", [False, True])
def test_quantize_many_near_ties(r, pow2):
    """FP32 rows with few significant bits: thousands of exact and near ties against peaks of every size."""
    rng = np.random.default_rng(3)
    x = rng.integers(-255, 256, (400, 512)) * 2.0 ** rng.integers(-20, 20, (400, 1))
    x[:, 0] = 254 * 2.0 ** rng.integers(-20, 20, 400)
    x[::2] += x[::2] * 2.0 ** -23
    x = x.astype(np.float32).astype(np.float64)
    check_quantize(quantize(r, x, "fp32", pow2), x, pow2)


@pytest.mark.parametrize("pow2", [False, True])
@pytest.mark.parametrize("kind", ["fp32", "bf16"])
def test_quantize_zeros_infinities_nan_and_extremes(r, kind, pow2):
    big = 3.3895313892515355e38        # the largest bf16, beyond 127 * 2^121
    rows = np.zeros((10, 40))
    rows[1, 3] = np.nan
    rows[2, 39] = np.inf
    rows[3, 0] = -np.inf
    rows[4, 7] = big
    rows[5, :] = 127 * 2.0 ** 121      # the largest that is served
    rows[5, 5] = 1.0
    rows[6, 2] = 2.0 ** -130           # subnormal in FP32
    rows[7, :] = np.linspace(-1, 1, 40) * 2.0 ** -120
    rows[8, :] = 2.0 ** -133 * np.arange(40)
    rows[9, 11] = -0.0
    x = torch.from_numpy(rows).to(TORCH[kind]).double().numpy()
    got = quantize(r, x, kind, pow2)
    q, s = model.quantize(x, pow2)
    assert np.array_equal(got[0], q)
    assert np.array_equal(np.isnan(got[1]), np.isnan(s)) and np.isnan(got[1][1:5]).all()
    fine = ~np.isnan(s)
    assert np.all(np.abs(got[1][fine] - s[fine]) <= 2.0 ** -24 * s[fine] + 2.0 ** -149)
    out = Buffer(10, 40, "fp32")
    qb, sb = Buffer(10, 40, "int8", values=got[0]), Buffer(1, 10, "fp32", values=got[1][None])
    r.i8_restore(qb.address, sb.address, out.address, 40, 10, out_type=0)
    assert np.isnan(out.numpy()[1:5]).all() and np.isfinite(out.numpy()[5:]).all() and (out.numpy()[0] == 0).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,k,ldq,ldo,offset", [(1, 1, None, None, 0), (3, 16, None, None, 0), (37, 1001, 1008, None, 0), (5, 250, 256, 256, 0),
                                                   (64, 4096, None, None, 0), (9, 100, 101, 103, 1), (2, 70000, None, None, 0)])
def test_restore(r, kind, rows, k, ldq, ldo, offset):
    rng = np.random.default_rng(k)
    q = rng.integers(-128, 128, (rows, k)).astype(np.int8)
    s = np.exp(rng.standard_normal(rows)).astype(np.float32)
    s[0] = 0.0
    qb, sb, out = Buffer(rows, k, "int8", ldq, offset, q), Buffer(1, rows, "fp32", values=s[None]), Buffer(rows, k, kind, ldo, offset)
    r.i8_restore(qb.address, sb.address, out.address, k, rows, ldq=qb.ld, ldo=out.ld, out_type=KINDS.index(kind))
    torch.cuda.synchronize()
    assert out.untouched()
    # FP32 product (one rounding), then the rounding to the type: both restated in the same order
    assert np.array_equal(out.numpy(), model.restore(q, s, kind))


@pytest.mark.parametrize("kind", KINDS)
def test_power_of_two_checkpoint_round_trip(r, kind):
    """With power-of-two scales the restored value is s * q exactly, and at most half a scale from the input."""
    x = activations(np.random.default_rng(8), 64, 777, kind)
    q, s = quantize(r, x, kind, True)
    out = Buffer(64, 777, kind)
    qb, sb = Buffer(64, 777, "int8", values=q), Buffer(1, 64, "fp32", values=s[None])
    r.i8_restore(qb.address, sb.address, out.address, 777, 64, out_type=KINDS.index(kind))
    exact = q.astype(np.float64) * s[:, None]
    assert np.array_equal(out.numpy(), exact)
    assert np.all(np.abs(exact - x) <= 0.5 * s[:, None])
    peak = np.abs(x).max(1)
    assert np.all(127 * s >= peak) and np.all(127 * s / 2 < peak)


def rmsnorm(r, x, g, kind, residual=None, eps=1e-6, ld=None, ldq=None, offset=0, want_sum=True, inplace=None, roffset=None, goffset=0):
    rows, k = x.shape
    src, gb = Buffer(rows, k, kind, ld, offset, x), Buffer(1, k, kind, offset=goffset, values=g[None])
    res = Buffer(rows, k, kind, ld, offset if roffset is None else roffset, residual) if residual is not None else None
    total = {"x": src, "residual": res, None: Buffer(rows, k, kind, ld, offset) if want_sum else None}[inplace]
    q, s = Buffer(rows, k, "int8", ldq, offset), Buffer(1, rows, "fp32")
    r.i8_rmsnorm(src.address, gb.address, q.address, s.address, k, rows, residual=res.address if res else None,
                 sum_out=total.address if total else None, eps=eps, ldx=src.ld, ldr=src.ld, lds=src.ld, ldq=q.ld, x_type=KINDS.index(kind))
    torch.cuda.synchronize()
    assert q.untouched() and s.untouched() and src.untouched() and (total is None or total.untouched())
    return q.numpy(), s.numpy()[0], total.numpy() if total else None


def check_norm(got, x, g, kind, residual=None, eps=1e-6, passes=1):
    q, s, h = model.rmsnorm(x, g, eps, residual)
    assert np.array_equal(got[0], q)
    check_rounded(got[1], s, "fp32", (50 + 16 * passes) * 2.0 ** -24)
    if got[2] is not None:
        assert np.array_equal(got[2], model.round_to(h, kind), equal_nan=True)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("with_residual", [False, True])
@pytest.mark.parametrize("k", LENGTHS)
def test_rmsnorm(r, kind, with_residual, k):
    rng = np.random.default_rng(k + 1)
    rows = 3 if k > 20000 else 21
    x, g = activations(rng, rows, k, kind), activations(rng, 1, k, kind, 0.0)[0]
    res = activations(rng, rows, k, kind, 2.0) if with_residual else None
    check_norm(rmsnorm(r, x, g, kind, res), x, g, kind, res, passes=1 + k // 8192)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("inplace", ["x", "residual"])
@pytest.mark.parametrize("rows,k,ld,ldq,offset", [(4, 512, None, None, 0), (33, 1000, 1003, 1001, 5), (2, 40000, None, None, 0)])
def test_rmsnorm_sum_in_place_and_pitches(r, kind, inplace, rows, k, ld, ldq, offset):
    rng = np.random.default_rng(k)
    x, res = activations(rng, rows, k, kind), activations(rng, rows, k, kind)
    g = activations(rng, 1, k, kind, 0.0)[0]
    check_norm(rmsnorm(r, x, g, kind, res, ld=ld, ldq=ldq, offset=offset, inplace=inplace), x, g, kind, res, passes=1 + k // 8192)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("k,ld,ldq,offset,roffset,goffset", [(1000, 1001, 1000, 3, 3, 1), (1000, 1001, 1003, 3, 2, 0), (257, 257, 272, 0, 0, 5),
                                                             (9000, 9001, 9008, 1, 1, 0), (5, 7, 6, 2, 2, 0), (40, 41, 41, 7, 0, 3)])
def test_rmsnorm_rows_that_start_anywhere(r, kind, k, ld, ldq, offset, roffset, goffset):
    """Vectors shifted against the rows (all matrices alike) and rows that share no alignment at all."""
    rng = np.random.default_rng(k + ld)
    x, res = activations(rng, 23, k, kind), activations(rng, 23, k, kind)
    g = activations(rng, 1, k, kind, 0.0)[0]
    got = rmsnorm(r, x, g, kind, res, ld=ld, ldq=ldq, offset=offset, roffset=roffset, goffset=goffset)
    check_norm(got, x, g, kind, res, passes=1 + k // 8192)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("shift", range(8))
def test_quantize_and_restore_at_every_offset(r, kind, shift):
    """Rows of every start and several lengths within their 16-byte vectors, q at another offset."""
    for k in (1, 6, 17, 100, 1031):
        x = activations(np.random.default_rng(k), 13, k, kind)
        for pow2 in (False, True):
            got = quantize(r, x, kind, pow2, k + shift, k + 3, shift, 5)
            check_quantize(got, x, pow2)
        qb, sb, out = Buffer(13, k, "int8", k + 3, shift, got[0]), Buffer(1, 13, "fp32", values=got[1][None]), Buffer(13, k, kind, k + shift, 1)
        r.i8_restore(qb.address, sb.address, out.address, k, 13, ldq=qb.ld, ldo=out.ld, out_type=KINDS.index(kind))
        torch.cuda.synchronize()
        assert out.untouched() and np.array_equal(out.numpy(), model.restore(got[0], got[1], kind))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("eps", [0.0, 1e-6, 1e-2, 5.0])
def test_rmsnorm_eps_zero_rows_and_no_sum(r, kind, eps):
    rng = np.random.default_rng(5)
    x, g = activations(rng, 12, 300, kind), activations(rng, 1, 300, kind, 0.0)[0]
    g[::3] = 0.0
    if eps:
        x[4] = 0.0
    got = rmsnorm(r, x, g, kind, eps=eps, want_sum=False)
    check_norm(got, x, g, kind, eps=eps)
    if eps:
        assert got[1][4] == 0 and (got[0][4] == 0).all()


@pytest.mark.parametrize("kind", ["fp32", "bf16"])
def test_rmsnorm_rows_out_of_range(r, kind):
    rng = np.random.default_rng(6)
    x, g = activations(rng, 8, 200, kind), np.abs(activations(rng, 1, 200, kind, 0.0)[0]) + 0.5
    g = torch.from_numpy(g).to(TORCH[kind]).double().numpy()
    x[1, 7], x[2, 0], x[3, 199] = np.nan, np.inf, -np.inf
    x[4] *= 2.0 ** 90           # squares leave FP32, the norm does not
    x[5] *= 2.0 ** 120
    x = torch.from_numpy(x).to(TORCH[kind]).double().numpy()
    got = rmsnorm(r, x, g, kind)
    q, s, h = model.rmsnorm(x, g, 1e-6)
    assert np.array_equal(got[0], q) and np.isnan(got[1][1:4]).all() and np.isfinite(got[1][4:]).all()
    check_rounded(got[1], s, "fp32", 66 * 2.0 ** -24)


def test_same_bits_every_time_and_on_another_stream(r):
    rng = np.random.default_rng(9)
    x, res = activations(rng, 50, 5000, "bf16"), activations(rng, 50, 5000, "bf16")
    g = activations(rng, 1, 5000, "bf16", 0.0)[0]
    first = rmsnorm(r, x, g, "bf16", res)
    src, rb, gb = (Buffer(v.shape[0], 5000, "bf16", values=v) for v in (x, res, g[None]))
    q, s, total = Buffer(50, 5000, "int8"), Buffer(1, 50, "fp32"), Buffer(50, 5000, "bf16")
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    r.i8_rmsnorm(src.address, gb.address, q.address, s.address, 5000, 50, residual=rb.address, sum_out=total.address, x_type=2,
                 stream=side.cuda_stream)
    side.synchronize()
    assert np.array_equal(q.numpy(), first[0]) and np.array_equal(s.numpy()[0], first[1]) and np.array_equal(total.numpy(), first[2])
