"""The 8-bit linear layer on the device against the 64-bit definition.

The integer sum is exact.  Its conversion to FP32, the product with x_scale and the fused product with w_scale plus bias
round once each: (acc * sx) * sw has 3 roundings of 2^-24, and adding the bias rounds the total (the third rounding is the
fused one), so |y - exact| <= 2.01 * 2^-24 |acc sx sw| + 2^-24 |y| before the last rounding to Y's type."""
import numpy as np
import pytest
import torch

from i8_cases import CODES, HALF_STEP, SMALLEST, Buffer
from oracle import i8_model as model
from runner import api

pytestmark = pytest.mark.gpu

KINDS = ["fp32", "fp16", "bf16"]
AUTO, MAIN, SIMT, FEW, HALF = 0, 1, 2, 3, 4


@pytest.fixture(scope="module")
def runner(built):
    with api.SgemmRunner(*built.ensure(built.DEFAULT_I8)) as r:
        yield r


@pytest.fixture
def r(runner):
    runner.set_option("force_variant", AUTO)
    runner.set_option("split_k", 0)
    yield runner
    runner.set_option("force_variant", AUTO)
    runner.set_option("split_k", 0)


def problem(m, n, k, seed=0, extreme=False):
    rng = np.random.default_rng(seed)
    pick = (lambda *s: rng.choice(np.array([-128, 127, -127], dtype=np.int8), s)) if extreme else (lambda *s: rng.integers(-128, 128, s).astype(np.int8))
    return (pick(n, k), np.exp(rng.standard_normal(n)).astype(np.float32), pick(m, k),
            (np.exp(rng.standard_normal(m)) * 1e-3).astype(np.float32), rng.standard_normal(m).astype(np.float32))


def run(r, qx, sx, qw, sw, bias, kind, ldw=None, ldx=None, ldy=None, offset=0, yoffset=0, stream=0):
    (n, k), m = qx.shape, qw.shape[0]
    ceil16 = max(16, (k + 15) // 16 * 16)
    w, x = Buffer(m, k, "int8", ldw or ceil16, offset, qw), Buffer(n, k, "int8", ldx or ceil16, offset, qx)
    a, b = Buffer(1, m, "fp32", values=sw[None]), Buffer(1, n, "fp32", values=sx[None])
    bb = Buffer(1, m, "fp32", values=bias[None]) if bias is not None else None
    y = Buffer(n, m, kind, ldy, yoffset)
    torch.cuda.synchronize()
    r.i8_linear(w.address, a.address, x.address, b.address, y.address, m, n, k, bias=bb.address if bb else None, ldw=w.ld, ldx=x.ld,
                ldy=y.ld, y_type=CODES[kind], stream=stream)
    torch.cuda.synchronize()
    assert r.last_status()[0] == 0 and y.untouched()
    return y.numpy()


def check(got, qx, sx, qw, sw, bias, kind):
    exact = model.linear(qx, sx, qw, sw, bias)
    product = np.abs(model.linear(qx, sx, qw, sw))
    bound = (2.01 * 2.0 ** -24 * product + 2.0 ** -24 * np.abs(exact)) * (1 + HALF_STEP[kind]) + HALF_STEP[kind] * np.abs(exact) + SMALLEST[kind]
    if kind == "fp16":   # results beyond the type's range
        over = np.abs(exact) > 65504
        assert np.all(np.abs(got[over]) >= 65504)
        got, exact, bound = np.where(over, 0, got), np.where(over, 0, exact), np.where(over, 1, bound)
    worst = np.max(np.abs(got - exact) / bound)
    assert worst <= 1.0, worst


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 31, 33, 64, 65, 128, 129, 200, 300])
def test_token_counts(r, kind, n):
    args = problem(300, n, 520, n)
    check(run(r, *args, kind), *args, kind)


@pytest.mark.parametrize("variant", [MAIN, SIMT, FEW, HALF])
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (2, 3, 16), (127, 1, 129), (128, 16, 128), (129, 17, 127), (256, 256, 256), (257, 255, 1000),
                                   (1000, 130, 90), (512, 300, 2048), (40, 600, 4097)])
def test_every_kernel_on_ragged_shapes(r, variant, m, n, k):
    r.set_option("force_variant", variant)
    args = problem(m, n, k, m + n + k)
    for kind in KINDS:
        check(run(r, *args, kind), *args, kind)
        assert r.info("last_variant") == variant


@pytest.mark.parametrize("parts", [1, 2, 4, 8])
@pytest.mark.parametrize("n", [1, 16, 30, 64, 100, 250])
def test_cut_k_gives_the_same_bits(r, parts, n):
    """K cut over the CTAs of a cluster, including more parts than K has stages: the integer sum is the same."""
    r.set_option("force_variant", FEW)
    for k in (64, 500, 3000):
        args = problem(200, n, k, n + k)
        r.set_option("split_k", 1)
        want = run(r, *args, "fp32")
        check(want, *args, "fp32")
        r.set_option("split_k", parts)
        assert np.array_equal(run(r, *args, "fp32"), want) and r.info("last_split_k") == parts


def test_all_kernels_agree_bit_for_bit(r):
    args = problem(700, 333, 1500, 2)
    outs = []
    for variant in (MAIN, SIMT, FEW, HALF):
        r.set_option("force_variant", variant)
        outs.append(run(r, *args, "fp32"))
    assert all(np.array_equal(outs[0], out) for out in outs[1:])


@pytest.mark.parametrize("variant", [MAIN, SIMT, FEW, HALF])
def test_largest_k_and_extreme_values_stay_exact(r, variant):
    """K = 131071 of -128 * -128: one below the 32-bit limit."""
    r.set_option("force_variant", variant)
    k = 131071
    qx, qw = np.full((3, k), -128, dtype=np.int8), np.full((130, k), -128, dtype=np.int8)
    qw[1, ::2] = 127
    sx, sw = np.ones(3, dtype=np.float32), np.ones(130, dtype=np.float32)
    check(run(r, qx, sx, qw, sw, None, "fp32"), qx, sx, qw, sw, None, "fp32")
    args = problem(140, 20, 5000, 1, extreme=True)
    check(run(r, *args, "fp32"), *args, "fp32")


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("k,ldw,ldx,ldy,offset,yoffset", [(100, 112, 128, None, 0, 0), (100, 100, 100, 261, 0, 1), (257, 257, 300, 300, 0, 3), (100, 112, 112, None, 5, 0),
                                                         (96, 96, 96, 1000, 16, 7), (1, 1, 1, None, 0, 0)])
def test_pitches_and_unaligned_operands(r, kind, k, ldw, ldx, ldy, offset, yoffset):
    for n in (3, 140):
        args = problem(260, n, k, k + n)
        check(run(r, *args, kind, ldw, ldx, ldy, offset, yoffset), *args, kind)
        aligned = ldw % 16 == 0 and ldx % 16 == 0 and offset % 16 == 0
        assert (r.info("last_variant") != SIMT) == aligned


def test_no_bias_no_features_and_empty_outputs(r):
    qx, sx, qw, sw, bias = problem(70, 9, 64, 4)
    check(run(r, qx, sx, qw, sw, None, "bf16"), qx, sx, qw, sw, None, "bf16")
    got = run(r, qx[:, :0], sx, qw[:, :0], sw, bias, "fp32")
    assert np.array_equal(got, np.tile(bias.astype(np.float64), (9, 1)))
    r.i8_linear(0, 0, 0, 0, 0, 0, 5, 3, y_type=0)
    r.i8_linear(0, 0, 0, 0, 0, 5, 0, 3, y_type=0)


def test_scales_that_are_not_finite_reach_their_row_only(r):
    for n in (5, 300):
        qx, sx, qw, sw, bias = problem(150, n, 200, 6)
        sx[2], sw[7] = np.nan, np.inf
        got = run(r, qx, sx, qw, sw, bias, "bf16")
        assert np.isnan(got[2]).all() and not np.isfinite(got[:, 7]).any()
        keep_n, keep_m = np.arange(n) != 2, np.arange(150) != 7
        check(got[np.ix_(keep_n, keep_m)], qx[keep_n], sx[keep_n], qw[keep_m], sw[keep_m], bias[keep_m], "bf16")


def test_large_problem_on_a_sample(r):
    """Many tiles per CTA pair: both accumulators and every ring phase are used over and over."""
    m, n, k = 4000, 4100, 1100
    args = problem(m, n, k, 12)
    for variant in (MAIN, HALF):
        r.set_option("force_variant", variant)
        got = run(r, *args, "bf16", ldy=4008)
        cols = np.arange(0, n, 13)
        check(got[cols], args[0][cols], args[1][cols], *args[2:], "bf16")


def test_concurrent_streams_and_captured_graphs(r):
    """Two captured calls replayed side by side on two streams, and eager calls beside them: no shared workspace to collide in."""
    args = problem(512, 24, 4096, 3)
    want = run(r, *args, "fp32")
    qx, sx, qw, sw, bias = args
    w, x = Buffer(512, 4096, "int8", values=qw), Buffer(24, 4096, "int8", values=qx)
    a, b, c = (Buffer(1, len(v), "fp32", values=v[None]) for v in (sw, sx, bias))
    outs = [torch.empty(24, 512, device="cuda") for _ in range(3)]
    call = lambda y, s: r.i8_linear(w.view, a.view, x.view, b.view, y, 512, 24, 4096, bias=c.view, stream=s.cuda_stream)   # noqa: E731
    torch.cuda.synchronize()
    graphs, streams = [], [torch.cuda.Stream() for _ in range(2)]
    for y, s in zip(outs, streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            call(y, s)
        graphs.append(g)
    for _ in range(20):
        for y in outs:
            y.fill_(float("nan"))
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        call(outs[2], torch.cuda.current_stream())
        torch.cuda.synchronize()
        for y in outs:
            assert np.array_equal(y.double().cpu().numpy(), want)
    assert r.last_status()[0] == 0
