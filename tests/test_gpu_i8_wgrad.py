"""The weight gradient from an 8-bit checkpoint against the 64-bit definition.

Products of 16-bit values are exact in FP32.  The tensor core adds 16 tokens at a time into its accumulator with truncation (two
guard bits: an error below 2^-23 of the largest partial sum per addition, of which there are at most 64 in a chain), and chains and parts
are added with round-to-nearest.  So an error is below (64 + chains + parts) * 2^-23 of the sum of magnitudes S; then alpha and beta
round twice more (2^-23 of S at most) and the result rounds to its type."""
import numpy as np
import pytest
import torch

from i8_cases import CODES, HALF_STEP, SMALLEST, TORCH, Buffer, activations
from oracle import i8_model as model
from runner import api

pytestmark = pytest.mark.gpu

AUTO, TENSOR, SIMT = 0, 1, 2


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


def problem(m, n, tokens, kind, seed=0, pow2=True):
    rng = np.random.default_rng(seed)
    q, s = model.quantize(activations(rng, tokens, m, "bf16") if tokens else np.zeros((0, m)), pow2)
    dy = torch.from_numpy(rng.standard_normal((tokens, n)) * 0.1 * np.exp(rng.standard_normal((tokens, 1)))).to(TORCH[kind]).double().numpy()
    return q, s.astype(np.float32), dy


def run(r, q, s, dy, kind, out, c=None, alpha=1.0, beta=0.0, inplace=False, ldq=None, lddy=None, lddw=None, offset=0, ooffset=0):
    (tokens, m), n = q.shape, dy.shape[1]
    qb = Buffer(tokens, m, "int8", ldq or (m + 15) // 16 * 16, offset, q)
    g = Buffer(tokens, n, kind, lddy or (n + 7) // 8 * 8, offset, dy)
    sb = Buffer(1, tokens, "fp32", values=s[None])
    d = Buffer(n, m, out, lddw, ooffset, c if inplace else None)
    cb = d if inplace else Buffer(n, m, out, lddw, ooffset, c) if c is not None else None
    torch.cuda.synchronize()
    r.i8_wgrad(qb.address, sb.address, g.address, d.address, m, n, tokens, c=cb.address if cb else None, alpha=alpha, beta=beta, ldq=qb.ld,
               lddy=g.ld, ldc=d.ld, lddw=d.ld, dy_type=CODES[kind], dw_type=CODES[out])
    torch.cuda.synchronize()
    assert r.last_status()[0] == 0 and d.untouched()
    return d.numpy()


def check(got, q, s, dy, kind, out, c=None, alpha=1.0, beta=0.0):
    want, size = model.wgrad(q, s, dy, kind, alpha, c, beta)
    chains = q.shape[0] // 512 + 8
    error = (64 + chains + 2) * 2.0 ** -23 * size
    bound = error + HALF_STEP[out] * (np.abs(want) + error) + SMALLEST[out]
    assert np.max(np.abs(got - want) / bound) <= 1.0


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("variant", [TENSOR, SIMT])
@pytest.mark.parametrize("m,n,tokens", [(1, 1, 1), (16, 8, 3), (130, 70, 63), (256, 256, 64), (257, 300, 65), (100, 513, 200), (600, 100, 1000), (128, 128, 2500)])
def test_shapes_types_and_kernels(r, kind, variant, m, n, tokens):
    r.set_option("force_variant", variant)
    p = problem(m, n, tokens, kind, m + n)
    for out in ("fp32", "bf16", "fp16"):
        check(run(r, *p, kind, out), *p, kind, out)
        assert r.info("last_variant") == variant


@pytest.mark.parametrize("parts", [1, 2, 3, 4])
@pytest.mark.parametrize("tokens", [100, 256, 1111, 5000])
def test_cut_tokens(r, parts, tokens):
    r.set_option("split_k", parts)
    p = problem(300, 270, tokens, "bf16", tokens)
    c = np.random.default_rng(1).standard_normal((270, 300))
    c = c.astype(np.float32).astype(np.float64)
    first = run(r, *p, "bf16", "fp32", c, 0.5, -2.0)
    check(first, *p, "bf16", "fp32", c, 0.5, -2.0)
    assert r.info("last_split_k") == min(parts, (tokens + 63) // 64)
    for _ in range(3):
        assert np.array_equal(run(r, *p, "bf16", "fp32", c, 0.5, -2.0), first)


@pytest.mark.parametrize("variant", [TENSOR, SIMT])
@pytest.mark.parametrize("out", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("inplace", [False, True])
def test_accumulation(r, variant, out, inplace):
    r.set_option("force_variant", variant)
    p = problem(200, 150, 300, "bf16", 3)
    c = torch.from_numpy(np.random.default_rng(2).standard_normal((150, 200))).to(TORCH[out]).double().numpy()
    check(run(r, *p, "bf16", out, c, 1.0, 1.0, inplace), *p, "bf16", out, c, 1.0, 1.0)
    check(run(r, *p, "bf16", out, c, 0.25, 3.0, inplace), *p, "bf16", out, c, 0.25, 3.0)
    # beta = 0 reads neither C nor what D held
    check(run(r, *p, "bf16", out, np.full((150, 200), np.nan), 1.0, 0.0, inplace), *p, "bf16", out)


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
def test_scales_that_are_no_powers_of_two(r, kind):
    """The checkpoint's values are then rounded to dY's type, as restore gives them."""
    p = problem(140, 90, 500, kind, 5, pow2=False)
    for variant in (TENSOR, SIMT):
        r.set_option("force_variant", variant)
        check(run(r, *p, kind, "fp32"), *p, kind, "fp32")


@pytest.mark.parametrize("ldq,lddy,lddw,offset,ooffset", [(160, 96, 144, 0, 0), (141, 90, 140, 0, 0), (144, 91, 141, 0, 1), (144, 96, 150, 3, 5), (144, 96, None, 16, 3)])
def test_pitches_and_unaligned_operands(r, ldq, lddy, lddw, offset, ooffset):
    p = problem(140, 90, 333, "bf16", 6)
    check(run(r, *p, "bf16", "bf16", ldq=ldq, lddy=lddy, lddw=lddw, offset=offset, ooffset=ooffset), *p, "bf16", "bf16")
    tma = ldq % 16 == 0 and lddy % 8 == 0 and offset % 16 == 0
    assert r.info("last_variant") == (TENSOR if tma else SIMT)


def test_no_tokens_and_tokens_of_zeros(r):
    q, s, dy = problem(40, 30, 0, "bf16")
    c = np.random.default_rng(3).standard_normal((30, 40)).astype(np.float32).astype(np.float64)
    assert (run(r, q, s, dy, "bf16", "fp32") == 0).all()
    assert np.array_equal(run(r, q, s, dy, "bf16", "fp32", c, 1.0, 1.0), c)
    q, s, dy = problem(40, 30, 80, "bf16")
    q[10:20], s[10:20] = 0, 0.0
    check(run(r, q, s, dy, "bf16", "fp32"), q, s, dy, "bf16", "fp32")


def test_a_token_out_of_range_makes_the_gradient_nan(r):
    q, s, dy = problem(50, 40, 90, "bf16")
    q[33], s[33] = 0, np.nan
    for variant in (TENSOR, SIMT):
        r.set_option("force_variant", variant)
        assert np.isnan(run(r, q, s, dy, "bf16", "fp32")).all()


def test_same_signed_sums_do_not_drift(r):
    """8192 tokens of one sign: truncation inside the tensor core would pile up without the chains.  A chain is at most 64
    additions, each off by less than 2^-24 of a partial sum that grows evenly to the chain's (half of it on average): 32 *
    2^-24; the 14 chains' sums add 14 * 2^-24 at most.  One chain of 512 additions could be off by 256 * 2^-24."""
    tokens = 8192
    q = np.full((tokens, 256), 100, dtype=np.int8)
    q[:, ::3] = 77
    s = np.full(tokens, 2.0 ** -6, dtype=np.float32)
    dy = torch.from_numpy(np.abs(np.random.default_rng(4).standard_normal((tokens, 256))) + 0.1).bfloat16().double().numpy()
    got = run(r, q, s, dy, "bf16", "fp32")
    want, _ = model.wgrad(q, s, dy, "bf16")
    check(got, q, s, dy, "bf16", "fp32")
    assert np.max(np.abs(got / want - 1)) < 46 * 2.0 ** -24


def test_many_tiles_per_pair(r):
    p = problem(2600, 4500, 700, "bf16", 9)
    got = run(r, *p, "bf16", "bf16")
    rows = np.arange(0, 4500, 37)
    check(got[rows], p[0], p[1], p[2][:, rows], "bf16", "bf16")


def test_gradient_against_differences(r):
    """d/dW of sum(dY * (V W^T)) taken by differences: the loss is linear in W, so a difference of any step gives the derivative, up to
    64-bit rounding; the checkpoint's V comes from the device's own quantize and restore."""
    rng = np.random.default_rng(11)
    tokens, m, n = 96, 48, 40
    x = Buffer(tokens, m, "bf16", values=activations(rng, tokens, m, "bf16"))
    q, s, v = Buffer(tokens, m, "int8"), Buffer(1, tokens, "fp32"), Buffer(tokens, m, "bf16")
    r.i8_quantize(x.view, q.view, s.view, m, tokens, pow2=True)
    r.i8_restore(q.view, s.view, v.view, m, tokens)
    values = v.numpy()
    dy = torch.from_numpy(rng.standard_normal((tokens, n))).bfloat16().double().numpy()
    got = run(r, q.numpy(), s.numpy()[0].astype(np.float32), dy, "bf16", "fp32")
    weight = rng.standard_normal((n, m))
    loss = lambda w: float(np.sum(dy * (values @ w.T)))   # noqa: E731
    for i, j in [(0, 0), (3, 47), (39, 12), (17, 30)]:
        bumped = weight.copy()
        bumped[i, j] += 1.0
        lowered = weight.copy()
        lowered[i, j] -= 1.0
        size = np.sum(np.abs(dy[:, i] * values[:, j]))
        assert abs((loss(bumped) - loss(lowered)) / 2 - got[i, j]) <= 80 * 2.0 ** -23 * size + 1e-9


def test_captured_graph_and_streams(r):
    q, s, dy = problem(512, 384, 4096, "bf16", 13)
    want = run(r, q, s, dy, "bf16", "fp32")
    qb, sb, g = Buffer(4096, 512, "int8", values=q), Buffer(1, 4096, "fp32", values=s[None]), Buffer(4096, 384, "bf16", values=dy)
    outs = [torch.empty(384, 512, device="cuda") for _ in range(2)]
    streams, graphs = [torch.cuda.Stream() for _ in range(2)], []
    torch.cuda.synchronize()
    for y, st in zip(outs, streams):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            r.i8_wgrad(qb.view, sb.view, g.view, y, 512, 384, 4096, stream=st.cuda_stream)
        graphs.append(graph)
    for _ in range(10):
        for y in outs:
            y.fill_(float("nan"))
        torch.cuda.synchronize()
        for graph, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                graph.replay()
        torch.cuda.synchronize()
        for y in outs:
            assert np.array_equal(y.double().cpu().numpy(), want)
