"""The weight gradient against the host model of the tensor core's arithmetic, bit for bit: chains of 32 additions of 16 tokens inside the tensor core
(512 tokens), each added to a running sum in FP32 that starts as beta * C; cut tokens are added in the order of their parts."""
import numpy as np
import pytest

from oracle import i8_model as model
from oracle import tensor_model
from test_gpu_i8_wgrad import TENSOR, problem, r, run, runner  # noqa: F401

pytestmark = pytest.mark.gpu

CHAIN = 512      # tokens


def predicted(q, s, dy, kind, c, alpha, beta, parts, chain=CHAIN):
    """[channels, features] in FP32 as the kernel computes it."""
    tokens = q.shape[0]
    values, g = model.restore(q, s, kind).astype(np.float32), dy.astype(np.float32)
    blocks = (tokens + 63) // 64
    total = None
    for part in range(parts):
        first, last = blocks * part // parts * 64, min(tokens, blocks * (part + 1) // parts * 64)
        start = np.float32(beta) * c.astype(np.float32) if beta and part == 0 else np.zeros((dy.shape[1], q.shape[1]), dtype=np.float32)
        for t in range(first, last, chain):
            end = min(last, t + chain)
            start = tensor_model._fma_f32(tensor_model.accumulate(g[t:end].T, values[t:end], terms=1, mma_k=16), np.float32(alpha), start)
        total = start if total is None else (total + start).astype(np.float32)
    return total


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("parts", [1, 3])
@pytest.mark.parametrize("tokens", [1, 16, 100, 512, 513, 1111, 5000])
@pytest.mark.parametrize("alpha, beta", [(1.0, 0.0), (0.75, -1.25)])
def test_gradient_equals_the_model_bit_for_bit(r, kind, parts, tokens, alpha, beta):   # noqa: F811
    r.set_option("force_variant", TENSOR)
    r.set_option("split_k", parts)
    q, s, dy = problem(40, 24, tokens, kind, tokens)
    c = np.random.default_rng(7).standard_normal((24, 40)).astype(np.float32).astype(np.float64)
    got = run(r, q, s, dy, kind, "fp32", c if beta else None, alpha, beta)
    used = r.info("last_split_k")
    assert used == min(parts, (tokens + 63) // 64)
    want = predicted(q, s, dy, kind, c, alpha, beta, used)
    assert np.array_equal(got, want)
    if tokens > 2000 and parts == 1:     # the comparison tells the length of the chains
        assert not np.array_equal(want, predicted(q, s, dy, kind, c, alpha, beta, used, 2 * CHAIN))
        assert not np.array_equal(want, predicted(q, s, dy, kind, c, alpha, beta, used, CHAIN // 2))


def test_same_signed_sums_of_8192_tokens(r):   # noqa: F811
    """Truncation inside the tensor core drifts: an addition loses half a unit in the last place on average, at most 2^-24 of the partial sum.  Over a
    chain of 32 additions to an evenly growing sum that is 16.5 * 2^-24 of the chain; adding up the 16 chains, rounded to nearest,
    is off by 16 * 2^-24 at most: 32.5 * 2^-24."""
    tokens = 8192
    q = np.full((tokens, 256), 100, dtype=np.int8)
    q[:, ::3] = 77
    s = np.full(tokens, 2.0 ** -6, dtype=np.float32)
    dy = model.round_bf16(np.abs(np.random.default_rng(4).standard_normal((tokens, 256))) + 0.1)
    got = run(r, q, s, dy, "bf16", "fp32")
    want, _ = model.wgrad(q, s, dy, "bf16")
    assert np.max(np.abs(got / want - 1)) <= 32.5 * 2.0 ** -24
