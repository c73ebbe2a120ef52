"""The linear layer on wide outputs with few tokens, by the kernel that the plan takes there, and the binding's checks on the GPU's own tensors.
The integer sum is exact, its conversion and the two products are one rounding each, the bias's addition is fused with the second."""
import numpy as np
import pytest
import torch

from i8_cases import HALF_STEP, SMALLEST, TORCH
from runner import api

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def r(built):
    with api.SgemmRunner(*built.ensure(built.DEFAULT_I8)) as runner:
        yield runner


@pytest.mark.parametrize("kind", ["bf16", "fp32"])
@pytest.mark.parametrize("tokens, channels, features", [(1, 12288, 4096), (1, 57345, 272), (3, 100003, 144), (16, 40000, 1040), (17, 28673, 512), (33, 20001, 2048),
                                                        (64, 65536, 128), (100, 14337, 1024), (128, 40000, 384)])
def test_wide_outputs_for_few_tokens(r, kind, tokens, channels, features):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(channels)
    w = torch.randint(-127, 128, (channels, features), dtype=torch.int8, device="cuda", generator=gen)
    x = torch.randint(-127, 128, (tokens, features), dtype=torch.int8, device="cuda", generator=gen)
    sw, sx = (torch.rand(n, device="cuda", generator=gen) + 0.01 for n in (channels, tokens))
    bias = torch.randn(channels, device="cuda", generator=gen)
    y = torch.full((tokens + 1, channels), 77.0, dtype=TORCH[kind], device="cuda")
    r.i8_linear(w, sw, x, sx, y, channels, tokens, features, bias=bias)
    torch.cuda.synchronize()
    assert r.last_status()[0] == 0
    product = (x.double() @ w.double().T) * sx.double()[:, None] * sw.double()
    want = product + bias.double()
    # of the product: the sum's conversion and the product with x_scale; then one rounding of the fused step and one to the type
    error = 2 * 2.0 ** -24 * (1 + 2.0 ** -24) * product.abs()
    error = error + 2.0 ** -24 * (want.abs() + error)
    bound = error + HALF_STEP[kind] * (want.abs() + error) + SMALLEST[kind]
    assert bool(((y[:tokens].double() - want).abs() <= bound).all())
    assert bool((y[tokens] == 77.0).all())


def test_short_tensors_and_other_devices_are_refused_on_the_gpu(r):
    q, s = torch.zeros(16, 32, dtype=torch.int8, device="cuda"), torch.zeros(16, device="cuda")
    y, p = torch.zeros(16, 16, device="cuda"), torch.nn.Parameter(torch.zeros(16, device="cuda"))
    r.i8_linear(q, p, q, s, y, 16, 16, 32, bias=p)
    for args in ((q[:15], s, q, s, y), (q, s[:15], q, s, y), (q, s, q[:, :31], s, y), (q, s, q, s[1:], y), (q, s, q, s, y[:15]), (q, s, q.cpu(), s, y),
                 (q, s, q, s.cpu(), y), (q, s, q, s, y.to("meta"))):
        with pytest.raises(ValueError):
            r.i8_linear(*args, 16, 16, 32)
    with pytest.raises(ValueError):
        r.i8_linear(q, s, q, s, y, 16, 16, 32, bias=s[:3])
    torch.cuda.synchronize()
    assert np.array_equal(y.detach().cpu().numpy(), np.zeros((16, 16)))
