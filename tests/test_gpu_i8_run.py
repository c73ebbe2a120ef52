"""The 8-bit operators together, as a program uses them: a block of a network that answers with 8-bit layers, a training step whose
activations are kept in 8 bits beside the framework's BF16 products, and the runner program on an INT8 kernel."""
import json

import numpy as np
import pytest
import torch

from i8_cases import HALF_STEP, activations, check_rounded
from oracle import i8_model as model
from runner import api
from test_gpu_runner_cli import run_cli

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def r(built):
    with api.SgemmRunner(*built.ensure(built.DEFAULT_I8)) as runner:
        yield runner


def tensor(values, dtype=torch.bfloat16):
    return torch.from_numpy(np.ascontiguousarray(values)).to("cuda", dtype)


def weights8(r, rng, channels, features):
    w = tensor(rng.standard_normal((channels, features)) * 0.05, torch.float32)
    q, s = torch.empty(channels, features, dtype=torch.int8, device="cuda"), torch.empty(channels, device="cuda")
    r.i8_quantize(w, q, s, features, channels)
    return q, s


@pytest.mark.parametrize("tokens", [1, 24, 300])
def test_a_block_of_8_bit_layers(r, tokens):
    """residual + norm -> linear -> 8 bits again -> linear, eagerly and as a captured graph: every step against its definition on what
    the step before it gave."""
    rng = np.random.default_rng(tokens)
    k, hidden = 512, 1200
    x, res = tensor(activations(rng, tokens, k, "bf16")), tensor(activations(rng, tokens, k, "bf16"))
    gamma = tensor(1 + 0.1 * rng.standard_normal(k))
    (q1, s1), (q2, s2) = weights8(r, rng, hidden, k), weights8(r, rng, k, hidden)
    bias = tensor(rng.standard_normal(hidden), torch.float32)
    new = lambda *shape, dtype: torch.empty(*shape, dtype=dtype, device="cuda")   # noqa: E731
    a, sa, up = new(tokens, k, dtype=torch.int8), new(tokens, dtype=torch.float32), new(tokens, hidden, dtype=torch.bfloat16)
    b, sb, out = new(tokens, hidden, dtype=torch.int8), new(tokens, dtype=torch.float32), new(tokens, k, dtype=torch.bfloat16)
    total = new(tokens, k, dtype=torch.bfloat16)

    def block(stream):
        r.i8_rmsnorm(x, gamma, a, sa, k, tokens, residual=res, sum_out=total, eps=1e-5, stream=stream)
        r.i8_linear(q1, s1, a, sa, up, hidden, tokens, k, bias=bias, stream=stream)
        r.i8_quantize(up, b, sb, hidden, tokens, stream=stream)
        r.i8_linear(q2, s2, b, sb, out, k, tokens, hidden, stream=stream)

    block(torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    eager = [t.clone() for t in (a, sa, total, up, b, sb, out)]
    host = lambda t: (t if t.dtype == torch.int8 else t.double()).cpu().numpy()   # noqa: E731
    q, s, h = model.rmsnorm(host(x), host(gamma), 1e-5, host(res))
    assert np.array_equal(host(a), q) and np.array_equal(host(total), model.round_to(h, "bf16"))
    check_rounded(host(sa), s, "fp32", 66 * 2.0 ** -24)
    for got, qx, sx, qw, sw, c in ((up, a, sa, q1, s1, bias), (out, b, sb, q2, s2, None)):
        y = model.linear(host(qx), host(sx), host(qw), host(sw), host(c) if c is not None else None)
        product = np.abs(model.linear(host(qx), host(sx), host(qw), host(sw)))
        bound = 1.01 * (3 * 2.0 ** -24 * (product + np.abs(y))) + HALF_STEP["bf16"] * np.abs(y)
        assert np.all(np.abs(host(got) - y) <= bound)
    assert np.array_equal(host(b), model.quantize(host(up))[0])
    graph = torch.cuda.CUDAGraph()
    stream = torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=stream):
        block(stream.cuda_stream)
    for t in (a, sa, total, up, b, sb, out):
        t.zero_()
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    for t, want in zip((a, sa, total, up, b, sb, out), eager):
        assert torch.equal(t, want)
    assert r.last_status()[0] == 0


def test_a_training_step_with_8_bit_checkpoints(r, built):
    """Y = X W^T in BF16 on the framework's own product, X kept in 8 bits, the gradients of W and X from it: W's against the formula
    on the kept values and, loosely, on X itself; X's is the framework's BF16 product as before."""
    rng = np.random.default_rng(5)
    tokens, k, n = 640, 384, 256
    x, w = activations(rng, tokens, k, "bf16", 0.3), rng.standard_normal((n, k)) * 0.05
    X, W = tensor(x), tensor(w)
    w = W.double().cpu().numpy()
    dy = rng.standard_normal((tokens, n))
    dY = tensor(dy)
    dy = dY.double().cpu().numpy()
    Y, dX = torch.empty(tokens, n, device="cuda"), torch.empty(tokens, k, device="cuda")
    q, s = torch.empty(tokens, k, dtype=torch.int8, device="cuda"), torch.empty(tokens, device="cuda")
    grad = torch.full((n, k), 0.25, device="cuda")
    # forward: column-major Y (n x tokens) = W^T-stored (K x n) times X (K x tokens): the transposed-A kernel
    with api.SgemmRunner(*built.ensure("bf16_tc_128x256x32_s4_tn")) as tn, api.SgemmRunner(*built.ensure("bf16_tc2_256x256x64_s6")) as nn:
        tn.launch(W, X, None, Y, n, tokens, k, lda=k, ldb=k)
        r.i8_quantize(X, q, s, k, tokens, pow2=True)
        # backward: dX (k x tokens) = W (k x n) dY (n x tokens), dW (k x n) += kept X (k x tokens) dY^T
        nn.launch(W, dY, None, dX, k, tokens, n)
        r.i8_wgrad(q, s, dY, grad, k, n, tokens, c=grad, beta=1.0)
        torch.cuda.synchronize()
        assert tn.last_status()[0] == 0 and nn.last_status()[0] == 0 and r.last_status()[0] == 0
    kept = q.cpu().numpy().astype(np.float64) * s.double().cpu().numpy()[:, None]
    assert np.all(np.abs(kept - x) <= 0.5 * s.double().cpu().numpy()[:, None])
    want, size = dy.T @ kept + 0.25, np.abs(dy).T @ np.abs(kept) + 0.25
    assert np.all(np.abs(grad.double().cpu().numpy() - want) <= 80 * 2.0 ** -23 * size)
    # against the gradient from unrounded activations: each token's error is at most half its scale
    full = dy.T @ x + 0.25
    assert np.all(np.abs(want - full) <= np.abs(dy).T @ np.repeat(0.5 * s.double().cpu().numpy()[:, None], k, 1) + 1e-9)
    assert np.all(np.abs(Y.double().cpu().numpy() - x @ w.T) <= 2.0 ** -18 * (np.abs(x) @ np.abs(w).T))
    assert np.all(np.abs(dX.double().cpu().numpy() - dy @ w) <= 2.0 ** -18 * (np.abs(dy) @ np.abs(w)))


def test_tensors_of_the_wrong_kind_are_refused(r):
    q, s = torch.zeros(16, 32, dtype=torch.int8, device="cuda"), torch.zeros(16, device="cuda")
    y = torch.zeros(16, 16, device="cuda")
    r.i8_linear(q, s, q, s, y, 16, 16, 32)
    for bad in (dict(w=q.float()), dict(w_scale=s.double()), dict(x_scale=s.bfloat16()), dict(x=q.cpu()), dict(bias=s.half()), dict(y=q),
                dict(x=torch.zeros(32, 16, dtype=torch.int8, device="cuda").t())):
        args = dict(w=q, w_scale=s, x=q, x_scale=s, y=y, bias=None)
        args.update(bad)
        with pytest.raises((TypeError, ValueError)):
            r.i8_linear(args["w"], args["w_scale"], args["x"], args["x_scale"], args["y"], 16, 16, 32, bias=args["bias"])
    with pytest.raises(TypeError):
        r.i8_rmsnorm(y, s.half(), q, s, 16, 16)
    with pytest.raises(OverflowError):
        r.i8_linear(q, s, q, s, y, 16, 2 ** 32, 32)
    with pytest.raises(api.SgemmError, match="K above 131071"):
        r.i8_linear(q, s, q, s, y, 16, 16, 131072, ldw=131072, ldx=131072)
    with pytest.raises(api.SgemmError, match="leading dimension"):
        r.i8_linear(q, s, q, s, y, 16, 16, 32, ldw=31)
    x16 = torch.zeros(64 * 64, device="cuda")
    with pytest.raises(api.SgemmError, match="sgemm_i8"):     # the FP32-result calls refuse this cubin
        r.launch(x16, x16, None, x16, 8, 8, 8)
    with pytest.raises(api.SgemmError, match="sgemm_i8"):
        r.workspace_bytes(256, 256, 256)


def test_leading_dimensions_come_from_two_dimensional_tensors(r):
    """Rows inside wider buffers without a leading dimension in the call; rows that overlap are refused."""
    rng = np.random.default_rng(2)
    x = tensor(rng.standard_normal((20, 96)), torch.float32)
    q, s, out = torch.zeros(20, 64, dtype=torch.int8, device="cuda"), torch.zeros(20, device="cuda"), torch.zeros(20, 80, device="cuda")
    r.i8_quantize(x[:, :50], q[:, :50], s, 50, 20)
    r.i8_restore(q, s, out[:, 3:53], 50, 20)
    torch.cuda.synchronize()
    want, scale = model.quantize(x.double().cpu().numpy()[:, :50])
    assert np.array_equal(q.cpu().numpy()[:, :50], want) and (q[:, 50:] == 0).all()
    assert np.array_equal(out[:, 3:53].double().cpu().numpy(), model.restore(want, s.double().cpu().numpy(), "fp32"))
    assert (out[:, :3] == 0).all() and (out[:, 53:] == 0).all()
    with pytest.raises(ValueError, match="apart"):
        r.i8_quantize(x[:1].expand(20, 96), q, s, 50, 20)
    r.i8_quantize(x[:1].expand(1, 96), q, s, 50, 1)


def test_other_cubins_refuse_the_8_bit_calls(built):
    q, s = torch.zeros(16, 32, dtype=torch.int8, device="cuda"), torch.zeros(16, device="cuda")
    with api.SgemmRunner(*built.ensure(built.DEFAULT_SIMT)) as other:
        with pytest.raises(api.SgemmError, match="INT8"):
            other.i8_restore(q, s, torch.zeros(16, 32, device="cuda"), 32, 16)


def test_bounded_wait_self_test_on_the_int8_cubin(r):
    r.wait_selftest(5, 0x1234)
    with pytest.raises(api.SgemmError, match="gave up"):
        r.last_status()
    assert r.last_status()[0] == 0


@pytest.mark.parametrize("m,n,k", [(512, 768, 640), (300, 5, 1000)])
def test_runner_program_on_an_int8_kernel(built, tmp_path, m, n, k):
    ret = run_cli(built, built.DEFAULT_I8, m, n, k, 1, env={"SGEMM_JSON": str(tmp_path / "r.json"), "SGEMM_SEED": "3"})
    assert ret.returncode == 0, ret.stdout + ret.stderr
    lines = ret.stdout.split("\n")
    assert lines[0].startswith("cpuGemm func: ") and lines[1].startswith("SIMT gemm: ") and lines[4].startswith("ASM gemm: ")
    assert lines[2].startswith("Gflops: ") and lines[3].startswith("GiB/s: ") and lines[7] == f"# of mismatches: 0/{m * n}"
    rec = json.loads((tmp_path / "r.json").read_text())
    assert rec["variant"] == "tcgen05_int8" and rec["mismatches"] == 0 and rec["tflops"] > 0 and "tcgen05 INT8" in ret.stderr
