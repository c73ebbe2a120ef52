"""The 64-bit model of the 8-bit operators against exact rational arithmetic, the INT8 configuration of the generator, and the Python
binding's handling of arguments: everything of the 8-bit operators that needs no GPU besides the entry points' own checks."""
from fractions import Fraction

import numpy as np
import pytest
import torch

from generator import generator as g
from oracle import i8_model as model
from runner import api

F, I8 = g.DataType.FP32, g.DataType.INT8


def exact_round(x: Fraction) -> int:
    """Nearest integer, halves to the even one."""
    return round(x)


@pytest.mark.parametrize("seed", range(4))
def test_model_rounds_the_exact_quotient(seed):
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((6, 50)).astype(np.float32)
    x[1] = np.arange(-25, 25) / 2.0          # a peak of 12.5: many quotients next to halves
    x[2] = np.concatenate([np.arange(-24.5, 25, 1.0), ])[:50]
    x[2, 0] = 127.0                          # exact ties
    x[3] = 0.0
    q, s = model.quantize(x)
    for row in range(6):
        peak = max(abs(Fraction(float(v))) for v in x[row])
        for j in range(50):
            want = exact_round(127 * Fraction(float(x[row, j])) / peak) if peak else 0
            assert q[row, j] == want
        assert s[row] == pytest.approx(float(peak) / 127, rel=1e-15)
    q, s = model.quantize(x, pow2=True)
    for row in range(6):
        peak = max(abs(Fraction(float(v))) for v in x[row])
        if not peak:
            assert s[row] == 0 and (q[row] == 0).all()
            continue
        scale = Fraction(s[row])
        assert 127 * scale >= peak and 127 * scale / 2 < peak and np.frexp(s[row])[0] == 0.5
        assert all(q[row, j] == exact_round(Fraction(float(x[row, j])) / scale) for j in range(50))


def test_model_of_rows_out_of_range():
    x = np.zeros((4, 3))
    x[0, 1], x[1, 0], x[2, 2], x[3, 1] = np.nan, np.inf, 1.5 * model.LARGEST, model.LARGEST
    for pow2 in (False, True):
        q, s = model.quantize(x, pow2)
        assert np.isnan(s[:3]).all() and (q[:3] == 0).all() and np.isfinite(s[3])
        assert abs(q[3, 1]) == 127 and np.isfinite(model.restore(q, s, "fp32")[3]).all()


def test_int8_configuration_and_its_refusals():
    cfg = g.tensor_config(256, 128, 6, cluster=2, trans_a=True, ab_type=I8)
    assert cfg.tile_size == (256, 256) and cfg.mfma == (128, 256, 1, 32) and cfg.stages == 6 and cfg.num_workitems == 384
    assert cfg.lds_usage_bytes == 6 * (128 + 128) * 128 + 1280 and cfg.acc_chain == 0 and cfg.companion_config() is None
    d = cfg.to_dict()
    assert (d["a_type"], d["b_type"], d["cd_type"]) == (3, 3, 0) and d["trans_a"] and not d["trans_b"]
    for kw in (dict(trans_a=False), dict(trans_b=True), dict(cluster=1), dict(bk=64), dict(split="inkernel"), dict(acc_chain=128),
               dict(epilogue_warps=4), dict(a_major="k"), dict(stages=9)):
        args = dict(bn=256, bk=128, stages=6, cluster=2, trans_a=True, ab_type=I8)
        args.update(kw)
        with pytest.raises(RuntimeError):
            g.tensor_config(**args)
    with pytest.raises(RuntimeError):      # A and B have one type
        g.GemmSolutionConfig(I8, F, F, F, (128, 256, 1, 32), (2, 1), (1, 1), 128, True, False)
    with pytest.raises(RuntimeError):      # the atom's K is that of the type
        g.GemmSolutionConfig(I8, I8, F, F, (128, 256, 1, 16), (2, 1), (1, 1), 128, True, False)
    with pytest.raises(RuntimeError):
        g.simt_config().__class__(I8, I8, F, F, (1, 1, 1, 1), (16, 16), (8, 8), 16, True, False)


def test_int8_source_and_recommendation(built):
    cfg = g.tensor_config(256, 128, 6, cluster=2, trans_a=True, ab_type=I8)
    src = g.gemm(None, "k", "sm_100a", cfg, g.GemmOptimizations(1, wgm=4), g.default_arguments())
    assert "#define I8_BN 256" in src and "#define I8_STAGES 6" in src and "#define OPT_WGM 4" in src
    assert "kind::i8" in src and "cp.async.bulk.tensor" in src and "i8_wgrad" in src and "i8_rmsnorm" in src
    # no load of a tile into several CTAs at once (only commits are multicast)
    assert all("tcgen05.commit" in line for line in src.split("\n") if "multicast::cluster" in line)
    assert built.recommend(16, 4096, 4096, operands="int8") == built.DEFAULT_I8 in built.REGISTRY
    parsed = api.parse_config(built.ensure(built.DEFAULT_I8)[1])
    assert parsed.a_type == 3 and parsed.trans_a == 1 and parsed.dynamic_smem_bytes == cfg.lds_usage_bytes


class Recorder:
    """Stands in for SgemmRunner: notes the arguments that the binding could not take by itself."""

    def __init__(self):
        self.asked = []

    def _addr(self, x, name, code=-1):
        self.asked.append((name, code))
        return 1 << 20


def test_binding_takes_addresses_and_asks_about_the_rest(built):
    native = api._native()
    r = Recorder()
    # a NULL handle: the C call answers, nothing is launched
    assert native.i8_restore(r, 0, 0, 1 << 20, 1 << 20, 1 << 20, 8, 4, 0, 0, 2, 0) == -1 and not r.asked
    q, s, out = torch.zeros(4, 8, dtype=torch.int8), torch.zeros(4), torch.zeros(4, 8, dtype=torch.bfloat16)
    assert native.i8_restore(r, 0, 0, q, s, out, 8, 4, 0, 0, None, 0) == -1            # CPU tensors: not on the handle's GPU
    assert r.asked == [("q", 3), ("scale", 0), ("out", -1)]
    with pytest.raises(TypeError, match="type with an address"):
        native.i8_restore(r, 0, 0, 1 << 20, 1 << 20, 1 << 20, 8, 4, 0, 0, None, 0)     # an address without its type
    with pytest.raises(TypeError):
        native.i8_restore(r, 0, 0, q, s, q, 8, 4, 0, 0, None, 0)                       # int8 is no output type
    with pytest.raises(OverflowError):
        native.i8_restore(r, 0, 0, 1 << 20, 1 << 20, 1 << 20, 1 << 32, 4, 0, 0, 0, 0)
    with pytest.raises(OverflowError):
        native.i8_restore(r, 0, 0, 1 << 20, 1 << 20, 1 << 20, -1, 4, 0, 0, 0, 0)
    with pytest.raises(TypeError):
        native.i8_restore(r, 0, 0, 1 << 20, 1 << 20, 1 << 20, "8", 4, 0, 0, 0, 0)
    with pytest.raises(ValueError, match="apart"):
        native.i8_restore(r, 0, 0, q[:1].expand(4, 8), s, out, 8, 4, 0, 0, None, 0)
    with pytest.raises(TypeError, match="arguments"):
        native.i8_restore(r, 0, 0, q)
    for name, count in (("i8_linear", 14), ("i8_quantize", 10), ("i8_rmsnorm", 15), ("i8_wgrad", 17)):
        with pytest.raises(TypeError, match="arguments"):
            getattr(native, name)(*[0] * (count + 2))


def test_operands_are_checked_by_name():
    runner = api.SgemmRunner.__new__(api.SgemmRunner)
    runner.device, runner._h = -1, None          # (CPU tensors lie on "device" -1)
    x = torch.zeros(4, 8)
    assert runner._addr(x, "x") == x.data_ptr() and runner._addr(None, "bias", 0) == 0 and runner._addr(64, "w", 3) == 64
    with pytest.raises(TypeError, match="x is torch.float32, the call takes int8"):
        runner._addr(x, "x", 3)
    with pytest.raises(ValueError, match="contiguous"):
        runner._addr(x.t(), "x")
    runner.device = 0
    with pytest.raises(ValueError, match="lies on cpu"):
        runner._addr(x, "x")
    with pytest.raises(api.SgemmError, match="closed"):
        runner.i8_restore(0, 0, 0, 1, 1, out_type=0)


def bare_runner(device=-1):
    runner = api.SgemmRunner.__new__(api.SgemmRunner)
    runner.device, runner._h = device, None
    return runner


@pytest.mark.parametrize("name", ["w_scale", "x_scale", "scale", "bias", "gamma"])
def test_vectors_with_gaps_are_refused(name):
    r = bare_runner()
    for x in (torch.zeros(4, 3)[:, :1], torch.zeros(8)[::2], torch.zeros(1).expand(4), torch.zeros(1, 1).expand(4, 1)):
        with pytest.raises(ValueError, match="contiguous"):
            r._addr(x, name, 0)
    for x in (torch.zeros(4), torch.zeros(4, 1), torch.zeros(1, 4), torch.zeros(4, 3)[1]):
        assert r._addr(x, name, 0) == x.data_ptr()


def test_rows_at_uneven_distances_are_refused():
    r = bare_runner()
    base = torch.zeros(3, 6, 16)
    for x in (base[:, :4], base[:, :4, :8], base[::2], base.transpose(0, 1), torch.zeros(6, 16).expand(3, 6, 16)):
        with pytest.raises(ValueError, match="one distance"):
            r._addr(x, "x")
    for x in (base, base[..., :8], base[:1, :4], base[1:2, 2:5, :3], base[:, :1], base[:, :, :8][1], torch.zeros(2, 3, 6, 16)[..., :8]):
        assert r._addr(x, "x") == x.data_ptr()
    with pytest.raises(ValueError, match="one distance"):
        r._addr(torch.zeros(2, 3, 6, 16)[:, :2], "x")


def test_host_arrays_are_refused(built):
    with pytest.raises(TypeError, match="ndarray"):
        bare_runner()._addr(np.zeros(4, np.float32), "scale", 0)
    with pytest.raises(TypeError, match="ndarray"):
        api._native().i8_restore(bare_runner(), 0, -1, np.zeros((4, 8), np.int8), 1, 1, 8, 4, 0, 0, 0, 0)


def test_a_type_that_is_not_the_tensors_is_refused(built):
    bf16 = torch.zeros(4, 8, dtype=torch.bfloat16)
    for code in (0, 1):
        with pytest.raises(TypeError, match="element type"):
            api._native().i8_restore(bare_runner(), 0, -1, 1 << 20, 1 << 20, bf16, 8, 4, 0, 0, code, 0)
    # its own type, and storage of another kind with the type said: only the NULL handle stops these
    assert api._native().i8_restore(bare_runner(), 0, -1, 1 << 20, 1 << 20, bf16, 8, 4, 0, 0, 2, 0) == -1
    assert api._native().i8_restore(bare_runner(), 0, -1, 1 << 20, 1 << 20, torch.zeros(4, 16, dtype=torch.uint8), 8, 4, 0, 0, 2, 0) == -1


@pytest.mark.parametrize("shape, stride, rows, pitch", [
    ((4, 8), (8, 1), 8, 8), ((4, 8), (24, 1), 8, 24), ((1, 8), (3, 1), 8, 8), ((1, 8), (32, 1), 8, 32), ((2, 3, 8), (36, 12, 1), 8, 12),
    ((5, 1, 8), (8, 40, 1), 8, 8), ((5, 1, 8), (8, 1, 1), 8, 8), ((5, 1, 1, 8), (16, 9, 77, 1), 8, 16), ((1, 1, 8), (99, 16, 1), 8, 16),
    ((8,), (1,), 8, 8), ((4, 8), (0, 1), 8, None), ((5, 1, 8), (4, 40, 1), 8, None)])
def test_pitch_is_that_of_the_rows(built, shape, stride, rows, pitch):
    x = torch.empty(4096, dtype=torch.int8).as_strided(shape, stride)
    if pitch is None:
        with pytest.raises(ValueError, match="elements apart"):
            api._native().pitch(x, rows)
    else:
        assert api._native().pitch(x, rows) == pitch


def test_pitch_of_a_transposed_batch_of_one(built):
    x = torch.zeros(1, 5, 16, dtype=torch.int8).transpose(0, 1)
    assert x.is_contiguous() and x.stride(-2) == 80 and api._native().pitch(x, 16) == 16
