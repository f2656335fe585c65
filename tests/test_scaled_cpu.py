"""The 8-bit linear layer without a GPU: the oracle's own arithmetic, plan refusals, C ABI refusals."""

from __future__ import annotations

import ctypes

import ml_dtypes
import numpy as np
import pytest
import torch

from oracle import scaled as oracle
from tpu_cake_b200 import _native
from tpu_cake_b200 import scaled_cuda_lowering as scaled

E4M3 = np.dtype(ml_dtypes.float8_e4m3fn)


def test_oracle_rounds_like_the_format():
    # Every e4m3 value rounds to itself, and the midpoints between neighbours go to the even code.
    codes = np.arange(0x7F, dtype=np.uint8)
    values = codes.view(E4M3).astype(np.float64)
    assert np.array_equal(oracle.round_e4m3(values), values) and values[-1] == 448
    middles = (values[:-1] + values[1:]) / 2
    assert np.array_equal(oracle.round_e4m3(middles), values[codes[:-1] + (codes[:-1] & 1)])
    generator = np.random.default_rng(0)
    v = generator.uniform(-448, 448, 20000).astype(np.float32)
    v[:5000] *= 2.0**-12
    assert np.array_equal(oracle.round_e4m3(v.astype(np.float64)), v.astype(E4M3).astype(np.float64))


@pytest.mark.parametrize("largest, scale", [(448.0, 1.0), (np.nextafter(448.0, 1e9), 2.0), (224.0, 0.5), (1e-45, 2.0**-127),
                                            (0.0, 1.0), (3.4e38, 2.0**120), (np.inf, np.nan), (np.nan, np.nan)])
def test_oracle_scale_is_the_least_power_of_two(largest, scale):
    row = np.zeros((1, 130))
    row[0, 7] = -largest if np.isfinite(largest) else largest
    got = oracle.group_scales(row)
    assert got.shape == (1, 2) and got[0, 1] == 1.0
    assert np.isnan(got[0, 0]) if np.isnan(scale) else got[0, 0] == scale


def test_plans_refuse_what_they_do_not_run():
    for arguments in ({"columns": 0}, {"columns": 8, "input_dtype": "f64"}, {"columns": 8, "gate": "gelu"}):
        with pytest.raises(ValueError):
            scaled.CudaQuantizeRowsPlan(name="p", **arguments)
    for arguments in ({"columns": 0}, {"columns": scaled.MAX_NORM_COLUMNS + 1}, {"columns": 8, "input_dtype": "i8"},
                      {"columns": 8, "input_dtype": "bf16", "weight_dtype": "f16"}, {"columns": 8, "epsilon": -1.0},
                      {"columns": 8, "epsilon": float("nan")}):
        with pytest.raises(ValueError):
            scaled.CudaRmsNormQuantizePlan(name="p", **arguments)
    for arguments in ({"n": 0, "k": 8}, {"n": 8, "k": 0}, {"n": 1 << 30, "k": 8}, {"n": 8, "k": 1 << 27}, {"n": 8, "k": 8, "output_dtype": "f16"},
                      {"n": 8, "k": 8, "tile": 160}, {"n": 8, "k": 8, "tile": 256, "k_split": 2}, {"n": 8, "k": 8, "k_split": 2}, {"n": 8, "k": 8, "tile": 192, "k_split": 2},
                      {"n": 8, "k": 8, "tile": 16, "k_split": 9}):
        with pytest.raises(ValueError):
            scaled.CudaScaledMatmulPlan(name="p", **arguments)


def test_plan_sources_tell_plans_apart():
    a = scaled.CudaScaledMatmulPlan(name="p", n=256, k=512)
    assert a.source_sha256() == scaled.CudaScaledMatmulPlan(name="p", n=256, k=512).source_sha256()
    assert a.source_sha256() != scaled.CudaScaledMatmulPlan(name="p", n=256, k=512, output_dtype="f32").source_sha256()
    assert "cake_scaled_matmul_sm100" in a.render_executable_source()
    assert "cake_rms_norm_quantize_sm100" in scaled.CudaRmsNormQuantizePlan(name="p", columns=64).render_executable_source()
    assert "cake_quantize_rows_sm100" in scaled.CudaQuantizeRowsPlan(name="p", columns=64).render_executable_source()


@pytest.mark.parametrize("columns, pitch", [(1, 128), (16, 128), (100, 128), (128, 128), (1000, 1024)])
def test_codes_get_the_pitch_the_matmul_wants(columns, pitch):
    codes = scaled.empty_codes(3, columns, torch.device("cpu"))
    assert tuple(codes.shape) == (3, columns) and codes.stride() == (pitch, 1) and codes.dtype == torch.float8_e4m3fn
    assert tuple(scaled.empty_scales(3, columns, torch.device("cpu")).shape) == (3, -(-columns // 128))


class _Recorder:
    """An executable that records the binding calls instead of making them."""

    index = 0

    def __init__(self, plan=None):
        self.calls, self.plan, self.binding = [], plan, self
        self.desc_address = self.status_address = 0

    def record(self, *arguments):
        self.calls.append(arguments)
        return tuple(arguments[-2:])

    quantize_rows = rms_norm_quantize = scaled_matmul = record


def test_invoke_refuses_what_a_plan_does_not_take():
    recorder = _Recorder()
    x, weight = torch.zeros(4, 100, dtype=torch.bfloat16), torch.ones(100, dtype=torch.bfloat16)
    norm = scaled.CudaRmsNormQuantizePlan(name="p", columns=100)
    with pytest.raises(ValueError, match="residual"):
        norm.invoke(recorder, x, weight)
    plain = scaled.CudaRmsNormQuantizePlan(name="p", columns=100, with_residual=False)
    with pytest.raises(ValueError, match="residual"):
        plain.invoke(recorder, x, weight, x)
    with pytest.raises(ValueError, match="residual_out"):
        plain.invoke(recorder, x, weight, residual_out=x)
    matmul = scaled.CudaScaledMatmulPlan(name="p", n=32, k=256)
    with pytest.raises(ValueError, match="another plan"):
        matmul.invoke(_Recorder(scaled.CudaScaledMatmulPlan(name="p", n=32, k=512)), None, None, None, None)
    assert not recorder.calls
    norm.invoke(recorder, x, weight, x)
    same = _Recorder(scaled.CudaScaledMatmulPlan(name="p", n=32, k=256))
    matmul.invoke(same, 1, 2, 3, 4)
    assert len(recorder.calls) == 1 and same.calls == [(0, 0, 0, 1, 2, 3, 4, None)]


F32, BF16, CODES, SCALES = 0, 1, 3, 4


def test_row_operands_are_checked():
    check = _native.load_torch_binding().check_rows
    x = torch.zeros(4, 100, dtype=torch.bfloat16)
    assert check(x, 100, BF16, "x", -1, -1) == (4, 100) and check(x[::2], 100, BF16, "x", -1, 2) == (2, 200)
    assert check(x[:1].expand(1, 100), 100, BF16, "x", -1, 1)[0] == 1 and check(x[:0], 100, BF16, "x", -1, -1)[0] == 0
    assert check(torch.zeros(3, 7).to(torch.float8_e4m3fn), 7, CODES, "codes", -1, 3) == (3, 7)
    assert check(torch.ones(3, 2).to(torch.float8_e8m0fnu), 2, SCALES, "scales", -1, 3) == (3, 2)
    for wrong in (x.float(), x[:, :99], x[0], x.t(), x[None], None, 7, x.to_sparse()):
        with pytest.raises(ValueError, match="x must be a BFloat16 tensor of shape"):
            check(wrong, 100, BF16, "x", -1, -1)
    with pytest.raises(ValueError, match=r"out must be a Float tensor of shape \(5, 100\)"):
        check(x.float(), 100, F32, "out", -1, 5)
    for wrong in (torch.zeros(4, 200, dtype=torch.bfloat16)[:, ::2], x[:1].expand(4, 100), torch.zeros(400, dtype=torch.bfloat16).as_strided((4, 100), (99, 1))):
        with pytest.raises(ValueError, match="contiguous rows that do not overlap"):
            check(wrong, 100, BF16, "x", -1, -1)
    with pytest.raises(ValueError, match="x must be on cuda:0"):
        check(x, 100, BF16, "x", 0, -1)
    with pytest.raises(TypeError, match="6 arguments"):
        check(x)


def test_binding_calls_refuse_tensors_that_are_not_on_the_device():
    binding = _native.load_torch_binding()
    x, weight = torch.zeros(4, 100, dtype=torch.bfloat16), torch.ones(100, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="x must be on cuda:0"):
        binding.quantize_rows(0, x, 100, BF16, 0, None, None)
    with pytest.raises(ValueError, match="x must be a BFloat16 tensor of shape .rows, 200."):
        binding.quantize_rows(0, x, 100, BF16, 1, None, None)
    with pytest.raises(ValueError, match="x must be on cuda:0"):
        binding.rms_norm_quantize(0, x, 100, BF16, weight, BF16, 1e-5, x, None, None, None)
    desc = _native.ScaledMatmulDesc(n=32, k=100, out_dtype=1, tile=0, k_split=0)
    with pytest.raises(ValueError, match="lhs must be a Float8_e4m3fn tensor"):
        binding.scaled_matmul(0, ctypes.addressof(desc), 0, x, None, None, None, None)
    for call in (binding.quantize_rows, binding.rms_norm_quantize, binding.scaled_matmul, binding.init):
        with pytest.raises(TypeError, match="arguments"):
            call()


def _quantize(**overrides):
    arguments = dict(x=1 << 20, dtype=1, x_stride=128, gate=0, rows=2, cols=128, q=1 << 20, q_stride=128, scales=1 << 20, scales_stride=1, stream=None)
    arguments.update(overrides)
    return _native.load().cake_quantize_rows_enqueue(*arguments.values())


@pytest.mark.parametrize("overrides, code, fragment", [
    ({"cols": 0}, _native.CAKE_ERR_INVALID_ARGUMENT, "columns"),
    ({"cols": 1 << 40}, _native.CAKE_ERR_INVALID_ARGUMENT, "columns"),
    ({"rows": 1 << 30, "cols": 129, "x_stride": 129, "q_stride": 129, "scales_stride": 2}, _native.CAKE_ERR_UNSUPPORTED, "below 2^31"),
    ({"x_stride": 1 << 32}, _native.CAKE_ERR_UNSUPPORTED, "below 2^32"),
    ({"rows": -1}, _native.CAKE_ERR_INVALID_ARGUMENT, "rows"),
    ({"rows": 1 << 31}, _native.CAKE_ERR_INVALID_ARGUMENT, "rows"),
    ({"dtype": 7}, _native.CAKE_ERR_INVALID_ARGUMENT, "dtype"),
    ({"gate": 2}, _native.CAKE_ERR_INVALID_ARGUMENT, "gate"),
    ({"x": None}, _native.CAKE_ERR_INVALID_ARGUMENT, "null"),
    ({"scales": None}, _native.CAKE_ERR_INVALID_ARGUMENT, "null"),
    ({"x": (1 << 20) + 1}, _native.CAKE_ERR_INVALID_ARGUMENT, "aligned"),
    ({"x_stride": 127}, _native.CAKE_ERR_INVALID_ARGUMENT, "stride"),
    ({"gate": 1}, _native.CAKE_ERR_INVALID_ARGUMENT, "stride"),
    ({"q_stride": 0}, _native.CAKE_ERR_INVALID_ARGUMENT, "stride"),
    ({"scales_stride": 0}, _native.CAKE_ERR_INVALID_ARGUMENT, "stride"),
])
def test_quantize_refuses_bad_arguments(overrides, code, fragment):
    assert _quantize(**overrides) == code
    assert fragment in _native.load().cake_last_error().decode()


def test_no_rows_is_no_work():
    assert _quantize(rows=0, x=None, q=None, scales=None) == _native.CAKE_OK
    assert _norm(rows=0, x=None, weight=None, q=None, scales=None) == _native.CAKE_OK


def _norm(**overrides):
    arguments = dict(x=1 << 20, dtype=1, x_stride=128, residual=None, residual_stride=0, residual_out=None, residual_out_stride=0, weight=1 << 20,
                     weight_dtype=1, epsilon=1e-5, rows=2, cols=128, q=1 << 20, q_stride=128, scales=1 << 20, scales_stride=1, stream=None)
    arguments.update(overrides)
    return _native.load().cake_rms_norm_quantize_enqueue(*arguments.values())


@pytest.mark.parametrize("overrides, code, fragment", [
    ({"cols": 0}, _native.CAKE_ERR_UNSUPPORTED, "columns"),
    ({"cols": 32769}, _native.CAKE_ERR_UNSUPPORTED, "columns"),
    ({"weight_dtype": 2}, _native.CAKE_ERR_UNSUPPORTED, "weight"),
    ({"epsilon": -1.0}, _native.CAKE_ERR_INVALID_ARGUMENT, "epsilon"),
    ({"epsilon": float("nan")}, _native.CAKE_ERR_INVALID_ARGUMENT, "epsilon"),
    ({"dtype": 9, "weight_dtype": 0}, _native.CAKE_ERR_INVALID_ARGUMENT, "dtype"),
    ({"weight": None}, _native.CAKE_ERR_INVALID_ARGUMENT, "null"),
    ({"weight": (1 << 20) + 1}, _native.CAKE_ERR_INVALID_ARGUMENT, "aligned"),
    ({"residual": 1 << 20}, _native.CAKE_ERR_INVALID_ARGUMENT, "come together"),
    ({"residual_out": 1 << 20}, _native.CAKE_ERR_INVALID_ARGUMENT, "come together"),
    ({"residual": 1 << 20, "residual_out": 1 << 20, "residual_stride": 128}, _native.CAKE_ERR_INVALID_ARGUMENT, "stride"),
    ({"x_stride": 5}, _native.CAKE_ERR_INVALID_ARGUMENT, "stride"),
])
def test_norm_refuses_bad_arguments(overrides, code, fragment):
    assert _norm(**overrides) == code
    assert fragment in _native.load().cake_last_error().decode()


def _matmul(**overrides):
    desc = dict(n=128, k=128, out_dtype=1, tile=0, k_split=0)
    arguments = dict(m=2, lhs=1 << 20, lhs_stride=128, lhs_scales=1 << 20, lhs_scales_stride=1, rhs=1 << 20, rhs_stride=128, rhs_scales=1 << 20,
                     rhs_scales_stride=1, out=1 << 20, out_stride=128, status=None, stream=None)
    for name, value in overrides.items():
        (desc if name in desc else arguments)[name] = value
    return _native.load().cake_scaled_matmul_enqueue(ctypes.byref(_native.ScaledMatmulDesc(**desc)), *arguments.values())


@pytest.mark.parametrize("overrides, code, fragment", [
    ({"n": 0}, _native.CAKE_ERR_INVALID_ARGUMENT, "extents"),
    ({"k": 1 << 27}, _native.CAKE_ERR_INVALID_ARGUMENT, "extents"),
    ({"n": 1 << 30}, _native.CAKE_ERR_INVALID_ARGUMENT, "extents"),
    ({"out_dtype": 2}, _native.CAKE_ERR_INVALID_ARGUMENT, "out_dtype"),
    ({"tile": 160}, _native.CAKE_ERR_UNSUPPORTED, "tile"),
    ({"k_split": 9, "tile": 16}, _native.CAKE_ERR_INVALID_ARGUMENT, "k_split"),
    ({"k_split": 2}, _native.CAKE_ERR_INVALID_ARGUMENT, "k_split"),
    ({"k_split": 2, "tile": 224}, _native.CAKE_ERR_INVALID_ARGUMENT, "k_split"),
    ({"m": -1}, _native.CAKE_ERR_INVALID_ARGUMENT, "m must"),
    ({"m": 1 << 30}, _native.CAKE_ERR_INVALID_ARGUMENT, "m must"),
    ({"lhs": None}, _native.CAKE_ERR_INVALID_ARGUMENT, "null"),
    ({"rhs_scales": None}, _native.CAKE_ERR_INVALID_ARGUMENT, "null"),
    ({"lhs": (1 << 20) + 8}, _native.CAKE_ERR_INVALID_ARGUMENT, "16-byte aligned"),
    ({"rhs_stride": 136}, _native.CAKE_ERR_INVALID_ARGUMENT, "multiples of 16"),
    ({"lhs_stride": 112}, _native.CAKE_ERR_INVALID_ARGUMENT, "at least k"),
    ({"lhs_scales_stride": 0}, _native.CAKE_ERR_INVALID_ARGUMENT, "scales row stride"),
    ({"rhs_scales_stride": 0}, _native.CAKE_ERR_INVALID_ARGUMENT, "scales row stride"),
    ({"out_stride": 127}, _native.CAKE_ERR_INVALID_ARGUMENT, "output row stride"),
    ({"out": (1 << 20) + 1}, _native.CAKE_ERR_INVALID_ARGUMENT, "aligned to its elements"),
    ({"status": (1 << 20) + 2}, _native.CAKE_ERR_INVALID_ARGUMENT, "status_device"),
])
def test_scaled_matmul_refuses_bad_arguments(overrides, code, fragment):
    assert _matmul(**overrides) == code
    assert fragment in _native.load().cake_last_error().decode()


def test_null_descriptor_is_an_error_and_no_rows_are_no_work():
    assert ctypes.sizeof(_native.ScaledMatmulDesc) == 32
    assert _native.load().cake_scaled_matmul_enqueue(None, 1, *[None, 0] * 5, None, None) == _native.CAKE_ERR_INVALID_ARGUMENT
    assert _matmul(m=0, lhs=None, lhs_scales=None, rhs=None, rhs_scales=None, out=None) == _native.CAKE_OK


def test_mlp_plan_and_runner_refuse_bad_shapes(tmp_path):
    from tpu_cake_b200 import cli, scaled_runner

    plan = scaled.CudaScaledMlpPlan(name="layer", hidden=640, inner=1000)
    assert plan.up.n == 2000 and plan.up.k == 640 and plan.down.n == 640 and plan.down.k == 1000 and plan.gate.gate == "silu"
    for kernel in ("cake_rms_norm_quantize_sm100", "cake_scaled_matmul_sm100", "cake_quantize_rows_sm100"):
        assert kernel in plan.render_executable_source()
    for wrong in ({"hidden": scaled.MAX_NORM_COLUMNS + 1, "inner": 8}, {"hidden": 8, "inner": 0}):
        with pytest.raises(ValueError):
            scaled.CudaScaledMlpPlan(name="layer", **wrong)
    with pytest.raises(ValueError, match="up must be"):
        plan.quantize_weights(None, None, torch.zeros(4, 4), torch.zeros(4, 4))
    with pytest.raises(ValueError, match="positive"):
        scaled_runner.run_scaled_mlp(tmp_path / "out", rows=0, hidden=64, inner=64)
    if not torch.cuda.is_available():
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            cli.main(["run-scaled-mlp", str(tmp_path / "out")])
    assert not (tmp_path / "out").exists()


def test_runner_bounds_reject_a_wrong_scale():
    from tpu_cake_b200 import scaled_runner

    v = torch.randn(4, 300, generator=torch.Generator().manual_seed(0)).double()
    codes, scales = oracle.quantize(v.numpy())
    codes = torch.from_numpy(codes).float().to(torch.float8_e4m3fn)
    byte = torch.from_numpy(np.log2(scales) + 127).to(torch.uint8)
    assert scaled_runner._check_codes(codes, byte.view(torch.float8_e8m0fnu), v) <= 1
    byte[2, 1] += 1
    assert scaled_runner._check_codes(codes, byte.view(torch.float8_e8m0fnu), v) > 1
    lhs, rhs = v, torch.randn(7, 300, generator=torch.Generator().manual_seed(1)).double()
    out = (lhs @ rhs.t()).to(torch.bfloat16)
    assert scaled_runner._check_matmul(out, lhs, rhs) <= 1
    out[1, 2] *= 1.02
    assert scaled_runner._check_matmul(out, lhs, rhs) > 1
