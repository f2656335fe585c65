"""The 8-bit linear layer on the GPU against the float64 oracle.

Tolerances. Quantising x itself is exact: codes and scales equal the oracle's. After arithmetic in f32 (gate,
norm) a value v may differ from the oracle's by a relative DELTA before it is rounded, so the code times its
scale lies within half a step of the exact v moved by that much: 2^-4 |v| for normal codes (three mantissa
bits), 2^-10 s below 2^-6. DELTA for silu(g) u: 2^t within 2^-22 and the reciprocal within 2^-23 (the
hardware estimates' documented bounds), a correction, a sum and two products: 4 + 2 + 1 + 1 + 2 = 10 times 2^-24,
below 2^-20. For the norm: at most 40 sequential and 15 tree additions of squares (half of
that error reaches the root), quotient, root, two products: below 64 * 2^-24 = 2^-18.
Matmul: products of codes and powers of two are exact in f32; k additions in f32 are off by at most
k 2^-24 S with S = sum |lhs| |rhs|, and the output's own rounding by 2^-8 |out| (bf16) or nothing (f32).
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import scaled as oracle
from tpu_cake_b200 import scaled_cuda_lowering as scaled

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
GATE_DELTA = 2.0**-20
NORM_DELTA = 2.0**-18


def numpy64(tensor) -> np.ndarray:
    return tensor.detach().double().cpu().numpy()


def scale_values(scales) -> np.ndarray:
    """e8m0 bytes as the values they stand for, by the format's definition."""
    byte = scales.contiguous().view(torch.uint8).cpu().numpy().astype(np.float64)
    return np.where(byte == 255, np.nan, np.exp2(byte - 127))


def activations(seed, rows, cols, dtype, device, pad=0):
    generator = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols + pad, generator=generator)
    x[:, ::37] *= 25.0
    return x.to(DTYPES[dtype]).to(device)[:, :cols]


def operand(seed, rows, k, device, *, exact=False, scale_pad=0, row_pad=0):
    """Codes and scales; ``exact``: small enough that any order of summation in f32 is exact."""
    generator = torch.Generator().manual_seed(seed)
    if exact:
        values = torch.randint(-3, 4, (rows, k), generator=generator).float()
        bytes_ = torch.randint(126, 129, (rows, -(-k // 128) + scale_pad), generator=generator)
    else:
        values = (torch.randn(rows, k, generator=generator) * 60).clamp(-448, 448)
        bytes_ = torch.randint(115, 130, (rows, -(-k // 128) + scale_pad), generator=generator)
    pitch = -(-k // 16) * 16 + row_pad
    codes = torch.full((rows, pitch), float("nan")).to(torch.float8_e4m3fn)  # what lies between rows must not matter
    codes[:, :k] = values.to(torch.float8_e4m3fn)
    scales = bytes_.to(torch.uint8).view(torch.float8_e8m0fnu)
    return codes.to(device)[:, :k], scales.to(device)[:, : -(-k // 128)]


def check_close(codes, scales, expected, delta):
    expected_codes, expected_scales = oracle.quantize(expected)
    got_scales = scale_values(scales)
    assert np.array_equal(got_scales, expected_scales, equal_nan=True)
    step = oracle.expand(got_scales, expected.shape[1])
    error = np.abs(numpy64(codes) * step - expected)
    assert np.all(error <= (2.0**-4 * (1 + delta) + delta) * np.abs(expected) + 2.0**-10 * step)
    # A code only changes where a value lies within delta of a border, borders being 2^-4 apart or more.
    assert np.mean(numpy64(codes) != expected_codes) <= 64 * delta


# ------------------------------------------------------------------------------------------ quantise


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows, cols, pad", [(1, 1, 0), (1, 8, 0), (3, 127, 0), (2, 128, 0), (5, 129, 3), (64, 1000, 0), (7, 1024, 64), (33, 4100, 1), (1, 16384, 0), (70, 8192, 0)])
def test_quantize_is_exact(cuda_device, dtype, rows, cols, pad):
    x = activations(rows * 7 + cols, rows, cols, dtype, cuda_device, pad)
    plan = scaled.CudaQuantizeRowsPlan(name="t", columns=cols, input_dtype=dtype)
    codes, scales = plan.invoke(plan.build(cuda_device), x)
    expected_codes, expected_scales = oracle.quantize(numpy64(x))
    assert codes.stride(0) % 128 == 0
    assert np.array_equal(numpy64(codes), expected_codes)
    assert np.array_equal(scale_values(scales), expected_scales)


def test_quantize_special_groups(cuda_device):
    x = torch.zeros(6, 300)
    x[0, 0], x[0, 128], x[0, 299] = float("nan"), float("inf"), float("-inf")
    x[1] = 0.0
    x[1, 5] = -0.0
    x[2, :128], x[2, 128:256], x[2, 256:] = 448.0, 448.00003, 3.4e38
    x[3, :128], x[3, 128:256], x[3, 256:] = 1e-45, 1e-38, 2.0**-120
    x[4] = torch.linspace(-500, 500, 300)
    x[5] = torch.exp2(torch.linspace(-40, 9, 300))
    plan = scaled.CudaQuantizeRowsPlan(name="t", columns=300, input_dtype="f32")
    codes, scales = plan.invoke(plan.build(cuda_device), x.to(cuda_device))
    expected_codes, expected_scales = oracle.quantize(x.double().numpy())
    assert np.array_equal(scale_values(scales), expected_scales, equal_nan=True)
    assert np.array_equal(numpy64(codes), expected_codes, equal_nan=True)
    assert np.isnan(expected_scales[0]).all() and np.isnan(numpy64(codes)[0]).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows, cols, pad", [(1, 1, 0), (2, 100, 5), (3, 128, 0), (65, 1032, 0), (17, 1001, 1), (4, 16384, 0)])
def test_gated_quantize(cuda_device, dtype, rows, cols, pad):
    x = activations(rows + cols, rows, 2 * cols, dtype, cuda_device, pad)
    plan = scaled.CudaQuantizeRowsPlan(name="t", columns=cols, input_dtype=dtype, gate="silu")
    codes, scales = plan.invoke(plan.build(cuda_device), x)
    check_close(codes, scales, oracle.silu_and_mul(numpy64(x)), GATE_DELTA)


def test_gate_far_from_zero(cuda_device):
    # exp(-g) overflows below about -88: the product is -0 there, and up to 1 times u above.
    gate = torch.tensor([-3e38, -200.0, -104.0, -88.0, -20.0, -0.0, 0.0, 20.0, 200.0, 3e38])
    x = torch.cat([gate, torch.tensor([1.0, 2.0, -3.0, 1e4, 5.0, 1.0, 7.0, -1.0, 2.0, 0.5])])[None].to(cuda_device)
    plan = scaled.CudaQuantizeRowsPlan(name="t", columns=10, input_dtype="f32", gate="silu")
    codes, scales = plan.invoke(plan.build(cuda_device), x)
    check_close(codes, scales, oracle.silu_and_mul(numpy64(x)), GATE_DELTA)


# ------------------------------------------------------------------------------------------ norm


@pytest.mark.parametrize("dtype, weight_dtype", [("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16"), ("f16", "f32"), ("f32", "f32")])
@pytest.mark.parametrize("rows, cols, pad", [(1, 1, 0), (9, 64, 0), (3, 129, 3), (2, 1024, 0), (5, 1025, 0), (1, 4096, 0), (4, 4104, 8), (3, 8192, 0), (2, 8200, 0), (2, 16384, 0), (2, 16390, 1), (1, 32768, 0)])
@pytest.mark.parametrize("with_residual", [False, True])
def test_rms_norm(cuda_device, dtype, weight_dtype, rows, cols, pad, with_residual):
    x = activations(rows + cols, rows, cols, dtype, cuda_device, pad)
    residual = activations(rows + cols + 1, rows, cols, dtype, cuda_device, pad) if with_residual else None
    weight = (1 + 0.2 * torch.randn(cols, generator=torch.Generator().manual_seed(cols))).to(DTYPES[weight_dtype]).to(cuda_device)
    plan = scaled.CudaRmsNormQuantizePlan(name="t", columns=cols, input_dtype=dtype, weight_dtype=weight_dtype, epsilon=1e-5, with_residual=with_residual)
    codes, scales, summed = plan.invoke(plan.build(cuda_device), x, weight, residual)
    expected, _h = oracle.rms_norm(numpy64(x), numpy64(weight), 1e-5, None if residual is None else numpy64(residual))
    check_close(codes, scales, expected, NORM_DELTA)
    if with_residual:
        assert torch.equal(summed, (x.float() + residual.float()).to(DTYPES[dtype]))
    else:
        assert summed is None


@pytest.mark.parametrize("which", ["residual", "x"])
def test_rms_norm_updates_the_residual_in_place(cuda_device, which):
    x, residual = activations(1, 5, 5000, "bf16", cuda_device), activations(2, 5, 5000, "bf16", cuda_device)
    weight = torch.ones(5000, dtype=torch.bfloat16, device=cuda_device)
    plan = scaled.CudaRmsNormQuantizePlan(name="t", columns=5000)
    executable = plan.build(cuda_device)
    codes, scales, summed = plan.invoke(executable, x, weight, residual)
    target = x if which == "x" else residual
    again = plan.invoke(executable, x, weight, residual, residual_out=target)
    assert again[2] is target and torch.equal(target, summed)
    assert torch.equal(again[0].view(torch.uint8), codes.view(torch.uint8)) and torch.equal(again[1].view(torch.uint8), scales.view(torch.uint8))


def test_rms_norm_special_rows(cuda_device):
    x = torch.randn(4, 400, generator=torch.Generator().manual_seed(0))
    x[0] = 0.0
    x[1, 3] = float("nan")
    x[2, 3] = float("inf")
    plan = scaled.CudaRmsNormQuantizePlan(name="t", columns=400, input_dtype="f32", weight_dtype="f32", epsilon=0.0, with_residual=False)
    codes, scales, _ = plan.invoke(plan.build(cuda_device), x.to(cuda_device), torch.ones(400, device=cuda_device))
    with np.errstate(invalid="ignore", divide="ignore"):
        # 0 / 0 in the row of zeros without epsilon; the row's infinity leaves zeros elsewhere.
        assert np.isnan(numpy64(codes)[:2]).all() and np.isnan(scale_values(scales)[:2]).all()
        assert np.isnan(numpy64(codes)[2, :128]).all() and np.isnan(scale_values(scales)[2, 0])
        assert (numpy64(codes)[2, 128:] == 0).all() and (scale_values(scales)[2, 1:] == 1).all()
        expected, _h = oracle.rms_norm(x[3:].double().numpy(), np.ones(400), 0.0)
    check_close(codes[3:], scales[3:], expected, NORM_DELTA)


def test_rows_leave_what_lies_around_them(cuda_device):
    """Outputs that are slices of wider buffers, at odd offsets: nothing outside them is written."""
    x = activations(3, 6, 300, "bf16", cuda_device)
    held_codes = torch.full((8, 333), 7, dtype=torch.uint8, device=cuda_device)
    held_scales = torch.full((8, 9), 9, dtype=torch.uint8, device=cuda_device)
    codes, scales = held_codes[1:7, 5:305].view(torch.float8_e4m3fn), held_scales[1:7, 3:6].view(torch.float8_e8m0fnu)
    plan = scaled.CudaQuantizeRowsPlan(name="t", columns=300)
    plan.invoke(plan.build(cuda_device), x, codes=codes, scales=scales)
    expected_codes, expected_scales = oracle.quantize(numpy64(x))
    assert np.array_equal(numpy64(codes.contiguous()), expected_codes) and np.array_equal(scale_values(scales), expected_scales)
    norm = scaled.CudaRmsNormQuantizePlan(name="t", columns=300, with_residual=False)
    norm.invoke(norm.build(cuda_device), x, torch.ones(300, dtype=torch.bfloat16, device=cuda_device), codes=codes, scales=scales)
    held_codes[1:7, 5:305] = 7
    held_scales[1:7, 3:6] = 9
    assert (held_codes == 7).all() and (held_scales == 9).all()


# ------------------------------------------------------------------------------------------ matmul


def run_matmul(device, m, n, k, *, seed=0, exact=True, output_dtype="f32", tile=0, k_split=0, **layout):
    lhs, lhs_scales = operand(seed, m, k, device, exact=exact, **layout)
    rhs, rhs_scales = operand(seed + 1, n, k, device, exact=exact, **layout)
    plan = scaled.CudaScaledMatmulPlan(name="t", n=n, k=k, output_dtype=output_dtype, tile=tile, k_split=k_split)
    executable = plan.build(device)
    out = plan.invoke(executable, lhs, lhs_scales, rhs, rhs_scales)
    assert executable.status() == (0, 0, 0, 0)
    executable.close()
    a, b = numpy64(lhs) * oracle.expand(scale_values(lhs_scales), k), numpy64(rhs) * oracle.expand(scale_values(rhs_scales), k)
    return out, a @ b.T, np.abs(a) @ np.abs(b).T


@pytest.mark.parametrize("tile, k_split", [(16, 1), (16, 2), (16, 3), (16, 8), (32, 1), (32, 4), (64, 1), (64, 2), (128, 1), (128, 5), (192, 0), (224, 0), (256, 0), (0, 0)])
@pytest.mark.parametrize("m, n, k", [(1, 1, 1), (1, 128, 128), (16, 128, 1024), (5, 300, 520), (33, 129, 650), (130, 225, 140), (200, 448, 2048)])
def test_matmul_is_exact_where_f32_is(cuda_device, m, n, k, tile, k_split):
    # Codes -3..3 and scales 1/2, 1, 2: sums of multiples of 1/4 below 36 k, which f32 holds exactly.
    out, expected, _ = run_matmul(cuda_device, m, n, k, seed=m + n + k, tile=tile, k_split=k_split)
    assert np.array_equal(numpy64(out), expected)


@pytest.mark.parametrize("output_dtype", ["bf16", "f32"])
@pytest.mark.parametrize("m, n, k", [(1, 1024, 4096), (64, 777, 2000), (300, 520, 1111), (257, 1300, 384), (512, 640, 8192)])
def test_matmul_random(cuda_device, m, n, k, output_dtype):
    out, expected, magnitude = run_matmul(cuda_device, m, n, k, seed=k, exact=False, output_dtype=output_dtype)
    rounding = 2.0**-8 if output_dtype == "bf16" else 0.0
    assert np.all(np.abs(numpy64(out) - expected) <= rounding * np.abs(expected) + k * 2.0**-24 * magnitude * (1 + rounding))
    relative = np.linalg.norm(numpy64(out) - expected) / np.linalg.norm(expected)
    assert relative <= (2.0**-8 if output_dtype == "bf16" else 1e-5)


@pytest.mark.parametrize("layout", [{"scale_pad": 1}, {"scale_pad": 3}, {"row_pad": 16}, {"row_pad": 48, "scale_pad": 2}])
@pytest.mark.parametrize("tile, k_split", [(16, 3), (64, 1), (128, 0), (224, 0)])
def test_matmul_takes_strided_operands(cuda_device, layout, tile, k_split):
    out, expected, _ = run_matmul(cuda_device, 70, 260, 1300, tile=tile, k_split=k_split, **layout)
    assert np.array_equal(numpy64(out), expected)


@pytest.mark.parametrize("output_dtype", ["bf16", "f32"])
@pytest.mark.parametrize("tile, k_split", [(16, 2), (32, 1), (128, 0), (192, 0)])
@pytest.mark.parametrize("offset, width", [(0, 304), (8, 320), (1, 303), (3, 305)])
def test_matmul_writes_its_rows_only(cuda_device, output_dtype, tile, k_split, offset, width):
    m, n, k = 37, 290, 260
    lhs, lhs_scales = operand(5, m, k, cuda_device, exact=True)
    rhs, rhs_scales = operand(6, n, k, cuda_device, exact=True)
    held = torch.full((m + 2, width), 1234.0, dtype=DTYPES[output_dtype], device=cuda_device)
    before = held.clone()
    out = held[1 : m + 1, offset : offset + n]
    plan = scaled.CudaScaledMatmulPlan(name="t", n=n, k=k, output_dtype=output_dtype, tile=tile, k_split=k_split)
    executable = plan.build(cuda_device)
    assert plan.invoke(executable, lhs, lhs_scales, rhs, rhs_scales, out=out) is out
    expected = oracle.matmul(numpy64(lhs), scale_values(lhs_scales), numpy64(rhs), scale_values(rhs_scales))
    assert torch.equal(out.cpu(), torch.from_numpy(expected).to(DTYPES[output_dtype]))
    out.fill_(1234.0)
    assert torch.equal(held, before)
    executable.close()


def test_matmul_nan_codes_and_scales_stay_in_their_rows(cuda_device):
    for tile in (16, 128):
        lhs, lhs_scales = operand(1, 40, 300, cuda_device, exact=True)
        rhs, rhs_scales = operand(2, 150, 300, cuda_device, exact=True)
        lhs.view(torch.uint8)[3, 299] = 0x7F
        lhs_scales.view(torch.uint8)[7, 1] = 255
        rhs.view(torch.uint8)[149, 0] = 0xFF
        rhs_scales.view(torch.uint8)[4, 2] = 255
        plan = scaled.CudaScaledMatmulPlan(name="t", n=150, k=300, output_dtype="f32", tile=tile)
        out = numpy64(plan.invoke(plan.build(cuda_device), lhs, lhs_scales, rhs, rhs_scales))
        expected = oracle.matmul(numpy64(lhs), scale_values(lhs_scales), numpy64(rhs), scale_values(rhs_scales))
        assert np.isnan(expected[3]).all() and np.isnan(expected[:, 4]).all()
        assert np.array_equal(out, expected, equal_nan=True)


def test_matmul_extreme_scales(cuda_device):
    # Scales from 2^-127 on: products of two small ones underflow as f32 does, a small and a large one do not.
    codes = torch.full((16, 128), 2.0).to(torch.float8_e4m3fn).to(cuda_device)
    low = torch.full((16, 1), 0, dtype=torch.uint8, device=cuda_device).view(torch.float8_e8m0fnu)
    high = torch.full((16, 1), 247, dtype=torch.uint8, device=cuda_device).view(torch.float8_e8m0fnu)
    plan = scaled.CudaScaledMatmulPlan(name="t", n=16, k=128, output_dtype="f32")
    out = plan.invoke(plan.build(cuda_device), codes, low, codes, high)
    assert torch.equal(out, torch.full_like(out, 512.0 * 2.0**-7))


def test_no_rows(cuda_device):
    rhs, rhs_scales = operand(2, 64, 256, cuda_device)
    plan = scaled.CudaScaledMatmulPlan(name="t", n=64, k=256)
    assert tuple(plan.invoke(plan.build(cuda_device), rhs[:0], rhs_scales[:0], rhs, rhs_scales).shape) == (0, 64)
    quantize = scaled.CudaQuantizeRowsPlan(name="t", columns=256)
    codes, scales = quantize.invoke(quantize.build(cuda_device), torch.empty(0, 256, dtype=torch.bfloat16, device=cuda_device))
    assert tuple(codes.shape) == (0, 256) and tuple(scales.shape) == (0, 2)


# ------------------------------------------------------------------------------------------ together


class Mlp:
    """norm -> gate and up projection -> gated activation -> down projection, as a decoder layer runs it."""

    def __init__(self, device, hidden, inner, seed=0):
        generator = torch.Generator().manual_seed(seed)
        self.norm_weight = (1 + 0.1 * torch.randn(hidden, generator=generator)).to(torch.bfloat16).to(device)
        self.up = (torch.randn(2 * inner, hidden, generator=generator) * hidden**-0.5).to(torch.bfloat16).to(device)
        self.down = (torch.randn(hidden, inner, generator=generator) * inner**-0.5).to(torch.bfloat16).to(device)
        self.norm = scaled.CudaRmsNormQuantizePlan(name="norm", columns=hidden)
        self.up_plan = scaled.CudaScaledMatmulPlan(name="up", n=2 * inner, k=hidden)
        self.gate = scaled.CudaQuantizeRowsPlan(name="gate", columns=inner, gate="silu")
        self.down_plan = scaled.CudaScaledMatmulPlan(name="down", n=hidden, k=inner)
        self.rows = self.norm.build(device)
        self.up_executable, self.down_executable = self.up_plan.build(device), self.down_plan.build(device)
        self.up8 = scaled.CudaQuantizeRowsPlan(name="w", columns=hidden).invoke(self.rows, self.up)
        self.down8 = scaled.CudaQuantizeRowsPlan(name="w", columns=inner).invoke(self.rows, self.down)

    def __call__(self, x, residual, out=None):
        codes, scales, summed = self.norm.invoke(self.rows, x, self.norm_weight, residual, residual_out=residual)
        up = self.up_plan.invoke(self.up_executable, codes, scales, *self.up8)
        return self.down_plan.invoke(self.down_executable, *self.gate.invoke(self.rows, up), *self.down8, out=out), summed

    def reference(self, x, residual):
        def bf16(values):
            return torch.from_numpy(values).to(torch.bfloat16).double().numpy()

        normed, h = oracle.rms_norm(numpy64(x), numpy64(self.norm_weight), 1e-5, numpy64(residual))
        up = bf16(oracle.matmul(*oracle.quantize(normed), *oracle.quantize(numpy64(self.up))))
        return oracle.matmul(*oracle.quantize(oracle.silu_and_mul(up)), *oracle.quantize(numpy64(self.down))), bf16(h)


@pytest.mark.parametrize("rows", [1, 5, 64, 300])
def test_mlp_runs_as_a_layer(cuda_device, rows):
    mlp = Mlp(cuda_device, 640, 1000)
    x, residual = activations(1, rows, 640, "bf16", cuda_device), activations(2, rows, 640, "bf16", cuda_device)
    expected, expected_residual = mlp.reference(x, residual)
    out, summed = mlp(x, residual)
    # The bf16 rounding of the intermediate and the 8-bit rounding after it see values that differ in the last
    # f32 bits: a value next to a border moves by a whole bf16 step (2^-7), an 8-bit one by 2^-3. At most a few in
    # a thousand are next to one, sqrt(0.004) 2^-3 of the norm together, beside the output's own 2^-8.
    assert np.linalg.norm(numpy64(out) - expected) <= (2.0**-8 + 2.0**-7) * np.linalg.norm(expected)
    assert np.linalg.norm(numpy64(summed) - expected_residual) <= 2.0**-8 * np.linalg.norm(expected_residual)


def test_mlp_in_a_graph_on_another_stream_and_twice_at_once(cuda_device):
    mlp = Mlp(cuda_device, 512, 768)
    streams = [torch.cuda.Stream(cuda_device) for _ in range(2)]
    inputs = [(activations(10 + i, 20 + i, 512, "bf16", cuda_device), activations(20 + i, 20 + i, 512, "bf16", cuda_device)) for i in range(2)]
    expected = [mlp(x, r.clone()) for x, r in inputs]
    held = [(x, r.clone(), torch.zeros_like(x)) for x, r in inputs]
    torch.cuda.synchronize(cuda_device)
    graphs = []
    for stream, (x, r, out) in zip(streams, held, strict=True):
        with torch.cuda.stream(stream):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                mlp(x, r, out)
        graphs.append(graph)
    for _ in range(3):
        for (x, r, out), (_, r0) in zip(held, inputs, strict=True):
            r.copy_(r0)
            out.zero_()
        torch.cuda.synchronize(cuda_device)
        for stream, graph in zip(streams, graphs, strict=True):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize(cuda_device)
        for (_, r, out), (want, want_residual) in zip(held, expected, strict=True):
            assert torch.equal(out, want) and torch.equal(r, want_residual)


def test_repeats_give_the_same_bits(cuda_device):
    for m, n, k in ((3, 2048, 4096), (300, 500, 1500)):
        lhs, lhs_scales = operand(1, m, k, cuda_device)
        rhs, rhs_scales = operand(2, n, k, cuda_device)
        plan = scaled.CudaScaledMatmulPlan(name="t", n=n, k=k, output_dtype="f32")
        executable = plan.build(cuda_device)
        first = plan.invoke(executable, lhs, lhs_scales, rhs, rhs_scales)
        for _ in range(5):
            assert torch.equal(plan.invoke(executable, lhs, lhs_scales, rhs, rhs_scales), first)
        executable.close()


def test_entry_points_refuse_what_tensor_maps_cannot_hold(cuda_device):
    lhs, lhs_scales = operand(1, 4, 256, cuda_device)
    plan = scaled.CudaScaledMatmulPlan(name="t", n=4, k=256)
    executable = plan.build(cuda_device)
    packed = torch.zeros(4 * 260 + 16, dtype=torch.uint8, device=cuda_device)
    bad_pitch = packed[: 4 * 260].view(4, 260)[:, :256].view(torch.float8_e4m3fn)
    bad_base = packed[8 : 8 + 4 * 256].view(4, 256).view(torch.float8_e4m3fn)
    from tpu_cake_b200 import _native

    with pytest.raises(_native.CakeError, match="multiples of 16"):
        plan.invoke(executable, bad_pitch, lhs_scales, lhs, lhs_scales)
    with pytest.raises(_native.CakeError, match="16-byte aligned"):
        plan.invoke(executable, lhs, lhs_scales, bad_base, lhs_scales)
    with pytest.raises(ValueError, match="must be on"):
        plan.invoke(executable, lhs.cpu(), lhs_scales, lhs, lhs_scales)


@pytest.mark.parametrize("rows", [3, 200])
def test_mlp_plan_gives_what_its_calls_give(cuda_device, rows):
    mlp = Mlp(cuda_device, 640, 1000)
    x, residual = activations(1, rows, 640, "bf16", cuda_device), activations(2, rows, 640, "bf16", cuda_device)
    plan = scaled.CudaScaledMlpPlan(name="layer", hidden=640, inner=1000)
    executable = plan.build(cuda_device)
    weights = plan.quantize_weights(executable, mlp.norm_weight, mlp.up, mlp.down)
    out, summed = plan.invoke(executable, weights, x, residual)
    want, want_residual = mlp(x, residual.clone())
    assert executable.status() == (0, 0, 0, 0)
    assert torch.equal(out, want) and torch.equal(summed, want_residual)
    executable.close()


def test_run_scaled_mlp_writes_a_bundle(cuda_device, tmp_path):
    import json

    from tpu_cake_b200 import cli

    assert cli.main(["run-scaled-mlp", str(tmp_path / "out"), "--rows", "33", "--hidden", "520", "--inner", "776", "--measured-iterations", "3"]) == 0
    result = json.loads((tmp_path / "out" / "result.json").read_text())
    assert result["passed"] and result["median_ns"] > 0 and max(result["share_of_bound"].values()) <= 1
    assert {a["role"] for a in result["artifacts"]} >= {"contract", "lowered_source", "correctness", "execution_ledger", "source_state"}
    with pytest.raises(FileExistsError):
        cli.main(["run-scaled-mlp", str(tmp_path / "out")])


# ------------------------------------------------------------------------------------------ far apart, first calls


def test_rows_more_than_32_bits_apart(cuda_device):
    """Row strides of 2^31 + 8 elements: the third row starts beyond 2^32 elements (8 GiB)."""
    stride = (1 << 31) + 8
    held = torch.empty(2 * stride + 512, dtype=torch.bfloat16, device=cuda_device)
    x = held.as_strided((3, 512), (stride, 1))
    x.copy_(activations(1, 3, 512, "bf16", cuda_device))
    expected = oracle.quantize(numpy64(x))
    plan = scaled.CudaQuantizeRowsPlan(name="t", columns=512)
    codes, scales = plan.invoke(plan.build(cuda_device), x)
    assert np.array_equal(numpy64(codes), expected[0]) and np.array_equal(scale_values(scales), expected[1])
    norm = scaled.CudaRmsNormQuantizePlan(name="t", columns=512)
    residual = activations(2, 3, 512, "bf16", cuda_device)
    summed = (x.float() + residual.float()).to(torch.bfloat16)
    want, _h = oracle.rms_norm(numpy64(x), np.ones(512), 1e-5, numpy64(residual))
    codes, scales, _ = norm.invoke(norm.build(cuda_device), x, torch.ones(512, dtype=torch.bfloat16, device=cuda_device), residual, residual_out=x)
    check_close(codes, scales, want, NORM_DELTA)
    assert torch.equal(x, summed)


@pytest.mark.parametrize("m, n, k, tile", [(40000, 65540, 130, 0), (40000, 65540, 130, 128), (40000, 65539, 130, 224)])
def test_matmul_outputs_beyond_32_bits(cuda_device, m, n, k, tile):
    """2.6 billion outputs: checked where the last rows and columns lie."""
    lhs, lhs_scales = operand(1, m, k, cuda_device, exact=True)
    rhs, rhs_scales = operand(2, n, k, cuda_device, exact=True)
    plan = scaled.CudaScaledMatmulPlan(name="t", n=n, k=k, tile=tile)
    executable = plan.build(cuda_device)
    out = plan.invoke(executable, lhs, lhs_scales, rhs, rhs_scales)
    assert executable.status() == (0, 0, 0, 0)
    for rows in (slice(0, 8), slice(32760, 32776), slice(m - 40, m)):
        expected = oracle.matmul(numpy64(lhs[rows]), scale_values(lhs_scales[rows]), numpy64(rhs), scale_values(rhs_scales))
        assert torch.equal(out[rows].cpu(), torch.from_numpy(expected).to(torch.bfloat16))


FIRST_CALL_IN_A_CAPTURE = """
import sys, torch
sys.path.insert(0, {root!r})
import __graft_entry__
__graft_entry__.load_package()
from tpu_cake_b200 import scaled_cuda_lowering as scaled
device = torch.device("cuda", 0)
x = torch.randn(300, 512, device=device).to(torch.bfloat16)
w = torch.randn({n}, 512, device=device).to(torch.bfloat16)
quantize = scaled.CudaQuantizeRowsPlan(name="t", columns=512)
matmul = scaled.CudaScaledMatmulPlan(name="t", n={n}, k=512)
rows, product = quantize.build(device), matmul.build(device)
def layer():
    return matmul.invoke(product, *quantize.invoke(rows, x), *quantize.invoke(rows, w))
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = layer()
graph.replay()
torch.cuda.synchronize()
assert torch.equal(out, layer()) and product.status() == (0, 0, 0, 0)
x.mul_(2)
graph.replay()
torch.cuda.synchronize()
assert torch.equal(out, layer())
"""


@pytest.mark.parametrize("n", [64, 20000])
def test_the_first_call_of_a_process_may_be_captured(cuda_device, n):
    import subprocess
    import sys
    from pathlib import Path

    root = str(Path(__file__).resolve().parent.parent)
    done = subprocess.run([sys.executable, "-c", FIRST_CALL_IN_A_CAPTURE.format(root=root, n=n)], capture_output=True, text=True, timeout=180, check=False)
    assert done.returncode == 0, done.stderr[-2000:]


def test_calls_on_two_streams_overlap(cuda_device):
    """Wide and narrow matmuls and row kernels of two streams at once, many times: no call sees another."""
    streams = [torch.cuda.Stream(cuda_device) for _ in range(3)]
    work = []
    for i, (m, n, k) in enumerate(((300, 2048, 1024), (5, 4096, 2048), (70, 1000, 1500))):
        x = activations(i, m, k, "bf16", cuda_device)
        w = activations(10 + i, n, k, "bf16", cuda_device)
        quantize, matmul = scaled.CudaQuantizeRowsPlan(name="t", columns=k), scaled.CudaScaledMatmulPlan(name="t", n=n, k=k, output_dtype="f32")
        rows, product = quantize.build(cuda_device), matmul.build(cuda_device)
        weights = quantize.invoke(rows, w)
        work.append((matmul, product, quantize, rows, x, weights, matmul.invoke(product, *quantize.invoke(rows, x), *weights)))
    torch.cuda.synchronize(cuda_device)
    results = [[] for _ in work]
    for _ in range(20):
        for stream, (matmul, product, quantize, rows, x, weights, _want), got in zip(streams, work, results, strict=True):
            with torch.cuda.stream(stream):
                got.append(matmul.invoke(product, *quantize.invoke(rows, x), *weights))
    torch.cuda.synchronize(cuda_device)
    for (_m, product, _q, _r, _x, _w, want), got in zip(work, results, strict=True):
        assert product.status() == (0, 0, 0, 0) and all(torch.equal(g, want) for g in got)


def test_invoke_refuses_wrong_operands(cuda_device):
    plan = scaled.CudaQuantizeRowsPlan(name="p", columns=100)
    executable = plan.build(cuda_device)
    x, weight = torch.zeros(4, 100, dtype=torch.bfloat16, device=cuda_device), torch.ones(100, dtype=torch.bfloat16, device=cuda_device)
    for wrong in (x.float(), x[:, :99], x[0], x.t(), torch.zeros(4, 200, dtype=torch.bfloat16, device=cuda_device)[:, ::2], x[:1].expand(4, 100), None, x.cpu()):
        with pytest.raises(ValueError, match="x must"):
            plan.invoke(executable, wrong)
    with pytest.raises(ValueError, match="codes must"):
        plan.invoke(executable, x, codes=torch.zeros(3, 100, device=cuda_device).to(torch.float8_e4m3fn))
    with pytest.raises(ValueError, match="scales must"):
        plan.invoke(executable, x, scales=torch.ones(4, 2, device=cuda_device).to(torch.float8_e8m0fnu))
    with pytest.raises(ValueError, match="x must"):
        scaled.CudaQuantizeRowsPlan(name="p", columns=100, gate="silu").invoke(executable, x)
    norm = scaled.CudaRmsNormQuantizePlan(name="p", columns=100)
    for wrong in (weight.float(), weight[:99], torch.ones(200, dtype=torch.bfloat16, device=cuda_device)[::2], weight.cpu(), None):
        with pytest.raises(ValueError, match="weight must"):
            norm.invoke(executable, x, wrong, x)
    with pytest.raises(ValueError, match="residual must"):
        norm.invoke(executable, x, weight, x[:3])
    with pytest.raises(ValueError, match="residual_out must"):
        norm.invoke(executable, x, weight, x, residual_out=x.float())
    matmul = scaled.CudaScaledMatmulPlan(name="p", n=32, k=256)
    product = matmul.build(cuda_device)
    lhs, lhs_scales = operand(1, 4, 256, cuda_device)
    rhs, rhs_scales = operand(2, 32, 256, cuda_device)
    for wrong in ((lhs[:, :255], lhs_scales, rhs, rhs_scales), (lhs, lhs_scales[:3], rhs, rhs_scales), (lhs, lhs_scales, rhs[:31], rhs_scales[:31]),
                  (lhs, lhs_scales, rhs, rhs_scales[:, :1]), (lhs.view(torch.float8_e5m2), lhs_scales, rhs, rhs_scales),
                  (lhs, lhs_scales.view(torch.uint8), rhs, rhs_scales), (lhs, lhs_scales.cpu(), rhs, rhs_scales)):
        with pytest.raises(ValueError):
            matmul.invoke(product, *wrong)
    with pytest.raises(ValueError, match="out must"):
        matmul.invoke(product, lhs, lhs_scales, rhs, rhs_scales, out=torch.zeros(4, 32, device=cuda_device))


@pytest.mark.parametrize("tile, k_split", [(0, 0), (16, 1), (256, 0)])
def test_matmul_longest_contraction(cuda_device, tile, k_split):
    """2^27 - 1 codes a row, zero but for the first and the last of them: sums of 600 exact products."""
    k = (1 << 27) - 1
    sides = []
    for seed, rows in ((1, 1), (2, 2)):
        generator = torch.Generator().manual_seed(seed)
        codes = torch.zeros(rows, -(-k // 16) * 16, dtype=torch.uint8, device=cuda_device).view(torch.float8_e4m3fn)[:, :k]
        scales = torch.full((rows, -(-k // 128)), 126, dtype=torch.uint8, device=cuda_device).view(torch.float8_e8m0fnu)
        values = torch.randint(-3, 4, (rows, 600), generator=generator).float()
        codes[:, :300], codes[:, -300:] = values[:, :300].to(cuda_device).to(torch.float8_e4m3fn), values[:, 300:].to(cuda_device).to(torch.float8_e4m3fn)
        sides.append((codes, scales, values))
    expected = sides[0][2] @ sides[1][2].t() * 0.25
    plan = scaled.CudaScaledMatmulPlan(name="t", n=2, k=k, output_dtype="f32", tile=tile, k_split=k_split)
    executable = plan.build(cuda_device)
    out = plan.invoke(executable, *sides[0][:2], *sides[1][:2])
    assert executable.status() == (0, 0, 0, 0)
    assert torch.equal(out.cpu(), expected)
