"""The 8-bit gated MLP layer as a run bundle: seeded inputs, a correctness gate on every call of the layer,
then timed calls. ``cli run-scaled-mlp``.

The reference has no 8-bit path; the bundle and its ledger are those of its matmul run
(src/tpu_cake/runner.py:486-559: single-use directory, CREATED ... TIMED, REJECTED on a numerical
mismatch, device synchronised after every call, median). The gate computes each call's definition in
float64 from the inputs that the call itself had, so that no call hides behind another's rounding:

  codes and scales   |code * scale - v| <= half a step of e4m3, v moved by its own f32 arithmetic (2^-18)
  matmul             k 2^-24 sum |lhs| |rhs| for the f32 accumulation, 2^-8 |out| for the rounding to bf16
"""

from __future__ import annotations

import json
import math
import statistics
import time
from dataclasses import asdict
from pathlib import Path

import torch

from . import run_artifacts
from . import scaled_cuda_lowering as scaled
from .identity import semantic_sha256
from .run_ledger import RunLedger, RunState

SEED = 97
CHECKED_ROWS = 256
F32_ARITHMETIC = 2.0**-18


def _inputs(rows: int, hidden: int, inner: int, device: torch.device) -> dict[str, torch.Tensor]:
    generator = torch.Generator().manual_seed(SEED)

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=generator) * scale).to(torch.bfloat16).to(device)

    return {"x": normal(rows, hidden), "residual": normal(rows, hidden), "norm": normal(hidden, scale=0.1) + 1,
            "up": normal(2 * inner, hidden, scale=hidden**-0.5), "down": normal(hidden, inner, scale=inner**-0.5)}


def _values(codes: torch.Tensor, scales: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(code * scale, scale per element) in float64."""
    spread = torch.exp2(scales.view(torch.uint8).double() - 127).repeat_interleave(scaled.GROUP_COLUMNS, dim=1)[:, : codes.shape[1]]
    return codes.double() * spread, spread


def _check_codes(codes, scales, expected: torch.Tensor) -> float:
    """The largest error as a share of what is allowed."""
    got, spread = _values(codes, scales)
    allowed = (2.0**-4 * (1 + F32_ARITHMETIC) + F32_ARITHMETIC) * expected.abs() + 2.0**-10 * spread
    return float(((got - expected).abs() / allowed).max())


def _check_matmul(out, lhs: torch.Tensor, rhs: torch.Tensor) -> float:
    expected = lhs @ rhs.t()
    allowed = 2.0**-8 * expected.abs() + rhs.shape[1] * 2.0**-24 * (1 + 2.0**-8) * (lhs.abs() @ rhs.abs().t())
    return float(((out.double() - expected).abs() / allowed.clamp(min=1e-300)).max())


def check_layer(plan: scaled.CudaScaledMlpPlan, executable, weights: scaled.ScaledMlpWeights, x, residual) -> dict[str, float]:
    """Every call of the layer against its definition: the largest error of each as a share of its bound."""
    codes, scales, summed = plan.norm.invoke(executable.rows, x, weights.norm, residual)
    h = x.double() + residual.double()
    shares = {"norm": _check_codes(codes, scales, h / torch.sqrt(h.square().mean(dim=1, keepdim=True) + plan.epsilon) * weights.norm.double()),
              "residual": float(((summed.double() - h).abs() / (2.0**-8 * h.abs()).clamp(min=1e-300)).max())}
    projected = plan.up.invoke(executable.up, codes, scales, *weights.up)
    shares["up"] = _check_matmul(projected, _values(codes, scales)[0], _values(*weights.up)[0])
    codes, scales = plan.gate.invoke(executable.rows, projected)
    gate, up = projected.double().split(plan.inner, dim=1)
    shares["gate"] = _check_codes(codes, scales, gate * torch.sigmoid(gate) * up)
    out = plan.down.invoke(executable.down, codes, scales, *weights.down)
    shares["down"] = _check_matmul(out, _values(codes, scales)[0], _values(*weights.down)[0])
    executable.status()
    return shares


def run_scaled_mlp(output_dir: Path, *, rows: int, hidden: int, inner: int, warmup_iterations: int = 3, measured_iterations: int = 10) -> dict:
    """Runs the layer and writes its bundle under ``output_dir``, which must not exist. Raises when a call
    misses its bound; the bundle's ledger then ends in REJECTED."""
    if min(rows, hidden, inner, measured_iterations) < 1 or warmup_iterations < 0:
        raise ValueError("rows, hidden, inner and measured iterations must be positive")
    plan = scaled.CudaScaledMlpPlan(name="scaled-mlp", hidden=hidden, inner=inner)
    if not torch.cuda.is_available():
        raise RuntimeError("the 8-bit MLP layer needs a CUDA device: the CUDA backend has no CPU fallback")
    device = torch.device("cuda", torch.cuda.current_device())
    output_dir = Path(output_dir)
    output_dir.mkdir(parents=True, exist_ok=False)
    artifacts: list[run_artifacts.ArtifactReference] = []
    contract = {"workload": "scaled-mlp", "rows": rows, "hidden": hidden, "inner": inner, "seed": SEED, "epsilon": plan.epsilon,
                "warmup_iterations": warmup_iterations, "measured_iterations": measured_iterations, "source_sha256": plan.source_sha256()}
    run_id = semantic_sha256("scaled-mlp-run", json.dumps(contract, sort_keys=True))
    run_artifacts.write_json(output_dir, output_dir / "contract.json", contract, "contract", artifacts)
    run_artifacts.source_state(output_dir, artifacts)
    run_artifacts.write_text(output_dir, output_dir / "lowered_cuda.py", plan.render_executable_source(), "lowered_source", artifacts)
    with RunLedger(output_dir / "ledger.sqlite") as ledger:
        ledger.create(run_id, contract)
        ledger.transition(run_id, RunState.VERIFIED, {"source_sha256": plan.source_sha256()})
        ledger.transition(run_id, RunState.LOWERED, {"kernels": ["cake_rms_norm_quantize_sm100", "cake_scaled_matmul_sm100", "cake_quantize_rows_sm100"]})
        executable = plan.build(device)
        inputs = _inputs(rows, hidden, inner, device)
        weights = plan.quantize_weights(executable, inputs["norm"], inputs["up"], inputs["down"])
        ledger.transition(run_id, RunState.COMPILED, {"device_kind": torch.cuda.get_device_name(device)})

        # Rows are independent: the gate takes the first of them.
        checked = min(rows, CHECKED_ROWS)
        shares = check_layer(plan, executable, weights, inputs["x"][:checked], inputs["residual"][:checked])
        shares["up weights"] = _check_codes(*weights.up, inputs["up"].double())
        shares["down weights"] = _check_codes(*weights.down, inputs["down"].double())
        run_artifacts.write_json(output_dir, output_dir / "correctness.json", {"checked_rows": checked, "share_of_bound": shares}, "correctness", artifacts)
        if not all(math.isfinite(s) and s <= 1 for s in shares.values()):
            ledger.transition(run_id, RunState.REJECTED, {"reason": "numerical mismatch", "share_of_bound": shares})
            raise ValueError(f"SCALED_MLP_CORRECTNESS_FAILED share_of_bound={shares}")
        ledger.transition(run_id, RunState.CORRECT, {"share_of_bound": shares})

        samples = []
        for iteration in range(warmup_iterations + measured_iterations):
            started = time.perf_counter_ns()
            plan.invoke(executable, weights, inputs["x"], inputs["residual"])
            torch.cuda.synchronize(device)
            if iteration >= warmup_iterations:
                samples.append(time.perf_counter_ns() - started)
        executable.status()
        result = {"run_id": run_id, **contract, "passed": True, "share_of_bound": shares, "samples_ns": samples,
                  "median_ns": float(statistics.median(samples)), "flops": 6 * rows * hidden * inner}
        ledger.transition(run_id, RunState.TIMED, {"median_ns": result["median_ns"]})
    artifacts.append(run_artifacts.reference_of(output_dir, output_dir / "ledger.sqlite", "execution_ledger"))
    result["artifacts"] = [asdict(a) for a in artifacts]
    (output_dir / "result.json").write_text(json.dumps(result, indent=2, sort_keys=True) + "\n")
    return result
