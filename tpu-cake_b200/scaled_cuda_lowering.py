"""CUDA backend plans of the 8-bit linear layer: row quantisation, RMS norm with 8-bit output, and the
block-scaled matmul that takes both.

The reference has one matmul, in bf16 (src/tpu_cake/pallas_lowering.py:44-50); ``CudaScaledMatmulPlan``
is its local contraction at half the bytes and twice the tensor rate, and the two row plans make its
operands. Operands are pairs (codes, scales): codes ``torch.float8_e4m3fn`` [rows, columns] with
contiguous rows whose pitch is a multiple of 16 bytes, scales ``torch.float8_e8m0fnu``
[rows, ceil(columns / 128)], one power of two per 128 consecutive columns of a row:

  scale   the least 2^e >= 2^-127 with max |v| <= 448 * 2^e over the group; 1 for a group of zeros; NaN
          for a group that holds an infinity or a NaN, whose codes are then NaN throughout
  code    v / scale rounded to nearest even

Plans are built for a width and a type and serve any number of rows, zero included. Calls are
asynchronous on the device's current stream, allocate their outputs from torch unless they are given,
use no workspace and keep nothing between calls, so they can be captured into CUDA graphs.
"""

from __future__ import annotations

import ctypes
from dataclasses import dataclass
from functools import cached_property

import torch

from . import _native
from .identity import text_sha256

GROUP_COLUMNS = 128
CODE_DTYPE = torch.float8_e4m3fn
SCALE_DTYPE = torch.float8_e8m0fnu
MAX_NORM_COLUMNS = 32768
_CAKE_DTYPES = {"bf16": _native.CAKE_DTYPE_BF16, "f16": _native.CAKE_DTYPE_F16, "f32": _native.CAKE_DTYPE_F32}
_GATES = {"none": _native.CAKE_GATE_NONE, "silu": _native.CAKE_GATE_SILU}


def scale_columns(columns: int) -> int:
    """Scales of a row of ``columns`` codes."""
    return -(-columns // GROUP_COLUMNS)


def empty_codes(rows: int, columns: int, device: torch.device) -> torch.Tensor:
    """Uninitialised codes with a row pitch of whole 128-byte lines: the matmul takes multiples of 16 bytes,
    but its 128-byte reads of a row then touch two lines each (1001 x 5000 x 4096: 32 us against 26)."""
    if columns % 128 == 0:
        return torch.empty(rows, columns, dtype=CODE_DTYPE, device=device)
    return torch.empty(rows, -(-columns // 128) * 128, dtype=CODE_DTYPE, device=device)[:, :columns]


def empty_scales(rows: int, columns: int, device: torch.device) -> torch.Tensor:
    return torch.empty(rows, -(-columns // GROUP_COLUMNS), dtype=SCALE_DTYPE, device=device)


class RowQuantizeExecutable:
    """What a plan runs on: a device and the compiled binding. The row kernels keep nothing else."""

    def __init__(self, device: torch.device):
        self.binding = _native.load_torch_binding()
        self.index = torch.cuda.current_device() if device.index is None else device.index
        self.device = torch.device("cuda", self.index)

    def close(self) -> None:
        """Nothing to release: here for the executables' common surface."""


class ScaledMatmulExecutable(RowQuantizeExecutable):
    """A matmul plan's descriptor and its status word on a GPU."""

    def __init__(self, plan: "CudaScaledMatmulPlan", desc: _native.ScaledMatmulDesc, device: torch.device):
        super().__init__(device)
        self.plan = plan
        self._desc = desc
        self.desc_address = ctypes.addressof(desc)
        self._status = torch.zeros(4, dtype=torch.int32).to(self.device)  # there when the copy returns, for any stream
        self.status_address = self._status.data_ptr()

    def status(self) -> tuple[int, int, int, int]:
        """Waits for the current stream's work and reads the status word; raises if a bounded wait ran out."""
        code, *details = self._status.tolist()
        if code:
            self._status.zero_()
            raise _native.CakeError(_native.CAKE_ERR_TIMEOUT, "device-side bounded wait ran out: block={} tile={} where={}".format(*details))
        return (code, *details)


def _outputs(result):
    """A binding call's outputs; its error code raises."""
    if type(result) is int:
        _native.check(result)
    return result


def _source(kind: str, kernel: str, plan, fields: tuple[str, ...]) -> str:
    lines = [f"# cake-b200 lowered {kind}", f"name = {plan.name!r}", f"kernel = {kernel!r}"]
    lines += [f"{field} = {getattr(plan, field)!r}" for field in fields]
    return "\n".join([*lines, f"group_columns = {GROUP_COLUMNS}", "codes = 'e4m3'", "scales = 'e8m0'", "abi_version = 1"]) + "\n"


def _device(device: torch.device | None) -> torch.device:
    return device or torch.device("cuda", torch.cuda.current_device())


@dataclass(frozen=True)
class CudaQuantizeRowsPlan:
    """codes, scales of ``x`` [rows, columns], or with ``gate="silu"`` of silu(gate) * up with ``x`` =
    [rows, gate | up] (2 * columns wide), computed in f32."""

    name: str
    columns: int
    input_dtype: str = "bf16"
    gate: str = "none"

    def __post_init__(self) -> None:
        if self.columns < 1:
            raise ValueError(f"columns must be positive, got {self.columns}")
        if self.input_dtype not in _CAKE_DTYPES:
            raise ValueError(f"input dtype must be one of {tuple(_CAKE_DTYPES)}, got {self.input_dtype}")
        if self.gate not in _GATES:
            raise ValueError(f"gate must be one of {tuple(_GATES)}, got {self.gate}")

    def render_executable_source(self) -> str:
        return _source("row quantisation", "cake_quantize_rows_sm100", self, ("columns", "input_dtype", "gate"))

    def source_sha256(self) -> str:
        return text_sha256(self.render_executable_source())

    def build(self, device: torch.device | None = None) -> RowQuantizeExecutable:
        return RowQuantizeExecutable(_device(device))

    def invoke(self, executable: RowQuantizeExecutable, x, *, codes=None, scales=None) -> tuple[torch.Tensor, torch.Tensor]:
        return _outputs(executable.binding.quantize_rows(executable.index, x, self.columns, _CAKE_DTYPES[self.input_dtype], _GATES[self.gate], codes, scales))


@dataclass(frozen=True)
class CudaRmsNormQuantizePlan:
    """codes, scales of h / sqrt(mean(h^2) + epsilon) * weight with h = x + residual (or x alone), all in
    f32, and h rounded to the input type as the next layer's residual."""

    name: str
    columns: int
    input_dtype: str = "bf16"
    weight_dtype: str = "bf16"
    epsilon: float = 1e-5
    with_residual: bool = True

    def __post_init__(self) -> None:
        if not 1 <= self.columns <= MAX_NORM_COLUMNS:
            raise ValueError(f"a norm's row is held on chip: columns must be 1 to {MAX_NORM_COLUMNS}, got {self.columns}")
        if self.input_dtype not in _CAKE_DTYPES:
            raise ValueError(f"input dtype must be one of {tuple(_CAKE_DTYPES)}, got {self.input_dtype}")
        if self.weight_dtype not in (self.input_dtype, "f32"):
            raise ValueError(f"weight dtype must be the input's or f32, got {self.weight_dtype}")
        if not self.epsilon >= 0:
            raise ValueError(f"epsilon must not be negative, got {self.epsilon}")

    def render_executable_source(self) -> str:
        return _source("RMS norm with 8-bit output", "cake_rms_norm_quantize_sm100", self,
                       ("columns", "input_dtype", "weight_dtype", "epsilon", "with_residual"))

    def source_sha256(self) -> str:
        return text_sha256(self.render_executable_source())

    def build(self, device: torch.device | None = None) -> RowQuantizeExecutable:
        return RowQuantizeExecutable(_device(device))

    def invoke(self, executable: RowQuantizeExecutable, x, weight, residual=None, *, codes=None, scales=None, residual_out=None):
        """Returns (codes, scales, new residual or None). ``residual_out`` may be ``residual`` or ``x``."""
        if (residual is not None) != self.with_residual:
            raise ValueError("residual must be given to a plan with residual, and to no other")
        if residual is None and residual_out is not None:
            raise ValueError("residual_out needs a plan with residual")
        return _outputs(executable.binding.rms_norm_quantize(executable.index, x, self.columns, _CAKE_DTYPES[self.input_dtype], weight,
                                                             _CAKE_DTYPES[self.weight_dtype], self.epsilon, residual, codes, scales, residual_out))


@dataclass(frozen=True)
class CudaScaledMatmulPlan:
    """out [m, n] = lhs [m, k] rhs [n, k]^T over dequantised operands, accumulated in f32 and rounded once
    to ``output_dtype``. ``tile`` and ``k_split`` override the library's choice (0): tiles of 16, 32, 64 or
    128 tokens by 128 columns with 1 to 8 blocks sharing a tile's contraction, or of 256 tokens by 192,
    224 or 256 columns. Runs on one mesh position."""

    name: str
    n: int
    k: int
    output_dtype: str = "bf16"
    tile: int = 0
    k_split: int = 0

    def __post_init__(self) -> None:
        if not (0 < self.n < 1 << 30 and 0 < self.k < 1 << 27):
            raise ValueError(f"scaled matmul extents must be n = 1 to 2^30 - 1 and k = 1 to 2^27 - 1, got n={self.n} k={self.k}")
        if self.output_dtype not in ("bf16", "f32"):
            raise ValueError(f"output dtype must be f32 or bf16, got {self.output_dtype}")
        if self.tile not in (0, 16, 32, 64, 128, 192, 224, 256):
            raise ValueError(f"tile must be 0, 16, 32, 64, 128, 192, 224 or 256, got {self.tile}")
        if not 0 <= self.k_split <= 8 or (self.k_split > 1 and self.tile not in (16, 32, 64, 128)):
            raise ValueError(f"k_split must be 0 to 8, and above 1 only with tile 16, 32, 64 or 128, got {self.k_split}")

    def render_executable_source(self) -> str:
        return _source("block-scaled matmul", "cake_scaled_matmul_sm100", self, ("n", "k", "output_dtype", "tile", "k_split"))

    def source_sha256(self) -> str:
        return text_sha256(self.render_executable_source())

    def build(self, device: torch.device | None = None) -> ScaledMatmulExecutable:
        desc = _native.ScaledMatmulDesc(n=self.n, k=self.k, out_dtype=_CAKE_DTYPES[self.output_dtype], tile=self.tile, k_split=self.k_split)
        return ScaledMatmulExecutable(self, desc, _device(device))

    def invoke(self, executable: ScaledMatmulExecutable, lhs, lhs_scales, rhs, rhs_scales, *, out=None) -> torch.Tensor:
        if executable.plan is not self and executable.plan != self:
            raise ValueError(f"the executable was built from another plan: {executable.plan}")
        return _outputs(executable.binding.scaled_matmul(executable.index, executable.desc_address, executable.status_address,
                                                         lhs, lhs_scales, rhs, rhs_scales, out))


@dataclass(frozen=True)
class ScaledMlpWeights:
    """A layer's parameters as the kernels take them: the norm's vector and the two projections as (codes, scales)."""

    norm: torch.Tensor
    up: tuple[torch.Tensor, torch.Tensor]    # [2 * inner, hidden]: gate rows, then up rows
    down: tuple[torch.Tensor, torch.Tensor]  # [hidden, inner]


class ScaledMlpExecutable:
    """The executables of a layer's four calls on one GPU."""

    def __init__(self, plan: "CudaScaledMlpPlan", device: torch.device):
        self.rows = plan.norm.build(device)
        self.up = plan.up.build(device)
        self.down = plan.down.build(device)
        self.device = self.rows.device

    def status(self) -> tuple[int, int, int, int]:
        """Raises if a matmul's bounded wait ran out."""
        self.up.status()
        return self.down.status()

    def close(self) -> None:
        """Nothing to release: here for the executables' common surface."""


@dataclass(frozen=True)
class CudaScaledMlpPlan:
    """The 8-bit gated MLP of a decoder layer, four calls: residual addition, norm and quantisation; the gate
    and up projection; silu(gate) * up and quantisation; the down projection."""

    name: str
    hidden: int
    inner: int
    epsilon: float = 1e-5

    def __post_init__(self) -> None:
        self.norm, self.up, self.gate, self.down  # their own checks

    @cached_property
    def norm(self) -> CudaRmsNormQuantizePlan:
        return CudaRmsNormQuantizePlan(name=f"{self.name}-norm", columns=self.hidden, epsilon=self.epsilon)

    @cached_property
    def up(self) -> CudaScaledMatmulPlan:
        return CudaScaledMatmulPlan(name=f"{self.name}-up", n=2 * self.inner, k=self.hidden)

    @cached_property
    def gate(self) -> CudaQuantizeRowsPlan:
        return CudaQuantizeRowsPlan(name=f"{self.name}-gate", columns=self.inner, gate="silu")

    @cached_property
    def down(self) -> CudaScaledMatmulPlan:
        return CudaScaledMatmulPlan(name=f"{self.name}-down", n=self.hidden, k=self.inner)

    def render_executable_source(self) -> str:
        return "".join(plan.render_executable_source() for plan in (self.norm, self.up, self.gate, self.down))

    def source_sha256(self) -> str:
        return text_sha256(self.render_executable_source())

    def build(self, device: torch.device | None = None) -> ScaledMlpExecutable:
        return ScaledMlpExecutable(self, _device(device))

    def quantize_weights(self, executable: ScaledMlpExecutable, norm, up, down) -> ScaledMlpWeights:
        """bf16 parameters to what ``invoke`` takes, once when a model is loaded: ``up`` [2 * inner, hidden] is
        the gate projection's rows followed by the up projection's, ``down`` [hidden, inner]."""
        if not isinstance(up, torch.Tensor) or not isinstance(down, torch.Tensor) or up.shape != (2 * self.inner, self.hidden) \
                or down.shape != (self.hidden, self.inner):
            raise ValueError(f"up must be [{2 * self.inner}, {self.hidden}] and down [{self.hidden}, {self.inner}]")
        return ScaledMlpWeights(
            norm=norm,
            up=CudaQuantizeRowsPlan(name=f"{self.name}-up-weights", columns=self.hidden).invoke(executable.rows, up),
            down=CudaQuantizeRowsPlan(name=f"{self.name}-down-weights", columns=self.inner).invoke(executable.rows, down),
        )

    def invoke(self, executable: ScaledMlpExecutable, weights: ScaledMlpWeights, x, residual, *, out=None, residual_out=None):
        """(layer output bf16 [rows, hidden], x + residual): bf16 ``x`` and ``residual`` [rows, hidden]."""
        codes, scales, summed = self.norm.invoke(executable.rows, x, weights.norm, residual, residual_out=residual_out)
        projected = self.up.invoke(executable.up, codes, scales, *weights.up)
        return self.down.invoke(executable.down, *self.gate.invoke(executable.rows, projected), *weights.down, out=out), summed
