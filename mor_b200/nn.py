"""Training-loop callers of the fake-quantization operators.

``MoRLinear`` applies the operators to the input, the weight and (optionally) the incoming
gradient of a linear layer, with the straight-through gradients that ``mor_b200.ops``
registers (mor/ops.py:15-156 of the reference), and can emit one log line per quantized
tensor in the format that the reference's log tooling parses
(train_logs/process_example_logs.py:38-72):

    <rank>: Tensor <name> at counter <c> step <s> tensor dimension: <R>x<C>
    global_non_zero: <n> global_error: <e> relative_error: <e / n> histogram [h0, ..., h12]

The histogram counts 128 x 128 blocks by their mean relative error in bins of 0.005 (the
tooling labels bin i with (i + 1) * 0.005 and uses the first twelve); the last bin
collects everything from 0.060 up.  The numbers in the line come from the operator itself
(``global_nnz``, ``global_error``); the histogram is computed from input and output with
ordinary tensor operations and is a logging aid, not part of the bit-exact path.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Callable, List, Optional

import torch
from torch import Tensor

from . import ops

HIST_BINS = 13
HIST_WIDTH = 0.005


@dataclass
class QuantConfig:
    """``kind``: "block" (block scaling, global-mantissa scale by default), "block_delayed" (the same in one
    pass over the tensor, with the tensor amax of the previous call: delayed scaling), "row" (one scale per
    row), "mx" (1 x 32 groups, E8M0 scale, single pass), "mor" (per-block format choice), "none"."""
    kind: str = "block"
    block_rows: int = 128
    block_cols: int = 128
    ss_mode: int = 1
    threshold: float = 0.045
    elem_format: int = 0          # mx: 0 E4M3, 1 E5M2, 3 E2M3
    mor_mode: int = 1             # mor: 1 relative-error criterion, 101 dynamic range
    clamp_threshold: float = 1e-15


@dataclass
class QuantStats:
    meta: Optional[Tensor] = None
    global_amax: Optional[Tensor] = None
    global_nnz: Optional[Tensor] = None
    global_error: Optional[Tensor] = None


def fake_quantize_tensor(t: Tensor, cfg: QuantConfig, state: Optional[dict] = None):
    """Fake-quantizes a tensor of any rank >= 1 (viewed as ``[-1, last]``); returns ``(out, QuantStats)``.
    ``state`` carries the amax from call to call for the "block_delayed" kind (first call: two passes)."""
    if cfg.kind == "none":
        return t, QuantStats()
    x = t.reshape(-1, t.shape[-1])
    if not x.is_contiguous():
        x = x.contiguous()
    r, c = x.shape
    if cfg.kind == "block":
        out, meta, amax, nnz, err = ops.fake_quantize_block_scaling(x, r, c, cfg.block_rows, cfg.block_cols,
                                                                    cfg.threshold, cfg.ss_mode)
        st = QuantStats(meta, amax, nnz, err)
    elif cfg.kind == "block_delayed":
        prev = None if state is None else state.get("amax")
        if prev is None:   # nothing to go by yet: the two-pass form, whose amax seeds the next call
            out, meta, amax, nnz, err = ops.fake_quantize_block_scaling(x, r, c, 128, 128, cfg.threshold, cfg.ss_mode)
        else:
            out, meta, amax, nnz, err = ops.fake_quantize_block_scaling_delayed(x, r, c, 128, 128, cfg.threshold,
                                                                                cfg.ss_mode, prev)
        if state is not None:
            state["amax"] = amax.detach()
        st = QuantStats(meta, amax, nnz, err)
    elif cfg.kind == "row":
        out, meta, amax, nnz, err = ops.fake_quantize_channel_scaling(x, r, c, 1, c, cfg.threshold, cfg.ss_mode)
        st = QuantStats(meta, amax, nnz, err)
    elif cfg.kind == "mx":
        out, _ = ops.fake_quantize_mx(x, r, c, 32, cfg.elem_format, 2)
        st = QuantStats()
    elif cfg.kind == "mor":
        out, meta = ops.fake_quantize(x, r, c, cfg.block_rows, cfg.block_cols, cfg.clamp_threshold, cfg.mor_mode, 1)
        st = QuantStats(meta=meta)
    else:
        raise ValueError(f"unknown quantization kind {cfg.kind!r}")
    return out.reshape(t.shape), st


def block_error_histogram(x: Tensor, out: Tensor, block_rows: int = 128, block_cols: int = 128) -> List[int]:
    """Counts blocks by mean relative error |(out - x) / x| over their non-zero elements, bins of 0.005."""
    x2 = x.reshape(-1, x.shape[-1]).float()
    o2 = out.reshape(-1, out.shape[-1]).float()
    r, c = x2.shape
    br, bc = min(block_rows, r), min(block_cols, c)
    r2, c2 = (r // br) * br, (c // bc) * bc
    x2, o2 = x2[:r2, :c2], o2[:r2, :c2]
    nz = x2 != 0
    rel = torch.where(nz, ((o2 - x2) / torch.where(nz, x2, torch.ones_like(x2))).abs(), torch.zeros_like(x2))
    blocks = lambda a: a.reshape(r2 // br, br, c2 // bc, bc).sum(dim=(1, 3))  # noqa: E731
    mean = blocks(rel) / blocks(nz.float()).clamp(min=1.0)
    idx = (mean / HIST_WIDTH).floor().clamp(0, HIST_BINS - 1).long().flatten()
    return torch.bincount(idx, minlength=HIST_BINS).tolist()


def format_log_line(rank: int, name: str, counter: int, step: int, rows: int, cols: int, global_nnz: int,
                    global_error: float, histogram: List[int]) -> str:
    """One line in the format parsed by train_logs/process_example_logs.py:38-72 (plain decimals only)."""
    rel = global_error / global_nnz if global_nnz else 0.0
    return (f"{rank}: Tensor {name} at counter {counter} step {step} tensor dimension: {rows}x{cols} "
            f"global_non_zero: {global_nnz} global_error: {global_error:.6f} relative_error: {rel:.10f} "
            f"histogram [{', '.join(str(int(h)) for h in histogram)}]")


class TensorLogger:
    """Collects log lines; ``sink`` receives each line (``print`` by default).  Logging synchronises the
    stream (it reads scalars back), so enable it for the steps you want to look at, not for every step."""

    def __init__(self, sink: Callable[[str], None] = print, rank: int = 0, every: int = 1):
        self.sink, self.rank, self.every = sink, rank, max(1, every)
        self.step = 0
        self.counter = 0

    def wants(self) -> bool:
        return self.step % self.every == 0

    def log(self, name: str, x: Tensor, out: Tensor, st: QuantStats, cfg: QuantConfig) -> Optional[str]:
        if st.global_nnz is None or not self.wants():
            return None
        x2 = x.reshape(-1, x.shape[-1])
        line = format_log_line(self.rank, name, self.counter, self.step, x2.shape[0], x2.shape[1],
                               int(st.global_nnz.item()), float(st.global_error.item()),
                               block_error_histogram(x, out, cfg.block_rows, cfg.block_cols))
        self.counter += 1
        self.sink(line)
        return line


class _QuantizeGrad(torch.autograd.Function):
    """Identity in the forward pass; fake-quantizes the gradient that flows back."""

    @staticmethod
    def forward(ctx, x: Tensor, layer: "MoRLinear") -> Tensor:
        ctx.layer = layer
        return x.view_as(x)

    @staticmethod
    def backward(ctx, grad: Tensor):
        layer = ctx.layer
        g = grad.contiguous()
        gq, st = fake_quantize_tensor(g, layer.grad_cfg, layer._state["grad"])
        if layer.logger is not None:
            layer.logger.log(f"{layer.log_name}.grad_output", g, gq, st, layer.grad_cfg)
        return gq, None


class MoRLinear(torch.nn.Linear):
    """``torch.nn.Linear`` whose input, weight and (optionally) output gradient are fake-quantized.

    Tensors must be CUDA bfloat16 (float32 is accepted by the block and row kinds) with dimensions that the
    chosen block shape divides; the matrix product itself is torch's."""

    def __init__(self, in_features: int, out_features: int, bias: bool = True, device=None, dtype=torch.bfloat16,
                 input_cfg: Optional[QuantConfig] = None, weight_cfg: Optional[QuantConfig] = None,
                 grad_cfg: Optional[QuantConfig] = None, logger: Optional[TensorLogger] = None, name: str = "linear"):
        super().__init__(in_features, out_features, bias=bias, device=device, dtype=dtype)
        self.input_cfg = input_cfg or QuantConfig()
        self.weight_cfg = weight_cfg or QuantConfig()
        self.grad_cfg = grad_cfg or QuantConfig(kind="none")
        self.logger = logger
        self.log_name = name
        self._state = {"input": {}, "weight": {}, "grad": {}}   # amax carried between calls (delayed scaling)

    def forward(self, x: Tensor) -> Tensor:
        xq, sx = fake_quantize_tensor(x, self.input_cfg, self._state["input"])
        wq, sw = fake_quantize_tensor(self.weight, self.weight_cfg, self._state["weight"])
        if self.logger is not None:
            self.logger.log(f"{self.log_name}.input", x, xq, sx, self.input_cfg)
            self.logger.log(f"{self.log_name}.weight", self.weight, wq, sw, self.weight_cfg)
        y = torch.nn.functional.linear(xq, wq, self.bias)
        if self.grad_cfg.kind != "none" and torch.is_grad_enabled():
            y = _QuantizeGrad.apply(y, self)
        return y


# --------------------------------------------------------------------------- linear layer on microscaled operands
MX_FORMATS = {"e4m3": 0, "e5m2": 1, "e2m1": 4}
MX_INPUT_TYPES = {"e4m3": (torch.bfloat16,), "e5m2": (torch.bfloat16,), "e2m1": (torch.bfloat16, torch.float32)}   # what is quantised to them


def _mx_quantize(x: Tensor, elem_format: int):
    """Codes and scale bytes of a ``[rows, cols]`` tensor in groups of 32 columns."""
    r, c = x.shape
    return ops.quantize_mx_fp4(x, r, c, 32) if elem_format == 4 else ops.quantize_mx(x, r, c, 32, elem_format, operand=True)


def mx_linear(x: Tensor, weight: Tensor, bias: Optional[Tensor] = None, elem_format: int = 0) -> Tensor:
    """``x @ weight.T + bias`` on microscaled operands: ``x`` ``[..., in]`` and ``weight`` ``[out, in]`` are quantised in
    groups of 32 along ``in`` (a multiple of 32) and multiplied as codes; the result is bfloat16, and so is the bias that is
    added to the sums (one of another type is rounded first).  ``elem_format``: 0 E4M3,
    1 E5M2 (bfloat16 inputs), 4 E2M1 (bfloat16 or float32).  A group that holds an infinity or a NaN counts as NaN in whole,
    in the product and in the gradients.  The gradients are straight-through: those of a linear layer
    fed the quantised values, computed from the codes, which are all that the forward pass keeps of ``x`` and ``weight``
    -- one byte (E2M1: half a byte) and a thirty-second per element in place of two; they have no gradient of their own.
    Each call quantises the weight it is given; for serving see :meth:`MXLinear.pack`.  To dispatch modes, tracing and
    profiles by operator the layer is one operator, ``mor::mx_linear``: what it is made of is called inside."""
    if elem_format not in MX_FORMATS.values():
        raise ValueError(f"elem_format must be one of {sorted(MX_FORMATS.values())}, got {elem_format}")
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"x [..., in] and weight [out, in] expected, got {tuple(x.shape)} and {tuple(weight.shape)}")
    return torch.ops.mor.mx_linear.default(x, weight, bias, elem_format)


class MXLinear(torch.nn.Linear):
    """``torch.nn.Linear`` computed by :func:`mx_linear`; ``elem_format`` "e4m3", "e5m2" (bfloat16) or "e2m1"
    (bfloat16 or float32)."""

    def __init__(self, in_features: int, out_features: int, bias: bool = True, device=None, dtype=torch.bfloat16,
                 elem_format: str = "e4m3"):
        if elem_format not in MX_FORMATS:
            raise ValueError(f"elem_format must be one of {sorted(MX_FORMATS)}, got {elem_format!r}")
        if in_features % 32:
            raise ValueError(f"in_features must be a multiple of 32, got {in_features}")
        if (dtype or torch.get_default_dtype()) not in MX_INPUT_TYPES[elem_format]:
            raise ValueError(f"dtype for {elem_format} must be one of {MX_INPUT_TYPES[elem_format]}, got {dtype or torch.get_default_dtype()}")
        super().__init__(in_features, out_features, bias=bias, device=device, dtype=dtype)
        self.elem_format = elem_format

    def forward(self, x: Tensor) -> Tensor:
        return mx_linear(x, self.weight, self.bias, MX_FORMATS[self.elem_format])

    def pack(self) -> "PackedMXLinear":
        """The layer for serving: its weights quantised once, without the originals."""
        return PackedMXLinear(self)

    def extra_repr(self) -> str:
        return f"{super().extra_repr()}, elem_format={self.elem_format}"


class PackedMXLinear(torch.nn.Module):
    """Forward-only linear layer that holds its weights as codes and scale bytes (made by :meth:`MXLinear.pack`)."""

    def __init__(self, layer: MXLinear):
        super().__init__()
        self.in_features, self.out_features, self.elem_format = layer.in_features, layer.out_features, layer.elem_format
        with torch.no_grad():
            codes, scales = _mx_quantize(layer.weight.detach(), MX_FORMATS[layer.elem_format])
        self.register_buffer("payload", codes.contiguous())
        self.register_buffer("scales", scales.contiguous())
        self.register_buffer("bias", None if layer.bias is None else layer.bias.detach().to(torch.bfloat16, copy=True))

    def forward(self, x: Tensor) -> Tensor:
        return torch.ops.mor.mx_linear_packed.default(x, self.payload, self.scales, self.bias, MX_FORMATS[self.elem_format])
