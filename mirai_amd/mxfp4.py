"""MXFP4 tensors: OCP microscaled 4-bit floats, quantised and read back on the GPU.

Blocks of 32 elements along the last axis share one power of two X =
2^clamp(floor(log2 max|x|) - 2, -127, 125); an element is x / X rounded to nearest
(ties to even) on 0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives, what lies above 6
to 6. A block that holds a NaN or an infinity reads back as NaN.

Expert weights take this form with ``quant_format="mxfp4"``, the rows of
``CompressedGroupedExperts.grouped_linear`` with ``activations="mxfp4"``.
"""

from __future__ import annotations

import math
from dataclasses import dataclass

import torch

from . import _native as nat

MX_BLOCK = 32


@dataclass
class MXFP4Tensor:
    """codes uint8 [..., 16 B], scales uint8 [..., B] of a [..., cols] tensor with
    B = ceil(cols / 32) blocks a row: element 2 i of a row in the low nibble of its
    byte i (sign, 2 exponent bits, 1 fraction bit; zeros past cols), the scale byte
    log2 X + 127, or 255 for a block of NaN."""

    codes: torch.Tensor
    scales: torch.Tensor
    cols: int

    @property
    def shape(self) -> tuple[int, ...]:
        return (*self.codes.shape[:-1], self.cols)

    def nbytes(self) -> int:
        return self.codes.numel() + self.scales.numel()


def mxfp4_quantize(x: torch.Tensor) -> MXFP4Tensor:
    """x [..., cols] (any floating type; bf16 and fp32 are read as they are, others
    as fp32) in MXFP4. Rows may lie any distance apart. Carries no gradient."""
    shape = x.shape
    if len(shape) < 1 or shape[-1] < 1:
        raise ValueError(f"mxfp4_quantize takes [..., cols] with cols >= 1, got {tuple(shape)}.")
    if not x.is_floating_point():
        raise ValueError(f"mxfp4_quantize takes a floating-point tensor, got {x.dtype}.")
    device = nat.require_gpu(x)
    if x.dtype not in (torch.bfloat16, torch.float32):
        x = x.detach().float()
    *lead, cols = shape
    if x.is_contiguous():
        flat, rows, ldx = x, math.prod(lead), cols
    else:
        # A view where the rows are evenly spaced, else a copy.
        flat = x.detach().reshape(-1, cols)
        if flat.stride(1) != 1 or flat.stride(0) < cols:
            flat = flat.contiguous()
        rows, ldx = flat.shape[0], max(flat.stride(0), cols)
    blocks = -(-cols // MX_BLOCK)
    codes = torch.empty((*lead, 16 * blocks), dtype=torch.uint8, device=device)
    scales = torch.empty((*lead, blocks), dtype=torch.uint8, device=device)
    with nat.on_device(device):
        nat.call("mx_mxfp4_quantize", flat.data_ptr(), nat.dtype_code(flat.dtype), rows, cols, ldx,
                 codes.data_ptr(), scales.data_ptr(), nat.stream(device))
    return MXFP4Tensor(codes, scales, cols)


def mxfp4_dequantize(q: MXFP4Tensor, *, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The [..., cols] values ``q`` stands for, in bf16 or fp32 (both hold them
    exactly, but for scales above 2^125, which only other quantisers produce)."""
    cols, blocks = int(q.cols), -(-int(q.cols) // MX_BLOCK)
    lead = q.codes.shape[:-1]
    if (cols < 1 or q.codes.dtype != torch.uint8 or q.scales.dtype != torch.uint8
            or q.codes.shape != (*lead, 16 * blocks) or q.scales.shape != (*lead, blocks)):
        raise ValueError(f"an MXFP4 tensor of {cols} columns holds uint8 codes [..., {16 * blocks}] "
                         f"and scales [..., {blocks}], got {tuple(q.codes.shape)} "
                         f"{q.codes.dtype} and {tuple(q.scales.shape)} {q.scales.dtype}.")
    code = nat.dtype_code(dtype)
    device = nat.require_gpu(q.codes, q.scales)
    codes, scales = q.codes.contiguous(), q.scales.contiguous()
    if codes.data_ptr() % 4:
        codes = codes.clone()
    out = torch.empty((*lead, cols), dtype=dtype, device=device)
    rows = math.prod(lead)
    with nat.on_device(device):
        nat.call("mx_mxfp4_dequantize", codes.data_ptr(), scales.data_ptr(), rows, cols,
                 out.data_ptr(), code, nat.stream(device))
    return out
