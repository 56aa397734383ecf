"""Weights of 8 bits: e4m3 numbers with one fp32 scale for each block of 128 x 128, and the product over them.

A matrix entry stands for ``value * scale`` of its block (the layout that 8-bit checkpoints come in: ``weight`` and ``weight_scale_inv``).
``fp8_linear`` rounds its rows to e4m3 too, one scale for each run of 128 of a row, and multiplies on the tensor cores in 8 bits; sums are
fp32.  ``mlp.Fp8GatedMLP`` is the gated feed-forward of such matrices, ``mlp.FewTokenExperts`` takes stacks of them as experts."""

from __future__ import annotations

import torch

from extensions_b200.tiny_llm_ext_b200 import blocks

BLOCK = 128
LARGEST = 448.0  # of the e4m3 numbers


def _blocks(n: int) -> int:
    return -(-n // BLOCK)


class Fp8Weights:
    """``values [.., N, K]`` (``torch.float8_e4m3fn``) and ``scales [.., ceil(N / 128), ceil(K / 128)]`` fp32; leading dimensions are stacks
    of matrices.  Rows are kept in a multiple of 16 bytes: the values are copied once where they are not laid out so."""

    def __init__(self, values: torch.Tensor, scales: torch.Tensor):
        if values.dtype != torch.float8_e4m3fn or values.dim() < 2 or values.numel() == 0:
            raise ValueError("Fp8Weights: values must be float8_e4m3fn [.., outputs, inputs]")
        n, k = values.shape[-2:]
        if scales.dtype != torch.float32 or scales.shape != (*values.shape[:-2], _blocks(n), _blocks(k)):
            raise ValueError(f"Fp8Weights: scales must be float32 {(*values.shape[:-2], _blocks(n), _blocks(k))}, one for each block of {BLOCK}")
        if scales.device != values.device:
            raise ValueError("Fp8Weights: values and scales on two devices")
        self.shape = tuple(values.shape)
        self.scales = scales.contiguous()
        pad = -k % 16
        raw = values.contiguous().view(torch.uint8)
        if pad or raw.data_ptr() % 16:
            wide = torch.zeros((*values.shape[:-1], k + pad), dtype=torch.uint8, device=values.device)
            wide[..., :k] = raw
            raw = wide
        self.values = raw.view(torch.float8_e4m3fn)  # [.., N, K rounded up to 16], zero behind K

    @property
    def device(self) -> torch.device:
        return self.values.device

    @staticmethod
    def from_tensor(weight: torch.Tensor) -> "Fp8Weights":
        """The matrix (or stack) rounded to this form: a block's largest magnitude becomes 448."""
        if weight.dim() < 2 or weight.numel() == 0 or not weight.is_floating_point():
            raise ValueError("Fp8Weights.from_tensor: a floating-point tensor [.., outputs, inputs]")
        if weight.dim() > 2:  # a matrix at a time: fp32 copies of a whole stack of experts would not fit beside it
            parts = [Fp8Weights.from_tensor(w) for w in weight.reshape(-1, *weight.shape[-2:])]
            lead, k = weight.shape[:-2], weight.shape[-1]
            stack = torch.stack([p.values[..., :k].view(torch.uint8) for p in parts]).view(torch.float8_e4m3fn)
            scales = torch.stack([p.scales for p in parts])
            return Fp8Weights(stack.reshape(*lead, *stack.shape[1:]), scales.reshape(*lead, *scales.shape[1:]))
        n, k = weight.shape
        w = torch.nn.functional.pad(weight.to(torch.float32), (0, -k % BLOCK, 0, -n % BLOCK)).reshape(_blocks(n), BLOCK, _blocks(k), BLOCK)
        most = w.abs().amax(dim=(1, 3), keepdim=True)
        if not bool(torch.isfinite(most).all()):
            raise ValueError("Fp8Weights.from_tensor: the weights hold infinities or NaN")
        most = most.clamp_min(2.0**-100)
        q = (w * (torch.full_like(most, LARGEST) / most)).clamp(-LARGEST, LARGEST).to(torch.float8_e4m3fn)
        q = q.view(torch.uint8).reshape(_blocks(n) * BLOCK, -1)[:n, :k].contiguous().view(torch.float8_e4m3fn)
        return Fp8Weights(q, (most / torch.full_like(most, LARGEST)).reshape(_blocks(n), _blocks(k)))

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The matrix that the numbers stand for."""
        n, k = self.shape[-2:]
        wide = self.scales.repeat_interleave(BLOCK, -2)[..., :n, :].repeat_interleave(BLOCK, -1)[..., :k]
        return (self.values[..., :k].to(torch.float32) * wide).to(dtype)


def fp8_linear(x: torch.Tensor, w: Fp8Weights, bias: torch.Tensor | None = None) -> torch.Tensor:
    """``x [.., K]`` (bf16 or fp32) times the transposed matrix -> ``[.., N]`` in ``x``'s dtype, any number of rows from none up."""
    if len(w.shape) != 2:
        raise ValueError("fp8_linear: one matrix, not a stack")
    return blocks.fp8_linear_of(x, w.values, w.scales, w.shape[1], bias)


def interleaved(gate: Fp8Weights, up: Fp8Weights):
    """The two first projections of a feed-forward as one matrix: runs of 128 rows of either in turn, zero behind the last feature -> (values, scales)."""
    (n, _), kp = gate.shape, gate.values.shape[-1]
    runs = _blocks(n)
    values = torch.zeros((2, runs * BLOCK, kp), dtype=torch.uint8, device=gate.device)
    values[0, :n], values[1, :n] = gate.values.view(torch.uint8), up.values.view(torch.uint8)
    values = values.reshape(2, runs, BLOCK, kp).transpose(0, 1).reshape(2 * runs * BLOCK, kp)
    return values.view(torch.float8_e4m3fn), torch.stack([gate.scales, up.scales], dim=1).reshape(2 * runs, -1).contiguous()
