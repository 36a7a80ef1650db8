"""Quantisation: block-scaled fp8 (e4m3) in plain PyTorch, the oracle for what
``AllToAll.dispatch_quant`` fuses into the send, and rows of 8-bit integers, the input of
``grouped_gemm_int8``.

One fp32 scale per ``block`` (128) consecutive columns of a row:
``scale = max(amax, 1e-4) / 448`` and ``q = round_to_e4m3(x * (448 / max(amax, 1e-4)))``.
"""

from __future__ import annotations

import torch

from . import _ops


def per_token_block_quant(x: torch.Tensor, block: int = 128,
                          pow2: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    """x: [m, hidden] -> (q [m, hidden] float8_e4m3fn, scale [m, ceil(hidden / block)] fp32).
    With ``pow2`` the scale is the smallest power of two that is not below ``amax / 448``."""
    m, hidden = x.shape
    nblk = (hidden + block - 1) // block
    xf = x.to(torch.float32)
    pad = nblk * block - hidden
    if pad:
        xf = torch.nn.functional.pad(xf, (0, pad))
    v = xf.view(m, nblk, block)
    amax = v.abs().amax(dim=2).clamp(min=1e-4)
    if pow2:
        scale = torch.exp2(torch.ceil(torch.log2(amax / 448.0)))
        q = (v / scale.unsqueeze(2)).clamp(-448.0, 448.0)
    else:
        scale = amax / 448.0
        q = (v * (448.0 / amax).unsqueeze(2)).clamp(-448.0, 448.0)
    q = q.to(torch.float8_e4m3fn).view(m, nblk * block)[:, :hidden]
    return q.contiguous(), scale.contiguous()


def block_dequant(q: torch.Tensor, scale: torch.Tensor, block: int = 128) -> torch.Tensor:
    """Inverse of ``per_token_block_quant`` in fp32."""
    hidden = q.size(-1)
    s = scale.repeat_interleave(block, dim=-1)[..., :hidden]
    return q.to(torch.float32) * s


def quantize_rows_int8(x: torch.Tensor, counts: torch.Tensor | None = None,
                       out: torch.Tensor | None = None, out_scale: torch.Tensor | None = None,
                       ) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows of 8-bit integers with one fp32 scale each: ``x ~= q * scale``.

    ``x`` [rows, k] or [experts, rows, k] in bf16, fp16 or fp32 (weights, one row per channel, or
    activations).  With ``a = max(max |x|, 1e-30)`` of a row, ``scale = a * (1 / 127)`` and ``q =
    round(x * (127 * (1 / a)))``, ties to even, within [-127, 127]; each step is rounded to fp32, the
    reciprocals too, so a value on the border of two integers goes where its rounded product lies.
    A row with an infinity or a NaN gets that as its scale and zeros in place of the values, so
    that what is computed with the row is not finite either.  ``counts`` [experts] int32, with x of
    [experts, rows, k]: rows at or beyond an expert's count are left as they are.
    """
    if x.requires_grad and torch.is_grad_enabled():
        raise ValueError("quantize_rows_int8: no gradient is recorded here; use torch.no_grad() or detach()")
    if out is None and out_scale is None:
        return _ops.quantize_rows_int8(x, counts)
    if out is None:
        out = torch.empty(x.shape, dtype=torch.int8, device=x.device)
    if out_scale is None:
        out_scale = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
    _ops.quantize_rows_int8_out(x, counts, out, out_scale)
    return out, out_scale


def quantize_rows_int8_reference(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Plain PyTorch statement of ``quantize_rows_int8`` for finite rows."""
    v = x.to(torch.float32)
    amax = v.abs().amax(dim=-1).clamp(min=1e-30)
    q = torch.round(v * (127.0 * amax.reciprocal()).unsqueeze(-1)).clamp(-127, 127).to(torch.int8)
    # (As a tensor, so that the reciprocal is rounded to fp32 on every device.)
    return q, amax * torch.full_like(amax, 127.0).reciprocal()
