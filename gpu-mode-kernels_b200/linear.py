"""Dense products with bias, activation and residual in their epilogue: what stands beside the routed experts of a layer
-- the router's logits, shared experts, projections.

All work is in liba2a.so (``a2a_linear``); there is no CPU or PyTorch fallback.  The reference has no counterpart: its
layer is the all-to-all around a placeholder (amd-distributed/all2all/reference.py:256-270).
"""
from __future__ import annotations

import ctypes as C
from typing import Optional

import torch

from . import _lib

DTYPES = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_FP16, torch.float32: _lib.DTYPE_FP32}
_SIXTEEN = (torch.bfloat16, torch.float16)


def refuse(message: str):
    raise _lib.A2AError(_lib.A2A_ERR_CONFIG, message)


def failed(code: int):
    """Raise for a status code of a product."""
    if code == _lib.A2A_ERR_TIMEOUT:
        raise _lib.A2AError(code, "a wait inside an earlier product on this GPU ran out, and what it left is not valid; nothing has been launched now "
                                  "(linear.check() clears this)")
    _lib.check(code)


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether the bytes from the first to the last element of two strided tensors meet."""
    if a.numel() == 0 or b.numel() == 0:
        return False
    ends = [t.data_ptr() + t.element_size() * (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride()))) for t in (a, b)]
    return a.data_ptr() < ends[1] and b.data_ptr() < ends[0]


def linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, *, activation: str = "none",
           residual: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """``act(x @ weight.T + bias) + residual`` on the current stream.

    ``x`` ``[..., inputs]`` and ``weight`` ``[outputs, inputs]`` are bf16 or fp16 CUDA tensors, rows contiguous (a matrix's rows may lie
    further apart), ``inputs`` and the distance of rows a multiple of 8, starts on 16 bytes.  ``activation``: ``"none"``, ``"relu"``, ``"gelu"``
    (by the error function), ``"silu"``, or ``"swiglu"``: ``weight`` ``[2 * outputs, inputs]`` holds gate rows before up rows and the result is
    ``silu(gate) * up``.  ``bias`` has the weight's rows, in its type or fp32; ``residual`` the result's shape and type.  ``out_dtype``: the
    type of ``x`` (default) or ``torch.float32``.  Sums and the epilogue are fp32, with one rounding at the end.  For inference: no gradient is
    recorded.  Raises where an earlier product on this GPU has recorded an error (``check``).
    """
    out = _lib.host().linear(x, weight, bias, activation, residual, out_dtype)
    if out is not None:
        return out if type(out) is not int else failed(out)
    # something is wrong, or unusual: look again, one thing at a time
    if x.dtype not in _SIXTEEN or not x.is_cuda or x.dim() < 1:
        refuse(f"x must be a bf16 or fp16 CUDA tensor [..., inputs], got {x.dtype} {tuple(x.shape)} on {x.device}")
    device = x.get_device()
    if device != torch.cuda.current_device():
        with torch.cuda.device(device):
            return linear(x, weight, bias, activation=activation, residual=residual, out_dtype=out_dtype)
    inputs = x.shape[-1]
    if weight.dtype != x.dtype or weight.dim() != 2 or weight.shape[1] != inputs or weight.get_device() != device:
        refuse(f"weight must be [outputs, {inputs}] {x.dtype} on {x.device}, got {tuple(weight.shape)} {weight.dtype} on {weight.device}")
    if activation not in _lib.ACTIVATION:
        refuse(f"activation must be one of {', '.join(_lib.ACTIVATION)}, got {activation!r}")
    rows = weight.shape[0]
    outputs = rows // 2 if activation == "swiglu" else rows
    if outputs == 0 or (activation == "swiglu" and rows % 2):
        refuse(f"weight has {rows} rows" + (", and swiglu takes an even number: gate rows and up rows" if rows else ""))
    if inputs < 8 or inputs % 8 or inputs > _lib.MAX_PRODUCT or outputs > _lib.MAX_OUTPUTS:
        refuse(f"inputs must be a multiple of 8 up to {_lib.MAX_PRODUCT}, outputs at most {_lib.MAX_OUTPUTS}, got {inputs} and {outputs}")
    out_dtype = out_dtype or x.dtype
    if out_dtype not in (x.dtype, torch.float32):
        refuse(f"out_dtype must be {x.dtype} or torch.float32, got {out_dtype}")
    if weight.stride(1) != 1 or (rows > 1 and (weight.stride(0) < inputs or weight.stride(0) % 8)) or weight.data_ptr() % 16:
        refuse("weight must have contiguous rows, 16-byte aligned")
    if bias is not None and (bias.dtype not in (x.dtype, torch.float32) or tuple(bias.shape) != (rows,) or not bias.is_contiguous()
                             or bias.get_device() != device):
        refuse(f"bias must be a contiguous [{rows}] of {x.dtype} or torch.float32 on {x.device}, got {tuple(bias.shape)} {bias.dtype}")
    shape = (*x.shape[:-1], outputs)
    if residual is not None and (residual.dtype != out_dtype or tuple(residual.shape) != shape or residual.get_device() != device):
        refuse(f"residual must be {shape} {out_dtype} on {x.device}, got {tuple(residual.shape)} {residual.dtype} on {residual.device}")
    y = torch.empty(shape, dtype=out_dtype, device=x.device)
    # matrices as they lie, where one stride gives the rows; else copies
    flat = x if x.dim() == 2 else x.reshape(-1, inputs)
    if flat.stride(1) != 1 or flat.stride(0) < inputs or flat.stride(0) % 8 or flat.data_ptr() % 16:
        flat = flat.contiguous()
        if flat.data_ptr() % 16:
            flat = flat.clone()
    tokens = flat.shape[0]
    if tokens == 0:
        return y
    if tokens > _lib.MAX_ROWS:
        refuse(f"at most {_lib.MAX_ROWS} rows, got {tokens}")
    add = None
    if residual is not None:
        add = residual if residual.dim() == 2 else residual.reshape(-1, outputs)
        if add.stride(1) != 1 or add.stride(0) < 0:
            add = add.contiguous()
    args = _lib.Linear(flat.data_ptr(), weight.data_ptr(), 0 if bias is None else bias.data_ptr(), 0 if add is None else add.data_ptr(),
                       y.data_ptr(), flat.stride(0) if tokens > 1 else inputs, weight.stride(0) if rows > 1 else inputs,
                       0 if add is None else add.stride(0), outputs, tokens, inputs, outputs, DTYPES[x.dtype], DTYPES[out_dtype],
                       DTYPES[x.dtype if bias is None else bias.dtype], _lib.ACTIVATION[activation])
    rc = _lib.load().a2a_linear(C.byref(args), _lib.current_stream())
    if rc != 0:
        failed(rc)
    return y


def check() -> None:
    """Raise if a product (``linear``, ``moe_layer``, ``expert_mlp``) on the current device has recorded an error since the last look, and forget it
    (synchronises the device).  A wait inside a kernel that ran out is recorded when it does, after the call has returned: without this the next product
    raises, and launches nothing; replays of a captured graph do not look."""
    code = C.c_int32()
    _lib.check(_lib.load().a2a_product_status(C.byref(code)))
    if code.value != 0:
        raise _lib.A2AError(code.value, "a wait inside a product on this GPU ran out: what it left is not valid; the record has been cleared")
