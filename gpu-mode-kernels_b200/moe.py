"""The layer around the all-to-all: the gate that chooses a token's experts, and the experts themselves.

``topk_gate``   indices and weights, as ``custom_kernel`` and ``A2AContext`` take them, from the router's logits.
``moe_layer``   a whole layer for a few tokens on one GPU: experts' products and their weighted sum.
``expert_mlp``  the experts' products on the rows a dispatch has left: the real expert op between ``A2AContext.dispatch_recv``
                and ``expert_done`` (``A2AContext.experts`` calls it there).

Experts are SwiGLU ones: ``down (silu(gate x) * up x)``, ``gate_up`` ``[experts, 2 * inner, hidden]`` with gate rows before up rows,
``down`` ``[experts, hidden, inner]``.  All work is in liba2a.so; there is no CPU or PyTorch fallback.  In the reference the
experts are a placeholder (amd-distributed/all2all/reference.py:262) and the choice is random (reference.py:33-43).
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Tuple

import torch

from . import _lib
from .linear import DTYPES, _overlap, failed, linear, refuse

_SIXTEEN = (torch.bfloat16, torch.float16)


def topk_gate(logits: torch.Tensor, k: int, *, score: str = "softmax", bias: Optional[torch.Tensor] = None, renormalize: bool = True,
              scale: float = 1.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(indices [tokens, k] int32, weights [tokens, k] fp32)`` from ``logits`` ``[tokens, experts]`` (fp32, bf16 or fp16).

    Scores are the softmax or the sigmoid of the logits.  The k largest logits are chosen, or with ``bias`` ``[experts]`` fp32 the
    k largest ``score + bias`` (in 64 bits; the bias is not part of the weights), in descending order, ties to the lowest index.  Weights are the
    chosen scores, divided by their sum with ``renormalize`` (however small that is; 0 where all chosen logits are -inf), times ``scale``.  A logit of -inf excludes an expert while k
    others are there; a row of nothing else gets weights 0 with softmax.  NaN ranks first, and the weights of its row are NaN with softmax.
    For inference: no gradient is recorded.
    """
    out = _lib.host().gate(logits, k, score, bias, renormalize, scale)
    if out is not None:
        return out if type(out) is not int else _lib.check(out)
    # something is wrong, or unusual: look again, one thing at a time
    if logits.dtype not in DTYPES or not logits.is_cuda or logits.dim() != 2:
        refuse(f"logits must be a [tokens, experts] CUDA tensor of fp32, bf16 or fp16, got {tuple(logits.shape)} {logits.dtype} on {logits.device}")
    device = logits.get_device()
    if device != torch.cuda.current_device():
        with torch.cuda.device(device):
            return topk_gate(logits, k, score=score, bias=bias, renormalize=renormalize, scale=scale)
    tokens, experts = logits.shape
    if tokens > _lib.MAX_ROWS or not 1 <= experts <= _lib.MAX_EXPERTS or not 1 <= k <= min(experts, _lib.MAX_TOPK):
        refuse(f"1 to {_lib.MAX_EXPERTS} experts, and 1 to {_lib.MAX_TOPK} of them chosen, not {k} of {experts}; at most {_lib.MAX_ROWS} tokens")
    if score not in _lib.SCORE:
        refuse(f"score must be one of {', '.join(_lib.SCORE)}, got {score!r}")
    if bias is not None and (bias.dtype is not torch.float32 or tuple(bias.shape) != (experts,) or not bias.is_contiguous()
                             or bias.get_device() != device):
        refuse(f"bias must be a contiguous [{experts}] torch.float32 on {logits.device}, got {tuple(bias.shape)} {bias.dtype} on {bias.device}")
    if experts > 1 and logits.stride(1) != 1 or logits.stride(0) < 0:
        logits = logits.contiguous()
    indices = torch.empty(tokens, k, dtype=torch.int32, device=logits.device)
    weights = torch.empty(tokens, k, dtype=torch.float32, device=logits.device)
    args = _lib.Gate(logits.data_ptr(), logits.stride(0), 0 if bias is None else bias.data_ptr(), indices.data_ptr(), weights.data_ptr(),
                     tokens, experts, k, DTYPES[logits.dtype], _lib.SCORE[score], renormalize, scale)
    rc = _lib.load().a2a_gate(C.byref(args), _lib.current_stream())
    if rc != 0:
        _lib.check(rc)
    return indices, weights


def route(x: torch.Tensor, router: torch.Tensor, k: int, *, score: str = "softmax", bias: Optional[torch.Tensor] = None,
          renormalize: bool = True, scale: float = 1.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """``topk_gate`` of the fp32 logits ``x @ router.T``: from token rows ``[tokens, hidden]`` to what a dispatch takes."""
    return topk_gate(linear(x, router, out_dtype=torch.float32), k, score=score, bias=bias, renormalize=renormalize, scale=scale)


def _check_experts(gate_up: torch.Tensor, down: torch.Tensor, hidden: int, dtype: torch.dtype, device: int) -> Tuple[int, int]:
    """Number and inner size of the experts."""
    if gate_up.dim() != 3 or down.dim() != 3:
        refuse(f"gate_up must be [experts, 2 * inner, hidden] and down [experts, hidden, inner], got {tuple(gate_up.shape)} and {tuple(down.shape)}")
    experts, inner = down.shape[0], down.shape[2]
    if tuple(gate_up.shape) != (experts, 2 * inner, hidden) or down.shape[1] != hidden:
        refuse(f"gate_up must be [experts, 2 * inner, {hidden}] and down [experts, {hidden}, inner], got {tuple(gate_up.shape)} and {tuple(down.shape)}")
    for name, t in (("gate_up", gate_up), ("down", down)):
        if t.dtype != dtype or t.get_device() != device or not t.is_contiguous() or t.data_ptr() % 16:
            refuse(f"{name} must be a contiguous {dtype} tensor on cuda:{device}, 16-byte aligned, got {t.dtype} on {t.device}")
    if not 1 <= experts <= _lib.MAX_EXPERTS:
        refuse(f"1 to {_lib.MAX_EXPERTS} experts, got {experts}")
    for name, n in (("hidden", hidden), ("inner", inner)):
        if n < 8 or n % 8 or n > _lib.MAX_PRODUCT:
            refuse(f"{name} must be a multiple of 8 up to {_lib.MAX_PRODUCT}, got {n}")
    return experts, inner


def moe_layer(x: torch.Tensor, indices: torch.Tensor, weights: torch.Tensor, gate_up: torch.Tensor, down: torch.Tensor, *,
              residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``y[t] = residual[t] + sum_k weights[t, k] * expert_{indices[t, k]}(x[t])`` for up to 256 tokens ``[tokens, hidden]``.

    ``x``, the experts and ``residual`` (or None) share one type, bf16 or fp16; ``indices`` int32 and ``weights`` fp32 are ``[tokens, k]``.  An
    index outside the experts marks none (a padded token's row is its residual, or 0); the same expert twice counts twice.  Sums are fp32;
    an expert's inner values are rounded to the type, since the second product takes 16-bit operands, and the result once.
    More tokens go through ``A2AContext`` with ``experts`` between dispatch and combine.  For inference: no gradient is recorded.
    Raises where an earlier product on this GPU has recorded an error (``linear.check``).
    """
    out = _lib.host().layer(x, indices, weights, gate_up, down, residual)
    if out is not None:
        return out if type(out) is not int else failed(out)
    # something is wrong, or unusual: look again, one thing at a time
    if x.dtype not in _SIXTEEN or not x.is_cuda or x.dim() != 2 or not x.is_contiguous():
        refuse(f"x must be a contiguous bf16 or fp16 CUDA tensor [tokens, hidden], got {x.dtype} {tuple(x.shape)} on {x.device}")
    device = x.get_device()
    if device != torch.cuda.current_device():
        with torch.cuda.device(device):
            return moe_layer(x, indices, weights, gate_up, down, residual=residual)
    tokens, hidden = x.shape
    if tokens > _lib.MAX_LAYER_TOKENS:
        refuse(f"at most {_lib.MAX_LAYER_TOKENS} tokens, got {tokens}: more go through A2AContext.experts")
    experts, inner = _check_experts(gate_up, down, hidden, x.dtype, device)
    topk = indices.shape[1] if indices.dim() == 2 else 0
    if not 1 <= topk <= _lib.MAX_TOPK:
        refuse(f"indices must be [{tokens}, k] with k from 1 to {_lib.MAX_TOPK}, got {tuple(indices.shape)}")
    for name, t, dtype in (("indices", indices, torch.int32), ("weights", weights, torch.float32)):
        if t.dtype is not dtype or tuple(t.shape) != (tokens, topk) or not t.is_contiguous() or t.get_device() != device:
            refuse(f"{name} must be a contiguous [{tokens}, {topk}] {dtype} on {x.device}, got {tuple(t.shape)} {t.dtype} on {t.device}")
    if residual is not None and (residual.dtype != x.dtype or residual.shape != x.shape or not residual.is_contiguous()
                                 or residual.get_device() != device):
        refuse(f"residual must be a contiguous {tuple(x.shape)} {x.dtype} on {x.device}, got {tuple(residual.shape)} {residual.dtype}")
    if x.data_ptr() % 16:
        x = x.clone()
    y = torch.empty_like(x)
    if tokens == 0:
        return y
    lib = _lib.load()
    space = torch.empty(lib.a2a_layer_workspace(tokens, topk, hidden, inner), dtype=torch.uint8, device=x.device)
    args = _lib.Layer(x.data_ptr(), indices.data_ptr(), weights.data_ptr(), gate_up.data_ptr(), down.data_ptr(),
                      0 if residual is None else residual.data_ptr(), y.data_ptr(), space.data_ptr(), space.numel(),
                      tokens, topk, experts, hidden, inner, DTYPES[x.dtype])
    rc = lib.a2a_layer(C.byref(args), _lib.current_stream())
    if rc != 0:
        failed(rc)
    return y


def expert_mlp(rows: torch.Tensor, counts: torch.Tensor, gate_up: torch.Tensor, down: torch.Tensor,
               out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Every expert on its rows: ``rows`` ``[local experts, world, capacity, hidden]`` and ``counts`` ``[world, 4, local experts]`` int32 as
    ``A2AContext.expert_buffers`` gives them; row i of slab (l, s) is valid for ``i < counts[s, 0, l]``.

    The results go where the rows are, or to ``out`` of the same shape and type, which is returned; what lies behind a slab's
    valid rows is left as it is.  Sums are fp32; inner values and results are rounded to the type of the rows.  Raises where an earlier product
    on this GPU has recorded an error (``linear.check``).
    """
    if rows.dtype not in _SIXTEEN or not rows.is_cuda or rows.dim() != 4 or not rows.is_contiguous():
        refuse(f"rows must be a contiguous bf16 or fp16 CUDA tensor [local experts, world, capacity, hidden], got {rows.dtype} "
               f"{tuple(rows.shape)} on {rows.device}")
    device = rows.get_device()
    if device != torch.cuda.current_device():
        with torch.cuda.device(device):
            return expert_mlp(rows, counts, gate_up, down, out)
    local, world, capacity, hidden = rows.shape
    experts, inner = _check_experts(gate_up, down, hidden, rows.dtype, device)
    if experts != local:
        refuse(f"rows of {local} experts, and weights of {experts}")
    if not 1 <= world <= _lib.MAX_WORLD or not 1 <= capacity <= 65535:
        refuse(f"1 to {_lib.MAX_WORLD} ranks and a capacity of 1 to 65535, got {world} and {capacity}")
    if counts.dtype is not torch.int32 or tuple(counts.shape) != (world, 4, local) or not counts.is_contiguous() or counts.get_device() != device:
        refuse(f"counts must be a contiguous [{world}, 4, {local}] torch.int32 on {rows.device}, got {tuple(counts.shape)} {counts.dtype}")
    if rows.data_ptr() % 16:
        refuse("rows must be 16-byte aligned")
    out = rows if out is None else out
    if out.dtype != rows.dtype or out.shape != rows.shape or not out.is_contiguous() or out.get_device() != device:
        refuse(f"out must be a contiguous {tuple(rows.shape)} {rows.dtype} on {rows.device}, got {tuple(out.shape)} {out.dtype}")
    if out.data_ptr() != rows.data_ptr() and _overlap(out, rows):
        refuse("out overlaps rows without being the same")
    lib = _lib.load()
    space = torch.empty(lib.a2a_experts_workspace(local, world, capacity, inner), dtype=torch.uint8, device=rows.device)
    args = _lib.Experts(rows.data_ptr(), counts.data_ptr(), gate_up.data_ptr(), down.data_ptr(), out.data_ptr(), space.data_ptr(),
                        space.numel(), local, world, capacity, hidden, inner, DTYPES[rows.dtype])
    rc = lib.a2a_experts(C.byref(args), _lib.current_stream())
    if rc != 0:
        failed(rc)
    return out
