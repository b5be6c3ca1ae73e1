"""The SwiGLU layer as a mixture of experts, for up to 64 tokens (swb_moe).

    logits = router x,  experts = the topk largest,  w = softmax
    y_t = sum_j w_tj down_e (SiLU(gate_e x_t) * (up_e x_t))

Ties go to the lowest index and a NaN logit counts as the largest. ``renormalize``: the
softmax runs over the selected logits, so that a token's weights sum to one; else over all
logits. The product of the activations keeps fp32's range in either type (swb_moe states its
precision). Like ``swiglu_out`` the call adds no bias and no residual, writes buffers the caller
owns, launches on the current CUDA stream and allocates nothing.
"""
from __future__ import annotations

import torch

from . import _lib
from .binding import _check
from .mx4 import _TYPES, _call, _check_packed

MAX_TOKENS = _lib.SWB_MOE_MAX_TOKENS


def _check_sizes(tokens: int, experts: int, topk: int, inter: int) -> None:
    """Here too, since the library's arguments are 32 bits wide and ctypes cuts longer ones."""
    _check(0 <= tokens <= MAX_TOKENS and 0 < experts <= _lib.SWB_MOE_MAX_EXPERTS
           and 0 < topk <= min(experts, _lib.SWB_MOE_MAX_TOPK) and 0 < inter <= _lib.SWB_MOE_MAX_DIM, "invalid shape")


def moe_workspace(tokens: int, experts: int, topk: int, inter: int, device=None) -> torch.Tensor:
    """A zeroed workspace for calls of up to these sizes, one per stream of calls (calls that may
    overlap on the GPU, captured ones included, need one each)."""
    _check_sizes(tokens, experts, topk, inter)
    n = _lib.lib().swb_moe_workspace_bytes(tokens, experts, topk, inter)
    return torch.zeros(n, dtype=torch.uint8, device=device or "cuda")


def moe_out(x: torch.Tensor, router: torch.Tensor, gate: torch.Tensor, up: torch.Tensor, down: torch.Tensor,
            y: torch.Tensor, workspace: torch.Tensor, topk: int, *, renormalize: bool = True,
            gate_scales: torch.Tensor | None = None, up_scales: torch.Tensor | None = None,
            down_scales: torch.Tensor | None = None, ids: torch.Tensor | None = None,
            weights: torch.Tensor | None = None) -> None:
    """The layer into ``y`` [tokens, hidden].

    x: [tokens, hidden] fp16 or bf16, rows contiguous; router: [experts, hidden] of x's type;
    gate, up: [experts, inter, hidden] and down: [experts, hidden, inter] of x's type, or all
    three four-bit codes with their scales (``mx4_quantize``; inter is then read from gate).
    ids [tokens, topk] int32 and weights [tokens, topk] fp32 receive the selection.
    """
    _check(x.is_cuda and x.dtype in (torch.float16, torch.bfloat16) and x.dim() == 2,
           "x must be a CUDA FP16 or BF16 matrix")
    device, dtype = x.device, x.dtype
    tokens, hidden = x.shape
    pitch = x.stride(0) if tokens > 1 else hidden
    _check((hidden <= 1 or x.stride(1) == 1) and pitch >= hidden, "x must have contiguous rows")
    _check(router.dim() == 2 and router.size(1) == hidden, "router must be [experts, hidden]")
    _check(gate.dim() == 3, "gate must be [experts, inter, hidden]")
    experts, inter = router.size(0), gate.size(1)
    _check_sizes(tokens, experts, topk, inter)
    _check(0 < hidden <= _lib.SWB_MOE_MAX_DIM, "invalid shape")
    four_bit = gate_scales is not None
    _check(four_bit == (up_scales is not None) == (down_scales is not None),
           "scales belong to all three matrices or to none")
    if four_bit:
        _check_packed(gate, gate_scales, (experts, inter), hidden, device)
        _check_packed(up, up_scales, (experts, inter), hidden, device)
        _check_packed(down, down_scales, (experts, hidden), inter, device)
        typed = (router, y)
    else:
        _check(gate.shape == (experts, inter, hidden) and up.shape == gate.shape
               and down.shape == (experts, hidden, inter), "incompatible weights")
        typed = (router, y, gate, up, down)
    for t in typed:
        if t.dtype != dtype or t.device != device or not t.is_contiguous():
            raise RuntimeError("router, weights and y must be contiguous, of x's type and on its device")
        if t.requires_grad:
            raise RuntimeError("inference only: disable gradients")
    _check(not x.requires_grad and (weights is None or not weights.requires_grad), "inference only: disable gradients")
    _check(y.shape == x.shape, "y must have x's shape")
    _check(workspace.device == device and workspace.dtype == torch.uint8 and workspace.is_contiguous(),
           "workspace must come from moe_workspace on x's device")
    for t, kind in ((ids, torch.int32), (weights, torch.float32)):
        if t is not None and (t.dtype != kind or t.device != device or not t.is_contiguous()
                              or t.shape != (tokens, topk)):
            raise RuntimeError("ids (int32) and weights (fp32) must be contiguous [tokens, topk]")
    flags = (_lib.SWB_MOE_MX4 if four_bit else 0) | (_lib.SWB_MOE_RENORMALIZE if renormalize else 0)
    _call(device, _lib.lib().swb_moe, _TYPES[dtype], flags, x.data_ptr(), pitch, router.data_ptr(), gate.data_ptr(),
          up.data_ptr(), down.data_ptr(), gate_scales.data_ptr() if four_bit else None,
          up_scales.data_ptr() if four_bit else None, down_scales.data_ptr() if four_bit else None, y.data_ptr(),
          None if ids is None else ids.data_ptr(), None if weights is None else weights.data_ptr(), tokens, hidden,
          inter, experts, topk, workspace.data_ptr(), workspace.numel())


def moe(x: torch.Tensor, router: torch.Tensor, gate: torch.Tensor, up: torch.Tensor, down: torch.Tensor, topk: int,
        **kwargs) -> torch.Tensor:
    """Allocating wrapper of ``moe_out`` (output and workspace; the options are ``moe_out``'s)."""
    _check(x.dim() == 2 and router.dim() == 2 and gate.dim() == 3, "invalid dimensions")
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    workspace = moe_workspace(x.size(0), router.size(0), topk, gate.size(1), x.device)
    moe_out(x, router, gate, up, down, y, workspace, topk, **kwargs)
    return y
