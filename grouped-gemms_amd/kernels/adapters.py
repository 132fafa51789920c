"""Low-rank adapters of many requests beside a shared projection.

``lora_grouped_mm`` adds to the output of a projection that all tokens share
(e.g. ``triton_mxfp8_grouped_mm`` with one expert) the adapter of each token's
request, all adapters of the batch in one call:

  ``out[t] = base[t] + scales[a] * (x[t] @ down[a]^T) @ up[a]``

``a`` is the token's adapter; a token without one keeps ``base``.  The tokens are
grouped by ``token_plan(adapter_ids, L)``, made once per batch for all layers.
No counterpart in the reference, whose grouped GEMM takes full weights only.

``up`` is stored rank-major, ``(L, r, N)``: with the long side of both factors
contiguous the gradients run on the forward's kernels (an ``(N, r)`` factor from
elsewhere is transposed once, when it is loaded).
"""

from __future__ import annotations

from typing import Optional

import torch

from . import _lib
from ._common import _OUT_CODES, _require, _stream_handle
from .routing import TokenPlan, _check_plan, _row_stride, _same_device


def _ptr(t: Optional[torch.Tensor]):
    return t.data_ptr() if t is not None else None


def _factor(w: torch.Tensor) -> tuple:
    """``(w, rank stride, adapter stride)`` of a factor with its long side contiguous."""
    _, r, K = w.shape
    st = w.stride()
    if (st[2] != 1 and K > 1) or (st[1] < K and r > 1):
        w = w.contiguous()
        st = w.stride()
    return w, st[1] if r > 1 else K, st[0]


def _shrink(x, w, plan, M, code):
    L, r, K = w.shape
    h = torch.empty(_lib.lora_hidden_floats(M, L, r, K), dtype=torch.float32, device=x.device)
    x, ld = _row_stride(x)
    w, ld_r, ld_l = _factor(w)
    _lib.check(_lib.calls().mxgg_lora_shrink(x.data_ptr(), code, K, ld, w.data_ptr(), ld_r, ld_l,
                                             r, plan.src.data_ptr(), plan.offs.data_ptr(), L, M, h.data_ptr(),
                                             _stream_handle(x.device)))
    return h


def _expand(h, w, plan, T, M, code, scales, base, out):
    L, r, N = w.shape
    ldb = 0
    if base is not None:
        base, ldb = _row_stride(base)
    w, ld_r, ld_l = _factor(w)
    _lib.check(_lib.calls().mxgg_lora_expand(h.data_ptr(), h.shape[0], w.data_ptr(), code, N, ld_r,
                                             ld_l, r, _ptr(scales), _ptr(base), ldb, out.data_ptr(),
                                             max(out.stride(0), N), plan.rows.data_ptr(), T, plan.src.data_ptr(),
                                             plan.offs.data_ptr(), L, M, _stream_handle(h.device)))
    return out


def _outer(h, x, L, r, plan, M, code, scales):
    x, ld = _row_stride(x)
    K = x.shape[1]
    out = torch.empty((L, r, K), dtype=x.dtype, device=x.device)
    floats = _lib.lora_outer_floats(M, L, r, K)
    ws = torch.empty(floats, dtype=torch.float32, device=x.device) if floats else None
    _lib.check(_lib.calls().mxgg_lora_outer(h.data_ptr(), h.shape[0], x.data_ptr(), code, K, ld, r, _ptr(scales),
                                            plan.src.data_ptr(), plan.offs.data_ptr(), L, M, out.data_ptr(), _ptr(ws),
                                            floats, _stream_handle(x.device)))
    return out


class _LoraGroupedMM(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, down, up, base, scales, plan, T, M, code):
        h = _shrink(x, down, plan, M, code)
        out = torch.empty((T, up.shape[2]), dtype=x.dtype, device=x.device)
        _expand(h, up, plan, T, M, code, scales, base, out)
        ctx.save_for_backward(x, down, up, scales, h, *plan)
        ctx.args = T, M, code, base is not None
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        x, down, up, scales, h, *plan = ctx.saved_tensors
        plan = TokenPlan(*plan)
        T, M, code, based = ctx.args
        L, r, K = down.shape
        gx = gdown = gup = None
        if ctx.needs_input_grad[0] or ctx.needs_input_grad[1]:
            u = _shrink(g, up, plan, M, code)
            if ctx.needs_input_grad[0]:
                gx = _expand(u, down, plan, T, M, code, scales, None,
                             torch.empty((T, K), dtype=x.dtype, device=x.device))
            if ctx.needs_input_grad[1]:
                gdown = _outer(u, x, L, r, plan, M, code, scales)
        if ctx.needs_input_grad[2]:
            gup = _outer(h, g, L, r, plan, M, code, scales)
        return gx, gdown, gup, g if based else None, None, None, None, None, None


def lora_grouped_mm(x: torch.Tensor, down: torch.Tensor, up: torch.Tensor, plan: TokenPlan, *,
                    scales: Optional[torch.Tensor] = None, base: Optional[torch.Tensor] = None,
                    out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``out[t] = base[t] + scales[a] * (x[t] @ down[a]^T) @ up[a]``, a the token's adapter.

    Args:
        x: ``(T, K)`` bf16 or fp16.
        down: ``(L, r, K)``, up: ``(L, r, N)`` of x's type; r up to 512, L up to 1024.
        plan: ``token_plan(adapter_ids, L)`` of the ``(T,)`` adapter ids, -1 for none.
        scales: ``(L,)`` f32 factor of each adapter (None: 1).
        base: ``(T, N)`` of x's type, the shared projection's output (None: zeros).
        out: where to put the result without gradients; ``base`` itself adds in place.

    Sums are f32 and rounded once, to x's type.  Differentiable in ``x``,
    ``down``, ``up`` and ``base``.
    """
    _require(x, "x")
    code = _OUT_CODES.get(x.dtype)
    if x.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"x dtype {x.dtype} is neither bf16 nor fp16")
    T, k, M = _check_plan(plan, x.device)
    if k != 1:
        raise ValueError(f"the plan gives {k} adapters to a token, expected 1")
    if x.dim() != 2 or x.shape[0] != T:
        raise ValueError(f"x must be ({T}, K) for this plan, got {tuple(x.shape)}")
    if down.dim() != 3 or up.dim() != 3 or down.shape[:2] != up.shape[:2] or down.shape[2] != x.shape[1]:
        raise ValueError(f"down must be (L, r, {x.shape[1]}) and up (L, r, N); got {tuple(down.shape)} and {tuple(up.shape)}")
    if plan.offs.shape[0] != down.shape[0]:
        raise ValueError(f"the plan has {plan.offs.shape[0]} groups, down has L={down.shape[0]}")
    N = up.shape[2]
    for name, t in (("down", down), ("up", up), ("base", base), ("out", out)):
        if t is None:
            continue
        if t.dtype != x.dtype:
            raise TypeError(f"{name} dtype {t.dtype} is not x's {x.dtype}")
        _same_device(t, name, x.device)
        if name in ("base", "out") and tuple(t.shape) != (T, N):
            raise ValueError(f"{name} must be ({T}, {N}), got {tuple(t.shape)}")
    if scales is not None:
        if scales.dtype != torch.float32 or tuple(scales.shape) != (down.shape[0],):
            raise ValueError(f"scales must be float32 ({down.shape[0]},), got {scales.dtype} {tuple(scales.shape)}")
        _same_device(scales, "scales", x.device)
        scales = scales.contiguous()
    if torch.is_grad_enabled() and (x.requires_grad or down.requires_grad or up.requires_grad
                                    or (base is not None and base.requires_grad)):
        if out is not None:
            raise ValueError("out cannot be given where gradients are recorded")
        if T == 0:
            raise ValueError("a batch without tokens has no gradients to record")
        return _LoraGroupedMM.apply(x, down, up, base, scales, plan, T, M, code)
    if out is None:
        out = torch.empty((T, N), dtype=x.dtype, device=x.device)
    elif out.stride(1) != 1 and N > 1:
        raise ValueError("out must have a contiguous last dim")
    if T == 0:
        return out
    return _expand(_shrink(x, down, plan, M, code), up, plan, T, M, code, scales, base, out)
