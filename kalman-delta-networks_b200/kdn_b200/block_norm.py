"""The norms around a block: what joins a block's output to the residual stream
and normalises the sum for the next block, in one kernel each way.

    u = act(gate) * scale * norm(y) * post_weight      (norm after the block, gate, residual scale)
    z = alpha * x + u                                  (residual stream)
    h = norm(z) * weight                               (norm before the next block)
    norm(t) = t / sqrt(mean(t^2) + eps)

The reference's ``Block.forward`` (lit_gpt/model.py:265-299) takes the two
middle steps (``x + mixer(norm_1(x))``, then ``norm_2``) as separate kernels;
the norm after the block, the gate and the scale are those of sandwich-norm,
gated and LayerScale blocks.  Everything is computed in fp32 and rounded once
per output; the backward forms z again from x and y, so its gradients are
those of the unrounded sum.  Weight gradients are summed in a fixed order.
"""
from __future__ import annotations

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from . import _native as N
from .norm_gated import _ACTIVATIONS

# A norm over one value is its sign; its gradient is of the order of eps, which fp32 cannot resolve beside 1.
MIN_WIDTH, MAX_WIDTH = 2, 8192
_DTYPES = (torch.bfloat16, torch.float32)


def _rows(t, D):
    """[..., D] as [rows, D] with contiguous rows that do not overlap, or one row for all (a view where the strides allow
    one).  ``empty_like`` of it is contiguous, whatever the rows' stride."""
    if t.ndim != 2:
        t = t.reshape(-1, D)
    apart, inner = t.stride()
    return t if inner == 1 and (apart >= D or apart == 0 or t.shape[0] <= 1) else t.contiguous()


def _args(x, y, gate, weight, post_weight, scale, z, h, rstd, alpha, swish, eps):
    """The C arguments (None: absent) in the order of the fields."""
    return N.KdnBlockNormArgs(
        x.dtype == torch.bfloat16, (x if y is None else y).dtype == torch.bfloat16, weight.dtype == torch.bfloat16, swish,
        x.shape[0], x.shape[1], alpha, eps,
        x.data_ptr(), None if y is None else y.data_ptr(), None if gate is None else gate.data_ptr(),
        x.stride(0), 0 if y is None else y.stride(0), 0 if gate is None else gate.stride(0),
        weight.data_ptr(), None if post_weight is None else post_weight.data_ptr(),
        None if scale is None else scale.data_ptr(), None if z is None else z.data_ptr(),
        None if h is None else h.data_ptr(), None if rstd is None else rstd.data_ptr())


def _forward(x, y, gate, weight, post_weight, scale, alpha, swish, eps, want_rstd):
    """x, y, gate as [rows, D].  Returns (z or None, h, rstd or None), contiguous."""
    lib = N.load_library()
    h = torch.empty_like(x if y is None else y)
    z = None if y is None else torch.empty_like(x)
    rstd = x.new_empty((2, x.shape[0]), dtype=torch.float32) if want_rstd else None
    a = _args(x, y, gate, weight, post_weight, scale, z, h, rstd, alpha, swish, eps)
    N.launch(lib.kdn_block_norm_fwd, a, x, "kdn_block_norm_fwd")
    return z, h, rstd


class _BlockNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, y, gate, weight, post_weight, scale, alpha, swish, eps):
        z, h, rstd = _forward(x, y, gate, weight, post_weight, scale, alpha, swish, eps, True)
        ctx.save_for_backward(x, y, gate, weight, post_weight, scale, rstd)
        ctx.meta = (alpha, swish, eps)
        ctx.set_materialize_grads(False)
        # without a block z is x; it is handed on here so that its cotangent reaches the kernel (one rounding of the sum)
        return x if z is None else z, h

    @staticmethod
    @once_differentiable
    def backward(ctx, dz, dh):
        if dz is None and dh is None:
            return (None,) * 9
        saved = ctx.saved_tensors
        inputs, needed = saved[:6], ctx.needs_input_grad[:6]
        a = _args(*inputs, None, None, saved[6], *ctx.meta)
        if dz is not None:
            dz = dz.contiguous()
            a.dz = dz.data_ptr()
        if dh is not None:
            dh = dh.contiguous()
            a.dh = dh.data_ptr()
        else:  # z does not depend on the weight
            needed = (*needed[:3], False, *needed[4:])
        grads = [torch.empty_like(t) if n else None for t, n in zip(inputs, needed)]
        for name, g in zip(("dx", "dy", "dgate", "dweight", "dpost", "dscale"), grads):
            if g is not None:
                setattr(a, name, g.data_ptr())
        lib = N.load_library()
        x = inputs[0]
        if any(needed[3:]):
            ws = x.new_empty(lib.kdn_block_norm_workspace_bytes(a.rows, a.D), dtype=torch.uint8)
            a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
        N.launch(lib.kdn_block_norm_bwd, a, x, "kdn_block_norm_bwd")
        return (*grads, None, None, None)


def _validate(x, y, weight, post_weight, gate, scale, alpha, activation):
    if activation not in _ACTIVATIONS:
        raise ValueError(f"Unsupported activation: {activation}")
    if x.ndim < 1 or not MIN_WIDTH <= x.shape[-1] <= MAX_WIDTH:
        raise ValueError(f"kdn_b200 block_norm: the last axis must be {MIN_WIDTH} to {MAX_WIDTH} wide, got {tuple(x.shape)}")
    D = x.shape[-1]
    if x.dtype not in _DTYPES:
        raise TypeError(f"x must be bf16 or fp32, got {x.dtype}")
    if y is None:
        if post_weight is not None or gate is not None or scale is not None or alpha != 1.0:
            raise ValueError("post_weight, gate, scale and alpha need a block output y")
    else:
        if y.shape != x.shape:
            raise ValueError(f"x and y must have the same shape, got {tuple(x.shape)} and {tuple(y.shape)}")
        if y.dtype != x.dtype and (x.dtype, y.dtype) != (torch.float32, torch.bfloat16):
            raise TypeError(f"y must have x's dtype, or be bf16 beside an fp32 x; got x {x.dtype}, y {y.dtype}")
    if gate is not None and (gate.shape != y.shape or gate.dtype != y.dtype):
        raise ValueError(f"gate must have y's shape and dtype, got {tuple(gate.shape)} {gate.dtype}")
    if weight is None:
        raise TypeError("weight must be a tensor")
    for name, w in (("weight", weight), ("post_weight", post_weight), ("scale", scale)):
        if w is None:
            continue
        if w.ndim != 1 or w.shape[0] != D:
            raise ValueError(f"{name} must have shape [{D}], got {tuple(w.shape)}")
        if w.dtype is not weight.dtype or w.dtype not in _DTYPES:
            raise TypeError("weight, post_weight and scale must share one dtype, bf16 or fp32")
    device = x.device
    for t in (y, weight, post_weight, gate, scale):
        if t is not None and t.device != device:
            raise ValueError("all block_norm tensors must share one CUDA device")
    if not x.is_cuda:
        N.require_cuda(x)
    return D


def block_norm(x, y, weight, *, post_weight=None, gate=None, scale=None, alpha=1.0, activation="sigmoid", eps=1e-5):
    """Join block output ``y`` to the residual stream ``x`` and normalise for the next block; returns ``(z, h)``.

    x [..., D] bf16 or fp32; y and gate [..., D] in x's dtype, or bf16 beside an fp32 x; weight, post_weight and scale [D]
    (one dtype, bf16 or fp32).  ``post_weight`` None: no norm after the block; ``gate`` None: no gate; ``scale`` None: 1.
    ``alpha`` is a Python number multiplying x.  z has x's dtype, h has y's.  With ``y`` None (before the first block) z
    is x itself and h = norm(x) * weight.  Differentiable in every tensor, once and in reverse mode.
    """
    alpha, eps = float(alpha), float(eps)
    fast = N.host()
    if fast is not None and y is not None and weight is not None and activation in _ACTIVATIONS:
        out = fast.block_norm(x, y, weight, post_weight, gate, scale, alpha, _ACTIVATIONS[activation], eps, MIN_WIDTH,
                              MAX_WIDTH)
        if out is not None:
            return out
    D = _validate(x, y, weight, post_weight, gate, scale, alpha, activation)
    swish = _ACTIVATIONS[activation]
    shape = x.shape
    x2 = _rows(x, D)
    y2 = None if y is None else _rows(y, D)
    g2 = None if gate is None else _rows(gate, D)
    leaves = [t for t in (x, y, gate, weight, post_weight, scale) if t is not None]
    # forward-mode tangents go to the function too: it refuses them (no jvp) instead of dropping them
    if (torch.is_grad_enabled() and any([t.requires_grad for t in leaves])) or N.has_tangent(*leaves):
        weight, post_weight, scale = [None if w is None else w.contiguous() for w in (weight, post_weight, scale)]
        z, h = _BlockNormFunction.apply(x2, y2, g2, weight, post_weight, scale, alpha, swish, eps)
        if y is None and not x.requires_grad:
            z = None
    else:
        weight, post_weight, scale = [None if w is None else w.contiguous()
                                      for w in (weight, post_weight, scale)]
        z, h, _ = _forward(x2, y2, g2, weight, post_weight, scale, alpha, swish, eps, False)
    if len(shape) != 2:
        z, h = None if z is None else z.view(shape), h.view(shape)
    return (x if z is None else z), h


class BlockNorm(nn.Module):
    """Module form: holds ``weight`` and, when asked for, ``post_weight`` (ones) and ``scale`` (``scale_init``)."""

    def __init__(self, hidden_size, *, post_norm=False, scale_init=None, alpha=1.0, eps=1e-5, activation="sigmoid",
                 device=None, dtype=None):
        super().__init__()
        if activation not in _ACTIVATIONS:
            raise ValueError(f"Unsupported activation: {activation}")
        self.hidden_size, self.alpha, self.eps, self.activation = hidden_size, alpha, eps, activation
        ones = lambda: nn.Parameter(torch.ones(hidden_size, device=device, dtype=dtype))  # noqa: E731
        self.weight = ones()
        self.post_weight = ones() if post_norm else None
        self.scale = None
        if scale_init is not None:
            self.scale = nn.Parameter(torch.full((hidden_size,), float(scale_init), device=device, dtype=dtype))

    def forward(self, x, y=None, gate=None):
        if y is None:
            return block_norm(x, None, self.weight, eps=self.eps)
        return block_norm(x, y, self.weight, post_weight=self.post_weight, gate=gate, scale=self.scale,
                          alpha=self.alpha, activation=self.activation, eps=self.eps)


__all__ = ("BlockNorm", "block_norm")
