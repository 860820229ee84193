"""One new token per sequence through a KDN mixer: the serving form of the
operators the mixers train with (``lit_gpt/iso_kdn.py:219-314``,
``lit_gpt/diag_kdn.py:245-355``).  The reference's mixers reject caches; here a
pool of per-sequence states (:class:`KDNState`) replaces a key-value cache,
and one kernel (``kdn_step``) does everything between the block's input
projections and its output projection: the short convolution, the q / k
normalisation, the gates, the covariance gain, the memory update and readout,
and the gated output norm.

    step = IsoKDNStep(conv_weight, A_log, dt_bias, norm_weight, omega_bias=..., r_bias=..., omega_min=..., r_min=...)
    state = KDNState.allocate("iso", num_slots, H, D, device="cuda")
    state.reset(slots, initial_precision)                    # or state.store(...) after a prompt
    y = step(state, qkv, decay_raw, omega_r_raw, out_gate, slots)   # [B, H*D], once per token

The arithmetic is fp32 throughout: the convolution's outputs, the normalised
q and k and the readout, which the training path rounds to bf16 between its
kernels, are not rounded here.

The step serves and has no derivative: parameters are taken detached, and in
grad mode an output of inputs that require gradients raises when its backward
is asked for (forward-mode tangents are refused at once).
"""
from __future__ import annotations

import math
from numbers import Real

import torch

from . import _native as N
from .norm_gated import _ACTIVATIONS
from .short_conv import GROUPS, KERNEL_WIDTH

HEAD_DIMS = (64, 128)
DIAG_R_MIN = 0.01  # the diagonal frontend's constant (diag_kdn_chunk.py:2237)
_ACT_DTYPES = (torch.bfloat16, torch.float32)
_SLOT_DTYPES = (torch.int32, torch.int64)


class KDNState:
    """The states of ``num_slots`` sequences of one layer.

    * ``memory`` fp32 [num_slots, H, D, D] (key-major, as the scan's states)
    * ``covariance`` fp32 [num_slots, H] (iso) or [num_slots, H, D] (diag)
    * ``window`` bf16 or fp32 [num_slots, 3, 3*H*D]: the last three rows of the
      raw q | k | v projections, oldest first (the convolution's past)

    The tensors are the caller's and are updated in place.
    """

    def __init__(self, memory, covariance, window):
        if memory.ndim != 4 or memory.shape[2] != memory.shape[3]:
            raise ValueError(f"memory must be [num_slots, H, D, D], got {tuple(memory.shape)}")
        n, H, D, _ = memory.shape
        if H < 1 or D not in HEAD_DIMS:
            raise ValueError(f"kdn_b200 step: H >= 1 and D in {HEAD_DIMS} required, got H={H}, D={D}")
        if tuple(covariance.shape) not in ((n, H), (n, H, D)):
            raise ValueError(f"covariance must be {(n, H)} (iso) or {(n, H, D)} (diag), got {tuple(covariance.shape)}")
        if tuple(window.shape) != (n, KERNEL_WIDTH - 1, GROUPS * H * D):
            raise ValueError(f"window must be {(n, KERNEL_WIDTH - 1, GROUPS * H * D)}, got {tuple(window.shape)}")
        if memory.dtype != torch.float32 or covariance.dtype != torch.float32:
            raise TypeError("memory and covariance must be FP32")
        if window.dtype not in _ACT_DTYPES:
            raise TypeError(f"window must be bf16 or fp32, got {window.dtype}")
        for name, t in (("memory", memory), ("covariance", covariance), ("window", window)):
            if not t.is_contiguous():
                raise ValueError(f"{name} must be contiguous")
            if t.device != memory.device:
                raise ValueError("all state tensors must share one device")
        if memory.data_ptr() % 16:
            raise ValueError("memory must be 16-byte aligned")
        self.memory, self.covariance, self.window = memory, covariance, window
        self.variant = "iso" if covariance.ndim == 2 else "diag"
        self.num_slots, self.num_heads, self.head_dim = n, H, D
        self.layout = (self.variant, H, D)

    @classmethod
    def allocate(cls, variant, num_slots, num_heads, head_dim=128, *, dtype=torch.bfloat16, device="cuda"):
        """A pool of empty states (zero memory, zero past, covariance zero until :meth:`reset`)."""
        if variant not in ("iso", "diag"):
            raise ValueError(f"variant must be 'iso' or 'diag', got {variant!r}")
        cov = (num_slots, num_heads) if variant == "iso" else (num_slots, num_heads, head_dim)
        return cls(torch.zeros(num_slots, num_heads, head_dim, head_dim, device=device),
                   torch.zeros(cov, device=device),
                   torch.zeros(num_slots, KERNEL_WIDTH - 1, GROUPS * num_heads * head_dim, dtype=dtype,
                               device=device))

    def reset(self, slots, initial_precision):
        """Start new sequences at ``slots`` (a tensor or list of slot numbers, or a slice): empty memory and past, covariance
        ``1 / initial_precision`` ([H], the frontend's output).  Plain indexing, here and in :meth:`store`: slots outside
        the pool, which mark idle rows of a step, have to be left out."""
        if tuple(initial_precision.shape) != (self.num_heads,):
            raise ValueError(f"initial_precision must be [{self.num_heads}], got {tuple(initial_precision.shape)}")
        prior = 1.0 / initial_precision.float()
        self.memory[slots] = 0.0
        self.window[slots] = 0
        self.covariance[slots] = prior if self.variant == "iso" else prior[:, None].expand(-1, self.head_dim)

    def store(self, slots, memory, covariance, qkv_tail):
        """Put the states after a prompt at ``slots``: ``memory`` and ``covariance`` as the scan and the gain return them
        (``sequence_parallel.iso_segment`` / ``diag_segment``) and ``qkv_tail`` [n, t, 3*H*D], the prompt's last
        rows of the raw projections (fewer than three: the prompt was shorter, zeros go before them)."""
        tail = qkv_tail[:, -(KERNEL_WIDTH - 1):]
        self.memory[slots] = memory
        self.covariance[slots] = covariance
        window = torch.zeros(tail.shape[0], KERNEL_WIDTH - 1, tail.shape[2], dtype=self.window.dtype,
                             device=self.window.device)
        if tail.shape[1]:
            window[:, -tail.shape[1]:] = tail
        self.window[slots] = window


def _fp32_param(name, t, shape, device):
    if tuple(t.shape) != shape and t.numel() != math.prod(shape):
        raise ValueError(f"{name} must have shape {shape}, got {tuple(t.shape)}")
    if t.device != device:
        raise ValueError("all step parameters must share one device")
    if t.dtype not in _ACT_DTYPES:
        raise TypeError(f"{name} must be bf16 or fp32, got {t.dtype}")
    t = t.detach().float().reshape(shape).contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _finite(name, value):
    if isinstance(value, bool) or not isinstance(value, Real):
        raise TypeError(f"{name} must be a Python scalar, got {type(value).__name__}")
    if not math.isfinite(float(value)):
        raise ValueError(f"{name} must be finite, got {value!r}")
    return float(value)


class _StepFunction(torch.autograd.Function):
    """A step on inputs that require gradients: an error where one is asked for, not a graph that ends in silence."""

    @staticmethod
    def forward(ctx, launch, *inputs):
        return launch()

    @staticmethod
    def backward(ctx, dy):
        raise RuntimeError("kdn_b200 step: the token step has no gradient (train on the chunked operators)")


class _Step:
    """The parameters of one mixer laid out for ``kdn_step`` (fp32 copies where
    they are not fp32 already: make a new step after changing parameters)."""

    variant: str

    def __init__(self, conv_weight, A_log, dt_bias, norm_weight, omega_bias, r_bias, omega_min, r_min, posterior_scale,
                 norm_eps, activation):
        if conv_weight.ndim < 2 or conv_weight.shape[-1] != KERNEL_WIDTH or conv_weight.shape[0] % GROUPS:
            raise ValueError(f"conv_weight must be [3*H*D, {KERNEL_WIDTH}], got {tuple(conv_weight.shape)}")
        if A_log.ndim != 1 or not A_log.shape[0]:
            raise ValueError(f"A_log must be [H], got {tuple(A_log.shape)}")
        if activation not in _ACTIVATIONS:
            raise ValueError(f"Unsupported activation: {activation}")
        H, channels, device = A_log.shape[0], conv_weight.shape[0] // GROUPS, conv_weight.device
        D = channels // H
        if channels != H * D or D not in HEAD_DIMS:
            raise ValueError(f"kdn_b200 step: head dimension must be one of {HEAD_DIMS}, got {channels} channels "
                             f"for {H} heads")
        self.num_heads, self.head_dim, self.device = H, D, device
        self.layout = (self.variant, H, D)
        p = {"conv_weight": _fp32_param("conv_weight", conv_weight, (GROUPS * channels, KERNEL_WIDTH), device),
             "A_log": _fp32_param("A_log", A_log, (H,), device),
             "dt_bias": _fp32_param("dt_bias", dt_bias, (channels,), device)}
        for name, t, shape in (("norm_weight", norm_weight, (D,)), ("omega_bias", omega_bias, (H,)),
                               ("r_bias", r_bias, (H,))):
            if t is not None:
                p[name] = _fp32_param(name, t, shape, device)
        self.parameters = p
        a = N.KdnStepArgs()
        a.variant = N.KDN_ISO if self.variant == "iso" else N.KDN_DIAG
        a.swish = _ACTIVATIONS[activation]
        a.H, a.D = H, D
        for name, t in p.items():
            setattr(a, name, t.data_ptr())
        a.omega_min, a.r_min = _finite("omega_min", omega_min), _finite("r_min", r_min)
        a.posterior_scale, a.eps = posterior_scale, _finite("norm_eps", norm_eps)
        a.scale = D ** -0.5
        self._args = bytes(a)

    def _fits(self, state, qkv):
        return isinstance(state, KDNState) and state.layout == self.layout and self.device == qkv.device

    def _run(self, state, slots, qkv, rows):
        """Checks the token's tensors, launches and returns y.  rows: (argument, tensor, width) of those beside qkv."""
        H, channels, dtype = self.num_heads, self.num_heads * self.head_dim, qkv.dtype
        if not isinstance(state, KDNState) or state.variant != self.variant:
            raise TypeError(f"state must be a KDNState of the {self.variant} variant")
        if state.num_heads != H or state.head_dim != self.head_dim:
            raise ValueError(f"state holds {state.num_heads} heads of {state.head_dim}, the step {H} of {self.head_dim}")
        if qkv.ndim != 2 or qkv.shape[1] != GROUPS * channels:
            raise ValueError(f"qkv must be [B, {GROUPS * channels}], got {tuple(qkv.shape)}")
        B, device = qkv.shape[0], qkv.device
        if dtype not in _ACT_DTYPES or dtype != state.window.dtype:
            raise TypeError(f"qkv must be bf16 or fp32 as the state's window ({state.window.dtype}), got {dtype}")
        if qkv.stride(1) != 1:
            raise ValueError(f"qkv's rows must be contiguous, got strides {qkv.stride()}")
        for name, t, width in rows:
            if t.ndim != 2 or t.shape[0] != B or t.shape[1] != width:
                raise ValueError(f"{name} must be {(B, width)}, got {tuple(t.shape)}")
            if t.dtype is not dtype:
                raise TypeError(f"{name} must have qkv's dtype {dtype}, got {t.dtype}")
            if t.stride(1) != 1 and width > 1:
                raise ValueError(f"{name}'s rows must be contiguous, got strides {t.stride()}")
            if t.device != device:
                raise ValueError("all step tensors must share one CUDA device")
        if slots is None:
            if state.num_slots < B:
                raise ValueError(f"without slots the pool must hold {B} states, got {state.num_slots}")
        else:
            if slots.ndim != 1 or slots.shape[0] != B or slots.dtype not in _SLOT_DTYPES or not slots.is_contiguous():
                raise ValueError(f"slots must be a contiguous int32 or int64 [{B}] tensor, got {tuple(slots.shape)} "
                                 f"{slots.dtype}")
            if slots.device != device:
                raise ValueError("all step tensors must share one CUDA device")
        if state.memory.device != device or self.device != device:
            raise ValueError("all step tensors must share one CUDA device")
        if not qkv.is_cuda:
            N.require_cuda(qkv)
        inputs = (qkv, *(t for _, t, _ in rows))
        if N.has_tangent(*inputs):
            raise NotImplementedError("kdn_b200 step: the token step has no jvp (forward-mode derivative)")
        if torch.is_grad_enabled() and any([t.requires_grad for t in inputs]):
            return _StepFunction.apply(lambda: self._launch(state, slots, *inputs), *inputs)
        return self._launch(state, slots, *inputs)

    def _launch(self, state, slots, qkv, *rows):
        lib = N.load_library()
        B = qkv.shape[0]
        y = qkv.new_empty((B, self.num_heads * self.head_dim))
        a = N.KdnStepArgs.from_buffer_copy(self._args)
        a.act_bf16 = qkv.dtype == torch.bfloat16
        a.B, a.num_slots = B, state.num_slots
        a.qkv, a.qkv_stride = qkv.data_ptr(), qkv.stride(0)
        self._rows(a, *rows)
        if slots is not None:
            a.slots, a.slots_i64 = slots.data_ptr(), slots.dtype == torch.int64
        a.memory, a.covariance = state.memory.data_ptr(), state.covariance.data_ptr()
        a.window, a.y = state.window.data_ptr(), y.data_ptr()
        N.launch(lib.kdn_step, a, qkv, "kdn_step")
        return y


class IsoKDNStep(_Step):
    """The isotropic mixer's token step.

    conv_weight [3*H*D, 4] (the packed q | k | v convolution), A_log [H],
    dt_bias [H*D], norm_weight [D] or None (the output norm's), omega_bias and
    r_bias [H]; omega_min, r_min, info_scale as the gate frontend and
    ``iso_kdn_gain`` take them; activation and norm_eps of the output norm.
    """

    variant = "iso"

    def __init__(self, conv_weight, A_log, dt_bias, norm_weight, *, omega_bias, r_bias, omega_min, r_min,
                 info_scale=None, norm_eps=1e-5, activation="sigmoid"):
        D = conv_weight.shape[0] // GROUPS // max(A_log.shape[0] if A_log.ndim else 0, 1)
        scale = 1.0
        if info_scale is not None:
            scale = _finite("info_scale", info_scale) / max(D, 1)
            if scale <= 0:
                raise ValueError(f"info_scale must be positive and finite, got {info_scale!r}")
        super().__init__(conv_weight, A_log, dt_bias, norm_weight, omega_bias, r_bias, omega_min, r_min, scale,
                         norm_eps, activation)

    def __call__(self, state, qkv, decay_raw, omega_r_raw, out_gate, slots=None):
        """One token per row: qkv [B, 3*H*D], decay_raw [B, H*D], omega_r_raw [B, 2*H] (omega | r), out_gate [B, H*D],
        all of one dtype (bf16 or fp32, the window's), rows contiguous and apart (or one for all); slots [B] int32 / int64
        (None: row b uses slot b; a slot outside the pool marks an idle row, output zero; no slot twice).
        Returns y [B, H*D] and updates the states in place."""
        fast = N.host()
        if fast is not None and self._fits(state, qkv):
            y = fast.step(self._args, state.memory, state.covariance, state.window, qkv, decay_raw, omega_r_raw, None,
                          out_gate, slots)
            if y is not None:
                return y
        H = self.num_heads
        channels = H * self.head_dim
        return self._run(state, slots, qkv, (("decay_raw", decay_raw, channels), ("omega_r_raw", omega_r_raw, 2 * H),
                                             ("out_gate", out_gate, channels)))

    def _rows(self, a, decay_raw, omega_r_raw, out_gate):
        a.decay_raw, a.decay_stride = decay_raw.data_ptr(), decay_raw.stride(0)
        a.omega_raw, a.omega_stride = omega_r_raw.data_ptr(), omega_r_raw.stride(0)
        a.r_raw = omega_r_raw.data_ptr() + self.num_heads * omega_r_raw.element_size()  # the row's second half
        a.r_stride = omega_r_raw.stride(0)
        a.gate, a.gate_stride = out_gate.data_ptr(), out_gate.stride(0)


class DiagKDNStep(_Step):
    """The diagonal mixer's token step: conv_weight [3*H*D, 4] (the q, k and v
    convolutions' weights one after the other), A_log [H], dt_bias [H*D] or
    [H, D], norm_weight [D] or None."""

    variant = "diag"

    def __init__(self, conv_weight, A_log, dt_bias, norm_weight, *, norm_eps=1e-5, activation="sigmoid"):
        super().__init__(conv_weight, A_log, dt_bias, norm_weight, None, None, 0.0, DIAG_R_MIN, 1.0, norm_eps,
                         activation)

    def __call__(self, state, qkv, retention_raw, omega_raw, r_raw, out_gate, slots=None):
        """As :meth:`IsoKDNStep.__call__`, with retention_raw and omega_raw [B, H*D] and r_raw [B, H]."""
        fast = N.host()
        if fast is not None and self._fits(state, qkv):
            y = fast.step(self._args, state.memory, state.covariance, state.window, qkv, retention_raw, omega_raw, r_raw,
                          out_gate, slots)
            if y is not None:
                return y
        channels = self.num_heads * self.head_dim
        return self._run(state, slots, qkv, (("retention_raw", retention_raw, channels),
                                             ("omega_raw", omega_raw, channels), ("r_raw", r_raw, self.num_heads),
                                             ("out_gate", out_gate, channels)))

    def _rows(self, a, retention_raw, omega_raw, r_raw, out_gate):
        a.decay_raw, a.decay_stride = retention_raw.data_ptr(), retention_raw.stride(0)
        a.omega_raw, a.omega_stride = omega_raw.data_ptr(), omega_raw.stride(0)
        a.r_raw, a.r_stride = r_raw.data_ptr(), r_raw.stride(0)
        a.gate, a.gate_stride = out_gate.data_ptr(), out_gate.stride(0)


__all__ = ("KDNState", "IsoKDNStep", "DiagKDNStep")
