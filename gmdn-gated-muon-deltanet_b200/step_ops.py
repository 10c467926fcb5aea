"""Operators of the training step around the mixer, on the library's own kernels.

``layer_norm(x, weight, bias, eps)`` / ``rms_norm(x, weight, bias, eps)``
    the norm over the model width, optionally of ``x + residual`` (a block's
    residual add and the norm after it in one pass, train_ablation.py:197-246),
    differentiable in the input, the residual, the weight and the bias.

``token_logprobs(logits, targets)``
    log probability of a given token per row of logits, with the row's entropy
    and its top alternatives, differentiable in the logits (the trainer's loss
    is minus its mean, train_ablation.py:197-246).

``pack8`` / ``unpack8``, ``act8_forward`` / ``act8_backward``, ``mlp8``
    activations kept in 8 bits between the forward and the backward: any
    tensor; a GELU or SwiGLU whose backward reads the checkpoint; and an MLP
    whose saved activations are all 8-bit (train_ablation.py:202-205).

Derivatives are of the first order and reverse mode; second ones, and forward
mode, raise.  All run only on CUDA tensors, bf16 or fp32, through
``libgmdn_b200.so``.  The
operators below them are registered in C++ (``csrc/torch_ops.cpp``) with their
autograd formulas; here are their fake kernels (for torch.compile), the
arguments' checks and the public names.
"""

from __future__ import annotations

import math
from typing import NamedTuple, Optional

import torch
import torch.nn.functional as F
from torch import Tensor
from torch.autograd.forward_ad import unpack_dual
from torch.autograd.function import once_differentiable

from ._lib import load_torch_ops
from .ops import _f32_flag, _require_cuda

__all__ = ["layer_norm", "rms_norm", "token_logprobs", "TokenLogprobs", "pack8", "unpack8",
           "Packed8", "act8_forward", "act8_backward", "Act8Saved", "mlp8"]

# The mixer's ops need libgmdn_b200.so alone: without libgmdn_torch.so the package still imports,
# and the calls of this module raise why.
try:
    load_torch_ops()
    _unloaded = None
except ImportError as e:
    _unloaded = str(e)


def _op(name: str):
    if _unloaded is None:
        return getattr(torch.ops.gmdn, name).default

    def missing(*_args):
        raise ImportError(_unloaded)
    return missing


def _register_fake(name: str):
    return torch.library.register_fake(f"gmdn::{name}") if _unloaded is None else lambda f: f


_norm_fwd = _op("norm_fwd")
_token_logprobs_fwd = _op("token_logprobs_fwd")
_pack8, _unpack8 = _op("pack8"), _op("unpack8")
_act8_fwd, _act8_bwd = _op("act8_fwd"), _op("act8_bwd")
MAX_TOP_K = 64
BLOCK8 = 128   # consecutive elements that share a scale


def _same_device(name: str, first: Tensor, *others: Optional[Tensor]) -> None:
    """Every tensor on one CUDA device: a kernel would fault on another's memory."""
    device = first.device
    if device.type != "cuda":
        _require_cuda(name, first)
    for t in others:
        if t is not None and t.device != device:
            _require_cuda(name, t)
            raise ValueError(f"{name}: tensors on {device} and {t.device}")


# ---------------------------------------------------------------------------
# norm over the model width
# ---------------------------------------------------------------------------

@_register_fake("norm_fwd")
def _(x, residual, weight, bias, eps, center, out_f32):
    D = x.shape[-1]
    y = x.new_empty(x.shape, dtype=torch.float32 if out_f32 else torch.bfloat16)
    if residual is None:
        h = x.new_empty(0)
    else:
        h = x.new_empty(x.shape, dtype=torch.promote_types(x.dtype, residual.dtype))
    return y, h, x.new_empty(2 if center else 1, x.numel() // D if D else 0, dtype=torch.float32)


@_register_fake("norm_bwd")
def _(s, stats, weight, dy, dh, center, want_bf16, want_f32, want_w, want_b):
    def out(wanted, dtype, shape):
        return s.new_empty(shape if wanted else (0,), dtype=dtype)

    D = s.shape[-1]
    return (out(want_bf16, torch.bfloat16, s.shape), out(want_f32, torch.float32, s.shape),
            out(want_w, torch.float32, (D,)), out(want_b, torch.float32, (D,)))


def _norm(name: str, center: bool, x: Tensor, weight: Optional[Tensor], bias: Optional[Tensor],
          eps: float, residual: Optional[Tensor], out_dtype: Optional[torch.dtype]):
    if x.dim() < 1:
        raise ValueError(f"{name}: x must have a last axis to normalise")
    D = x.shape[-1]
    for what, t in (("weight", weight), ("bias", bias)):
        if t is not None and t.shape != (D,):
            raise ValueError(f"{name}: {what} must be ({D},), got {tuple(t.shape)}")
    if residual is not None and residual.shape != x.shape:
        raise ValueError(f"{name}: residual {tuple(residual.shape)} != x {tuple(x.shape)}")
    if not eps >= 0.0:
        raise ValueError(f"{name}: eps must be >= 0, got {eps}")
    _f32_flag(x, "x")
    if residual is not None:
        _f32_flag(residual, "residual")
    out_dtype = x.dtype if out_dtype is None else out_dtype
    if out_dtype not in (torch.bfloat16, torch.float32):
        raise TypeError(f"out_dtype must be bfloat16 or float32, got {out_dtype}")
    _same_device(name, x, weight, bias, residual)
    # the parameters' casts are differentiable: their gradients come back in their own types
    if weight is not None and weight.dtype != torch.float32:
        weight = weight.float()
    if bias is not None and bias.dtype != torch.float32:
        bias = bias.float()
    y, h, _ = _norm_fwd(x, residual, weight, bias, eps, center, out_dtype == torch.float32)
    return y if residual is None else (y, h)


def layer_norm(x: Tensor, weight: Optional[Tensor] = None, bias: Optional[Tensor] = None,
               eps: float = 1e-5, *, residual: Optional[Tensor] = None,
               out_dtype: Optional[torch.dtype] = None):
    """Layer norm of x, or of x + residual, over the last axis.

    x: (..., D), bf16 or fp32, any D; weight, bias: (D,) or None; residual:
    like x in shape, bf16 or fp32 of its own.  Returns y (..., D) in out_dtype
    (default x's); with a residual (y, h) where h = x + residual in fp32 if
    either is fp32, and the norm reads the rounded h.  Statistics and sums are
    fp32, y is rounded once.  Differentiable in x, residual, weight and bias;
    the parameters' gradients are summed in a fixed order (equal calls give
    equal bits).
    """
    return _norm("layer_norm", True, x, weight, bias, eps, residual, out_dtype)


def rms_norm(x: Tensor, weight: Optional[Tensor] = None, bias: Optional[Tensor] = None,
             eps: Optional[float] = None, *, residual: Optional[Tensor] = None,
             out_dtype: Optional[torch.dtype] = None):
    """``layer_norm`` without the mean: y = s / sqrt(mean(s^2) + eps) * weight
    [+ bias], s = x or x + residual.  eps: None for nn.RMSNorm's default
    (float32 machine epsilon)."""
    return _norm("rms_norm", False, x, weight, bias,
                 torch.finfo(torch.float32).eps if eps is None else eps, residual, out_dtype)


# ---------------------------------------------------------------------------
# token log probabilities
# ---------------------------------------------------------------------------

class TokenLogprobs(NamedTuple):
    """What ``token_logprobs`` returns; a field that was not asked for is None."""
    logprobs: Optional[Tensor]       # (...) fp32
    entropy: Optional[Tensor]        # (...) fp32
    top_logprobs: Optional[Tensor]   # (..., top_k) fp32, falling
    top_ids: Optional[Tensor]        # (..., top_k) int64


@_register_fake("token_logprobs_fwd")
def _(logits, targets, entropy, top_k, ignore_index):
    shape = logits.shape[:-1]

    def out(wanted, size, dtype=torch.float32):
        return logits.new_empty(size if wanted else (0,), dtype=dtype)

    return (out(targets is not None, shape), out(entropy, shape),
            out(top_k > 0, (*shape, top_k)), out(top_k > 0, (*shape, top_k), torch.int64),
            logits.new_empty(*shape, 4, dtype=torch.float32))


@_register_fake("token_logprobs_bwd")
def _(logits, targets, ids, stats, g_lp, g_ent, g_top, ignore_index):
    return logits.new_empty(logits.shape)


def token_logprobs(logits: Tensor, targets: Optional[Tensor] = None, *, entropy: bool = False,
                   top_k: int = 0, ignore_index: int = -100) -> TokenLogprobs:
    """Log probability of a given token for each row of logits, in one pass.

    logits: (..., V), bf16 or fp32; rows may be strided (a shifted view such as
    ``logits[:, :-1]`` or the live columns of a padded head is read in place).
    targets: (...) int64 or int32, or None for no log probabilities; a target
    equal to ignore_index gives 0 and no gradient, any other outside [0, V)
    gives NaN.  A row whose cotangents are all 0 has a zero gradient whatever it
    holds.  entropy: also the entropy of each row's distribution.  top_k:
    also the log probabilities and columns of the top_k (at most 64) largest
    logits, falling, ties to the lowest column.

    A column at -inf has probability 0; a row of nothing else has log
    probability -inf, entropy 0 and a zero gradient.  A row that holds a NaN or
    +inf gives NaN.  Differentiable in the logits through logprobs, entropy and
    top_logprobs.
    """
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError(f"logits must be (..., V) with V >= 1, got {tuple(logits.shape)}")
    V = logits.shape[-1]
    _f32_flag(logits, "logits")
    if not 0 <= top_k <= min(MAX_TOP_K, V):
        raise ValueError(f"top_k must be in [0, min({MAX_TOP_K}, V = {V})], got {top_k}")
    if targets is None and not entropy and not top_k:
        raise ValueError("token_logprobs: nothing asked for (no targets, entropy or top_k)")
    if targets is not None:
        if targets.shape != logits.shape[:-1]:
            raise ValueError(f"targets must be {tuple(logits.shape[:-1])}, "
                             f"got {tuple(targets.shape)}")
        if targets.dtype not in (torch.int64, torch.int32):
            raise TypeError(f"targets must be int64 or int32, got {targets.dtype}")
    _same_device("token_logprobs", logits, targets)
    if targets is not None and targets.dtype == torch.int32:
        targets = targets.long()
    lp, ent, tops, ids, _ = _token_logprobs_fwd(logits, targets, bool(entropy), int(top_k),
                                                int(ignore_index))
    return TokenLogprobs(None if targets is None else lp, ent if entropy else None,
                         tops if top_k else None, ids if top_k else None)


# ---------------------------------------------------------------------------
# activations in 8 bits
# ---------------------------------------------------------------------------

class Packed8(NamedTuple):
    """A tensor in 8 bits: codes int8 in its shape, one fp32 scale for each 128
    consecutive elements, and the type it comes back in."""
    codes: Tensor
    scales: Tensor
    dtype: torch.dtype


class Act8Saved(NamedTuple):
    """The 8-bit checkpoint of an activation's inputs (gate: SwiGLU only)."""
    x: Packed8
    gate: Optional[Packed8]


def _codes_like(x):
    return (x.new_empty(x.shape, dtype=torch.int8),
            x.new_empty((x.numel() + BLOCK8 - 1) // BLOCK8, dtype=torch.float32))


@_register_fake("pack8")
def _(x):
    return _codes_like(x)


@_register_fake("unpack8")
def _(codes, scales, f32):
    return codes.new_empty(codes.shape, dtype=torch.float32 if f32 else torch.bfloat16)


@_register_fake("act8_fwd")
def _(x, gate):
    codes, scales = _codes_like(x)
    g = (codes.new_empty(0), scales.new_empty(0)) if gate is None else _codes_like(x)
    return x.new_empty(x.shape), codes, scales, *g


@_register_fake("act8_bwd")
def _(codes, scales, gcodes, gscales, dy, restore):
    return (dy.new_empty(dy.shape), dy.new_empty(dy.shape if gcodes is not None else 0),
            dy.new_empty(dy.shape if restore else 0))


def _check_packed(name: str, p: Packed8) -> None:
    if p.codes.dtype != torch.int8 or p.scales.dtype != torch.float32:
        raise TypeError(f"{name}: codes must be int8 and scales float32, got {p.codes.dtype} and "
                        f"{p.scales.dtype}")
    if p.dtype not in (torch.bfloat16, torch.float32):
        raise TypeError(f"{name}: a checkpoint comes back in bfloat16 or float32, not {p.dtype}")
    if p.scales.dim() != 1 or p.scales.numel() != (p.codes.numel() + BLOCK8 - 1) // BLOCK8:
        raise ValueError(f"{name}: {tuple(p.codes.shape)} codes need one scale for each {BLOCK8} "
                         f"elements, got {tuple(p.scales.shape)}")


def pack8(x: Tensor) -> Packed8:
    """x (bf16 or fp32, any shape) in 8 bits.  128 consecutive elements share a
    scale, a = their largest magnitude: an element comes back as
    round(x * 127 / a) * a / 127, off by at most a / 254 and rounding.  Blocks
    with a below 2^-100 come back as zeros, blocks that hold a NaN or an
    infinity as NaN.  Not differentiable: the result is a checkpoint."""
    _f32_flag(x, "x")
    _require_cuda("pack8", x)
    return Packed8(*_pack8(x.detach()), x.dtype)


def unpack8(packed: Packed8) -> Tensor:
    """The tensor that ``pack8`` kept, in its shape and type."""
    _check_packed("unpack8", packed)
    _same_device("unpack8", packed.codes, packed.scales)
    return _unpack8(packed.codes, packed.scales, packed.dtype == torch.float32)


def act8_forward(x: Tensor, gate: Optional[Tensor] = None) -> tuple[Tensor, Act8Saved]:
    """GELU(x) (exact), or SiLU(gate) * x with a gate, and the 8-bit checkpoint
    of its inputs for ``act8_backward``.  x, gate: one shape and type, bf16 or
    fp32.  Not seen by autograd, in reverse or forward mode (``mlp8`` is the
    differentiable form)."""
    _f32_flag(x, "x")
    if gate is not None and (gate.shape != x.shape or gate.dtype != x.dtype):
        raise ValueError(f"gate must be like x, {tuple(x.shape)} {x.dtype}, got "
                         f"{tuple(gate.shape)} {gate.dtype}")
    _same_device("act8_forward", x, gate)
    y, codes, scales, gcodes, gscales = _act8_fwd(
        x.detach(), None if gate is None else gate.detach())
    return y, Act8Saved(Packed8(codes, scales, x.dtype),
                        None if gate is None else Packed8(gcodes, gscales, x.dtype))


def act8_backward(saved: Act8Saved, dy: Tensor, restore: bool = True):
    """(dx, dgate, y) from the checkpoint of ``act8_forward`` and the cotangent
    dy: dgate is None without a gate; y is the activation of the restored
    inputs (for the weight gradient of the projection that read it), None
    unless restore."""
    x, gate = saved
    _check_packed("act8_backward", x)
    if dy.shape != x.codes.shape or dy.dtype != x.dtype:
        raise ValueError(f"dy must be {tuple(x.codes.shape)} {x.dtype}, got {tuple(dy.shape)} "
                         f"{dy.dtype}")
    if gate is not None:
        _check_packed("act8_backward", gate)
        if gate.codes.shape != x.codes.shape or gate.dtype != x.dtype:
            raise ValueError("act8_backward: the gate's checkpoint is not like the input's")
    parts = [x.codes, x.scales] + ([None, None] if gate is None else [gate.codes, gate.scales])
    _same_device("act8_backward", dy, *parts)
    dx, dgate, y = _act8_bwd(*parts, dy.detach(), bool(restore))
    return dx, dgate if gate is not None else None, y if restore else None


def _has_tangent(*tensors: Optional[Tensor]) -> bool:
    """A forward-mode tangent on any of them (it needs no requires_grad)."""
    return any(t is not None and unpack_dual(t).tangent is not None for t in tensors)


def _rows(t: Tensor) -> Tensor:
    """(..., D) as a matrix; a D of 0 leaves nothing to infer the rows from."""
    return t.reshape(math.prod(t.shape[:-1]), t.shape[-1])


class _Mlp8Function(torch.autograd.Function):
    """down(act(up x)) that keeps x and the activation's inputs in 8 bits; the
    weight gradients are products with the restored tensors."""

    @staticmethod
    def forward(ctx, x, w_up, w_down, w_gate):
        rows = _rows(x)
        up = F.linear(rows, w_up)
        y, saved = act8_forward(up, None if w_gate is None else F.linear(rows, w_gate))
        kept = pack8(rows) if w_up.requires_grad or (w_gate is not None and w_gate.requires_grad) \
            else None
        ctx.dtype, ctx.shape, ctx.gated = x.dtype, x.shape, w_gate is not None
        ctx.kept = kept is not None
        ctx.save_for_backward(w_up, w_down, w_gate, saved.x.codes, saved.x.scales,
                              *(saved.gate[:2] if ctx.gated else ()),
                              *(kept[:2] if ctx.kept else ()))
        return F.linear(y, w_down).view(*x.shape[:-1], w_down.shape[0])

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        if _has_tangent(dout):
            raise RuntimeError("mlp8: no forward-mode derivative of its backward")
        # the products in the forward's type, whatever the caller's autocast asks for
        with torch.autocast("cuda", enabled=False):
            return _Mlp8Function.grads(ctx, dout)

    @staticmethod
    def grads(ctx, dout):
        w_up, w_down, w_gate, codes, scales, *more = ctx.saved_tensors
        gate = Packed8(*more[:2], ctx.dtype) if ctx.gated else None
        saved = Act8Saved(Packed8(codes, scales, ctx.dtype), gate)
        need = ctx.needs_input_grad
        dout = _rows(dout).to(ctx.dtype)
        dup, dgate, y = act8_backward(saved, dout @ w_down, restore=need[2])
        dx = dw_up = dw_gate = dw_down = None
        if need[2]:
            dw_down = dout.mT @ y
        if ctx.kept:
            rows = unpack8(Packed8(*more[-2:], ctx.dtype))
            dw_up = dup.mT @ rows if need[1] else None
            dw_gate = dgate.mT @ rows if ctx.gated and need[3] else None
        if need[0]:
            dx = dup @ w_up
            if ctx.gated:
                dx = torch.addmm(dx, dgate, w_gate)
            dx = dx.view(ctx.shape)
        return dx, dw_up, dw_down, dw_gate


def mlp8(x: Tensor, w_up: Tensor, w_down: Tensor, w_gate: Optional[Tensor] = None) -> Tensor:
    """GELU(x w_up^T) w_down^T, or (SiLU(x w_gate^T) * (x w_up^T)) w_down^T, whose
    saved activations are 8-bit: x and the activation's inputs, 1 byte an
    element instead of the 2 or 4 of each plus the activation's output that
    autograd keeps.  The forward is not changed by the checkpoint; the weight
    gradients and the activation's derivative read the restored tensors.

    x: (..., D); w_up, w_gate: (F, D); w_down: (D_out, F); one type, bf16 or
    fp32 (under autocast they are cast to its type first, as nn.Linear's are).
    """
    weights = [w_up, w_down] + ([] if w_gate is None else [w_gate])
    if x.dim() < 1 or any(w.dim() != 2 for w in weights):
        raise ValueError("mlp8: x must be (..., D) and the weights matrices")
    if w_up.shape[1] != x.shape[-1] or w_down.shape[1] != w_up.shape[0] or \
            (w_gate is not None and w_gate.shape != w_up.shape):
        raise ValueError(f"mlp8: x {tuple(x.shape)} does not fit w_up {tuple(w_up.shape)}, w_down "
                         f"{tuple(w_down.shape)}"
                         + ("" if w_gate is None else f", w_gate {tuple(w_gate.shape)}"))
    _same_device("mlp8", x, *weights)
    if torch.is_autocast_enabled("cuda"):
        dt = torch.get_autocast_dtype("cuda")
        x, w_up, w_down = x.to(dt), w_up.to(dt), w_down.to(dt)
        w_gate = None if w_gate is None else w_gate.to(dt)
    _f32_flag(x, "x")
    for w in (w_up, w_down, w_gate):
        if w is not None and w.dtype != x.dtype:
            raise TypeError(f"mlp8: x is {x.dtype}, a weight {w.dtype}")
    recorded = torch.is_grad_enabled() and any(t.requires_grad for t in (x, *weights))
    # a tangent goes to autograd too, which refuses it
    if not recorded and not _has_tangent(x, *weights):
        y, _ = act8_forward(F.linear(x, w_up), None if w_gate is None else F.linear(x, w_gate))
        return F.linear(y, w_down)
    return _Mlp8Function.apply(x, w_up, w_down, w_gate)
