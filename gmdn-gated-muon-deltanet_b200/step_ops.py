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

All run only on CUDA tensors, bf16 or fp32, through ``libgmdn_b200.so``.  Like
the mixer's, each is a torch.library custom op with a fake kernel (and autograd
where it is differentiable), which torch.compile and dispatch modes see; an
eager call on plain tensors goes to the library directly, because the
dispatcher's bookkeeping costs more than a small call's kernel.
"""

from __future__ import annotations

from typing import NamedTuple, Optional

import torch
import torch.nn.functional as F
from torch import Tensor
from torch.autograd.function import once_differentiable

from ._lib import check, lib
from .ops import _aligned, _f32_flag, _require_cuda

__all__ = ["layer_norm", "rms_norm", "token_logprobs", "TokenLogprobs", "pack8", "unpack8",
           "Packed8", "act8_forward", "act8_backward", "Act8Saved", "mlp8"]

MAX_TOP_K = 64
_PLAIN = (Tensor, torch.nn.Parameter, type(None))


def _eager(*tensors: Optional[Tensor]) -> bool:
    """Plain tensors, no tracing and no dispatch mode: nothing else has to see
    the call, so it may go to the library directly."""
    if torch.compiler.is_compiling() or torch._C._len_torch_dispatch_stack():
        return False
    for t in tensors:
        if type(t) not in _PLAIN:
            return False
    return True


def _run(what: str, fn, device: torch.device, *args) -> None:
    """The library call on the device's current stream, with that device current."""
    index = device.index
    if index == torch._C._cuda_getDevice():
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        check(rc, what)


def _at(t: Optional[Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _same_device(name: str, first: Tensor, *others: Optional[Tensor]) -> None:
    """Every tensor on one CUDA device: a kernel would fault on another's memory."""
    device = first.device
    if device.type != "cuda":
        _require_cuda(name, first)
    for t in others:
        if t is not None and t.device != device:
            _require_cuda(name, t)
            raise ValueError(f"{name}: tensors on {device} and {t.device}")


def _once(backward):
    """A Function's backward without a second derivative: asking for one (grad
    mode on) raises when it is used.  The wrapper that does this is left out
    where grad mode is off, as in every plain backward."""
    strict = once_differentiable(backward)

    def run(ctx, *grads):
        return strict(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)

    return staticmethod(run)


def _needs_grad(*tensors: Optional[Tensor]) -> bool:
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


# ---------------------------------------------------------------------------
# norm over the model width
# ---------------------------------------------------------------------------

def _norm_fwd_call(x: Tensor, residual: Optional[Tensor], weight: Optional[Tensor],
                   bias: Optional[Tensor], eps: float, center: bool,
                   out_f32: bool) -> tuple[Tensor, Optional[Tensor], Tensor]:
    D = x.shape[-1]
    rows = x.numel() // D if D else 0
    y = torch.empty_like(x, dtype=torch.float32 if out_f32 else torch.bfloat16)
    h = None
    if residual is not None:
        h = torch.empty_like(residual if residual.dtype == torch.float32 else x)
    stats = torch.empty((2 if center else 1, rows), dtype=torch.float32, device=x.device)
    at = stats.data_ptr()
    _run("gmdn_norm_fwd", lib.gmdn_norm_fwd, x.device, x.data_ptr(), _at(residual), _at(weight),
         _at(bias), y.data_ptr(), _at(h), at, at + 4 * rows if center else None, rows, D, eps,
         center, x.dtype == torch.float32,
         residual is not None and residual.dtype == torch.float32, out_f32)
    return y, h, stats


def _norm_bwd_call(s: Tensor, stats: Tensor, weight: Optional[Tensor], dy: Tensor,
                   dh: Optional[Tensor], center: bool, want_bf16: bool, want_f32: bool,
                   want_w: bool, want_b: bool) -> tuple[Optional[Tensor], ...]:
    D = s.shape[-1]
    rows = s.numel() // D if D else 0

    da = torch.empty_like(s, dtype=torch.bfloat16) if want_bf16 else None
    db = torch.empty_like(s, dtype=torch.float32) if want_f32 else None
    dweight = torch.empty(D, dtype=torch.float32, device=s.device) if want_w else None
    dbias = torch.empty(D, dtype=torch.float32, device=s.device) if want_b else None
    nbytes = lib.gmdn_norm_bwd_workspace_bytes(rows, D) if want_w or want_b else 0
    ws = torch.empty(nbytes, dtype=torch.uint8, device=s.device) if nbytes else None
    at = stats.data_ptr()
    _run("gmdn_norm_bwd", lib.gmdn_norm_bwd, s.device, s.data_ptr(), at,
         at + 4 * rows if center else None, _at(weight), dy.data_ptr(), _at(dh),
         _at(da), _at(db), _at(dweight), _at(dbias), _at(ws), nbytes, rows, D, center, s.dtype == torch.float32, dy.dtype == torch.float32,
         dh is not None and dh.dtype == torch.float32, False, True)
    return da, db, dweight, dbias


@torch.library.custom_op("gmdn::norm_fwd", mutates_args=())
def _norm_fwd(x: Tensor, residual: Optional[Tensor], weight: Optional[Tensor],
              bias: Optional[Tensor], eps: float, center: bool,
              out_f32: bool) -> tuple[Tensor, Tensor, Tensor]:
    y, h, stats = _norm_fwd_call(x, residual, weight, bias, eps, center, out_f32)
    return y, x.new_empty(0) if h is None else h, stats


@_norm_fwd.register_fake
def _(x, residual, weight, bias, eps, center, out_f32):
    D = x.shape[-1]
    y = x.new_empty(x.shape, dtype=torch.float32 if out_f32 else torch.bfloat16)
    h = x.new_empty(0) if residual is None else \
        torch.empty_like(residual if residual.dtype == torch.float32 else x)
    return y, h, x.new_empty(2 if center else 1, x.numel() // D if D else 0, dtype=torch.float32)


@torch.library.custom_op("gmdn::norm_bwd", mutates_args=())
def _norm_bwd(s: Tensor, stats: Tensor, weight: Optional[Tensor], dy: Tensor,
              dh: Optional[Tensor], center: bool, want_bf16: bool, want_f32: bool, want_w: bool,
              want_b: bool) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    got = _norm_bwd_call(s, stats, weight, dy, dh, center, want_bf16, want_f32, want_w, want_b)
    types = (torch.bfloat16, torch.float32, torch.float32, torch.float32)
    return tuple(s.new_empty(0, dtype=t) if g is None else g for g, t in zip(got, types))


@_norm_bwd.register_fake
def _(s, stats, weight, dy, dh, center, want_bf16, want_f32, want_w, want_b):
    def out(wanted, dtype, shape):
        return s.new_empty(shape if wanted else (0,), dtype=dtype)

    D = s.shape[-1]
    return (out(want_bf16, torch.bfloat16, s.shape), out(want_f32, torch.float32, s.shape),
            out(want_w, torch.float32, (D,)), out(want_b, torch.float32, (D,)))


def _norm_setup(ctx, inputs, output):
    x, residual, weight, bias, eps, center, out_f32 = inputs
    _, h, stats = output
    ctx.save_for_backward(x if residual is None else h, stats, weight)
    ctx.types = (x.dtype, None if residual is None else residual.dtype)
    ctx.center, ctx.out_f32 = center, out_f32
    ctx.set_materialize_grads(False)


def _norm_backward(ctx, dy, dh, _dstats):
    s, stats, weight = ctx.saved_tensors
    dy_type = torch.float32 if ctx.out_f32 else torch.bfloat16
    dy = torch.zeros_like(s, dtype=dy_type) if dy is None else _aligned(dy.to(dy_type))
    if ctx.types[1] is None:
        dh = None   # without a residual, h is a placeholder
    elif dh is not None:
        dh = _aligned(dh)
    need = ctx.needs_input_grad
    wanted = [t for t, n in zip(ctx.types, need) if n]
    call = _norm_bwd_call if _eager(s, dy, dh) else torch.ops.gmdn.norm_bwd
    da, db, dweight, dbias = call(s, stats, weight, dy, dh, ctx.center, torch.bfloat16 in wanted,
                                  torch.float32 in wanted, need[2], need[3])
    of = {torch.bfloat16: da, torch.float32: db, None: None}
    return (of[ctx.types[0]] if need[0] else None, of[ctx.types[1]] if need[1] else None,
            dweight if need[2] else None, dbias if need[3] else None, None, None, None)


_norm_fwd.register_autograd(_norm_backward, setup_context=_norm_setup)


class _NormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, *args):
        got = _norm_fwd_call(*args)
        _norm_setup(ctx, args, got)
        return got

    backward = _once(_norm_backward)


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
    args = (_aligned(x), None if residual is None else _aligned(residual),
            None if weight is None else _aligned(weight.float()),
            None if bias is None else _aligned(bias.float()), float(eps), center,
            out_dtype == torch.float32)
    if not _eager(*args[:4]):
        y, h, _ = torch.ops.gmdn.norm_fwd(*args)
    elif _needs_grad(*args[:4]):
        y, h, _ = _NormFunction.apply(*args)
    else:
        y, h, _ = _norm_fwd_call(*args)
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


def _rows_of(logits: Tensor):
    """(batch, length, stride_b, stride_t) of the rows of a tensor whose rows
    are contiguous, or None where two strides do not reach every row."""
    dims = [(n, s) for n, s in zip(logits.shape[:-1], logits.stride()[:-1]) if n != 1]
    if logits.shape[-1] > 1 and logits.stride(-1) != 1:
        return None
    merged: list = []
    for n, s in dims:
        if merged and merged[-1][1] == n * s:
            merged[-1] = (merged[-1][0] * n, s)
        else:
            merged.append((n, s))
    if len(merged) > 2:
        return None
    while len(merged) < 2:
        merged.insert(0, (1, 0))
    (b, sb), (t, st) = merged
    return b, t, sb, st


def _logprobs_fwd_call(logits: Tensor, targets: Optional[Tensor], entropy: bool, top_k: int,
                       ignore_index: int) -> tuple[Optional[Tensor], ...]:
    shape, V = logits.shape[:-1], logits.shape[-1]
    if (rows := _rows_of(logits)) is None:
        logits = logits.contiguous()
        rows = _rows_of(logits)

    stats = torch.empty((*shape, 4), dtype=torch.float32, device=logits.device)
    lp = stats.new_empty(shape) if targets is not None else None
    ent = stats.new_empty(shape) if entropy else None
    tops = ids = None
    if top_k:
        tops = stats.new_empty((*shape, top_k))
        ids = torch.empty((*shape, top_k), dtype=torch.int64, device=logits.device)
    b, t, sb, st = rows
    _run("gmdn_token_logprobs_fwd", lib.gmdn_token_logprobs_fwd, logits.device, logits.data_ptr(),
         _at(targets), _at(lp), _at(ent), _at(tops), _at(ids), stats.data_ptr(), b, t, sb, st, V,
         top_k, ignore_index, logits.dtype == torch.float32)
    return lp, ent, tops, ids, stats


def _logprobs_bwd_call(logits: Tensor, targets: Optional[Tensor], ids: Optional[Tensor],
                       stats: Tensor, g_lp: Optional[Tensor], g_ent: Optional[Tensor],
                       g_top: Optional[Tensor], ignore_index: int) -> Tensor:
    if (rows := _rows_of(logits)) is None:
        logits = logits.contiguous()
        rows = _rows_of(logits)
    grad = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    b, t, sb, st = rows
    _run("gmdn_token_logprobs_bwd", lib.gmdn_token_logprobs_bwd, logits.device, logits.data_ptr(),
         _at(targets), stats.data_ptr(), _at(ids), _at(g_lp), _at(g_ent), _at(g_top),
         grad.data_ptr(), b, t, sb, st, logits.shape[-1], 0 if g_top is None else g_top.shape[-1],
         ignore_index, logits.dtype == torch.float32)
    return grad


@torch.library.custom_op("gmdn::token_logprobs_fwd", mutates_args=())
def _logprobs_fwd(logits: Tensor, targets: Optional[Tensor], entropy: bool, top_k: int,
                  ignore_index: int) -> tuple[Tensor, Tensor, Tensor, Tensor, Tensor]:
    *got, stats = _logprobs_fwd_call(logits, targets, entropy, top_k, ignore_index)
    types = (torch.float32, torch.float32, torch.float32, torch.int64)
    return (*(logits.new_empty(0, dtype=t) if g is None else g for g, t in zip(got, types)), stats)


@_logprobs_fwd.register_fake
def _(logits, targets, entropy, top_k, ignore_index):
    shape = logits.shape[:-1]

    def out(wanted, size, dtype=torch.float32):
        return logits.new_empty(size if wanted else (0,), dtype=dtype)

    return (out(targets is not None, shape), out(entropy, shape),
            out(top_k > 0, (*shape, top_k)), out(top_k > 0, (*shape, top_k), torch.int64),
            logits.new_empty(*shape, 4, dtype=torch.float32))


@torch.library.custom_op("gmdn::token_logprobs_bwd", mutates_args=())
def _logprobs_bwd(logits: Tensor, targets: Optional[Tensor], ids: Optional[Tensor],
                  stats: Tensor, g_lp: Optional[Tensor], g_ent: Optional[Tensor],
                  g_top: Optional[Tensor], ignore_index: int) -> Tensor:
    return _logprobs_bwd_call(logits, targets, ids, stats, g_lp, g_ent, g_top, ignore_index)


@_logprobs_bwd.register_fake
def _(logits, targets, ids, stats, g_lp, g_ent, g_top, ignore_index):
    return logits.new_empty(logits.shape)


def _logprobs_setup(ctx, inputs, output):
    logits, targets, entropy, top_k, ignore_index = inputs
    _, _, _, ids, stats = output
    if ids is not None:
        ctx.mark_non_differentiable(ids)
    ctx.save_for_backward(logits, targets, ids if top_k else None, stats)
    ctx.ignore_index, ctx.entropy = ignore_index, entropy
    ctx.set_materialize_grads(False)


def _logprobs_backward(ctx, g_lp, g_ent, g_top, _g_ids, _g_stats):
    logits, targets, ids, stats = ctx.saved_tensors
    g = [None if t is None else t.float().contiguous()
         for t in (g_lp if targets is not None else None, g_ent if ctx.entropy else None,
                   g_top if ids is not None else None)]
    call = _logprobs_bwd_call if _eager(logits, *g) else torch.ops.gmdn.token_logprobs_bwd
    return call(logits, targets, ids, stats, *g, ctx.ignore_index), None, None, None, None


_logprobs_fwd.register_autograd(_logprobs_backward, setup_context=_logprobs_setup)


class _LogprobsFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, *args):
        got = _logprobs_fwd_call(*args)
        _logprobs_setup(ctx, args, got)
        return got

    backward = _once(_logprobs_backward)


def token_logprobs(logits: Tensor, targets: Optional[Tensor] = None, *, entropy: bool = False,
                   top_k: int = 0, ignore_index: int = -100) -> TokenLogprobs:
    """Log probability of a given token for each row of logits, in one pass.

    logits: (..., V), bf16 or fp32; rows may be strided (a shifted view such as
    ``logits[:, :-1]`` or the live columns of a padded head is read in place).
    targets: (...) int64 or int32, or None for no log probabilities; a target
    equal to ignore_index gives 0 and no gradient, any other outside [0, V)
    gives NaN.  entropy: also the entropy of each row's distribution.  top_k:
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
    if targets is not None:
        targets = targets.long().contiguous()
    args = (logits, targets, bool(entropy), int(top_k), int(ignore_index))
    if not _eager(logits, targets):
        lp, ent, tops, ids, _ = torch.ops.gmdn.token_logprobs_fwd(*args)
    elif _needs_grad(logits):
        lp, ent, tops, ids, _ = _LogprobsFunction.apply(*args)
    else:
        lp, ent, tops, ids, _ = _logprobs_fwd_call(*args)
    return TokenLogprobs(None if targets is None else lp, ent if entropy else None,
                         tops if top_k else None, ids if top_k else None)


# ---------------------------------------------------------------------------
# activations in 8 bits
# ---------------------------------------------------------------------------

BLOCK8 = 128   # consecutive elements that share a scale


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


def _aligned32(t: Tensor) -> Tensor:
    """Contiguous and 32-byte aligned, as ``_aligned`` is for 16."""
    t = _aligned(t)
    try:
        return t if t.data_ptr() % 32 == 0 else t.clone()
    except RuntimeError:   # traced tensors have no storage
        return t


def _codes_like(x: Tensor) -> tuple[Tensor, Tensor]:
    return (torch.empty_like(x, dtype=torch.int8),
            torch.empty((x.numel() + BLOCK8 - 1) // BLOCK8, dtype=torch.float32, device=x.device))


def _pack8_call(x: Tensor) -> tuple[Tensor, Tensor]:
    codes, scales = _codes_like(x)
    _run("gmdn_pack8", lib.gmdn_pack8, x.device, x.data_ptr(), codes.data_ptr(), scales.data_ptr(),
         x.numel(), x.dtype == torch.float32)
    return codes, scales


def _unpack8_call(codes: Tensor, scales: Tensor, f32: bool) -> Tensor:
    x = torch.empty_like(codes, dtype=torch.float32 if f32 else torch.bfloat16)
    _run("gmdn_unpack8", lib.gmdn_unpack8, codes.device, codes.data_ptr(), scales.data_ptr(),
         x.data_ptr(), codes.numel(), f32)
    return x


def _act8_fwd_call(x: Tensor, gate: Optional[Tensor]) -> tuple[Tensor, Tensor, Tensor, Tensor,
                                                               Tensor]:
    y = torch.empty_like(x)
    codes, scales = _codes_like(x)
    if gate is None:
        gcodes, gscales = codes.new_empty(0), scales.new_empty(0)
    else:
        gcodes, gscales = _codes_like(gate)
    _run("gmdn_act8_fwd", lib.gmdn_act8_fwd, x.device, x.data_ptr(), _at(gate), y.data_ptr(),
         codes.data_ptr(), scales.data_ptr(), gcodes.data_ptr(), gscales.data_ptr(), x.numel(),
         x.dtype == torch.float32)
    return y, codes, scales, gcodes, gscales


def _act8_bwd_call(codes: Tensor, scales: Tensor, gcodes: Optional[Tensor],
                   gscales: Optional[Tensor], dy: Tensor,
                   restore: bool) -> tuple[Tensor, Tensor, Tensor]:
    dx = torch.empty_like(dy)
    dgate = torch.empty_like(dy) if gcodes is not None else dy.new_empty(0)
    y = torch.empty_like(dy) if restore else dy.new_empty(0)
    _run("gmdn_act8_bwd", lib.gmdn_act8_bwd, dy.device, codes.data_ptr(), scales.data_ptr(),
         _at(gcodes), _at(gscales), dy.data_ptr(), dx.data_ptr(),
         dgate.data_ptr() if gcodes is not None else None, y.data_ptr() if restore else None,
         dy.numel(), dy.dtype == torch.float32)
    return dx, dgate, y


@torch.library.custom_op("gmdn::pack8", mutates_args=())
def _pack8_op(x: Tensor) -> tuple[Tensor, Tensor]:
    return _pack8_call(x)


@torch.library.custom_op("gmdn::unpack8", mutates_args=())
def _unpack8_op(codes: Tensor, scales: Tensor, f32: bool) -> Tensor:
    return _unpack8_call(codes, scales, f32)


@torch.library.custom_op("gmdn::act8_fwd", mutates_args=())
def _act8_fwd_op(x: Tensor, gate: Optional[Tensor]) -> tuple[Tensor, Tensor, Tensor, Tensor,
                                                            Tensor]:
    return _act8_fwd_call(x, gate)


@torch.library.custom_op("gmdn::act8_bwd", mutates_args=())
def _act8_bwd_op(codes: Tensor, scales: Tensor, gcodes: Optional[Tensor],
                 gscales: Optional[Tensor], dy: Tensor,
                 restore: bool) -> tuple[Tensor, Tensor, Tensor]:
    return _act8_bwd_call(codes, scales, gcodes, gscales, dy, restore)


@_pack8_op.register_fake
def _(x):
    return _codes_like(x)


@_unpack8_op.register_fake
def _(codes, scales, f32):
    return codes.new_empty(codes.shape, dtype=torch.float32 if f32 else torch.bfloat16)


@_act8_fwd_op.register_fake
def _(x, gate):
    codes, scales = _codes_like(x)
    g = (codes.new_empty(0), scales.new_empty(0)) if gate is None else _codes_like(gate)
    return torch.empty_like(x), codes, scales, *g


@_act8_bwd_op.register_fake
def _(codes, scales, gcodes, gscales, dy, restore):
    return (torch.empty_like(dy),
            torch.empty_like(dy) if gcodes is not None else dy.new_empty(0),
            torch.empty_like(dy) if restore else dy.new_empty(0))


def _check_packed(name: str, p: Packed8) -> None:
    if p.codes.dtype != torch.int8 or p.scales.dtype != torch.float32:
        raise TypeError(f"{name}: codes must be int8 and scales float32, got {p.codes.dtype} and "
                        f"{p.scales.dtype}")
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
    x = _aligned32(x.detach())
    call = _pack8_call if _eager(x) else torch.ops.gmdn.pack8
    return Packed8(*call(x), x.dtype)


def unpack8(packed: Packed8) -> Tensor:
    """The tensor that ``pack8`` kept, in its shape and type."""
    _check_packed("unpack8", packed)
    _same_device("unpack8", packed.codes, packed.scales)
    codes, scales = _aligned32(packed.codes), _aligned32(packed.scales)
    call = _unpack8_call if _eager(codes, scales) else torch.ops.gmdn.unpack8
    return call(codes, scales, packed.dtype == torch.float32)


def act8_forward(x: Tensor, gate: Optional[Tensor] = None) -> tuple[Tensor, Act8Saved]:
    """GELU(x) (exact), or SiLU(gate) * x with a gate, and the 8-bit checkpoint
    of its inputs for ``act8_backward``.  x, gate: one shape and type, bf16 or
    fp32.  Not recorded by autograd (``mlp8`` is the differentiable form)."""
    _f32_flag(x, "x")
    if gate is not None and (gate.shape != x.shape or gate.dtype != x.dtype):
        raise ValueError(f"gate must be like x, {tuple(x.shape)} {x.dtype}, got "
                         f"{tuple(gate.shape)} {gate.dtype}")
    _same_device("act8_forward", x, gate)
    x, gate = _aligned32(x.detach()), None if gate is None else _aligned32(gate.detach())
    call = _act8_fwd_call if _eager(x, gate) else torch.ops.gmdn.act8_fwd
    y, codes, scales, gcodes, gscales = call(x, gate)
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
    parts = [None if t is None else _aligned32(t) for t in parts]
    dy = _aligned32(dy.detach())
    call = _act8_bwd_call if _eager(dy, *parts) else torch.ops.gmdn.act8_bwd
    dx, dgate, y = call(*parts, dy, bool(restore))
    return dx, dgate if gate is not None else None, y if restore else None


class _Mlp8Function(torch.autograd.Function):
    """down(act(up x)) that keeps x and the activation's inputs in 8 bits; the
    weight gradients are products with the restored tensors."""

    @staticmethod
    def forward(ctx, x, w_up, w_down, w_gate):
        rows = x.reshape(-1, x.shape[-1])
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
        w_up, w_down, w_gate, codes, scales, *more = ctx.saved_tensors
        gate = Packed8(*more[:2], ctx.dtype) if ctx.gated else None
        saved = Act8Saved(Packed8(codes, scales, ctx.dtype), gate)
        need = ctx.needs_input_grad
        dout = dout.reshape(-1, dout.shape[-1]).to(ctx.dtype)
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
    return _Mlp8Function.apply(x, w_up, w_down, w_gate)
