"""Plain 64-bit forms of the training step's operators (norm, token log
probabilities, 8-bit activation checkpoints), differentiable by autograd."""
import math

import torch

BLOCK8 = 128


def norm(x, weight=None, bias=None, eps=1e-5, residual=None, center=True):
    """(y, h) in fp64; with a residual h is the sum rounded to its stored type
    (a constant shift for autograd, as the kernel treats it)."""
    s = x.double()
    if residual is not None:
        total = s + residual.double()
        stored = torch.promote_types(x.dtype, residual.dtype)
        s = total + (total.to(stored).double() - total).detach()
    h = s
    c = s - s.mean(-1, keepdim=True) if center else s
    y = c / torch.sqrt((c * c).mean(-1, keepdim=True) + eps)
    if weight is not None:
        y = y * weight.double()
    if bias is not None:
        y = y + bias.double()
    return y, h


def token_logprobs(logits, targets=None, top_k=0, ignore_index=-100):
    """(logprobs, entropy, top_logprobs, top_ids) in fp64 for rows that hold a
    finite logit and no NaN or +inf; a row of nothing but -inf: (-inf, 0)."""
    z = logits.double()
    empty = (z == -math.inf).all(-1, keepdim=True)
    z = torch.where(empty, torch.zeros_like(z), z)
    lp = torch.log_softmax(z, -1)
    p = lp.exp()
    entropy = -(p * torch.where(p > 0, lp, torch.zeros_like(lp))).sum(-1)
    entropy = torch.where(empty[..., 0], torch.zeros_like(entropy), entropy)
    lp = torch.where(empty, torch.full_like(lp, -math.inf), lp)
    got = None
    if targets is not None:
        skip = targets == ignore_index
        at = torch.where(skip, torch.zeros_like(targets), targets)
        got = lp.gather(-1, at[..., None])[..., 0]
        got = torch.where(skip, torch.zeros_like(got), got)
    ids = torch.sort(logits.detach().float(), dim=-1, descending=True,
                     stable=True).indices[..., :top_k]
    return got, entropy, lp.gather(-1, ids), ids


def pack8(x):
    """(codes, scales) by the definition: the two factors of a block are fp32
    numbers, the product with the first is exact in fp64."""
    flat = x.detach().reshape(-1).double().cpu()
    n = flat.numel()
    v = torch.cat([flat, flat.new_zeros(-n % BLOCK8)]).view(-1, BLOCK8)
    a = v.abs().amax(1)
    bad = ~torch.isfinite(v).all(1)
    tiny = a < 2.0 ** -100
    use = torch.where(bad | tiny, torch.ones_like(a), a)
    r = (127.0 / use).float().double()
    s = (use * torch.tensor(1.0 / 127.0, dtype=torch.float32).double()).float()
    q = torch.round(v * r[:, None])
    q[bad | tiny] = 0.0
    s = torch.where(bad, torch.full_like(s, math.nan), torch.where(tiny, torch.zeros_like(s), s))
    return q.view(-1)[:n].to(torch.int8).view(x.shape), s


def unpack8(codes, scales):
    """Restored values in fp64."""
    flat = codes.reshape(-1).double()
    s = scales.double().repeat_interleave(BLOCK8)[:flat.numel()]
    return (flat * s).view(codes.shape)


def act(x, gate=None):
    """GELU(x) or SiLU(gate) * x in fp64."""
    x = x.double()
    if gate is None:
        return 0.5 * x * torch.special.erfc(-x / math.sqrt(2.0))
    gate = gate.double()
    return gate * torch.sigmoid(gate) * x
