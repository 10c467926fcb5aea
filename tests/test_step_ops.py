"""The training step's operators without a GPU: their refusals, at the ops and
at the C ABI, and the 64-bit oracle against differences."""
import ctypes

import pytest
import torch

from conftest import load_pkg
from oracle import step_oracle as so

NULL = ctypes.c_void_p(None)
FAKE = ctypes.c_void_p(0x1000)   # never dereferenced: the checks fail first
ODD = ctypes.c_void_p(0x1008)


def _lib():
    return load_pkg()._lib.lib


def test_refuses_cpu_tensors():
    pkg = load_pkg()
    x = torch.zeros(4, 16)
    calls = [lambda: pkg.layer_norm(x), lambda: pkg.rms_norm(x, torch.ones(16)),
             lambda: pkg.token_logprobs(x, torch.zeros(4, dtype=torch.int64)),
             lambda: pkg.pack8(x), lambda: pkg.act8_forward(x),
             lambda: pkg.unpack8(pkg.Packed8(torch.zeros(4, dtype=torch.int8), torch.zeros(1),
                                             torch.float32)),
             lambda: pkg.mlp8(x, torch.zeros(32, 16), torch.zeros(16, 32))]
    for call in calls:
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


@pytest.mark.parametrize("bad, error", [
    (lambda p, x: p.layer_norm(torch.zeros(())), ValueError),
    (lambda p, x: p.layer_norm(x, torch.ones(15)), ValueError),
    (lambda p, x: p.layer_norm(x, None, torch.ones(2, 16)), ValueError),
    (lambda p, x: p.layer_norm(x, residual=torch.zeros(1, 16)), ValueError),
    (lambda p, x: p.layer_norm(x, eps=-1.0), ValueError),
    (lambda p, x: p.rms_norm(x, eps=float("nan")), ValueError),
    (lambda p, x: p.rms_norm(x.half()), TypeError),
    (lambda p, x: p.rms_norm(x, residual=x.double()), TypeError),
    (lambda p, x: p.rms_norm(x, out_dtype=torch.float16), TypeError),
    (lambda p, x: p.token_logprobs(torch.zeros(4, 0)), ValueError),
    (lambda p, x: p.token_logprobs(x), ValueError),
    (lambda p, x: p.token_logprobs(x, top_k=17), ValueError),
    (lambda p, x: p.token_logprobs(torch.zeros(4, 100), top_k=65), ValueError),
    (lambda p, x: p.token_logprobs(x, top_k=-1), ValueError),
    (lambda p, x: p.token_logprobs(x, torch.zeros(3, dtype=torch.int64)), ValueError),
    (lambda p, x: p.token_logprobs(x, torch.zeros(4)), TypeError),
    (lambda p, x: p.token_logprobs(x.half(), torch.zeros(4, dtype=torch.int64)), TypeError),
    (lambda p, x: p.pack8(x.to(torch.float16)), TypeError),
    (lambda p, x: p.act8_forward(x, x.bfloat16()), ValueError),
    (lambda p, x: p.act8_forward(x, torch.zeros(4, 8)), ValueError),
    (lambda p, x: p.unpack8(p.Packed8(x, torch.zeros(1), torch.float32)), TypeError),
    (lambda p, x: p.unpack8(p.Packed8(torch.zeros(129, dtype=torch.int8), torch.zeros(1),
                                      torch.float32)), ValueError),
    (lambda p, x: p.unpack8(p.Packed8(torch.zeros(4, dtype=torch.int8), torch.zeros(1),
                                      torch.float16)), TypeError),
    (lambda p, x: p.act8_backward(p.Act8Saved(p.Packed8(torch.zeros(4, 16, dtype=torch.int8),
                                                        torch.zeros(1), torch.float32), None),
                                  x.bfloat16()), ValueError),
    (lambda p, x: p.mlp8(x, torch.zeros(32, 15), torch.zeros(16, 32)), ValueError),
    (lambda p, x: p.mlp8(x, torch.zeros(32, 16), torch.zeros(16, 31)), ValueError),
    (lambda p, x: p.mlp8(x, torch.zeros(32, 16), torch.zeros(16, 32), torch.zeros(31, 16)),
     ValueError),
])
def test_refuses_bad_arguments(bad, error):
    with pytest.raises(error):
        bad(load_pkg(), torch.zeros(4, 16))


def test_norm_abi_refusals():
    lib = _lib()

    def fwd(x=FAKE, h=NULL, res=NULL, mean=FAKE, rows=4, width=16, eps=1e-5, center=1):
        return lib.gmdn_norm_fwd(x, res, FAKE, NULL, FAKE, h, FAKE, mean, rows, width, eps, center,
                                 0, 0, 0, NULL)

    assert fwd(rows=-1) == 1 and fwd(width=-1) == 1
    assert fwd(rows=1 << 59, width=1 << 20) == 2
    assert fwd(x=NULL) == 1 and fwd(mean=NULL) == 1 and fwd(res=FAKE) == 1
    assert fwd(x=ODD) == 1 and "aligned" in lib.gmdn_last_error_string().decode()
    assert fwd(eps=-1.0) == 1 and fwd(eps=float("nan")) == 1
    assert fwd(rows=0, x=NULL) == 0
    need = lib.gmdn_norm_bwd_workspace_bytes(1000, 768)
    assert need > 0 and lib.gmdn_norm_bwd_workspace_bytes(0, 768) == 0

    def bwd(s=FAKE, ws=FAKE, nbytes=need, dw=FAKE):
        return lib.gmdn_norm_bwd(s, FAKE, FAKE, FAKE, FAKE, NULL, FAKE, NULL, dw, NULL, ws, nbytes,
                                 1000, 768, 1, 0, 0, 0, 0, 0, NULL)

    assert bwd(s=NULL) == 1 and bwd(s=ODD) == 1
    assert bwd(ws=NULL) == 3 and bwd(nbytes=need - 1) == 3


def test_token_logprobs_abi_refusals():
    lib = _lib()

    def fwd(logits=FAKE, targets=FAKE, lp=FAKE, tops=NULL, ids=NULL, stats=FAKE, batch=2, length=3,
            vocab=100, k=0, f32=0):
        return lib.gmdn_token_logprobs_fwd(logits, targets, lp, NULL, tops, ids, stats, batch,
                                           length, 300, 100, vocab, k, -100, f32, NULL)

    assert fwd(batch=-1) == 1 and fwd(vocab=0) == 1 and fwd(logits=NULL) == 1
    assert fwd(batch=1 << 31, length=1 << 29) == 2
    assert fwd(k=65) == 1 and fwd(k=-1) == 1 and fwd(vocab=5, k=6) == 1
    assert fwd(k=3) == 1 and fwd(targets=NULL) == 1     # null outputs / targets
    assert fwd(logits=ctypes.c_void_p(0x1002), f32=1) == 1
    assert fwd(stats=ODD) == 1
    assert fwd(batch=0, logits=NULL) == 0

    def bwd(stats=FAKE, g_top=NULL, ids=NULL, out=FAKE, targets=FAKE):
        return lib.gmdn_token_logprobs_bwd(FAKE, targets, stats, ids, FAKE, NULL, g_top, out, 2, 3,
                                           300, 100, 100, 0, -100, 0, NULL)

    assert bwd(stats=NULL) == 1 and bwd(out=NULL) == 1 and bwd(g_top=FAKE) == 1
    assert bwd(targets=NULL) == 1 and bwd(out=ODD) == 1


def test_act8_abi_refusals():
    lib = _lib()
    assert lib.gmdn_pack8(FAKE, FAKE, NULL, 10, 0, NULL) == 1
    assert lib.gmdn_pack8(ODD, FAKE, FAKE, 10, 0, NULL) == 1
    assert lib.gmdn_pack8(FAKE, FAKE, FAKE, -1, 0, NULL) == 1
    assert lib.gmdn_pack8(NULL, NULL, NULL, 0, 0, NULL) == 0
    assert lib.gmdn_unpack8(NULL, FAKE, FAKE, 10, 0, NULL) == 1
    assert lib.gmdn_act8_fwd(FAKE, FAKE, FAKE, FAKE, FAKE, NULL, FAKE, 10, 0, NULL) == 1
    assert lib.gmdn_act8_bwd(FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, NULL, NULL, 10, 0, NULL) == 1
    assert lib.gmdn_act8_bwd(FAKE, FAKE, NULL, NULL, FAKE, FAKE, NULL, ODD, 10, 0, NULL) == 1


# ---- the oracle itself ---------------------------------------------------------

def _difference(f, x, v, h=1e-6):
    return (f(x + h * v) - f(x - h * v)) / (2 * h)


@pytest.mark.parametrize("center", [True, False])
def test_oracle_norm_gradient_against_differences(center):
    g = torch.Generator().manual_seed(1)
    x, v, c = (torch.randn(3, 17, generator=g, dtype=torch.float64) for _ in range(3))
    w = torch.randn(17, generator=g, dtype=torch.float64)

    def f(t):
        return (so.norm(t, w, None, 1e-5, None, center)[0] * c).sum()

    x.requires_grad_(True)
    (grad,) = torch.autograd.grad(f(x), x)
    want = _difference(lambda t: f(t).item(), x.detach(), v)
    # central differences: truncation ~ h^2, rounding ~ 2^-53 |f| / h
    assert abs((grad * v).sum().item() - want) < 1e-7


def test_oracle_logprobs_gradient_against_differences():
    g = torch.Generator().manual_seed(2)
    z, v = (torch.randn(3, 40, generator=g, dtype=torch.float64) for _ in range(2))
    z[1, 5:] = -float("inf")
    v[1, 5:] = 0.0
    t = torch.tensor([4, -100, 39])
    a, b = torch.randn(3, generator=g, dtype=torch.float64), torch.randn(3, 4, generator=g,
                                                                           dtype=torch.float64)

    def f(x):
        lp, ent, tops, _ = so.token_logprobs(x, t, 4)
        return (lp * a).sum() + (ent * a).sum() + (tops * b).sum()

    z.requires_grad_(True)
    (grad,) = torch.autograd.grad(f(z), z)
    want = _difference(lambda x: f(x).item(), z.detach(), v)
    assert abs((torch.nan_to_num(grad) * v).sum().item() - want) < 1e-7


def test_oracle_pack8_is_within_half_a_step():
    g = torch.Generator().manual_seed(3)
    x = torch.randn(1000, generator=g) * torch.exp(3 * torch.randn(1000, generator=g))
    codes, scales = so.pack8(x)
    back = so.unpack8(codes, scales)
    assert int(codes.abs().max()) == 127
    # half a step a / 254; 127 of the scale's and the factor's relative 2^-24 more
    step = scales.double().repeat_interleave(128)[:1000]
    assert ((back - x.double()).abs() <= step * (0.5 + 4 * 127 * 2.0 ** -24)).all()
