"""The step operators at the borders between their ways: sizes, types, views and
cotangents that the other tests pass by."""
import math

import pytest
import torch

from conftest import load_pkg
from oracle import step_oracle as so
from test_gpu_step_ops import BF, EPS, FP, U, _check_norm, _gen, _norm_case, _within

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D", [6001, 6009, 6010, 6073, 6130, 6137, 6138, 12025, 12026, 12101, 12273,
                               12281, 12282])
def test_norm_odd_widths_around_48_kb_of_shared_memory(D):
    """An odd width's weight and bias copies lie in shared memory beside the kernel's own
    kilobyte: together they pass 48 KB before the copies alone do (from 6010 with both, from
    12026 with one)."""
    pkg = load_pkg()
    _check_norm(pkg, _norm_case(5, D, True, FP, None, FP))
    _check_norm(pkg, _norm_case(5, D, False, BF, FP, BF, bias=False))


@pytest.mark.parametrize("dtype", [BF, FP])
def test_logprobs_bad_targets_without_cotangents_have_no_gradient(dtype):
    """A target outside the columns gives NaN; where the caller drops that value (a cotangent
    of 0), the row has a zero gradient like any other without cotangents."""
    pkg = load_pkg()
    t = torch.tensor([1, -1, 60, 3, 50, -100]).cuda()
    z = torch.randn(6, 50, generator=_gen(1)).to(dtype).cuda().requires_grad_(True)
    lp = pkg.token_logprobs(z, t).logprobs
    good = (t >= 0) & (t < 50)
    (g,) = torch.autograd.grad(torch.where(good, lp, 0.0).sum(), z, retain_graph=True)
    (want,) = torch.autograd.grad(pkg.token_logprobs(z[good], t[good]).logprobs.sum(), z)
    assert torch.equal(g, want) and torch.equal(g[~good], torch.zeros_like(g[~good]))
    cot = torch.tensor([0.0, 0.0, 1.0, 0.0, math.nan, 1.0]).cuda()
    (g,) = torch.autograd.grad(lp, z, cot)
    assert torch.isnan(g).all(-1).tolist() == [False, False, True, False, True, False]
    assert torch.equal(g[[0, 1, 3, 5]], torch.zeros_like(g[:4]))
    # with another cotangent the row has that one's gradient alone
    got = pkg.token_logprobs(z, t, entropy=True)
    b = torch.randn(6, generator=_gen(2)).cuda()
    (g,) = torch.autograd.grad([got.logprobs, got.entropy], z, [torch.zeros(6).cuda(), b])
    ent = pkg.token_logprobs(z, None, entropy=True).entropy
    (want,) = torch.autograd.grad(ent, z, b)
    assert torch.equal(g, want)
