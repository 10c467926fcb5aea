"""GPU parity of the training step's operators with their 64-bit oracles, at
the sizes and masks where they can go wrong.

Bounds.  U is half a step of the output's type (bf16 2^-8, fp32 2^-24,
relative), the last rounding.  Inside, everything is fp32: an operation is off
by EPS = 2^-24 of its result, a sum of n terms added in a chain of c by c EPS
of the sum of magnitudes.  The longest chain of a row sum is width / 32 terms
in a lane (one warp a row) and 16 joins; CHAIN(width) counts it.
"""
import copy
import math

import pytest
import torch
import torch.nn.functional as F

from conftest import load_pkg
from oracle import step_oracle as so

pytestmark = pytest.mark.gpu

EPS = 2.0 ** -24
BF, FP = torch.bfloat16, torch.float32


def U(dtype):
    return torch.finfo(dtype).eps / 2


def CHAIN(width):
    return width / 32 + 16


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _within(got, want, bound, what):
    got, want = got.detach().double().cpu(), want.detach().double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    bad = ~((got - want).abs() <= bound.cpu() if torch.is_tensor(bound) else
            (got - want).abs() <= bound)
    bad &= ~(torch.isnan(got) & torch.isnan(want)) & (got != want)
    if bad.any():
        i = int(bad.flatten().nonzero()[0])
        b = (bound.double().cpu().expand_as(want) if torch.is_tensor(bound) else
             torch.full_like(want, bound)).flatten()[i].item()
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} outside; at {i} "
                             f"{got.flatten()[i].item()} for {want.flatten()[i].item()} +- {b}")


# ---------------------------------------------------------------------------
# norm
# ---------------------------------------------------------------------------

def _norm_case(rows, D, center, x_dt, res_dt, out_dt, weight=True, bias=True, offset=0.3, seed=0,
               eps=1e-5):
    g = _gen(seed + 7 * D + rows)
    x = (torch.randn(rows, D, generator=g) * torch.exp(torch.randn(rows, 1, generator=g))
         + offset).to(x_dt)
    res = None if res_dt is None else (torch.randn(rows, D, generator=g) * 2).to(res_dt)
    w = 1 + 0.3 * torch.randn(D, generator=g) if weight else None
    b = 0.3 * torch.randn(D, generator=g) if bias else None
    dy = torch.randn(rows, D, generator=g).to(out_dt)
    dh = None if res is None else torch.randn(rows, D, generator=g).to(
        torch.promote_types(x_dt, res_dt))
    return dict(x=x, res=res, w=w, b=b, dy=dy, dh=dh, center=center, out=out_dt, eps=eps)


def _run_norm(pkg, c):
    leaves = {n: None if c[n] is None else c[n].cuda().requires_grad_(True)
              for n in ("x", "res", "w", "b")}
    call = pkg.layer_norm if c["center"] else pkg.rms_norm
    got = call(leaves["x"], leaves["w"], leaves["b"], c["eps"], residual=leaves["res"],
               out_dtype=c["out"])
    outs = [got] if c["res"] is None else list(got)
    cots = [c["dy"].cuda()] + ([c["dh"].cuda()] if c["res"] is not None else [])
    live = {n: t for n, t in leaves.items() if t is not None}
    grads = dict(zip(live, torch.autograd.grad(outs, list(live.values()), cots)))
    return outs, grads


def _check_norm(pkg, c):
    outs, grads = _run_norm(pkg, c)
    ref = {n: None if c[n] is None else c[n].double().requires_grad_(True)
           for n in ("x", "res", "w", "b")}
    stored = None if c["res"] is None else torch.promote_types(c["x"].dtype, c["res"].dtype)
    y, h = so.norm(c["x"], ref["w"], ref["b"], c["eps"], c["res"], c["center"])
    # the same again, differentiable in x and the residual (both fp64 here, so h is shifted to
    # its stored value by hand)
    s = ref["x"] if c["res"] is None else ref["x"] + ref["res"]
    if stored is not None:
        s = s + (h - s).detach()
    y, _ = so.norm(s, ref["w"], ref["b"], c["eps"], None, c["center"])
    live = {n: t for n, t in ref.items() if t is not None}
    cots = c["dy"].double()
    loss = (y * cots).sum() + (0.0 if c["dh"] is None else (s * c["dh"].double()).sum())
    want = dict(zip(live, torch.autograd.grad(loss, list(live.values()))))

    D = c["x"].shape[-1]
    s = h.detach()
    ch = CHAIN(D) * EPS
    mean = s.mean(-1, keepdim=True) if c["center"] else torch.zeros_like(s[:, :1])
    rstd = 1 / torch.sqrt(((s - mean) ** 2).mean(-1, keepdim=True) + c["eps"])
    w = torch.ones(D, dtype=torch.float64) if c["w"] is None else c["w"].double()
    b = torch.zeros(D, dtype=torch.float64) if c["b"] is None else c["b"].double()
    xh = (s - mean) * rstd
    # s - mean is off by an ulp of the mean and of itself; rstd by a chain
    xh_err = ch * xh.abs() + 4 * EPS * (mean.abs() + s.abs()) * rstd
    if c["center"]:
        # the mean itself is a chained sum: fl(sum d) is off by ch sum|d|, however near 0 the
        # mean is, and every xh of the row moves by that over D times rstd
        xh_err = xh_err + ch * (s - mean).abs().mean(-1, keepdim=True) * rstd
    _within(outs[0], y, U(c["out"]) * y.abs() + xh_err * w.abs() + 4 * EPS * (b.abs() + y.abs()),
            "y")
    assert outs[0].dtype == c["out"]
    if c["res"] is not None:
        assert outs[1].dtype == stored
        assert torch.equal(outs[1].cpu(), h.to(stored)), "h"
    g = c["dy"].double() * w
    top = (g.abs().mean(-1, keepdim=True) + g.abs())
    along = (g * xh).abs().mean(-1, keepdim=True)
    ds = want["x"]
    inner = ch * (top + xh.abs() * along) + xh_err * along \
        + xh.abs() * (xh_err * g.abs()).mean(-1, keepdim=True)
    dh = torch.zeros_like(s) if c["dh"] is None else c["dh"].double()
    # ds is the same sum for x and the residual, each rounded to its type
    bound = inner * rstd + ch * rstd * (top + xh.abs() * along) + 4 * EPS * (dh.abs() + ds.abs())
    _within(grads["x"], ds, bound + U(c["x"].dtype) * ds.abs(), "dx")
    assert grads["x"].dtype == c["x"].dtype
    if c["res"] is not None:
        _within(grads["res"], want["res"], bound + U(c["res"].dtype) * ds.abs(), "dres")
        assert grads["res"].dtype == c["res"].dtype
    dy = c["dy"].double()
    # a column's chain: at most rows / 8 rows in a thread, then at most 64 joins
    col = (c["x"].shape[0] / 8 + 64) * EPS
    if c["w"] is not None:
        _within(grads["w"], want["w"], col * (dy * xh).abs().sum(0) + (dy.abs() * xh_err).sum(0)
                + U(FP) * want["w"].abs(), "dw")
    if c["b"] is not None:
        _within(grads["b"], want["b"], col * dy.abs().sum(0) + U(FP) * want["b"].abs(), "db")


@pytest.mark.parametrize("rows, D", [(1, 1), (3, 2), (2, 7), (5, 8), (1, 31), (9, 64), (33, 100),
                                     (1, 768), (300, 768), (1000, 1000), (17, 1283), (40, 2048),
                                     (7, 4096), (5, 8192), (3, 12345), (2, 16384), (2, 40000),
                                     (2, 40001), (4099, 136)])
@pytest.mark.parametrize("center", [True, False])
def test_norm_sizes(rows, D, center):
    pkg = load_pkg()
    for dt, res in ((BF, FP), (FP, None)):
        _check_norm(pkg, _norm_case(rows, D, center, dt, res, dt))


@pytest.mark.parametrize("rows, D", [(20000, 13), (12001, 64), (9001, 101), (5000, 129), (4000, 257),
                                     (3001, 513), (2000, 761), (2500, 775), (2501, 1030),
                                     (1200, 4081), (1201, 4083), (700, 8177), (650, 8179),
                                     (300, 8191), (40, 16370), (3, 16383),
                                     (300, 16384), (320, 8200), (301, 8185), (299, 8193),
                                     (303, 12345), (200, 16377), (150, 16378)])
def test_norm_ragged_widths(rows, D):
    """Rows at every alignment, each CTA walking many of them, at the borders
    between the ways a width is held."""
    pkg = load_pkg()
    _check_norm(pkg, _norm_case(rows, D, True, BF, FP, BF))
    _check_norm(pkg, _norm_case(rows, D, False, FP, None, FP, bias=False))


def test_norm_neighbours_stay_out():
    """Infinities and NaN in a row stay in it, whatever shares its memory groups."""
    pkg = load_pkg()
    for D in (5, 100, 769, 1283, 8203):
        c = _norm_case(24, D, True, FP, BF, FP)
        clean, cg = _run_norm(pkg, c)
        c["x"][7] = math.inf
        c["x"][8, 0] = math.nan
        c["dh"][11, -1] = math.nan
        dirty, dg = _run_norm(pkg, c)
        keep = [r for r in range(24) if r not in (7, 8)]
        for a, b in zip(clean, dirty):
            assert torch.equal(a[keep], b[keep])
        assert torch.isnan(dirty[0][7]).all() and torch.isnan(dirty[0][8]).all()
        keep.remove(11)
        assert torch.equal(cg["x"][keep], dg["x"][keep])
        assert torch.isnan(dg["x"][11, -1]) and not torch.isnan(dg["x"][11, :-1]).any()


@pytest.mark.parametrize("x_dt", [BF, FP])
@pytest.mark.parametrize("res_dt", [None, BF, FP])
@pytest.mark.parametrize("out_dt", [BF, FP])
def test_norm_types(x_dt, res_dt, out_dt):
    pkg = load_pkg()
    for D in (96, 1536, 777):
        for center, weight, bias in ((True, True, True), (False, True, False),
                                     (True, False, False), (False, False, True)):
            _check_norm(pkg, _norm_case(65, D, center, x_dt, res_dt, out_dt, weight, bias))


def test_norm_large_mean_and_constant_rows():
    """A mean of 3000 beside a deviation of 1: the centred sum of squares keeps
    what the sum of squares loses; rows of one value give the bias."""
    pkg = load_pkg()
    for D in (768, 1283, 9000):
        _check_norm(pkg, _norm_case(20, D, True, FP, None, FP, offset=3000.0))
    x = torch.full((3, 768), 7.5, device="cuda")
    b = torch.randn(768, generator=_gen(1)).cuda()
    assert torch.equal(pkg.layer_norm(x, torch.ones(768, device="cuda"), b), b.expand(3, 768))
    assert torch.equal(pkg.rms_norm(torch.zeros(3, 768, device="cuda")),
                       torch.zeros(3, 768, device="cuda"))


def test_norm_strided_misaligned_and_empty():
    pkg = load_pkg()
    base = torch.randn(40, 3, 200, generator=_gen(2)).cuda()
    w = torch.randn(200, generator=_gen(3)).cuda()
    for x in (base[:, 1], base.transpose(0, 1), base[..., 3:103]):
        ww = w[:x.shape[-1]]
        xg = x.detach().requires_grad_(True)
        y = pkg.rms_norm(xg, ww, None, 1e-6)
        want = pkg.rms_norm(x.contiguous().clone(), ww.clone(), None, 1e-6)
        assert torch.equal(y, want) and y.shape == x.shape
        (dx,) = torch.autograd.grad(y, xg, torch.ones((), device="cuda").expand(y.shape))
        assert dx.shape == x.shape
    odd = torch.randn(64 * 10 + 1, generator=_gen(4)).cuda()[1:].view(10, 64)   # 4-byte aligned
    assert torch.equal(pkg.layer_norm(odd), pkg.layer_norm(odd.clone()))
    for shape in ((0, 64), (3, 0), (2, 0, 64)):
        x = torch.empty(shape, device="cuda", requires_grad=True)
        w = torch.ones(shape[-1], device="cuda", requires_grad=True)
        y = pkg.layer_norm(x, w)
        y.sum().backward()
        assert y.shape == x.shape and x.grad.shape == x.shape
        assert torch.equal(w.grad, torch.zeros_like(w))


def test_norm_partial_cotangents_and_frozen_inputs():
    """Only h used, only y used, inputs that need no gradient, bf16 parameters."""
    pkg = load_pkg()
    c = _norm_case(33, 256, True, BF, FP, BF)
    x, r = c["x"].cuda().requires_grad_(True), c["res"].cuda().requires_grad_(True)
    w = c["w"].cuda().to(BF).requires_grad_(True)
    y, h = pkg.layer_norm(x, w, residual=r)
    dx, dr = torch.autograd.grad(h, [x, r], c["dh"].cuda(), retain_graph=True)
    assert torch.equal(dr, c["dh"].cuda()) and torch.equal(dx, c["dh"].cuda().to(BF))
    both = torch.autograd.grad([y, h], [x, r, w], [c["dy"].cuda(), torch.zeros_like(h)],
                               retain_graph=True)
    only = torch.autograd.grad(y, [x, r, w], c["dy"].cuda(), retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(both, only)) and only[2].dtype == BF
    y2, _ = pkg.layer_norm(x.detach(), w, residual=r.detach())
    (dw,) = torch.autograd.grad(y2, w, c["dy"].cuda())
    assert torch.equal(dw, only[2])
    y3, _ = pkg.layer_norm(x, w.detach(), residual=r.detach())
    (dx3,) = torch.autograd.grad(y3, x, c["dy"].cuda())
    assert torch.equal(dx3, only[0])
    with pytest.raises(RuntimeError):   # no second derivative, and it says so
        (g,) = torch.autograd.grad(y.float().sum(), x, create_graph=True)
        g.float().sum().backward()


def test_norm_gradient_against_differences():
    pkg = load_pkg()
    c = _norm_case(6, 300, True, FP, FP, FP)
    _, grads = _run_norm(pkg, c)
    v = {n: torch.randn(c[n].shape, generator=_gen(9), dtype=torch.float64)
         for n in ("x", "res", "w", "b")}

    def loss(h):
        p = {n: c[n].double() + h * v[n] for n in v}
        s = p["x"] + p["res"]
        y, _ = so.norm(s, p["w"], p["b"], c["eps"])
        return ((y * c["dy"].double()).sum() + (s * c["dh"].double()).sum()).item()

    want = (loss(1e-6) - loss(-1e-6)) / 2e-6
    got = sum((grads[n].double().cpu() * v[n]).sum().item() for n in v)
    # the rounded h moves y by 2^-24; sums of ~4000 fp32 terms of size <= 30
    assert abs(got - want) < 4000 * 30 * 16 * EPS


def test_norm_repeats_bit_for_bit_and_on_another_stream():
    pkg = load_pkg()
    c = _norm_case(5000, 768, False, BF, FP, BF)
    _, a = _run_norm(pkg, c)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _, b = _run_norm(pkg, c)
    torch.cuda.synchronize()
    assert all(torch.equal(a[n], b[n]) for n in a)


# ---------------------------------------------------------------------------
# token log probabilities
# ---------------------------------------------------------------------------

def _logits(rows, V, dtype, seed=0, scale=3.0):
    return (torch.randn(rows, V, generator=_gen(seed + V)) * scale).to(dtype)


def _check_logprobs(pkg, z, t, top_k, ignore=-100, grads=True, cuda_z=None):
    """z (rows, V) on the CPU; cuda_z: the same values as a GPU view."""
    V = z.shape[-1]
    zg = (z.cuda() if cuda_z is None else cuda_z).detach().requires_grad_(True)
    got = pkg.token_logprobs(zg, t.cuda(), entropy=True, top_k=top_k, ignore_index=ignore)
    zr = z.double().requires_grad_(True)
    lp, ent, tops, ids = so.token_logprobs(zr, t, top_k, ignore)
    full = so.token_logprobs(z)[1]
    m = z.double().amax(-1).clamp_min(-1e300)
    # logprob = (x - m) - log S: two roundings of each part; S: an exponential is off by 2^-22
    # and by 2^-23 of its argument (weighted by p: at most the entropy and log V), a chain
    spread = full.abs() + math.log(V) + 1
    s_err = 2.0 ** -22 + 2.0 ** -23 * spread + (V / 32 + 32) * EPS
    log_s = (torch.logsumexp(torch.where((z == -math.inf).all(-1, keepdim=True), 0.0, z.double()),
                             -1) - torch.where(m.isfinite() & (m > -1e300), m, 0.0)).abs()

    def err(v):
        far = torch.where(v.isfinite(), v.abs(), torch.zeros_like(v))
        pad = (...,) + (None,) * (v.dim() - 1)
        return 4 * EPS * (far + log_s[pad]) + s_err[pad]

    _within(got.logprobs, lp, err(lp), "logprobs")
    # entropy = log S - Q / S, Q = sum e^c c of magnitude <= S spread
    _within(got.entropy, ent, 4 * EPS * (ent.abs() + log_s) + s_err * (2 + spread), "entropy")
    if top_k:
        assert torch.equal(got.top_ids.cpu(), ids), "top_ids"
        _within(got.top_logprobs, tops, err(tops), "top_logprobs")
    if not grads:
        return
    gen = _gen(5)
    a, b = (torch.randn(len(z), generator=gen) for _ in range(2))
    k = torch.randn(len(z), top_k, generator=gen)
    outs, cots = [got.logprobs, got.entropy], [a, b]
    if top_k:
        outs.append(got.top_logprobs)
        cots.append(k)
    (gz,) = torch.autograd.grad(outs, zg, [c.cuda() for c in cots])
    empty = (z == -math.inf).all(-1)
    p = torch.softmax(
        torch.where(empty[:, None], 0.0, z.double()), -1)
    live = (t != ignore) & ~empty
    al = torch.where(live, a, torch.zeros_like(a)).double()
    w = al + k.double().sum(-1)
    lpz = torch.where(p > 0, torch.log(p.clamp_min(1e-320)), torch.zeros_like(p))
    H = ent.detach()[:, None]
    want = -p * (w[:, None] + b.double()[:, None] * (lpz + H))
    want.scatter_add_(1, torch.where(live, t, torch.zeros_like(t))[:, None], al[:, None])
    want.scatter_add_(1, ids, k.double())
    want[empty] = 0.0
    size = w.abs()[:, None] + b.double().abs()[:, None] * (lpz.abs() + H + 1)
    bound = p * size * (s_err[:, None] * (4 + spread[:, None]) + 8 * EPS * (lpz.abs() + 4)) \
        + U(z.dtype) * want.abs() + 8 * EPS * want.abs()
    # a column that is target and alternative sums up to 1 + top_k cotangents, and -p w beside
    hits = torch.zeros_like(want)
    hits.scatter_add_(1, torch.where(live, t, torch.zeros_like(t))[:, None], al.abs()[:, None])
    hits.scatter_add_(1, ids, k.double().abs())
    # p below the smallest normal number, 2^-126, is 0 in the kernel: that times the factor of p
    bound = bound + 8 * EPS * (hits + p * size) + 2.0 ** -126 * (1 + size)
    _within(gz, want, bound, "grad")
    assert gz.dtype == z.dtype


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("rows, V, k", [(1, 1, 1), (3, 2, 2), (5, 7, 3), (4, 33, 0), (9, 100, 64),
                                        (2, 511, 20), (6, 513, 1), (37, 4096, 5), (1, 32000, 20),
                                        (4, 32000, 64), (300, 1000, 8), (3, 50021, 20),
                                        (1, 262144, 64), (2, 131073, 7), (1300, 130, 2)])
def test_logprobs_sizes(dtype, rows, V, k):
    pkg = load_pkg()
    z = _logits(rows, V, dtype)
    t = torch.randint(0, V, (rows,), generator=_gen(rows))
    _check_logprobs(pkg, z, t, k)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("V", [50, 4096, 50021])
def test_logprobs_masks(dtype, V):
    """Columns at -inf and at the type's lowest value, rows that keep one column
    or none, a lone large logit, a constant row, ignored targets."""
    pkg = load_pkg()
    z = _logits(9, V, dtype)
    z[0, V // 2:] = -math.inf
    z[1, :-1] = -math.inf
    z[2] = -math.inf
    z[3, V // 3:] = torch.finfo(dtype).min
    z[4] = torch.finfo(dtype).min
    z[5] = 1.0
    z[6, 7] = 1000.0
    z[7, ::2] = -math.inf
    z[8] = 30000.0
    t = torch.tensor([0, V - 1, 3, 1, V - 1, 0, 7, -100, 2])
    for k in (0, 5, 40):
        _check_logprobs(pkg, z, t, k)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("V", [3000, 32000, 70001])
def test_logprobs_orders_and_ties(dtype, V):
    """Rows that put many of the largest together: sorted either way, in one
    run, heavy ties, all zeros of both signs."""
    pkg = load_pkg()
    z = _logits(8, V, FP)
    z[0] = torch.sort(z[0]).values
    z[1] = torch.sort(z[1], descending=True).values
    z[2, 1000:1064] += 50.0
    z[3] = torch.round(z[3])
    z[4] = 0.0
    z[4, ::3] = -0.0
    z[5, torch.arange(0, V, max(1, V // 64))[:64]] = 100.0
    z[6] = -torch.arange(V) / V
    z[7] = torch.arange(V) // 8 % 5
    z = z.to(dtype)
    t = torch.randint(0, V, (8,), generator=_gen(3))
    for k in (1, 20, 64):
        _check_logprobs(pkg, z, t, k, grads=k == 20)


def test_logprobs_bad_rows_and_targets():
    pkg = load_pkg()
    z = _logits(6, 5000, FP)
    z[1, 4000] = math.nan
    z[2, 17] = math.inf
    z[3, :] = -math.inf
    z[3, 9] = math.nan
    t = torch.tensor([0, 1, 17, 9, 5000, -1]).cuda()
    zg = z.cuda().requires_grad_(True)
    got = pkg.token_logprobs(zg, t, entropy=True, top_k=4)
    assert torch.isnan(got.logprobs).tolist() == [False, True, True, True, True, True]
    assert torch.isnan(got.entropy).tolist() == [False, True, True, True, False, False]
    assert torch.isnan(got.top_logprobs).all(-1).tolist() == [False, True, True, True, False, False]
    for r in (1, 2, 3):
        assert got.top_ids[r].tolist() == [0, 1, 2, 3]
    (g,) = torch.autograd.grad(got.logprobs.sum(), zg)
    assert torch.isnan(g).any(-1).tolist() == [False, True, True, True, True, True]
    # ignored rows stay 0 whatever they hold, when nothing but the logprob is asked for
    lp = pkg.token_logprobs(z.cuda(), torch.full((6,), -100).cuda()).logprobs
    assert torch.equal(lp, torch.zeros(6, device="cuda"))


def test_logprobs_ignored_rows_have_no_gradient():
    """Padded positions may hold anything: their cotangents are 0, so is their
    gradient, and the other rows do not see them."""
    pkg = load_pkg()
    for V in (100, 5001):
        z = _logits(6, V, BF)
        t = torch.tensor([1, -100, 2, -100, -100, 3])
        clean = z.cuda().requires_grad_(True)
        (want,) = torch.autograd.grad(pkg.token_logprobs(clean, t.cuda()).logprobs.sum(), clean)
        z[1] = math.nan
        z[3, 5] = math.inf
        z[4] = -math.inf
        zg = z.cuda().requires_grad_(True)
        got = pkg.token_logprobs(zg, t.cuda(), top_k=3)
        (g,) = torch.autograd.grad([got.logprobs, got.top_logprobs], zg,
                                   [torch.ones(6, device="cuda"), torch.zeros(6, 3, device="cuda")])
        assert torch.equal(g, want)
        assert torch.equal(g[[1, 3, 4]], torch.zeros_like(g[:3]))
        # a cotangent on an alternative of such a row is not lost
        got = pkg.token_logprobs(zg, t.cuda(), top_k=3)
        cot = torch.zeros(6, 3, device="cuda")
        cot[1, 2] = 1.0
        (g,) = torch.autograd.grad(got.top_logprobs, zg, cot)
        assert torch.isnan(g[1]).all() and not torch.isnan(g[2:]).any()


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("V", [64, 1001, 32000])
def test_logprobs_views(dtype, V):
    """Shifted, sliced, transposed and broadcast rows, at every alignment."""
    pkg = load_pkg()
    base = _logits(3 * 5, V + 9, dtype).view(3, 5, V + 9)
    cb = base.cuda()
    t = torch.randint(0, V, (3, 4), generator=_gen(1))
    for off in (0, 1, 3, 8):
        view = base[:, :-1, off:off + V]
        cview = cb[:, :-1, off:off + V]
        got = pkg.token_logprobs(cview, t.cuda(), entropy=True, top_k=6)
        want = pkg.token_logprobs(view.contiguous().cuda(), t.cuda(), entropy=True, top_k=6)
        assert torch.equal(got.top_ids, want.top_ids)
        for a, b in zip(got[:3], want[:3]):
            # another alignment is another order of the same sums
            assert torch.allclose(a, b, rtol=0, atol=(2 ** -20) * (math.log(V) + 30))
        flat = view.reshape(-1, V)
        tt = t.reshape(-1)
        zz = cview.detach()
        _check_logprobs(pkg, flat, tt, 0, cuda_z=zz.reshape(-1, V))
        zg = zz.requires_grad_(True)
        g1 = torch.autograd.grad(pkg.token_logprobs(zg, t.cuda()).logprobs.sum(), zg)[0]
        zc = view.contiguous().cuda().requires_grad_(True)
        g2 = torch.autograd.grad(pkg.token_logprobs(zc, t.cuda()).logprobs.sum(), zc)[0]
        assert (g1.float() - g2.float()).abs().max() <= U(dtype) * 2 + 2 ** -18
    tr = cb.transpose(0, 1)[:, :, :V]
    a = pkg.token_logprobs(tr, None, entropy=True).entropy
    b = pkg.token_logprobs(tr.contiguous(), None, entropy=True).entropy
    assert a.shape == (5, 3) and torch.allclose(a, b, rtol=0, atol=1e-4)
    ex = cb[:1, :1, :V].expand(3, 4, V)
    a = pkg.token_logprobs(ex, t.cuda().int()).logprobs
    b = pkg.token_logprobs(ex.contiguous(), t.cuda()).logprobs
    assert torch.allclose(a, b, rtol=0, atol=1e-4)
    cols = cb.permute(0, 2, 1)[:, :V]    # rows that are not contiguous are copied
    a = pkg.token_logprobs(cols, None, top_k=2)
    assert torch.equal(a.top_ids, pkg.token_logprobs(cols.contiguous(), None, top_k=2).top_ids)
    one = pkg.token_logprobs(cb[0, 0], torch.tensor(3).cuda(), top_k=3)
    assert one.logprobs.shape == () and one.top_ids.shape == (3,)
    none = pkg.token_logprobs(cb[:0], None, top_k=2, entropy=True)
    assert none.entropy.shape == (0, 5) and none.top_ids.shape == (0, 5, 2)
    assert none.logprobs is None


def test_logprobs_gradient_against_differences():
    pkg = load_pkg()
    z = _logits(4, 900, FP, scale=2.0)
    t = torch.tensor([5, 899, -100, 0])
    a = torch.randn(4, generator=_gen(1)).double()
    k = torch.randn(4, 3, generator=_gen(2)).double()
    zg = z.cuda().requires_grad_(True)
    got = pkg.token_logprobs(zg, t.cuda(), entropy=True, top_k=3)
    (g,) = torch.autograd.grad(got[:3], zg, [a.float().cuda(), a.float().cuda(), k.float().cuda()])
    v = torch.randn(4, 900, generator=_gen(3), dtype=torch.float64)

    def loss(h):
        lp, ent, tops, _ = so.token_logprobs(z.double() + h * v, t, 3)
        return ((lp + ent) * a).sum().item() + (tops * k).sum().item()

    want = (loss(1e-6) - loss(-1e-6)) / 2e-6
    assert abs((g.double().cpu() * v).sum().item() - want) < 1e-4


# ---------------------------------------------------------------------------
# activations in 8 bits
# ---------------------------------------------------------------------------

def _acts(n, dtype, seed=0):
    g = _gen(seed + n)
    x = 2 * torch.randn(n, generator=g) * torch.exp(torch.randn((n + 99) // 100, generator=g)
                                                    .repeat_interleave(100)[:n])
    return x.to(dtype)


SIZES = [1, 2, 15, 16, 17, 127, 128, 129, 1000, 4096, 4111, 128 * 1000 + 5, 1 << 20]


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("n", SIZES)
def test_pack8_codes_are_the_definitions(dtype, n):
    pkg = load_pkg()
    x = _acts(n, dtype)
    p = pkg.pack8(x.cuda())
    codes, scales = so.pack8(x)
    assert torch.equal(p.codes.cpu(), codes) and torch.equal(p.scales.cpu(), scales)
    back = pkg.unpack8(p)
    # one fp32 product, then the type's rounding
    want = (codes.float() * scales.repeat_interleave(128)[:n]).to(dtype)
    assert torch.equal(back.cpu(), want) and back.dtype == dtype


def test_pack8_special_blocks():
    pkg = load_pkg()
    x = _acts(128 * 10, FP).view(10, 128)
    x[0] = 0.0
    x[1] = x[1] * 2.0 ** -110           # below the smallest kept magnitude
    x[2, 5] = math.nan
    x[3, 6] = -math.inf
    x[4] = torch.linspace(-3.4e38, 3.4e38, 128)     # its range overflows: infinities and NaN
    x[5] = 2.0 ** -100                  # exactly the smallest kept
    x[6] = 2.0 ** -149
    x[7] = (torch.arange(128) - 64).float() + 0.5   # borders between codes
    x[8] = torch.arange(128).float() * 2.0 - 127.0  # every odd code: exact
    x[9] = torch.linspace(-1.0, 1.0, 128) * 3.4e38  # up to the type's largest
    p = pkg.pack8(x.cuda())
    codes, scales = so.pack8(x)
    back = pkg.unpack8(p).cpu()
    assert not torch.isfinite(x[4]).any()
    assert torch.isnan(back[2:5]).all()
    assert torch.equal(torch.isnan(p.scales.cpu()), torch.isnan(scales))
    keep = [0, 1, 5, 6, 7, 8, 9]
    assert torch.equal(p.codes.cpu()[keep], codes[keep])
    assert torch.equal(p.scales.cpu()[keep], scales[keep])
    assert torch.equal(back[[0, 1, 6]], torch.zeros(3, 128))
    assert torch.equal(back[8], x[8])


def test_pack8_views_and_empty():
    pkg = load_pkg()
    x = _acts(4000, BF).view(40, 100).cuda()
    for v in (x.t(), x[:, 3:50], x[::2], x.flatten()[1:], x[:0], x.new_empty(0)):
        p = pkg.pack8(v)
        assert p.codes.shape == v.shape
        assert torch.equal(pkg.unpack8(p), pkg.unpack8(pkg.pack8(v.contiguous().clone())))
    # a slice of a checkpoint that starts at a block is a checkpoint
    p = pkg.pack8(_acts(1024, FP).cuda())
    tail = pkg.Packed8(p.codes[256:], p.scales[2:], p.dtype)
    assert torch.equal(pkg.unpack8(tail), pkg.unpack8(p)[256:])


def _act_grads(x, gate, dy):
    x = x.clone().requires_grad_(True)
    gate = None if gate is None else gate.clone().requires_grad_(True)
    y = so.act(x, gate)
    return y.detach(), torch.autograd.grad(y, [x] if gate is None else [x, gate], dy.double())


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("n", SIZES)
def test_act8(dtype, gated, n):
    pkg = load_pkg()
    x, gate, dy = _acts(n, dtype), _acts(n, dtype, 1) if gated else None, _acts(n, dtype, 2)
    y, saved = pkg.act8_forward(x.cuda(), None if gate is None else gate.cuda())
    for kept, t in ((saved.x, x), (saved.gate, gate)):
        if t is not None:
            codes, scales = so.pack8(t)
            assert torch.equal(kept.codes.cpu(), codes) and torch.equal(kept.scales.cpu(), scales)
    # GELU: the share P is within 2e-7 of erf's (a published approximation's bound, halved, and
    # fp32 roundings) or 8 ulp; SwiGLU: a sigmoid within 2^-21, three products
    far = (x.double().abs() * (2e-7 if dtype == BF else 8 * EPS) if not gated else
           (x.double() * gate.double()).abs() * 2.0 ** -21)
    want = so.act(x, gate)
    _within(y, want, far + (U(dtype) + 8 * EPS) * want.abs(), "y")
    xr = so.unpack8(*so.pack8(x))
    gr = None if gate is None else so.unpack8(*so.pack8(gate))
    want_y, grads = _act_grads(xr, gr, dy)
    dx, dgate, back = pkg.act8_backward(saved, dy.cuda())
    d = dy.double().abs()
    if gated:
        a = gr.abs()
        fars = [d * a * 2.0 ** -20, d * xr.abs() * (1 + a) * 2.0 ** -20]
        far = (xr * gr).abs() * 2.0 ** -20
    else:
        # P, and x phi(x) with an exponential of x^2 / 2
        fars = [d * ((2e-7 if dtype == BF else 8 * EPS) * (1 + xr.abs())
                     + 2.0 ** -21 * xr.abs() * torch.exp(-xr * xr / 2) * (1 + xr * xr))]
        far = xr.abs() * (2e-7 if dtype == BF else 8 * EPS)
    _within(dx, grads[0], fars[0] + (U(dtype) + 16 * EPS) * grads[0].abs(), "dx")
    if gated:
        _within(dgate, grads[1], fars[1] + (U(dtype) + 16 * EPS) * grads[1].abs(), "dgate")
    else:
        assert dgate is None
    _within(back, want_y, far + (U(dtype) + 16 * EPS) * want_y.abs(), "restored y")
    again = pkg.act8_backward(saved, dy.cuda(), restore=False)
    assert again[2] is None and torch.equal(again[0], dx)


def test_act8_tails():
    """Far arguments of both signs: the exponentials neither overflow nor lose
    the small side."""
    pkg = load_pkg()
    for dtype in (BF, FP):
        x = torch.cat([torch.linspace(-40, 40, 1280), torch.tensor([-1e4, 1e4, 0.0, -0.0])]).to(dtype)
        dy = torch.ones_like(x)
        for gate in (None, x.flip(0).clone()):
            y, saved = pkg.act8_forward(x.cuda(), None if gate is None else gate.cuda())
            want = so.act(x, gate)
            far = x.double().abs() * (2e-7 if dtype == BF else 8 * EPS) if gate is None else \
                (x.double() * gate.double()).abs() * 2.0 ** -21
            _within(y, want, far + (U(dtype) + 8 * EPS) * want.abs(), "y")
            dx, dgate, back = pkg.act8_backward(saved, dy.cuda())
            assert torch.isfinite(dx).all() and torch.isfinite(back).all()
            assert dgate is None or torch.isfinite(dgate).all()


def test_act8_fp32_gelu_keeps_its_digits():
    """The small side too: P(x) is a product t q e, relative to it the fit (2e-8), 11
    roundings of which those of the sum's leading terms count in full (3.5e-7 in a model of
    them), the exponential (2^-22) and the reciprocal (2^-23): 8e-7 and y's own rounding.
    For |x| < 1 it is 1/2 + x R: two half ulps of at most 1 over P >= 0.158, 4e-7."""
    pkg = load_pkg()
    x = torch.cat([torch.linspace(-12, 12, 1 << 18), torch.linspace(-1.01, 1.01, 1 << 16),
                   torch.tensor([1.0, -1.0, 14.0, 15.0, 16.0, 1e6, 1e-30, -1e-30])])
    y, _ = pkg.act8_forward(x.cuda())
    want = x.double() * torch.special.erfc(-x.double() / 2.0 ** 0.5) / 2
    rel = ((y.cpu().double() - want) / want.abs().clamp_min(2.0 ** -126)).abs()
    print("largest relative error", rel.max().item())
    assert rel.max() <= 8e-7 + EPS
    inf = float("inf")
    bad, _ = pkg.act8_forward(torch.tensor([inf, -inf, float("nan"), 3.0]).cuda())
    assert bad[0] == inf and bad[1].isnan() and bad[2].isnan()


# ---------------------------------------------------------------------------
# the MLP, and the operators together
# ---------------------------------------------------------------------------

def _restored(pkg, t):
    return pkg.unpack8(pkg.pack8(t))


@pytest.mark.parametrize("gated", [False, True])
def test_mlp8_gradients(gated):
    """fp32 against the formulas with restored tensors in fp64, every subset of
    leaves, and the memory that autograd keeps."""
    pkg = load_pkg()
    g = _gen(11)
    x = torch.randn(6, 50, 96, generator=g).cuda().requires_grad_(True)
    ws = [(torch.randn(s, generator=g) / 10).cuda().requires_grad_(True)
          for s in ((200, 96), (64, 200), (200, 96))[:3 if gated else 2]]
    dout = torch.randn(6, 50, 64, generator=g).cuda()
    out = pkg.mlp8(x, *ws)
    grads = torch.autograd.grad(out, [x, *ws], dout, retain_graph=True)
    with torch.no_grad():
        rows = x.reshape(-1, 96)
        up = F.linear(rows, ws[0])
        gate = F.linear(rows, ws[2]) if gated else None
        ur, gr = _restored(pkg, up), _restored(pkg, gate) if gated else None
        xr = _restored(pkg, rows).double()
        d = dout.reshape(-1, 64).double()
        dyv = d @ ws[1].double()
    cpu = [None if t is None else t.cpu() for t in (ur, gr)]
    yr, da = _act_grads(*[None if t is None else t.double() for t in cpu], dyv.cpu())
    da = [t.cuda() for t in da]
    want_x = da[0] @ ws[0].double() + (da[1] @ ws[2].double() if gated else 0.0)
    want = [want_x.view_as(x), da[0].mT @ xr, d.mT @ yr.cuda()] + \
        ([da[1].mT @ xr] if gated else [])
    plain = so.act(up.cpu(), None if gate is None else gate.cpu()).cuda() @ ws[1].double().mT
    # products of up to 300 fp32 terms of size ~ 1
    assert (out.double().view_as(plain) - plain).abs().max() < 1e-4 * plain.abs().max()
    for a, b in zip(grads, want):
        assert (a.double() - b).abs().max() < 1e-4 * b.abs().max()
    (gx,) = torch.autograd.grad(pkg.mlp8(x, *[w.detach() for w in ws]), x, dout)
    assert torch.equal(gx, grads[0])
    (gd,) = torch.autograd.grad(pkg.mlp8(x.detach(), ws[0].detach(), ws[1],
                                         *[w.detach() for w in ws[2:]]), ws[1], dout)
    assert torch.equal(gd, grads[2])
    with torch.no_grad():
        assert torch.equal(pkg.mlp8(x, *ws), out)


def test_mlp8_autocast_and_kept_memory():
    pkg = load_pkg()
    g = _gen(12)
    x = torch.randn(4096, 512, generator=g).cuda().to(BF).requires_grad_(True)
    w1 = (torch.randn(2048, 512, generator=g) / 20).cuda().requires_grad_(True)
    w2 = (torch.randn(512, 2048, generator=g) / 40).cuda().requires_grad_(True)
    with torch.autocast("cuda", dtype=BF):
        pkg.mlp8(x, w1, w2)
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        out = pkg.mlp8(x, w1, w2)
    kept = torch.cuda.memory_allocated() - before - out.numel() * 2
    # 1 B and 1/32 B of scales an element of x and of the hidden layer, two cast weights
    assert kept < (x.numel() + 4096 * 2048) * 1.04 + 2 * 2 * w1.numel() + (1 << 20)
    out.float().square().mean().backward()
    assert out.dtype == BF and w1.grad.dtype == FP and x.grad.dtype == BF
    ref = F.linear(F.gelu(F.linear(x.detach(), w1.detach().to(BF))), w2.detach().to(BF))
    assert (out - ref).abs().max() <= 3 * U(BF) * ref.abs().max() + 0.02
    with pytest.raises(TypeError):
        pkg.mlp8(x, w1, w2)     # bf16 with fp32 weights outside autocast


@pytest.mark.parametrize("gated", [False, True])
def test_mlp8_backward_under_another_autocast(gated):
    """An fp32 forward's backward inside an autocast region keeps fp32: equal bits."""
    pkg = load_pkg()
    g = _gen(13)
    x = torch.randn(70, 64, generator=g).cuda().requires_grad_(True)
    ws = [(torch.randn(s, generator=g) / 8).cuda().requires_grad_(True)
          for s in ((130, 64), (64, 130), (130, 64))[:3 if gated else 2]]
    dout = torch.randn(70, 64, generator=g).cuda()
    want = torch.autograd.grad(pkg.mlp8(x, *ws), [x, *ws], dout)
    out = pkg.mlp8(x, *ws)
    with torch.autocast("cuda", dtype=BF):
        got = torch.autograd.grad(out, [x, *ws], dout)
    for a, b in zip(got, want):
        assert a.dtype == FP and torch.equal(a, b)


def _block(pkg, p, idx, targets):
    """Two residual branches and the head on the operators, as a model uses them."""
    h = p["emb"][idx]
    y = pkg.rms_norm(h, p["n1"], out_dtype=p["dt"])
    branch = F.linear(y, p["w"].to(p["dt"]))
    y, h = pkg.rms_norm(branch, p["n2"], residual=h, out_dtype=p["dt"])
    y, h = pkg.layer_norm(pkg.mlp8(y, p["w1"].to(p["dt"]), p["w2"].to(p["dt"])), p["n3"], p["b3"],
                          residual=h, out_dtype=p["dt"])
    got = pkg.token_logprobs(F.linear(y, p["emb"].to(p["dt"])), targets, entropy=True, top_k=3)
    return -got.logprobs.mean() - 0.01 * got.entropy.mean() + 0.01 * got.top_logprobs.mean(), got


def _block_plain(p, idx, targets, restored):
    h = p["emb"][idx]
    y, _ = so.norm(h, p["n1"], None, torch.finfo(FP).eps, None, False)
    h = h + F.linear(y, p["w"])
    y, _ = so.norm(h, p["n2"], None, torch.finfo(FP).eps, None, False)
    y = F.linear(so.act(F.linear(y, p["w1"])), p["w2"])
    h = h + y
    y, _ = so.norm(h, p["n3"], p["b3"])
    lp, ent, tops, _ = so.token_logprobs(F.linear(y, p["emb"]), targets, 3)
    return -lp.mean() - 0.01 * ent.mean() + 0.01 * tops.mean()


def _params(dt, V=1001, D=128, Fh=512):
    g = _gen(21)
    r = lambda *s: torch.randn(*s, generator=g) / 8
    return dict(emb=r(V, D) * 4, w=r(D, D), w1=r(Fh, D), w2=r(D, Fh), n1=1 + r(D), n2=1 + r(D),
                n3=1 + r(D), b3=r(D), dt=dt), torch.randint(0, V, (2, 40), generator=g), \
        torch.randint(0, V, (2, 40), generator=g)


def test_operators_together_against_fp64():
    """A block and the loss in fp32: the only inexact step is the 8-bit
    checkpoint, half a step of 1 / 254 of a block's largest magnitude, in the
    MLP's gradients."""
    pkg = load_pkg()
    p, idx, t = _params(FP)
    leaves = [n for n in p if n != "dt"]
    gp = {n: p[n].cuda().requires_grad_(True) if n != "dt" else FP for n in p}
    loss, _ = _block(pkg, gp, idx.cuda(), t.cuda())
    grads = torch.autograd.grad(loss, [gp[n] for n in leaves])
    dp = {n: p[n].double().requires_grad_(True) if n != "dt" else None for n in p}
    want = _block_plain(dp, idx, t, False)
    wg = torch.autograd.grad(want, [dp[n] for n in leaves])
    # fp32 through five products of up to 512 terms and three norms
    assert abs(loss.item() - want.item()) < 1e-5 * abs(want.item())
    for n, a, b in zip(leaves, grads, wg):
        exact = n in ("n3", "b3")      # nothing of the checkpoint reaches these
        assert (a.double().cpu() - b).norm() <= (1e-5 if exact else 2e-2) * b.norm(), n


@pytest.mark.parametrize("dt", [BF, FP])
def test_operators_in_a_captured_graph(dt):
    """The run of them captured, replayed on new inputs; equal to plain calls."""
    pkg = load_pkg()
    p, idx, t = _params(dt)
    leaves = [n for n in p if n != "dt"]
    gp = {n: p[n].cuda().requires_grad_(True) if n != "dt" else dt for n in p}
    idx, t = idx.cuda(), t.cuda()

    def step():
        loss, got = _block(pkg, gp, idx, t)
        return (loss.detach(), got.top_ids, *torch.autograd.grad(loss, [gp[n] for n in leaves]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    t.copy_((t + 1) % 1001)
    with torch.no_grad():
        gp["n2"].mul_(1.5)
    graph.replay()
    want = step()
    torch.cuda.synchronize()
    for n, a, b in zip(["loss", "ids", *leaves], out, want):
        if n == "emb":   # torch's embedding gradient adds with atomics
            assert (a - b).norm() <= 1e-5 * b.norm()
        else:
            assert torch.equal(a, b), n


def test_two_streams_at_once():
    """Calls that overlap on two streams share nothing."""
    pkg = load_pkg()
    p, idx, t = _params(BF, V=5003)
    leaves = [n for n in p if n != "dt"]
    gp = {n: p[n].cuda().requires_grad_(True) if n != "dt" else BF for n in p}
    idx, t = idx.cuda(), t.cuda()
    shifted = (t + 7) % 5003

    def step(targets):
        loss, got = _block(pkg, gp, idx, targets)
        return (loss.detach(), got.top_ids,
                *torch.autograd.grad(loss, [gp[n] for n in leaves if n != "emb"]))

    want = [step(t), step(shifted)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        got = [None, None]
        for i, (s, targets) in enumerate(zip(streams, (t, shifted))):
            with torch.cuda.stream(s):
                got[i] = step(targets)
        torch.cuda.synchronize()
        for a, b in zip(want, got):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_the_same_tensor_twice_and_nothing_at_all():
    pkg = load_pkg()
    x = torch.randn(9, 200, generator=_gen(1)).cuda().requires_grad_(True)
    w = torch.randn(200, generator=_gen(2)).cuda().requires_grad_(True)
    y, h = pkg.rms_norm(x, w, w, 1e-5, residual=x)      # x + x, and w as weight and bias
    cot = torch.randn(9, 200, generator=_gen(3)).cuda()
    gx, gw = torch.autograd.grad([y, h], [x, w], [cot, cot])
    xr, wr = x.detach().double().requires_grad_(True), w.detach().double().requires_grad_(True)
    yr, hr = so.norm(2 * xr, wr, wr, 1e-5, None, False)
    ex, ew = torch.autograd.grad([yr, hr], [xr, wr], [cot.double()] * 2)
    # fp32 through sums of 200 and of 9
    assert (gx - ex).abs().max() < 64 * EPS * ex.abs().max()
    assert (gw - ew).abs().max() < 64 * EPS * ew.abs().max()
    a = _acts(1000, BF).cuda()
    y, saved = pkg.act8_forward(a, a)
    _within(y, so.act(a.cpu(), a.cpu()), (U(BF) + 2.0 ** -20) * so.act(a.cpu(), a.cpu()).abs(), "y")
    for shape in ((0, 16), (3, 0, 16)):
        x = torch.empty(shape, device="cuda", requires_grad=True)
        w1 = torch.randn(32, 16, device="cuda", requires_grad=True)
        w2 = torch.randn(8, 32, device="cuda", requires_grad=True)
        out = pkg.mlp8(x, w1, w2, w1)
        out.sum().backward()
        assert out.shape == (*shape[:-1], 8) and x.grad.shape == x.shape
        assert not w1.grad.any() and not w2.grad.any()
    empty = torch.empty(0, 5, device="cuda")
    y, saved = pkg.act8_forward(empty, empty)
    dx, dgate, back = pkg.act8_backward(saved, empty)
    assert y.shape == dx.shape == dgate.shape == back.shape == (0, 5)


def test_opcheck():
    """The dispatcher's view of every op: schema, fake kernels, autograd."""
    pkg = load_pkg()
    utils = ("test_schema", "test_autograd_registration", "test_faketensor",
             "test_aot_dispatch_static")
    ops = torch.ops.gmdn
    g = _gen(31)
    x = torch.randn(6, 64, generator=g).cuda().requires_grad_(True)
    r = torch.randn(6, 64, generator=g).cuda().to(BF).requires_grad_(True)
    w = torch.randn(64, generator=g).cuda().requires_grad_(True)
    torch.library.opcheck(ops.norm_fwd.default, (x, r, w, None, 1e-5, True, False), test_utils=utils)
    torch.library.opcheck(ops.norm_fwd.default, (x, None, None, w, 1e-5, False, True),
                          test_utils=utils)
    t = torch.tensor([1, 2, 3, -100, 5, 6]).cuda()
    torch.library.opcheck(ops.token_logprobs_fwd.default, (x, t, True, 3, -100), test_utils=utils)
    torch.library.opcheck(ops.token_logprobs_fwd.default, (x, None, True, 0, -100),
                          test_utils=utils)
    half = ("test_schema", "test_faketensor")
    xd = x.detach()
    torch.library.opcheck(ops.pack8.default, (xd,), test_utils=half)
    codes, scales = ops.pack8(xd)
    torch.library.opcheck(ops.unpack8.default, (codes, scales, True), test_utils=half)
    torch.library.opcheck(ops.act8_fwd.default, (xd, xd), test_utils=half)
    torch.library.opcheck(ops.act8_bwd.default, (codes, scales, None, None, xd, True),
                          test_utils=half)


def test_dispatcher_route_equals_the_direct_one():
    """Under a dispatch mode the calls go through the registered ops, with the
    same bits and gradients."""
    from torch.utils._python_dispatch import TorchDispatchMode
    seen = []

    class Watch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))

    pkg = load_pkg()
    p, idx, t = _params(FP)
    leaves = [n for n in p if n not in ("dt", "emb")]
    gp = {n: p[n].cuda().requires_grad_(True) if n != "dt" else FP for n in p}

    def step():
        loss, _ = _block(pkg, gp, idx.cuda(), t.cuda())
        return (loss.detach(), *torch.autograd.grad(loss, [gp[n] for n in leaves]))

    want = step()
    with Watch():
        got = step()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    for name in ("norm_fwd", "norm_bwd", "token_logprobs_fwd", "token_logprobs_bwd", "pack8",
                 "unpack8", "act8_fwd", "act8_bwd"):
        assert any(name in s for s in seen), name


def test_compiled_block_matches_eager():
    pkg = load_pkg()
    torch._dynamo.reset()
    p, idx, t = _params(FP)
    idx, t = idx.cuda(), t.cuda()
    leaves = [n for n in p if n != "dt"]

    def grads(fn):
        gp = {n: p[n].cuda().requires_grad_(True) if n != "dt" else FP for n in p}
        loss = fn(gp)
        return loss.detach(), torch.autograd.grad(loss, [gp[n] for n in leaves])

    la, ga = grads(lambda gp: _block(pkg, gp, idx, t)[0])
    lb, gb = grads(torch.compile(lambda gp: _block(pkg, gp, idx, t)[0], dynamic=False))
    assert torch.allclose(la, lb, rtol=1e-5)
    for n, a, b in zip(leaves, ga, gb):
        # another order of the plain parts can move a code by one: as far as the checkpoint goes
        assert (a - b).norm() <= 2e-2 * b.norm() + 1e-12, n


def test_double_backward_is_refused():
    pkg = load_pkg()
    z = torch.randn(4, 50, generator=_gen(1)).cuda().requires_grad_(True)
    lp = pkg.token_logprobs(z, torch.zeros(4, dtype=torch.int64).cuda()).logprobs
    (g,) = torch.autograd.grad(lp.sum(), z, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_offsets_past_32_bits():
    """A row and a block whose element offsets need 33 bits."""
    pkg = load_pkg()
    V, rows = 50021, 43000                       # 2.15e9 elements
    z = torch.zeros(rows, V, dtype=BF, device="cuda")
    z[-1, 777] = 5.0
    z[-1, -1] = 6.0
    got = pkg.token_logprobs(z, torch.full((rows,), 777, device="cuda"), top_k=2)
    want = 5.0 - math.log(V - 2 + math.exp(5.0) + math.exp(6.0))
    assert abs(got.logprobs[-1].item() - want) < 1e-5
    assert got.top_ids[-1].tolist() == [V - 1, 777] and got.top_ids[0].tolist() == [0, 1]
    g = torch.ops.gmdn.token_logprobs_bwd(
        z, torch.full((rows,), 777, device="cuda"), None,
        torch.tensor([[0.0, math.log(V), math.log(V), 0.0]], device="cuda").expand(rows, 4)
        .contiguous(), torch.ones(rows, device="cuda"), None, None, -100)
    assert abs(g[-2, 777].item() - 1.0) < 2 ** -8 and abs(g[-2, 5].item() * V + 1.0) < 2 ** -7
    del g
    p = pkg.pack8(z)
    assert p.codes[-1, 777] == 127
    back = pkg.unpack8(p)
    assert back[-1, -1].item() == 6.0 and back[0, 0].item() == 0.0
    del p, back
    y = pkg.rms_norm(z, None, None, 1.0)
    want = 6.0 / math.sqrt((25.0 + 36.0) / V + 1.0)
    assert abs(y[-1, -1].item() - want) <= 2 ** -8 * want
