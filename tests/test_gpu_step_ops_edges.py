"""The step operators at the borders between their ways: sizes, types, views and
cotangents that the other tests pass by."""
import math

import pytest
import torch
import torch.autograd.forward_ad as fw

from conftest import load_pkg
from oracle import step_oracle as so
from test_gpu_step_ops import (BF, EPS, FP, U, _check_logprobs, _check_norm, _gen, _norm_case,
                               _within)

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


@pytest.mark.parametrize("gated", [False, True])
def test_mlp8_refuses_forward_mode(gated):
    pkg = load_pkg()
    g = _gen(3)
    ps = [torch.randn(s, generator=g).cuda() for s in ((3, 64), (128, 64), (64, 128), (128, 64))]
    ps = ps[:4 if gated else 3]
    for grad in (False, True):
        for i, p in enumerate(ps):
            with torch.set_grad_enabled(grad), fw.dual_level(), \
                    pytest.raises((RuntimeError, NotImplementedError)):
                pkg.mlp8(*ps[:i], fw.make_dual(p, torch.ones_like(p)), *ps[i + 1:])
            with torch.set_grad_enabled(grad), pytest.raises((RuntimeError, NotImplementedError)):
                torch.func.jvp(lambda d: pkg.mlp8(*ps[:i], d, *ps[i + 1:]), (p,), (p,))
    x = ps[0].clone().requires_grad_(True)
    out = pkg.mlp8(x, *ps[1:])
    with fw.dual_level(), pytest.raises((RuntimeError, NotImplementedError)):
        torch.autograd.grad(out, x, fw.make_dual(torch.ones_like(out), torch.ones_like(out)))
    with fw.dual_level():       # no tangent among the inputs: nothing to refuse
        plain = pkg.mlp8(x.detach(), *ps[1:])
    assert torch.equal(plain, out)


def test_mlp8_without_gradients_compiles_whole():
    pkg = load_pkg()
    torch._dynamo.reset()
    g = _gen(4)
    ps = [torch.randn(s, generator=g).cuda() for s in ((40, 64), (128, 64), (64, 128))]
    got = torch.compile(lambda *p: pkg.mlp8(*p), fullgraph=True, dynamic=False)(*ps)
    assert torch.allclose(got, pkg.mlp8(*ps), rtol=1e-5, atol=1e-4)


@pytest.mark.parametrize("x_dt, res_dt", [(BF, FP), (FP, BF), (BF, BF), (FP, FP)])
@pytest.mark.parametrize("D", [64, 1283, 16384])
def test_norm_with_only_h_used(x_dt, res_dt, D):
    """Without a cotangent of y the gradient is that of h, whatever the rows hold."""
    pkg = load_pkg()
    c = _norm_case(4, D, True, x_dt, res_dt, BF)
    c["x"][1, 5 % D] = math.inf
    c["x"][2, 3 % D] = math.nan
    leaves = [c[n].cuda().requires_grad_(True) for n in ("x", "res", "w", "b")]
    for call in (pkg.layer_norm, pkg.rms_norm):
        _, h = call(leaves[0], leaves[2], leaves[3], 1e-5, residual=leaves[1])
        dh = c["dh"].cuda()
        dx, dr, dw, db = torch.autograd.grad(h, leaves, dh)
        assert torch.equal(dx, dh.to(x_dt)) and torch.equal(dr, dh.to(res_dt))
        assert not dw.any() and not db.any() and dw.shape == db.shape == (D,)
        (dx,) = torch.autograd.grad(
            call(leaves[0], residual=leaves[1].detach())[1], leaves[0], dh)
        assert torch.equal(dx, dh.to(x_dt))


@pytest.mark.parametrize("gated", [False, True])
def test_mlp8_of_no_width(gated):
    """A width of 0 anywhere: the shapes and zeros that nn.Linear gives."""
    pkg = load_pkg()
    for lead in ((5,), (2, 3), ()):
        for D, Fh, Do in ((0, 8, 4), (4, 0, 3), (4, 8, 0), (0, 0, 0)):
            ps = [torch.randn(s, generator=_gen(5)).cuda().requires_grad_(True)
                  for s in ((*lead, D), (Fh, D), (Do, Fh), (Fh, D))[:4 if gated else 3]]
            out = pkg.mlp8(*ps)
            assert out.shape == (*lead, Do) and not out.any()
            grads = torch.autograd.grad(out, ps, torch.ones_like(out))
            for g, p in zip(grads, ps):
                assert g.shape == p.shape and not g.any()
            with torch.no_grad():
                assert pkg.mlp8(*ps).shape == out.shape


def _half_step(v, dtype):
    """Half the distance between the type's numbers around v (of the subnormal ones below)."""
    e = torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -126)))
    return torch.exp2(e) * U(dtype)


def _tails(dtype):
    """Arguments of both signs where P, the sigmoid and their products stay normal numbers."""
    x = torch.cat([torch.linspace(-13, 13, 1 << 14), torch.linspace(-3, 3, 1 << 12)])
    # blocks of 128 around one magnitude, so that the 8-bit values are as far out as the input's
    return x.sort().values.to(dtype)


@pytest.mark.parametrize("dtype", [BF, FP])
def test_gelu_keeps_its_digits_on_the_small_side(dtype):
    """Relative to y, dx and the restored y themselves.  P is within 5.4e-5 (bf16: the fit) or
    8e-7 (fp32: see the fp32 test of y) of its value, e^(-x^2 / 2) within 2^-22 and, for bf16,
    two roundings of its exponent, x^2 / 2 EPS each; then at most 8 fp32 roundings of terms no
    larger than P and |x| phi, and the output's own.  Below 2^-126 the exponential is 0."""
    pkg = load_pkg()
    x = _tails(dtype)
    rel = 5.4e-5 if dtype == BF else 8e-7   # beyond the roundings counted in check()

    def share(v):
        return torch.special.erfc(-v / math.sqrt(2.0)) / 2

    def check(got, want, terms, exponent, what):
        fp32 = 8 * EPS * terms + 2.0 ** -126 * 16
        _within(got, want, exponent + fp32 + _half_step(want, dtype) * (1 + 2.0 ** -8), what)

    def parts(v):
        v = v.double()
        phi = torch.exp(-v * v / 2) / math.sqrt(2 * math.pi)
        e_err = 2.0 ** -22 + (v * v * EPS if dtype == BF else 0.0)
        return v, share(v), phi, (rel + e_err) * share(v), e_err * phi

    y, saved = pkg.act8_forward(x.cuda())
    v, P, phi, P_err, phi_err = parts(x)
    check(y, v * P, v.abs() * P, v.abs() * P_err, "y")
    dx, _, back = pkg.act8_backward(saved, torch.ones_like(x).cuda())
    v, P, phi, P_err, phi_err = parts(so.unpack8(*so.pack8(x)).float())
    check(back, v * P, v.abs() * P, v.abs() * P_err, "restored y")
    check(dx, P + v * phi, P + v.abs() * phi, P_err + v.abs() * phi_err, "dx")


@pytest.mark.parametrize("dtype", [BF, FP])
def test_swiglu_keeps_its_digits_on_the_small_side(dtype):
    """Relative: the sigmoid is 1 / (1 + e^-a), off by 2^-21 and, for bf16, by the rounding of
    its exponent, |a| 2 EPS (log2 e and the product); dgate's slope is the sum of sig, silu and
    -silu sig.  A sigmoid below 2^-126 is 0."""
    pkg = load_pkg()
    a = torch.cat([_tails(dtype).float() * 6, _tails(dtype).float()]).sort().values.to(dtype)
    u = torch.linspace(0.5, 3.0, a.numel()).to(dtype)
    y, saved = pkg.act8_forward(u.cuda(), a.cuda())
    dx, dgate, back = pkg.act8_backward(saved, torch.ones_like(u).cuda())

    def parts(t):
        t = t.double()
        sig = torch.sigmoid(t)
        return t, sig, 2.0 ** -21 + (2 * EPS * t.abs() if dtype == BF else 0.0)

    def check(got, want, size, rel, what):
        _within(got, want, size * (rel + 8 * EPS) + 2.0 ** -125 * 300
                + _half_step(want, dtype) * (1 + 2.0 ** -8), what)

    t, sig, rel = parts(a)
    check(y, t * sig * u.double(), (t * sig * u.double()).abs(), rel, "y")
    t, sig, rel = parts(so.unpack8(*so.pack8(a)).float())
    w = so.unpack8(*so.pack8(u)).float().double()
    check(back, t * sig * w, (t * sig * w).abs(), rel, "restored y")
    check(dx, t * sig, (t * sig).abs(), rel, "dx")
    check(dgate, w * sig * (1 + t * (1 - sig)), w * sig * (1 + 2 * t.abs()), 2 * rel, "dgate")


@pytest.mark.parametrize("V", [400, 401])
def test_logprobs_fp32_gradient_keeps_its_digits(V):
    """The gradient's -p relative to itself, down to e^-85, in EPS: the exponential 4 (2^-22) and
    its correction 2; 1 / S and the products 3; S: a thread's chunk, a warp's and the warps'
    joins 14 adds, and the exponentials of the columns that make it, 4 + 1.5 |c| each.  The logits
    are multiples of 2^-8, so x - max is exact.  Below 2^-126 the exponential is 0."""
    pkg = load_pkg()
    z = torch.round(torch.rand(64, V, generator=_gen(V)) * -90 * 256) / 256
    z[:, 7] = 2.0
    t = torch.full((64,), 7)
    zg = z.cuda().requires_grad_(True)
    got = pkg.token_logprobs(zg, t.cuda(), entropy=True)
    lp = torch.log_softmax(z.double(), -1)
    p = lp.exp()
    c = z.double() - z.double().amax(-1, keepdim=True)
    s_err = 14 + 4 + 1.5 * (p * c.abs()).sum(-1, keepdim=True)
    rel = (s_err + 4 + 2 + 3) * EPS
    tiny = 2.0 ** -126
    others = torch.arange(V) != 7
    (g,) = torch.autograd.grad(got.logprobs.sum(), zg, retain_graph=True)
    _within(g.cpu()[:, others], -p[:, others], (p * rel + tiny)[:, others], "-p")
    # the entropy's: p (logprob + H) with log S, the logprob and H off by 2 EPS of themselves each
    H = -(p * lp).sum(-1, keepdim=True)
    (g,) = torch.autograd.grad(got.entropy.sum(), zg)
    size = lp.abs() + H + torch.log(torch.exp(c).sum(-1, keepdim=True)).abs()
    _within(g, -p * (lp + H), p * size * (rel + 8 * EPS) + p * (s_err * EPS * 4) + 100 * tiny,
            "entropy")


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("V", [64, 1001, 5003, 32000])
def test_logprobs_of_the_views_themselves(dtype, V):
    """Rows at every alignment, read in place: outputs and the gradient (whose rows lie at
    another alignment) element by element against the oracle, with entropy and alternatives."""
    pkg = load_pkg()
    base = (torch.randn(15, V + 9, generator=_gen(V)) * 3).to(dtype)
    cb = base.cuda()
    t = torch.randint(0, V, (15,), generator=_gen(1))
    t[4] = -100
    for off in range(9 if dtype == BF else 5):
        view = cb[:, off:off + V]
        seen = []

        class Calls:      # the call that the check makes, with the tensor that it is given
            @staticmethod
            def token_logprobs(z, *args, **kw):
                seen.append((z.data_ptr(), z.stride()))
                return pkg.token_logprobs(z, *args, **kw)

        for k in (0, 6):
            _check_logprobs(Calls, base[:, off:off + V], t, k, cuda_z=view)
        assert seen == [(view.data_ptr(), (V + 9, 1))] * 2
        # the same rows as a shifted batch: equal bits
        cube = cb.view(3, 5, V + 9)[:, :-1, off:off + V]
        keep = [r for r in range(15) if r % 5 != 4]
        flat = view.detach().requires_grad_(True)
        zg = cube.detach().requires_grad_(True)
        assert zg.data_ptr() == view.data_ptr() and zg.stride() == (5 * (V + 9), V + 9, 1)
        for kw in (dict(entropy=True, top_k=6), dict(entropy=True), dict(top_k=3), dict()):
            a = pkg.token_logprobs(flat, t.cuda(), **kw)
            b = pkg.token_logprobs(zg, t[keep].view(3, 4).cuda(), **kw)
            cots = [torch.randn(x.shape, generator=_gen(7)).cuda() for x in a[:3] if x is not None]
            for x, y in zip(a, b):
                assert (x is None) == (y is None)
                assert x is None or torch.equal(x[keep], y.reshape(12, *y.shape[2:]))
            (ga,) = torch.autograd.grad([x for x in a[:3] if x is not None], flat, cots)
            (gb,) = torch.autograd.grad([x for x in b[:3] if x is not None], zg,
                                        [c[keep].view(3, 4, *c.shape[1:]) for c in cots])
            assert torch.equal(ga[keep], gb.reshape(12, V))


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("rows, V, parts", [(160, 20003, 1), (2, 131073, 8)])
def test_logprobs_alternatives_in_few_threads(dtype, rows, V, parts):
    """Large logits that fall to 40 of the 128 groups of threads which give the bound: it is
    then taken from the others, and more columns lie above it than are listed (1024)."""
    pkg = load_pkg()
    E = 16 // dtype.itemsize     # elements of a 16-byte chunk
    z = torch.randn(rows, V, generator=_gen(V))
    col = torch.arange(V)
    most = []
    for r in range(rows):
        off = r * V % E                              # where the row starts in its first chunk
        chunk = (col + off) // E
        per = -(-((off + V - 1) // E + 1) // parts)
        raised = chunk % per % 128 < 40
        z[r, raised] = 20.0 + torch.rand(int(raised.sum()), generator=_gen(r)) * 10
        most.append(int((raised & (chunk < per)).sum()))
    assert min(most) > 1024
    z = z.to(dtype)              # bf16: about a hundred values, hundreds of ties each
    t = torch.randint(0, V, (rows,), generator=_gen(3))
    _check_logprobs(pkg, z, t, 64, grads=rows < 10)
    _check_logprobs(pkg, z, t, 7, grads=False)


def test_odd_and_wide_rows_in_a_captured_graph():
    """Shared memory beyond 48 KB, clusters of two CTAs and of eight, captured and replayed on
    new inputs: equal to plain calls."""
    pkg = load_pkg()
    cases = []
    for D in (1283, 6101, 8192, 12101, 16384):
        c = _norm_case(200, D, True, FP, BF, BF)
        cases.append({n: c[n].cuda().requires_grad_(n in ("x", "res", "w", "b"))
                      for n in ("x", "res", "w", "b", "dy", "dh")})
    z = torch.randn(4, 50021, generator=_gen(1)).cuda().requires_grad_(True)
    t = torch.randint(0, 50021, (4,), generator=_gen(2)).cuda()

    def step():
        out = []
        for c in cases:
            y, h = pkg.layer_norm(c["x"], c["w"], c["b"], residual=c["res"], out_dtype=BF)
            out += [y.detach(), *torch.autograd.grad([y, h], [c[n] for n in ("x", "res", "w", "b")],
                                                     [c["dy"], c["dh"]])]
        got = pkg.token_logprobs(z, t, entropy=True, top_k=20)
        loss = got.logprobs.sum() + got.entropy.sum() + got.top_logprobs.sum()
        return out + [got.top_ids, loss.detach(), *torch.autograd.grad(loss, [z])]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    with torch.no_grad():
        z.neg_()
        for c in cases:
            c["x"].mul_(-1.5)
    graph.replay()
    want = step()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_logprobs_gradient_from_stats_without_the_sum():
    """Stats whose fourth number is 0: 1 / S is e^(-log S), off by the logarithm's rounding."""
    load_pkg()
    ops = torch.ops.gmdn
    z = torch.randn(5, 300, generator=_gen(1)).cuda()
    t = torch.tensor([0, 299, -100, 7, 8]).cuda()
    stats = ops.token_logprobs_fwd(z, t, True, 0, -100)[4]
    g = torch.randn(5, generator=_gen(2)).cuda()
    want = ops.token_logprobs_bwd(z, t, None, stats, g, g, None, -100)
    stats[:, 3] = 0.0
    got = ops.token_logprobs_bwd(z, t, None, stats, g, g, None, -100)
    # log S ~ 4 rounded to 2^-22 / 2, expf 2 ulp; a gradient's terms are below |g| (1 + |lp| + H)
    assert (got - want).abs().max() <= 16 * EPS * g.abs().max()


def _small_block(pkg):
    g = _gen(9)
    w, w1, w2 = (torch.randn(s, generator=g).cuda().requires_grad_(True)
                 for s in ((64,), (96, 64), (64, 96)))

    def loss(x, t):
        y, h = pkg.rms_norm(x, w, residual=x)
        y = pkg.mlp8(y, w1, w2) + h
        got = pkg.token_logprobs(y, t, entropy=True, top_k=2)
        return got.entropy.mean() - got.logprobs.mean()
    x = torch.randn(7, 64, generator=g).cuda().requires_grad_(True)
    t = torch.randint(0, 64, (7,), generator=g).cuda()
    return loss, x, t, [x, w, w1, w2]


def test_saved_tensors_elsewhere_and_recomputed():
    """Saved tensors moved to the host and back, and a forward run again in the backward."""
    from torch.utils.checkpoint import checkpoint
    loss, x, t, leaves = _small_block(load_pkg())
    want = torch.autograd.grad(loss(x, t), leaves)
    with torch.autograd.graph.save_on_cpu():
        a = loss(x, t)
    for got in (torch.autograd.grad(a, leaves),
                torch.autograd.grad(checkpoint(loss, x, t, use_reentrant=False), leaves)):
        assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_compiled_for_any_number_of_rows():
    torch._dynamo.reset()
    loss, _, _, (_, *weights) = _small_block(load_pkg())
    compiled = torch.compile(loss, dynamic=True)
    for n in (3, 5, 130, 1):
        x = torch.randn(n, 64, generator=_gen(n)).cuda()
        t = torch.randint(0, 64, (n,), generator=_gen(n)).cuda()
        for a, b in zip(torch.autograd.grad(compiled(x, t), weights),
                        torch.autograd.grad(loss(x, t), weights)):
            # the plain parts may add in another order, and move a code by one
            assert (a - b).norm() <= 2e-2 * b.norm() + 1e-12


def test_threads_on_their_own_streams():
    import threading
    loss, x, t, leaves = _small_block(load_pkg())
    want = torch.autograd.grad(loss(x, t), leaves)
    torch.cuda.synchronize()
    wrong = []

    def run(i):
        try:
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                for _ in range(10):
                    got = torch.autograd.grad(loss(x, t), leaves)
                    s.synchronize()
                    if not all(torch.equal(p, q) for p, q in zip(got, want)):
                        wrong.append(i)
        except Exception as e:   # noqa: BLE001 - reported below
            wrong.append(e)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(4)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not wrong
