"""The language model on the step's operators (fused norms and loss, 8-bit MLP
checkpoints) against the same model on torch's."""
import math

import pytest
import torch
import torch.nn.functional as F

from conftest import load_pkg
from test_training import _training

pytestmark = pytest.mark.gpu


def _models(tr, mlp, **options):
    """The plain model and one with the options, same weights, head dim 64."""
    torch.manual_seed(3)
    a = tr.LanguageModel(331, 128, 2, 2, "delta", chunk=64, mlp=mlp).cuda()
    b = tr.LanguageModel(331, 128, 2, 2, "delta", chunk=64, mlp=mlp, **options).cuda()
    b.load_state_dict(a.state_dict())
    g = torch.Generator().manual_seed(4)
    idx = torch.randint(0, 331, (2, 129), generator=g).cuda()
    return a, b, idx[:, :-1], idx[:, 1:]


def _grads(model, idx, targets):
    model.zero_grad()
    _, loss = model(idx, targets)
    loss.backward()
    return loss.item(), {n: p.grad.double() for n, p in model.named_parameters()}


@pytest.mark.parametrize("mlp", ["gelu", "swiglu"])
def test_fused_model_equals_the_plain_one(mlp):
    """fp32: the same function; what differs is the order of fp32 sums."""
    load_pkg()
    tr = _training()
    a, b, idx, targets = _models(tr, mlp, fused=True)
    la, ga = _grads(a, idx, targets)
    lb, gb = _grads(b, idx, targets)
    assert abs(la - lb) <= 1e-5 * abs(la)
    for n in ga:
        assert (ga[n] - gb[n]).norm() <= 1e-4 * ga[n].norm(), n
    with torch.no_grad():
        assert (a(idx)[0] - b(idx)[0]).abs().max() <= 1e-5 * a(idx)[0].abs().max()
    # ignored targets leave the mean, as cross_entropy has it
    targets = targets.clone()
    targets[0, 5:] = -100
    assert abs(a(idx, targets)[1].item() - b(idx, targets)[1].item()) <= 1e-5 * abs(la)


@pytest.mark.parametrize("fused", [False, True])
@pytest.mark.parametrize("mlp", ["gelu", "swiglu"])
def test_act8_model_gradients(mlp, fused):
    """fp32: the forward is the plain one's; a stored value is off by half a step, a / 254 for
    a block's largest a, of uniform error: 1 / (254 sqrt 3) of a, and a is about 3 deviations
    of a block of 128 normal values, so 0.7 % of the value's deviation.  It enters a gradient
    of the MLP once or twice and those before it through the activation's slope."""
    load_pkg()
    tr = _training()
    a, b, idx, targets = _models(tr, mlp, fused=fused, act8=True)
    la, ga = _grads(a, idx, targets)
    lb, gb = _grads(b, idx, targets)
    assert abs(la - lb) <= 1e-5 * abs(la)
    for n in ga:
        assert (ga[n] - gb[n]).norm() <= 3e-2 * ga[n].norm(), n
    moved = [n for n in ga if "mlp" in n and (ga[n] - gb[n]).norm() > 1e-4 * ga[n].norm()]
    assert moved   # the checkpoint is what the gradients read


def test_training_step_runs_with_both(tmp_path):
    """Steps under bf16 autocast run the operators' kernels and keep less memory; the
    checkpoint loads into either model."""
    pkg = load_pkg()
    tr = _training()
    g = torch.Generator().manual_seed(8)
    idx = torch.randint(0, 1000, (8, 513), generator=g).cuda()
    peak = {}
    for on in (False, True):
        torch.manual_seed(7)
        model = tr.LanguageModel(1000, 256, 2, 4, "delta", chunk=64, fused=on, act8=on).cuda()
        opts = tr.build_optimizers(model)
        tr.train_step(model, opts, idx[:, :-1], idx[:, 1:])
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        pkg._lib.prof_report()
        pkg._lib.prof_enable(True)
        loss = tr.train_step(model, opts, idx[:, :-1], idx[:, 1:])
        torch.cuda.synchronize()
        pkg._lib.prof_enable(False)
        names = set(pkg._lib.prof_report())
        ours = {"norm_fwd", "norm_bwd", "token_logprobs_fwd", "token_logprobs_bwd", "pack8",
                "unpack8", "act8_fwd", "act8_bwd"}
        assert names & ours == (ours if on else set())
        assert math.isfinite(loss.item())
        assert all(torch.isfinite(p.grad).all() for p in model.parameters())
        peak[on] = torch.cuda.max_memory_allocated()
    assert peak[True] < peak[False]
    path = str(tmp_path / "ck.pt")
    tr.save_checkpoint(path, model, vocab=1000, d_model=256, n_layers=2, n_heads=4, inner="delta",
                       chunk=64, outer="muon", step=2, seed=7, data_seed=8, args={},
                       final_val_loss=0.0, final_val_ppl=1.0)
    again, _ = tr.load_checkpoint(path, fused=True, act8=True)
    plain, _ = tr.load_checkpoint(path)
    x = idx[:2, :64]
    with torch.no_grad():
        la, lb = again.cuda()(x)[0], plain.cuda()(x)[0]
    assert (la - lb).abs().max() <= 1e-4 * lb.abs().max()


def test_score():
    tr = _training()
    a, b, idx, targets = _models(tr, "gelu", fused=True)
    targets = targets.clone()
    targets[1, :3] = -100
    got = b.score(idx, targets, top_k=4)
    with torch.no_grad():
        lp = F.log_softmax(a(idx)[0].double(), -1)
    want = lp.gather(-1, targets.clamp_min(0)[..., None])[..., 0].masked_fill(targets == -100, 0.0)
    # logits through 2 layers of fp32 products
    assert (got.logprobs.double() - want).abs().max() < 1e-4
    assert (got.entropy.double() + (lp.exp() * lp).sum(-1)).abs().max() < 1e-4
    top = lp.topk(4, -1)
    assert (got.top_logprobs.double() - top.values).abs().max() < 1e-4
    assert not got.logprobs.requires_grad
    assert b.score(idx).logprobs is None
