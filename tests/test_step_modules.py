"""LanguageModel(fused=, act8=) and modules that are not as it made them: hooks,
replacements and wrappers are called, not read past.  On the CPU, with the
step's operators in their plain forms."""
import copy

import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

from test_training import _training


class Mixer(nn.Module):
    """A stand-in for the mixer, which needs a GPU."""

    def __init__(self, d_model, n_heads, inner, chunk, ns_steps):
        super().__init__()
        self.out = nn.Linear(d_model, d_model, bias=False)

    def set_gate_priors(self):
        pass

    def forward(self, x):
        return self.out(torch.tanh(x))


class Scaled(nn.Module):
    """A wrapper."""

    def __init__(self, inner):
        super().__init__()
        self.inner = inner
        self.weight = getattr(inner, "weight", None)
        self.bias, self.eps = None, 1e-6

    def forward(self, x):
        return 2.0 * self.inner(x)


@pytest.fixture
def tr(monkeypatch):
    tr = _training()
    calls = []

    def rms_norm(x, w, b, eps, residual=None, out_dtype=None):
        calls.append("norm")
        h = x if residual is None else x + residual
        y = F.rms_norm(h, (h.shape[-1],), w, eps)
        return y if residual is None else (y, h)

    def mlp8(x, up, down, gate=None):
        calls.append("mlp8")
        u = F.linear(x, up)
        return F.linear(F.gelu(u) if gate is None else F.silu(F.linear(x, gate)) * u, down)

    monkeypatch.setattr(tr.step_ops, "rms_norm", rms_norm)
    monkeypatch.setattr(tr.step_ops, "mlp8", mlp8)
    tr.calls = calls
    yield tr
    del tr.calls


def _pair(tr, mlp, change):
    """Logits of the plain model and of the one with both options, both changed alike."""
    torch.manual_seed(1)
    a = tr.LanguageModel(50, 16, 2, 2, "delta", mixer_cls=Mixer, mlp=mlp)
    b = tr.LanguageModel(50, 16, 2, 2, "delta", mixer_cls=Mixer, mlp=mlp, fused=True, act8=True)
    b.load_state_dict(a.state_dict())
    change(a)
    change(b)
    idx = torch.arange(24).view(2, 12)
    tr.calls.clear()
    with torch.no_grad():
        return a(idx)[0], b(idx)[0]


def _hook(pick):
    return lambda m: pick(m).register_forward_hook(lambda mod, args, out: out * 1.5)


def _pre_hook(pick):
    return lambda m: pick(m).register_forward_pre_hook(lambda mod, args: (args[0] * 1.5,))


def _set(path, make):
    def change(m):
        *way, last = path.split(".")
        at = m
        for w in way:
            at = at[int(w)] if w.isdigit() else getattr(at, w)
        torch.manual_seed(2)
        if last.isdigit():
            at[int(last)] = make(at[int(last)])
        else:
            setattr(at, last, make(getattr(at, last)))
    return change


def _own_forward(m):
    norm = m.blocks[0].n1
    norm.forward = lambda x: 3.0 * F.rms_norm(x, (x.shape[-1],))


PLAIN = 5 + 2    # norms and MLPs of two blocks that the operators compute
CHANGES = [
    ("gelu", lambda m: None, PLAIN), ("swiglu", lambda m: None, PLAIN),
    ("gelu", _hook(lambda m: m.blocks[0].n1), PLAIN - 1),
    ("gelu", _pre_hook(lambda m: m.blocks[1].n2), PLAIN - 1),
    ("gelu", _hook(lambda m: m.norm_f), PLAIN - 1),
    ("gelu", _hook(lambda m: m.blocks[0].mlp), PLAIN - 1),
    ("gelu", _hook(lambda m: m.blocks[0].mlp[0]), PLAIN - 1),
    ("gelu", _pre_hook(lambda m: m.blocks[0].mlp[1]), PLAIN - 1),
    ("gelu", _hook(lambda m: m.blocks[0].mlp[2]), PLAIN - 1),
    ("swiglu", _hook(lambda m: m.blocks[1].mlp), PLAIN - 1),
    ("swiglu", _pre_hook(lambda m: m.blocks[1].mlp.gate), PLAIN - 1),
    ("swiglu", _hook(lambda m: m.blocks[1].mlp.up), PLAIN - 1),
    # a hooked block runs as a block: its norms are called, its MLP stays on mlp8
    ("gelu", _hook(lambda m: m.blocks[0]), PLAIN - 2), ("gelu", _hook(lambda m: m.blocks[1]),
                                                       PLAIN - 2),
    ("gelu", _set("blocks.0.mlp.1", lambda old: nn.GELU(approximate="tanh")), PLAIN - 1),
    ("gelu", _set("blocks.0.mlp.1", lambda old: nn.ReLU()), PLAIN - 1),
    ("gelu", _set("blocks.0.mlp.0", lambda old: nn.Linear(16, 64)), PLAIN - 1),
    ("gelu", _set("blocks.0.mlp.2", lambda old: nn.Linear(64, 16)), PLAIN - 1),
    ("gelu", _set("blocks.0.mlp.2", Scaled), PLAIN - 1),
    ("gelu", _set("blocks.0.mlp", lambda old: nn.Sequential(*old, nn.Tanh())), PLAIN - 1),
    ("swiglu", _set("blocks.0.mlp.out", lambda old: nn.Linear(64, 16)), PLAIN - 1),
    ("gelu", _set("blocks.0.n1", lambda old: nn.LayerNorm(16)), PLAIN - 1),
    ("gelu", _set("blocks.1.n2", Scaled), PLAIN - 1),
    ("gelu", _set("norm_f", Scaled), PLAIN - 1),
    ("gelu", _set("blocks.1", Scaled), PLAIN - 2),
    ("gelu", _own_forward, PLAIN - 1),
    ("gelu", lambda m: nn.utils.parametrizations.weight_norm(m.blocks[0].mlp[0]), PLAIN - 1),
]


@pytest.mark.parametrize("case", range(len(CHANGES)))
def test_a_changed_module_is_called(tr, case):
    mlp, change, used = CHANGES[case]
    plain, ours = _pair(tr, mlp, change)
    # fp32, the same operations in another order of adds at most
    assert (plain - ours).abs().max() <= 1e-5 * plain.abs().max()
    assert len(tr.calls) == used


def test_a_global_hook_sees_every_module(tr):
    seen = []
    handle = nn.modules.module.register_module_forward_hook(
        lambda mod, args, out: seen.append(type(mod).__name__))
    try:
        plain, ours = _pair(tr, "gelu", lambda m: None)
    finally:
        handle.remove()
    assert len(seen) % 2 == 0 and seen[:len(seen) // 2] == seen[len(seen) // 2:]
    assert torch.equal(plain, ours) and not tr.calls


def test_a_copied_model_stays_on_the_operators(tr):
    a = tr.LanguageModel(50, 16, 2, 2, "delta", mixer_cls=Mixer, fused=True, act8=True)
    with torch.no_grad():
        copy.deepcopy(a)(torch.arange(6).view(1, 6))
    assert len(tr.calls) == PLAIN
