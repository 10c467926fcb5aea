"""libgmdn_torch.so: built against one torch, needed by the step operators alone."""
import importlib.util
import os
import shutil
import subprocess
import sys

import pytest
import torch

from conftest import PKG_NAME, ROOT, load_pkg

PKG = os.path.join(ROOT, PKG_NAME)

PROBE = f"""
import importlib, torch
pkg = importlib.import_module("{PKG_NAME}")
assert pkg.state_scan and pkg.chunk_fast_weight and torch.ops.gmdn is not None
from importlib import import_module
step = import_module("{PKG_NAME}.step_ops")
step._same_device = step._require_cuda = lambda *a: None      # past the refusal of CPU tensors
x = torch.zeros(4, 16)
for call in (lambda: pkg.layer_norm(x), lambda: pkg.token_logprobs(x, None, entropy=True),
             lambda: pkg.pack8(x), lambda: pkg.act8_forward(x),
             lambda: pkg.mlp8(x, torch.zeros(8, 16), torch.zeros(4, 8))):
    try:
        call()
    except ImportError as e:
        print("refused:", e)
"""


def _copy(tmp_path):
    """The package without its op library; the C library is linked in."""
    to = tmp_path / PKG_NAME
    to.mkdir()
    for f in os.listdir(PKG):
        if f.endswith(".py"):
            shutil.copy(os.path.join(PKG, f), to / f)
    os.symlink(load_pkg()._lib.LIB_PATH, to / "libgmdn_b200.so")
    return to


def _run(tmp_path):
    env = {**os.environ, "PYTHONPATH": str(tmp_path)}
    res = subprocess.run([sys.executable, "-c", PROBE], cwd=tmp_path, env=env, capture_output=True,
                         text=True)
    assert res.returncode == 0, res.stderr
    return [line for line in res.stdout.splitlines() if line.startswith("refused:")]


def test_the_package_imports_without_the_op_library(tmp_path):
    _copy(tmp_path)
    said = _run(tmp_path)
    assert len(said) == 5 and all("libgmdn_torch.so is missing" in s for s in said)


def test_the_package_imports_with_an_op_library_that_does_not_load(tmp_path):
    (_copy(tmp_path) / "libgmdn_torch.so").write_bytes(b"not a library")
    said = _run(tmp_path)
    assert len(said) == 5 and all("does not load" in s for s in said)


def test_an_op_library_of_another_torch_is_not_loaded(tmp_path):
    to = _copy(tmp_path)
    (to / "libgmdn_torch.so").write_bytes(b"not even opened")
    (to / "_build").mkdir()
    (to / "_build" / "libgmdn_torch.torch_version").write_text("1.0.0")
    said = _run(tmp_path)
    assert len(said) == 5 and all("built against torch 1.0.0" in s for s in said)


@pytest.fixture
def build():
    spec = importlib.util.spec_from_file_location("gmdn_build", os.path.join(PKG, "build.py"))
    b = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(b)
    return b


def test_the_op_library_is_stale_for_another_torch(build, tmp_path, monkeypatch):
    assert build._torch_version(build._torch_dir()) == torch.__version__
    lib, stamp = tmp_path / "lib.so", tmp_path / "version"
    lib.write_bytes(b"")
    monkeypatch.setattr(build, "TORCH_LIB", str(lib))
    monkeypatch.setattr(build, "TORCH_STAMP", str(stamp))
    assert build._torch_stale("2.0")              # nothing says what it was built against
    stamp.write_text("2.0")
    assert not build._torch_stale("2.0") and build._torch_stale("2.1")
    os.utime(lib, (1, 1))
    assert build._torch_stale("2.0")


def test_without_torch_the_c_library_alone_is_built(build, monkeypatch, capsys):
    monkeypatch.setattr(build.importlib.util, "find_spec", lambda name: None)
    assert build.build_torch() is None
    assert "torch not found" in capsys.readouterr().err
