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
