"""The step operators' own checks, below the Python ones: a refusal is an
exception with its message.  The kernels' entries are reached through the
dispatcher with CPU tensors; every call is refused before it touches a device.
"""
import ctypes

import pytest
import torch

from conftest import load_pkg

NULL = ctypes.c_void_p(None)
FAKE = ctypes.c_void_p(0x1000)   # never dereferenced: the checks fail first
CUDA = torch._C.DispatchKeySet(torch._C.DispatchKey.CUDA)


def _op(name):
    load_pkg()
    return getattr(torch.ops.gmdn, name).default


@pytest.mark.parametrize("name, args, error, message", [
    ("norm_fwd", (torch.zeros(3, 8), None, torch.zeros(7), None, 1e-5, True, True), RuntimeError,
     "expected 8 float32 values"),
    ("norm_fwd", (torch.zeros(3, 8).half(), None, None, None, 1e-5, True, True), TypeError,
     "must be bfloat16 or float32, got Half"),
    ("norm_fwd", (torch.zeros(3, 8), torch.zeros(2, 8), None, None, 1e-5, True, True),
     RuntimeError, "differ in shape"),
    ("norm_fwd", (torch.zeros(3, 8), torch.zeros(3, 8, device="meta"), None, None, 1e-5, True,
                  True), RuntimeError, "tensors on cpu and meta"),
    ("norm_bwd", (torch.zeros(3, 8), torch.zeros(2, 4), None, torch.zeros(3, 8), None, True, False,
                  True, False, False), RuntimeError, "expected 6 float32 values"),
    ("token_logprobs_fwd", (torch.zeros(3, 0), None, True, 0, -100), RuntimeError, "logits must be"),
    ("token_logprobs_bwd", (torch.zeros(3, 9), None, None, torch.zeros(3, 3), None, None, None,
                            -100), RuntimeError, "expected 12 float32 values"),
    ("unpack8", (torch.zeros(300, dtype=torch.int8), torch.zeros(2), True), ValueError,
     "one scale for each 128"),
])
def test_a_refusal_is_an_exception(name, args, error, message):
    with pytest.raises(error, match=message):
        _op(name).redispatch(CUDA, *args)


@pytest.mark.parametrize("width", [64, 768, 1283, 8192, 16384, 40000])
@pytest.mark.parametrize("s_f32", [0, 1])
def test_norm_abi_refuses_a_dh_of_another_type(width, s_f32):
    """The kernels read dh as h is stored: another type would be read past its end."""
    lib = load_pkg()._lib.lib

    def bwd(dh, dh_f32):
        return lib.gmdn_norm_bwd(FAKE, FAKE, FAKE, FAKE, FAKE, dh, FAKE, NULL, NULL, NULL, NULL, 0,
                                 -1 if dh_f32 == s_f32 or not dh.value else 100, width, 1, s_f32, 0,
                                 dh_f32, 0, 0, NULL)

    assert bwd(FAKE, 1 - s_f32) == 1
    assert "type of s" in lib.gmdn_last_error_string().decode()
    assert bwd(FAKE, s_f32) == 1 and bwd(NULL, 1 - s_f32) == 1   # refused for their size alone
    assert "negative size" in lib.gmdn_last_error_string().decode()


@pytest.mark.skipif(torch.cuda.is_available(), reason="the pointers are not a device's")
@pytest.mark.parametrize("width", [64, 768, 2048, 1283, 16384, 12345, 40000])
def test_without_a_device_every_launch_is_an_error(width):
    """Occupancy queries and launches fail and say so; a call after them starts clean."""
    lib = load_pkg()._lib.lib
    for _ in range(2):
        assert lib.gmdn_norm_fwd(FAKE, NULL, FAKE, FAKE, FAKE, NULL, FAKE, FAKE, 10000, width, 1e-5, 1,
                                 0, 0, 0, NULL) == 4
        assert "norm_fwd" in lib.gmdn_last_error_string().decode()
        for dw in (FAKE, NULL):
            need = lib.gmdn_norm_bwd_workspace_bytes(10000, width)
            assert lib.gmdn_norm_bwd(FAKE, FAKE, FAKE, FAKE, FAKE, NULL, FAKE, NULL, dw, NULL, FAKE,
                                     need, 10000, width, 1, 0, 0, 0, 0, 0, NULL) == 4
            assert "norm_bwd" in lib.gmdn_last_error_string().decode()
        assert lib.gmdn_norm_fwd(NULL, NULL, NULL, NULL, NULL, NULL, NULL, NULL, 0, width, 1e-5, 1, 0,
                                 0, 0, NULL) == 0


def test_norm_abi_refuses_a_misaligned_workspace():
    lib = load_pkg()._lib.lib
    need = lib.gmdn_norm_bwd_workspace_bytes(1000, 768)
    for at in (0x1001, 0x1002, 0x1004, 0x1008):
        assert lib.gmdn_norm_bwd(FAKE, FAKE, FAKE, FAKE, FAKE, NULL, FAKE, NULL, FAKE, NULL,
                                 ctypes.c_void_p(at), need, 1000, 768, 1, 0, 0, 0, 0, 0, NULL) == 1
        assert "workspace" in lib.gmdn_last_error_string().decode()
