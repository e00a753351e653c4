"""After a failed self-test of the 8-bit kernels, their calls are refused (no GPU here: the failure is
set from the host, as the library sets it when it starts)."""
import ctypes as C

import pytest

from tests.test_fp8_refusals import P, desc, moe
from tierlm_amd import lib

EIO = -1
CALLS = {"fp8_pack": lambda: lib.tlm_hip_fp8_pack(P, 128, P, 1, 16, 128, P, None),
         "fp8_quantize": lambda: lib.tlm_hip_fp8_quantize(0, P, 128, 128, 1, P, P, None),
         "fp8_matmul": lambda: lib.tlm_hip_fp8_matmul(P, 16, 128, P, P, 1, 0, P, 16, None),
         "fp8_moe": lambda: moe(desc())}


@pytest.fixture
def failed():
    note = getattr(lib, "_Z15tlmh_set_failedi")           # tlmh_set_failed(int), of the library's own start
    note.argtypes, note.restype = [C.c_int], None
    yield note
    note(0)


@pytest.mark.parametrize("name", CALLS)
def test_a_failed_self_test_refuses_the_call(failed, name):
    import torch
    if torch.cuda.is_available():
        pytest.skip("addresses that a launch would follow")
    failed(1 << 28)
    assert CALLS[name]() == EIO
    msg = lib.tlm_hip_errmsg()
    assert name.encode() in msg and b"self-test" in msg


def test_other_failures_and_empty_calls_do_not(failed):
    import torch
    if torch.cuda.is_available():
        pytest.skip("addresses that a launch would follow")
    failed(1 << 28)
    assert moe(desc(), T=0) == 0 and lib.tlm_hip_fp8_matmul(P, 16, 128, P, P, 0, 0, P, 16, None) == 0
    failed((1 << 14) | (1 << 29) | (1 << 30))
    CALLS["fp8_matmul"]()                                  # no device: another error
    assert b"self-test" not in lib.tlm_hip_errmsg()
