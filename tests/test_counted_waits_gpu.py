"""The wait with a limit of polls, which the kernels of linear attention's prompts use: it ends, says so, and soon."""
import ctypes as C
import time

import pytest
import torch

from h100_gdn_cuda_b200 import _cabi as cabi

pytestmark = pytest.mark.gpu


def status():
    word = C.c_int(-1)
    cabi.check(cabi.load().gdn_device_status(torch.cuda.current_device(), C.byref(word)), "status")
    return word.value


def test_a_limit_of_polls_is_reached():
    """1000 polls of at most 4 us each, beside a wait of one cycle; 8 would say that a wait came back as if its barrier had completed."""
    lib, stream = cabi.load(), torch.cuda.current_stream().cuda_stream
    assert status() == 0
    cabi.check(lib.gdn_selftest_bounded_wait(1, stream), "selftest")
    torch.cuda.synchronize()
    assert status() == 7 and status() == 0
    begin = time.perf_counter()
    for _ in range(10):
        cabi.check(lib.gdn_selftest_bounded_wait(1, stream), "selftest")
    torch.cuda.synchronize()
    assert time.perf_counter() - begin < 1.0  # 10 x 1000 x 4 us, and as much again for a slow host
    assert status() == 7 and status() == 0
