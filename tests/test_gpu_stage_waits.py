"""No bounded wait ran out in whatever ran before in this process (GPU only; collected after the tests of the kernels that
wait)."""
import ctypes as C

import pytest

from halo_flash_b200 import lib

pytestmark = pytest.mark.gpu


def test_no_wait_ran_out_in_any_test_before():
    n, err = C.c_uint(99), C.create_string_buffer(256)
    assert lib().cdll.halo_b200_stage_timeouts(C.byref(n), err, len(err)) == 0 and n.value == 0
