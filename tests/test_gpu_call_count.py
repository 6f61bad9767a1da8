"""Every call of an entry point is counted, through ctypes or through the extension module (GPU only)."""
import pytest
import torch

from halo_flash_b200 import HaloError, lib, ops
from tests.test_gpu_attention import BF16, DEV, _i32

pytestmark = pytest.mark.gpu


def test_calls_of_ops_are_counted():
    q, k = torch.zeros(3, 4, 64, dtype=BF16, device=DEV), torch.zeros(3, 2, 64, dtype=BF16, device=DEV)
    kc, vc = (torch.zeros(2, 8, 2, 64, dtype=BF16, device=DEV) for _ in range(2))
    cu, lens, slot = _i32([0, 3]), _i32([3]), torch.arange(3, device=DEV)
    calls = [lambda: ops.paged_plan(_i32([[0]]), _i32([0]), lens, _i32([0, 1]), 8, slot), lambda: ops.paged_store(k, k, kc, vc, slot),
             lambda: ops.attention_packed(q, k, k, cu, torch.empty_like(q)),
             lambda: ops.attention_paged(q, kc, vc, _i32([[0]]), lens, cu, torch.empty_like(q)), lambda: ops.silu_mul(q.float(), q.float())]
    for call in calls:
        before = lib().calls
        call()
        assert lib().calls == before + 1
    before = lib().calls
    with pytest.raises(HaloError):  # a refused call was a call
        ops.attention_packed(q, k, k, cu, torch.empty_like(q), scale=-1.0)
    assert lib().calls == before + 1
