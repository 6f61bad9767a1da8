"""The plan called from several host threads at once through the C ABI, which holds no lock (GPU only)."""
import threading

import pytest
import torch

from halo_flash_b200 import lib
from tests.test_gpu_attention import DEV, _i32

pytestmark = pytest.mark.gpu


def test_plans_of_different_sizes_from_several_threads():
    """Batches whose prefix sums take 49 to 131 KB of shared memory, planned at once: each call launches what it needs."""
    errors, tokens = [], 64

    def plans(batch):
        try:
            s = torch.cuda.Stream()
            past, fresh, table = (torch.zeros(batch, dtype=torch.int32, device=DEV) for _ in range(3))
            cu, slot = torch.full((batch + 1,), 7, dtype=torch.int32, device=DEV), torch.zeros(tokens, dtype=torch.int64, device=DEV)
            free = _i32([1, 2, 3])
            fresh[:3] = 20
            torch.cuda.synchronize()
            for _ in range(3000):
                lib().call("paged_plan", s.cuda_stream, table.data_ptr(), 1, 1, past.data_ptr(), fresh.data_ptr(), free.data_ptr(), 3, 32,
                           slot.data_ptr(), None, cu.data_ptr(), None, None, batch, tokens)
            s.synchronize()
            want = torch.arange(batch + 1, device=DEV).clamp(max=3) * 20
            assert torch.equal(cu.long(), want) and slot.tolist() == [32 + i for i in range(20)] + [64 + i for i in range(20)] + [96 + i for i in range(20)] + [-1] * 4
        except Exception as e:  # noqa: BLE001 - handed to the test
            errors.append(e)

    threads = [threading.Thread(target=plans, args=(b,)) for b in (6200, 9000, 12000, 16384)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors[0]
