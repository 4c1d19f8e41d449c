"""Page plans of as many requests as the default shared-memory limit holds, and a few more or less."""

import pytest
import torch

from mint_b200.ops import _ext, paged_plan

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [6100, 6135, 6136, 6140, 6143, 6144, 6200])
def test_plan_request_counts_around_the_default_shared_memory_limit(n):
    i32 = {"dtype": torch.int32, "device": "cuda"}
    seq = torch.arange(n, **i32) % 16
    got = paged_plan(seq, torch.ones(n, **i32), torch.arange(n, **i32)[:, None].contiguous(), torch.arange(n, 2 * n, **i32),
                     torch.zeros(1, **i32), page_size=16, n_tokens=n)
    row = torch.arange(n)
    fresh = (row % 16 == 0).long()
    page = torch.where(fresh == 1, n + torch.cumsum(fresh, 0) - 1, row)
    assert got.rows.tolist() == row.tolist() and got.positions.tolist() == (row % 16).tolist()
    assert got.slots.tolist() == (page * 16 + row % 16).tolist() and int(got.free_head) == int(fresh.sum())
    _ext.check_device_status()
