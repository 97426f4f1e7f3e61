"""GPU checks of the paged operators where their documented limits are."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def cp():
    import cuda_primitives

    return cuda_primitives


def test_release_of_the_largest_table_that_names_one_page_everywhere(cp):
    """Almost 2^31 entries name page 0 and the stack is full: their places pass 2^31, and nothing is written."""
    batch, most, pool = 32, (1 << 26) - 1, (1 << 27) - 1
    t = cp.PageTable.allocate(batch, most, pool, 16)
    t.pages.zero_()
    t.held.fill_(most)
    assert int(t.free_count) + batch * most > 1 << 31
    cp.cuda_release_pages_(t, torch.zeros((batch,), dtype=torch.int64).cuda())
    assert int(t.free_count) == pool and (t.held == 0).all()
    assert all((row == -1).all() for row in t.pages)
    assert torch.equal(t.free_pages, torch.arange(pool - 1, -1, -1, dtype=torch.int32, device="cuda"))
