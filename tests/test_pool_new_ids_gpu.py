"""A compaction tells the pages' new ids to whoever keeps page ids elsewhere."""
import pytest
import torch

from ananta_ocr_b200.page_pool import PagePool

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("pages", [1, 7, 200])
@pytest.mark.parametrize("apart", [False, True])
def test_new_ids_follow_the_moves(pages, apart):
    pool, other = PagePool(pages, 8, 64, 16), PagePool(pages, 8, 64, 16)
    rows = torch.arange(8, dtype=torch.int32, device="cuda")
    pool.reserve(rows, 16 * torch.tensor([9, 1, 30, 4, 2, 40, 3, 11], dtype=torch.int32, device="cuda"))
    pool.free(rows[::3].contiguous())
    data = torch.arange(pages, dtype=torch.int32, device="cuda")[:, None]
    old_table, old_ref, old_data = pool.block_table.clone(), pool.ref.clone(), data.clone()
    ids = torch.full((pages,), -9, dtype=torch.int32, device="cuda")
    moved = pool.compact([data], into=other if apart else None, new_ids=ids)
    now = other if apart else pool
    held = old_ref > 0
    assert moved.item() == (ids != torch.arange(pages, device="cuda")).sum().item()
    assert torch.equal(now.block_table, torch.where(old_table < 0, old_table, ids[old_table.clamp(min=0).long()]))
    assert torch.equal(data[ids[held].long()], old_data[held])
    assert ids[held].sort().values.tolist() == list(range(int(held.sum())))
    assert torch.equal(ids[~held], torch.arange(pages, dtype=torch.int32, device="cuda")[~held])


def test_wrong_new_ids_raise():
    pool = PagePool(10, 2, 4, 16)
    data = torch.zeros(10, 1, device="cuda")
    for bad in (torch.zeros(9, dtype=torch.int32, device="cuda"), torch.zeros(10, dtype=torch.int64, device="cuda"),
                torch.zeros(20, dtype=torch.int32, device="cuda")[::2], torch.zeros(10, dtype=torch.int32)):
        with pytest.raises(ValueError, match="new_ids"):
            pool.compact([data], new_ids=bad)
