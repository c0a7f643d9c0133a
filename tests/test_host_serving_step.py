"""CPU tests: a step without its new rows is refused."""
import pytest
import torch

import kernelfuser_b200 as kf


@pytest.mark.parametrize("k,v", [(False, True), (True, False), (False, False)])
def test_a_step_needs_both_new_rows(k, v):
    # (one row without the other used to become an attention over whatever the newest row's place holds)
    q, row = torch.zeros(2, 4, 1, 128, dtype=torch.bfloat16), torch.zeros(2, 2, 1, 128, dtype=torch.bfloat16)
    cache = kf.PagedCache.allocate(5, 16, 2, 128, device="cpu")
    pages, lengths = torch.zeros(2, 2, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="Expected K/V"):
        kf.decode_step(q, row if k else None, row if v else None, cache, pages, lengths)
