"""Arguments of route_topk that the library's 32-bit integers would read as others."""
import pytest
import torch

import jangq_b200 as jq
from jangq_b200 import JangqError

WRAP = 1 << 32


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [dict(groups=WRAP + 8, groups_kept=4), dict(groups=8, groups_kept=WRAP + 4), dict(groups=8, groups_kept=4, group_top=WRAP + 2),
                                dict(groups=8, groups_kept=4, group_top=1 - WRAP), dict(groups=WRAP + 1), dict(groups_kept=1 - WRAP), dict(group_top=1 << 40)])
def test_groups_beyond_32_bits(kw):
    with pytest.raises(JangqError):
        jq.route_topk(torch.zeros((3, 64), device="cuda"), 2, **kw)
