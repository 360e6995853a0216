"""Index scores on either side of the rule that groups query rows, against every row alone."""
import pytest
import torch

from opfoundry_b200 import api
from test_front_edges import problem

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("s_q,H", [(5, 64), (6, 64), (9, 64), (10, 64), (17, 64), (8, 32), (9, 32), (18, 32), (19, 32), (18, 16), (19, 16), (36, 16), (37, 16)])
def test_scores_of_groups_are_those_of_each_row(built_lib, fp8, s_q, H):
    """Groups of 256 columns in equal parts, or of 512 with places that have no row: the bits of every row alone, single positions and blocks."""
    B, kv_len = 9, 3000
    x = problem(B, s_q, H, kv_len, fp8, seed=s_q)
    for block in (1, 32, 128):
        whole = api.index_scores(kv_len=kv_len, s_q=s_q, block=block, **x)
        for r in range(s_q):
            alone = api.index_scores(x["q"][r::s_q], x["weights"][r::s_q], x["index_cache"], x["valid_len"][r::s_q].contiguous(), kv_len, block=block,
                                     block_table=x["block_table"])
            assert torch.equal(alone, whole[r::s_q])
