"""A step without tokens, and calls of the largest number of rows."""
import pytest
import torch

from opfoundry_b200 import api
from front_util import E4M3, rope_table

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fp8", [False, True])
def test_an_empty_step(built_lib, fp8):
    """No tokens through all operators of a step, and nothing is written."""
    i32 = dict(dtype=torch.int32, device="cuda")
    rt, pos, table = rope_table(64, 8).cuda(), torch.empty(0, **i32), torch.zeros(1, 2, **i32)
    index = api.index_cache_pages(2, fp8)
    kv = torch.full((128, 656), 3, dtype=torch.uint8, device="cuda") if fp8 else torch.full((128, 576), 3.0, dtype=torch.bfloat16, device="cuda")
    x = torch.empty(0, 576, dtype=torch.bfloat16, device="cuda")
    q = torch.empty(0, 4, 128, dtype=torch.bfloat16, device="cuda")
    api.append_cache(x[:, :512], x[:, 512:], kv, rt, pos, block_table=table, index_key=q[:, 0], index_cache=index)
    q8, k8, _, _ = api.norm_rotate(q, rt, pos, k=q, out_dtype=E4M3 if fp8 else torch.bfloat16)
    s = api.index_scores(q8, torch.empty(0, 4, device="cuda"), index, pos, 128, block=64, block_table=table)
    idx = api.block_select(s, 2, 64, pos)
    assert q8.shape == k8.shape == (0, 4, 128) and s.shape == (0, 2) and idx.shape == (0, 128)
    assert (kv == 3).all() and (index == 0).all()


def test_an_empty_step_of_single_positions(built_lib):
    q, pos = torch.empty(0, 4, 128, dtype=torch.bfloat16, device="cuda"), torch.empty(0, dtype=torch.int32, device="cuda")
    s = api.index_scores(q, torch.empty(0, 4, device="cuda"), api.index_cache_pages(2, False), pos, 128)
    assert s.shape == (0, 128) and api.topk_select(s, 16, pos).shape == (0, 16)


def test_block_select_of_the_most_rows(built_lib):
    """2^31 - 3 rows: rounded up to eight rows a CTA their number passes 31 bits."""
    rows = 2 ** 31 - 3
    s = torch.zeros(rows, 1, device="cuda")
    out = torch.full((rows, 1), 7, dtype=torch.int32, device="cuda")
    api.block_select(s, 1, 1, out=out)
    assert not out.any()
