"""Refusals at the borders of the front end's argument blocks, before anything is launched (no GPU)."""
import ctypes as C

import pytest
import torch

from opfoundry_b200 import api
from test_front_args import ALIGN, BASE, NULL, SHAPE, append_args, refused, rotate_args, scores_args


@pytest.mark.parametrize("rows", [650, 639, 1])
def test_append_refuses_parts_of_fp8_index_pages(built_lib, rows):
    """A page's scales stand behind its keys: those of a part of a page would lie behind the cache."""
    for changes in (dict(), dict(kv=None)):
        refused(built_lib.dsa_v32_append_cache, append_args, dict(kv_dtype=api.KV_FP8, num_kv_rows=rows) | changes, SHAPE)


@pytest.mark.parametrize("changes", [dict(kv_dtype=api.KV_BF16, num_kv_rows=650), dict(kv_dtype=api.KV_FP8, num_kv_rows=650, index_cache=None),
                                     dict(kv_dtype=api.KV_FP8, num_kv_rows=640)])
def test_append_takes_rows_without_pages_of_scales(built_lib, changes):
    a = append_args()
    for k, v in (changes | dict(num_tokens=0)).items():
        setattr(a, k, v)
    assert built_lib.dsa_v32_append_cache(C.byref(a), None) == 0


def test_block_select_of_no_rows(built_lib):
    """Empty tensors have the address 0; shapes are checked all the same."""
    assert built_lib.dsa_v32_block_select(None, 10, None, 0, 10, 64, 4, 0, 0, None, None) == 0
    assert built_lib.dsa_v32_block_select(None, 10, None, 0, 10, 64, 4, 3, 2, None, None) == SHAPE
    for scores, out in ((None, BASE), (BASE, None)):
        assert built_lib.dsa_v32_block_select(scores, 10, None, 1, 10, 64, 4, 0, 0, out, None) == NULL


def test_topk_select_of_no_rows(built_lib):
    """The lists of single positions, from the same scores."""
    assert built_lib.dsa_v32_topk_select(None, 10, None, 0, 10, 4, None, None) == 0
    assert built_lib.dsa_v32_topk_select(None, 9, None, 0, 10, 4, None, None) == SHAPE
    for scores, out in ((None, BASE), (BASE, None)):
        assert built_lib.dsa_v32_topk_select(scores, 10, None, 1, 10, 4, out, None) == NULL


def test_center_belongs_to_a_norm(built_lib):
    """Without a weight there is no norm whose mean could be subtracted; the values would pass as they are."""
    refused(built_lib.dsa_v32_norm_rotate, rotate_args, dict(center=1), NULL)
    refused(built_lib.dsa_v32_norm_rotate, rotate_args, dict(center=1, k_weight=BASE), NULL)      # there are no keys
    refused(built_lib.dsa_v32_append_cache, append_args, dict(index_center=1), NULL)
    # (strides that are refused later: the call gets past the checks of the norm)
    refused(built_lib.dsa_v32_norm_rotate, rotate_args, dict(center=1, q_weight=BASE, stride_q_head=120), SHAPE)
    refused(built_lib.dsa_v32_norm_rotate, rotate_args, dict(center=1, k_weight=BASE, k_heads=1, k=BASE, k_out=BASE, stride_k_row=128, stride_ko_row=128, stride_q_head=120), SHAPE)
    refused(built_lib.dsa_v32_append_cache, append_args, dict(index_center=1, index_weight=BASE, stride_index_key=120), SHAPE)
    refused(built_lib.dsa_v32_append_cache, append_args, dict(index_center=1, index_cache=None, stride_latent=504), SHAPE)


@pytest.mark.parametrize("kv_len,block", [(0, 1), (-5, 1), (64, 0), (64, -64)])
def test_index_scores_of_no_columns(kv_len, block):
    """Refused before the result's shape is formed from them."""
    q, w, cache = torch.zeros(2, 4, 128, dtype=torch.bfloat16), torch.zeros(2, 4), torch.zeros(128, 128, dtype=torch.bfloat16)
    with pytest.raises(AssertionError):
        api.index_scores(q, w, cache, None, kv_len, block=block)


@pytest.mark.parametrize("num_selected,block", [(0, 64), (-1, 64), (4, 0), (4, -1)])
def test_block_select_of_no_positions(num_selected, block):
    with pytest.raises(AssertionError):
        api.block_select(torch.zeros(2, 10), num_selected, block)


@pytest.mark.parametrize("fn,make,fields", [("norm_rotate", rotate_args, ["q_scale", "k_scale", "head_weight", "positions"]), ("append_cache", append_args, ["positions", "seq_ids", "block_table"]),
                                            ("index_scores", scores_args, ["valid_len", "block_table", "status", "weights", "out"])])
def test_words_off_their_boundary_are_refused(built_lib, fn, make, fields):
    for f in fields:
        for off in (1, 2, 3):
            changes = {f: BASE + off}
            if f in ("q_scale", "k_scale", "head_weight"):
                changes = dict(out_dtype=2, q_scale=BASE, k_heads=1, k=BASE, k_out=BASE, k_scale=BASE, stride_k_row=128, stride_ko_row=128) | changes
            refused(getattr(built_lib, "dsa_v32_" + fn), make, changes, ALIGN)


def test_block_select_refuses_words_off_their_boundary(built_lib):
    for at in (0, 2, 9):
        args = [BASE, 10, BASE, 1, 10, 64, 4, 0, 0, BASE]
        args[at] = BASE + 2
        assert built_lib.dsa_v32_block_select(*args, None) == ALIGN
