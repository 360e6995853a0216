"""What the front end's entry points refuse, before anything is launched (no GPU)."""
import ctypes as C

import pytest

from opfoundry_b200 import api

BUF = (C.c_uint8 * 8192)()
BASE = (C.addressof(BUF) + 255) & ~255
NULL, SHAPE, ALIGN, DTYPE = -1, -2, -3, -5


def refused(fn, make, changes, want):
    a = make()
    for k, v in changes.items():
        setattr(a, k, v)
    assert fn(C.byref(a), None) == want, changes


def rotate_args():
    a = api.NormRotateArgs()
    a.q = a.q_out = a.cos_sin = a.positions = BASE
    a.stride_q_row = a.stride_qo_row = 512
    a.stride_q_head = a.stride_qo_head = 128
    a.num_tokens, a.q_heads, a.head_dim, a.rope_dim, a.max_positions, a.eps = 2, 4, 128, 64, 10, 1e-6
    return a


@pytest.mark.parametrize("changes,want", [
    (dict(q=None), NULL), (dict(q_out=None), NULL), (dict(cos_sin=None), NULL), (dict(positions=None), NULL), (dict(k_heads=2), NULL), (dict(out_dtype=2), NULL),
    (dict(q_bias=BASE), NULL),
    (dict(num_tokens=-1), SHAPE), (dict(q_heads=0), SHAPE), (dict(k_heads=-1), SHAPE), (dict(head_dim=0), SHAPE), (dict(head_dim=1032), SHAPE), (dict(head_dim=12), SHAPE),
    (dict(rope_dim=24), SHAPE), (dict(rope_dim=-16), SHAPE), (dict(rope_begin=4), SHAPE), (dict(rope_begin=72), SHAPE), (dict(max_positions=0), SHAPE),
    (dict(eps=-1.0), SHAPE), (dict(eps=float("nan")), SHAPE), (dict(stride_q_head=120), SHAPE), (dict(stride_qo_row=504), SHAPE),
    (dict(in_dtype=2), DTYPE), (dict(out_dtype=1), DTYPE), (dict(head_weight=BASE), DTYPE),
    (dict(q=BASE + 8), ALIGN), (dict(q_out=BASE + 8), ALIGN), (dict(q_weight=BASE + 4), ALIGN), (dict(cos_sin=BASE + 4), ALIGN), (dict(stride_q_head=132, stride_q_row=528), ALIGN),
    (dict(stride_qo_row=516), ALIGN)])
def test_norm_rotate_refuses(built_lib, changes, want):
    refused(built_lib.dsa_v32_norm_rotate, rotate_args, changes, want)


def append_args():
    a = api.AppendArgs()
    a.latent = a.rope = a.index_key = a.kv = a.index_cache = a.cos_sin = a.positions = a.block_table = BASE
    a.stride_latent = a.stride_rope = 576
    a.stride_index_key, a.num_kv_rows, a.num_tokens, a.s_q, a.num_seqs = 128, 640, 3, 1, 3
    a.block_table_stride, a.page_block_size, a.max_positions, a.eps = 4, 64, 100, 1e-6
    return a


@pytest.mark.parametrize("changes,want", [
    (dict(kv=None, index_cache=None), NULL), (dict(latent=None), NULL), (dict(rope=None), NULL), (dict(index_key=None), NULL), (dict(positions=None), NULL),
    (dict(cos_sin=None), NULL), (dict(index_bias=BASE), NULL),
    (dict(num_tokens=-1), SHAPE), (dict(s_q=0), SHAPE), (dict(max_positions=0), SHAPE), (dict(num_kv_rows=0), SHAPE), (dict(num_kv_rows=2 ** 31), SHAPE),
    (dict(page_block_size=0), SHAPE), (dict(page_block_size=48), SHAPE), (dict(page_block_size=8), SHAPE), (dict(block_table_stride=0), SHAPE),
    (dict(block_table=None, kv_batch_stride_rows=-1), SHAPE), (dict(stride_latent=504), SHAPE), (dict(stride_rope=56), SHAPE), (dict(stride_index_key=120), SHAPE),
    (dict(eps=float("inf")), SHAPE), (dict(in_dtype=2), DTYPE), (dict(kv_dtype=2), DTYPE),
    (dict(latent=BASE + 8), ALIGN), (dict(rope=BASE + 2), ALIGN), (dict(kv=BASE + 8), ALIGN), (dict(index_cache=BASE + 8), ALIGN), (dict(stride_latent=580), ALIGN),
    (dict(stride_index_key=132), ALIGN), (dict(latent_weight=BASE + 4), ALIGN), (dict(cos_sin=BASE + 8), ALIGN)])
def test_append_refuses(built_lib, changes, want):
    refused(built_lib.dsa_v32_append_cache, append_args, changes, want)


def scores_args():
    a = api.IndexScoresArgs()
    a.q = a.weights = a.index_cache = a.out = a.block_table = BASE
    a.stride_q_row, a.stride_q_head, a.stride_w_row, a.stride_o_row, a.num_index_rows = 8192, 128, 64, 100, 640
    a.total_q, a.H, a.s_q, a.kv_len, a.block, a.block_table_stride, a.page_block_size, a.cache_dtype = 4, 64, 2, 100, 1, 2, 64, api.KV_FP8
    return a


@pytest.mark.parametrize("changes,want", [
    (dict(q=None), NULL), (dict(weights=None), NULL), (dict(index_cache=None), NULL), (dict(out=None), NULL),
    (dict(total_q=3), SHAPE), (dict(total_q=-2), SHAPE), (dict(s_q=0), SHAPE), (dict(H=0), SHAPE), (dict(H=65), SHAPE), (dict(kv_len=0), SHAPE), (dict(kv_len=2 ** 31 - 10), SHAPE),
    (dict(block=0), SHAPE), (dict(block=48), SHAPE), (dict(block=256), SHAPE), (dict(page_block_size=8), SHAPE), (dict(page_block_size=96), SHAPE), (dict(num_index_rows=0), SHAPE),
    (dict(num_index_rows=650), SHAPE), (dict(num_index_rows=2 ** 31), SHAPE), (dict(block_table_stride=0), SHAPE), (dict(block_table=None, kv_batch_stride_rows=100), SHAPE),
    (dict(stride_q_head=112), SHAPE), (dict(stride_q_row=8000), SHAPE), (dict(stride_w_row=63), SHAPE), (dict(stride_o_row=99), SHAPE), (dict(cache_dtype=2), DTYPE),
    (dict(q=BASE + 8), ALIGN), (dict(index_cache=BASE + 8), ALIGN), (dict(stride_q_head=136, stride_q_row=9000), ALIGN), (dict(weights=BASE + 2), ALIGN), (dict(out=BASE + 1), ALIGN)])
def test_index_scores_refuses(built_lib, changes, want):
    refused(built_lib.dsa_v32_index_scores, scores_args, changes, want)


@pytest.mark.parametrize("args,want", [
    ((None, 10, None, 1, 10, 64, 4, 0, 0, BASE), NULL), ((BASE, 10, None, 1, 10, 64, 4, 0, 0, None), NULL), ((BASE, 9, None, 1, 10, 64, 4, 0, 0, BASE), SHAPE),
    ((BASE, 10, None, -1, 10, 64, 4, 0, 0, BASE), SHAPE), ((BASE, 10, None, 1, 0, 64, 4, 0, 0, BASE), SHAPE), ((BASE, 10, None, 1, 10, 0, 4, 0, 0, BASE), SHAPE),
    ((BASE, 10, None, 1, 10, 64, 0, 0, 0, BASE), SHAPE), ((BASE, 10, None, 1, 10, 64, 4, -1, 0, BASE), SHAPE), ((BASE, 10, None, 1, 10, 64, 4, 3, 2, BASE), SHAPE),
    ((BASE, 10, None, 1, 10, 2 ** 30, 4, 0, 0, BASE), SHAPE)])
def test_block_select_refuses(built_lib, args, want):
    assert built_lib.dsa_v32_block_select(*args, None) == want


def test_nothing_to_do_is_fine(built_lib):
    for fn, make in ((built_lib.dsa_v32_norm_rotate, rotate_args), (built_lib.dsa_v32_append_cache, append_args)):
        a = make()
        a.num_tokens = 0
        assert fn(C.byref(a), None) == 0
    a = scores_args()
    a.total_q = 0
    assert built_lib.dsa_v32_index_scores(C.byref(a), None) == 0
    assert built_lib.dsa_v32_block_select(BASE, 10, None, 0, 10, 64, 4, 0, 0, BASE, None) == 0


def test_null_arguments(built_lib):
    for fn in (built_lib.dsa_v32_norm_rotate, built_lib.dsa_v32_append_cache, built_lib.dsa_v32_index_scores):
        assert fn(None, None) == NULL
