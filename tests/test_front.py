"""The front end (norm and rotation, append, index scores, block selection) against 64 bits, and a run of it before the attention."""
import math

import pytest
import torch

from opfoundry_b200 import api
from front_util import (E4M3, block_select_plain, check_bf16, check_e4m3, index_keys64, index_scores64, norm_rotate64, physical_rows, rope_table)

pytestmark = pytest.mark.gpu


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


# ------------------------------------------------------------------ norm and rotation
@pytest.mark.parametrize("D,R,begin", [(64, 64, 0), (128, 64, 0), (128, 128, 0), (192, 64, 128), (256, 16, 8), (576, 64, 512), (24, 16, 8), (1024, 256, 768), (8, 0, 0), (520, 512, 8)])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("norm,dtype,fp8", [("none", torch.bfloat16, False), ("rms", torch.float32, True), ("layer", torch.bfloat16, True), ("rms", torch.float32, False)])
def test_norm_rotate(built_lib, D, R, begin, interleaved, norm, dtype, fp8):
    g = gen(D + R)
    T, H, Hk, P = 13, 5, 2, 300
    table = rope_table(R, P) if R else None
    pos = torch.randint(0, P, (T,), generator=g).to(torch.int32)
    pos[0], pos[1] = 0, P - 1
    dead = torch.zeros(T, dtype=torch.bool)
    if R:
        pos[2], pos[3] = -1, P        # padding
        dead[2:4] = True
    xs, w, b = [], [None, None], [None, None]
    for i, h in enumerate((H, Hk)):
        x = torch.randn(T, h, D + 8, generator=g).to(dtype)[..., :D]          # rows that are not dense
        if h > 1:
            x[5, 1] = 0
        xs.append(x)
        if norm != "none":
            w[i] = 1 + 0.2 * torch.randn(D, generator=g)
            if norm == "layer":
                b[i] = 0.3 * torch.randn(D, generator=g)
    gate = torch.randn(T, H, generator=g) if fp8 else None
    cu = lambda t: None if t is None else t.cuda()  # noqa: E731
    q, k = (x.cuda() for x in xs)
    od = E4M3 if fp8 else torch.bfloat16
    q_out = torch.full((T, H + 1, D + 16), 7.0, device="cuda").to(od)
    k_out = torch.full((T, Hk, D), 7.0, device="cuda").to(od)
    sc = dict(q_scale=torch.full((T, H), 7.0, device="cuda"), k_scale=torch.full((T, Hk), 7.0, device="cuda")) if fp8 else {}
    r = api.norm_rotate(q, cu(table), pos.cuda(), k=k, q_weight=cu(w[0]), k_weight=cu(w[1]), q_bias=cu(b[0]), k_bias=cu(b[1]), center=norm == "layer",
                        rope_begin=begin, interleaved=interleaved, head_weight=cu(gate), q_out=q_out[:, 1:, 8:8 + D], k_out=k_out, **sc)
    assert (q_out[:, 0].float() == 7).all() and (q_out[..., :8].float() == 7).all() and (q_out[..., 8 + D:].float() == 7).all()
    live = ~dead
    for i, (x, out, scale) in enumerate(zip(xs, (r[0], r[1]), (r[2], r[3]))):
        y, m = norm_rotate64(x, w[i], b[i], norm == "layer", 1e-6, table, pos, begin, interleaved)
        out = out.cpu()
        assert (out[dead].float() == 7).all()
        if fp8:
            scale = scale.cpu()
            assert (scale[dead] == 7).all()
            scale = scale[live].double()
            if i == 0:
                scale = scale / gate[live].double()
            check_e4m3(out[live], scale[..., None], y[live], m[live], D)
        else:
            check_bf16(out[live], y[live], m[live])


@pytest.mark.parametrize("weight", [False, True])
def test_norm_rotate_in_place_and_alone(built_lib, weight):
    """In place (without a norm only the rotated part is touched), one token of one head, no tokens."""
    g = gen(1)
    for T, H, D, R, begin in ((1, 1, 576, 64, 512), (70, 3, 128, 128, 0), (0, 4, 128, 64, 0)):
        x = torch.randn(T, H, D, generator=g).to(torch.bfloat16)
        pos = torch.randint(0, 50, (T,), generator=g).to(torch.int32)
        w = 1 + torch.rand(D, generator=g) if weight else None
        q = x.cuda()
        api.norm_rotate(q, rope_table(R, 50).cuda(), pos.cuda(), q_weight=None if w is None else w.cuda(), rope_begin=begin, interleaved=False, q_out=q)
        y, m = norm_rotate64(x, w, None, False, 1e-6, rope_table(R, 50), pos, begin, False)
        check_bf16(q.cpu(), y, m)
        if not weight:
            assert torch.equal(q.cpu()[..., :begin], x[..., :begin])


def test_norm_rotate_special_values(built_lib):
    """Infinities and NaN stay in their own head; zeros have the scale 1; far positions take the table's row."""
    T, H, D = 4, 4, 128
    x = torch.randn(T, H, D, generator=gen(3)).to(torch.bfloat16)
    x[0, 0, 5], x[1, 1, 70], x[2, 2] = float("nan"), float("inf"), 0
    pos = torch.tensor([0, 1, 65535, 3], dtype=torch.int32)
    table = rope_table(64, 65536)
    out, _, scale, _ = api.norm_rotate(x.cuda(), table.cuda(), pos.cuda(), out_dtype=E4M3)
    out, scale = out.cpu(), scale.cpu()
    bad = torch.zeros(T, H, dtype=torch.bool)
    bad[0, 0] = bad[1, 1] = True
    y, m = norm_rotate64(x, table=table, pos=pos)
    check_e4m3(out[~bad], scale[~bad][:, None], y[~bad], m[~bad], D)
    assert out[0, 0].float().isnan().any() and scale[1, 1].isinf() and scale[2, 2] == 1 and (out[2, 2].float() == 0).all()


# ------------------------------------------------------------------ append
def make_caches(g, pages, page, fp8):
    rows = pages * page
    if fp8:
        return (torch.randint(0, 120, (rows, 656), generator=g).to(torch.uint8), torch.randint(0, 120, (pages, page * 132), generator=g).to(torch.uint8))
    return torch.randn(rows, 576, generator=g).to(torch.bfloat16), torch.randn(rows, 128, generator=g).to(torch.bfloat16)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("page,paged", [(64, True), (16, True), (256, True), (64, False)])
@pytest.mark.parametrize("dtype,norm,pairs", [(torch.bfloat16, True, (True, False)), (torch.float32, False, (False, True))])
def test_append(built_lib, fp8, page, paged, dtype, norm, pairs):
    g = gen(page)
    B, per, pages, T, P = 5, 6, 40, 203, 4096
    table = torch.randperm(pages, generator=g)[:B * per].view(B, per).to(torch.int32) if paged else None
    if paged:
        table[1, 2], table[2, 3] = -1, pages            # a page that is not there, one outside the cache
    stride = 8 * page
    seq = torch.randint(0, B, (T,), generator=g).to(torch.int32)
    pos = torch.zeros(T, dtype=torch.int32)
    for b in range(B):                                   # distinct positions of a sequence, some behind its table or rows
        mine = (seq == b).nonzero()[:, 0]
        pos[mine] = torch.randperm(10 * page, generator=g)[:len(mine)].to(torch.int32)
    pos[0], seq[1], seq[2], pos[3] = -1, -1, B + 3 if paged else 99, P
    latent = torch.randn(T, 576, generator=g).to(dtype)
    key = torch.randn(T, 136, generator=g).to(dtype)[:, 8:]
    latent[7, :128], key[9] = 0, 0
    lw = 1 + 0.2 * torch.randn(512, generator=g) if norm else None
    iw, ib = (1 + 0.2 * torch.randn(128, generator=g), 0.3 * torch.randn(128, generator=g)) if norm else (None, None)
    rt = rope_table(64, P)
    kv, index = make_caches(g, pages, page, fp8)
    dkv, dindex = kv.cuda(), index.cuda()
    dl, dk = latent.cuda(), torch.zeros(T, 136, dtype=dtype, device="cuda")[:, 8:]
    dk.copy_(key)
    cu = lambda t: None if t is None else t.cuda()  # noqa: E731
    api.append_cache(dl[:, :512], dl[:, 512:], dkv, rt.cuda(), pos.cuda(), seq_ids=seq.cuda(), block_table=cu(table), page_block_size=page,
                     kv_batch_stride_rows=stride, latent_weight=cu(lw), index_key=dk, index_cache=dindex, index_weight=cu(iw), index_bias=cu(ib),
                     index_center=norm, interleaved=pairs[0], index_interleaved=pairs[1])
    rows = physical_rows(seq, torch.where(pos < P, pos, -1), pages * page, table, page, stride)
    ok = rows >= 0
    assert 20 < ok.sum() < T and len(set(rows[ok].tolist())) == ok.sum()
    other = torch.ones(pages * page, dtype=torch.bool)
    other[rows[ok]] = False
    gkv, gindex = dkv.cpu(), dindex.cpu()
    y, m = norm_rotate64(latent[:, None, :512], lw)
    ry, rm = norm_rotate64(latent[:, None, 512:], table=rt, pos=pos, interleaved=pairs[0])
    ky, km = norm_rotate64(key[:, None], iw, ib, norm, 1e-6, rt, pos, 0, pairs[1])
    y, m, ry, rm, ky, km = (t[ok][:, 0] for t in (y, m, ry, rm, ky, km))
    assert torch.equal(gkv[other], kv[other])
    got = gkv[rows[ok]]
    if fp8:
        check_e4m3(got[:, :512].contiguous().view(E4M3), got[:, 512:528].contiguous().view(torch.float32), y, m, 128)
        check_bf16(got[:, 528:].contiguous().view(torch.bfloat16), ry, rm)
        keys, scales = gindex[:, :page * 128].reshape(-1, 128), gindex[:, page * 128:].contiguous().view(torch.float32).view(-1)
        check_e4m3(keys[rows[ok]].view(E4M3), scales[rows[ok]][:, None], ky, km, 128)
        assert torch.equal(keys[other], index[:, :page * 128].reshape(-1, 128)[other])
        assert torch.equal(gindex[:, page * 128:].reshape(-1, 4)[other], index[:, page * 128:].reshape(-1, 4)[other])
    else:
        check_bf16(got[:, :512], y, m)
        check_bf16(got[:, 512:], ry, rm)
        check_bf16(gindex[rows[ok]], ky, km)
        assert torch.equal(gindex[other], index[other])


@pytest.mark.parametrize("fp8", [False, True])
def test_append_one_cache_alone(built_lib, fp8):
    """Either cache without the other gives the same bytes; a decode step's tokens go by s_q; no tokens, nothing written."""
    g = gen(8)
    B, s_q, pages = 3, 2, 12
    table = torch.randperm(pages, generator=g)[:B * 4].view(B, 4).to(torch.int32).cuda()
    pos = torch.tensor([0, 1, 63, 64, 200, 201], dtype=torch.int32, device="cuda")
    x, key, rt = torch.randn(6, 576, generator=g).bfloat16().cuda(), torch.randn(6, 128, generator=g).bfloat16().cuda(), rope_table(64, 300).cuda()
    kv, index = (t.cuda() for t in make_caches(g, pages, 64, fp8))
    both, alone = (kv.clone(), index.clone()), (kv.clone(), index.clone())
    args = dict(s_q=s_q, block_table=table)
    api.append_cache(x[:, :512], x[:, 512:], both[0], rt, pos, index_key=key, index_cache=both[1], **args)
    api.append_cache(x[:, :512], x[:, 512:], alone[0], rt, pos, **args)
    api.append_cache(None, None, None, rt, pos, index_key=key, index_cache=alone[1], **args)
    assert torch.equal(both[0], alone[0]) and torch.equal(both[1], alone[1])
    assert not torch.equal(both[0], kv) and not torch.equal(both[1], index)
    if fp8:       # the latents' bytes are those of the packer
        want = api.pack_fp8_rows(x[:, :512].float().contiguous(), x[:, 512:].contiguous())
        rows = physical_rows(torch.arange(6) // s_q, pos.cpu(), pages * 64, table.cpu())
        assert torch.equal(both[0][rows.cuda()][:, :528], want[:, :528])
    api.append_cache(x[:0, :512], x[:0, 512:], both[0], rt, pos[:0], **args)
    assert torch.equal(both[0], alone[0])


# ------------------------------------------------------------------ index scores
def make_index(g, pages, page, fp8):
    if not fp8:
        return torch.randn(pages * page, 128, generator=g).to(torch.bfloat16)
    keys = (torch.randn(pages, page * 128, generator=g) * 100).to(E4M3).view(torch.uint8)
    return torch.cat([keys, (torch.rand(pages, page, generator=g) * 0.01 + 0.005).view(torch.uint8)], 1)


def run_scores(g, *, B, s_q, H, kv_len, fp8, block, page=64, paged=True, valid=None, weights=None, spread=False):
    per = -(-kv_len // page)
    pages = B * per + 1
    index = make_index(g, pages, page, fp8)
    table = torch.randperm(pages, generator=g)[:B * per].view(B, per).to(torch.int32) if paged else None
    rows = B * s_q
    q = (torch.randn(rows, H, 128, generator=g) * (100 if fp8 else 1)).to(E4M3 if fp8 else torch.bfloat16)
    if weights is None:
        weights = torch.randn(rows, H, generator=g)
    cols = -(-kv_len // block)
    dq, dw, buf = q.cuda(), weights.cuda(), torch.full((rows, cols + 3), 7.0, device="cuda")
    if spread:        # rows and heads apart
        wide = torch.zeros(rows, H + 1, 144, dtype=torch.uint8 if fp8 else torch.bfloat16, device="cuda")
        wide = wide.view(E4M3) if fp8 else wide
        wide[:, :H, :128] = dq
        dq = wide[:, :H, :128]
        wbuf = torch.zeros(rows, H + 5, device="cuda")
        wbuf[:, :H] = dw
        dw = wbuf[:, :H]
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    api.index_scores(dq, dw, index.cuda(), None if valid is None else valid.cuda(), kv_len, s_q=s_q, block=block, block_table=None if table is None else table.cuda(),
                     page_block_size=page, kv_batch_stride_rows=per * page, out=buf[:, :cols], status=status)
    got = buf.cpu()
    assert int(status) == 0 and (got[:, cols:] == 7).all()
    want, tol = index_scores64(q, weights, index, valid, kv_len, s_q, block, table, page, per * page)
    return got[:, :cols].double(), want, tol, (dq, dw, index, table)


def check_scores(got, want, tol):
    assert torch.equal(got.isinf(), want.isinf()) and torch.equal(got.isnan(), want.isnan())
    fine = want.isfinite()
    bad = (got - want)[fine].abs() > tol[fine]
    assert not bad.any(), ((got - want)[fine].abs() / tol[fine].clamp(min=1e-30)).max()
    assert torch.equal(got[want.isinf()], want[want.isinf()])


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("B,s_q,H,kv_len,block", [(1, 1, 64, 1, 1), (3, 1, 64, 1000, 1), (2, 2, 64, 640, 1), (2, 3, 32, 129, 1), (1, 130, 64, 777, 1), (2, 9, 40, 513, 16),
                                                  (1, 41, 16, 700, 64), (2, 5, 1, 300, 128), (3, 17, 8, 260, 2), (1, 8, 64, 4096, 32), (5, 4, 33, 127, 64)])
def test_index_scores(built_lib, fp8, B, s_q, H, kv_len, block):
    g = gen(kv_len + H)
    valid = torch.randint(0, kv_len + 1, (B * s_q,), generator=g).to(torch.int32)
    valid[0] = kv_len
    if B * s_q > 2:
        valid[1], valid[2] = 0, 1
    check_scores(*run_scores(g, B=B, s_q=s_q, H=H, kv_len=kv_len, fp8=fp8, block=block, valid=valid, spread=block % 3 == 1)[:3])


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("page,paged", [(16, True), (32, True), (128, True), (512, True), (64, False), (256, False)])
def test_index_scores_pages(built_lib, fp8, page, paged):
    g = gen(page)
    check_scores(*run_scores(g, B=3, s_q=2, H=64, kv_len=1100, fp8=fp8, block=1, page=page, paged=paged)[:3])
    check_scores(*run_scores(g, B=2, s_q=20, H=32, kv_len=900, fp8=fp8, block=64, page=page, paged=paged, valid=torch.arange(861, 901).to(torch.int32))[:3])


@pytest.mark.parametrize("fp8", [False, True])
def test_index_scores_missing_pages_and_special_values(built_lib, fp8):
    """Pages that are negative or outside the cache count as no positions; NaN and infinite keys stay in their own position, and in
    places that no row sees they reach nothing."""
    g = gen(5)
    kv_len, page = 700, 64
    index = make_index(g, 16, page, fp8)
    table = torch.randperm(11, generator=g)[None].to(torch.int32)
    table[0, 3], table[0, 5], table[0, 7] = -1, 16, 2 ** 30
    rows = physical_rows(0, torch.arange(kv_len), 16 * 64, table, page)
    for p, v in ((10, float("nan")), (130, float("inf")), (650, float("nan"))):
        r = int(rows[p])
        if fp8:
            index[r // page, page * 128 + 4 * (r % page):page * 128 + 4 * (r % page) + 4] = torch.tensor([v]).view(torch.uint8)
            if v != v:
                index[r // page, (r % page) * 128 + 3] = 0x7F
        else:
            index[r] = torch.rand(128, generator=g).bfloat16()
            index[r, 17] = v
    q = torch.randn(2, 64, 128, generator=g).abs()
    q = (q * 100).to(E4M3) if fp8 else q.bfloat16()
    w = torch.rand(2, 64, generator=g)
    valid = torch.tensor([640, 200], dtype=torch.int32)
    for block in (1, 32):
        got = api.index_scores(q.cuda(), w.cuda(), index.cuda(), valid.cuda(), kv_len, s_q=2, block=block, block_table=table.cuda()).cpu().double()
        want, tol = index_scores64(q, w, index, valid, kv_len, 2, block, table, page)
        check_scores(got, want, tol)
        if block == 1:
            assert got[0, 10].isnan() and not got[0, 130].isfinite() and (got[:, 192:256] == -math.inf).all() and (got[:, 640:] == -math.inf).all()


# ------------------------------------------------------------------ block selection
@pytest.mark.parametrize("rows,blocks,n,block,first,local", [(1, 1, 1, 64, 0, 0), (9, 100, 7, 64, 1, 2), (70, 513, 32, 64, 0, 0), (5, 2048, 32, 64, 1, 1), (3, 300, 300, 16, 0, 0),
                                                             (4, 33, 40, 64, 2, 2), (6, 5000, 100, 16, 0, 3), (3, 40001, 500, 4, 3, 0), (12, 257, 16, 128, 8, 8), (2, 64, 2048, 1, 0, 0),
                                                             (40, 1000, 512, 1, 0, 0), (7, 97, 5, 7, 1, 1)])
def test_block_select(built_lib, rows, blocks, n, block, first, local):
    g = gen(blocks + n)
    buf = torch.randn(rows, blocks + 5, generator=g)
    s = buf[:, :blocks]
    s[0] = torch.round(s[0] * 2) / 2
    if rows > 4:
        s[1] = 0
        s[2, ::7], s[2, ::5] = float("nan"), float("inf")
        s[3, ::2], s[3, 1::4], s[4] = -math.inf, float("nan"), float("nan")
    valid = torch.randint(0, blocks * block + 1, (rows,), generator=g).to(torch.int32)
    valid[0] = blocks * block
    if rows > 6:
        valid[5], valid[6] = 0, 1
        valid[2:5] = blocks * block - 1
    elif rows > 2:
        valid[1], valid[2] = -5, 2 ** 31 - 1
    want = block_select_plain(s, n, block, valid, first, local)
    dev = buf.cuda()[:, :blocks]
    assert torch.equal(api.block_select(dev, n, block, valid.cuda(), first=first, local=local).cpu(), want)
    assert torch.equal(api.block_select(dev, n, block, first=first, local=local).cpu(), block_select_plain(s, n, block, None, first, local))


def test_block_select_of_single_positions_is_topk_select(built_lib):
    s = torch.randn(20, 3001, generator=gen(2)).cuda()
    valid = torch.randint(0, 3002, (20,), generator=gen(3)).to(torch.int32).cuda()
    assert torch.equal(api.block_select(s, 128, 1, valid), api.topk_select(s, 128, valid))


# ------------------------------------------------------------------ together
@pytest.mark.parametrize("fp8", [True, False])
@pytest.mark.parametrize("block", [1, 64])
def test_decode_steps_from_projections_to_output(built_lib, oracle, fp8, block):
    """A prompt is appended, then decode steps: queries and caches, scores, lists, attention; the lists against the scores that the kernel
    gave, the scores against 64 bits on the caches that it wrote, the attention against the oracle on its lists; one step also as a replayed graph."""
    import numpy as np
    from helpers import TOL_BF16, TOL_FP8, check_lse, check_out
    g = gen(21)
    B, H, Hi, page, per, topk = 3, 16, 32, 64, 6, 128
    pages = B * per
    table = torch.randperm(pages, generator=g).view(B, per).to(torch.int32).cuda()
    rt = rope_table(64, 1024).cuda()
    kv = torch.zeros(pages * page, 656, dtype=torch.uint8, device="cuda") if fp8 else torch.zeros(pages * page, 576, dtype=torch.bfloat16, device="cuda")
    index = api.index_cache_pages(pages, fp8, page)
    lens = [300, 127, 64]
    lw, iw, ib = (1 + 0.1 * torch.randn(512, generator=g)).cuda(), (1 + 0.1 * torch.randn(128, generator=g)).cuda(), (0.1 * torch.randn(128, generator=g)).cuda()
    rnd = lambda *s: torch.randn(*s, generator=g).to(torch.bfloat16).cuda()  # noqa: E731
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    opt = dict(block_table=table, latent_weight=lw, index_cache=index, index_weight=iw, index_bias=ib, index_center=True, index_interleaved=False)
    x = rnd(sum(lens), 576)
    api.append_cache(x[:, :512], x[:, 512:], kv, rt, ints([p for n in lens for p in range(n)]), seq_ids=ints([b for b, n in enumerate(lens) for _ in range(n)]),
                     index_key=rnd(sum(lens), 128), **opt)
    plan = api.mla_decode_plan_create(B, H, topk)
    pos, valid = ints(lens), ints([n + 1 for n in lens])
    x, key, qi, gate, q_pe, q = rnd(B, 576), rnd(B, 128), rnd(B, Hi, 128), torch.randn(B, Hi, generator=g).cuda(), rnd(B, H, 64), rnd(B, H, 576)
    out, lse = torch.empty(B, H, 512, dtype=torch.bfloat16, device="cuda"), torch.empty(B, H, device="cuda")
    scores, idx = torch.empty(B, -(-per * page // block), device="cuda"), torch.empty(B, topk, dtype=torch.int32, device="cuda")
    q8 = torch.empty(B, Hi, 128, dtype=E4M3 if fp8 else torch.bfloat16, device="cuda")
    w8 = torch.empty(B, Hi, device="cuda") if fp8 else gate
    scale = 1.0 / math.sqrt(192.0)

    def step():
        api.append_cache(x[:, :512], x[:, 512:], kv, rt, pos, index_key=key, **opt)
        api.norm_rotate(q_pe, rt, pos, q_out=q[..., 512:])
        api.norm_rotate(qi, rt, pos, interleaved=False, q_out=q8, **(dict(head_weight=gate, q_scale=w8) if fp8 else {}))
        api.index_scores(q8, w8, index, valid, per * page, block=block, block_table=table, out=scores)
        api.block_select(scores, topk // block, block, valid, local=1, out=idx)
        api.mla_decode_launch_pipeline(q, kv, idx, plan, scale, block_table=table, page_block_size=page, out=out, lse=lse, check=False)

    def check():
        torch.cuda.synchronize()
        v = valid.cpu()
        want, tol = index_scores64(q8.cpu(), w8.cpu(), index.cpu(), v, per * page, 1, block, table.cpu(), page)
        check_scores(scores.cpu().double(), want, tol)
        assert torch.equal(idx.cpu(), block_select_plain(scores.cpu(), topk // block, block, v, 0, 1))
        bits = lambda t: t.view(torch.int16).cpu().numpy().view(np.uint16)  # noqa: E731
        r_out, r_lse = oracle.sparse_mla(bits(q), kv.cpu().numpy() if fp8 else bits(kv), idx.cpu().numpy(), scale, kv_is_fp8=fp8,
                                         block_table=table.cpu().numpy(), page_block_size=page)
        check_out(bits(out), r_out, **(TOL_FP8 if fp8 else TOL_BF16))
        check_lse(lse.cpu().numpy(), r_lse)

    step()
    check()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step()
    for _ in range(3):       # the next tokens
        pos += 1
        valid += 1
        x.copy_(rnd(B, 576))
        key.copy_(rnd(B, 128))
        qi.copy_(rnd(B, Hi, 128))
        out.fill_(float("nan"))
        graph.replay()
        check()
