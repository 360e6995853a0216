"""The front end's edges: rows that see nothing, more groups than are dealt out, streams, offsets past 32 bits, calls that the Python side refuses."""
import math

import pytest
import torch

from opfoundry_b200 import api
from front_util import E4M3, check_bf16, check_e4m3, index_scores64, norm_rotate64, rope_table

pytestmark = pytest.mark.gpu


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def problem(B, s_q, H, kv_len, fp8, seed=0, page=64):
    """Inputs of index_scores on the device, the lengths ragged, some zero."""
    g = gen(seed)
    per = -(-kv_len // page)
    if fp8:
        keys = (torch.randn(B * per, page * 128, generator=g) * 100).clamp(-448, 448).to(E4M3).view(torch.uint8)
        index = torch.cat([keys, (torch.rand(B * per, page, generator=g) * 0.01 + 0.005).view(torch.uint8)], 1)
    else:
        index = torch.randn(B * per * page, 128, generator=g).bfloat16()
    q = torch.randn(B * s_q, H, 128, generator=g) * (100 if fp8 else 1)
    q = q.clamp(-448, 448).to(E4M3 if fp8 else torch.bfloat16)
    valid = torch.randint(0, kv_len + 1, (B * s_q,), generator=g).to(torch.int32)
    return dict(q=q.cuda(), weights=torch.randn(B * s_q, H, generator=g).cuda(), index_cache=index.cuda(), valid_len=valid.cuda(),
                block_table=torch.randperm(B * per, generator=g).view(B, per).to(torch.int32).cuda())


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("s_q,block", [(1, 1), (8, 64), (3, 16)])
def test_scores_of_rows_that_see_nothing(built_lib, fp8, s_q, block):
    """No row sees a position: every column is written, with -inf."""
    x = problem(3, s_q, 64, 1000, fp8)
    x["valid_len"].zero_()
    out = torch.full((3 * s_q, -(-1000 // block)), 7.0, device="cuda")
    api.index_scores(kv_len=1000, s_q=s_q, block=block, out=out, **x)
    assert (out == -math.inf).all()
    x["block_table"].fill_(-1)              # nor is there a page
    x["valid_len"].fill_(1000)
    assert (api.index_scores(kv_len=1000, s_q=s_q, block=block, out=out, **x) == -math.inf).all()


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("s_q,H", [(1, 64), (24, 16), (3, 40)])
def test_scores_of_many_sequences_are_those_of_each_half(built_lib, fp8, s_q, H):
    """1100 sequences take items in turn, 550 are dealt out evenly: the same bits, and one sequence against 64 bits."""
    B, kv_len = 1100, 300
    x = problem(B, s_q, H, kv_len, fp8, seed=s_q)
    whole = api.index_scores(kv_len=kv_len, s_q=s_q, **x)
    r = B // 2 * s_q
    for a, b in ((slice(0, r), slice(0, B // 2)), (slice(r, None), slice(B // 2, None))):
        part = api.index_scores(x["q"][a], x["weights"][a], x["index_cache"], x["valid_len"][a], kv_len, s_q=s_q, block_table=x["block_table"][b])
        assert torch.equal(part, whole[a])
    a = slice((B - 1) * s_q, B * s_q)
    want, tol = index_scores64(x["q"][a].cpu(), x["weights"][a].cpu(), x["index_cache"].cpu(), x["valid_len"][a].cpu(), kv_len, s_q, 1, x["block_table"][-1:].cpu(), 64)
    got = whole[a].cpu().double()
    assert torch.equal(got.isinf(), want.isinf()) and ((got - want)[want.isfinite()].abs() <= tol[want.isfinite()]).all()


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("s_q,H", [(2, 64), (3, 64), (4, 64), (3, 40), (7, 32), (13, 16), (8, 64)])
def test_scores_of_several_rows_are_those_of_each(built_lib, fp8, s_q, H):
    """However many rows share a tile and its accumulators: the bits of every row alone, time and again."""
    B, kv_len = 40, 6000
    x = problem(B, s_q, H, kv_len, fp8, seed=H)
    whole = api.index_scores(kv_len=kv_len, s_q=s_q, **x)
    for r in range(s_q):
        alone = api.index_scores(x["q"][r::s_q], x["weights"][r::s_q], x["index_cache"], x["valid_len"][r::s_q].contiguous(), kv_len, block_table=x["block_table"])
        assert torch.equal(alone, whole[r::s_q])
    for _ in range(20):
        assert torch.equal(api.index_scores(kv_len=kv_len, s_q=s_q, **x), whole)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("H,block", [(64, 1), (64, 64), (32, 1), (16, 128), (24, 32)])
def test_scores_of_a_chunk_are_those_of_its_rows(built_lib, fp8, H, block):
    """Full tiles of query rows on every SM, time and again, against one row a tile (the rows as sequences of one shared cache)."""
    T, kv_len = 2048, 8192
    x = problem(1, T, H, kv_len, fp8, seed=H)
    x.pop("block_table")
    alone = api.index_scores(kv_len=kv_len, block=block, **x)
    for _ in range(10):
        assert torch.equal(api.index_scores(kv_len=kv_len, s_q=T, block=block, **x), alone)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
def test_many_tokens_are_those_of_few(built_lib, fp8, dtype, interleaved):
    """5003 tokens in one call, where a warp takes several tokens or heads, give the bits of calls of 100; every seventh is padding."""
    g = gen(9)
    T, H, Hk, P = 5003, 9, 2, 6000
    pages = -(-P // 64)
    rt, pos = rope_table(64, P).cuda(), torch.randperm(P, generator=g)[:T].to(torch.int32)
    pos[::7] = -1
    pos = pos.cuda()
    table = torch.randperm(pages, generator=g)[None].to(torch.int32).cuda()
    x, key, q, k = (torch.randn(T, *s, generator=g).to(dtype).cuda() for s in ((576,), (128,), (H, 128), (Hk, 128)))
    w, iw, ib = (1 + 0.1 * torch.randn(n, generator=g).cuda() for n in (512, 128, 128))
    got = []
    for step in (T, 100):
        kv = torch.full((pages * 64, 656), 7, dtype=torch.uint8, device="cuda") if fp8 else torch.full((pages * 64, 576), 7.0, dtype=torch.bfloat16, device="cuda")
        index = api.index_cache_pages(pages, fp8)
        od = E4M3 if fp8 else torch.bfloat16
        qo, ko = torch.full((T, H, 128), 7.0, device="cuda").to(od), torch.full((T, Hk, 128), 7.0, device="cuda").to(od)
        qs, ks = (torch.full((T, n), 7.0, device="cuda") if fp8 else None for n in (H, Hk))
        for a in range(0, T, step):
            b = slice(a, a + step)
            api.append_cache(x[b, :512], x[b, 512:], kv, rt, pos[b], s_q=T, block_table=table, latent_weight=w, index_key=key[b], index_cache=index, index_weight=iw,
                             index_bias=ib, index_center=True, interleaved=interleaved)
            api.norm_rotate(q[b], rt, pos[b], k=k[b], q_weight=iw, q_bias=ib, k_weight=iw, center=True, interleaved=interleaved, q_out=qo[b], k_out=ko[b],
                            **(dict(q_scale=qs[b], k_scale=ks[b]) if fp8 else {}))
        got.append([kv, index, qo.view(torch.uint8), ko.view(torch.uint8)] + ([qs, ks] if fp8 else []))
    for a, b in zip(*got):
        assert torch.equal(a, b)
    assert (got[0][2].view(E4M3 if fp8 else torch.bfloat16)[::7].float() == 7).all()


def test_calls_on_two_streams_at_once(built_lib):
    """Every operator on two side streams at the same time gives the bits that it gives alone."""
    xs = [problem(4, 2, 64, 20000, True, seed=s) for s in (1, 2)]
    qs = [torch.randn(300, 64, 128, generator=gen(s)).bfloat16().cuda() for s in (1, 2)]
    pos, rt = torch.arange(300, dtype=torch.int32, device="cuda"), rope_table(64, 300).cuda()
    row = [torch.randn(300, 576, generator=gen(s + 5)).bfloat16().cuda() for s in (1, 2)]
    table = torch.arange(5, dtype=torch.int32, device="cuda")[None]

    def all_of(i):
        kv, index = torch.zeros(320, 656, dtype=torch.uint8, device="cuda"), api.index_cache_pages(5, True)
        s = api.index_scores(kv_len=20000, s_q=2, block=64, **xs[i])
        idx = api.block_select(s, 16, 64, xs[i]["valid_len"], first=1, local=1)
        q8, _, scale, _ = api.norm_rotate(qs[i], rt, pos, out_dtype=E4M3)
        api.append_cache(row[i][:, :512], row[i][:, 512:], kv, rt, pos, s_q=300, block_table=table, index_key=qs[i][:, 0], index_cache=index)
        return s, idx, q8.view(torch.uint8), scale, kv, index

    alone = [all_of(i) for i in (0, 1)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in (0, 1)], [[], []]
    for _ in range(5):
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                got[i].append(all_of(i))
    torch.cuda.synchronize()
    for i in (0, 1):
        for r in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(alone[i], r))


def test_caches_of_more_than_32_bits_of_bytes(built_lib):
    """Rows whose byte offsets pass 2^32 in both fp8 caches and in a bf16 index cache."""
    g = gen(4)
    pages, page, T = 540000, 64, 150
    rt, pos = rope_table(64, 512).cuda(), torch.arange(T, dtype=torch.int32, device="cuda")
    table = torch.tensor([[pages - 1, 3, pages - 2]], dtype=torch.int32, device="cuda")
    x, key = torch.randn(T, 576, generator=g).bfloat16().cuda(), torch.randn(T, 128, generator=g).bfloat16().cuda()
    small = torch.tensor([[1, 0, 2]], dtype=torch.int32, device="cuda")
    rows = [(b * page, b * page + page) for b in (pages - 1, 3, pages - 2)]
    for fp8 in (True, False):
        index = torch.empty(pages, page * 132, dtype=torch.uint8, device="cuda") if fp8 else torch.empty(pages * page, 128, dtype=torch.bfloat16, device="cuda")
        near = api.index_cache_pages(3, fp8)
        q = torch.randn(2, 64, 128, generator=g).cuda().to(E4M3 if fp8 else torch.bfloat16)
        w, valid = torch.randn(2, 64, generator=g).cuda(), torch.tensor([T - 1, T], dtype=torch.int32, device="cuda")
        s = []
        for cache, t in ((index, table), (near, small)):
            api.append_cache(None, None, None, rt, pos, s_q=T, block_table=t, index_key=key, index_cache=cache)
            s.append(api.index_scores(q, w, cache, valid, T, s_q=2, block_table=t))
        assert torch.equal(s[0], s[1]) and s[0][:, :T - 1].isfinite().all()
        del index, near
    kv, near = torch.empty(pages * page, 656, dtype=torch.uint8, device="cuda"), torch.zeros(3 * page, 656, dtype=torch.uint8, device="cuda")
    for cache, t in ((kv, table), (near, small)):
        api.append_cache(x[:, :512], x[:, 512:], cache, rt, pos, s_q=T, block_table=t)
    far = torch.cat([kv[a:b] for a, b in rows])[:T]
    assert torch.equal(far, torch.cat([near[64:128], near[:64], near[128:]])[:T])


def test_outputs_of_more_than_32_bits_of_elements(built_lib):
    g = gen(6)
    # scores: 2200 rows over 2^20 columns, of which the cache holds 128
    q, w, cache = torch.randn(2200, 1, 128, generator=g).bfloat16(), torch.rand(2200, 1, generator=g), torch.randn(128, 128, generator=g).bfloat16()
    out = api.index_scores(q.cuda(), w.cuda(), cache.cuda(), None, 1 << 20, s_q=2200, kv_batch_stride_rows=128)
    want = torch.relu(q[-1, 0].double() @ cache.double().T) * w[-1].double()
    tol = (q[-1, 0].double().abs() @ cache.double().abs().T) * w[-1].double() * 200 * 2.0 ** -23
    assert ((out[-1, :128].cpu().double() - want).abs() <= tol).all() and (out[-1, 128:] == -math.inf).all() and (out[0, 128:] == -math.inf).all()
    del out
    # lists: 2^20 + 9 rows of 2048 positions
    rows = (1 << 20) + 9
    s = torch.zeros(rows, 40, device="cuda")
    s[-1] = torch.randn(40, generator=g).cuda()
    idx = api.block_select(s, 32, 64)
    best = s[-1].cpu().topk(32).indices.sort().values
    assert torch.equal(idx[-1].cpu().long(), (best[:, None] * 64 + torch.arange(64)).flatten())
    assert torch.equal(idx[-2], torch.arange(2048, dtype=torch.int32, device="cuda"))
    del idx, s
    # heads: 2^31 and some values
    T, H = 33000, 512
    x = torch.randn(1, H, 128, generator=g).bfloat16()
    big = x.cuda().repeat(T, 1, 1)
    pos = torch.arange(T, dtype=torch.int32, device="cuda") % 100
    out, _, scale, _ = api.norm_rotate(big, rope_table(64, 100).cuda(), pos, out_dtype=E4M3)
    y, m = norm_rotate64(x, table=rope_table(64, 100), pos=pos[-1:].cpu())
    check_e4m3(out[-1:].cpu(), scale[-1:].cpu()[..., None], y, m, 128)
    api.norm_rotate(big, rope_table(64, 100).cuda(), pos, q_out=big)
    check_bf16(big[-1:].cpu(), y, m)


def test_python_side_refuses(built_lib):
    """What the argument blocks cannot show: types, shapes, memory layout, the device."""
    rt, pos = rope_table(64, 8).cuda(), torch.zeros(2, dtype=torch.int32, device="cuda")
    q = torch.zeros(2, 4, 128, dtype=torch.bfloat16, device="cuda")
    refused = (AssertionError, api.DsaError)
    for kw in (dict(q=q.half()), dict(q=q.cpu()), dict(positions=pos.long()), dict(positions=pos[:1]), dict(positions=None), dict(cos_sin=rt.double()), dict(cos_sin=rt.cpu()),
               dict(q=q.transpose(1, 2)), dict(q=q[:, :1].expand(2, 4, 128)), dict(q_out=q.float()), dict(q_out=q[:, :3]), dict(q_weight=torch.ones(64, device="cuda")),
               dict(q_weight=torch.ones(128, device="cuda", dtype=torch.bfloat16)), dict(k=q.float()), dict(k=q[:1]), dict(k_weight=torch.ones(128, device="cuda")),
               dict(head_weight=torch.ones(2, 4, device="cuda")), dict(q=q[..., 4:124])):
        with pytest.raises(refused):
            api.norm_rotate(**(dict(q=q, cos_sin=rt, positions=pos) | kw))
    x, kv, key = torch.zeros(2, 576, dtype=torch.bfloat16, device="cuda"), torch.zeros(128, 576, dtype=torch.bfloat16, device="cuda"), q[:, 0]
    index, table = api.index_cache_pages(2, False), torch.zeros(2, 1, dtype=torch.int32, device="cuda")
    good = dict(latent=x[:, :512], rope=x[:, 512:], kv=kv, cos_sin=rt, positions=pos, block_table=table, index_key=key, index_cache=index)
    for kw in (dict(latent=None), dict(rope=None), dict(latent=x[:, :256]), dict(rope=x[:1, 512:]), dict(latent=x[:, :512].float()), dict(kv=kv.float()), dict(kv=kv[:, :512]), dict(kv=kv.cpu()), dict(index_key=None),
               dict(index_cache=None), dict(index_cache=api.index_cache_pages(2, True)), dict(index_cache=api.index_cache_pages(3, False)), dict(block_table=table.long()),
               dict(block_table=torch.zeros(2, 4, dtype=torch.int32, device="cuda")[:, ::2]), dict(cos_sin=rt[:, :32].contiguous()), dict(seq_ids=pos[:1]), dict(latent_weight=torch.ones(576, device="cuda")), dict(page_block_size=48)):
        with pytest.raises(refused):
            api.append_cache(**(good | kw))
    kv.fill_(3)
    x.fill_(1)
    api.append_cache(**(good | dict(block_table=table.T[:, ::2])))        # a dense table of one sequence: the other's token is not written
    assert (kv[0] != 3).any() and (kv[1:] == 3).all()
    good = dict(q=q, weights=torch.zeros(2, 4, device="cuda"), index_cache=index, valid_len=pos, kv_len=64, block_table=table)
    for kw in (dict(q=q.float()), dict(index_cache=api.index_cache_pages(2, True)), dict(weights=torch.zeros(2, 3, device="cuda")), dict(weights=torch.zeros(2, 4)),
               dict(weights=torch.zeros(1, 4, device="cuda").expand(2, 4)), dict(valid_len=pos[:1]), dict(kv_len=0), dict(block=3), dict(out=torch.zeros(2, 63, device="cuda")),
               dict(block_table=table[:1]), dict(s_q=3), dict(page_block_size=32, index_cache=api.index_cache_pages(2, True))):
        with pytest.raises(refused):
            api.index_scores(**(good | kw))
    s = torch.zeros(2, 10, device="cuda")
    for kw in (dict(scores=s.double()), dict(scores=s.cpu()), dict(scores=s.T), dict(scores=s[:1].expand(2, 10)), dict(valid_len=pos[:1]), dict(num_selected=0), dict(first=3, local=2),
               dict(out=torch.zeros(2, 4, dtype=torch.int32, device="cuda")), dict(out=torch.zeros(2, 256, device="cuda"))):
        with pytest.raises(refused):
            api.block_select(**(dict(scores=s, num_selected=4, block=64) | kw))
    torch.cuda.synchronize()
