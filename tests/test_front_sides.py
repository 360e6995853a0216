"""Norm and rotation where queries and keys are treated differently: a norm on one side only.  Heads of up to 128 values share warps, whose lanes may be of
both sides and of units behind the last."""
import pytest
import torch

from opfoundry_b200 import api
from front_util import E4M3, check_bf16, check_e4m3, norm_rotate64, rope_table

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D,R,begin", [(24, 16, 8), (64, 64, 0), (128, 64, 64), (256, 64, 0)])
@pytest.mark.parametrize("T,H,Hk", [(1, 5, 1), (13, 1, 1), (7, 3, 4), (5500, 5, 2)])
@pytest.mark.parametrize("side", ["q", "k"])
@pytest.mark.parametrize("center", [True, False])
@pytest.mark.parametrize("fp8", [False, True])
def test_norm_on_one_side(built_lib, D, R, begin, T, H, Hk, side, center, fp8):
    """The side with a weight is normed, the other one rotated only.  5500 tokens: four heads a unit (7 heads x 8 lanes x 5500 threads fill the device)."""
    g = torch.Generator()
    g.manual_seed(D + T)
    P = 64
    table, pos = rope_table(R, P), torch.randint(0, P, (T,), generator=g).to(torch.int32)
    q, k = (1.0 + torch.randn(T, H, D, generator=g)).bfloat16(), (torch.randn(T, Hk, D, generator=g) - 2.0).bfloat16()
    w, b = 1 + 0.2 * torch.randn(D, generator=g), 0.3 * torch.randn(D, generator=g)
    r = api.norm_rotate(q.cuda(), table.cuda(), pos.cuda(), k=k.cuda(), center=center, rope_begin=begin, interleaved=D == 64, out_dtype=E4M3 if fp8 else torch.bfloat16,
                        **{side + "_weight": w.cuda(), side + "_bias": b.cuda()})
    for i, (n, x) in enumerate((("q", q), ("k", k))):
        y, m = norm_rotate64(x, w if n == side else None, b if n == side else None, center, 1e-6, table, pos, begin, D == 64)
        if fp8:
            check_e4m3(r[i].cpu(), r[2 + i].cpu()[..., None], y, m, D)
        else:
            check_bf16(r[i].cpu(), y, m)


@pytest.mark.parametrize("H,Hk", [(1, 0), (1, 1), (2, 0), (3, 0), (5, 1)])
def test_few_heads_of_many_tokens(built_lib, H, Hk):
    """One head a unit or four, by how many places of four have a head: the bits of a call of few tokens."""
    g = torch.Generator()
    g.manual_seed(H)
    T, P = 30000, 128
    table, pos = rope_table(64, P).cuda(), torch.randint(0, P, (T,), generator=g).to(torch.int32).cuda()
    q, k = torch.randn(T, H, 128, generator=g).bfloat16().cuda(), torch.randn(T, Hk, 128, generator=g).bfloat16().cuda() if Hk else None
    w = (1 + 0.2 * torch.randn(128, generator=g)).cuda()
    at = slice(29950, 30000)
    for fp8 in (False, True):
        args = dict(q_weight=w, k_weight=w if Hk else None, center=True, interleaved=False, out_dtype=E4M3 if fp8 else torch.bfloat16)
        whole = api.norm_rotate(q, table, pos, k=k, **args)
        few = api.norm_rotate(q[at], table, pos[at], k=None if k is None else k[at], **args)
        for a, b in zip(whole, few):
            assert (a is None) == (b is None) and (a is None or torch.equal(a[at].view(torch.uint8), b.view(torch.uint8)))
