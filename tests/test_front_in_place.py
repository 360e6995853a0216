"""Norm and rotation in place: heads that are read and written by several lanes, through loads that see stores in order."""
import os
import re

import pytest
import torch

from front_util import check_bf16, norm_rotate64, rope_table

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def body(text, start):
    """The braces' contents from the first one behind `start` on."""
    i = text.index("{", text.index(start))
    depth = 0
    for j in range(i, len(text)):
        depth += (text[j] == "{") - (text[j] == "}")
        if depth == 0:
            return text[i:j]
    raise AssertionError("no end of " + start)


@pytest.mark.parametrize("kernel", ["norm_rotate_kernel(", "norm_rotate_long_kernel("])
def test_vectors_that_may_be_written_are_not_read_through_the_read_only_path(kernel):
    """__ldg promises that nobody writes the data while the kernel runs, and its loads may cross barriers.  Every load from x goes by kApart, which is false
    where the output may be the input."""
    with open(os.path.join(ROOT, "opfoundry_b200", "csrc", "norm_rotate.cu")) as f:
        text = f.read()
    b = body(text, kernel)
    assert re.search(r"constexpr bool kApart = kE4m3 \|\| sizeof\(In\) != 2;", b)
    assert not re.search(r"__ldg\([^)]*\bx\b", b)
    loads = re.findall(r"load8(<\w+>)?\(x\b", b) + re.findall(r"Raw<In, kPairs(?:, (\w+))?> raw\b", b)
    assert loads and all(m.strip("<>") == "kApart" for m in loads), loads


@pytest.mark.gpu
@pytest.mark.parametrize("D,R,begin", [(576, 64, 512), (1024, 1024, 0), (1024, 512, 256), (520, 512, 8), (264, 256, 0), (768, 768, 0), (128, 128, 0), (256, 64, 64)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norm", ["none", "rms", "layer"])
def test_in_place(built_lib, D, R, begin, interleaved, norm):
    """q and k inside one buffer of wider rows; what lies between them, and the padding tokens, keep their bytes."""
    from opfoundry_b200 import api
    g = torch.Generator()
    g.manual_seed(D + begin)
    T, H, Hk, P = 301, 6, 2, 400
    table, pos = rope_table(R, P), torch.randperm(P, generator=g)[:T].to(torch.int32)
    pos[::50] = -1
    x = torch.randn(T, H + Hk + 1, D, generator=g).bfloat16()
    w = [1 + 0.2 * torch.randn(D, generator=g) if norm != "none" else None for _ in range(2)]
    b = [0.3 * torch.randn(D, generator=g) if norm == "layer" else None for _ in range(2)]
    cu = lambda t: None if t is None else t.cuda()  # noqa: E731
    args = dict(q_weight=cu(w[0]), k_weight=cu(w[1]), q_bias=cu(b[0]), k_bias=cu(b[1]), center=norm == "layer", rope_begin=begin, interleaved=interleaved)
    for _ in range(5):
        buf = x.cuda()
        q, k = buf[:, :H], buf[:, H + 1:]
        apart = api.norm_rotate(q, table.cuda(), pos.cuda(), k=k, q_out=q.clone(), k_out=k.clone(), **args)
        api.norm_rotate(q, table.cuda(), pos.cuda(), k=k, q_out=q, k_out=k, **args)
        assert torch.equal(q, apart[0]) and torch.equal(k, apart[1])
    got, live = buf.cpu(), pos >= 0
    assert torch.equal(got[:, H], x[:, H]) and torch.equal(got[~live], x[~live])
    for i, (a, e) in enumerate(((0, H), (H + 1, H + 1 + Hk))):
        y, m = norm_rotate64(x[:, a:e], w[i], b[i], norm == "layer", 1e-6, table, pos, begin, interleaved)
        check_bf16(got[live, a:e], y[live], m[live])
