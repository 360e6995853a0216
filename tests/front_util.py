"""The front end's operators in 64 bits (torch, CPU), and the inputs their tests share."""
import math

import torch

E4M3 = torch.float8_e4m3fn


def rope_table(R, n):
    inv = 10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64) / R)
    a = torch.arange(n, dtype=torch.float64)[:, None] * inv
    return torch.cat([a.cos(), a.sin()], 1).float()


def norm_rotate64(x, weight=None, bias=None, center=False, eps=1e-6, table=None, pos=None, begin=0, interleaved=True):
    """x [tokens, heads, D] -> (y, m): y in 64 bits, m the sum of the magnitudes of the terms that y is made of."""
    x = x.double()
    y, m = x, x.abs()
    if weight is not None:
        if center:
            m = m + m.mean(-1, keepdim=True)
            y = y - y.mean(-1, keepdim=True)
        r = 1 / (y.pow(2).mean(-1, keepdim=True) + eps).sqrt()
        y, m = y * r * weight.double(), m * r * weight.double().abs()
        if bias is not None:
            y, m = y + bias.double(), m + bias.double().abs()
    if table is not None:
        R = table.shape[1]
        t = table.double()[pos.long().clamp(0, table.shape[0] - 1)][:, None]
        c, s = t[..., :R // 2], t[..., R // 2:]
        i = torch.arange(R // 2)
        a, b = (begin + 2 * i, begin + 2 * i + 1) if interleaved else (begin + i, begin + i + R // 2)
        y0, m0, y, m = y, m, y.clone(), m.clone()
        y[..., a], y[..., b] = y0[..., a] * c - y0[..., b] * s, y0[..., a] * s + y0[..., b] * c
        m[..., a] = m[..., b] = m0[..., a] + m0[..., b]
    return y, m


# fp32 steps of a value: at most 37 roundings in a sum of squares (32 values a lane, five exchanges), half of them in its root, a
# dozen in mean, norm, affine and rotation: under 64 roundings of 2^-24 of the terms
F32 = 64 * 2.0 ** -24


def check_bf16(got, y, m):
    """Rounded once to bf16: half a step, 2^-8 of the value, over the fp32 steps."""
    bad = (got.double() - y).abs() > 2.0 ** -8 * y.abs() + (1 + 2.0 ** -8) * F32 * m
    assert not bad.any(), ((got.double() - y).abs().max(), bad.sum())


def check_e4m3(codes, scale, y, m, group):
    """codes [..., n] e4m3 and scales [..., n / group] (without factors): the scale to the fp32 steps of the largest term, a value to half a
    step (2^-4 of it, or of the smallest step 2^-9 of the scale) over them."""
    y, m, v = (t.double().unflatten(-1, (-1, group)) for t in (y, m, codes.float()))
    amax, mmax = y.abs().amax(-1), m.amax(-1)
    want = torch.where(amax > 0, amax / 448, torch.ones_like(amax))
    tol = F32 * mmax / 448 + 2.0 ** -22 * want
    assert ((scale.double() - want).abs() <= tol).all(), (scale.double() - want).abs().max()
    s = scale.double()[..., None]
    err = (v * s - y).abs()
    # (1.01: a quotient's own rounding may carry it over a border)
    bad = err > 1.01 * torch.maximum(2.0 ** -4 * y.abs(), 2.0 ** -10 * s) + 2 * F32 * mmax[..., None]
    assert not bad.any(), (err.max(), bad.sum())


def index_keys64(cache, rows, page):
    """Keys [..., 128] in 64 bits and scales [...] of physical rows of an index cache (CPU tensors); rows < 0 give zeros."""
    r = rows.clamp(min=0)
    if cache.dtype == torch.uint8:
        keys = cache[:, :page * 128].contiguous().view(E4M3).view(-1, 128)
        scales = cache[:, page * 128:].contiguous().view(torch.float32).view(-1)
        return keys.view(torch.uint8)[r].view(E4M3).double(), scales[r].double()
    return cache[r].double(), torch.ones(r.shape, dtype=torch.float64)


def physical_rows(seq, pos, num_rows, block_table=None, page=64, stride=0):
    """Physical row of (sequence, position), -1 where there is none."""
    seq, pos = torch.as_tensor(seq).long(), torch.as_tensor(pos).long()
    seq, pos = torch.broadcast_tensors(seq, pos)
    ok = (seq >= 0) & (pos >= 0)
    if block_table is not None:
        ok &= (seq < block_table.shape[0]) & (pos // page < block_table.shape[1])
        p = block_table.long()[seq.clamp(0, block_table.shape[0] - 1), (pos // page).clamp(0, block_table.shape[1] - 1)]
        ok &= p >= 0
        row = p * page + pos % page
    else:
        if stride > 0:
            ok &= pos < stride
        row = seq * stride + pos
    return torch.where(ok & (row < num_rows), row, torch.full_like(row, -1))


def index_scores64(q, weights, cache, valid, kv_len, s_q=1, block=1, block_table=None, page=64, stride=0):
    """(scores, tol) [rows, ceil(kv_len / block)] in 64 bits.  tol: a sum of 128 products, 64 heads and a few factors more, every
    rounding at most 2^-23 of the terms' magnitudes (the tensor cores' own sums keep no less)."""
    n_rows = cache.shape[0] * page if cache.dtype == torch.uint8 else cache.shape[0]
    total_q = q.shape[0]
    cols = -(-kv_len // block)
    out = torch.full((total_q, cols * block), -math.inf, dtype=torch.float64)
    tol = torch.zeros(total_q, cols * block, dtype=torch.float64)
    pos = torch.arange(kv_len)
    for i in range(total_q):
        rows = physical_rows(i // s_q, pos, n_rows, block_table, page, stride)
        k, ks = index_keys64(cache, rows, page)
        d = q[i].double() @ k.T
        w = weights[i].double()[:, None]
        s = (torch.where(d < 0, torch.zeros_like(d), d) * w).sum(0) * ks
        ok = (rows >= 0) & (pos < (kv_len if valid is None else int(valid[i])))
        out[i, :kv_len] = torch.where(ok, s, torch.full_like(s, -math.inf))
        tol[i, :kv_len] = torch.where(ok, ((q[i].double().abs() @ k.abs().T) * w.abs()).sum(0) * ks.abs(), torch.zeros_like(s)) * 200 * 2.0 ** -23
    out, tol = out.unflatten(1, (cols, block)), tol.unflatten(1, (cols, block))
    return out.amax(-1), tol.nan_to_num(0.0).amax(-1)


def block_select_plain(scores, num_selected, block, valid=None, first=0, local=0):
    """The selection by sorting, row by row."""
    rows, blocks = scores.shape
    out = torch.full((rows, num_selected * block), -1, dtype=torch.int32)
    for i in range(rows):
        n = blocks * block if valid is None else min(max(int(valid[i]), 0), blocks * block)
        live = -(-n // block)
        s = [-math.inf if math.isnan(v) else v for v in scores[i, :live].tolist()]
        nan = [math.isnan(v) for v in scores[i, :live].tolist()]
        forced = [b < first or b >= live - local for b in range(live)]
        order = sorted(range(live), key=lambda b: (not forced[b], nan[b] and not forced[b], -s[b], b) if not forced[b] else (False, False, 0.0, b))
        pos = [p for b in sorted(order[:num_selected]) for p in range(b * block, min((b + 1) * block, n))]
        out[i, :len(pos)] = torch.tensor(pos, dtype=torch.int32)
    return out
