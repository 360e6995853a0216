"""The front end of the sparse attention: norms of queries and keys with the position rotation, the append to the paged
caches, the index scores of blocks of positions, and the selection of blocks as lists of positions.

A case is a dict of plain values.  `listed()` are the ones that are followed; `draw()` gives others of the same ranges.
Each operator stands here in its plain form, elementary torch operations in 32 bits, and, where `own` is true, as the
call of the library that a program makes.
"""
import math

import torch

own = False

PAGE = 64                    # positions of a page of the caches
D_INDEX = 128                # values of an index key
D_LATENT, D_ROPE = 512, 64   # values of a cache row of the attention
EPS = 1e-6
E4M3 = torch.float8_e4m3fn


# ------------------------------------------------------------------ the cases
def rotate(T, H, D, *, Hk=0, R=64, begin=0, pairs=True, norm="none", fp8=False, gate=False, wide=0, fp32=False):
    """wide > D: the heads are the last D values of rows of `wide` values in the buffer that is written."""
    return dict(kind="rotate", T=T, H=H, D=D, Hk=Hk, R=R, begin=begin, pairs=pairs, norm=norm, fp8=fp8, gate=gate, wide=wide, fp32=fp32)


def append(B, T, *, fp8=True, index=True, norm=True, fp32=False):
    """T new tokens of B sequences: as many each where B divides T, else ragged."""
    return dict(kind="append", B=B, T=T, fp8=fp8, index=index, norm=norm, fp32=fp32)


def scores(B, kv_len, *, s_q=1, H=64, fp8=True, block=1, even=False):
    """even: all sequences have kv_len positions; otherwise theirs lie between a half of it and all."""
    return dict(kind="scores", B=B, kv_len=kv_len, s_q=s_q, H=H, fp8=fp8, block=block, even=even)


def select(rows, kv_len, *, block=64, blocks=32, causal=False):
    return dict(kind="select", rows=rows, kv_len=kv_len, block=block, blocks=blocks, causal=causal)


def listed():
    return [
        # the index queries of a decode step of four sequences: rotated, quantised, the scales folded into the heads' weights
        dict(rotate(4, 64, D_INDEX, fp8=True, gate=True), name="rotate_index_decode"),
        # norms and rotation of queries and keys of a prompt's odd-sized chunk, halves rotated against each other
        dict(rotate(4091, 64, D_INDEX, Hk=8, R=128, pairs=False, norm="rms"), name="rotate_qk_norm_prefill"),
        # the rotary part of the attention's queries, from the projection's output to its place in rows of 576 values
        dict(rotate(2048, 128, D_ROPE, wide=576), name="rotate_mla_q_prefill"),
        # one token of one sequence into the bf16 caches
        dict(append(1, 1, fp8=False), name="append_bf16_b1"),
        # a decode step of 64 sequences into the fp8 caches
        dict(append(64, 64), name="append_fp8_b64"),
        # a packed prefill batch of seven prompts into the fp8 caches
        dict(append(7, 16380), name="append_fp8_prefill"),
        # the scores of one user's decode step
        dict(scores(1, 32768, even=True), name="scores_fp8_b1"),
        # a decode batch of ragged lengths, with one speculative token
        dict(scores(64, 32768, s_q=2), name="scores_fp8_b64_mtp"),
        # the last chunk of a prompt, a score for every position: the largest case
        dict(scores(1, 16384, s_q=4096), name="scores_fp8_prefill"),
        # an odd-sized chunk on a bf16 cache, 32 heads, the best of each page
        dict(scores(1, 7001, s_q=1500, H=32, fp8=False, block=64), name="scores_bf16_blocks"),
        # the lists of a decode batch over long contexts
        dict(select(64, 131072), name="select_decode"),
        # the lists of a prefill chunk
        dict(select(4096, 16384, causal=True), name="select_prefill"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case: the kinds of work above with sizes over their whole range."""
    kind = rng.choice(["rotate", "append", "scores", "scores", "select"])
    if kind == "rotate":
        what = rng.choice(["index", "norm", "mla"])
        T = _log_int(rng, 1, 4096)
        if what == "index":
            return rotate(T, rng.choice([64, 64, 32, 16]), D_INDEX, fp8=True, gate=rng.random() < 0.7, fp32=rng.random() < 0.3)
        if what == "mla":
            return rotate(T, rng.choice([128, 64, 16]), D_ROPE, pairs=rng.random() < 0.7, wide=576)
        D = rng.choice([64, 128, 128, 192, 256])
        return rotate(T, rng.choice([8, 16, 32, 40, 64]), D, Hk=rng.choice([1, 2, 8]), R=rng.choice([64, D]) if D <= 128 else 64,
                      begin=rng.choice([0, D - 64]) if D > 128 else 0, pairs=rng.random() < 0.5, norm=rng.choice(["rms", "layer"]), fp32=rng.random() < 0.3)
    if kind == "append":
        B = _log_int(rng, 1, 128)
        return append(B, B if rng.random() < 0.4 else max(B, _log_int(rng, 1, 16384)), fp8=rng.random() < 0.6, index=rng.random() < 0.8,
                      norm=rng.random() < 0.7, fp32=rng.random() < 0.3)
    if kind == "select":
        block = rng.choice([16, 32, 64, 64, 128])
        causal = rng.random() < 0.5
        return select(_log_int(rng, 64, 4096) if causal else _log_int(rng, 1, 160), _log_int(rng, 2000, 16384) if causal else _log_int(rng, 2000, 131072),
                      block=block, blocks=max(4, rng.choice([2048, 2048, 1024]) // block), causal=causal)
    fp8, H = rng.random() < 0.6, rng.choice([64, 64, 32, 16])
    block = rng.choice([1, 1, 64, 64, 32, 16, 128])
    if rng.random() < 0.5:      # decode
        B = _log_int(rng, 1, 96)
        return scores(B, _log_int(rng, 1000, 131072 if B < 16 else 40000), s_q=rng.choice([1, 1, 2, 3]), H=H, fp8=fp8, block=block, even=rng.random() < 0.3)
    T = _log_int(rng, 20, 3000)
    return scores(1, T + _log_int(rng, 1, 12000), s_q=T, H=H, fp8=fp8, block=block)


# ------------------------------------------------------------------ what a program has in hand before the call
def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = {"rotate": _prepare_rotate, "append": _prepare_append, "scores": _prepare_scores, "select": _prepare_select}[case["kind"]](case, g, seed)
    s["case"] = case
    return s


def _randn(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def _rope_table(R, max_positions):
    """fp32 [positions, R]: R / 2 cosines, then R / 2 sines; the angles are formed in 64 bits."""
    inv = 10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64, device="cuda") / R)
    a = torch.arange(max_positions, dtype=torch.float64, device="cuda")[:, None] * inv
    return torch.cat([a.cos(), a.sin()], dim=1).float()


MAX_POS = 32768


def _prepare_rotate(c, g, seed):
    T, H, D, Hk = c["T"], c["H"], c["D"], c["Hk"]
    dt = torch.float32 if c["fp32"] else torch.bfloat16
    s = dict(q=_randn(g, T, H, D, dtype=dt), k=_randn(g, T, Hk, D, dtype=dt) if Hk else None, table=_rope_table(c["R"], MAX_POS),
             pos=torch.randint(0, MAX_POS, (T,), generator=g, device="cuda").to(torch.int32))
    for n in ("q", "k"):
        s[n + "w"] = 1 + _randn(g, D, scale=0.1) if c["norm"] != "none" else None
        s[n + "b"] = _randn(g, D, scale=0.1) if c["norm"] == "layer" else None
    s["gate"] = _randn(g, T, H, scale=H ** -0.5) if c["gate"] else None
    od = E4M3 if c["fp8"] else torch.bfloat16
    s["q_out"] = torch.zeros(T, H, c["wide"] or D, dtype=torch.bfloat16, device="cuda").to(od)[..., (c["wide"] or D) - D:]
    s["k_out"] = torch.empty(T, Hk, D, dtype=od, device="cuda") if Hk else None
    s["q_scale"] = torch.empty(T, H, device="cuda") if c["fp8"] else None
    s["k_scale"] = torch.empty(T, Hk, device="cuda") if c["fp8"] and Hk else None
    return s


def _tokens(c, seed):
    """Per sequence its number of new tokens: equal, or cut at places that the seed gives."""
    B, T = c["B"], c["T"]
    if T % B == 0:
        return [T // B] * B
    r = torch.Generator()
    r.manual_seed(seed)
    cuts = [0] + sorted((torch.randperm(T - 1, generator=r)[:B - 1] + 1).tolist()) + [T]
    return [b - a for a, b in zip(cuts, cuts[1:])]


def _prepare_append(c, g, seed):
    B, T = c["B"], c["T"]
    new = _tokens(c, seed)
    r = torch.Generator()
    r.manual_seed(seed + 1)
    old = torch.randint(0, 200, (B,), generator=r).tolist()      # positions that are in the cache already
    per = max(-(-(o + n) // PAGE) for o, n in zip(old, new))
    lens = [-(-(o + n) // PAGE) for o, n in zip(old, new)]
    pages = -(-(T + 200 * B) // PAGE) + B                        # the pool holds them wherever the cuts lie
    order = torch.randperm(pages, generator=r).tolist()
    table = torch.full((B, per), -1, dtype=torch.int32)
    at = 0
    for b in range(B):
        table[b, :lens[b]] = torch.tensor(order[at:at + lens[b]], dtype=torch.int32)
        at += lens[b]
    pos = torch.cat([torch.arange(o, o + n) for o, n in zip(old, new)]).to(torch.int32)
    seq = torch.cat([torch.full((n,), b) for b, n in enumerate(new)]).to(torch.int32)
    dt = torch.float32 if c["fp32"] else torch.bfloat16
    proj = _randn(g, T, D_LATENT + D_ROPE, dtype=dt)             # one projection gives both parts
    rows = pages * PAGE
    s = dict(latent=proj[:, :D_LATENT], rope=proj[:, D_LATENT:], pos=pos.cuda(), seq=seq.cuda(), block_table=table.cuda(), table=_rope_table(D_ROPE, MAX_POS))
    if c["fp8"]:
        s["kv"] = torch.zeros(rows, 656, dtype=torch.uint8, device="cuda")
        s["kv"][:, :512] = _randn(g, rows, 512, scale=100.0).to(E4M3).view(torch.uint8)
        s["kv"][:, 512:528] = (torch.rand(rows, 4, generator=g, device="cuda") * 0.01 + 0.005).view(torch.uint8)
        s["kv"][:, 528:] = _randn(g, rows, 64, dtype=torch.bfloat16).view(torch.uint8)
    else:
        s["kv"] = _randn(g, rows, 576, dtype=torch.bfloat16)
    s["lw"] = 1 + _randn(g, D_LATENT, scale=0.1) if c["norm"] else None
    s["index"] = s["key"] = s["iw"] = s["ib"] = None
    if c["index"]:
        s["key"] = _randn(g, T, D_INDEX, dtype=dt)
        s["iw"], s["ib"] = 1 + _randn(g, D_INDEX, scale=0.1), _randn(g, D_INDEX, scale=0.1)
        s["index"] = _index_cache(g, pages, c["fp8"])
    return s


def _index_cache(g, pages, fp8):
    """Pages of PAGE keys of 128 values: bf16, or e4m3 with the keys' fp32 scales behind them."""
    if not fp8:
        return _randn(g, pages * PAGE, D_INDEX, dtype=torch.bfloat16)
    cache = torch.empty(pages, PAGE * (D_INDEX + 4), dtype=torch.uint8, device="cuda")
    for p0 in range(0, pages, 4096):
        n = min(4096, pages - p0)
        cache[p0:p0 + n, :PAGE * D_INDEX] = _randn(g, n, PAGE * D_INDEX, scale=150.0).to(E4M3).view(torch.uint8)
    cache[:, PAGE * D_INDEX:] = (torch.rand(pages, PAGE, generator=g, device="cuda") * 0.01 + 0.005).view(torch.uint8)
    return cache


def _lengths(c, seed):
    """Positions that each sequence has."""
    r = torch.Generator()
    r.manual_seed(seed)
    n = torch.randint(max(c["s_q"], c["kv_len"] // 2), c["kv_len"] + 1, (c["B"],), generator=r)
    n[-1] = c["kv_len"]
    return torch.full_like(n, c["kv_len"]) if c["even"] or c["B"] == 1 else n


def _prepare_scores(c, g, seed):
    B, s_q, H, kv_len = c["B"], c["s_q"], c["H"], c["kv_len"]
    lens = _lengths(c, seed)
    per = -(-kv_len // PAGE)
    q = _randn(g, B * s_q, H, D_INDEX, scale=100.0 if c["fp8"] else 1.0)
    return dict(q=q.to(E4M3 if c["fp8"] else torch.bfloat16), weights=_randn(g, B * s_q, H, scale=(1e-3 if c["fp8"] else 0.1) * H ** -0.5),
                index=_index_cache(g, B * per, c["fp8"]), block_table=torch.randperm(B * per, generator=g, device="cuda").to(torch.int32).view(B, per),
                # the rows of a sequence are its last positions
                valid=(lens[:, None] - s_q + 1 + torch.arange(s_q)[None, :]).reshape(-1).to(torch.int32).cuda(),
                out=torch.empty(B * s_q, -(-kv_len // c["block"]), device="cuda"))


def _prepare_select(c, g, seed):
    rows, kv_len, block = c["rows"], c["kv_len"], c["block"]
    sc = _randn(g, rows, -(-kv_len // block))
    sc = torch.where(torch.rand(sc.shape, generator=g, device="cuda") < 0.1, (sc * 4).round() / 4, sc)      # some are equal
    if c["causal"]:
        valid = (kv_len - rows + 1 + torch.arange(rows)).clamp(min=1).to(torch.int32).cuda()
    else:
        valid = torch.randint(max(1, kv_len // 2), kv_len + 1, (rows,), generator=g, device="cuda").to(torch.int32)
    return dict(scores=sc, valid=valid, out=torch.empty(rows, c["blocks"] * block, dtype=torch.int32, device="cuda"))


FIRST, LOCAL = 1, 2          # blocks that are always selected: the first of a row and its last ones


# ------------------------------------------------------------------ one pass
def run(s):
    c = s["case"]
    if c["kind"] == "rotate":
        if own:
            from opfoundry_b200 import api
            r = api.norm_rotate(s["q"], s["table"], s["pos"], k=s["k"], q_weight=s["qw"], k_weight=s["kw"], q_bias=s["qb"], k_bias=s["kb"],
                                center=c["norm"] == "layer", eps=EPS, rope_begin=c["begin"], interleaved=c["pairs"], head_weight=s["gate"],
                                q_out=s["q_out"], k_out=s["k_out"], q_scale=s["q_scale"], k_scale=s["k_scale"])
            return [x for x in r if x is not None]
        return _plain_rotate(s)
    if c["kind"] == "append":
        if own:
            from opfoundry_b200 import api
            api.append_cache(s["latent"], s["rope"], s["kv"], s["table"], s["pos"], seq_ids=s["seq"], block_table=s["block_table"], page_block_size=PAGE,
                             latent_weight=s["lw"], index_key=s["key"], index_cache=s["index"], index_weight=s["iw"], index_bias=s["ib"], index_center=True,
                             eps=EPS)
        else:
            _plain_append(s)
        return _cache_values(s)
    if c["kind"] == "scores":
        if own:
            from opfoundry_b200 import api
            return api.index_scores(s["q"], s["weights"], s["index"], s["valid"], c["kv_len"], s_q=c["s_q"], block=c["block"],
                                    block_table=s["block_table"], page_block_size=PAGE, out=s["out"])
        return _plain_scores(s)
    if own:
        from opfoundry_b200 import api
        return api.block_select(s["scores"], c["blocks"], c["block"], s["valid"], first=FIRST, local=LOCAL, out=s["out"])
    return _plain_select(s)


def _normed_rotated(x, w, b, center, cs, begin, pairs):
    """x [tokens, heads, D]; cs [tokens, R]; w, b: [D] or None.  In 32 bits."""
    x = x.float()
    if center:
        x = x - x.mean(-1, keepdim=True)
    if w is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w
        if b is not None:
            x = x + b
    R = cs.shape[1]
    cos, sin = cs[:, None, :R // 2], cs[:, None, R // 2:]
    r = x[..., begin:begin + R]
    u, v = (r[..., 0::2], r[..., 1::2]) if pairs else (r[..., :R // 2], r[..., R // 2:])
    u, v = u * cos - v * sin, u * sin + v * cos
    r = torch.stack([u, v], dim=-1).flatten(-2) if pairs else torch.cat([u, v], dim=-1)
    return torch.cat([x[..., :begin], r, x[..., begin + R:]], dim=-1)


def _quantised(y, group):
    """y [..., n] in groups of `group` values: e4m3 values and the groups' scales."""
    y = y.unflatten(-1, (-1, group))
    amax = y.abs().amax(-1, keepdim=True)
    scale = torch.where(amax > 0, amax / 448.0, 1.0)
    return (y / scale).flatten(-2).to(E4M3), scale[..., 0]


def _plain_rotate(s):
    c, cs = s["case"], s["table"][s["pos"].long()]
    r, scales = [], []
    for n in ("q", "k"):
        if s[n] is None:
            continue
        y = _normed_rotated(s[n], s[n + "w"], s[n + "b"], c["norm"] == "layer", cs, c["begin"], c["pairs"])
        if c["fp8"]:
            codes, scale = _quantised(y, c["D"])
            s[n + "_out"].copy_(codes)
            scales.append(scale[..., 0] * s["gate"] if n == "q" and c["gate"] else scale[..., 0])
        else:
            s[n + "_out"].copy_(y)
        r.append(s[n + "_out"])
    return r + scales


def _plain_append(s):
    c, cs = s["case"], s["table"][s["pos"].long()]
    pos, seq = s["pos"].long(), s["seq"].long()
    page = s["block_table"][seq, pos // PAGE].long()
    row = page * PAGE + pos % PAGE
    y = s["latent"].float()
    if c["norm"]:
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * s["lw"]
    rope = _normed_rotated(s["rope"][:, None, :], None, None, False, cs, 0, True)[:, 0].to(torch.bfloat16)
    if c["fp8"]:
        codes, scale = _quantised(y, 128)
        s["kv"][row] = torch.cat([codes.view(torch.uint8), scale.view(torch.uint8), rope.view(torch.uint8)], dim=1)
    else:
        s["kv"][row] = torch.cat([y.to(torch.bfloat16), rope], dim=1)
    if c["index"]:
        k = _normed_rotated(s["key"][:, None, :], s["iw"], s["ib"], True, cs, 0, True)[:, 0]
        if c["fp8"]:
            codes, scale = _quantised(k, D_INDEX)
            keys, scales = _index_views(s["index"])
            keys.view(torch.uint8)[page, pos % PAGE] = codes.view(torch.uint8)
            scales[page, pos % PAGE] = scale[:, 0]
        else:
            s["index"][row] = k.to(torch.bfloat16)


def _index_views(cache):
    """Keys [pages, PAGE, 128] e4m3 and scales [pages, PAGE] of an fp8 index cache."""
    return cache[:, :PAGE * D_INDEX].unflatten(1, (PAGE, D_INDEX)).view(E4M3), cache[:, PAGE * D_INDEX:].view(torch.float32)


def _cache_values(s):
    """The caches as the values that they hold."""
    c, r = s["case"], {}
    if c["fp8"]:
        r |= dict(latent=s["kv"][:, :512].view(E4M3), latent_scale=s["kv"][:, 512:528].view(torch.float32), rope=s["kv"][:, 528:].view(torch.bfloat16))
    else:
        r |= dict(rows=s["kv"])
    if c["index"]:
        r |= dict(zip(("key", "key_scale"), _index_views(s["index"]))) if c["fp8"] else dict(key=s["index"])
    return r


def _plain_scores(s):
    c = s["case"]
    B, s_q, H, kv_len, block = c["B"], c["s_q"], c["H"], c["kv_len"], c["block"]
    pages = s["block_table"].long()
    if c["fp8"]:
        keys, scales = _index_views(s["index"])
        k = keys.view(torch.uint8)[pages].view(E4M3).float().reshape(B, -1, D_INDEX)
        ks = scales[pages].reshape(B, 1, -1)
    else:
        k, ks = s["index"].unflatten(0, (-1, PAGE))[pages].float().reshape(B, -1, D_INDEX), None
    n = k.shape[1]
    dots = torch.bmm(s["q"].float().reshape(B, s_q * H, D_INDEX), k.transpose(1, 2)).clamp_(min=0)
    r = torch.bmm(s["weights"].reshape(B * s_q, 1, H), dots.reshape(B * s_q, H, n)).reshape(B, s_q, n)
    r = (r * ks if c["fp8"] else r).reshape(B * s_q, n)[:, :kv_len]
    r = r.masked_fill(torch.arange(kv_len, device=r.device) >= s["valid"][:, None], -math.inf)
    if block > 1:
        r = torch.nn.functional.pad(r, (0, -kv_len % block), value=-math.inf).unflatten(1, (-1, block)).amax(-1)
    return r


def _plain_select(s):
    c, sc = s["case"], s["scores"]
    block, n, valid = c["block"], c["blocks"], s["valid"].long()[:, None]
    col = torch.arange(sc.shape[1], device=sc.device)
    live = (valid + block - 1) // block
    sc = sc.masked_fill((col < FIRST) | (col >= live - LOCAL), math.inf).masked_fill(col >= live, -math.inf)
    best = sc.sort(dim=1, descending=True, stable=True).indices[:, :n]
    if best.shape[1] < n:
        best = torch.nn.functional.pad(best, (0, n - best.shape[1]), value=1 << 40)
    best = torch.where(best < live, best, 1 << 40).sort(dim=1).values
    p = (best[:, :, None] * block + torch.arange(block, device=sc.device)).flatten(1)
    return torch.where(p < valid, p, -1).to(torch.int32)


# ------------------------------------------------------------------ from the definitions, in 64 bits
def exact(case, seed):
    return {"rotate": _exact_rotate, "append": _exact_append, "scores": _exact_scores, "select": _exact_select}[case["kind"]](prepare(case, seed))


def _turned(x, w, b, center, table, pos, begin, pairs):
    """Norm, then each pair as a complex number times exp(i angle), the table's numbers taken as they are."""
    x = x.double()
    mean = x.sum(-1, keepdim=True) / x.shape[-1] if center else 0.0
    if w is not None:
        x = (x - mean) / ((x - mean).pow(2).sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt() * w.double() + (0.0 if b is None else b.double())
    R = table.shape[1]
    first = torch.arange(R // 2, device=x.device) * (2 if pairs else 1) + begin
    second = first + (1 if pairs else R // 2)
    t = table[pos.long()].double()
    z = torch.complex(x[..., first], x[..., second]) * torch.complex(t[:, None, :R // 2], t[:, None, R // 2:])
    y = x.clone()
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _scaled(y, group):
    """(y in units of its groups' scales, scales): amax / 448, or 1."""
    g = y.reshape(*y.shape[:-1], -1, group)
    m = g.abs().max(-1).values / 448
    m = m + (m == 0)
    return (g / m[..., None]).reshape(y.shape), m


def _exact_rotate(s):
    c, r, scales = s["case"], [], []
    for n in ("q", "k"):
        if s[n] is not None:
            y = _turned(s[n], s[n + "w"], s[n + "b"], c["norm"] == "layer", s["table"], s["pos"], c["begin"], c["pairs"])
            if c["fp8"]:
                y, m = _scaled(y, c["D"])
                scales.append(m[..., 0] * (s["gate"].double() if n == "q" and c["gate"] else 1.0))
            r.append(y)
    return r + scales


def _exact_append(s):
    c, v = s["case"], {k: x.double() for k, x in _cache_values(s).items()}
    pos, seq = s["pos"].long(), s["seq"].long()
    page, at = s["block_table"].long()[seq, pos // PAGE], pos % PAGE
    row = page * PAGE + at
    y = s["latent"].double()
    if c["norm"]:
        y = y / (y.pow(2).sum(-1, keepdim=True) / D_LATENT + EPS).sqrt() * s["lw"].double()
    rope = _turned(s["rope"][:, None], None, None, False, s["table"], s["pos"], 0, True)[:, 0]
    if c["fp8"]:
        v["latent"][row], v["latent_scale"][row] = _scaled(y, 128)
        v["rope"][row] = rope
    else:
        v["rows"][row] = torch.cat([y, rope], 1)
    if c["index"]:
        k = _turned(s["key"][:, None], s["iw"], s["ib"], True, s["table"], s["pos"], 0, True)[:, 0]
        if c["fp8"]:
            k, m = _scaled(k, D_INDEX)
            v["key"][page, at], v["key_scale"][page, at] = k, m[:, 0]
        else:
            v["key"][row] = k
    return v


def _exact_scores(s):
    c = s["case"]
    r = torch.full((c["B"] * c["s_q"], -(-c["kv_len"] // c["block"])), -math.inf, dtype=torch.float64, device="cuda")
    valid, pages = s["valid"].tolist(), s["block_table"].long()
    for b in range(c["B"]):
        if c["fp8"]:
            keys, scales = _index_views(s["index"])
            k = keys.view(torch.uint8)[pages[b]].view(E4M3).double().flatten(0, 1) * scales[pages[b]].double().flatten()[:, None]
        else:
            k = s["index"].unflatten(0, (-1, PAGE))[pages[b]].double().flatten(0, 1)
        for i in range(b * c["s_q"], (b + 1) * c["s_q"], 64):
            e = min(i + 64, (b + 1) * c["s_q"])
            n = max(valid[i:e])
            d = (torch.relu(s["q"][i:e].double() @ k[:n].T) * s["weights"][i:e].double()[:, :, None]).sum(1)
            d[torch.arange(n, device="cuda")[None, :] >= s["valid"][i:e, None]] = -math.inf
            m = -(-n // c["block"])
            full = torch.full((e - i, m * c["block"]), -math.inf, dtype=torch.float64, device="cuda")
            full[:, :n] = d
            r[i:e, :m] = full.reshape(e - i, m, -1).max(-1).values
    return r


def _exact_select(s):
    """By ranks: a block is selected when fewer than `blocks` stand before it."""
    c, sc = s["case"], s["scores"].double()
    block, n, nb = c["block"], c["blocks"], sc.shape[1]
    if sc.numel() * nb > 2e10:
        return None
    r = torch.full((c["rows"], n * block), -1, dtype=torch.int32, device="cuda")
    col, order = torch.arange(nb, device="cuda"), torch.arange(n * block, device="cuda")
    step = max(1, int(2e8 // (nb * nb)))
    for i in range(0, c["rows"], step):
        x, valid = sc[i:i + step].clone(), s["valid"][i:i + step].long()[:, None]
        live = -(-valid // block)
        x[(col < FIRST) | (col >= live - LOCAL)] = math.inf
        ahead = (x[:, None, :] > x[:, :, None]) | ((x[:, None, :] == x[:, :, None]) & (col[None, None, :] < col[None, :, None]))
        taken = ((ahead & (col < live)[:, None, :]).sum(2) < n) & (col < live)
        p = col[None, :, None] * block + torch.arange(block, device="cuda")
        p = p.expand(x.shape[0], nb, block)[taken[:, :, None].expand(-1, nb, block) & (p < valid[:, :, None])].to(torch.int32)
        count = torch.minimum(taken.sum(1) * block, taken.sum(1) * block - (live * block - valid)[:, 0])
        r[i:i + step][order[None, :] < count[:, None]] = p
    return r


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    c = case
    if c["kind"] == "rotate":
        heads = c["H"] + c["Hk"]
        per = (4 if c["fp32"] else 2) * c["D"] + (c["D"] + 4 if c["fp8"] else 2 * c["D"])
        return {"bytes": c["T"] * (heads * per + 4 + (4 * c["H"] if c["gate"] else 0)) + min(c["T"], MAX_POS) * 4 * c["R"], "flops": 0}
    if c["kind"] == "append":
        x = 4 if c["fp32"] else 2
        per = x * (D_LATENT + D_ROPE) + (656 if c["fp8"] else 1152) + 8
        if c["index"]:
            per += x * D_INDEX + (D_INDEX + 4 if c["fp8"] else 2 * D_INDEX)
        return {"bytes": c["T"] * per + min(c["T"], MAX_POS) * 4 * D_ROPE, "flops": 0}
    if c["kind"] == "scores":
        # sequences of ragged lengths have three quarters of the longest on the average
        n = c["kv_len"] * (1.0 if c["even"] or c["B"] == 1 else 0.75)
        pairs = c["B"] * c["s_q"] * max(1.0, n - (c["s_q"] - 1) / 2)
        rows = c["B"] * c["s_q"]
        return {"bytes": c["B"] * n * (D_INDEX + 4 if c["fp8"] else 2 * D_INDEX) + rows * (c["H"] * (D_INDEX * (1 if c["fp8"] else 2) + 4) + 4)
                + 4 * rows * -(-c["kv_len"] // c["block"]), "flops": 2 * c["H"] * D_INDEX * pairs}
    valid = sum(max(1, c["kv_len"] - c["rows"] + 1 + i) for i in range(c["rows"])) if c["causal"] else c["rows"] * 0.75 * c["kv_len"]
    return {"bytes": 4 * valid / c["block"] + 4 * c["rows"] * c["blocks"] * c["block"] + 4 * c["rows"], "flops": 0}
