"""Performance cases of the paged 4-bit KV cache: the tables that place tokens in pages, the
writer and the reader of the pages, and the attention over them.

``kind`` picks the calls of a case:

  tables  build_block_tables: block tables and slot maps of a step from request lengths
  append  store_kv4 of new tokens, then load_kv4 of the contexts for a prompt kernel
  attend  attend_kv4: causal attention over the pages, whole context or a window
  nsa     nsa_attend_kv4: compressed tokens, selected blocks and window, gated and mixed

A page holds ``page`` tokens of every KV group: k [pages, G, page, dk/2] bytes (element 2i in
the low nibble of byte i, e2m1) with one scale byte (e8m0) for each 32 elements, k_scale [pages,
G, page, dk/32], and the same for v.  ``own`` false: plain torch operations.  ``own`` true: the
framework's calls.  ``exact``: the definitions in 64 bits.
"""
import math
import random
import sys
from pathlib import Path

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp32": torch.float32}
_LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _nsa():
    p = str(Path(__file__).resolve().parents[1] / "nsa-test_amd")
    if p not in sys.path:
        sys.path.insert(0, p)
    import nsa

    return nsa


# ------------------------------------------------------------------------------- cases
def _case(name, kind, **kw):
    c = dict(name=name, kind=kind, B=1, page=64, lo=1, hi=1)
    if kind in ("attend", "nsa"):
        c.update(dtype="bf16", rows=1)
    if kind == "nsa":
        c.update(n=16, w=512, l=32, d=16, lp=64)
    c.update(kw)
    return c


def listed():
    return [
        # one decoding step of a server: 64 requests, a token each
        _case("tables_decode", "tables", B=64, lo=100, hi=32000, new_lo=1, new_hi=1, packed=False),
        # prompts of one scheduling step, packed without padding, some of them continued
        _case("tables_prompts", "tables", B=48, lo=0, hi=8192, new_lo=1, new_hi=4096, packed=True),
        # one token joins a short fp32 context, read back whole: a toy model's step
        _case("append_token_fp32", "append", dtype="fp32", G=2, dk=64, dv=64, lo=300, hi=300, chunk=1, page=16),
        # prompts taken in chunks: 512 tokens of 8 requests stored, their contexts read back for the
        # prompt kernels, at the default layer's heads
        _case("append_chunk", "append", dtype="bf16", B=8, G=4, dk=192, dv=128, lo=513, hi=8192, chunk=512),
        # a single short request over its whole context
        _case("attend_short", "attend", H=8, G=2, dk=64, dv=64, lo=700, hi=700, w=0),
        # a ragged batch over the last 512 tokens
        _case("attend_window_batch", "attend", B=32, H=32, G=2, dk=128, dv=128, lo=200, hi=8192, w=512),
        # four tokens of each request verified at once, fp32, 4 heads a group, small pages
        _case("attend_verify_fp32", "attend", dtype="fp32", B=4, H=16, G=4, dk=64, dv=64, lo=300, hi=5001, w=0, rows=4,
              page=16),
        # one request over a long context, at the default layer's heads
        _case("attend_long", "attend", H=64, G=4, dk=192, dv=128, lo=131072, hi=131072, w=0),
        # one layer of a small fp32 model served: a single request, its prompt of 1000 tokens behind it
        _case("nsa_short_fp32", "nsa", dtype="fp32", H=8, G=2, dk=64, dv=64, lo=1000, hi=1000, w=256),
        # a ragged batch of requests at the default layer's heads
        _case("nsa_batch", "nsa", B=32, H=64, G=4, dk=192, dv=128, lo=200, hi=16384),
        # long requests at the long-context configuration's heads
        _case("nsa_long_batch", "nsa", B=16, H=32, G=2, dk=128, dv=128, lo=16001, hi=32000),
    ]


def _logint(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


_HEADS = [(8, 2), (16, 4), (16, 1), (32, 2), (64, 4)]
_DIMS = [(32, 32), (64, 64), (128, 128), (192, 128)]


def draw(rng):
    kind = rng.choice(["tables", "append", "attend", "attend", "nsa", "nsa"])
    c = _case("", kind)
    del c["name"]
    c["page"] = rng.choice([16, 32, 64, 64, 128])
    if kind == "tables":
        c["B"] = _logint(rng, 1, 256)
        c["packed"] = rng.random() < 0.5
        c["hi"] = _logint(rng, 64, 32000)
        c["lo"] = rng.choice([0, 1, c["hi"] // 3])
        c["new_hi"] = _logint(rng, 1, max(1, 65536 // c["B"]))
        c["new_lo"] = rng.choice([0, 1, c["new_hi"]])
        return c
    c["H"], c["G"] = rng.choice(_HEADS)
    c["dk"], c["dv"] = rng.choice(_DIMS)
    c["dtype"] = "fp32" if rng.random() < 0.25 else "bf16"
    width = c["G"] * (c["dk"] + c["dv"])
    if kind == "append":
        del c["H"]
        c["B"] = _logint(rng, 1, 16)
        c["hi"] = _logint(rng, 2, min(16384, 16384 * 1280 // (c["B"] * width)))
        c["lo"] = max(1, c["hi"] // rng.choice([1, 2, 8]))
        c["chunk"] = _logint(rng, 1, c["lo"])
        return c
    c["B"] = _logint(rng, 1, 48)
    tokens = 131072 * 1280 // width
    if kind == "attend":
        c["w"] = rng.choice([0, 0, 128, 512])
        c["rows"] = rng.choice([1, 1, 1, 2, 5])
        c["hi"] = _logint(rng, 8, min(131072, tokens // (c["B"] * c["rows"])))
    else:
        c["w"] = rng.choice([128, 256, 512, 512])
        c["n"] = rng.choice([4, 8, 16, 16])
        c["hi"] = _logint(rng, 64, min(32000, tokens // c["B"]))
    c["lo"] = max(c["rows"], c["hi"] // rng.choice([1, 2, 16]))
    return c


def _spread(salt, B, lo, hi):
    """B whole numbers of [lo, hi], evenly over the logarithm, the largest among them."""
    rng = random.Random(f"{salt} {B} {lo} {hi}")
    out = [_logint(rng, max(lo, 1), hi) if rng.random() < 0.9 else lo for _ in range(B)]
    out[rng.randrange(B)] = hi
    return out


def _lengths(c):
    return _spread("lengths", c["B"], c["lo"], c["hi"])


def _new(c):
    return _spread("new", c["B"], c["new_lo"], c["new_hi"])


def _pages(n, page):
    return -(-n // page)


def _n_cmp(c, tokens):
    """Compressed tokens completed by that many tokens (block i covers i d .. i d + l - 1)."""
    return (tokens - c["l"]) // c["d"] + 1 if tokens >= c["l"] else 0


def work(c):
    B = c["B"]
    if c["kind"] == "tables":
        news, lens = _new(c), _lengths(c)
        rows = sum(news) if c["packed"] else B * max(news)
        fresh = sum(_pages(a + b, c["page"]) - _pages(a, c["page"]) for a, b in zip(lens, news))
        # slot, position and sequence of each row; page numbers read and written; per-request counts
        return {"bytes": rows * 16 + fresh * 8 + B * 16, "flops": 0}
    es = 4 if c["dtype"] == "fp32" else 2
    row = c["G"] * (c["dk"] + c["dv"])
    if c["kind"] == "append":
        new = B * c["chunk"]
        tokens = sum(_lengths(c))
        # new rows read and stored in 4 bits, the older rows read in 4 bits, every row of the padded
        # result written
        return {"bytes": new * row * es + tokens * row * 17 // 32 + B * max(_lengths(c)) * row * es, "flops": 0}
    keys = pairs = 0
    for n in _lengths(c):
        if c["kind"] == "attend":
            w = c["w"] or n
            keys += min(n, w + c["rows"] - 1)
            pairs += sum(min(n - i, w) for i in range(c["rows"]))
        else:
            own_block = (n - 1) // c["lp"]
            k = (_n_cmp(c, n) + min(n, c["w"])
                 + min(c["n"], own_block + 1) * c["lp"] - (c["lp"] - (n - own_block * c["lp"])))
            keys += k
            pairs += k
    io = B * c["rows"] * c["H"] * (c["dk"] + c["dv"]) * es
    return {"bytes": keys * row * 17 // 32 + io, "flops": 2 * pairs * c["H"] * (c["dk"] + c["dv"])}


# ------------------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _quantize(x):
    """x [..., d] fp32 -> e2m1 codes [..., d/2] (two a byte) and e8m0 scales [..., d/32]."""
    xb = x.unflatten(-1, (-1, 32))
    _, ex = torch.frexp(xb.abs().amax(-1))  # amax = m 2^ex, m in [0.5, 1)
    e = (ex - 3 + 127).clamp(1, 254)
    y = xb * torch.exp2((127 - e).float()).unsqueeze(-1)
    a = y.abs()
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
    code = (code + 8 * (y < 0)).to(torch.uint8).flatten(-2)
    return code[..., 0::2] | (code[..., 1::2] << 4), e.to(torch.uint8)


def _pool(g, n_pages, G, page, d, spread):
    """Pages of quantised normal values, the channels of different size (log-normal)."""
    codes = torch.empty(n_pages, G, page, d // 2, dtype=torch.uint8, device="cuda")
    scales = torch.empty(n_pages, G, page, d // 32, dtype=torch.uint8, device="cuda")
    size = torch.exp(spread * torch.randn(G, 1, d, device="cuda", generator=g))
    step = max(1, (1 << 26) // (G * page * d))
    for i in range(0, n_pages, step):
        n = min(step, n_pages - i)
        codes[i:i + n], scales[i:i + n] = _quantize(torch.randn(n, G, page, d, device="cuda", generator=g) * size)
    return codes, scales


def _tables(g, counts, extra, n_pages):
    """Block tables [B, W] int32 over a random order of the pool's pages, -1 behind a request's own;
    the pages left over in order."""
    B, W = len(counts), max(counts) + extra
    perm = torch.randperm(n_pages, device="cuda", generator=g).to(torch.int32)
    n = torch.tensor(counts, device="cuda")
    first = torch.cumsum(n, 0) - n
    j = torch.arange(W, device="cuda")
    t = torch.where(j < n[:, None], perm[(first[:, None] + j).clamp(max=n_pages - 1)], -1).to(torch.int32)
    return t.contiguous(), perm[sum(counts):].contiguous()


def _cache(g, c, counts, extra=1, spare=3):
    n_pages = sum(counts) + spare
    s = {}
    s["tables"], s["free"] = _tables(g, counts, extra, n_pages)
    s["k"], s["ks"] = _pool(g, n_pages, c["G"], c["page"], c["dk"], 0.5)
    s["v"], s["vs"] = _pool(g, n_pages, c["G"], c["page"], c["dv"], 0.0)
    if own:
        s["kv"] = _nsa().PagedKV4(s["k"], s["ks"], s["v"], s["vs"])
    return s


def _i32(xs):
    return torch.tensor(xs, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    c, g = case, _gen(seed)
    lens = _lengths(c)
    s = {"case": c, "lengths": _i32(lens), "max_len": max(lens)}
    if c["kind"] == "tables":
        news = _new(c)
        fresh = [_pages(a + b, c["page"]) - _pages(a, c["page"]) for a, b in zip(lens, news)]
        counts = [_pages(a, c["page"]) for a in lens]
        width = max(_pages(a + b, c["page"]) for a, b in zip(lens, news))
        s["tables"], s["free"] = _tables(g, counts, width - max(counts) + 1, sum(counts) + sum(fresh) + 9)
        s["new"] = _i32(news)
        s["used"] = _i32([2])  # two pages of the list are taken already
        s["rows"] = sum(news) if c["packed"] else c["B"] * max(news)
        s["per"] = 0 if c["packed"] else max(news)
        return s
    dt = _DT[c["dtype"]]
    if c["kind"] == "append":
        s.update(_cache(g, c, [_pages(n, c["page"]) for n in lens]))
        N = c["B"] * c["chunk"]
        s["kn"] = torch.randn(N, c["G"], c["dk"], device="cuda", generator=g).to(dt)
        s["vn"] = torch.randn(N, c["G"], c["dv"], device="cuda", generator=g).to(dt)
        p = s["lengths"].long()[:, None] - c["chunk"] + torch.arange(c["chunk"], device="cuda")
        s["slots"] = (s["tables"].long().gather(1, p // c["page"]) * c["page"] + p % c["page"]).reshape(-1)
        return s
    B, H, R = c["B"], c["H"], c["rows"]
    s["scale"] = 1.0 / math.sqrt(c["dk"])
    s["q"] = torch.randn(B, R, H, c["dk"], device="cuda", generator=g).to(dt).transpose(1, 2)
    if c["kind"] == "attend":
        s.update(_cache(g, c, [_pages(n, c["page"]) for n in lens]))
        return s
    s["cmp"] = _cache(g, c, [_pages(_n_cmp(c, n), c["page"]) for n in lens])
    counts = [_pages(n, c["page"]) for n in lens]
    s["sel"] = _cache(g, c, counts)
    win = _cache(g, c, counts)
    win["tables"] = s["sel"]["tables"]  # a token has the same slot in both
    s["win"] = win
    # the initial and the local blocks, then others by a random score; -1 where there are no more
    nb = _pages(max(lens), c["lp"])
    t = s["lengths"].long() - 1
    sc = torch.rand(B, c["G"], nb, device="cuda", generator=g)
    blk = torch.arange(nb, device="cuda")
    last = (t // c["lp"])[:, None, None]
    sc = sc + 2.0 * ((blk == last) | (blk == last - 1) | (blk == 0))
    sc = torch.where(blk <= last, sc, -1.0)
    top = torch.topk(sc, min(c["n"], nb), dim=-1)
    idx = torch.where(top.values >= 0, top.indices, -1)
    idx = torch.cat([idx, torch.full((B, c["G"], c["n"] - idx.shape[-1]), -1, device="cuda")], dim=-1)
    s["indices"] = idx.unsqueeze(2).contiguous()
    s["gates"] = torch.randn(B, R, H, 3, device="cuda", generator=g).to(dt).permute(0, 2, 1, 3)
    if own:
        s["cfg"] = _nsa().NSAConfig(head_dim_qk=c["dk"], head_dim_v=c["dv"], n_heads=H, n_kv_groups=c["G"], n=c["n"],
                                    w=c["w"], l=c["l"], d=c["d"], l_prime=c["lp"])
    return s


# ------------------------------------------------------------------------- plain forms
def _plain_tables(s):
    c = s["case"]
    P, tables, lens, new = c["page"], s["tables"], s["lengths"].long(), s["new"].long()
    have = (lens + P - 1) // P
    need = (lens + new + P - 1) // P - have
    first = torch.cumsum(need, 0) - need + s["used"].long()
    j = torch.arange(tables.shape[1], device="cuda")
    i = j - have[:, None]
    fresh = s["free"][(first[:, None] + i).clamp(0, s["free"].shape[0] - 1)]
    tables.copy_(torch.where((i >= 0) & (i < need[:, None]), fresh, tables))
    ends = torch.cumsum(new, 0)
    r = torch.arange(s["rows"], device="cuda")
    if s["per"]:
        b, i = r // s["per"], r % s["per"]
        ok = i < new[b]
    else:
        b = torch.searchsorted(ends, r, right=True)
        i = r - (ends - new)[b]
        ok = torch.ones_like(r, dtype=torch.bool)
    p = lens[b] + i
    page = tables[b, (p // P).clamp(max=tables.shape[1] - 1)].long()
    slots = torch.where(ok, page * P + p % P, -1)
    offsets = torch.cat([torch.zeros(1, dtype=torch.int64, device="cuda"), ends])
    info = torch.stack([ends[-1], s["used"][0] + need.sum(), torch.zeros_like(ends[-1])])
    return (tables, slots, torch.where(ok, p, -1).int(), torch.where(ok, b, -1).int(), offsets.int(), (lens + new).int(),
            info.int())


def _values(codes, scales):
    """The values that codes [..., d/2] with scales [..., d/32] stand for, fp32 [..., d]."""
    lv = torch.tensor(_LEVELS + tuple(-x for x in _LEVELS), device="cuda")
    b = torch.arange(256, device="cuda")
    pair = torch.stack([lv[b & 15], lv[b >> 4]], -1)
    x = pair.index_select(0, codes.reshape(-1).int()).view(*codes.shape[:-1], -1, 32)
    return (x * torch.exp2(scales.float() - 127.0).unsqueeze(-1)).flatten(-2)


def _take(codes, scales, slots):
    """Rows at slots [B, G or 1, n] of every group: fp32 [B, G, n, d] (slot -1: row 0)."""
    G, P = codes.shape[1], codes.shape[2]
    sl = slots.clamp(min=0).expand(-1, G, -1)
    pg, r, g = sl // P, sl % P, torch.arange(G, device="cuda")[:, None]
    return _values(codes[pg, g, r], scales[pg, g, r])


def _slots_of(tables, page, pos):
    """Slots of positions pos [B, g, n]; -1 where pos < 0."""
    B = pos.shape[0]
    j = (pos.clamp(min=0) // page).clamp(max=tables.shape[1] - 1).reshape(B, -1)
    return torch.where(pos >= 0, tables.long().gather(1, j).view(pos.shape) * page + pos % page, -1)


def _plain_append(s):
    c = s["case"]
    P, slots = c["page"], s["slots"]
    for name, x in (("k", s["kn"]), ("v", s["vn"])):
        codes, scales = _quantize(x.float())
        s[name][slots // P, :, slots % P] = codes
        s[name + "s"][slots // P, :, slots % P] = scales
    pos = torch.arange(s["max_len"], device="cuda")
    pos = torch.where(pos < s["lengths"][:, None], pos, -1).unsqueeze(1)
    sl = _slots_of(s["tables"], P, pos)
    keep = (sl >= 0).unsqueeze(-1)
    return tuple((_take(s[n], s[n + "s"], sl) * keep).to(s["kn"].dtype) for n in ("k", "v"))


def _plain_source(q, src, page, pos, mask, scale):
    """softmax(scale q K^T) V in fp32 over the keys at positions pos [B, g, n]; q [B,G,m,dk] fp32,
    mask [B, 1 or G, 1 or m, n] of visible keys.  A row that sees none is zero."""
    sl = _slots_of(src["tables"], page, pos)
    k, v = _take(src["k"], src["ks"], sl), _take(src["v"], src["vs"], sl)
    x = torch.matmul(q * scale, k.transpose(-1, -2).contiguous())
    x = x.masked_fill(~mask, float("-inf"))
    m = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(torch.isfinite(m), m, 0.0))
    z = p.sum(-1, keepdim=True)
    return torch.matmul(p, v) / torch.where(z > 0, z, 1.0)


def _plain_attend(s):
    c = s["case"]
    B, H, G, R = c["B"], c["H"], c["G"], c["rows"]
    lens = s["lengths"].long()
    n = s["max_len"] if not c["w"] else min(s["max_len"], c["w"] + R - 1)
    lo = (lens - n).clamp(min=0) if c["w"] else torch.zeros_like(lens)
    pos = lo[:, None] + torch.arange(n, device="cuda")
    pos = torch.where(pos < lens[:, None], pos, -1)[:, None]                   # [B,1,n]
    at = (lens[:, None] - R + torch.arange(R, device="cuda"))[:, None, :, None]  # [B,1,R,1]
    mask = (pos[:, :, None] >= 0) & (pos[:, :, None] <= at)
    if c["w"]:
        mask &= pos[:, :, None] > at - c["w"]
    hpg = H // G
    q = s["q"].float().reshape(B, G, hpg * R, c["dk"])
    mask = mask.unsqueeze(2).expand(B, 1, hpg, R, n).reshape(B, 1, hpg * R, n)
    o = _plain_source(q, s, c["page"], pos, mask, s["scale"])
    return o.view(B, H, R, c["dv"]).to(s["q"].dtype)


def _plain_nsa(s):
    c = s["case"]
    B, H, G = c["B"], c["H"], c["G"]
    lens = s["lengths"].long()
    t = (lens - 1)[:, None, None]
    q = s["q"].float().reshape(B, G, H // G, c["dk"])
    i = torch.arange(max(_n_cmp(c, s["max_len"]), 1), device="cuda")
    ps = [torch.where(i * c["d"] + c["l"] - 1 <= t, i, -1)]
    idx = s["indices"][:, :, 0]
    p = (idx.unsqueeze(-1) * c["lp"] + torch.arange(c["lp"], device="cuda")).flatten(-2)
    ps.append(torch.where((idx.repeat_interleave(c["lp"], -1) >= 0) & (p <= t), p, -1))
    p = t - torch.arange(min(c["w"], s["max_len"]), device="cuda")
    ps.append(p.clamp(min=-1))
    gate = torch.sigmoid(s["gates"].float())  # [B,H,1,3]
    out = 0.0
    for k, (name, pos) in enumerate(zip(("cmp", "sel", "win"), ps)):
        o = _plain_source(q, s[name], c["page"], pos, (pos >= 0).unsqueeze(2), s["scale"])
        out = out + gate[..., k:k + 1] * o.view(B, H, 1, c["dv"])
    return out.to(s["q"].dtype)


def run(s):
    c = s["case"]
    kind = c["kind"]
    if not own:
        with torch.no_grad():
            return {"tables": _plain_tables, "append": _plain_append, "attend": _plain_attend, "nsa": _plain_nsa}[kind](s)
    nsa = _nsa()
    if kind == "tables":
        t = nsa.build_block_tables(s["tables"], s["lengths"], s["new"], s["free"], s["used"], c["page"], s["rows"],
                                   row_stride=s["per"])
        return s["tables"], t.slots, t.positions, t.sequences, t.offsets, t.lengths, t.info
    if kind == "append":
        nsa.store_kv4(s["kv"], s["kn"], s["vn"], s["slots"])
        return nsa.load_kv4(s["kv"], s["tables"], s["lengths"], s["max_len"], dtype=s["kn"].dtype)
    if kind == "attend":
        return nsa.attend_kv4(s["q"], s["kv"], s["tables"], s["lengths"], s["scale"], window=c["w"] or None)
    return nsa.nsa_attend_kv4(s["q"], s["cmp"]["kv"], s["sel"]["kv"], s["win"]["kv"], s["cmp"]["tables"], s["sel"]["tables"],
                              s["lengths"], s["indices"], s["gates"], s["scale"], s["cfg"])


# ------------------------------------------------------------------------ definitions
def _exact_values(codes, scales):
    """float64 values of e2m1 codes and e8m0 scales, from the formats' fields."""
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    man, exp = (c & 1).double(), ((c >> 1) & 3).double()
    mag = torch.where(exp > 0, (1 + man / 2) * 2.0 ** (exp - 1), man / 2)
    mag = torch.where(c >= 8, -mag, mag)
    return mag * (2.0 ** (scales.double() - 127)).repeat_interleave(32, -1)


def _exact_round(x):
    """Rows [..., d] as 4 bits hold them: each block of 32 over 2^(floor(log2 max) - 2), to the nearest
    level (ties to the even code), 6 at most."""
    x = x.double().unflatten(-1, (-1, 32))
    big = x.abs().amax(-1, keepdim=True)
    e = torch.floor(torch.log2(torch.where(big > 0, big, 1.0))) - 2
    e = torch.where(big > 0, e, -126.0).clamp(min=-126)
    y = x / 2.0 ** e
    lv = torch.tensor(_LEVELS, dtype=torch.float64, device=x.device)
    a = y.abs().clamp(max=6.0)
    hi = torch.searchsorted(lv, a.contiguous()).clamp(max=7)
    lo = (hi - 1).clamp(min=0)
    up, down = lv[hi] - a, a - lv[lo]
    k = torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    return (torch.sign(y) * lv[k] * 2.0 ** e).flatten(-2)


def _exact_rows(src, b, page, pos):
    """K and V [G, n, d] of request b at positions pos (a tensor)."""
    pg = src["tables"][b].long()[pos // page]
    r = pos % page
    return [_exact_values(src[n][pg, :, r], src[n + "s"][pg, :, r]).transpose(0, 1).contiguous() for n in ("k", "v")]


def _exact_softmax(q, k, v, scale):
    """q [G, m, dk], k [G, n, dk], v [G, n, dv] -> [G, m, dv], all float64."""
    if k.shape[1] == 0:
        return q.new_zeros(*q.shape[:2], v.shape[-1])
    x = torch.matmul(q, k.transpose(-1, -2).contiguous()) * scale
    return torch.matmul(torch.softmax(x, -1), v)


def exact(case, seed):
    global own
    c = case
    if c["kind"] == "tables":
        return _exact_tables(c, seed)
    was, own = own, False
    try:
        s = prepare(c, seed)
    finally:
        own = was
    lens = _lengths(c)
    P, G, H = c["page"], c["G"], c["H"] if "H" in c else 0
    if c["kind"] == "append":
        out = []
        for n, new in (("k", s["kn"]), ("v", s["vn"])):
            x = torch.zeros(c["B"], G, s["max_len"], new.shape[-1], dtype=torch.float64, device="cuda")
            fresh = _exact_round(new).view(c["B"], c["chunk"], G, -1).transpose(1, 2)
            for b, m in enumerate(lens):
                pos = torch.arange(m, device="cuda")
                x[b, :, :m] = _exact_rows(s, b, P, pos)[0 if n == "k" else 1]
                x[b, :, m - c["chunk"]:m] = fresh[b]
            out.append(x)
        return tuple(out)
    out = torch.zeros(c["B"], H, c["rows"], c["dv"], dtype=torch.float64, device="cuda")
    for b, m in enumerate(lens):
        for i in range(c["rows"]):
            t = m - c["rows"] + i
            q = s["q"][b, :, i].double().view(G, H // G, -1)
            if c["kind"] == "attend":
                pos = torch.arange(max(0, t - c["w"] + 1) if c["w"] else 0, t + 1, device="cuda")
                out[b, :, i] = _exact_softmax(q, *_exact_rows(s, b, P, pos), s["scale"]).reshape(H, -1)
                continue
            gate = 1 / (1 + torch.exp(-s["gates"][b, :, i].double()))
            pos = torch.arange(_n_cmp(c, t + 1), device="cuda")
            o = _exact_softmax(q, *_exact_rows(s["cmp"], b, P, pos), s["scale"]).reshape(H, -1) * gate[:, :1]
            for g in range(G):
                rows = []
                for blk in sorted({x for x in s["indices"][b, g, i].tolist() if x >= 0}):
                    rows += range(blk * c["lp"], min((blk + 1) * c["lp"], t + 1))
                k, v = _exact_rows(s["sel"], b, P, torch.tensor(rows, device="cuda"))
                hs = slice(g * (H // G), (g + 1) * (H // G))
                o[hs] += _exact_softmax(q[g:g + 1], k[g:g + 1], v[g:g + 1], s["scale"])[0] * gate[hs, 1:2]
            pos = torch.arange(max(0, t - c["w"] + 1), t + 1, device="cuda")
            o += _exact_softmax(q, *_exact_rows(s["win"], b, P, pos), s["scale"]).reshape(H, -1) * gate[:, 2:]
            out[b, :, i] = o
    return out


def _exact_tables(c, seed):
    s = prepare(c, seed)
    P, lens, news = c["page"], _lengths(c), _new(c)
    tables, free = s["tables"].tolist(), s["free"].tolist()
    used = s["used"].item()
    slots, positions, seqs, offsets = [-1] * s["rows"], [-1] * s["rows"], [-1] * s["rows"], [0]
    for b, (m, n) in enumerate(zip(lens, news)):
        r0 = b * s["per"] if s["per"] else offsets[-1]
        for i in range(n):
            p = m + i
            if p % P == 0:
                tables[b][p // P] = free[used]
                used += 1
            slots[r0 + i], positions[r0 + i], seqs[r0 + i] = tables[b][p // P] * P + p % P, p, b
        offsets.append(offsets[-1] + n)
    t64 = torch.tensor(slots, dtype=torch.int64, device="cuda")
    return (_i32(tables), t64, _i32(positions), _i32(seqs), _i32(offsets), _i32([a + b for a, b in zip(lens, news)]),
            _i32([offsets[-1], used, 0]))
