"""GPU tests of what an NSAPagedKVCache holds and gives, against results made apart from it: the compressed values of
the layer's own NSAKVCache, and 64-bit attention for the types and batches that take other ways."""
import pytest
import torch

import paged_ref as ref
from nsa import NSAAttention, NSAPagedKVCache
from nsa.kernels import score_and_select
from test_gpu_paged_module import _cfg, _check_state, _held, _single

pytestmark = pytest.mark.gpu


def _near(got, want):
    """Rows that the pages hold against the 4-bit form of rows made another way.  In 16 bits the two may round another
    way, by 2^-8 of a value, where their fp32 sums (apart by some 2^-24 a term) lie at a border: one value in
    2^-8 / (terms 2^-24) or fewer.  Of those, one in 2^-2 / 2^-8 lies at a border of the 4-bit levels (2^-2 of a
    value apart or more).  One in a hundred is far above that; each by a level, half its block's largest at most."""
    assert got.shape == want.shape
    if want.numel() == 0:
        return
    assert (got != want).double().mean() < 1e-2
    pad = -want.shape[-1] % 32
    blocks = lambda t: torch.nn.functional.pad(t, (0, pad)).unflatten(-1, (-1, 32))
    diff, most = blocks((got - want).abs()).amax(-1), blocks(want.abs()).amax(-1)
    assert (diff <= 0.5 * most).all()


def _check_values(m, cfg, cache, xs, dev, dtype):
    """cache.cmp's values are those of each sequence's own NSAKVCache (and the rest of the state is)."""
    for b, c in enumerate(_check_state(m, cfg, cache, xs, dev, dtype)):
        a = c.n_act
        _, v4 = _held(cache, cache._blocks, cache.cmp, b, a)
        _near(v4, ref.quantized(c.V_cmp[0, :, :a].float().cpu()))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("page,kw", [(16, {}), (64, dict(n_heads=16, n_kv_groups=1, use_bias=True)), (16, dict(l=40, d=8, l_prime=16)),
                                     (32, dict(head_dim_qk=48, head_dim_v=40, l=16, d=8, l_prime=16)),
                                     (16, dict(l=16, d=8, l_prime=16, head_dim_qk=192, head_dim_v=128, n_heads=4))])
@torch.no_grad()
def test_compressed_values_are_the_layers(dev, dtype, page, kw):
    """Prompts in pieces, blocks that single tokens complete (in the step's call and in calls of their own),
    and a request in a released one's place."""
    cfg = _cfg(**kw)
    torch.manual_seed(0)
    m = NSAAttention(cfg).to(dev, dtype).eval()
    B, D = 3, cfg.d_model
    cache = NSAPagedKVCache(cfg, B, 200, dev, dtype, page_size=page)
    g = torch.Generator().manual_seed(5)
    xs = [torch.zeros(0, D, device=dev, dtype=dtype) for _ in range(B)]

    def tokens(T):
        return torch.randn(B, T, D, generator=g).to(dev, dtype)

    def took(x, new):
        for b, n in enumerate(new):
            xs[b] = torch.cat([xs[b], x[b, :n]])

    for new in ([45, 0, 101], [3, 7, 1], [0, 70, 30]):
        x = tokens(max(new))
        m.prefill(x, cache, lengths=new)
        took(x, new)
        _check_values(m, cfg, cache, xs, dev, dtype)
    for i in range(2 * cfg.d + 3):  # every sequence completes blocks
        x, act = tokens(1), [True, i % 3 != 1, i % 2 == 0]
        m.decode(x, cache, output_attentions=i % 4 == 1, active=act)
        took(x, [int(a) for a in act])
    _check_values(m, cfg, cache, xs, dev, dtype)
    cache.release(1)
    xs[1] = xs[1][:0]
    x = tokens(50)
    m.prefill(x, cache, lengths=[2, 50, 0])
    took(x, [2, 50, 0])
    for i in range(cfg.d):
        x = tokens(1)
        m.decode(x, cache)
        took(x, [1] * B)
    _check_values(m, cfg, cache, xs, dev, dtype)


def _check_out(m, cfg, cache, out, info, x, q, z, b, half, auto):
    """Row b of a decode step over cache: out from the 64-bit attention of its query q [B,H,1,dk] (bits that the layer
    uses) over what the pages hold, gates from z [B,H,1,3]."""
    G, H, dk, n = cfg.n_kv_groups, cfg.n_heads, cfg.head_dim_qk, cache.lengths[b]
    p, a = n - 1, cache._blocks.host[b]
    npad = min(1 << max(a - 1, 0).bit_length(), cache.block_ends.shape[0])
    qb = q[b:b + 1].contiguous()
    idx = score_and_select(qb, cache.K_cmp[b:b + 1, :, :, :npad], cache.block_ends[:npad], m.scale, cfg, q_offset=p)
    got_idx = info["selected_indices"][b]
    assert torch.equal(got_idx, idx[0])
    gates = z[b, :, 0].double().cpu()
    gates = torch.softmax(gates, -1) if cfg.gate_mode == "softmax" else torch.sigmoid(gates)
    assert torch.allclose(info["gates"][b, 0].double().cpu(), gates, rtol=4 * half, atol=2.0 ** -20)
    qd = qb[0, :, 0].double().cpu().view(G, H // G, dk)
    mix = mag = torch.zeros(H, cfg.head_dim_v, dtype=torch.float64)
    A, most = 0.0, 0
    for k, (pg, pool) in enumerate(((cache._blocks, cache.cmp), (cache._tokens, cache.sel), (cache._tokens, cache.win))):
        kk, vv = _held(cache, pg, pool, b, a if k == 0 else n)
        o, s_abs = torch.zeros(2, G, H // G, cfg.head_dim_v, dtype=torch.float64)
        for g in range(G):
            if k == 1:
                bl = {i for i in got_idx[g, 0].tolist() if i >= 0}
                rows = sorted(r for i in bl for r in range(i * cfg.l_prime, min((i + 1) * cfg.l_prime, n)))
            else:
                rows = list(range(a)) if k == 0 else list(range(max(0, p - cfg.w + 1), p + 1))
            if rows:
                pr = torch.softmax(qd[g] @ kk[g, rows].T.contiguous() * m.scale, -1)
                o[g], s_abs[g] = pr @ vv[g, rows], pr @ vv[g, rows].abs()
                A = max(A, float((qd[g].abs() @ kk[g, rows].abs().T.contiguous()).max()) * m.scale)
                most = max(most, len(rows))
        mix = mix + gates[:, k:k + 1] * o.view(H, -1)
        mag = mag + gates[:, k:k + 1] * s_abs.view(H, -1)
    W = m.o_proj.weight.double().cpu()
    want = W @ mix.reshape(-1)
    if m.o_proj.bias is not None:
        want += m.o_proj.bias.double().cpu()
    # A weight, the mix and (under autocast) the projection's weight are each off by a half step of their type,
    # relative to sums of absolute values; the output by one of its own; fp32 sums as in paged_ref.bound (the
    # gates' exp and division 16 steps more), the projection's own over its inputs.
    fp32 = (2 * (dk + 16) * A + 2 * most + 80 + W.shape[1]) * 2.0 ** -24
    lim = (1.01 * (2 + auto) * half + fp32) * (W.abs() @ mag.reshape(-1)) + 1.01 * half * want.abs()
    err = (out[b, 0].double().cpu() - want).abs()
    assert (err <= lim).all(), (b, float(err.max()), float((err / lim).max()))


@pytest.mark.parametrize("B,dtype,held,auto,kw", [
    (70, torch.bfloat16, torch.bfloat16, False, {}), (70, torch.float32, torch.float32, False, dict(gate_mode="softmax")),
    (2, torch.float16, torch.float16, False, {}), (3, torch.float32, torch.bfloat16, False, dict(use_bias=True)),
    (3, torch.bfloat16, torch.float32, False, {}), (3, torch.float32, torch.float32, True, {}),
    (3, torch.float32, torch.bfloat16, True, dict(l=8, d=1, l_prime=16))])
@torch.no_grad()
def test_outputs_of_types_and_batches_that_take_other_ways(dev, B, dtype, held, auto, kw):
    """More sequences than a step's call takes, caches of another dtype than the tokens', fp16, autocast, at lengths of
    their own: rows of the output against 64-bit attention over what the pages hold, the rows in the pages and
    the compressed values against the layer's own cache."""
    cfg = _cfg(**kw)
    torch.manual_seed(0)
    m = NSAAttention(cfg).to(dev, dtype).eval()
    g = torch.Generator().manual_seed(7)
    a = NSAPagedKVCache(cfg, B, 100, dev, held, page_size=16)
    x = torch.randn(B, 90, cfg.d_model, generator=g).to(dev, dtype)
    lens = [1 + int(n) for n in torch.randint(0, 60, (B,), generator=g)]
    xs = [x[b, :n] for b, n in enumerate(lens)]
    look = sorted({0, 1, B // 2, B - 1})
    work = torch.bfloat16 if auto else dtype
    half = torch.finfo(work).eps / 2
    with torch.autocast("cuda", torch.bfloat16, enabled=auto):
        m.prefill(x, a, lengths=lens)
        for i in range(25):
            t = torch.randn(B, 1, cfg.d_model, generator=g).to(dev, dtype)
            act = (torch.rand(B, generator=g) < 0.8).tolist()
            q, z, _ = m._paged_inputs(t)
            # (apart from how it is made: operands under autocast and the output rounded, sums of fp32)
            xd, wd = t[:, 0].double().cpu(), m.q_proj.weight.double().cpu()
            want = xd @ wd.T + (0 if m.q_proj.bias is None else m.q_proj.bias.double().cpu())
            lim = 1.01 * half * want.abs() + ((3 if auto else 0) * half + cfg.d_model * 2.0 ** -24) * (xd.abs() @ wd.abs().T + 1)
            assert ((q.transpose(1, 2).flatten(2)[:, 0].double().cpu() - want).abs() <= lim).all()
            assert q.dtype == work and z.dtype == work
            att = i % 4 != 3
            out, info = m.decode(t, a, output_attentions=att, active=act)
            assert out.isfinite().all() and out.dtype == (torch.bfloat16 if auto else dtype)
            xs = [torch.cat([s, t[b]]) if act[b] else s for b, s in enumerate(xs)]
            if att:
                for b in look:
                    if act[b]:
                        _check_out(m, cfg, a, out, info, t, q, z, b, half, auto)
        assert a.lengths == [len(s) for s in xs] == a._tokens.lengths.tolist()
        for b in look:
            own = _single(m, cfg, xs[b], dev, held)
            rows = _single(m, cfg, xs[b], dev, torch.float32)  # the projections as they come: the pages take those
            n, nc = len(xs[b]), own.n_act
            for pool, kk, vv in ((a.sel, rows.k_sel, rows.v_sel), (a.win, rows.k_win, rows.v_win)):
                for got, r in zip(_held(a, a._tokens, pool, b, n), (kk, vv)):
                    _near(got, ref.quantized(r[0, :, :n].float().cpu()))
            assert a._blocks.host[b] == nc
            _near(_held(a, a._blocks, a.cmp, b, nc)[1], ref.quantized(own.V_cmp[0, :, :nc].float().cpu()))
