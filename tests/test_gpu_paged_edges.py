"""GPU tests of calls at the edge of the paged 4-bit cache."""
import math

import pytest
import torch

from nsa import NSAAttention, NSAConfig, NSAKVCache, NSAPagedKVCache, PagedKV4, attend_kv4, store_kv4

pytestmark = pytest.mark.gpu


def _cfg(**kw):
    a = dict(d_model=128, head_dim_qk=64, head_dim_v=64, n_heads=8, n_kv_groups=2, l=32, d=16, l_prime=32, n=4, w=40)
    a.update(kw)
    return NSAConfig(**a)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kw", [{}, dict(include_fixed_in_selection=False), dict(l=40, d=8, l_prime=16, include_fixed_in_selection=False)])
@torch.no_grad()
def test_a_released_sequence_leaves_nothing_to_the_next(dev, dtype, kw):
    """A request whose first compressed key overflowed to NaN is released; the next one, shorter than a block, gets
    what it gets in a cache that never held the first."""
    cfg = _cfg(**kw)
    torch.manual_seed(0)
    m = NSAAttention(cfg).to(dev, dtype).eval()
    m.compress_mlp[0].weight.mul_(10)
    g = torch.Generator().manual_seed(1)
    a, b = (NSAPagedKVCache(cfg, 2, 100, dev, dtype, page_size=16) for _ in range(2))
    m.prefill(torch.full((2, 70, cfg.d_model), 3e38, device=dev, dtype=dtype), a, lengths=[0, 70])
    assert a.K_cmp[1, :, :, 0].isnan().any()
    a.release(1)
    x = torch.randn(2, 60, cfg.d_model, generator=g).to(dev, dtype)
    for c in (a, b):
        m.prefill(x, c, lengths=[60, 5])
    for i in range(40):  # over the second sequence's first blocks
        x = torch.randn(2, 1, cfg.d_model, generator=g).to(dev, dtype)
        att = i % 3 != 2
        (oa, ia), (ob, ib) = (m.decode(x, c, output_attentions=att) for c in (a, b))
        assert oa.isfinite().all() and torch.equal(oa, ob), i
        if att:
            assert all(torch.equal(ia[k], ib[k]) for k in ib), i


@torch.no_grad()
def test_widths_that_the_scoring_refuses_leave_the_cache(dev):
    """A decode step whose queries the scoring does not take (rows of no 16 bytes) is refused before its
    token joins the cache."""
    cfg = _cfg(head_dim_qk=36, head_dim_v=32)
    m = NSAAttention(cfg).to(dev, torch.bfloat16).eval()
    cache = NSAPagedKVCache(cfg, 2, 100, dev, torch.bfloat16)
    x = torch.randn(2, 40, cfg.d_model, device=dev, dtype=torch.bfloat16)
    m.prefill(x, cache, lengths=[40, 3])
    before = [t.clone() for t in (cache._tokens.lengths, cache._tokens.tables, cache._tail, cache.sel.k)]
    for att in (False, True):
        with pytest.raises(ValueError, match="16 bytes"):
            m.decode(x[:, :1], cache, output_attentions=att)
    assert cache.lengths == [40, 3]
    assert all(torch.equal(s, t) for s, t in zip(before, (cache._tokens.lengths, cache._tokens.tables, cache._tail, cache.sel.k)))
    # the same widths in fp32 are 16-byte rows
    m = m.float()
    cache = NSAPagedKVCache(cfg, 2, 100, dev, torch.float32)
    m.prefill(x.float(), cache, lengths=[40, 3])
    assert m.decode(x[:, :1].float(), cache)[0].isfinite().all() and cache.lengths == [41, 4]


@torch.no_grad()
def test_window_of_any_size(dev):
    """A window past 32 bits is the whole context, in the step's one call as in calls of their own."""
    torch.manual_seed(0)
    m = NSAAttention(_cfg(w=1 << 40)).to(dev).eval()
    same = NSAAttention(_cfg(w=1000)).to(dev).eval()
    same.load_state_dict(m.state_dict())
    x = torch.randn(2, 61, 128, device=dev)
    outs = []
    for layer in (m, same):
        for att in (False, True):
            cache = NSAPagedKVCache(layer.config, 2, 100, dev, torch.float32)
            layer.prefill(x[:, :60], cache, lengths=[60, 9])
            outs.append(layer.decode(x[:, 60:], cache, output_attentions=att)[0])
    assert all(torch.equal(o, outs[0]) for o in outs)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_off_their_alignment(dev, dtype):
    """Queries, keys and values that start in the middle of 16 bytes: the results of aligned ones."""
    G, H, d, N = 2, 4, 64, 24

    def pair(*shape):  # the same numbers, aligned and one element into a buffer
        n = math.prod(shape)
        buf = torch.randn(n + 1, device=dev).to(dtype)
        off = buf[1:].view(shape)
        assert off.is_contiguous() and off.data_ptr() % 16
        return off.clone(), off

    k, v, q = pair(N, G, d), pair(N, G, d), pair(1, H, 1, d)
    slots, tab = torch.arange(N, device=dev), torch.tensor([[0, 1]], device=dev, dtype=torch.int32)
    lens = torch.tensor([N], device=dev, dtype=torch.int32)
    pools = [PagedKV4.empty(2, 16, G, d, d, dev) for _ in range(2)]
    for i, kv in enumerate(pools):
        store_kv4(kv, k[i], v[i], slots)
    assert all(torch.equal(s, t) for s, t in zip(pools[0]._tensors, pools[1]._tensors))
    a, b = (attend_kv4(q[i], pools[0], tab, lens, 0.125) for i in range(2))
    assert a.any() and torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@torch.no_grad()
def test_tokens_off_their_alignment(dev, dtype):
    """A token's rows that start in the middle of 16 bytes: the step of aligned ones, in either cache."""
    cfg = _cfg()
    torch.manual_seed(0)
    m = NSAAttention(cfg).to(dev, dtype).eval()
    x = torch.randn(2, 45, cfg.d_model, device=dev, dtype=dtype)
    buf = torch.empty(2 * cfg.d_model + 1, device=dev, dtype=dtype)
    t = buf[1:].view(2, 1, -1).copy_(x[:, :1])
    assert t.is_contiguous() and t.data_ptr() % 16
    for make in (NSAKVCache, NSAPagedKVCache):
        for att in (False, True):
            caches = [make(cfg, 2, 100, dev, dtype) for _ in range(2)]
            outs = []
            for c, token in zip(caches, (x[:, :1].contiguous(), t)):
                m.prefill(x, c)
                outs.append(m.decode(token, c, output_attentions=att)[0])
            assert outs[0].any() and torch.equal(*outs)


@torch.no_grad()
def test_release_in_a_capture_is_refused(dev):
    cfg = _cfg()
    m = NSAAttention(cfg).to(dev).eval()
    cache = NSAPagedKVCache(cfg, 2, 100, dev, torch.float32)
    x = torch.randn(2, 40, cfg.d_model, device=dev)
    m.prefill(x, cache)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="captured"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            x.neg()
            cache.release(1)
    torch.cuda.synchronize()
    assert cache.lengths == [40, 40] and cache._tokens.lengths.tolist() == [40, 40]
    cache.release(1)
    assert cache.lengths == [40, 0] and cache._tokens.lengths.tolist() == [40, 0]
