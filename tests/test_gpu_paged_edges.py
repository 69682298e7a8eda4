"""GPU tests of calls at the edge of the paged 4-bit cache."""
import pytest
import torch

from nsa import NSAAttention, NSAConfig, NSAPagedKVCache

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
