"""CPU tests of the paged 4-bit cache's host side: what the library and the Python calls refuse
before anything is launched, and the tests' own restatement of the format."""
import ctypes

import pytest
import torch

import nsa
import paged_ref as ref
from nsa import _lib

P = ctypes.c_void_p
ONE = P(4096)  # an address that a refused call never reads


def _err():
    return _lib.load().nsa_last_error().decode()


def _tables(n=2, width=4, n_free=8, page=16, rows=2, stride=0, st=4, ptr=ONE):
    return _lib.load().nsa_block_tables(ptr, st, n, width, ptr, ptr, ptr, n_free, ptr, page, rows, stride, *[ptr] * 6, None)


@pytest.mark.parametrize("kw,code", [
    (dict(n=0), 1), (dict(n=4097), 1), (dict(width=0), 1), (dict(n_free=-1), 1), (dict(rows=-1), 1), (dict(page=0), 1),
    (dict(page=8), 1), (dict(page=48), 1), (dict(page=2048), 1), (dict(stride=-1), 1), (dict(stride=2), 1),
    (dict(width=(1 << 26) + 1, st=1 << 27), 1), (dict(st=3), 3), (dict(ptr=None), 1)])
def test_block_tables_refusals(kw, code):
    assert _tables(**kw) == code and _err()


def _pages(**kw):
    a = dict(k=4096, k_scale=4096, v=4096, v_scale=4096, n_pages=4, page_size=16)
    a.update(kw)
    return _lib.Kv4Pages(**a)


@pytest.mark.parametrize("kw,code", [(dict(k=None), 1), (dict(v_scale=None), 1), (dict(n_pages=0), 1), (dict(page_size=24), 1),
                                     (dict(k=4097), 3)])
def test_pool_refusals(kw, code):
    lib, pg = _lib.load(), ctypes.byref(_pages(**kw))
    assert lib.nsa_kv4_store(pg, ONE, 64, 64, ONE, 64, 64, ONE, 1, 1, 64, 64, 0, None) == code
    assert lib.nsa_kv4_load(pg, ONE, 4, 4, ONE, ONE, ONE, 1, 1, 8, 64, 64, 0, None) == code


def test_store_and_load_refusals():
    lib, pg = _lib.load(), ctypes.byref(_pages())
    assert lib.nsa_kv4_store(pg, ONE, 64, 64, ONE, 64, 64, ONE, 1, 1, 64, 64, 7, None) == 1
    assert lib.nsa_kv4_store(pg, ONE, 64, 64, ONE, 64, 64, ONE, -1, 1, 64, 64, 0, None) == 1
    assert lib.nsa_kv4_store(pg, ONE, 65, 64, ONE, 64, 64, ONE, 2, 1, 64, 64, 0, None) == 3
    assert lib.nsa_kv4_store(pg, ONE, 64, 64, ONE, 64, 64, ONE, 2, 1, 48, 48, 0, None) == 2
    assert lib.nsa_kv4_store(pg, None, 64, 64, ONE, 64, 64, ONE, 2, 1, 64, 64, 0, None) == 1
    assert lib.nsa_kv4_store(pg, None, 64, 64, None, 64, 64, None, 0, 1, 64, 64, 0, None) == 0  # nothing to store
    assert lib.nsa_kv4_store(None, ONE, 64, 64, ONE, 64, 64, ONE, 1, 1, 64, 64, 0, None) == 1
    assert lib.nsa_kv4_load(pg, ONE, 4, 0, ONE, ONE, ONE, 1, 1, 8, 64, 64, 0, None) == 1
    assert lib.nsa_kv4_load(pg, ONE, 4, 4, ONE, ONE, ONE, 0, 1, 8, 64, 64, 0, None) == 1
    assert lib.nsa_kv4_load(pg, ONE, 4, 4, ONE, P(4100), ONE, 1, 1, 8, 64, 64, 0, None) == 3
    assert lib.nsa_kv4_load(pg, ONE, 4, 4, ONE, ONE, ONE, 1, 1, 8, 32, 64, 0, None) == 2


_POOL = _pages()


def _attn(**kw):
    a = _lib.Kv4AttnArgs()
    a.q = a.out = a.lengths = 4096
    a.pages[2], a.tables[2], a.stride_table[2], a.table_width[2] = ctypes.addressof(_POOL), 4096, 100, 100
    a.Z, a.H, a.n_kv_groups, a.n_ctx_q, a.head_dim_qk, a.head_dim_v, a.max_length = 2, 4, 2, 1, 64, 64, 4000
    a.l, a.d, a.n_slots, a.block_size_selection, a.window_size, a.gate_act, a.dtype, a.sm_scale = 32, 16, 4, 64, 1500, 0, 0, 1.0
    a.stride_qz = a.stride_oz = 256
    a.stride_qh = a.stride_oh = 64
    for k, v in kw.items():
        if k == "sel":
            a.pages[1], a.tables[1], a.stride_table[1], a.table_width[1] = ctypes.addressof(_POOL), 4096, 4, 4
            if v:
                a.pages[2] = None
        else:
            setattr(a, k, v)
    return a


def test_attention_refusals():
    lib = _lib.load()
    need = lib.nsa_kv4_attn_workspace_size(ctypes.byref(_attn()))
    assert need > 0 and need % 4 == 0
    bad = [dict(dtype=2), dict(Z=0), dict(H=3), dict(n_ctx_q=0), dict(max_length=0), dict(window_size=0), dict(Z=70000),
           dict(gates=4096, gate_act=3), dict(sel=False), dict(sel=True, n_slots=65), dict(sel=True, n_slots=0),
           dict(sel=True, block_size_selection=24), dict(sel=True, block_size_selection=0)]
    for kw in bad:
        a = _attn(**kw)
        assert lib.nsa_kv4_attn_workspace_size(ctypes.byref(a)) == 0, kw
        assert lib.nsa_kv4_attn(ctypes.byref(a), ONE, 1 << 30, None) == 1 and _err(), kw
    assert lib.nsa_kv4_attn(ctypes.byref(_attn(head_dim_qk=48)), ONE, 1 << 30, None) == 2
    assert lib.nsa_kv4_attn(ctypes.byref(_attn(stride_qh=65)), ONE, 1 << 30, None) == 3
    assert lib.nsa_kv4_attn(ctypes.byref(_attn(q=None)), ONE, 1 << 30, None) == 1
    assert lib.nsa_kv4_attn(ctypes.byref(_attn(sel=True, indices=None)), ONE, 1 << 30, None) == 1
    assert lib.nsa_kv4_attn(ctypes.byref(_attn()), ONE, need - 1, None) == 4
    assert lib.nsa_kv4_attn(ctypes.byref(_attn()), P(4104), need, None) == 4
    a = _attn()
    a.tables[2] = None
    assert lib.nsa_kv4_attn(ctypes.byref(a), ONE, need, None) == 1
    a = _attn()
    a.table_width[2] = 1 << 30
    assert lib.nsa_kv4_attn(ctypes.byref(a), ONE, 1 << 40, None) == 1


def test_pool_tensors_are_checked():
    kv = nsa.PagedKV4.empty(3, 16, 2, 80, 48, "cpu")
    assert kv.kernel_dims == (128, 128) and kv.head_dims == (80, 48) and kv.k.shape == (3, 2, 16, 64)
    k, ks, v, vs = kv.k, kv.k_scale, kv.v, kv.v_scale
    assert nsa.PagedKV4(k, ks, v, vs).head_dims == (128, 128)
    for bad in ((k.int(), ks, v, vs), (k[:, :1], ks, v, vs), (k, ks[..., :2], v, vs), (k[..., ::2], ks, v, vs), (v[..., :32].contiguous(), ks, v, vs),
                (k[:, :, :10].contiguous(), ks[:, :, :10].contiguous(), v[:, :, :10].contiguous(), vs[:, :, :10].contiguous()),
                (k[:0], ks[:0], v[:0], vs[:0])):
        with pytest.raises(ValueError):
            nsa.PagedKV4(*bad)
    with pytest.raises(ValueError):
        nsa.PagedKV4(k, ks, v, vs, (130, 48))
    with pytest.raises(ValueError):
        nsa.PagedKV4.empty(3, 16, 2, 256, 128, "cpu")


def test_cache_refusals():
    def make(batch=2, max_len=100, page_size=16, n_pages=None, **kw):
        cfg = nsa.NSAConfig(**{**dict(d_model=64, head_dim_qk=32, head_dim_v=32, n_heads=4, n_kv_groups=2), **kw})
        return nsa.NSAPagedKVCache(cfg, batch, max_len, "cpu", torch.float32, page_size, n_pages)

    c = make()
    assert c.sel.n_pages == 14 and c.cmp.n_pages == 2 and c.lengths == [0, 0]
    for kw in (dict(batch=0), dict(batch=4097), dict(max_len=0), dict(page_size=20), dict(n_pages=0), dict(l_prime=24, d=8, l=16),
               dict(n=65, n_fixed=3), dict(n_heads=130), dict(max_len=16 * 4096 + 32), dict(head_dim_qk=256)):
        with pytest.raises(ValueError):
            make(**kw)
    make(max_len=16 * 4095 + 32, n_pages=3)
    for new in ([1], [101, 0], [0, -1]):
        with pytest.raises(ValueError):
            c.check(new)
    with pytest.raises(ValueError, match="pages"):
        make(n_pages=3).check([40, 16])
    with pytest.raises(AttributeError):
        c.sel.k = c.sel.k


def test_packed_arguments_are_the_c_struct():
    """The packed form of nsa_kv4_attn_args has each field where ctypes (and C) have it."""
    from nsa import paged

    for packed, cls in ((paged._ATTN, _lib.Kv4AttnArgs), (paged._STEP, _lib.PagedStepArgs), (paged._BLOCKS, _lib.PagedBlocksArgs)):
        types = [t for _, f in cls._fields_ for t in ([f._type_] * f._length_ if hasattr(f, "_length_") else [f])]
        vals = [0.5 if t is ctypes.c_float else 1 + i for i, t in enumerate(types)]
        a = cls.from_buffer_copy(packed.pack(*vals).ljust(ctypes.sizeof(cls), b"\0"))
        got = []
        for name, _ in a._fields_:
            x = getattr(a, name)
            got += list(x) if hasattr(x, "__len__") else [x]
        assert got == vals and packed.size <= ctypes.sizeof(cls)


def test_step_refusals():
    def step(**kw):
        a = _lib.PagedStepArgs()
        for n in ("x", "tables", "cmp_tables", "lengths", "new_tokens", "free_pages", "used", "state", "tail", "k_cmp", "block_ends",
                  "out"):
            setattr(a, n, 4096)
        for i in range(3):
            a.pages[i] = ctypes.addressof(_POOL)
        for n, v in dict(Z=2, H=4, n_kv_groups=2, d_model=64, head_dim_qk=64, head_dim_v=64, gate_hidden=32, table_width=4,
                         cmp_table_width=4, n_free=4, n_blocks=8, max_length=64, l=32, d=16, l_prime=64, n=4, window_size=8, phases=3,
                         sm_scale=1.0).items():
            setattr(a, n, v)
        for n, v in kw.items():
            if n == "page":
                a.pages[v] = None
            else:
                setattr(a, n, v)
        return a

    lib = _lib.load()
    need = lib.nsa_paged_step_workspace_size(ctypes.byref(step()))
    assert need > 0
    for kw in (dict(Z=0), dict(Z=65), dict(H=3), dict(dtype=3), dict(n_blocks=0), dict(l=0), dict(n=0), dict(page=1), dict(phases=0),
               dict(phases=4), dict(tail=None), dict(used=None)):
        assert lib.nsa_paged_step(ctypes.byref(step(**kw)), ONE, 1 << 30, None) == 1 and _err(), kw
    assert lib.nsa_paged_step(ctypes.byref(step(head_dim_qk=48)), ONE, 1 << 30, None) == 2
    assert lib.nsa_paged_step(ctypes.byref(step(tail=4100)), ONE, 1 << 30, None) == 3
    assert lib.nsa_paged_step(ctypes.byref(step()), ONE, need - 1, None) == 4
    assert lib.nsa_paged_step(None, ONE, need, None) == 1
    bad, good = _blocks_args(closing=0), _blocks_args()
    assert lib.nsa_paged_step(ctypes.byref(step(blocks=ctypes.addressof(bad))), ONE, 1 << 30, None) == 1
    more = lib.nsa_paged_step_workspace_size(ctypes.byref(step(blocks=ctypes.addressof(good))))
    assert more >= need + lib.nsa_paged_blocks_workspace_size(ctypes.byref(good))


def _blocks_args(**kw):
    a = _lib.PagedBlocksArgs()
    for n in ("tables", "token_lengths", "lengths", "free_pages", "used", "state", "tail", "k_cmp", "E", "W1", "W2"):
        setattr(a, n, 4096)
    a.pages = ctypes.addressof(_POOL)
    for n, v in {**dict(Z=2, n_kv_groups=2, head_dim_qk=64, head_dim_v=64, table_width=4, n_free=4, l=32, closing=3), **kw}.items():
        setattr(a, n, v)
    return a


def test_blocks_refusals():
    lib, args = _lib.load(), _blocks_args
    need = lib.nsa_paged_blocks_workspace_size(ctypes.byref(args()))
    assert need > 0
    for kw in (dict(Z=0), dict(Z=65), dict(n_kv_groups=0), dict(dtype=3), dict(tail=None), dict(used=None), dict(W2=None), dict(pages=None)):
        a = args(**kw)
        assert lib.nsa_paged_blocks(ctypes.byref(a), ONE, 1 << 30, None) == 1 and _err(), kw
    for closing in (0, 4, 1 << 63):
        a = args(closing=closing)
        assert lib.nsa_paged_blocks(ctypes.byref(a), ONE, 1 << 30, None) == 1 and _err(), closing
    for kw in (dict(head_dim_qk=32, head_dim_v=32), dict(head_dim_qk=96), dict(l=128), dict(l=6), dict(l=0)):
        a = args(**kw)
        assert lib.nsa_paged_blocks(ctypes.byref(a), ONE, 1 << 30, None) == 2 and _err(), kw
    for kw in (dict(tail=4100), dict(k_cmp=4100), dict(stride_kn=6), dict(W1=4098)):
        a = args(**kw)
        assert lib.nsa_paged_blocks(ctypes.byref(a), ONE, 1 << 30, None) == 3 and _err(), kw
    assert lib.nsa_paged_blocks(ctypes.byref(args()), ONE, need - 1, None) == 4
    assert lib.nsa_paged_blocks(ctypes.byref(args()), None, need, None) == 4
    assert lib.nsa_paged_blocks(None, ONE, need, None) == 1


def test_calls_want_the_gpu():
    kv = nsa.PagedKV4.empty(3, 16, 2, 64, 64, "cpu")
    t, n = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    for f in (lambda: nsa.build_block_tables(t, n, n, n, n, 16, 1), lambda: nsa.load_kv4(kv, t, n, 4),
              lambda: nsa.store_kv4(kv, torch.zeros(1, 2, 64), torch.zeros(1, 2, 64), torch.zeros(1, dtype=torch.int64)),
              lambda: nsa.attend_kv4(torch.zeros(1, 2, 1, 64), kv, t, n, 1.0)):
        with pytest.raises(RuntimeError, match="GPU"):
            f()


def test_restated_format():
    x = torch.tensor([[0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.9] + [0.0] * 24, [1e-3] * 32])
    got = ref.quantized(x)
    assert got[0, :8].tolist() == [0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, 6.0]
    assert abs(got[1, 0].item() - 1e-3) <= 2.0 ** -3 * 1e-3  # a mantissa bit: half a step of 2^-2
    tab, slots, pos, seq, off, lens, info = ref.tables([[7, -1], [-1, -1]], [15, 0], [3, 1], [4, 5, 6], 1, 16, 4, 0)
    assert tab == [[7, 5], [6, -1]] and slots == [7 * 16 + 15, 5 * 16, 5 * 16 + 1, 6 * 16]
    assert pos == [15, 16, 17, 0] and seq == [0, 0, 0, 1] and off == [0, 3, 4] and lens == [18, 1] and info == [4, 3, 0]


def test_release_clears_the_compressed_keys():
    cfg = nsa.NSAConfig(d_model=64, head_dim_qk=32, head_dim_v=32, n_heads=4, n_kv_groups=2)
    c = nsa.NSAPagedKVCache(cfg, 2, 100, "cpu", torch.float32, 16)
    c._K_cmp.fill_(float("nan"))
    c.release(1)
    assert not c.K_cmp[1].any() and c.K_cmp[0].isnan().all()


def test_pools_of_one_table_have_pages_of_one_size():
    cfg = nsa.NSAConfig(d_model=64, head_dim_qk=64, head_dim_v=64, n_heads=4, n_kv_groups=2, n=4)
    cmp, sel, win = (nsa.PagedKV4.empty(3, p, 2, 64, 64, "cpu") for p in (64, 16, 32))
    t, n = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    q, idx, z = torch.zeros(1, 4, 1, 64), torch.zeros(1, 2, 1, 4, dtype=torch.int64), torch.zeros(1, 4, 1, 3)
    with pytest.raises(ValueError, match="pages of 16 and 32"):
        nsa.nsa_attend_kv4(q, cmp, sel, win, t, t, n, idx, z, 1.0, cfg)
    with pytest.raises(RuntimeError, match="GPU"):  # (the compressed tokens' table is another)
        nsa.nsa_attend_kv4(q, cmp, sel, sel, t, t, n, idx, z, 1.0, cfg)
    lib, a, other = _lib.load(), _attn(sel=False, gates=4096, gate_act=1, indices=4096), _pages(page_size=32)
    assert lib.nsa_kv4_attn_workspace_size(ctypes.byref(a)) > 0
    a.pages[1] = ctypes.addressof(other)
    assert lib.nsa_kv4_attn(ctypes.byref(a), ONE, 1 << 30, None) == 1 and "page sizes" in _err()
    a.tables[1] = 8192  # a table of its own
    assert lib.nsa_kv4_attn_workspace_size(ctypes.byref(a)) > 0


def test_gradients_are_refused():
    cfg = nsa.NSAConfig(d_model=64, head_dim_qk=64, head_dim_v=64, n_heads=4, n_kv_groups=2, n=4)
    kv = nsa.PagedKV4.empty(3, 16, 2, 64, 64, "cpu")
    t, n = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    q, idx, z = torch.zeros(1, 4, 1, 64), torch.zeros(1, 2, 1, 4, dtype=torch.int64), torch.zeros(1, 4, 1, 3)
    rows, slots = torch.zeros(1, 2, 64), torch.zeros(1, dtype=torch.int64)
    calls = {"q": lambda x: nsa.attend_kv4(x(q), kv, t, n, 1.0), "nsa q": lambda x: nsa.nsa_attend_kv4(x(q), kv, kv, kv, t, t, n, idx, z, 1.0, cfg),
             "gates": lambda x: nsa.nsa_attend_kv4(q, kv, kv, kv, t, t, n, idx, x(z), 1.0, cfg),
             "k": lambda x: nsa.store_kv4(kv, x(rows), rows, slots), "v": lambda x: nsa.store_kv4(kv, rows, x(rows), slots)}
    for name, f in calls.items():
        with pytest.raises(RuntimeError, match="not differentiable"):
            f(lambda y: y.clone().requires_grad_())
        with torch.no_grad(), pytest.raises(RuntimeError, match="GPU"):  # (on to the next check)
            f(lambda y: y.clone().requires_grad_())


def test_cache_refuses_what_a_decode_step_would():
    def make(batch=2, max_len=20, **kw):
        cfg = nsa.NSAConfig(**{**dict(d_model=64, head_dim_qk=32, head_dim_v=32, n_heads=16, n_kv_groups=16, l=2, d=2, l_prime=16), **kw})
        return nsa.NSAPagedKVCache(cfg, batch, max_len, "cpu", torch.float32, 16, 1)

    assert make(batch=4095).batch == 4095
    with pytest.raises(ValueError, match="65535 pairs"):
        make(batch=4096)
    d = 1 << 20
    assert make(batch=1, n_heads=2, n_kv_groups=1, head_dim_qk=4, head_dim_v=4, l=16, d=16, l_prime=d).config.l_prime == d
    with pytest.raises(ValueError, match="l_prime"):
        make(batch=1, n_heads=2, n_kv_groups=1, l_prime=d + 16)
    with pytest.raises(ValueError, match="max_len"):
        make(batch=1, n_heads=2, n_kv_groups=1, l=1 << 19, d=1 << 19, l_prime=1 << 19, max_len=(1 << 30) + 1)
