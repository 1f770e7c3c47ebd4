"""The 8-bit cache's refusals, which are checked before any GPU call, and its
number format's restatement."""
import ctypes

import numpy as np
import pytest

import kv8_ref as ref

FAKE = 1 << 20  # an aligned address that no refused call may read


def _cache(cbis, **kw):
    c = cbis.Kv8Cache(8, 32, 16, 10, FAKE, FAKE)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def _desc(cbis, **kw):
    a = cbis.Kv8AttnDesc()
    a.cache = _cache(cbis, **kw.pop("cache", {}))
    a.n_rows, a.n_heads = 4, 16
    a.q_dtype, a.q, a.ldq = cbis.F32, FAKE, 512
    a.out_dtype, a.out, a.ldo = cbis.BF16, FAKE, 512
    a.block_table, a.bt_stride, a.row_pos = FAKE, 8, FAKE
    for k, v in kw.items():
        setattr(a, k, v)
    return a


INVALID, UNSUPPORTED, WORKSPACE = 1, 2, 3


def test_page_bytes(cbis):
    f = cbis.kernels().cbis_kv8_page_bytes
    assert f(8, 32, 16) == 16 * 8 * 33 and f(1, 128, 64) == 64 * 129 and f(3, 64, 32) == 32 * 3 * 65
    for bad in ((0, 32, 16), (8, 48, 16), (8, 256, 16), (8, 32, 8), (8, 32, 24), (8, 32, 0), (-1, 32, 16)):
        assert f(*bad) == 0


@pytest.mark.parametrize("fn", ["cbis_kv8_scatter", "cbis_kv8_gather"])
def test_row_calls_refuse(cbis, fn):
    f = getattr(cbis.kernels(), fn)

    def call(cache=None, n=4, dt=0, k=FAKE, ldk=256, v=FAKE, ldv=256, page=FAKE, off=FAKE):
        c = _cache(cbis, **(cache or {}))
        rc = f(ctypes.byref(c), n, dt, k, ldk, v, ldv, page, off, None)
        if rc:
            assert fn in cbis.kernels().cbis_last_error().decode()
        return rc

    assert f(None, 4, 0, FAKE, 256, FAKE, 256, FAKE, FAKE, None) == INVALID
    assert call(n=0) == 0
    assert call(n=-1) == INVALID
    assert call(dt=2) == UNSUPPORTED
    for bad in ({"head_dim": 48}, {"page_size": 24}, {"page_size": 8}):
        assert call(cache=bad) == UNSUPPORTED
    for bad in ({"n_kv_heads": 0}, {"num_pages": 0}, {"k_pool": None}, {"v_pool": FAKE + 8}):
        assert call(cache=bad) == INVALID
    for bad in ({"k": None}, {"v": None}, {"page": None}, {"off": None}, {"ldk": 255}, {"ldv": 0}, {"k": FAKE + 2},
                {"page": FAKE + 2}):
        assert call(**bad) == INVALID


@pytest.mark.parametrize("fn", ["cbis_kv8_attention", "cbis_kv8_chunk_attention"])
def test_attention_refuses(cbis, fn):
    kern = cbis.kernels()
    chunk = "chunk" in fn

    def call(tiles=FAKE, n_tiles=2, **kw):
        a = _desc(cbis, **kw)
        rc = (getattr(kern, fn)(ctypes.byref(a), n_tiles, tiles, None) if chunk
              else getattr(kern, fn)(ctypes.byref(a), None))
        if rc:
            assert fn in kern.cbis_last_error().decode()
        return rc

    null = ctypes.POINTER(cbis.Kv8AttnDesc)()
    assert (getattr(kern, fn)(null, 1, FAKE, None) if chunk else getattr(kern, fn)(null, None)) == INVALID
    assert (call(n_tiles=0) if chunk else call(n_rows=0)) == 0
    for bad in ({"n_heads": 12}, {"n_heads": 0}, {"q": None}, {"out": None}, {"block_table": None}, {"ldq": 511},
                {"ldo": 100}, {"bt_stride": 0}, {"split_tokens": 63}, {"split_tokens": -64}, {"max_kv_len": -1},
                {"q": FAKE + 2}, {"out": FAKE + 1}, {"block_table": FAKE + 1},
                {"cache": {"num_pages": 0}}, {"cache": {"v_pool": None}}):
        assert call(**bad) == INVALID, bad
    for bad in ({"q_dtype": 2}, {"out_dtype": 2}, {"cache": {"head_dim": 96}}, {"cache": {"page_size": 17}}):
        assert call(**bad) == UNSUPPORTED, bad
    if chunk:
        assert call(n_tiles=-1) == INVALID and call(tiles=None) == INVALID and call(tiles=FAKE + 4) == INVALID
    else:
        assert call(n_rows=-1) == INVALID and call(row_pos=None) == INVALID
    # Splits without (enough) workspace.
    assert call(split_tokens=64, max_kv_len=128) == WORKSPACE
    a = _desc(cbis, split_tokens=64, max_kv_len=128)
    need = (kern.cbis_kv8_chunk_attention_workspace_size(ctypes.byref(a), 2) if chunk
            else kern.cbis_kv8_attention_workspace_size(ctypes.byref(a)))
    assert need == (2 * 64 if chunk else 4) * 2 * 16 * 33 * 4
    assert call(split_tokens=64, max_kv_len=128, workspace=FAKE, workspace_bytes=need - 1) == WORKSPACE
    assert call(split_tokens=64, max_kv_len=128, workspace=FAKE + 4, workspace_bytes=need) == INVALID


def test_workspace_size_of_bad_descriptors(cbis):
    kern = cbis.kernels()
    assert kern.cbis_kv8_attention_workspace_size(None) == 0
    assert kern.cbis_kv8_chunk_attention_workspace_size(None, 3) == 0
    for bad in ({"n_heads": 12}, {"cache": {"head_dim": 16}}, {"cache": {"page_size": 0}}, {"cache": {"n_kv_heads": 0}}):
        a = _desc(cbis, **bad)
        assert kern.cbis_kv8_attention_workspace_size(ctypes.byref(a)) == 0
        assert kern.cbis_kv8_chunk_attention_workspace_size(ctypes.byref(a), 3) == 0


def test_format_restatement():
    """The restated format keeps its promises: the scale is the least power of
    two that holds the slice, each value is off by at most half a step."""
    r = np.random.default_rng(0)
    x = (r.standard_normal((2000, 32)) * np.exp2(r.integers(-140, 120, (2000, 1)))).astype(np.float32)
    codes, byte = ref.quantise(x)
    e = byte.astype(int) - 127
    top = np.abs(x.astype(np.float64)).max(-1)
    assert (top <= np.ldexp(448.0, e)).all()
    assert ((top > np.ldexp(448.0, e - 1)) | (e == -126)).all()
    err = np.abs(ref.dequantise(codes, byte) - x)
    small = np.ldexp(1.0, e - 10)[:, None]
    assert (err <= np.maximum(2.0 ** -4 * np.abs(x.astype(np.float64)), small)).all()
    x[0, 3], x[1, 0] = np.nan, np.inf
    codes, byte = ref.quantise(x)
    assert (byte[:2] == 255).all() and (codes[:2] == 0).all() and np.isnan(ref.dequantise(codes, byte)[:2]).all()


def test_host_cache_of_fp8_pages(cbis):
    """PagedKVCache takes kv_dtype fp8 where the pages exist and refuses other
    geometries; its bookkeeping is the other dtypes'."""
    c = cbis.PagedKVCache(2, 8, 16, 3, 64, "fp8", alloc_device=False)
    s = c.allocate_sequence()
    assert c.ensure_capacity(s, 40) and c.pages(s) == [0, 1, 2] and c.num_free_pages() == 5
    c.close()
    for ps, hd in ((8, 32), (24, 32), (16, 48), (16, 16), (16, 256)):
        with pytest.raises(cbis.CbisError, match="fp8 K/V pages"):
            cbis.PagedKVCache(2, 8, ps, 3, hd, "fp8", alloc_device=False)


@pytest.mark.parametrize("heads", [1, 2, 5, 8, 16, 32, 40, 64])
@pytest.mark.parametrize("d", [32, 64, 128])
def test_workspace_bound_without_groups(cbis, heads, d):
    """What a runner sets aside once covers every step's calls: rows (64 to a tile)
    x splits x heads is at most 32768."""
    a = cbis.Kv8AttnDesc()
    a.cache.n_kv_heads, a.cache.head_dim, a.cache.page_size, a.cache.num_pages = heads, d, 16, 1
    a.n_heads, a.bt_stride, a.q_dtype = heads, 1 << 16, cbis.F32
    k = cbis.kernels()
    for out in (cbis.F32, cbis.BF16):
        a.out_dtype = out
        for kv in (1, 500, 1000, 2049, 5000, 10000, 20000, 32768, 100000, 1 << 20):
            a.max_kv_len = kv
            for n in (1, 2, 3, 4, 5, 7, 8, 12, 16, 24, 33, 64, 100, 200, 1000):
                a.n_rows = n
                assert k.cbis_kv8_attention_workspace_size(ctypes.byref(a)) <= 32768 * (d + 1) * 4
                assert k.cbis_kv8_chunk_attention_workspace_size(ctypes.byref(a), n) <= 32768 * (d + 1) * 4
