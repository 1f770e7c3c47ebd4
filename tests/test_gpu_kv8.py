"""The 8-bit paged K/V cache on the GPU against its 64-bit restatement."""
import ctypes

import numpy as np
import pytest

import kv8_ref as ref
from helpers import ptr, rng, stream, sync

pytestmark = pytest.mark.gpu

TORCH = {"f32": "float32", "bf16": "bfloat16"}


def _t(name):
    import torch
    return getattr(torch, TORCH[name])


def _cache(cbis, kv_heads, d, page_size, kpool, vpool):
    c = cbis.Kv8Cache()
    c.n_kv_heads, c.head_dim, c.page_size = kv_heads, d, page_size
    c.num_pages = kpool.numel() // ref.page_bytes(kv_heads, d, page_size)
    c.k_pool, c.v_pool = ptr(kpool), ptr(vpool)
    return c


def _rows(r, n, kv_heads, d):
    """K or V rows whose size varies from slice to slice, over many binades."""
    x = r.standard_normal((n, kv_heads, d)) * np.exp2(r.integers(-6, 7, (n, kv_heads, 1)))
    return x.astype(np.float32)


def _as(x, dtype, dev, pad=0):
    """[n, w] values on the device with `pad` more elements to a row, and the
    values that the type holds."""
    import torch
    n, w = x.shape
    t = torch.full((n, w + pad), float("nan"), dtype=_t(dtype), device=dev)
    t[:, :w] = torch.from_numpy(x).to(dev).to(_t(dtype))
    return t, t[:, :w].double().cpu().numpy()


# ---------------------------------------------------------------------------
# Write and read back.
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("kv_heads,d,page_size,n,pad", [
    (8, 32, 16, 1, 0), (8, 32, 16, 37, 0), (1, 32, 16, 5, 3), (64, 32, 16, 130, 0), (3, 64, 64, 200, 8),
    (4, 64, 16, 33, 1), (8, 128, 32, 97, 0), (5, 128, 16, 64, 4), (12, 32, 128, 300, 0)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_scatter_then_gather(cbis, dev, kv_heads, d, page_size, n, pad, dtype):
    """Codes and scale bytes equal the restatement's bit for bit in every slot
    written, every other byte stays, idle rows touch nothing; reading back
    gives the codes' values exactly."""
    import torch
    r = rng(kv_heads * 1000 + d + n)
    pages = n // page_size + 9
    size = pages * ref.page_bytes(kv_heads, d, page_size)
    before = r.integers(0, 256, (2, size), dtype=np.uint8)
    slots = r.permutation(pages * page_size)[:n]
    if n > 40:  # the first rows are consecutive tokens, as a prompt's are
        slots = np.concatenate([np.arange(n - 20) + 3, r.permutation(np.arange(n - 17, pages * page_size))[:20]])
    page, off = (slots // page_size).astype(np.int32), (slots % page_size).astype(np.int32)
    idle = np.array([-1, pages, 1 << 30, 0, 0], np.int32), np.array([0, 0, 0, -1, page_size], np.int32)
    if n > 4:
        page[2:2 + 5], off[2:2 + 5] = idle[0][:len(page[2:7])], idle[1][:len(off[2:7])]
    live = np.array([0 <= p < pages and 0 <= o < page_size for p, o in zip(page, off)])
    x = [_rows(r, n, kv_heads, d) for _ in range(2)]
    x[0][0] = 0.0
    x[1][0, 0] = np.float32(1e-42)
    x[1][n // 2, -1] = np.float32(3.4e38)
    x[0][n - 1, 0, 1], x[1][n - 1, -1, d - 1] = np.nan, -np.inf
    with np.errstate(over="ignore"):
        dk, kv = _as(x[0].reshape(n, -1), dtype, dev, pad)
        dv, vv = _as(x[1].reshape(n, -1), dtype, dev, pad)
    pools = [torch.from_numpy(b.copy()).to(dev) for b in before]
    c = _cache(cbis, kv_heads, d, page_size, *pools)
    dp, do = torch.from_numpy(page).to(dev), torch.from_numpy(off).to(dev)
    cbis.check(cbis.kernels().cbis_kv8_scatter(ctypes.byref(c), n, cbis.DTYPES[dtype], ptr(dk), dk.stride(0), ptr(dv),
                                               dv.stride(0), ptr(dp), ptr(do), stream()))
    sync()
    want = before.copy()
    for i in np.flatnonzero(live):
        for w, vals in enumerate((kv, vv)):
            ref.store(want[w], w == 1, kv_heads, d, page_size, page[i], off[i], vals[i].reshape(kv_heads, d))
    for w in range(2):
        assert np.array_equal(pools[w].cpu().numpy(), want[w]), "KV"[w]
    for out_dtype in ("f32", "bf16"):
        got = [torch.full((n, kv_heads * d + pad), 7.0, dtype=_t(out_dtype), device=dev) for _ in range(2)]
        cbis.check(cbis.kernels().cbis_kv8_gather(ctypes.byref(c), n, cbis.DTYPES[out_dtype], ptr(got[0]),
                                                  got[0].stride(0), ptr(got[1]), got[1].stride(0), ptr(dp), ptr(do),
                                                  stream()))
        sync()
        for w in range(2):
            g = got[w].double().cpu().numpy()
            assert (g[:, kv_heads * d:] == 7.0).all() and (g[~live] == 7.0).all()
            for i in np.flatnonzero(live):
                exact = ref.fetch(want[w], w == 1, kv_heads, d, page_size, page[i], off[i]).reshape(-1)
                held = torch.from_numpy(exact).to(_t(out_dtype)).double().numpy()
                assert np.array_equal(g[i, :kv_heads * d], held, equal_nan=True), (w, i)


def test_scatter_rounds_every_half_step(cbis, dev):
    """Every midpoint between two neighbouring codes, and the values just
    beside it, round to nearest even under scale 1 (one element of each slice
    is 448)."""
    import torch
    pos = ref.E4M3[:127]
    mid = (pos[1:] + pos[:-1]) / 2
    x = np.concatenate([pos, mid, mid * (1 + 2.0 ** -23), mid * (1 - 2.0 ** -23)])
    x = np.concatenate([x, -x]).astype(np.float32)
    n = -(-len(x) // 31)
    rows = np.full((n, 32), 448.0, np.float32)
    rows[:, 1:].reshape(-1)  # 31 values to a slice
    flat = np.zeros(n * 31, np.float32)
    flat[:len(x)] = x
    rows[:, 1:] = flat.reshape(n, 31)
    pools = [torch.zeros((n + 15) // 16 * ref.page_bytes(1, 32, 16), dtype=torch.uint8, device=dev) for _ in range(2)]
    c = _cache(cbis, 1, 32, 16, *pools)
    dx = torch.from_numpy(rows).to(dev)
    idx = torch.arange(n, dtype=torch.int32, device=dev)
    page, off = idx // 16, idx % 16
    cbis.check(cbis.kernels().cbis_kv8_scatter(ctypes.byref(c), n, cbis.F32, ptr(dx), 32, ptr(dx), 32, ptr(page),
                                               ptr(off), stream()))
    sync()
    for w in range(2):
        got = pools[w].cpu().numpy()
        want = np.zeros_like(got)
        for i in range(n):
            ref.store(want, w == 1, 1, 32, 16, i // 16, i % 16, rows[i:i + 1])
        assert np.array_equal(got, want)


# ---------------------------------------------------------------------------
# Attention.
# ---------------------------------------------------------------------------

class Case:
    """Sequences of `lengths` tokens cached in random pages; every other byte
    of the pools is 0xFF (e4m3's NaN, and a bad scale)."""

    def __init__(self, cbis, dev, kv_heads, d, page_size, lengths, seed, spread=3):
        import torch
        r = rng(seed)
        self.kv_heads, self.d, self.ps, self.lengths = kv_heads, d, page_size, lengths
        need = [-(-n // page_size) for n in lengths]
        pages = sum(need) + 3
        perm = r.permutation(pages)
        pools = np.full((2, pages * ref.page_bytes(kv_heads, d, page_size)), 255, np.uint8)
        self.table = np.full((len(lengths), max(1, max(need)) + 1), -5, np.int32)
        self.kv = []
        at = 0
        for i, n in enumerate(lengths):
            ids = perm[at:at + need[i]]
            at += need[i]
            self.table[i, :len(ids)] = ids
            both = []
            for w in range(2):
                x = r.standard_normal((n, kv_heads, d)) * np.exp2(r.integers(-spread, spread + 1, (n, kv_heads, 1)))
                if w == 0:  # K stays near 1: the scores' spread is what a model's is
                    x = r.standard_normal((n, kv_heads, d)) * np.exp2(r.integers(-1, 2, (n, kv_heads, 1)))
                for t in range(n):
                    ref.store(pools[w], w == 1, kv_heads, d, page_size, ids[t // page_size], t % page_size,
                              x[t].astype(np.float32))
                both.append(np.stack([ref.fetch(pools[w], w == 1, kv_heads, d, page_size, ids[t // page_size],
                                                t % page_size) for t in range(n)])
                            if n else np.zeros((0, kv_heads, d)))
            self.kv.append(both)
        self.pools = [torch.from_numpy(p).to(dev) for p in pools]
        self.cache = _cache(cbis, kv_heads, d, page_size, *self.pools)
        self.d_table = torch.from_numpy(self.table).to(dev)

    def desc(self, cbis, q, q_dtype, out, out_dtype, heads):
        a = cbis.Kv8AttnDesc()
        a.cache = self.cache
        a.n_heads = heads
        a.q_dtype, a.q, a.ldq = cbis.DTYPES[q_dtype], ptr(q), q.stride(0)
        a.out_dtype, a.out, a.ldo = cbis.DTYPES[out_dtype], ptr(out), out.stride(0)
        a.block_table, a.bt_stride = ptr(self.d_table), self.d_table.stride(0)
        return a

    def check(self, got, seq, pos, q, q_dtype, out_dtype, what=""):
        """One row's result against 64 bits."""
        n = max(0, pos + 1)
        k, v = (x[:n] for x in self.kv[seq])
        with np.errstate(invalid="ignore"):
            out, mag, big = ref.attend(q, k, v)
        tol = ref.tolerance(out, mag, big, n, self.d, np.nanmax(np.abs(v)) if n else 0.0, q_dtype, out_dtype)
        assert np.array_equal(np.isnan(out), np.isnan(got)), what
        fine = ~np.isnan(out)
        worst = (np.abs(got - out) / np.maximum(tol, 1e-300))[fine]
        assert (np.abs(got - out)[fine] <= tol[fine]).all(), (what, seq, pos, worst.max())


def _workspace(a, nbytes, dev):
    import torch
    w = torch.full((max(16, nbytes),), 255, dtype=torch.uint8, device=dev)
    a.workspace, a.workspace_bytes = ptr(w), nbytes
    return w


DTYPES = [("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16"), ("bf16", "f32")]
HEADS = [(8, 8, 32), (64, 64, 32), (5, 5, 32), (20, 20, 64), (12, 4, 64), (32, 8, 128), (28, 4, 128), (40, 2, 64),
         (17, 1, 128), (3, 3, 128)]
LENGTHS = [1, 200, 16, 17, 0, 63, 64, 65, 15, 130, 449, 2]


@pytest.mark.parametrize("heads,kv_heads,d", HEADS)
@pytest.mark.parametrize("q_dtype,out_dtype", DTYPES)
def test_decode(cbis, dev, heads, kv_heads, d, q_dtype, out_dtype):
    """Rows of every length at once, through a row list and a row -> sequence
    map, whole and in splits; rows that are not listed stay; padded strides."""
    import torch
    c = Case(cbis, dev, kv_heads, d, 16, LENGTHS, seed=heads + d)
    r = rng(5)
    n, w = len(LENGTHS), heads * d
    pad = 8 if heads % 2 == 0 else 3  # 3: rows off every vector's alignment
    q, qv = _as(r.standard_normal((n + 2, w)).astype(np.float32), q_dtype, dev, pad)
    rows = np.concatenate([np.arange(n - 1, 1, -1), [1]]).astype(np.int32) + 1  # rows 2 .. n; 0, 1 and n + 1 stay
    seq = np.concatenate([[0], r.permutation(n), [0]]).astype(np.int32)
    pos = np.array([LENGTHS[s] - 1 for s in seq], np.int32)
    d_rows, d_seq, d_pos = (torch.from_numpy(x).to(dev) for x in (rows, seq, pos))
    first = None
    for split, max_kv in ((0, 449), (64, 449), (128, 0), (64, 100)):
        out = torch.full((n + 2, w + pad), 7.0, dtype=_t(out_dtype), device=dev)
        a = c.desc(cbis, q, q_dtype, out, out_dtype, heads)
        a.n_rows, a.rows, a.row_bt, a.row_pos = len(rows), ptr(d_rows), ptr(d_seq), ptr(d_pos)
        a.max_kv_len, a.split_tokens = max_kv, split
        need = cbis.kernels().cbis_kv8_attention_workspace_size(ctypes.byref(a))
        assert (need > 0) == (split != 0) or split == 0
        ws = _workspace(a, need, dev)
        cbis.check(cbis.kernels().cbis_kv8_attention(ctypes.byref(a), stream()))
        sync()
        got = out.double().cpu().numpy()
        assert (got[:, w:] == 7.0).all()
        for i in range(n + 2):
            if i not in rows:
                assert (got[i] == 7.0).all()
                continue
            c.check(got[i, :w].reshape(heads, d), seq[i], pos[i], qv[i].reshape(heads, d), q_dtype, out_dtype,
                    f"split {split} max {max_kv}")
            if pos[i] < 0:
                assert (got[i, :w] == 0).all()
        del ws
        again = out.clone()
        _workspace(a, need, dev)
        ws = _workspace(a, need, dev)
        cbis.check(cbis.kernels().cbis_kv8_attention(ctypes.byref(a), stream()))
        sync()
        assert torch.equal(again.view(torch.int16 if out_dtype == "bf16" else torch.int32),
                           out.view(torch.int16 if out_dtype == "bf16" else torch.int32))
        first = again if first is None else first


@pytest.mark.parametrize("page_size", [16, 32, 128])
def test_decode_page_sizes_and_long_rows(cbis, dev, page_size):
    c = Case(cbis, dev, 2, 32, page_size, [2500, 1025, 4], seed=page_size)
    import torch
    q, qv = _as(rng(1).standard_normal((3, 8 * 32)).astype(np.float32), "f32", dev)
    pos = np.array([2499, 1024, 3], np.int32)
    d_pos = torch.from_numpy(pos).to(dev)
    out = torch.empty((3, 8 * 32), device=dev)
    a = c.desc(cbis, q, "f32", out, "f32", 8)
    a.n_rows, a.row_pos, a.max_kv_len = 3, ptr(d_pos), 2500
    ws = _workspace(a, cbis.kernels().cbis_kv8_attention_workspace_size(ctypes.byref(a)), dev)
    cbis.check(cbis.kernels().cbis_kv8_attention(ctypes.byref(a), stream()))
    sync()
    del ws
    for i in range(3):
        c.check(out[i].double().cpu().numpy().reshape(8, 32), i, pos[i], qv[i].reshape(8, 32), "f32", "f32")


TILES = [[(0, 1, 0, 0)], [(0, 64, 0, 0), (64, 36, 0, 64)], [(0, 7, 0, 100), (7, 64, 1, 130), (71, 3, 1, 194)],
         [(2, 5, 0, -2), (7, 17, 1, 15)], [(0, 64, 0, 386), (64, 63, 1, 386)]]


@pytest.mark.parametrize("heads,kv_heads,d", HEADS)
@pytest.mark.parametrize("q_dtype,out_dtype", DTYPES)
def test_chunk(cbis, dev, heads, kv_heads, d, q_dtype, out_dtype):
    """Tiles of every kind, whole and in splits: a single row, rows that start
    before position 0, tiles that end inside a cache tile, rows of no tile."""
    import torch
    c = Case(cbis, dev, kv_heads, d, 16, [450, 449], seed=heads + d + 1)
    w = heads * d
    r = rng(6)
    pad = 8 if heads % 2 == 0 else 3
    for k, tiles in enumerate(TILES):
        n = max(t[0] + t[1] for t in tiles) + 2
        q, qv = _as(r.standard_normal((n, w)).astype(np.float32), q_dtype, dev, pad)
        d_tiles = torch.tensor(tiles, dtype=torch.int32, device=dev)
        seq_pos = {t[0] + i: (t[2], t[3] + i) for t in tiles for i in range(t[1])}
        for split, max_kv in ((0, 450), (64, 0), (192, 300)):
            if split and k not in (2, 4):
                continue
            out = torch.full((n, w + pad), 7.0, dtype=_t(out_dtype), device=dev)
            a = c.desc(cbis, q, q_dtype, out, out_dtype, heads)
            a.max_kv_len, a.split_tokens = max_kv, split
            need = cbis.kernels().cbis_kv8_chunk_attention_workspace_size(ctypes.byref(a), len(tiles))
            ws = _workspace(a, need, dev)
            cbis.check(cbis.kernels().cbis_kv8_chunk_attention(ctypes.byref(a), len(tiles), ptr(d_tiles), stream()))
            sync()
            del ws
            got = out.double().cpu().numpy()
            assert (got[:, w:] == 7.0).all()
            some = set(r.choice(n, min(n, 24), replace=False)) | {t[0] + t[1] - 1 for t in tiles} | {t[0] for t in tiles}
            for i in range(n):
                if i not in seq_pos:
                    assert (got[i] == 7.0).all()
                elif i in some:
                    c.check(got[i, :w].reshape(heads, d), *seq_pos[i], qv[i].reshape(heads, d), q_dtype, out_dtype,
                            f"tiles {k} split {split}")


@pytest.mark.parametrize("heads,kv_heads,d", [(8, 8, 32), (8, 2, 128)])
@pytest.mark.parametrize("which", [0, 1], ids=["K", "V"])
def test_nan_slices_stay_with_their_head_and_rows(cbis, dev, heads, kv_heads, d, which):
    """A K or V slice of NaN (token 70, kv head 1) makes NaN of that kv head's
    heads in the rows that see the token, and of nothing else."""
    import torch
    c = Case(cbis, dev, kv_heads, d, 16, [100], seed=3)
    pool = c.pools[which].cpu().numpy()
    code, byte = ref.slot_index(kv_heads, d, 16, which == 1, c.table[0, 70 // 16], 70 % 16)
    pool[code[1]], pool[byte[1]] = 0, 255
    c.pools[which].copy_(torch.from_numpy(pool))
    c.kv[0][which][70, 1] = np.nan
    w = heads * d
    q, qv = _as(rng(2).standard_normal((100, w)).astype(np.float32), "f32", dev)
    pos = torch.arange(100, dtype=torch.int32, device=dev)
    zero = torch.zeros(100, dtype=torch.int32, device=dev)
    for form in ("decode", "decode split", "chunk", "chunk split"):
        out = torch.empty((100, w), device=dev)
        a = c.desc(cbis, q, "f32", out, "f32", heads)
        a.n_rows, a.row_bt, a.row_pos = 100, ptr(zero), ptr(pos)
        a.split_tokens = 64 if "split" in form else 0
        tiles = torch.tensor([(0, 64, 0, 0), (64, 36, 0, 64)], dtype=torch.int32, device=dev)
        k = cbis.kernels()
        if "decode" in form:
            ws = _workspace(a, k.cbis_kv8_attention_workspace_size(ctypes.byref(a)), dev)
            cbis.check(k.cbis_kv8_attention(ctypes.byref(a), stream()))
        else:
            ws = _workspace(a, k.cbis_kv8_chunk_attention_workspace_size(ctypes.byref(a), 2), dev)
            cbis.check(k.cbis_kv8_chunk_attention(ctypes.byref(a), 2, ptr(tiles), stream()))
        sync()
        del ws
        got = out.double().cpu().numpy().reshape(100, heads, d)
        for i in (0, 40, 64, 69, 70, 71, 99):
            c.check(got[i], 0, i, qv[i].reshape(heads, d), "f32", "f32", form)
        assert np.isnan(got[70:, heads // kv_heads]).all() and not np.isnan(got[:70]).any(), form


def test_pool_past_32_bits(cbis, dev):
    """Pages whose byte offsets pass 2^32 and 2^31 entries, in every call."""
    import torch
    kv_heads, d = 8, 128
    pb = ref.page_bytes(kv_heads, d, 16)
    pages = (1 << 32) // pb + 40
    pools = [torch.empty(pages * pb, dtype=torch.uint8, device=dev) for _ in range(2)]
    c = _cache(cbis, kv_heads, d, 16, *pools)
    ids = np.array([pages - 1, (1 << 31) // pb + 1, pages - 7], np.int32)
    n = 45
    r = rng(9)
    x = [_rows(r, n, kv_heads, d) for _ in range(2)]
    dk, dv = (torch.from_numpy(v.reshape(n, -1)).to(dev) for v in x)
    t = np.arange(n)
    page = torch.from_numpy(ids[t // 16]).to(dev)
    off = torch.from_numpy((t % 16).astype(np.int32)).to(dev)
    k = cbis.kernels()
    cbis.check(k.cbis_kv8_scatter(ctypes.byref(c), n, cbis.F32, ptr(dk), dk.stride(0), ptr(dv), dv.stride(0), ptr(page),
                                  ptr(off), stream()))
    back = [torch.empty_like(dk) for _ in range(2)]
    cbis.check(k.cbis_kv8_gather(ctypes.byref(c), n, cbis.F32, ptr(back[0]), dk.stride(0), ptr(back[1]), dk.stride(0),
                                 ptr(page), ptr(off), stream()))
    sync()
    held = []
    for w in range(2):
        held.append(ref.dequantise(*ref.quantise(x[w])))
        assert np.array_equal(back[w].double().cpu().numpy().reshape(n, kv_heads, d), held[w])
    q, qv = _as(r.standard_normal((n, 16 * d)).astype(np.float32), "f32", dev)
    table = torch.from_numpy(ids[None]).to(dev)
    zero = torch.zeros(n, dtype=torch.int32, device=dev)
    pos = torch.arange(n, dtype=torch.int32, device=dev)
    tiles = torch.tensor([(0, n, 0, 0)], dtype=torch.int32, device=dev)
    for form in ("decode", "chunk"):
        out = torch.empty((n, 16 * d), device=dev)
        a = cbis.Kv8AttnDesc()
        a.cache, a.n_heads, a.n_rows = c, 16, n
        a.q, a.ldq, a.out, a.ldo = ptr(q), 16 * d, ptr(out), 16 * d
        a.block_table, a.bt_stride, a.row_bt, a.row_pos = ptr(table), 3, ptr(zero), ptr(pos)
        if form == "decode":
            cbis.check(k.cbis_kv8_attention(ctypes.byref(a), stream()))
        else:
            cbis.check(k.cbis_kv8_chunk_attention(ctypes.byref(a), 1, ptr(tiles), stream()))
        sync()
        got = out.double().cpu().numpy().reshape(n, 16, d)
        for i in (0, 15, 16, 44):
            o, mag, big = ref.attend(qv[i].reshape(16, d), held[0][:i + 1], held[1][:i + 1])
            tol = ref.tolerance(o, mag, big, i + 1, d, np.abs(held[1][:i + 1]).max(), "f32", "f32")
            assert (np.abs(got[i] - o) <= tol).all(), (form, i)


def test_write_then_attend_in_a_graph(cbis, dev):
    """Scatter, decode with splits and chunk attention as a step would run them,
    captured on a stream of its own and replayed with new rows: every replay
    equals the eager calls bit for bit."""
    import torch
    kv_heads, d, heads, n = 4, 64, 8, 40
    c = Case(cbis, dev, kv_heads, d, 16, [200], seed=11)
    r = rng(12)
    width = (heads + 2 * kv_heads) * d
    qkv = torch.empty((n, width), device=dev)
    t = np.arange(160, 160 + n)
    page = torch.from_numpy(c.table[0][t // 16]).to(dev)
    off = torch.from_numpy((t % 16).astype(np.int32)).to(dev)
    pos = torch.from_numpy(t.astype(np.int32)).to(dev)
    zero = torch.zeros(n, dtype=torch.int32, device=dev)
    tiles = torch.tensor([(0, n, 0, 160)], dtype=torch.int32, device=dev)
    outs = [torch.zeros((n, heads * d), dtype=torch.bfloat16, device=dev) for _ in range(2)]
    k = cbis.kernels()
    descs, spaces = [], []
    for i in range(2):
        a = c.desc(cbis, qkv, "f32", outs[i], "bf16", heads)
        a.n_rows, a.row_bt, a.row_pos, a.max_kv_len, a.split_tokens = n, ptr(zero), ptr(pos), 200, 64
        need = (k.cbis_kv8_attention_workspace_size(ctypes.byref(a)) if i == 0
                else k.cbis_kv8_chunk_attention_workspace_size(ctypes.byref(a), 1))
        assert need > 0
        spaces.append(_workspace(a, need, dev))
        descs.append(a)

    def step():
        s = stream()
        cbis.check(k.cbis_kv8_scatter(ctypes.byref(c.cache), n, cbis.F32, ptr(qkv) + 4 * heads * d, width,
                                      ptr(qkv) + 4 * (heads + kv_heads) * d, width, ptr(page), ptr(off), s))
        cbis.check(k.cbis_kv8_attention(ctypes.byref(descs[0]), s))
        cbis.check(k.cbis_kv8_chunk_attention(ctypes.byref(descs[1]), 1, ptr(tiles), s))

    def fresh():
        x = r.standard_normal((n, width)).astype(np.float32)
        qkv.copy_(torch.from_numpy(x))
        return x

    fresh()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    for _ in range(4):
        x = fresh()
        g.replay()
        sync()
        replayed = [o.clone() for o in outs]
        for s in spaces:
            s.fill_(255)
        step()
        sync()
        for i in range(2):
            assert torch.equal(replayed[i].view(torch.int16), outs[i].view(torch.int16))
        kv = [ref.dequantise(*ref.quantise(x[:, (heads + w * kv_heads) * d:][:, :kv_heads * d].reshape(n, kv_heads, d)))
              for w in range(2)]
        for w in range(2):
            c.kv[0][w][160:] = kv[w]
        for i in (0, 7, n - 1):
            for o in outs:
                c.check(o[i].double().cpu().numpy().reshape(heads, d), 0, 160 + i,
                        x[i, :heads * d].astype(np.float64).reshape(heads, d), "f32", "bf16")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_scatter_extremes(cbis, dev, dtype):
    """Slices at the ends of fp32: subnormals, the largest finite values, maxima
    just below, at and above 448 * 2^e, signed zeros; and back in both types."""
    import torch
    r = rng(21)
    rows = [np.full(64, 3e-39), np.linspace(-1e-41, 1e-38, 64), r.standard_normal(64) * 3e38, np.full(64, -0.0),
            np.full(64, np.finfo(np.float32).max), np.full(64, 1.4e-45), r.standard_normal(64) * 1e-37]
    for e in (-126, -120, -3, 0, 5, 118):
        for m in (1.75, np.nextafter(np.float32(1.75), np.float32(2)), np.nextafter(np.float32(1.75), np.float32(1)),
                  1.7578125, 1.7421875, 1.0, 1.9921875):
            x = r.standard_normal(64) * 0.3
            x[r.integers(64)] = m
            rows.append(np.clip(x, -m, m) * 2.0 ** (e + 8))
    with np.errstate(over="ignore"):
        x = np.clip(np.stack(rows), -3.38e38, 3.38e38).astype(np.float32)
    n = len(x)
    dx, held = _as(x, dtype, dev)
    pools = [torch.zeros((n + 15) // 16 * ref.page_bytes(2, 32, 16), dtype=torch.uint8, device=dev) for _ in range(2)]
    c = _cache(cbis, 2, 32, 16, *pools)
    idx = torch.arange(n, dtype=torch.int32, device=dev)
    page, off = idx // 16, idx % 16
    k = cbis.kernels()
    cbis.check(k.cbis_kv8_scatter(ctypes.byref(c), n, cbis.DTYPES[dtype], ptr(dx), 64, ptr(dx), 64, ptr(page), ptr(off),
                                  stream()))
    back = {d: [torch.empty((n, 64), dtype=_t(d), device=dev) for _ in range(2)] for d in ("f32", "bf16")}
    for d, b in back.items():
        cbis.check(k.cbis_kv8_gather(ctypes.byref(c), n, cbis.DTYPES[d], ptr(b[0]), 64, ptr(b[1]), 64, ptr(page),
                                     ptr(off), stream()))
    sync()
    codes, byte = ref.quantise(held.reshape(n, 2, 32))
    exact = ref.dequantise(codes, byte).reshape(n, 64)
    for w in range(2):
        got = pools[w].cpu().numpy()
        want = np.zeros_like(got)
        for i in range(n):
            ref.store(want, w == 1, 2, 32, 16, i // 16, i % 16, held[i].reshape(2, 32))
        assert np.array_equal(got, want), "KV"[w]
        for d, b in back.items():
            with np.errstate(over="ignore"):
                stored = torch.from_numpy(exact.astype(np.float32)).to(_t(d)).double().numpy()
            assert np.array_equal(b[w].double().cpu().numpy(), stored), ("KV"[w], d)


@pytest.mark.parametrize("heads,kv_heads,d", [(16, 2, 32), (12, 1, 32), (24, 2, 64), (64, 2, 128), (9, 9, 32)])
@pytest.mark.parametrize("q_dtype,out_dtype", [("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16")])
def test_attention_other_groups(cbis, dev, heads, kv_heads, d, q_dtype, out_dtype):
    """Groups of 8, 12, 16 and 32 query heads (one, two or four kv heads to a
    workgroup's columns), every number of waves on a row, 128-token pages, V
    slices over 20 binades; both forms agree with 64 bits."""
    import torch
    c = Case(cbis, dev, kv_heads, d, 128, [700, 31], seed=heads, spread=10)
    w = heads * d
    n = 9
    q, qv = _as(rng(8).standard_normal((n, w)).astype(np.float32), q_dtype, dev)
    seq = np.array([0, 0, 1, 0, 1, 0, 0, 0, 0], np.int32)
    pos = np.array([699, 63, 30, 64, 0, 128, 250, 575, -1], np.int32)
    d_seq, d_pos = torch.from_numpy(seq).to(dev), torch.from_numpy(pos).to(dev)
    k = cbis.kernels()
    for split in (0, 64, 128, 192, 256, 512):
        out = torch.full((n, w), 7.0, dtype=_t(out_dtype), device=dev)
        a = c.desc(cbis, q, q_dtype, out, out_dtype, heads)
        a.n_rows, a.row_bt, a.row_pos, a.max_kv_len, a.split_tokens = n, ptr(d_seq), ptr(d_pos), 700, split
        ws = _workspace(a, k.cbis_kv8_attention_workspace_size(ctypes.byref(a)), dev)
        cbis.check(k.cbis_kv8_attention(ctypes.byref(a), stream()))
        sync()
        got = out.double().cpu().numpy().reshape(n, heads, d)
        for i in range(n):
            c.check(got[i], seq[i], pos[i], qv[i].reshape(heads, d), q_dtype, out_dtype, f"decode split {split}")
        tiles = torch.tensor([(0, 9, 0, 691)], dtype=torch.int32, device=dev)
        a.n_rows = 0
        ws = _workspace(a, k.cbis_kv8_chunk_attention_workspace_size(ctypes.byref(a), 1), dev)
        cbis.check(k.cbis_kv8_chunk_attention(ctypes.byref(a), 1, ptr(tiles), stream()))
        sync()
        del ws
        got = out.double().cpu().numpy().reshape(n, heads, d)
        for i in (0, 4, 8):
            c.check(got[i], 0, 691 + i, qv[i].reshape(heads, d), q_dtype, out_dtype, f"chunk split {split}")


def test_many_rows_and_tiles(cbis, dev):
    """Enough rows and tiles that waves no longer share keys: 700 rows of 8 heads
    of 32 (one wave to a row's heads), and the same rows as tiles."""
    import torch
    c = Case(cbis, dev, 8, 32, 16, [700], seed=33)
    q, qv = _as(rng(3).standard_normal((700, 256)).astype(np.float32), "f32", dev)
    pos = torch.arange(700, dtype=torch.int32, device=dev)
    many = pos.repeat(8)
    zero = torch.zeros(5600, dtype=torch.int32, device=dev)
    rows = (torch.arange(5600, dtype=torch.int32, device=dev) % 700).contiguous()
    tiles = torch.tensor([(at, min(64, 700 - at), 0, at) for at in range(0, 700, 64)] * 12, dtype=torch.int32, device=dev)
    k = cbis.kernels()
    for form in ("decode", "chunk"):
        out = torch.empty((700, 256), dtype=torch.bfloat16, device=dev)
        a = c.desc(cbis, q, "f32", out, "bf16", 8)
        a.row_bt, a.row_pos, a.max_kv_len = ptr(zero), ptr(many), 700
        if form == "decode":
            a.n_rows, a.rows = 5600, ptr(rows)
            assert k.cbis_kv8_attention_workspace_size(ctypes.byref(a)) == 0
            cbis.check(k.cbis_kv8_attention(ctypes.byref(a), stream()))
        else:
            assert k.cbis_kv8_chunk_attention_workspace_size(ctypes.byref(a), len(tiles)) == 0
            cbis.check(k.cbis_kv8_chunk_attention(ctypes.byref(a), len(tiles), ptr(tiles), stream()))
        sync()
        got = out.double().cpu().numpy().reshape(700, 8, 32)
        for i in (0, 15, 16, 63, 64, 300, 639, 640, 699):
            c.check(got[i], 0, i, qv[i].reshape(8, 32), "f32", "bf16", form)


def test_two_streams(cbis, dev):
    """Two attention calls with splits at once on two streams, each with its own
    workspace: the results of the calls alone, bit for bit."""
    import torch
    c = Case(cbis, dev, 4, 64, 16, [500, 300], seed=17)
    k = cbis.kernels()
    calls = []
    for i in range(2):
        q, _ = _as(rng(40 + i).standard_normal((30, 8 * 64)).astype(np.float32), "f32", dev)
        out = torch.empty((30, 8 * 64), device=dev)
        seq = torch.full((30,), i, dtype=torch.int32, device=dev)
        pos = torch.arange(200, 230, dtype=torch.int32, device=dev)
        a = c.desc(cbis, q, "f32", out, "f32", 8)
        a.n_rows, a.row_bt, a.row_pos, a.split_tokens, a.max_kv_len = 30, ptr(seq), ptr(pos), 64, 230
        ws = _workspace(a, k.cbis_kv8_attention_workspace_size(ctypes.byref(a)), dev)
        calls.append((a, out, (q, seq, pos, ws)))
    alone = []
    for a, out, _ in calls:
        cbis.check(k.cbis_kv8_attention(ctypes.byref(a), stream()))
        sync()
        alone.append(out.clone())
        out.zero_()
    streams = [torch.cuda.Stream() for _ in range(2)]
    sync()
    for _ in range(5):
        for (a, _, _), s in zip(calls, streams):
            cbis.check(k.cbis_kv8_attention(ctypes.byref(a), s.cuda_stream))
    sync()
    for (_, out, _), want in zip(calls, alone):
        assert torch.equal(out, want)


@pytest.mark.parametrize("heads,kv_heads,d", [(8, 8, 32), (8, 4, 64), (8, 2, 128)])
def test_positions_past_the_table(cbis, dev, heads, kv_heads, d):
    """A position past the table's 48 tokens, up to the largest int, reads those 48."""
    import torch
    c = Case(cbis, dev, kv_heads, d, 16, [48], seed=51)
    w, top = heads * d, 2**31 - 1
    q, qv = _as(rng(52).standard_normal((6, w)).astype(np.float32), "f32", dev)
    pos = torch.tensor([47, 48, 49, 4000, top - 1, top], dtype=torch.int32, device=dev)
    zero = torch.zeros(6, dtype=torch.int32, device=dev)
    tiles = torch.tensor([(0, 1, 0, 47), (1, 2, 0, 48), (3, 1, 0, 4000), (4, 2, 0, top)], dtype=torch.int32, device=dev)
    k = cbis.kernels()
    for form in ("decode", "chunk"):
        out = torch.empty((6, w), device=dev)
        a = c.desc(cbis, q, "f32", out, "f32", heads)
        a.bt_stride, a.n_rows, a.row_bt, a.row_pos = 3, 6, ptr(zero), ptr(pos)
        if form == "decode":
            ws = _workspace(a, k.cbis_kv8_attention_workspace_size(ctypes.byref(a)), dev)
            cbis.check(k.cbis_kv8_attention(ctypes.byref(a), stream()))
        else:
            ws = _workspace(a, k.cbis_kv8_chunk_attention_workspace_size(ctypes.byref(a), 4), dev)
            cbis.check(k.cbis_kv8_chunk_attention(ctypes.byref(a), 4, ptr(tiles), stream()))
        sync()
        del ws
        got = out.double().cpu().numpy().reshape(6, heads, d)
        for i in range(6):
            c.check(got[i], 0, 47, qv[i].reshape(heads, d), "f32", "f32", form)


@pytest.mark.parametrize("heads,kv_heads,d", [(8, 8, 32), (8, 4, 64), (8, 2, 128)])
@pytest.mark.parametrize("q_dtype,out_dtype", [("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16")])
def test_first_scores_of_minus_infinity(cbis, dev, heads, kv_heads, d, q_dtype, out_dtype):
    """The first 64 keys' scores fall below fp32's range (weight 0), the others' lie
    far below 0 themselves: their softmax is what comes out."""
    import torch
    c = Case(cbis, dev, kv_heads, d, 16, [164], seed=61)
    pool = c.pools[0].cpu().numpy()
    for t in range(164):
        x = np.full((kv_heads, d), -2.0**100 if t < 64 else -2.0**-25, np.float32)
        if t >= 64:  # the scores of the others differ by up to 32 * 3 / 8 / sqrt(d)
            x[:, 0] *= 1 + t % 4 / 8
        ref.store(pool, False, kv_heads, d, 16, c.table[0, t // 16], t % 16, x)
        c.kv[0][0][t] = ref.fetch(pool, False, kv_heads, d, 16, c.table[0, t // 16], t % 16)
    c.pools[0].copy_(torch.from_numpy(pool))
    w = heads * d
    q, qv = _as(np.full((64, w), 2.0**30, np.float32), q_dtype, dev)
    pos = torch.arange(100, 164, dtype=torch.int32, device=dev)
    zero = torch.zeros(64, dtype=torch.int32, device=dev)
    tiles = torch.tensor([(0, 64, 0, 100)], dtype=torch.int32, device=dev)
    k = cbis.kernels()
    for form, split in (("decode", 0), ("decode", 64), ("chunk", 0), ("chunk", 64)):
        out = torch.empty((64, w), dtype=_t(out_dtype), device=dev)
        a = c.desc(cbis, q, q_dtype, out, out_dtype, heads)
        a.n_rows, a.row_bt, a.row_pos, a.split_tokens, a.max_kv_len = 64, ptr(zero), ptr(pos), split, 164
        if form == "decode":
            ws = _workspace(a, k.cbis_kv8_attention_workspace_size(ctypes.byref(a)), dev)
            cbis.check(k.cbis_kv8_attention(ctypes.byref(a), stream()))
        else:
            ws = _workspace(a, k.cbis_kv8_chunk_attention_workspace_size(ctypes.byref(a), 1), dev)
            cbis.check(k.cbis_kv8_chunk_attention(ctypes.byref(a), 1, ptr(tiles), stream()))
        sync()
        del ws
        got = out.double().cpu().numpy().reshape(64, heads, d)
        for i in (0, 27, 28, 40, 63):
            kk, vv = (x[64:100 + i + 1] for x in c.kv[0])
            want, mag, big = ref.attend(qv[i].reshape(heads, d), kk, vv)
            tol = ref.tolerance(want, mag, big, 101 + i, d, np.abs(c.kv[0][1]).max(), q_dtype, out_dtype)
            assert (np.abs(got[i] - want) <= tol).all(), (form, split, i)


@pytest.mark.parametrize("heads,kv_heads,d", [h for h in HEADS if h[2] > 32])
@pytest.mark.parametrize("q_dtype,out_dtype", DTYPES)
def test_chunk_wide_table(cbis, dev, heads, kv_heads, d, q_dtype, out_dtype):
    """Short sequences in a table of 4096 tokens, which is what the call is laid out
    for: its widest workgroups, and splits most of which are empty."""
    import torch
    c = Case(cbis, dev, kv_heads, d, 16, [450, 449], seed=heads + d + 2)
    table = torch.full((2, 256), -5, dtype=torch.int32, device=dev)
    table[:, :c.d_table.shape[1]] = c.d_table
    w = heads * d
    r = rng(7)
    for tiles in (TILES[2], TILES[4]):
        n = max(t[0] + t[1] for t in tiles)
        q, qv = _as(r.standard_normal((n, w)).astype(np.float32), q_dtype, dev)
        d_tiles = torch.tensor(tiles, dtype=torch.int32, device=dev)
        out = torch.full((n, w), 7.0, dtype=_t(out_dtype), device=dev)
        for split in (0, 4096):
            a = c.desc(cbis, q, q_dtype, out, out_dtype, heads)
            a.block_table, a.bt_stride, a.split_tokens = ptr(table), 256, split
            need = cbis.kernels().cbis_kv8_chunk_attention_workspace_size(ctypes.byref(a), len(tiles))
            assert (need == 0) == (split == 4096)
            ws = _workspace(a, need, dev)
            cbis.check(cbis.kernels().cbis_kv8_chunk_attention(ctypes.byref(a), len(tiles), ptr(d_tiles), stream()))
            sync()
            del ws
            got = out.double().cpu().numpy()
            for row, rows, seq, pos in tiles:
                for i in {0, rows // 2, rows - 1}:
                    c.check(got[row + i].reshape(heads, d), seq, pos + i, qv[row + i].reshape(heads, d), q_dtype,
                            out_dtype, f"split {split}")


@pytest.mark.parametrize("heads,kv_heads,d", [(8, 8, 32), (8, 4, 64), (32, 8, 128), (28, 4, 128)])
@pytest.mark.parametrize("first", [20, 48, 4000])
def test_tiles_past_the_table(cbis, dev, heads, kv_heads, d, first):
    """Whole tiles whose rows lie past the table's 48 tokens, which end inside a
    block of 64: each sees those 48, once."""
    import torch
    c = Case(cbis, dev, kv_heads, d, 16, [48], seed=71)
    w = heads * d
    q, qv = _as(rng(72).standard_normal((70, w)).astype(np.float32), "f32", dev)
    tiles = torch.tensor([(0, 64, 0, first), (64, 6, 0, first + 64)], dtype=torch.int32, device=dev)
    out = torch.empty((70, w), device=dev)
    a = c.desc(cbis, q, "f32", out, "f32", heads)
    a.bt_stride = 3
    ws = _workspace(a, cbis.kernels().cbis_kv8_chunk_attention_workspace_size(ctypes.byref(a), 2), dev)
    cbis.check(cbis.kernels().cbis_kv8_chunk_attention(ctypes.byref(a), 2, ptr(tiles), stream()))
    sync()
    del ws
    got = out.double().cpu().numpy().reshape(70, heads, d)
    for i in (0, 1, 15, 16, 27, 28, 31, 32, 33, 47, 63, 64, 69):
        c.check(got[i], 0, min(first + i, 47), qv[i].reshape(heads, d), "f32", "f32", f"row {i}")


@pytest.mark.parametrize("heads,kv_heads,d", [(8, 8, 64), (16, 4, 64), (40, 8, 64), (4, 4, 128), (32, 8, 128), (28, 4, 128),
                                              (17, 1, 128), (24, 1, 64)])
@pytest.mark.parametrize("q_dtype,out_dtype", DTYPES)
def test_tiles_of_few_rows(cbis, dev, heads, kv_heads, d, q_dtype, out_dtype):
    """A few rows after many keys, whose waves share the keys: whole and in splits, laid
    out for long keys and for short ones; rows before position 0; a K and a V slice of
    NaN that only the later rows see."""
    import torch
    c = Case(cbis, dev, kv_heads, d, 16, [1300], seed=heads + d + 3)
    for which, token, head in ((0, 1293, kv_heads - 1), (1, 1292, 0)):
        pool = c.pools[which].cpu().numpy()
        code, byte = ref.slot_index(kv_heads, d, 16, which == 1, c.table[0, token // 16], token % 16)
        pool[code[head]], pool[byte[head]] = 0, 255
        c.pools[which].copy_(torch.from_numpy(pool))
        c.kv[0][which][token, head] = np.nan
    w = heads * d
    q, qv = _as(rng(82).standard_normal((20, w)).astype(np.float32), q_dtype, dev, 8)
    tiles = [(0, 4, 0, 1290), (4, 1, 0, 70), (5, 8, 0, -3), (13, 2, 0, 1023), (15, 1, 0, 0), (16, 1, 0, 1299)]
    d_tiles = torch.tensor(tiles, dtype=torch.int32, device=dev)
    for split, max_kv in ((0, 1300), (0, 40000), (64, 1300), (512, 1300)):
        table = torch.full((1, 2560), -5, dtype=torch.int32, device=dev)
        table[:, :c.d_table.shape[1]] = c.d_table
        out = torch.full((20, w + 8), 7.0, dtype=_t(out_dtype), device=dev)
        a = c.desc(cbis, q, q_dtype, out, out_dtype, heads)
        a.block_table, a.bt_stride, a.max_kv_len, a.split_tokens = ptr(table), 2560, max_kv, split
        need = cbis.kernels().cbis_kv8_chunk_attention_workspace_size(ctypes.byref(a), len(tiles))
        ws = _workspace(a, need, dev)
        cbis.check(cbis.kernels().cbis_kv8_chunk_attention(ctypes.byref(a), len(tiles), ptr(d_tiles), stream()))
        sync()
        del ws
        got = out.double().cpu().numpy()
        assert (got[17:] == 7.0).all() and (got[:, w:] == 7.0).all()
        for row, rows, seq, pos in tiles:
            for i in range(rows):
                c.check(got[row + i, :w].reshape(heads, d), seq, pos + i, qv[row + i].reshape(heads, d), q_dtype, out_dtype,
                        f"split {split} max {max_kv} row {row + i}")


@pytest.mark.parametrize("kv_heads,d,page_size,n,pad", [
    (1, 32, 16, 70, 0), (2, 32, 32, 150, 3), (3, 32, 16, 77, 0), (8, 32, 16, 170, 1), (1, 64, 16, 90, 1),
    (2, 64, 16, 48, 0), (4, 64, 32, 200, 2), (1, 128, 64, 130, 0), (2, 128, 16, 65, 4)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_narrow_rows(cbis, dev, kv_heads, d, page_size, n, pad, dtype):
    """Rows of which a wave takes several, or just does not."""
    test_scatter_then_gather(cbis, dev, kv_heads, d, page_size, n, pad, dtype)
