"""TransformerRunner, the scheduler and the tiers over an fp8 (8-bit pages)
K/V cache, against a 64-bit restatement of the step whose K and V slices go
through the cache's number format (tests/kv8_ref.py)."""
import ctypes

import numpy as np
import pytest
from scipy.special import erf

import kv8_ref as ref
from helpers import check_logits

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _torch_first(dev):
    """torch takes the device before the runtime does."""


def _ln(x):
    m = x.mean(-1, keepdims=True)
    return (x - m) / np.sqrt(((x - m) ** 2).mean(-1, keepdims=True) + 1e-5)


class Model:
    """The reference model's forward over one whole sequence in 64 bits, with
    the product's roundings: bf16 inputs of the linear calls for bf16 and fp8
    weights, K and V as the cache holds them."""

    def __init__(self, oracle, spec):
        self.o, self.s = oracle, spec
        self.w = oracle.synthetic_weights(spec, seed=0, pos_rows=spec.max_seq)

    def act(self, x):
        return self.o.round_bf16(x.astype(np.float32)).astype(np.float64) if self.s.act_bf16 else x

    def lin(self, x, name, bias=None):
        w = self.w.used[name].astype(np.float64)
        if name in self.w.scale:
            w = w * self.w.scale[name].astype(np.float64)[:, None]
        y = x @ w.T
        return y if bias is None else y + self.w.used[bias].astype(np.float64)

    def logits(self, ids):
        s, n = self.s, len(ids)
        x = self.w.used["tok_emb"].astype(np.float64)[ids] + self.w.used["pos_emb"].astype(np.float64)[:n]
        mask = np.triu(np.ones((n, n), bool), 1)
        for l in range(s.n_layers):
            p = f"l{l}."
            xn = self.act(_ln(x))
            q, k, v = (self.lin(xn, p + "w" + c, p + "b" + c).reshape(n, s.n_heads, s.head_dim) for c in "qkv")
            k, v = (ref.dequantise(*ref.quantise(t.astype(np.float32))) for t in (k, v))
            out = np.empty_like(q)
            for h in range(s.n_heads):
                a = q[:, h] @ k[:, h].T / np.sqrt(s.head_dim)
                a[mask] = -np.inf
                a = np.exp(a - a.max(1, keepdims=True))
                out[:, h] = a / a.sum(1, keepdims=True) @ v[:, h]
            x = x + self.lin(self.act(out.reshape(n, -1)), p + "wo", p + "bo")
            h = self.lin(self.act(_ln(x)), p + "fc1", p + "b1")
            x = x + self.lin(self.act(0.5 * h * (1 + erf(h / np.sqrt(2)))), p + "fc2", p + "b2")
        return self.lin(self.act(_ln(x)), "lm_head")


def _setup(cbis, oracle, wdt, heads, head_dim, layers=2, pages=64, rows=256):
    kw = dict(vocab=320, d_model=heads * head_dim, n_heads=heads, head_dim=head_dim, n_layers=layers, mlp=512,
              max_seq=512)
    cfg = cbis.ModelConfig.make(weight_dtype=wdt, kv_dtype="fp8", **kw)
    spec = oracle.ModelSpec(weight_dtype=wdt, **kw)
    weights = cbis.ModelWeights.synthetic(cfg, seed=0)
    cache = cbis.PagedKVCache(layers, pages, 16, heads, head_dim, "fp8", pages_per_seq=32)
    return weights, cache, cbis.TransformerRunner(weights, cache, rows), Model(oracle, spec)


@pytest.mark.parametrize("wdt", ["f32", "bf16", "fp8"])
@pytest.mark.parametrize("heads,head_dim", [(8, 32), (5, 64), (2, 128)])
def test_steps_match_the_restatement(cbis, oracle, wdt, heads, head_dim):
    """A mixed step (tiles and single rows), a chunk after cached rows, then
    decode steps whose shape repeats (a captured graph's replays)."""
    weights, cache, runner, model = _setup(cbis, oracle, wdt, heads, head_dim)
    r = np.random.default_rng(heads)
    seqs = [list(map(int, r.integers(0, 320, n))) for n in (3, 40, 150, 70)]
    sids = [cache.allocate_sequence() for _ in seqs]
    done = [0] * len(seqs)

    def step(counts, what):
        tok, pos, sid, want = [], [], [], []
        for i, c in enumerate(counts):
            for p in range(done[i], done[i] + c):
                assert cache.ensure_capacity(sids[i], p)
                tok.append(seqs[i][p]); pos.append(p); sid.append(sids[i])
            if c:
                want.append(model.logits(seqs[i][:done[i] + c])[done[i]:])
            done[i] += c
        got = runner.forward_step(tok, pos, sid)
        check_logits(got.astype(np.float64), np.concatenate(want), f"{wdt} {heads}x{head_dim} {what}")

    step([3, 40, 64, 7], "mixed")
    step([0, 0, 82, 60], "chunks after cached rows")
    for k in range(4):
        for s in seqs:
            s.append(int(r.integers(0, 320)))
        step([len(s) - d if d >= 1 else 0 for s, d in zip(seqs, done)] if k == 0 else [1] * 4, f"decode {k}")
    runner.close(); cache.close(); weights.close()


def test_greedy_schedules_agree(cbis, oracle):
    """The plain and the pipelined scheduler, whole and chunked prompts, graphs
    on and off: the same greedy tokens where the margin is not a rounding's."""
    r = np.random.default_rng(4)
    prompts = [list(map(int, r.integers(0, 320, n))) for n in (5, 33, 90, 17)]
    out = []
    for graphs, pipeline, chunk in ((True, False, 0), (False, False, 0), (True, True, 0), (True, False, 0)):
        weights, cache, runner, _ = _setup(cbis, oracle, "bf16", 8, 32)
        runner.set_graphs(graphs)
        out.append(cbis.run_continuous(runner, cache, prompts, [12] * 4, max_slots=4, prefill_chunk=chunk,
                                       pipeline=pipeline)[0])
        assert cache.num_free_pages() == cache.max_pages()
        runner.close(); cache.close(); weights.close()
    assert all(o == out[0] for o in out)


def test_tiers_move_fp8_pages(cbis, oracle, tmp_path):
    """A sequence's pages spilled to DRAM and NVMe and restored into other
    pages: the next decode step's logits are the same bit for bit."""
    weights, cache, runner, _ = _setup(cbis, oracle, "f32", 8, 32)
    ids = list(map(int, np.random.default_rng(7).integers(0, 320, 60)))
    a, b = cache.allocate_sequence(), cache.allocate_sequence()
    for sid in (a, b):
        assert cache.ensure_capacity(sid, 63)
    runner.forward_step(ids, list(range(60)), [a] * 60)
    first = runner.forward_step([9], [60], [a])
    mgr = cbis.TieredKVBlockManager(2, 16, 8, 32, tmp_path / "t.nvme", 8, 8, kv_dtype="fp8")
    assert mgr.raw_block_bytes() == 2 * 2 * 16 * 8 * 33
    for i, (src, dst) in enumerate(zip(cache.pages(a), cache.pages(b))):
        mgr.admit_gpu_resident(i, cache, src, 0)
        mgr.spill(i, "DRAM" if i % 2 else "NVME", 1)
        mgr.restore(i, cache, dst, 2)
    assert np.array_equal(runner.forward_step([9], [60], [b]), first)
    mgr.close(); runner.close(); cache.close(); weights.close()


def test_fill_normal_fills_every_slot(cbis, dev):
    """fill_normal of an fp8 cache: every slot of every layer reads back as
    finite normals of the given size."""
    import torch
    cache = cbis.PagedKVCache(3, 300, 16, 5, 64, "fp8")
    cache.fill_normal(3, 2.0)
    rows = 300 * 16
    idx = torch.arange(rows, dtype=torch.int32, device=dev)
    seen = []
    for l in range(3):
        c = cbis.Kv8Cache(5, 64, 16, 300, cache.k_base(l), cache.v_base(l))
        k, v = (torch.full((rows, 320), float("nan"), device=dev) for _ in range(2))
        page, off = idx // 16, idx % 16
        cbis.check(cbis.kernels().cbis_kv8_gather(ctypes.byref(c), rows, cbis.F32, k.data_ptr(), 320, v.data_ptr(), 320,
                                                  page.data_ptr(), off.data_ptr(), None))
        torch.cuda.synchronize()
        for x in (k, v):
            assert torch.isfinite(x).all()
            assert abs(float(x.std()) - 2.0) < 0.02 and abs(float(x.mean())) < 0.02
            seen.append(x.flatten()[:4096].cpu())
    assert all(not torch.equal(seen[i], seen[j]) for i in range(6) for j in range(i))
    cache.close()
