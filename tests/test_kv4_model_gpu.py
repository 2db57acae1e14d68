"""A model whose KV cache is held in 4 bits, step by step against the same model in numpy (64 bits, its rows coded as tests/_kv4.py codes
them): a prompt, tokens replayed from one graph, an eviction, and more tokens at their own positions."""
import ctypes as C

import numpy as np
import pytest

from libinferbit_b200 import _ffi
from tests import _cpu, _kv4
from tests._cpu import p
from tests.test_host_gpu import _tiny_model, host  # noqa: F401

pytestmark = pytest.mark.gpu


def _half(bits):
    return bits.view(np.float16).astype(np.float64)


def _dense(w, s, M, N, bits):
    if bits == 8:
        return w.reshape(M, N).astype(np.float64) * _half(s)[:, None]
    q = np.empty((M, N))
    q[:, 0::2], q[:, 1::2] = (w.reshape(M, N // 2) & 15) - 8.0, (w.reshape(M, N // 2) >> 4) - 8.0
    return q * _half(s)[:, None]


class Twin:
    def __init__(self, cfg, parts):
        layers, (hw, hs), emb, es, fn = parts
        self.cfg, self.emb, self.fn = cfg, emb.astype(np.float64) * _half(es)[:, None], _half(fn)
        self.layers = [([_dense(*t) for t in lin], [_half(n) for n in norms]) for lin, norms in layers]
        self.head = _dense(hw, hs, cfg.vocab, cfg.hidden, 8)
        hd, n_kv = cfg.head_dim, cfg.n_kv_heads
        self.cache = [[np.zeros((n_kv, 0, hd)), np.zeros((n_kv, 0, hd)), np.zeros((n_kv, 0))] for _ in layers]

    def step(self, tokens, pos):
        c = self.cfg
        norm = lambda x, w: x / np.sqrt((x * x).mean(1, keepdims=True) + c.eps) * w
        rows = lambda x: x.reshape(len(tokens), c.n_kv_heads, c.head_dim).transpose(1, 0, 2)
        held = lambda x: _kv4.values(*_kv4.quantise(x.astype(np.float32)))
        x = self.emb[tokens]
        for (lin, norms), cache in zip(self.layers, self.cache):
            h = norm(x, norms[0])
            q, k, v = (h @ w.T for w in lin[:3])
            row0 = cache[0].shape[1]
            cache[0] = np.concatenate([cache[0], held(rows(_kv4.rotate(k, c.n_kv_heads, pos, c.theta)))], 1)
            cache[1] = np.concatenate([cache[1], held(rows(v))], 1)
            out, weight, _, _ = _kv4.attention(_kv4.rotate(q, c.n_heads, pos, c.theta), cache[:2], c.n_heads, row0)
            cache[2] = np.concatenate([cache[2], np.zeros((c.n_kv_heads, len(tokens)))], 1) + weight
            x = x + out @ lin[3].T
            h = norm(x, norms[1])
            g = h @ lin[4].T
            x = x + (g / (1 + np.exp(-g)) * (h @ lin[5].T)) @ lin[6].T
        return norm(x, self.fn) @ self.head.T

    def evict(self, keep, sink, recent):
        for cache in self.cache:
            at = [_kv4.choose(w, keep, sink, recent) for w in cache[2]]
            for i in range(3):
                cache[i] = np.stack([a[r] for a, r in zip(cache[i], at)])


@pytest.mark.parametrize("graph", [1, 0])
def test_steps_over_a_cache_in_4_bits(host, graph):  # noqa: F811
    rng = np.random.default_rng(31)
    cfg = _ffi.ModelCfg(256, 512, 2, 8, 2, 32, 320, 40, 1e-5, 10000.0, 8, 4, 8)
    parts = _tiny_model(rng, cfg)
    layers, (hw, hs), emb, es, fn = parts
    m = host.ib_b200_model_create(host.ib_b200_ctx(), C.byref(cfg))
    for l, (lin, norms) in enumerate(layers):
        for i, (w, s, M, N, bits) in enumerate(lin):
            assert host.ib_b200_model_set_linear(m, l, i, p(w), p(s)) == 0
        assert host.ib_b200_model_set_norms(m, l, p(norms[0]), p(norms[1])) == 0
    assert host.ib_b200_model_set_linear(m, 0, 7, p(hw), p(hs)) == 0 and host.ib_b200_model_set_embedding(m, p(emb), p(es), p(fn)) == 0
    assert host.ib_b200_model_evict(m, 1, 1, 0, 0) != 0                       # an FP32 cache has no weights
    tok0 = np.zeros(1, np.int32)
    assert host.ib_b200_forward_step(m, p(tok0), 0, 1, None) == 0             # a graph over the FP32 cache, which must not be replayed afterwards
    assert host.ib_b200_model_kv4(m, 1) == 0 and host.ib_b200_model_kv4(m, 1) != 0
    host.ib_b200_model_use_graph(m, graph)
    twin, pos = Twin(cfg, parts), 0

    def step(B):
        nonlocal pos
        toks = rng.integers(0, cfg.vocab, B).astype(np.int32)
        got = np.empty((B, cfg.vocab), np.float32)
        assert host.ib_b200_forward_step(m, p(toks), pos, B, p(got)) == 0
        want = twin.step(toks, pos)
        scale = float(np.abs(want).max())
        assert _cpu.close(got, want, 2e-3, 2e-4 * max(1.0, scale)), (B, pos, float(np.max(np.abs(got - want))))
        pos += B

    for B in (20, 1, 1, 5, 1):
        step(B)
    k, v = (np.empty((pos, 64), np.float32) for _ in range(2))
    assert host.ib_b200_model_get_kv(m, 1, p(k), p(v), pos) == 0
    for got, want in ((k, twin.cache[1][0]), (v, twin.cache[1][1])):
        assert np.allclose(got.reshape(pos, 2, 32).transpose(1, 0, 2), want, rtol=2e-3, atol=1e-6)
    for n_pos, keep, sink, recent in ((pos + 20, 4, 0, 0), (pos, 0, 0, 0), (pos, pos + 1, 0, 0), (pos, 8, 5, 4), (pos, 8, -1, 0)):
        assert host.ib_b200_model_evict(m, n_pos, keep, sink, recent) != 0
    assert host.ib_b200_model_evict(m, pos, 10, 2, 4) == 0
    twin.evict(10, 2, 4)
    assert host.ib_b200_forward_step(m, p(tok0), pos - 1, 1, None) != 0       # that position is no row any more
    for B in (1, 1, 12, 1, 1, 8):                                             # past max_ctx in positions, within it in rows
        step(B)
    assert pos > cfg.max_ctx and host.ib_b200_forward_step(m, p(tok0), pos + 10, 1, None) != 0
    assert host.ib_b200_model_evict(m, pos, 12, 0, 6) == 0
    twin.evict(12, 0, 6)
    step(2)
    host.ib_b200_model_free(m)


def test_rows_set_by_the_host(host):  # noqa: F811
    """_set_kv codes the rows as they are (keys rotated already), _get_kv gives the values they are held as."""
    rng = np.random.default_rng(2)
    cfg = _ffi.ModelCfg(256, 512, 1, 8, 4, 32, 320, 50, 1e-5, 10000.0, 8, 4, 8)
    m = host.ib_b200_model_create(host.ib_b200_ctx(), C.byref(cfg))
    assert host.ib_b200_model_kv4(m, 0) == 0 and host.ib_b200_model_fill_random(m, 3, 50) == 0
    k, v = (rng.standard_normal((50, 128), dtype=np.float32) for _ in range(2))
    gk, gv = np.empty_like(k), np.empty_like(v)
    assert host.ib_b200_model_set_kv(m, 0, p(k), p(v), 50) == 0 and host.ib_b200_model_get_kv(m, 0, p(gk), p(gv), 50) == 0
    for got, x in ((gk, k), (gv, v)):
        assert np.array_equal(got, _kv4.values(*_kv4.quantise(x.reshape(50, 4, 32))).reshape(50, 128).astype(np.float32))
    host.ib_b200_model_free(m)
    cfg.head_dim, cfg.n_heads, cfg.n_kv_heads, cfg.hidden = 16, 16, 16, 256
    m = host.ib_b200_model_create(host.ib_b200_ctx(), C.byref(cfg))
    assert host.ib_b200_model_kv4(m, 0) != 0 and host.ib_b200_forward_step(m, p(np.zeros(1, np.int32)), 0, 1, None) == 0     # refused: the FP32 cache stays
    host.ib_b200_model_free(m)
