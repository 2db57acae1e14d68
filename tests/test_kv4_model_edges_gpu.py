"""A model whose 4-bit cache was cut, and what comes after: a new sequence, a cache filled anew."""
import ctypes as C

import numpy as np
import pytest

from libinferbit_b200 import _ffi
from tests import _cpu
from tests._cpu import p
from tests.test_host_gpu import _tiny_model, host  # noqa: F401
from tests.test_kv4_model_gpu import Twin

pytestmark = pytest.mark.gpu


def _step(host, m, toks, pos, vocab):
    got = np.empty((len(toks), vocab), np.float32)
    assert host.ib_b200_forward_step(m, p(toks), pos, len(toks), p(got)) == 0
    return got


@pytest.mark.parametrize("graph", [1, 0])
def test_a_new_sequence_after_an_eviction(host, graph):  # noqa: F811
    rng = np.random.default_rng(77)
    cfg = _ffi.ModelCfg(256, 512, 2, 8, 2, 32, 320, 40, 1e-5, 10000.0, 8, 4, 8)
    parts = _tiny_model(rng, cfg)
    layers, (hw, hs), emb, es, fn = parts
    m = host.ib_b200_model_create(host.ib_b200_ctx(), C.byref(cfg))
    for l, (lin, norms) in enumerate(layers):
        for i, (w, s, M, N, bits) in enumerate(lin):
            assert host.ib_b200_model_set_linear(m, l, i, p(w), p(s)) == 0
        assert host.ib_b200_model_set_norms(m, l, p(norms[0]), p(norms[1])) == 0
    assert host.ib_b200_model_set_linear(m, 0, 7, p(hw), p(hs)) == 0 and host.ib_b200_model_set_embedding(m, p(emb), p(es), p(fn)) == 0
    assert host.ib_b200_model_kv4(m, 1) == 0
    host.ib_b200_model_use_graph(m, graph)
    for turn in range(3):                                     # each a sequence of its own, cut and gone on with
        twin, pos = Twin(cfg, parts), 0
        for B in (12, 1, 1, 6, None, 1, 5, None, 1, 1):
            if B is None:
                assert host.ib_b200_model_evict(m, pos, 9, 2, 3) == 0
                twin.evict(9, 2, 3)
                continue
            toks = rng.integers(0, cfg.vocab, B).astype(np.int32)
            got, want = _step(host, m, toks, pos, cfg.vocab), twin.step(toks, pos)
            assert _cpu.close(got, want, 2e-3, 2e-4 * max(1.0, float(np.abs(want).max()))), (turn, pos)
            pos += B
    # refused steps leave the sequence as it is
    bad = np.zeros(1, np.int32)
    assert host.ib_b200_forward_step(m, p(bad), pos - 3, 1, None) != 0 and host.ib_b200_forward_step(m, p(bad), -1, 1, None) != 0
    assert host.ib_b200_forward_step(m, p(np.zeros(33, np.int32)), 0, 33, None) != 0
    toks = rng.integers(0, cfg.vocab, 2).astype(np.int32)
    got, want = _step(host, m, toks, pos, cfg.vocab), twin.step(toks, pos)
    assert _cpu.close(got, want, 2e-3, 2e-4 * max(1.0, float(np.abs(want).max())))
    host.ib_b200_model_free(m)


def test_a_cache_filled_anew_after_an_eviction(host):  # noqa: F811
    """The step behind the filled positions is that of a model that was never cut."""
    cfg = _ffi.ModelCfg(256, 512, 1, 8, 4, 32, 320, 64, 1e-5, 10000.0, 8, 4, 8)
    toks, outs = np.array([7], np.int32), []
    for cut in (False, True):
        m = host.ib_b200_model_create(host.ib_b200_ctx(), C.byref(cfg))
        assert host.ib_b200_model_kv4(m, 1) == 0 and host.ib_b200_model_fill_random(m, 5, 30) == 0
        if cut:
            _step(host, m, toks, 30, cfg.vocab)
            assert host.ib_b200_model_evict(m, 31, 8, 2, 2) == 0 and host.ib_b200_model_fill_random(m, 5, 30) == 0
        outs.append(_step(host, m, toks, 30, cfg.vocab))
        host.ib_b200_model_free(m)
    assert np.isfinite(outs[0]).all() and np.array_equal(*outs)
