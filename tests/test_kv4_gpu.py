"""The 4-bit KV cache: codes and scales bit for bit, attention and the weight of rows against 64 bits, eviction row for row."""
import numpy as np
import pytest

from tests import _kv4

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _free(backend):
    had = list(backend._bufs)
    yield
    for b in [b for b in backend._bufs if b not in had]:
        b.free()
        backend._bufs.remove(b)


def put(be, k, v, s, weight=None, decay=1.0):
    t = be.make_kv4(k.shape[0], k.shape[2] * 2, k.shape[1], weights=weight is not None, decay=decay)
    for b, a in zip(t._keep, (k, v, s.view(np.uint16)) + (() if weight is None else (weight.astype(np.float32),))):
        be.write(b, a)
    return t


def get(be, t):
    n, hd, rows = t.n_kv_heads, t.head_dim, t.max_rows
    k, v = (be.download(t._keep[i], np.uint8, n * rows * hd // 2).reshape(n, rows, hd // 2) for i in (0, 1))
    s = be.download(t._keep[2], np.uint16, n * rows * hd // 16).view(np.float16).reshape(n, rows, hd // 16)
    return (k, v, s) + ((be.download(t._keep[3], np.float32, n * rows).reshape(n, rows),) if t.weight else ())


def same(a, b):
    return np.array_equal(raw(a), raw(b)) or (np.array_equal(np.isnan(a), np.isnan(b)) and np.array_equal(a[~np.isnan(a)], b[~np.isnan(b)]))


def raw(a):
    return np.ascontiguousarray(a).view(np.uint8)


def rows_of(x, n_kv):
    return np.ascontiguousarray(x.reshape(x.shape[0], n_kv, -1).transpose(1, 0, 2))


@pytest.mark.parametrize("n_kv,hd,row0,pos0,B,theta", [(1, 32, 0, 0, 1, 10000.0), (8, 128, 5, 5, 3, 10000.0), (2, 64, 7, 100000, 9, 500000.0), (3, 96, 0, 3, 40, 0.0),
                                                        (5, 192, 11, 0, 2, 10000.0), (1, 256, 0, 77, 17, 10000.0), (4, 64, 130, 2000000, 65, 1000000.0)])
def test_rows_are_written_as_the_formula_says(backend, n_kv, hd, row0, pos0, B, theta):
    """Every code and scale of the new rows, the other rows untouched, and the read-back in the plain order."""
    be, rng = backend, np.random.default_rng(hd + B)
    max_rows = (row0 + B + 7) // 8 * 8 + 8
    k, v = (rng.standard_normal((B, n_kv * hd), dtype=np.float32) * np.float32(3) for _ in range(2))
    planes = _kv4.random_planes(rng, n_kv, hd, max_rows, row0)
    t = put(be, *planes, weight=rng.standard_normal((n_kv, max_rows)))
    before = get(be, t)
    dk, dv = be.upload(k), be.upload(v)
    be._check(be.lib.ibcu_kv4_write(be.ctx, t, dk.ptr, dv.ptr, row0, pos0, B, theta)); be.sync()
    after = get(be, t)
    kc, ks = _kv4.quantise(rows_of(_kv4.rotate(k, n_kv, pos0, theta).astype(np.float32), n_kv))
    vc, vs = _kv4.quantise(rows_of(v, n_kv))
    new = slice(row0, row0 + B)
    assert np.array_equal(after[0][:, new], _kv4.pack(kc, True)) and np.array_equal(after[1][:, new], _kv4.pack(vc, False))
    assert same(after[2][:, new], np.concatenate([ks, vs], -1)) and not after[3][:, new].any()
    for a, b in zip(before, after):
        old = [i for i in range(max_rows) if not row0 <= i < row0 + B]
        assert np.array_equal(raw(a[:, old]), raw(b[:, old]))
    assert np.array_equal(be.download(dk, np.float32, k.size), k.reshape(-1))
    ok, ov = be.alloc(k.nbytes), be.alloc(v.nbytes)
    be._check(be.lib.ibcu_kv4_read(be.ctx, t, ok.ptr, ov.ptr, row0, B)); be.sync()
    for o, c, s in ((ok, kc, ks), (ov, vc, vs)):
        assert np.array_equal(be.download(o, np.float32, k.size).reshape(B, n_kv, hd), _kv4.values(c, s).transpose(1, 0, 2).astype(np.float32))


def test_groups_out_of_the_ordinary(backend):
    """Zeros, values below the smallest scale, beyond the largest, Inf and NaN: each group by itself."""
    be, rng = backend, np.random.default_rng(1)
    x = rng.standard_normal((1, 256), dtype=np.float32).reshape(8, 32)
    x[0] = 0; x[1] *= 1e-9; x[2] *= 1e-6; x[3] *= 1e38; x[4, 3] = np.inf; x[5, 31] = np.nan; x[6] *= 8192 * 7; x[7, 0] = -np.inf
    x = x.reshape(1, 256)
    t = be.make_kv4(1, 256, 8)
    dx = be.upload(x)
    be._check(be.lib.ibcu_kv4_write(be.ctx, t, dx.ptr, dx.ptr, 2, 9, 1, 0.0)); be.sync()
    c, s = _kv4.quantise(x)
    k, v, sc = get(be, t)
    assert np.array_equal(k[0, 2], _kv4.pack(c, True)[0]) and np.array_equal(v[0, 2], _kv4.pack(c, False)[0])
    assert same(sc[0, 2], np.concatenate([s, s], -1)[0])
    assert np.isnan(s[0, [4, 5, 7]]).all() and s[0, 0] == 0 and s[0, 1] == 0 and s[0, 2] > 0 and s[0, 3] == 8192


SHAPES = [(1, 1, 32, 0, 1), (32, 8, 128, 0, 1), (32, 8, 128, 511, 1), (32, 4, 64, 3001, 6), (8, 1, 256, 100, 9), (6, 2, 96, 33, 5), (12, 12, 64, 257, 3), (10, 2, 192, 60, 8),
          (9, 1, 32, 17, 2), (24, 2, 64, 40, 3), (4, 4, 128, 0, 130), (8, 2, 64, 700, 70), (2, 1, 128, 9000, 1), (16, 16, 64, 1, 33), (40, 1, 128, 70, 1)]


@pytest.mark.parametrize("n_heads,n_kv,hd,row0,B", SHAPES)
def test_attention_and_weights(backend, n_heads, n_kv, hd, row0, B):
    """Heads in groups of 1 to 40, single positions and several, rows that end anywhere; what lies behind the last row is garbage."""
    be, rng = backend, np.random.default_rng(n_heads + hd + row0)
    R = row0 + B
    max_rows = (R + 7) // 8 * 8 + 16
    planes = _kv4.random_planes(rng, n_kv, hd, max_rows, R)
    q = rng.standard_normal((B, n_heads * hd), dtype=np.float32) * np.float32(1.5)
    old = rng.uniform(0, 2, (n_kv, max_rows)).astype(np.float32)
    want, weight, tol, wtol = _kv4.attention(q.astype(np.float64), _kv4.plane_values(*(p[:, :R] for p in planes)), n_heads, row0)
    dq, do = be.upload(q), be.alloc(q.nbytes)
    for decay, w0 in ((None, None), (1.0, old), (0.5, old), (0.0, np.full_like(old, np.nan))):
        t = put(be, *planes, weight=w0, decay=decay or 0.0)
        be._check(be.lib.ibcu_memset(be.ctx, do.ptr, 0xFF, q.nbytes))
        be._check(be.lib.ibcu_attention_kv4(be.ctx, t, dq.ptr, do.ptr, n_heads, row0, B)); be.sync()
        got = be.download(do, np.float32, q.size).reshape(q.shape)
        assert np.all(np.abs(got - want) <= tol), (decay, np.max(np.abs(got - want) / tol))
        if w0 is not None:
            after = get(be, t)[3]
            full = weight + (decay * w0[:, :R].astype(np.float64) if decay else 0.0)
            assert np.all(np.abs(after[:, :R] - full) <= wtol + 3 * 2.0 ** -24 * full), decay
            assert np.array_equal(after[:, R:], w0[:, R:], equal_nan=True)
        assert np.array_equal(be.download(dq, np.float32, q.size), q.reshape(-1))


@pytest.mark.parametrize("n_heads,n_kv,hd,row0,B", [(32, 8, 128, 0, 200), (16, 16, 64, 37, 400), (32, 4, 64, 1000, 333), (48, 48, 128, 61, 129), (32, 8, 128, 1, 257)])
def test_prompts(backend, n_heads, n_kv, hd, row0, B):
    """Enough columns for tiles of 128 on the tensor cores: tiles and rows that end anywhere, groups that do not divide a tile's positions."""
    test_attention_and_weights(backend, n_heads, n_kv, hd, row0, B)


@pytest.mark.parametrize("n_heads,n_kv,hd,row0,pos0,B,theta", [(32, 8, 128, 512, 512, 1, 10000.0), (32, 4, 64, 0, 0, 1, 10000.0), (8, 2, 128, 100, 5000, 4, 500000.0),
                                                                (6, 6, 96, 31, 31, 33, 10000.0), (4, 1, 256, 15, 70000, 2, 10000.0), (5, 1, 32, 3, 3, 1, 0.0), (32, 8, 128, 0, 0, 150, 10000.0),
                                                                (32, 8, 128, 5, 5, 200, 10000.0), (12, 12, 64, 70, 9000, 600, 500000.0)])
def test_decode_step(backend, n_heads, n_kv, hd, row0, pos0, B, theta):
    """One call: queries and keys rotated, the rows written as ibcu_kv4_write writes them, attention over them; inputs left alone."""
    be, rng = backend, np.random.default_rng(row0 + B)
    R = row0 + B
    max_rows = (R + 7) // 8 * 8
    planes = _kv4.random_planes(rng, n_kv, hd, max_rows, row0)
    q = rng.standard_normal((B, n_heads * hd), dtype=np.float32)
    k, v = (rng.standard_normal((B, n_kv * hd), dtype=np.float32) for _ in range(2))
    dq, dk, dv, do = be.upload(q), be.upload(k), be.upload(v), be.alloc(q.nbytes)
    t, t2 = put(be, *planes, weight=np.ones((n_kv, max_rows)), decay=0.0), put(be, *planes, weight=np.ones((n_kv, max_rows)))
    be._check(be.lib.ibcu_attention_decode_kv4(be.ctx, t, dq.ptr, dk.ptr, dv.ptr, do.ptr, n_heads, row0, pos0, B, theta))
    be._check(be.lib.ibcu_kv4_write(be.ctx, t2, dk.ptr, dv.ptr, row0, pos0, B, theta)); be.sync()
    a, b = get(be, t), get(be, t2)
    for x, y in zip(a[:3], b[:3]):
        assert np.array_equal(raw(x), raw(y))
    want, weight, tol, wtol = _kv4.attention(_kv4.rotate(q, n_heads, pos0, theta).astype(np.float32).astype(np.float64), _kv4.plane_values(*(p[:, :R] for p in b[:3])), n_heads, row0)
    got = be.download(do, np.float32, q.size).reshape(q.shape)
    assert np.all(np.abs(got - want) <= tol), np.max(np.abs(got - want) / tol)
    assert np.all(np.abs(a[3][:, :R] - weight) <= wtol + 2.0 ** -24 * weight)
    for d, x in ((dq, q), (dk, k), (dv, v)):
        assert np.array_equal(be.download(d, np.float32, x.size), x.reshape(-1))


@pytest.mark.parametrize("n_heads,n_kv,hd,row0,B,at", [(8, 2, 64, 0, 6, 3), (4, 4, 128, 29, 9, 30), (4, 1, 256, 60, 8, 67), (8, 8, 64, 0, 80, 33), (32, 8, 128, 200, 3, 201), (32, 8, 128, 100, 300, 250),
                                                       (32, 4, 64, 0, 300, 130)])
def test_a_later_row_does_not_reach_an_earlier_position(backend, n_heads, n_kv, hd, row0, B, at):
    """Row `at` holds NaN in key and value: positions that do not see it keep their bits, the others show it."""
    be, rng = backend, np.random.default_rng(at)
    R = row0 + B
    k, v, s = _kv4.random_planes(rng, n_kv, hd, (R + 7) // 8 * 8, R)
    q = be.upload(rng.standard_normal((B, n_heads * hd), dtype=np.float32))
    outs = []
    for poison in (False, True):
        if poison:
            s[:, at] = np.nan
        t, o = put(be, k, v, s, weight=np.zeros(k.shape[:2]), decay=0.0), be.alloc(B * n_heads * hd * 4)
        be._check(be.lib.ibcu_attention_kv4(be.ctx, t, q.ptr, o.ptr, n_heads, row0, B)); be.sync()
        outs.append(be.download(o, np.float32, B * n_heads * hd).reshape(B, -1))
    first = at - row0
    assert np.isfinite(outs[0]).all() and np.array_equal(outs[0][:first], outs[1][:first])
    assert np.isnan(outs[1][first:]).all()


def test_extreme_queries(backend):
    """A query of zeros weighs all rows alike, one of 1e30 picks the row of the largest score, Inf or NaN shows in its head alone."""
    be, rng = backend, np.random.default_rng(5)
    n_heads, n_kv, hd, row0 = 8, 2, 64, 99
    planes = _kv4.random_planes(rng, n_kv, hd, 104, 100)
    K, V = _kv4.plane_values(*(p[:, :100] for p in planes))
    q = rng.standard_normal((1, n_heads, hd)).astype(np.float32)
    q[0, 1] = 0; q[0, 2] *= np.float32(1e30); q[0, 3, 5] = np.inf; q[0, 4, 0] = np.nan; q[0, 5] *= np.float32(1e-30); q[0, 6] *= np.float32(1e-41)
    dq, do = be.upload(q), be.alloc(q.nbytes)
    be._check(be.lib.ibcu_attention_kv4(be.ctx, put(be, *planes), dq.ptr, do.ptr, n_heads, row0, 1)); be.sync()
    got = be.download(do, np.float32, q.size).reshape(n_heads, hd)
    mean = V.mean(1)
    tol = 700 * 2.0 ** -24 * np.abs(V).mean(1)
    for h in (1, 5, 6):
        assert np.all(np.abs(got[h] - mean[h // 4]) <= tol[h // 4] + 1e-28)
    best = np.argmax(K[0] @ q[0, 2].astype(np.float64))
    assert np.allclose(got[2], V[0, best], rtol=2.0 ** -20, atol=0)
    assert np.isnan(got[3]).all() and np.isnan(got[4]).all() and np.isfinite(got[[0, 1, 2, 5, 6, 7]]).all()


@pytest.mark.parametrize("n_kv,hd,rows,keep,sink,recent", [(1, 32, 1, 1, 0, 0), (8, 128, 4096, 1024, 4, 256), (2, 64, 1000, 999, 0, 0), (3, 96, 777, 100, 0, 100), (4, 64, 50, 50, 3, 9),
                                                            (5, 192, 2049, 1025, 1, 0), (1, 256, 5000, 7, 0, 1), (2, 64, 30001, 12345, 10, 500), (2, 32, 70001, 69999, 0, 3), (16, 32, 300, 5, 2, 2)])
@pytest.mark.parametrize("in_place", [False, True])
def test_eviction(backend, n_kv, hd, rows, keep, sink, recent, in_place):
    """Which rows stay, head by head, with weights that repeat, zeros of both signs, infinities and NaN; the rows themselves as they were."""
    be, rng = backend, np.random.default_rng(rows + keep)
    max_rows, dst_rows = (rows + 7) // 8 * 8 + 8, (keep + 7) // 8 * 8
    k, v, s = _kv4.random_planes(rng, n_kv, hd, max_rows, rows)
    w = np.exp(2 * rng.standard_normal((n_kv, max_rows))).astype(np.float16).astype(np.float32)
    w[rng.random(w.shape) < 0.2] = 1.0
    w[rng.random(w.shape) < 0.1] = 0.0
    w[rng.random(w.shape) < 0.05] = -0.0
    w[rng.random(w.shape) < 0.02] = np.nan
    w[rng.random(w.shape) < 0.02] = np.inf
    w[rng.random(w.shape) < 0.02] = -np.inf
    t = put(be, k, v, s, weight=w)
    d = t if in_place else put(be, *(np.zeros((n_kv, dst_rows, p.shape[2]), p.dtype) for p in (k, v, s)), weight=np.zeros((n_kv, dst_rows)))
    kept = be.alloc(n_kv * keep * 4)
    be._check(be.lib.ibcu_kv4_evict(be.ctx, t, d, rows, keep, sink, recent, None if in_place and keep % 2 else kept.ptr)); be.sync()
    got = get(be, d)
    for h in range(n_kv):
        at = _kv4.choose(w[h, :rows], keep, sink, recent)
        if not (in_place and keep % 2):
            assert np.array_equal(be.download(kept, np.int32, keep, 4 * h * keep), at)
        for a, b in zip((k, v, s, w), got):
            assert np.array_equal(raw(a[h, at]), raw(b[h, :keep]))
            if in_place:
                assert np.array_equal(raw(a[h, rows:]), raw(b[h, rows:]))


def test_prompt_then_eviction_then_decode(backend):
    """As they are used together: a prompt written and attended with weights, the cache cut in place to a budget, and further tokens
    at their own positions over the rows that stayed; the weights go on."""
    be, rng = backend, np.random.default_rng(8)
    n_heads, n_kv, hd, n, keep, sink, recent, theta = 16, 4, 64, 300, 90, 4, 30, 10000.0
    t = be.make_kv4(n_kv, hd, 304, weights=True)
    draw = lambda B, heads: rng.standard_normal((B, heads * hd), dtype=np.float32)
    q, k, v = draw(n, n_heads), draw(n, n_kv), draw(n, n_kv)
    d, o = [be.upload(x) for x in (q, k, v)], be.alloc(q.nbytes)
    be._check(be.lib.ibcu_attention_decode_kv4(be.ctx, t, *(b.ptr for b in d), o.ptr, n_heads, 0, 0, n, theta)); be.sync()
    planes = get(be, t)
    _, weight, _, wtol = _kv4.attention(_kv4.rotate(q, n_heads, 0, theta), _kv4.plane_values(*(p[:, :n] for p in planes[:3])), n_heads, 0)
    assert np.all(np.abs(planes[3][:, :n] - weight) <= wtol + 1e-6 * weight)
    be._check(be.lib.ibcu_kv4_evict(be.ctx, t, t, n, keep, sink, recent, None))
    held = [np.stack([p[h, _kv4.choose(planes[3][h, :n], keep, sink, recent)] for h in range(n_kv)]) for p in planes]
    total = held[3].astype(np.float64)
    for step in range(3):
        q, k, v = draw(1, n_heads), draw(1, n_kv), draw(1, n_kv)
        d = [be.upload(x) for x in (q, k, v)]
        be._check(be.lib.ibcu_attention_decode_kv4(be.ctx, t, *(b.ptr for b in d), o.ptr, n_heads, keep + step, n + step, 1, theta)); be.sync()
        kc, ks = _kv4.quantise(rows_of(_kv4.rotate(k, n_kv, n + step, theta).astype(np.float32), n_kv))
        vc, vs = _kv4.quantise(rows_of(v, n_kv))
        for i, new in enumerate((_kv4.pack(kc, True), _kv4.pack(vc, False), np.concatenate([ks, vs], -1))):
            held[i] = np.concatenate([held[i], new], 1)
        want, weight, tol, wtol = _kv4.attention(_kv4.rotate(q, n_heads, n + step, theta).astype(np.float32).astype(np.float64), _kv4.plane_values(*held[:3]), n_heads, keep + step)
        assert np.all(np.abs(be.download(o, np.float32, n_heads * hd) - want[0]) <= tol[0])
        total = np.concatenate([total, np.zeros((n_kv, 1))], 1) + weight
    after = get(be, t)
    assert np.all(np.abs(after[3][:, :keep + 3] - total) <= 1e-5 * total + 1e-9)
    for a, b in zip(after[:3], held[:3]):
        assert np.array_equal(raw(a[:, :keep + 3]), raw(b))


@pytest.mark.parametrize("n_heads,n_kv,hd,B,max_rows", [(32, 8, 128, 1, 1024), (8, 1, 64, 1, 4096), (16, 4, 64, 6, 600), (32, 8, 128, 40, 256), (32, 8, 128, 200, 512)])
def test_captured_at_a_device_place(backend, n_heads, n_kv, hd, B, max_rows):
    """One captured step serves every place: from an empty cache to a full one, rows and positions apart, weights summed up; the same as
    the launch for one place. A larger call in between makes the scratch grow, which the graph must survive."""
    import ctypes as C
    be, rng = backend, np.random.default_rng(B + hd)
    theta = 10000.0
    planes = _kv4.random_planes(rng, n_kv, hd, max_rows, max_rows)
    w0 = rng.uniform(0, 1, (n_kv, max_rows)).astype(np.float32)
    draw = lambda heads: rng.standard_normal((B, heads * hd), dtype=np.float32)
    q, k, v = draw(n_heads), draw(n_kv), draw(n_kv)
    d, o, at = [be.upload(x) for x in (q, k, v)], be.alloc(q.nbytes), be.upload(np.zeros(2, np.int32))
    t = put(be, *planes, weight=w0)
    call = lambda: be._check(be.lib.ibcu_attention_decode_kv4_at(be.ctx, t, *(x.ptr for x in d), o.ptr, n_heads, at.ptr, B, theta))
    call(); be.sync()
    gid = C.c_int()
    be._check(be.lib.ibcu_graph_begin(be.ctx)); call(); be._check(be.lib.ibcu_graph_end(be.ctx, C.byref(gid)))
    try:
        for i, (row0, pos0) in enumerate([(0, 0), (5, 9000), (max_rows // 2 + 3, max_rows // 2 + 3), (max_rows - B, 77)]):
            for b, a in zip(t._keep, planes):
                be.write(b, a.view(np.uint16) if a.dtype == np.float16 else a)
            be.write(t._keep[3], w0)
            be.write(at, np.array([row0, pos0], np.int32))
            if i == 2:
                big = put(be, *_kv4.random_planes(rng, 8, 128, 2000, 2000), weight=np.zeros((8, 2000)))
                x = be.upload(rng.standard_normal((300, 32 * 128), dtype=np.float32))
                be._check(be.lib.ibcu_attention_kv4(be.ctx, big, x.ptr, be.alloc(300 * 32 * 128 * 4).ptr, 32, 1700, 300))
            be._check(be.lib.ibcu_graph_launch(be.ctx, gid)); be.sync()
            got, after = be.download(o, np.float32, q.size).reshape(q.shape), get(be, t)
            held = [p.copy() for p in planes]
            kc, ks = _kv4.quantise(rows_of(_kv4.rotate(k, n_kv, pos0, theta).astype(np.float32), n_kv))
            vc, vs = _kv4.quantise(rows_of(v, n_kv))
            new = slice(row0, row0 + B)
            held[0][:, new], held[1][:, new], held[2][:, new] = _kv4.pack(kc, True), _kv4.pack(vc, False), np.concatenate([ks, vs], -1)
            for a, b in zip(after, held):
                assert np.array_equal(raw(a), raw(b))
            R = row0 + B
            want, weight, tol, wtol = _kv4.attention(_kv4.rotate(q, n_heads, pos0, theta).astype(np.float32).astype(np.float64), _kv4.plane_values(*(h[:, :R] for h in held)), n_heads, row0)
            assert np.all(np.abs(got - want) <= tol), (row0, np.max(np.abs(got - want) / tol))
            full = weight + np.where(np.arange(R) < row0, w0[:, :R], 0)
            assert np.all(np.abs(after[3][:, :R] - full) <= wtol + 3 * 2.0 ** -24 * full)
            assert np.array_equal(after[3][:, R:], w0[:, R:])
        # a place outside the cache writes nothing and is reported
        for row0, pos0 in ((max_rows - B + 1, 0), (-1, 0), (0, -5)):
            before = get(be, t)
            be.write(at, np.array([row0, pos0], np.int32))
            be._check(be.lib.ibcu_graph_launch(be.ctx, gid))
            assert be.lib.ibcu_sync(be.ctx) == -1 and b"outside the cache" in be.lib.ibcu_last_error(be.ctx)
            be.lib.ibcu_clear_error(be.ctx)
            for a, b in zip(get(be, t), before):
                assert np.array_equal(raw(a), raw(b))
    finally:
        be._check(be.lib.ibcu_graph_destroy(be.ctx, gid))


@pytest.mark.parametrize("n_heads,n_kv,hd,row0,B", [(32, 8, 128, 6000, 1), (8, 1, 128, 9001, 1), (64, 8, 64, 5000, 1), (32, 32, 96, 4200, 1), (4, 2, 256, 8193, 2), (8, 1, 64, 7000, 6), (16, 2, 192, 4097, 3),
                                                    (4, 4, 32, 20000, 1), (32, 8, 128, 4090, 6)])
def test_contexts_of_many_chunks(backend, n_heads, n_kv, hd, row0, B):
    """More chunks than a cluster has blocks, in tiles of 4, 8 and 16 columns."""
    test_attention_and_weights(backend, n_heads, n_kv, hd, row0, B)


@pytest.mark.parametrize("n_heads,n_kv,hd,row0,B", [(8, 1, 128, 8000, 640), (8, 1, 64, 8000, 900), (8, 2, 128, 12000, 60), (4, 1, 96, 12000, 100), (8, 1, 128, 30000, 1)])
def test_sums_over_many_rows_stay_exact(backend, n_heads, n_kv, hd, row0, B):
    """The tensor cores cut every addition off by up to 2^-23 of the sum, all in one direction. Within the 192 rows that a sum is theirs there are 36 additions, so that
    the outputs are off by at most 36 * 2^-23 of their size, and by about as much again from scores of 24 additions (less than 2 log2 units in size) and
    everything that is rounded. (All rows in one sum would be hundreds of additions: 5.7e-5 off.)"""
    be, rng = backend, np.random.default_rng(row0)
    R = row0 + B
    max_rows = (R + 7) // 8 * 8
    planes = _kv4.random_planes(rng, n_kv, hd, max_rows, R)
    q = rng.standard_normal((B, n_heads * hd), dtype=np.float32)
    dq, do = be.upload(q), be.alloc(q.nbytes)
    be._check(be.lib.ibcu_attention_kv4(be.ctx, put(be, *planes), dq.ptr, do.ptr, n_heads, row0, B)); be.sync()
    got = be.download(do, np.float32, q.size).reshape(B, n_heads, hd)
    K, V = _kv4.plane_values(*(p[:, :R] for p in planes))
    off = size = 0.0
    for h in range(n_heads):
        s = q.reshape(B, n_heads, hd)[:, h].astype(np.float64) @ K[h * n_kv // n_heads].T / np.sqrt(hd)
        p = np.where(np.arange(R)[None] <= row0 + np.arange(B)[:, None], np.exp(s - s.max(1, keepdims=True)), 0.0)
        want = p @ V[h * n_kv // n_heads] / p.sum(1, keepdims=True)
        off, size = off + ((got[:, h] - want) ** 2).sum(), size + (want ** 2).sum()
    assert np.sqrt(off / size) <= 2 * 36 * 2.0 ** -23, np.sqrt(off / size)


@pytest.mark.parametrize("n_kv,hd,rows,keep,sink,recent", [(1, 32, 150001, 100000, 3, 7), (40, 64, 3000, 900, 4, 100), (14, 128, 9000, 5000, 0, 0), (1, 64, 131072, 1, 0, 0)])
@pytest.mark.parametrize("in_place", [False, True])
def test_eviction_by_size(backend, n_kv, hd, rows, keep, sink, recent, in_place):
    """More rows than registers hold, more heads than clusters of eight or four have room, more kept rows than the choosing launch copies."""
    test_eviction(backend, n_kv, hd, rows, keep, sink, recent, in_place)


def test_eviction_by_weights_that_share_their_bits(backend):
    """Bounds that are found after one round, two or three, and the smallest there is."""
    be, rng = backend, np.random.default_rng(8)
    n_kv, hd, rows = 6, 32, 4096
    bits = np.empty((n_kv, rows), np.uint32)
    bits[0] = np.where(np.arange(rows) % 4 == 0, 0x41000000, 0x3F000000)                   # the first eight bits decide for 1024 rows
    bits[1] = 0x3F800000 + rng.permutation(rows).astype(np.uint32)                         # all but the last thirteen bits are equal
    bits[2] = 0                                                                             # zeros: the lowest rows
    bits[3] = 0x7FC00000                                                                    # NaN: the lowest rows
    bits[4] = np.where(np.arange(rows) % 4 == 1, 0x3F900000, 0x3F800000)
    bits[5] = np.where(np.arange(rows) < 1024, 0x80000000, 0xFF800000)                      # minus zero above minus infinity
    w = bits.view(np.float32)
    planes = _kv4.random_planes(rng, n_kv, hd, rows, rows)
    for keep in (1024, 1023, 1025, 1):
        src, dst = put(be, *planes, weight=w), be.make_kv4(n_kv, hd, rows, weights=True)
        kept = be.alloc(n_kv * keep * 4)
        be._check(be.lib.ibcu_kv4_evict(be.ctx, src, dst, rows, keep, 0, 0, kept.ptr)); be.sync()
        got = be.download(kept, np.int32, n_kv * keep).reshape(n_kv, keep)
        for h in range(n_kv):
            assert np.array_equal(got[h], _kv4.choose(w[h], keep, 0, 0)), (keep, h)


@pytest.mark.parametrize("n_heads,n_kv,hd,row0,B", [(32, 8, 128, 40, 1), (8, 1, 64, 5000, 1), (16, 4, 96, 11, 9), (32, 8, 128, 3, 200), (12, 3, 256, 0, 2)])
def test_activations_at_any_address(backend, n_heads, n_kv, hd, row0, B):
    """Queries, keys, values and outputs four bytes off a 16-byte boundary, and rows written and read back so: the same bits as on one."""
    be, rng = backend, np.random.default_rng(B)
    max_rows = (row0 + B + 7) // 8 * 8
    planes = _kv4.random_planes(rng, n_kv, hd, max_rows, row0 + B)
    draw = lambda heads: rng.standard_normal((B, heads * hd), dtype=np.float32)
    x = [draw(n_heads), draw(n_kv), draw(n_kv)]
    results = []
    for off in (0, 4):
        t = put(be, *planes, weight=np.zeros((n_kv, max_rows), np.float32))
        d = [be.alloc(a.nbytes + 16) for a in x]
        for b, a in zip(d, x):
            be.write(b, a, off)
        o, kb, vb = be.alloc(x[0].nbytes + 16), be.alloc(x[1].nbytes + 16), be.alloc(x[1].nbytes + 16)
        be._check(be.lib.ibcu_attention_decode_kv4(be.ctx, t, *(b.at(off) for b in d), o.at(off), n_heads, row0, row0 + 7, B, 10000.0))
        be._check(be.lib.ibcu_kv4_read(be.ctx, t, kb.at(off), vb.at(off), row0, B)); be.sync()
        raw_of = lambda b, n: be.download(b, np.float32, n + 4)[off // 4:off // 4 + n]
        results.append([raw_of(o, x[0].size), raw_of(kb, x[1].size), raw_of(vb, x[1].size)] + [raw(a) for a in get(be, t)])
    for a, b in zip(*results):
        assert np.array_equal(a, b, equal_nan=a.dtype.kind == "f")


def test_captured_eviction_in_place(backend):
    """A captured step and cut of the same cache, replayed over fresh contents."""
    import ctypes as C
    be, rng = backend, np.random.default_rng(3)
    n_kv, hd, rows, keep = 4, 64, 3000, 700
    planes = _kv4.random_planes(rng, n_kv, hd, rows, rows)
    t = put(be, *planes, weight=np.zeros((n_kv, rows), np.float32))
    kept = be.alloc(n_kv * keep * 4)
    call = lambda: be._check(be.lib.ibcu_kv4_evict(be.ctx, t, t, rows, keep, 4, 60, kept.ptr))
    call(); be.sync()
    gid = C.c_int()
    be._check(be.lib.ibcu_graph_begin(be.ctx)); call(); be._check(be.lib.ibcu_graph_end(be.ctx, C.byref(gid)))
    try:
        for _ in range(3):
            planes = _kv4.random_planes(rng, n_kv, hd, rows, rows)
            w = rng.exponential(1.0, (n_kv, rows)).astype(np.float32)
            for b, a in zip(t._keep, planes):
                be.write(b, a.view(np.uint16) if a.dtype == np.float16 else a)
            be.write(t._keep[3], w)
            be._check(be.lib.ibcu_graph_launch(be.ctx, gid)); be.sync()
            got, after = be.download(kept, np.int32, n_kv * keep).reshape(n_kv, keep), get(be, t)
            for h in range(n_kv):
                at = _kv4.choose(w[h], keep, 4, 60)
                assert np.array_equal(got[h], at)
                for a, b in zip(after, planes + (w,)):
                    assert np.array_equal(raw(a[h, :keep]), raw(b[h, at])) and np.array_equal(raw(a[h, keep:]), raw(b[h, keep:]))
    finally:
        be._check(be.lib.ibcu_graph_destroy(be.ctx, gid))


@pytest.mark.parametrize("n_heads,n_kv,hd,row0,B", [(8, 2, 64, 700, 1), (16, 2, 128, 700, 1), (8, 2, 96, 500, 30), (8, 2, 128, 900, 70), (8, 2, 64, 300, 1000), (8, 2, 128, 300, 700)])
def test_extreme_scores_in_every_form(backend, n_heads, n_kv, hd, row0, B):
    """Queries times 1e30 give each softmax one row, whose weight is 1, zeros weigh all rows alike, NaN stays in its own position and head, and a key of NaN in the positions
    that see it: for every kernel that a number of columns may reach."""
    be, rng = backend, np.random.default_rng(hd + B)
    R = row0 + B
    max_rows = (R + 7) // 8 * 8
    planes = _kv4.random_planes(rng, n_kv, hd, max_rows, R)
    group = n_heads // n_kv
    K, V = _kv4.plane_values(*(p[:, :R] for p in planes))
    q = rng.standard_normal((B, n_heads, hd)).astype(np.float32)
    q[:, 0] *= np.float32(1e30)
    q[:, 1] = 0
    q[B // 2, 2, 3] = np.nan
    t = put(be, *planes, weight=np.zeros((n_kv, max_rows), np.float32))
    dq, do = be.upload(q), be.alloc(q.nbytes)
    be._check(be.lib.ibcu_attention_kv4(be.ctx, t, dq.ptr, do.ptr, n_heads, row0, B)); be.sync()
    got = be.download(do, np.float32, q.size).reshape(q.shape)
    bad = np.isnan(got).any(2)
    assert bad[B // 2, 2] and bad.sum() == 1 and np.isnan(got[B // 2, 2]).all()
    s = q[:, 0].astype(np.float64) @ K[0].T
    s[np.arange(R)[None] > row0 + np.arange(B)[:, None]] = -np.inf
    best = s.argmax(1)
    assert np.allclose(got[:, 0], V[0, best], rtol=2.0 ** -18, atol=0)
    mean = np.cumsum(V[0], 0)[row0:] / np.arange(row0 + 1, R + 1)[:, None]
    size = np.cumsum(np.abs(V[0]), 0)[row0:] / np.arange(row0 + 1, R + 1)[:, None]
    assert np.all(np.abs(got[:, 1] - mean) <= 1500 * 2.0 ** -24 * size)
    w = get(be, t)[3]
    assert np.isnan(w[0, : row0 + B // 2 + 1]).all() and np.isfinite(w[1:, :R]).all()                  # the NaN query's weights
    assert np.allclose(w[1, :R].sum(), B * group, rtol=2.0 ** -12)
    # the same without the NaN query: every row has what it drew as the best one, and its shares
    q[B // 2, 2, 3] = 0
    q[:, 2:group] = q[:, :1]
    t = put(be, *planes, weight=np.zeros((n_kv, max_rows), np.float32))
    dq = be.upload(q)
    be._check(be.lib.ibcu_attention_kv4(be.ctx, t, dq.ptr, do.ptr, n_heads, row0, B)); be.sync()
    w = get(be, t)[3][0, :R]
    want = (group - 1) * np.bincount(best, minlength=R).astype(np.float64)
    share = 1.0 / np.arange(row0 + 1, R + 1)
    want += np.array([share[max(0, r - row0):].sum() for r in range(R)])
    assert np.allclose(w, want, rtol=2.0 ** -12, atol=1e-7)
    # a key that is not a number
    planes[2][0, row0 // 2, 0] = np.nan
    t = put(be, *planes, weight=np.zeros((n_kv, max_rows), np.float32))
    be._check(be.lib.ibcu_attention_kv4(be.ctx, t, dq.ptr, do.ptr, n_heads, row0, B)); be.sync()
    got = be.download(do, np.float32, q.size).reshape(q.shape)
    assert np.isnan(got[:, [0, *range(2, group)]]).all() and np.isfinite(got[:, group:]).all()


@pytest.mark.parametrize("n_heads,n_kv,hd,B,max_rows", [(8, 2, 128, 1, 40000), (64, 8, 64, 1, 20000), (8, 2, 96, 5, 30000), (4, 2, 64, 40, 20000), (32, 32, 32, 1, 9000)])
def test_captured_at_a_device_place_of_a_long_cache(backend, n_heads, n_kv, hd, B, max_rows):
    """Grids for a long cache and contexts that fill little of it, half and all."""
    test_captured_at_a_device_place(backend, n_heads, n_kv, hd, B, max_rows)
