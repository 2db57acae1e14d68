"""INT8 x INT8 products with a scale per token and per output row: codes bit for bit, results against 64 bits."""
import numpy as np
import pytest

from libinferbit_b200 import LinearT

pytestmark = pytest.mark.gpu
HALF = 2.0 ** -24                                 # half a step of FP32


@pytest.fixture(autouse=True)
def _free(backend):
    had = list(backend._bufs)
    yield
    for b in [b for b in backend._bufs if b not in had]:
        b.free()
        backend._bufs.remove(b)


def quantise(x):
    """codes and scales of FP32 rows"""
    amax = np.abs(x).max(1)
    s = (amax * (np.float32(1) / np.float32(127))).astype(np.float32)
    with np.errstate(all="ignore"):
        inv = (np.float32(1) / s).astype(np.float32)
        ok = np.isfinite(x).all(1) & (amax >= 2.0 ** -100)
        q = np.where(ok[:, None], np.rint(x * inv[:, None]), 0)
    s[amax < 2.0 ** -100] = 0
    s[~np.isfinite(x).all(1)] = np.nan
    return q.astype(np.int8), s


def tensors(be, rng, Ms, N, B, fp32=False, extra=0, add=False):
    """weights with their extremes, outputs with a row stride beyond M and something in them"""
    w = [rng.integers(-128, 128, (M, N), dtype=np.int8) for M in Ms]
    for a in w:
        a[-1] = -128
    s = [rng.uniform(0.001, 0.01, M).astype(np.float32 if fp32 else np.float16) for M in Ms]
    o = [rng.standard_normal((B, M + extra), dtype=np.float32) for M in Ms]
    do = [be.upload(a) for a in o]
    t = (LinearT * len(Ms))(*[LinearT(be.upload(a).ptr, be.upload(b).ptr, d.ptr, M, M + extra, int(fp32), int(add)) for a, b, d, M in zip(w, s, do, Ms)])
    return t, w, s, o, do


def check(be, w, s, o, do, q, sx, add):
    """The sum is exact; the two scales' product, the conversion of the sum, their product and, where added, the addition round once each."""
    for a, b, old, d in zip(w, s, o, do):
        B, M = q.shape[0], a.shape[0]
        y = (q.astype(np.float64) @ a.astype(np.float64).T) * b.astype(np.float64)[None] * sx.astype(np.float64)[:, None]
        want = old.astype(np.float64)
        want[:, :M] = y + (want[:, :M] if add else 0)
        got = be.download(d, np.float32, old.size).reshape(old.shape)
        assert np.array_equal(got[:, M:], old[:, M:])
        tol = 3.01 * HALF * np.abs(y) + (HALF * 1.01 * np.abs(want[:, :M]) if add else 0)
        bad = ~(np.abs(got[:, :M] - want[:, :M]) <= tol)
        assert not bad.any(), (np.argwhere(bad)[:5], bad.sum())


@pytest.mark.parametrize("N,B", [(1, 1), (7, 3), (128, 2), (4096, 5), (4099, 33), (14336, 2), (131072, 1), (16400, 4)])
def test_rows_are_quantised_as_the_formula_says(backend, N, B):
    be, rng = backend, np.random.default_rng(N)
    x = rng.standard_normal((B, N), dtype=np.float32) * np.exp(3 * rng.standard_normal((B, 1))).astype(np.float32)
    x[0, : N // 2] = np.float32(0.5)                          # ties
    x[0, 0] = np.float32(127)
    q, s = quantise(x)
    dx, dq, ds = be.upload(x), be.alloc(B * N), be.alloc(B * 4)
    be._check(be.lib.ibcu_quantize_rows_int8(be.ctx, dx.ptr, dq.ptr, ds.ptr, N, B)); be.sync()
    assert np.array_equal(be.download(dq, np.int8, B * N).reshape(B, N), q) and np.array_equal(be.download(ds, np.float32, B), s)


def test_rows_out_of_the_ordinary(backend):
    """Zeros, tiny and huge rows, Inf and NaN; a token that holds one of those gives NaN everywhere and leaves the others alone."""
    be, rng = backend, np.random.default_rng(0)
    N, M = 300, 70
    x = rng.standard_normal((8, N), dtype=np.float32)
    x[0] = 0; x[1] *= np.float32(1e-35); x[2] *= np.float32(1e-28); x[3] *= np.float32(1e37); x[4, 7] = np.inf; x[5, 299] = np.nan; x[6, 0] = -np.inf
    q, s = quantise(x)
    dx, dq, ds = be.upload(x), be.alloc(8 * N), be.alloc(8 * 4)
    be._check(be.lib.ibcu_quantize_rows_int8(be.ctx, dx.ptr, dq.ptr, ds.ptr, N, 8)); be.sync()
    assert np.array_equal(be.download(dq, np.int8, 8 * N).reshape(8, N), q)
    assert np.array_equal(be.download(ds, np.float32, 8), s, equal_nan=True)
    t, w, sc, o, do = tensors(be, rng, [M], N, 8)
    be._check(be.lib.ibcu_linear_w8a8_fp32(be.ctx, t, 1, dx.ptr, N, 8)); be.sync()
    got = be.download(do[0], np.float32, 8 * M).reshape(8, M)
    assert np.isnan(got[4:7]).all() and not got[:2].any()
    want = (q.astype(np.float64) @ w[0].astype(np.float64).T) * sc[0].astype(np.float64) * s.astype(np.float64)[:, None]
    rows = [2, 3, 7]
    assert np.all(np.abs(got[rows] - want[rows]) <= 3.01 * HALF * np.abs(want[rows]) + 1e-44)


SHAPES = [((1,), 1, 1), ((128,), 128, 1), ((64, 16, 16), 256, 1), ((4096,), 4096, 1), ((4096, 1024, 1024), 4096, 7), ((1003,), 2056, 37), ((130,), 4100, 16), ((257,), 129, 200), ((3,), 14336, 9),
          ((300, 1, 129, 40), 512, 65), ((512,), 1024, 256), ((1100,), 640, 515), ((128, 384), 2048, 130), ((40,), 131072, 3), ((5632,), 2048, 24), ((32000,), 256, 2)]


@pytest.mark.parametrize("Ms,N,B", SHAPES)
@pytest.mark.parametrize("fp32,add,extra", [(False, False, 0), (True, True, 3)])
def test_products(backend, Ms, N, B, fp32, add, extra):
    """Rows, columns and tokens that end anywhere in a tile, one tensor to four, the largest sums; both forms of the call, same bits."""
    be, rng = backend, np.random.default_rng(N + B)
    x = rng.standard_normal((B, N), dtype=np.float32)
    x[-1] = 127 if N > 100000 else x[-1]                      # 127 * -128 * 131072 is the largest sum there is
    q, sx = quantise(x)
    dx, dq, ds = be.upload(x), be.upload(q), be.upload(sx)
    outs = []
    for form in range(2):
        state = rng.bit_generator.state
        t, w, s, o, do = tensors(be, rng, Ms, N, B, fp32, extra, add)
        rng.bit_generator.state = state
        be._check(be.lib.ibcu_linear_w8a8_fp32(be.ctx, t, len(Ms), dx.ptr, N, B) if form else be.lib.ibcu_linear_w8a8(be.ctx, t, len(Ms), dq.ptr, ds.ptr, N, B)); be.sync()
        check(be, w, s, o, do, q, sx, add)
        outs.append([be.download(d, np.float32, a.size) for d, a in zip(do, o)])
    for a, b in zip(*outs):
        assert np.array_equal(a, b)


@pytest.mark.parametrize("off_w,off_x", [(1, 0), (0, 3), (8, 4)])
def test_operands_at_any_address(backend, off_w, off_x):
    """A slice of a tensor's columns is not one, but a tensor may begin anywhere."""
    be, rng = backend, np.random.default_rng(3)
    M, N, B = 200, 512, 20
    w, x = rng.integers(-128, 128, (M, N), dtype=np.int8), rng.integers(-127, 128, (B, N), dtype=np.int8)
    s, sx = rng.uniform(0.001, 0.01, M).astype(np.float16), rng.uniform(0.01, 0.1, B).astype(np.float32)
    dw, dx, do = be.alloc(w.nbytes + 16), be.alloc(x.nbytes + 16), be.upload(np.zeros((B, M), np.float32))
    be.write(dw, w, off_w); be.write(dx, x, off_x)
    t = (LinearT * 1)(LinearT(dw.at(off_w), be.upload(s).ptr, do.ptr, M, M, 0, 0))
    be._check(be.lib.ibcu_linear_w8a8(be.ctx, t, 1, dx.at(off_x), be.upload(sx).ptr, N, B)); be.sync()
    check(be, [w], [s], [np.zeros((B, M), np.float32)], [do], x, sx, False)


def test_many_tokens(backend):
    """More tokens than a grid's second dimension has blocks."""
    be, rng = backend, np.random.default_rng(4)
    M, N, B = 24, 32, 70001
    x = rng.standard_normal((B, N), dtype=np.float32)
    q, sx = quantise(x)
    t, w, s, o, do = tensors(be, rng, [M], N, B)
    be._check(be.lib.ibcu_linear_w8a8_fp32(be.ctx, t, 1, be.upload(x).ptr, N, B)); be.sync()
    check(be, w, s, o, do, q, sx, False)


def test_captured_and_replayed(backend):
    """A captured call computes from what its inputs hold when it is replayed, and a larger call in between does not disturb it."""
    import ctypes as C
    be, rng = backend, np.random.default_rng(6)
    M, N, B = 260, 1000, 40
    t, w, s, o, do = tensors(be, rng, [M], N, B)
    big, *_ = tensors(be, rng, [300], 2000, 90)
    dbig = be.upload(rng.standard_normal((90, 2000), dtype=np.float32))
    x = [rng.standard_normal((B, N), dtype=np.float32) for _ in range(3)]
    dx = be.upload(x[0])
    call = lambda: be._check(be.lib.ibcu_linear_w8a8_fp32(be.ctx, t, 1, dx.ptr, N, B))
    call(); be.sync()
    gid = C.c_int()
    be._check(be.lib.ibcu_graph_begin(be.ctx)); call(); be._check(be.lib.ibcu_graph_end(be.ctx, C.byref(gid)))
    try:
        for i in (1, 2):
            be.write(dx, x[i])
            be._check(be.lib.ibcu_linear_w8a8_fp32(be.ctx, big, 1, dbig.ptr, 2000, 90))
            be._check(be.lib.ibcu_graph_launch(be.ctx, gid)); be.sync()
            check(be, w, s, o, do, *quantise(x[i]), False)
    finally:
        be._check(be.lib.ibcu_graph_destroy(be.ctx, gid))


def run_both(be, rng, Ms, N, B, add, extra, fp32=False):
    x = rng.standard_normal((B, N), dtype=np.float32)
    q, sx = quantise(x)
    for form in range(2):
        t, w, s, o, do = tensors(be, rng, Ms, N, B, fp32, extra, add)
        be._check(be.lib.ibcu_linear_w8a8_fp32(be.ctx, t, len(Ms), be.upload(x).ptr, N, B) if form else be.lib.ibcu_linear_w8a8(be.ctx, t, len(Ms), be.upload(q).ptr, be.upload(sx).ptr, N, B)); be.sync()
        check(be, w, s, o, do, q, sx, add)


@pytest.mark.parametrize("Ms,N,B,add,extra", [((5000, 5000), 1040, 700, False, 1), ((14336,), 256, 512, True, 0), ((2300, 257, 5, 4000), 1153, 1027, False, 0), ((8192,), 4096, 257, True, 7)])
def test_large_products(backend, Ms, N, B, add, extra):
    """Tiles by pairs of blocks, with row tiles and tokens that end inside one."""
    run_both(backend, np.random.default_rng(B), Ms, N, B, add, extra)


@pytest.mark.parametrize("Ms,N", [((9000,), 512), ((70, 3, 2000), 4112), ((1, 1, 1, 1), 16), ((4737,), 1024), ((2048,), 8192), ((33, 900), 16400)])
@pytest.mark.parametrize("B", [1, 2, 3, 4])
def test_few_tokens(backend, Ms, N, B):
    run_both(backend, np.random.default_rng(N + B), Ms, N, B, B % 2 == 0, B - 1, B == 3)


def test_a_row_that_is_not_finite_stays_alone_among_few(backend):
    be, rng = backend, np.random.default_rng(9)
    M, N, B = 300, 512, 4
    x = rng.standard_normal((B, N), dtype=np.float32)
    x[1, 5], x[2] = np.inf, 0
    q, sx = quantise(x)
    t, w, s, o, do = tensors(be, rng, [M], N, B)
    be._check(be.lib.ibcu_linear_w8a8_fp32(be.ctx, t, 1, be.upload(x).ptr, N, B)); be.sync()
    got = be.download(do[0], np.float32, B * M).reshape(B, M)
    assert np.isnan(got[1]).all() and not got[2].any()
    want = (q.astype(np.float64) @ w[0].astype(np.float64).T) * s[0].astype(np.float64) * sx.astype(np.float64)[:, None]
    assert np.all(np.abs(got[[0, 3]] - want[[0, 3]]) <= 3.01 * HALF * np.abs(want[[0, 3]]))
