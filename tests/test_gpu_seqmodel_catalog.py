"""GPU: the sequence-model kernels as a compiled DAPHNE program reaches them - looked up in HIPcatalog.json by op mnemonic,
result and argument types, called with run-time objects - against plain numpy in 64 bits. The kernels' edge cases are in
test_gpu_seqmodel.py; this covers the layer above (shapes, results made by the kernel, placements, refusals)."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

F32, F64 = np.float32, np.float64
CPP = {np.dtype(F32): "float", np.dtype(F64): "double", np.dtype(np.int64): "int64_t", np.dtype(np.int8): "int8_t", np.dtype(np.uint8): "uint8_t"}


def dm(dt):
    return f"DenseMatrix<{CPP[np.dtype(dt)]}>"


@pytest.fixture(scope="module")
def rt():
    from catalog_caller import Runtime

    r = Runtime()
    yield r
    r.close()


def by_catalog(rt, mnemonic, res, args, *values):
    return rt.call(rt.find(mnemonic, res, args)["kernelFuncName"], *values)


def U(dt):
    return float(np.finfo(dt).eps) / 2


@pytest.mark.parametrize("dt", [F32, F64])
def test_embedding(rt, dt):
    rng = np.random.default_rng(1)
    table, ids, d = rng.standard_normal((30, 21)).astype(dt), rng.integers(0, 30, (50, 1)), rng.standard_normal((50, 21)).astype(dt)
    T, I, D = rt.matrix(table), rt.matrix(ids), rt.matrix(d)
    scalar = CPP[np.dtype(dt)]
    res = by_catalog(rt, "embeddingForward", [dm(dt)], [dm(dt), dm(np.int64), scalar], T, I, dt(0.5))
    assert res.where() == 2
    np.testing.assert_array_equal(res.to_numpy(), table[ids[:, 0]] * dt(0.5))
    g = by_catalog(rt, "embeddingBackward", [dm(dt)], [dm(dt), dm(np.int64), "size_t", scalar], D, I, 30, dt(2))
    want = np.zeros((30, 21), np.longdouble)
    np.add.at(want, ids[:, 0], d.astype(np.longdouble))
    mag = np.zeros((30, 21))
    np.add.at(mag, ids[:, 0], np.abs(d.astype(F64)))
    assert np.all(np.abs(g.to_numpy() - 2 * want) <= 52 * 2.0**-53 * 2 * mag + U(dt) * np.abs(2 * want) * 1.001)
    for m in (T, I, D, res, g):
        m.destroy()


@pytest.mark.parametrize("dt", [F32, F64])
def test_rms_norm_and_its_gradient(rt, dt):
    rng = np.random.default_rng(2)
    x, r, dy, ds = (rng.standard_normal((7, 33)).astype(dt) for _ in range(4))
    g = (1 + rng.random((1, 33))).astype(dt)
    X, R, G, DY, DS = (rt.matrix(a) for a in (x, r, g, dy, ds))
    y, s, inv = by_catalog(rt, "rmsNormForward", [dm(dt)] * 3, [dm(dt)] * 3 + [CPP[np.dtype(dt)]], X, R, G, dt(1e-5))
    h = x + r
    w = np.longdouble
    i = 1 / np.sqrt((h.astype(w) ** 2).mean(axis=1, keepdims=True) + w(dt(1e-5)))
    np.testing.assert_array_equal(s.to_numpy(), h)
    tol = (33 / 2 + 3) * 2.0**-53 + 3 * U(dt)
    assert np.all(np.abs(inv.to_numpy() - i) <= tol * i) and np.all(np.abs(y.to_numpy() - h * i * g) <= tol * np.abs(h * i * g) * 1.001)
    dx, dg = by_catalog(rt, "rmsNormBackward", [dm(dt)] * 2, [dm(dt)] * 5, s, inv, G, DY, DS)
    ii, u = inv.to_numpy().astype(w), dy.astype(w) * g
    k = ii * ii * (u * h).mean(axis=1, keepdims=True)
    mag = ii * (np.abs(u) + np.abs(h * k)) + np.abs(ds)
    assert np.all(np.abs(dx.to_numpy() - (ii * (u - h * k) + ds)) <= 6 * U(dt) * mag * 1.001 + 37 * 2.0**-53 * mag * 33)
    want = (dy * h * ii).sum(axis=0, keepdims=True)
    assert np.all(np.abs(dg.to_numpy() - want) <= (2 * U(dt) + 11 * 2.0**-53) * np.abs(dy * h * ii).sum(axis=0, keepdims=True) * 1.001)
    for m in (X, R, G, DY, DS, y, s, inv, dx, dg):
        m.destroy()


@pytest.mark.parametrize("dt", [F32, F64])
def test_gated_recurrence_and_its_gradient(rt, dt):
    rng = np.random.default_rng(3)
    n, c = 40, 9
    x, z, d = (rng.standard_normal((n, c)).astype(dt) for _ in range(3))
    h0, dl = rng.standard_normal((3, c)).astype(dt), rng.standard_normal((3, c)).astype(dt)
    starts = np.array([[0], [25], [25], [40]])
    X, Z, D, H0, DL, O = (rt.matrix(a) for a in (x, z, d, h0, dl, starts))
    res, last = by_catalog(rt, "gatedRecurrenceForward", [dm(dt)] * 2, [dm(dt)] * 3 + [dm(np.int64)], X, Z, H0, O)
    f = 1 / (1 + np.exp(-z.astype(F64)))
    h, ends = np.zeros((n, c)), h0.astype(F64)
    for s, (a, e) in enumerate(((0, 25), (25, 25), (25, 40))):
        for t in range(a, e):
            h[t] = f[t] * (h[t - 1] if t > a else h0[s]) + (1 - f[t]) * x[t]
        if e > a:
            ends[s] = h[e - 1]
    # at most 25 steps of two roundings and two gates (8 half steps and |z| each) of terms below 4
    tol = 25 * (2 + 2 * 14) * U(dt) * 4
    np.testing.assert_allclose(res.to_numpy(), h, rtol=0, atol=tol)
    np.testing.assert_allclose(last.to_numpy(), ends, rtol=0, atol=tol)
    dx, dz, dh0 = by_catalog(rt, "gatedRecurrenceBackward", [dm(dt)] * 3, [dm(dt)] * 6 + [dm(np.int64)], X, Z, res, H0, D, DL, O)
    gx, gz, g0 = np.zeros((n, c)), np.zeros((n, c)), dl.astype(F64)
    for s, (a, e) in enumerate(((0, 25), (25, 25), (25, 40))):
        for t in range(e - 1, a - 1, -1):
            g = d[t] + g0[s]
            gx[t], gz[t] = (1 - f[t]) * g, g * ((h[t - 1] if t > a else h0[s]) - x[t]) * f[t] * (1 - f[t])
            g0[s] = f[t] * g
    for got, want in ((dx, gx), (dz, gz), (dh0, g0)):
        np.testing.assert_allclose(got.to_numpy(), want, rtol=0, atol=16 * tol)  # G sums terms below 4 of up to 25 rows: below 16 here
    for m in (X, Z, D, H0, DL, O, res, last, dx, dz, dh0):
        m.destroy()


def test_quantised_weights(rt):
    rng = np.random.default_rng(4)
    w, x, r = rng.standard_normal((40, 96)).astype(F32), rng.standard_normal((3, 96)).astype(F32), rng.standard_normal((3, 96)).astype(F32)
    g = np.ones((1, 96), F32)
    W, X, R, G = rt.matrix(w), rt.matrix(x), rt.matrix(r), rt.matrix(g)
    codes, scales = by_catalog(rt, "quantizeQ4", [dm(np.uint8), dm(F32)], [dm(F32), "size_t"], W, 32)
    c = codes.to_numpy().astype(np.int64)
    c = ((np.stack((c & 15, c >> 4), -1).reshape(40, 96) ^ 8) - 8) * np.repeat(scales.to_numpy().astype(F64), 32, axis=1)
    assert np.all(np.abs(c - w) <= np.repeat(scales.to_numpy(), 32, axis=1) * 0.5001)
    y = by_catalog(rt, "matVecQ4", [dm(F32)], [dm(F32), dm(np.uint8), dm(F32), "size_t"], X, codes, scales, 32)
    mag = np.abs(x.astype(F64)) @ np.abs(c).T
    assert np.all(np.abs(y.to_numpy() - x.astype(F64) @ c.T) <= 32 * U(F32) * mag)
    q, qs, s, inv = by_catalog(rt, "rmsNormForwardQ8", [dm(np.int8)] + [dm(F32)] * 3, [dm(F32)] * 3 + ["float"], X, R, G, F32(1e-5))
    h = x + r
    most = np.abs(h).astype(F64).max(axis=1, keepdims=True)
    np.testing.assert_array_equal(q.to_numpy(), np.rint(h.astype(F64) * (127 / most)).astype(np.int8))
    y8 = by_catalog(rt, "matVecQ4Q8", [dm(F32)], [dm(np.int8), dm(F32), dm(np.uint8), dm(F32), "size_t"], q, qs, codes, scales, 32)
    xq = q.to_numpy().astype(F64) * qs.to_numpy()
    assert np.all(np.abs(y8.to_numpy() - xq @ c.T) <= 32 * U(F32) * (np.abs(xq) @ np.abs(c).T))
    for m in (W, X, R, G, codes, scales, y, q, qs, s, inv, y8):
        m.destroy()


def test_refusals_are_exceptions(rt):
    """A C++ exception must not cross ctypes: these calls go through the harness, which catches it and keeps its text."""
    import ctypes as C

    h = rt.harness
    for name in ("embedding", "rmsnorm", "recurrence", "q4"):
        getattr(h, f"th_seq_{name}").argtypes = [C.c_void_p] * 4

    def refused(name, match, *ms):
        assert getattr(h, f"th_seq_{name}")(rt.ctx, *[m.h for m in ms]) == 1
        assert match in h.th_last_error().decode()

    x, g, ids = rt.matrix(np.ones((4, 32), F32)), rt.matrix(np.ones((1, 31), F32)), rt.matrix(np.array([[3], [4]]))
    bad, two = rt.matrix(np.array([[0], [3], [2], [4]])), rt.matrix(np.zeros((2, 2), np.int64))
    refused("embedding", "'4'", x, ids, x)
    refused("embedding", "ids is 2 x 2", x, two, x)
    refused("rmsnorm", "gamma", x, x, g)
    refused("rmsnorm", "residual is 1 x 31", x, g, g)
    refused("recurrence", "offset", x, x, bad)
    refused("recurrence", "z is 1 x 31", x, g, bad)
    refused("q4", "multiple of 32", x, x, x)
    for m in (x, g, ids, bad, two):
        m.destroy()
