"""Infinite operands of the F32 GEMM and of linear_fwd / linear_bwd: infinity for
infinity and NaN for NaN of what 64-bit arithmetic on the same operands gives,
on every path (tensor cores and FFMA)."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

INF = np.inf


@pytest.fixture(scope="module")
def be():
    from orcaml_b200.backend import CudaBackend
    b = CudaBackend(0)
    yield b
    b.close()


def fill(n):
    """Values of 8 to 24 significant bits, zero, and values toward the ends of the range (below 2^-137
    the high part of a split value is zero)."""
    v = np.array([1.0, -1.0, 0.5, -2.0, 1 + 2.0 ** -9, -(1 + 2.0 ** -9 + 2.0 ** -18), 0.0, 3.0, -7.0, 1 / 3, 1e30, -1e-30,
                  1e-37, -1e-39, 2.0 ** -134, -(2.0 ** -136)], np.float64)
    return np.resize(v, n).astype(np.float32)


def product(a, b):
    """Rows of a times b in 64 bits, each product by itself."""
    with np.errstate(invalid="ignore", over="ignore"):
        return (a.astype(np.float64)[:, :, None] * b.astype(np.float64)[None]).sum(1)


def same_specials(got, want):
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.array_equal(np.isinf(got), np.isinf(want))
    assert np.array_equal(got[np.isinf(want)], want[np.isinf(want)].astype(np.float32))


def operands(m, k, n, rng):
    a = rng.standard_normal((m, k)).astype(np.float32)
    b = rng.standard_normal((k, n)).astype(np.float32)
    b[3], b[5] = fill(n), -fill(n)
    a[:, 3], a[:, 5] = np.clip(a[:, 3], -1, 1), np.clip(a[:, 5], -1, 1)
    a[0, 3], a[1, 5] = INF, -INF
    a[2, 3] = a[2, 5] = INF
    a[3, 4], a[3, 6] = INF, -INF
    b[7, :4] = [INF, -INF, 0.0, np.nan]
    a[0, 7], a[1, 7] = 1.0, 0.5
    a[4, 7] = INF
    return a, b


@pytest.mark.parametrize("path", [1, 2, 3, 4])
@pytest.mark.parametrize("a_mn,b_mn", [(False, False), (False, True), (True, True)])
@pytest.mark.parametrize("m,k,n", [(64, 64, 64), (1024, 96, 1024)])
def test_gemm(be, m, k, n, a_mn, b_mn, path):
    a, b = operands(m, k, n, np.random.default_rng(m + n))
    ab = be.from_f32_slice(list(a.T.shape if a_mn else a.shape), np.ascontiguousarray(a.T if a_mn else a))
    bb = be.from_f32_slice(list(b.shape if b_mn else b.T.shape), np.ascontiguousarray(b if b_mn else b.T))
    got = be.to_f32_vec(be.gemm_ex(m, n, k, ab, a_mn, bb, b_mn, path)).reshape(m, n)
    same_specials(got[:6], product(a[:6], b))
    assert np.isfinite(got[6:, 4:]).all()


@pytest.mark.parametrize("relu", [False, True])
@pytest.mark.parametrize("m,k,n", [(8, 40, 24), (1024, 96, 1024)])
def test_linear_fwd(be, m, k, n, relu):
    a, b = operands(m, k, n, np.random.default_rng(m))
    got = be.to_f32_vec(be.linear_fwd(be.from_f32_slice([m, k], a), be.from_f32_slice([k, n], b), None, m, k, n, relu=relu))
    got, want = got.reshape(m, n)[:6], product(a[:6], b)
    if relu:
        want = np.where(want > 0, want, 0.0)
    same_specials(got, want)


@pytest.mark.parametrize("m,k,n", [(8, 40, 24), (1024, 1024, 96)])
def test_linear_bwd(be, m, k, n):
    """dx under an infinite pre-activation of the layer below, dw of an infinite activation."""
    rng = np.random.default_rng(m)
    x, w, dy = (rng.standard_normal(s).astype(np.float32) for s in ((m, k), (k, n), (m, n)))
    x[2, 7], x[3] = INF, fill(k)
    dy[2], dy[3, 5] = fill(n), -INF
    w[:, 5] = fill(k)
    up = [be.from_f32_slice(list(v.shape), v) for v in (x, w, dy)]
    dx, dw, db = (be.to_f32_vec(v) for v in be.linear_bwd(*up, m, k, n, mask=up[0]))
    dx, dw = dx.reshape(m, k), dw.reshape(k, n)
    want = np.where(x[2:4] > 0, product(dy[2:4], w.T), 0.0)
    same_specials(dx[2:4], want)
    assert dx[2, 7] != 0.0
    same_specials(dw[7:8], product(x.T[7:8], dy))
    same_specials(dw[:, 5:6], product(x.T, dy[:, 5:6]))
    assert db[5] == -INF


def test_planes_that_pass_through_the_optimizer(be):
    """A parameter that overflows stays an infinity: p - lr * g of the largest values."""
    p = be.from_f32_slice([4], np.array([-3e38, 3e38, 1.0, -1e-40], np.float32))
    g = be.from_f32_slice([4], np.array([3e38, -3e38, 0.0, 0.0], np.float32))
    be.sgd_step(p, g, None, 1.0)
    assert np.array_equal(be.to_f32_vec(p), np.array([-INF, INF, 1.0, -1e-40], np.float32))
