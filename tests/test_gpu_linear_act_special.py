"""Infinite operands of the feed-forward operators: what 64-bit arithmetic on
the same operands gives, infinity for infinity and NaN for NaN, for each type,
activation and kind of product.  No tolerances: only the places and signs of
infinities and NaN are compared, and those follow from the operands alone."""
import math

import pytest

torch = pytest.importorskip("torch")

from tests.test_gpu_linear_act import TYPES, act64, be, gen_of, rand, sp  # noqa: E402,F401

pytestmark = pytest.mark.gpu

# One token and a few rows, whole and ragged tiles of many rows, rows whose
# starts are not 16-byte aligned.
SHAPES = [(4, 64, 64), (5, 200, 136), (300, 72, 264), (1100, 264, 1288), (1100, 265, 1287), (2320, 264, 2312)]


def values(t):
    """Values of 8, 16 and 24 significant bits, zero, and the extremes of the type's range."""
    v = [1.0, -1.0, 0.5, -2.0, 1 + 2.0 ** -9, -(1 + 2.0 ** -9 + 2.0 ** -18), 0.0, 3.0, -7.0, 1 / 3]
    if t == torch.float16:
        return v + [3e4, -6e-8]
    return v + [1e30, -1e-30, 1e-37, -1e-39] + ([2.0 ** -134, -(2.0 ** -149)] if t == torch.float32 else [])


def fill(n, t):
    v = torch.tensor(values(t), dtype=torch.float64)
    return v.repeat(n // len(v) + 1)[:n].to(t).cuda()


def same_specials(name, got, want):
    got = got.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{name}: NaN in other places"
    inf = torch.isinf(want)
    assert torch.equal(torch.isinf(got), inf), f"{name}: infinities in other places"
    assert torch.equal(got[inf], want[inf]), f"{name}: infinities of the other sign"


def product(a, b):
    """The rows of a times b in 64 bits, each product by itself."""
    return (a.double()[:, :, None] * b.double()[None]).sum(1)


@pytest.mark.parametrize("act", ["none", "relu", "gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("m,k,n", SHAPES)
@pytest.mark.parametrize("kind", list(TYPES))
def test_forward(be, kind, m, k, n, act):  # noqa: F811
    t = TYPES[kind]
    g = gen_of(m + n)
    x, w = rand(g, m, k, t=t), rand(g, k, n, scale=k ** -0.5, t=t)
    w[3], w[5] = fill(n, t), -fill(n, t)
    x[:, 3] = x[:, 3].clamp(-1, 1)
    x[0, 3] = math.inf
    x[1, 5] = -math.inf
    x[m - 1, 3], x[m - 1, 5] = math.inf, math.inf      # opposite infinities: NaN
    out, z = torch.empty(m, n, dtype=t, device="cuda"), torch.empty(m, n, dtype=t, device="cuda")
    be.linear_act_fwd(sp(be, x), sp(be, w), None, m, k, n, act=act, keep="z", out=sp(be, out), z=sp(be, z))
    rows = [0, 1, m - 1]
    z64 = product(x[rows], w)
    assert torch.isinf(z64[:2]).any() and torch.isnan(z64[2]).any()
    same_specials("z", z[rows], z64)
    want = act64(z64, act)
    if act in ("none", "relu"):
        same_specials("out", out[rows], want)
        assert torch.equal(out[rows][want == 0], want[want == 0].to(t))
    else:                                              # (far below zero they tend to 0)
        up = z64 != -math.inf
        same_specials("out", out[rows][up], want[up])
    rest = [i for i in range(m) if i not in rows]
    if t != torch.float16:                             # 3e4 times a few can pass F16's range
        assert torch.isfinite(out[rest]).all()


@pytest.mark.parametrize("m,k,n", [(4, 64, 64), (5, 200, 136), (300, 264, 72), (1100, 1288, 264), (1100, 1287, 265)])
@pytest.mark.parametrize("kind", list(TYPES))
def test_backward(be, kind, m, k, n):  # noqa: F811
    t = TYPES[kind]
    g = gen_of(m + k)
    x, w, dy = rand(g, m, k, t=t), rand(g, k, n, scale=n ** -0.5, t=t), rand(g, m, n, t=t)
    w[:, 3] = fill(k, t)
    x[2] = fill(k, t)
    dy[2, 3] = -math.inf
    dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty_like(dy[0])
    be.linear_act_bwd(sp(be, x), sp(be, w), sp(be, dy), m, k, n, dx=sp(be, dx), dw=sp(be, dw), db=sp(be, db))
    same_specials("dx", dx[2:3], product(dy[2:3], w.t()))
    same_specials("dw", dw[:, 3:4], product(x.t(), dy[:, 3:4]))
    assert db[3] == -math.inf
    # An infinite activation under finite gradients of few significant bits.
    dy = rand(g, m, n, t=t)
    dy[2] = fill(n, t)
    x[2, 7] = math.inf
    be.linear_act_bwd(sp(be, x), sp(be, w), sp(be, dy), m, k, n, dw=sp(be, dw), need_dx=False, need_db=False)
    same_specials("dw", dw[7:8], product(x.t()[7:8], dy))


@pytest.mark.parametrize("rows", [1, 300])
def test_both_operands_infinite(be, rows):  # noqa: F811
    """Infinity times infinity, by sign, in F32 (whose operands are split)."""
    m, k, n = rows, 64, 64
    x, w = torch.ones(m, k, device="cuda"), torch.ones(k, n, device="cuda")
    x[0, 9] = math.inf
    w[9, 0], w[9, 1], w[9, 2], w[9, 3] = math.inf, -math.inf, 0.0, math.nan
    out = torch.empty(m, n, device="cuda")
    be.linear_act_fwd(sp(be, x), sp(be, w), None, m, k, n, out=sp(be, out))
    assert out[0, 0] == math.inf and out[0, 1] == -math.inf
    assert torch.isnan(out[0, 2:4]).all() and (out[0, 4:] == math.inf).all()
    if m > 1:
        assert (out[1:, 0] == math.inf).all() and (out[1:, 1] == -math.inf).all()
        assert torch.equal(out[1:, 4:], torch.full_like(out[1:, 4:], k))


@pytest.mark.parametrize("m,n", [(3, 33), (64, 40), (5, 31)])
def test_new_checkpoints_have_all_their_bytes(be, m, n):  # noqa: F811
    """Storages that the calls make, in memory that held other bytes before."""
    import numpy as np
    from tests.test_gpu_linear_act import encode
    x = rand(gen_of(m), m, n)
    size = be.ckpt8_bytes(m, n)
    for _ in range(3):
        dirty = be.from_bytes([size], b"\xff" * size, 6)
        del dirty
        ck = be.ckpt8_pack(sp(be, x), m, n)
        assert np.array_equal(np.frombuffer(be.to_bytes(ck), np.uint8), encode(x))
        del ck


def test_empty_storage(be):  # noqa: F811
    from orcaml_b200 import _lib as L
    s = be.empty([3, 5])
    assert len(s) == 15 and s.device_ptr
    assert len(be.empty([0, 4])) == 0
    with pytest.raises(L.OrcaError):
        be.empty([3, -1])


@pytest.mark.parametrize("act,below", [("relu", 0.0), ("gelu", 0.0), ("gelu_tanh", math.nan), ("silu", math.nan)])
@pytest.mark.parametrize("kind", list(TYPES))
def test_activations_and_slopes_at_infinities(be, kind, act, below):  # noqa: F811
    """As the header says: +inf stays, -inf gives 0 or NaN, slopes are NaN but ReLU's."""
    t = TYPES[kind]
    z = torch.tensor([math.inf, -math.inf, math.nan, 1.0] * 40, device="cuda").to(t)
    none, one = be.span(None, 0, sp(be, z).dtype), torch.ones(1, device="cuda").to(t)
    out, dx = torch.empty_like(z), torch.empty_like(z)
    be.linear_act_fwd(none, none, sp(be, z), 1, 0, len(z), act=act, out=sp(be, out))
    be.linear_act_bwd(sp(be, z), sp(be, one), sp(be, torch.ones_like(z)), len(z), 1, 1, act=act, dx=sp(be, dx), need_dw=False,
                      need_db=False)
    nan = math.nan
    want = [math.inf, below, 0.0 if act == "relu" else nan]
    slope = [1.0, 0.0, 0.0] if act == "relu" else [nan, nan, nan]
    for got, w in ((out, want), (dx, slope)):
        got = got.view(-1, 4)[:, :3].float()
        w = torch.tensor(w, device="cuda").expand_as(got)
        assert torch.equal(torch.nan_to_num(got, nan=7.0, posinf=8.0), torch.nan_to_num(w, nan=7.0, posinf=8.0))
