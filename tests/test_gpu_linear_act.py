"""The feed-forward operators against plain 64-bit forms: linear with activation
and residual, forward and backward, and the 8-bit activation checkpoints.

Tolerances, all derived from the number formats:
  * a result rounded once to type t is off by at most u_t = finfo(t).eps / 2 of
    its value;
  * the F32 sums over K products are off by at most g(K) * sum |a||b|.  An
    accumulator step of the tensor core (16 products) loses less than 2^-22 of
    the magnitudes summed so far, so g = 2^-22 * (K / 16 + 16) covers one chain;
    F32 operands are summed in chains of 24 steps that are joined in F32;
  * activations have slopes of at most 1.13 (GELU's maximum is 1.129), slopes
    change by at most 0.81 per unit (GELU's second derivative at 0 is 0.798),
    and F32 evaluations are off by a few units of 2^-24.
"""
import ctypes
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
GROUP = 32


@pytest.fixture(scope="module")
def be():
    from orcaml_b200.backend import CudaBackend
    b = CudaBackend(0, stream=torch.cuda.current_stream().cuda_stream)
    yield b
    torch.cuda.synchronize()
    b.close()


def code_of(t):
    from orcaml_b200.backend import BF16, F16, F32, U8
    return {torch.bfloat16: BF16, torch.float16: F16, torch.float32: F32, torch.uint8: U8}[t]


def sp(be, t):
    if t is None:
        return None
    s = be.span(t.data_ptr(), t.numel(), code_of(t.dtype))
    s.owner = t          # alive as long as the span
    return s


def rand(gen, *shape, scale=1.0, t=torch.float32):
    return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(t)


def gen_of(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


# ---------------------------------------------------------------- 64-bit forms
def act64(z, act):
    if act == "relu":
        return torch.where(z > 0, z, 0.0)
    if act == "gelu":
        return 0.5 * z * torch.erfc(-z / math.sqrt(2))
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    if act == "silu":
        return z * torch.sigmoid(z)
    return z


def slope64(z, act):
    z = z.detach().clone().requires_grad_(True)
    if act == "none":
        return torch.ones_like(z).detach()
    return torch.autograd.grad(act64(z, act).sum(), z)[0]


def exps_at(m, n):
    return (m * n + 15) // 16 * 16


def groups_of(n):
    return (n + GROUP - 1) // GROUP


def encode(x):
    """The checkpoint's bytes of a [m, n] tensor, from the definition, in 64 bits on the CPU."""
    x = x.detach().cpu().double().numpy()
    m, n = x.shape
    codes = np.zeros((m, n), np.int8)
    exps = np.zeros((m, groups_of(n)), np.uint8)
    for g in range(groups_of(n)):
        v = x[:, g * GROUP:(g + 1) * GROUP]
        amax = np.abs(v).max(axis=1)
        fine = np.isfinite(v).all(axis=1)
        with np.errstate(divide="ignore", invalid="ignore"):
            e = np.where(amax > 0, np.frexp(np.where(fine, amax, 1.0))[1] - 1 - 6, -126)
        e = np.maximum(e, -126)
        q = np.clip(np.rint(np.where(fine[:, None], v, 0.0) * np.exp2(-e.astype(float))[:, None]), -127, 127)
        codes[:, g * GROUP:(g + 1) * GROUP] = q.astype(np.int8)
        exps[:, g] = np.where(fine, e + 127, 255)
    out = np.zeros(exps_at(m, n) + exps.size, np.uint8)
    out[:m * n] = codes.view(np.uint8).reshape(-1)
    out[exps_at(m, n):] = exps.reshape(-1)
    return out


def decode(buf, m, n):
    """Values (float64, on the GPU) and steps of a checkpoint's bytes."""
    q = buf[:m * n].view(torch.int8).view(m, n).double()
    e = buf[exps_at(m, n):exps_at(m, n) + m * groups_of(n)].view(m, groups_of(n)).double()
    step = torch.where(e == 255, math.nan, torch.exp2(e - 127))
    step = step.repeat_interleave(GROUP, dim=1)[:, :n]
    return q * step, step


def sum_error(k, t):
    if t == torch.float32:   # chains joined in F32; six products each
        return 2.0 ** -22 * 32 + 2.0 ** -24 * (6 * k / 64 / 8 + 8)
    return 2.0 ** -22 * (k / 16 + 16)


def check(name, got, want, bound):
    got = got.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{name}: NaN in other places"
    off = torch.where(torch.isnan(want), 0.0, (got - want).abs() - bound)
    worst = float(off.max()) if off.numel() else 0.0
    if worst > 0:
        i = int(off.argmax())
        raise AssertionError(f"{name}: element {i}: {got.flatten()[i]:.9g}, exact {want.flatten()[i]:.9g}, "
                             f"allowed off {bound.flatten()[i]:.3g}")


TINY = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24, torch.float32: 2.0 ** -149}


def rounding(v, t):
    return v.abs() * (torch.finfo(t).eps / 2) + TINY[t]


# ---------------------------------------------------------------- checkpoints
SHAPES8 = [(1, 1), (1, 33), (3, 31), (5, 32), (7, 40), (2, 4099), (64, 1001), (129, 1024), (300, 48)]


@pytest.mark.parametrize("m,n", SHAPES8)
@pytest.mark.parametrize("kind", list(TYPES))
def test_ckpt8_pack_is_the_definition(be, kind, m, n):
    t = TYPES[kind]
    x = rand(gen_of(m * 7 + n), m, n, scale=3.0).to(t)
    buf = torch.full((be.ckpt8_bytes(m, n) + 5,), 77, dtype=torch.uint8, device="cuda")
    assert be.ckpt8_bytes(m, n) == exps_at(m, n) + m * groups_of(n)
    buf[m * n:exps_at(m, n)] = 0
    be.ckpt8_pack(sp(be, x), m, n, out=sp(be, buf))
    want = encode(x)
    got = buf.cpu().numpy()
    assert np.array_equal(got[:len(want)], want)
    assert (got[len(want):] == 77).all()
    for out_t in TYPES.values():
        back = torch.empty(m, n, dtype=out_t, device="cuda")
        be.ckpt8_unpack(sp(be, buf), m, n, out=sp(be, back))
        values, _ = decode(buf, m, n)
        if out_t != torch.float16:
            assert torch.equal(back.double(), values)          # exact in BF16 and F32
        else:
            check("f16", back, values, rounding(values, out_t))


@pytest.mark.parametrize("kind", list(TYPES))
def test_ckpt8_special_values(be, kind):
    """Zeros, signed zeros, infinities, NaN, the type's extremes, subnormals,
    ties, and values that saturate the code."""
    t = TYPES[kind]
    top, low, sub = torch.finfo(t).max, torch.finfo(t).tiny, torch.finfo(t).smallest_normal / 4
    rows = [[0.0] * 70, [-0.0] * 70, [top] * 70, [-top, 1.0] * 35, [low] * 70, [sub] * 70,
            [math.inf] + [1.0] * 69, [1.0] * 40 + [math.nan] + [2.0] * 29, [-math.inf] * 70,
            [1.0, 0.5 / 64, 1.5 / 64, 2.5 / 64, -0.5 / 64, -1.5 / 64] + [0.0] * 64,
            [1.9921875, -1.9921875] * 35, [0.0] * 69 + [3.0]]
    x = torch.tensor(rows, dtype=torch.float64).to(t).cuda()
    m, n = x.shape
    buf = torch.zeros(be.ckpt8_bytes(m, n), dtype=torch.uint8, device="cuda")
    be.ckpt8_pack(sp(be, x), m, n, out=sp(be, buf))
    assert np.array_equal(buf.cpu().numpy(), encode(x))
    back = torch.empty(m, n, dtype=torch.float32, device="cuda")
    be.ckpt8_unpack(sp(be, buf), m, n, out=sp(be, back))
    back = back.cpu()
    assert torch.isnan(back[6, :32]).all() and torch.equal(back[6, 32:], torch.ones(38))
    assert torch.isnan(back[7, 32:64]).all() and torch.isnan(back[8]).all()
    assert torch.equal(back[9, :6], torch.tensor([1.0, 0.0, 2 / 64, 2 / 64, 0.0, -2 / 64]))


@pytest.mark.parametrize("act", ["relu", "gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("kind", list(TYPES))
def test_ckpt8_unpack_through_an_activation(be, kind, act):
    t, m, n = TYPES[kind], 37, 208
    x = rand(gen_of(5), m, n, scale=2.0).to(t)
    ck = be.ckpt8_pack(sp(be, x), m, n)
    out = torch.empty(m, n, dtype=t, device="cuda")
    be.ckpt8_unpack(ck, m, n, act=act, out=sp(be, out))
    buf = torch.from_numpy(np.frombuffer(be.to_bytes(ck), np.uint8).copy()).cuda()
    v, _ = decode(buf, m, n)
    want = act64(v, act)
    # 1 + erf and 1 + tanh lose relative accuracy in the tail: a few 2^-24 of |v|.
    check(act, out, want, rounding(want, t) + 2.0 ** -21 * v.abs())


@pytest.mark.parametrize("offset", [1, 3, 8])
def test_ckpt8_unaligned_memory(be, offset):
    m, n = 19, 64
    base = rand(gen_of(9), m * n + 16, t=torch.bfloat16)
    x = base[offset:offset + m * n]
    raw = torch.zeros(be.ckpt8_bytes(m, n) + 16, dtype=torch.uint8, device="cuda")
    buf = raw[offset:offset + be.ckpt8_bytes(m, n)]
    be.ckpt8_pack(sp(be, x), m, n, out=sp(be, buf))
    assert np.array_equal(buf.cpu().numpy(), encode(x.view(m, n)))
    out = torch.empty(m * n + 16, dtype=torch.bfloat16, device="cuda")[offset:offset + m * n]
    be.ckpt8_unpack(sp(be, buf), m, n, out=sp(be, out))
    assert torch.equal(out.view(m, n).double(), decode(buf, m, n)[0])


# ---------------------------------------------------------------- forward
# Tokens from one to several tiles; sizes of one, below, at and above tile
# borders, and odd.
FWD_SHAPES = [(1, 1, 1), (1, 64, 32), (2, 7, 5), (1, 4096, 1024), (8, 512, 512), (17, 100, 33),
              (33, 72, 264), (64, 1000, 784), (65, 1001, 517), (100, 130, 8), (129, 256, 300),
              (256, 512, 256), (257, 192, 1032), (300, 333, 777), (640, 784, 512), (1100, 264, 1288)]


def fwd_case(be, t, m, k, n, act, residual, keep, bias=True, seed=1, offset=0):
    g = gen_of(seed + m * 31 + k * 7 + n)

    def put(v):
        if v is None or not offset:
            return v
        base = torch.zeros(v.numel() + 64, dtype=v.dtype, device="cuda")
        base[offset:offset + v.numel()] = v.reshape(-1)
        return base[offset:offset + v.numel()].view(v.shape)

    x, w = put(rand(g, m, k, t=t)), put(rand(g, k, n, scale=k ** -0.5, t=t))
    b = put(rand(g, n, scale=0.3, t=t)) if bias else None
    r = put(rand(g, m, n, t=t)) if residual else None
    guard = 40
    out = torch.full((m * n + 2 * guard,), 7.0, dtype=t, device="cuda")
    body = out[guard:guard + m * n] if not offset else out[offset:offset + m * n]
    z = None
    if keep == "z":
        z = torch.full((m * n,), 7.0, dtype=t, device="cuda")
    elif keep == "ckpt8":
        z = torch.full((be.ckpt8_bytes(m, n),), 7, dtype=torch.uint8, device="cuda")
    be.linear_act_fwd(sp(be, x), sp(be, w), sp(be, b), m, k, n, act=act, residual=sp(be, r), keep=keep,
                      out=sp(be, body), z=sp(be, z))
    rest = torch.ones_like(out, dtype=torch.bool)
    start = guard if not offset else offset
    rest[start:start + m * n] = False
    assert (out[rest] == 7.0).all(), "written outside of out"
    z64 = x.double() @ w.double() + (b.double() if bias else 0.0)
    off = sum_error(k, t) * (x.double().abs() @ w.double().abs() + (b.double().abs() if bias else 0.0))
    off = off + 2.0 ** -23 * z64.abs()
    want = act64(z64, act) + (r.double() if residual else 0.0)
    check("out", body.view(m, n), want,
          1.01 * rounding(want, t) + 1.13 * off + 2.0 ** -21 * z64.abs() + 2.0 ** -23 * want.abs())
    if keep == "z":
        check("z", z.view(m, n), z64, 1.01 * rounding(z64, t) + off)
    elif keep == "ckpt8":
        v, step = decode(z, m, n)
        check("ckpt8", v, z64, step * torch.where(v.abs() >= 127 * step, 1.0, 0.5) * 1.0001 + off)
    return x, w, b, r, body.view(m, n), z


@pytest.mark.parametrize("m,k,n", FWD_SHAPES)
@pytest.mark.parametrize("kind", list(TYPES))
def test_forward(be, kind, m, k, n):
    i = FWD_SHAPES.index((m, k, n))
    acts = ["none", "relu", "gelu", "gelu_tanh", "silu"]
    keeps = [None, "z", "ckpt8"]
    fwd_case(be, TYPES[kind], m, k, n, acts[i % 5], i % 2 == 0, keeps[i % 3])
    fwd_case(be, TYPES[kind], m, k, n, acts[(i + 2) % 5], i % 2 == 1, keeps[(i + 1) % 3], bias=i % 3 != 0)


# Sizes that reach every tiling: several rounds of 256- and of 512-row tiles, a
# last round shared along the sum by two to five clusters, long sums of few
# tiles, borders inside the tiles.
LARGE = [(4096, 8192, 4608), (2320, 4104, 2312), (1100, 8200, 1096), (300, 16384, 520), (4100, 264, 5000),
         (8192, 8192, 8192)]


@pytest.mark.parametrize("m,k,n", LARGE)
def test_forward_large(be, m, k, n):
    i = LARGE.index((m, k, n))
    fwd_case(be, torch.bfloat16, m, k, n, "gelu" if i % 2 else "none", i % 3 == 0, [None, "ckpt8", "z"][i % 3])
    if m * k * n < 2 ** 36:
        fwd_case(be, torch.float16, m, k, n, "silu", True, None)
        fwd_case(be, torch.float32, m, k, n, "gelu_tanh", True, "z")


@pytest.mark.parametrize("act", ["none", "relu", "gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("kind", list(TYPES))
def test_forward_every_activation_and_keep(be, kind, act):
    for residual in (False, True):
        for keep in (None, "z", "ckpt8"):
            fwd_case(be, TYPES[kind], 264, 96, 320, act, residual, keep)
            fwd_case(be, TYPES[kind], 5, 200, 136, act, residual, keep)


@pytest.mark.parametrize("m,k,n", [(1, 128, 256), (20, 72, 40), (300, 136, 264)])
@pytest.mark.parametrize("offset", [1, 4])
def test_forward_unaligned_memory(be, m, k, n, offset):
    fwd_case(be, torch.bfloat16, m, k, n, "gelu", True, None, offset=offset)
    fwd_case(be, torch.float32, m, k, n, "silu", True, None, offset=offset)


@pytest.mark.parametrize("kind", list(TYPES))
def test_kept_checkpoint_is_the_packed_pre_activation(be, kind):
    """F32: the checkpoint the epilogue writes is bit for bit what packing the
    kept pre-activation gives, and running again gives the same bits."""
    t = TYPES[kind]
    for m, k, n in [(3, 64, 100), (270, 160, 520), (130, 72, 33)]:
        x, w, b, _, out, ck = fwd_case(be, t, m, k, n, "gelu", False, "ckpt8")
        again = fwd_case(be, t, m, k, n, "gelu", False, "ckpt8")
        assert torch.equal(out, again[4])
        keep = m * n
        assert torch.equal(ck[:keep], again[5][:keep]) and torch.equal(ck[exps_at(m, n):], again[5][exps_at(m, n):])
        if t == torch.float32:
            z = fwd_case(be, t, m, k, n, "gelu", False, "z")[5].view(m, n)
            want = encode(z)
            got = ck.cpu().numpy()
            assert np.array_equal(got[:keep], want[:keep])
            assert np.array_equal(got[exps_at(m, n):], want[exps_at(m, n):])


def test_forward_out_may_be_the_residual(be):
    for t in TYPES.values():
        for m, k, n in [(2, 64, 96), (300, 72, 264), (33, 50, 21)]:
            g = gen_of(3)
            x, w, r = rand(g, m, k, t=t), rand(g, k, n, scale=0.1, t=t), rand(g, m, n, t=t)
            out = torch.empty(m, n, dtype=t, device="cuda")
            be.linear_act_fwd(sp(be, x), sp(be, w), None, m, k, n, act="silu", residual=sp(be, r), out=sp(be, out))
            be.linear_act_fwd(sp(be, x), sp(be, w), None, m, k, n, act="silu", residual=sp(be, r), out=sp(be, r))
            assert torch.equal(out, r)


def test_forward_infinities_and_nan_stay_in_their_row(be):
    """A row of x with a NaN or an infinity gives a row without finite values;
    its checkpoint decodes to NaN; other rows are as without it."""
    for t in TYPES.values():
        for m, k, n in [(3, 64, 64), (300, 64, 264)]:
            g = gen_of(4)
            x, w = rand(g, m, k, t=t), rand(g, k, n, t=t)
            out = torch.empty(m, n, dtype=t, device="cuda")
            be.linear_act_fwd(sp(be, x), sp(be, w), None, m, k, n, out=sp(be, out))
            x2 = x.clone()
            x2[0, 5], x2[2, 7] = math.nan, math.inf
            got = torch.empty(m, n, dtype=t, device="cuda")
            ck = torch.zeros(be.ckpt8_bytes(m, n), dtype=torch.uint8, device="cuda")
            be.linear_act_fwd(sp(be, x2), sp(be, w), None, m, k, n, keep="ckpt8", out=sp(be, got), z=sp(be, ck))
            assert torch.isnan(got[0]).all() and not torch.isfinite(got[2]).any()
            ok = [i for i in range(m) if i not in (0, 2)]
            assert torch.equal(got[ok], out[ok])
            v, _ = decode(ck, m, n)
            assert torch.isnan(v[[0, 2]]).all() and torch.isfinite(v[ok]).all()


@pytest.mark.parametrize("kind", list(TYPES))
def test_empty_sizes(be, kind):
    t = TYPES[kind]
    e = torch.empty(0, dtype=t, device="cuda")
    b = rand(gen_of(1), 40, t=t)
    out = torch.empty(3, 40, dtype=t, device="cuda")
    be.linear_act_fwd(sp(be, e), sp(be, e), sp(be, b), 3, 0, 40, act="relu", out=sp(be, out))
    assert torch.equal(out, torch.where(b > 0, b, 0.0).to(t).expand(3, 40))
    be.linear_act_fwd(sp(be, e), sp(be, b), None, 0, 8, 5, out=sp(be, e))
    be.linear_act_fwd(sp(be, b), sp(be, e), None, 5, 8, 0, out=sp(be, e))
    be.ckpt8_pack(sp(be, e), 0, 9, out=sp(be, torch.empty(0, dtype=torch.uint8, device="cuda")))
    # No rows: gradients are zero.
    dw, db = torch.ones(8, 5, device="cuda"), torch.ones(5, device="cuda")
    be.linear_act_bwd(sp(be, e), sp(be, b), sp(be, e), 0, 8, 5, dx=sp(be, e), dw=sp(be, dw), db=sp(be, db))
    assert (dw == 0).all() and (db == 0).all()
    # No outputs of the layer: dx is the residual.
    dx, r = torch.ones(4, 10, dtype=t, device="cuda"), b.view(4, 10)
    be.linear_act_bwd(sp(be, r), sp(be, e), sp(be, e), 4, 10, 0, act="silu", residual=sp(be, r), dx=sp(be, dx),
                      dw=sp(be, e), db=sp(be, e))
    assert torch.equal(dx, r)
    # No inputs of the layer.
    dy, db = rand(gen_of(2), 4, 10, t=t), torch.ones(10, device="cuda")
    be.linear_act_bwd(sp(be, e), sp(be, e), sp(be, dy), 4, 0, 10, dx=sp(be, e), dw=sp(be, e), db=sp(be, db))
    check("db", db, dy.double().sum(0), 2.0 ** -22 * dy.double().abs().sum(0))
    torch.cuda.synchronize()


# ---------------------------------------------------------------- backward
BWD_SHAPES = [(1, 1, 1), (1, 64, 40), (3, 9, 5), (8, 512, 256), (33, 100, 72), (65, 1000, 784),
              (130, 517, 333), (256, 256, 512), (300, 264, 520), (1000, 136, 72), (520, 784, 1032)]


def bwd_case(be, t, m, k, n, act, packed, residual, grads, seed=2):
    g = gen_of(seed + m * 13 + k * 5 + n)
    x = rand(g, m, k, scale=1.5, t=t)
    w, dy = rand(g, k, n, scale=n ** -0.5, t=t), rand(g, m, n, scale=0.5, t=t)
    r = rand(g, m, k, t=t) if residual else None
    if packed:
        src = torch.zeros(be.ckpt8_bytes(m, k), dtype=torch.uint8, device="cuda")
        be.ckpt8_pack(sp(be, x), m, k, out=sp(be, src))
        v, _ = decode(src, m, k)
    else:
        src, v = x, x.double()
    gt = torch.float32 if grads == "f32" else t
    guard = 64                                     # elements behind each output

    def guarded(*shape, dtype):
        full = torch.full((math.prod(shape) + guard,), 9.0, dtype=dtype, device="cuda")
        return full, full[:math.prod(shape)].view(shape)

    (gx, dx), (gw, dw), (gb, db) = guarded(m, k, dtype=t), guarded(k, n, dtype=gt), guarded(n, dtype=gt)
    be.linear_act_bwd(sp(be, src), sp(be, w), sp(be, dy), m, k, n, act=act, x_ckpt8=packed, residual=sp(be, r),
                      dx=sp(be, dx), dw=sp(be, dw), db=sp(be, db))
    assert all((g[-guard:] == 9.0).all() for g in (gx, gw, gb)), "written behind an output"
    w64, dy64 = w.double(), dy.double()
    back = dy64 @ w64.t()
    s = slope64(v, act)
    want = back * s + (r.double() if residual else 0.0)
    off = sum_error(n, t) * (dy64.abs() @ w64.abs().t())
    # The slope in F32: a few 2^-24, of |v| in the tails' products.
    check("dx", dx, want, 1.01 * rounding(want, t) + 1.13 * off + 2.0 ** -20 * back.abs() * (1 + v.abs()))
    a = act64(v, act)
    aerr = 2.0 ** -21 * v.abs() if act != "none" else 0.0 * v
    if t != torch.float32 and (act != "none" or packed):
        aerr = aerr + rounding(a, t)                   # a is rounded to the operands' type
    want = a.t() @ dy64
    off = (a.abs() * sum_error(m, t) + aerr * 1.01).t() @ dy64.abs()
    check("dw", dw, want, 1.01 * rounding(want, gt) + off)
    want = dy64.sum(0)
    check("db", db, want, 1.01 * rounding(want, gt) + 2.0 ** -24 * (m / 8 + 16) * dy64.abs().sum(0))
    return src, w, dy, r, dx, dw, db


@pytest.mark.parametrize("m,k,n", BWD_SHAPES)
@pytest.mark.parametrize("kind", list(TYPES))
def test_backward(be, kind, m, k, n):
    i = BWD_SHAPES.index((m, k, n))
    acts = ["none", "relu", "gelu", "gelu_tanh", "silu"]
    for j, packed in enumerate((False, True)):
        bwd_case(be, TYPES[kind], m, k, n, acts[(i + j) % 5], packed, (i + j) % 2 == 0, "f32" if (i + j) % 3 else "same")


@pytest.mark.parametrize("m,k,n", [(n, m, k) for m, k, n in LARGE])
def test_backward_large(be, m, k, n):
    bwd_case(be, torch.bfloat16, m, k, n, "gelu", True, True, "same")
    bwd_case(be, torch.bfloat16, m, k, n, "none", (m + k) % 3 == 0, False, "f32")
    if m * k * n < 2 ** 36:
        bwd_case(be, torch.float16, m, k, n, "silu", False, True, "f32")
        bwd_case(be, torch.float32, m, k, n, "gelu_tanh", True, True, "same")


def test_backward_long_sums(be):
    """dX of a long sum over a wide output, in the largest tiles."""
    bwd_case(be, torch.bfloat16, 8192, 8192, 16384, "gelu", True, False, "same")


def test_matrices_past_32_bits(be):
    """More than 2^32 elements: rows at both ends and around 2^31 and 2^32."""
    t, m, n, k = torch.bfloat16, 2 ** 17 + 5, 2 ** 15, 64
    rows = torch.tensor([0, 1, 2 ** 16 - 1, 2 ** 16, 2 ** 17 - 1, 2 ** 17, m - 1], device="cuda")
    g = gen_of(50)
    x, w = rand(g, m, k, t=t), rand(g, k, n, scale=k ** -0.5, t=t)
    out = torch.empty(m, n, dtype=t, device="cuda")
    z8 = torch.empty(be.ckpt8_bytes(m, n), dtype=torch.uint8, device="cuda")
    be.linear_act_fwd(sp(be, x), sp(be, w), None, m, k, n, act="silu", keep="ckpt8", out=sp(be, out), z=sp(be, z8))
    z64 = x[rows].double() @ w.double()
    off = sum_error(k, t) * (x[rows].double().abs() @ w.double().abs())
    want = act64(z64, "silu")
    check("out", out[rows], want, 1.01 * rounding(want, t) + 1.13 * off + 2.0 ** -21 * z64.abs())
    values = torch.empty(m, n, dtype=t, device="cuda")
    be.ckpt8_unpack(sp(be, z8), m, n, out=sp(be, values))
    e = z8[exps_at(m, n):].view(m, n // GROUP)[rows].double()
    step = torch.exp2(e - 127).repeat_interleave(GROUP, dim=1)
    v = values[rows].double()
    check("ckpt8", v, z64, step * torch.where(v.abs() >= 127 * step, 1.0, 0.5) * 1.0001 + off)
    again = torch.empty_like(z8)
    be.ckpt8_pack(sp(be, values), m, n, out=sp(be, again))
    back = torch.empty_like(values)
    be.ckpt8_unpack(sp(be, again), m, n, out=sp(be, back))
    assert torch.equal(back[rows], values[rows])           # packing exact values changes nothing


def test_sums_shared_by_clusters_repeat_their_bits(be):
    t, (m, k, n) = torch.bfloat16, (1100, 8200, 1096)
    g = gen_of(40)
    x, w = rand(g, m, k, t=t), rand(g, k, n, scale=0.01, t=t)
    outs = [torch.empty(m, n, dtype=t, device="cuda") for _ in range(12)]
    for o in outs:
        be.linear_act_fwd(sp(be, x), sp(be, w), None, m, k, n, act="gelu", out=sp(be, o))
    assert all(torch.equal(o, outs[0]) for o in outs)


@pytest.mark.parametrize("act", ["none", "relu", "gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("kind", list(TYPES))
def test_backward_every_activation(be, kind, act):
    for packed in (False, True):
        for grads in ("f32", "same"):
            bwd_case(be, TYPES[kind], 264, 136, 72, act, packed, grads == "f32", grads)


@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
def test_slopes_in_the_tails(be, act):
    """dx of far, tiny and signed-zero pre-activations: with w = 1 it is the
    slope itself."""
    v = torch.tensor([0.0, -0.0, 1e-30, -1e-30, 3.0, -3.0, 5.5, -5.5, 9.0, -9.0, 30.0, -30.0, 1e4, -1e4, 1e20, -1e20,
                      3e38, -3e38], device="cuda")
    one = torch.ones(1, device="cuda")
    dx = torch.empty_like(v)
    be.linear_act_bwd(sp(be, v), sp(be, one), sp(be, torch.ones_like(v)), len(v), 1, 1, act=act, dx=sp(be, dx),
                      dw=sp(be, torch.empty_like(one)), db=sp(be, torch.empty_like(one)))
    want = slope64(v.double().clamp(-50, 50), act)
    check(act, dx, want, torch.full_like(want, 2.0 ** -20))


@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
def test_gradients_against_differences(be, act):
    """F32 gradients of sum(dy * (act(x) @ w + b)) along random directions
    against central differences of that sum in 64 bits.  The differences are
    off by h^2 / 6 of the third derivative along a unit direction (h = 1e-3)
    plus 2^-50 / h of the sum; both are below 1e-5 of the gradient's norm here."""
    m, k, n = 12, 24, 20
    g = gen_of(8)
    x, w, b = rand(g, m, k), rand(g, k, n, scale=0.3), rand(g, n)
    dy = rand(g, m, n)
    dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty_like(b)
    be.linear_act_bwd(sp(be, x), sp(be, w), sp(be, dy), m, k, n, act=act, dx=sp(be, dx), dw=sp(be, dw), db=sp(be, db))

    def total(xv, wv, bv):
        return float(((act64(xv, act) @ wv + bv) * dy.double()).sum())

    at = [x.double(), w.double(), b.double()]
    for i, grad in enumerate((dx, dw, db)):
        for s in range(3):
            d = torch.randn(at[i].shape, generator=g, device="cuda").double()
            d = d / d.norm()
            h = 1e-3
            up, down = list(at), list(at)
            up[i], down[i] = at[i] + h * d, at[i] - h * d
            diff = (total(*up) - total(*down)) / (2 * h)
            assert abs(diff - float((grad.double() * d).sum())) <= 1e-5 * float(grad.double().norm()) + 1e-6


def test_backward_parts_can_be_left_out(be):
    m, k, n, t = 70, 96, 40, torch.bfloat16
    src, w, dy, r, dx, dw, db = bwd_case(be, t, m, k, n, "gelu", True, True, "f32")
    for need in [(1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 0, 1)]:
        got = be.linear_act_bwd(sp(be, src) if need[0] or need[1] else None, sp(be, w) if need[0] else None, sp(be, dy),
                                m, k, n, act="gelu", x_ckpt8=bool(need[0] or need[1]), residual=sp(be, r) if need[0] else None,
                                need_dx=bool(need[0]), need_dw=bool(need[1]), need_db=bool(need[2]))
        for flag, a, b in zip(need, got, (dx, dw, db)):
            assert (a is not None) == bool(flag)
            if flag:
                raw = torch.from_numpy(np.frombuffer(be.to_bytes(a), np.uint8).copy())
                assert torch.equal(raw, b.cpu().contiguous().view(torch.uint8).reshape(-1))


# ---------------------------------------------------------------- used together
def ffn_block(be, x, w1, b1, w2, b2, dout, t, m, d, h):
    """out = x + gelu(x @ w1 + b1) @ w2 + b2 and its gradients, the hidden layer
    and the input kept in 8 bits only."""
    hidden, out = torch.empty(m, h, dtype=t, device="cuda"), torch.empty(m, d, dtype=t, device="cuda")
    z8 = torch.empty(be.ckpt8_bytes(m, h), dtype=torch.uint8, device="cuda")
    x8 = torch.empty(be.ckpt8_bytes(m, d), dtype=torch.uint8, device="cuda")
    be.ckpt8_pack(sp(be, x), m, d, out=sp(be, x8))
    be.linear_act_fwd(sp(be, x), sp(be, w1), sp(be, b1), m, d, h, act="gelu", keep="ckpt8", out=sp(be, hidden), z=sp(be, z8))
    be.linear_act_fwd(sp(be, hidden), sp(be, w2), sp(be, b2), m, h, d, residual=sp(be, x), out=sp(be, out))
    dz, dx = torch.empty(m, h, dtype=t, device="cuda"), torch.empty(m, d, dtype=t, device="cuda")
    dw2, db2 = torch.empty(h, d, device="cuda"), torch.empty(d, device="cuda")
    dw1, db1 = torch.empty(d, h, device="cuda"), torch.empty(h, device="cuda")
    be.linear_act_bwd(sp(be, z8), sp(be, w2), sp(be, dout), m, h, d, act="gelu", x_ckpt8=True, dx=sp(be, dz), dw=sp(be, dw2),
                      db=sp(be, db2))
    be.linear_act_bwd(sp(be, x8), sp(be, w1), sp(be, dz), m, d, h, x_ckpt8=True, residual=sp(be, dout), dx=sp(be, dx),
                      dw=sp(be, dw1), db=sp(be, db1))
    return out, z8, x8, (dx, dw1, db1, dw2, db2)


def ffn_inputs(t, m, d, h, seed=6):
    g = gen_of(seed)
    return (rand(g, m, d, t=t), rand(g, d, h, scale=d ** -0.5, t=t), rand(g, h, scale=0.1, t=t),
            rand(g, h, d, scale=h ** -0.5, t=t), rand(g, d, scale=0.1, t=t), rand(g, m, d, t=t))


@pytest.mark.parametrize("kind,m,d,h", [("bf16", 300, 256, 1024), ("f16", 77, 100, 36), ("f32", 130, 96, 264)])
def test_feed_forward_block(be, kind, m, d, h):
    """The block's output against 64 bits, and its gradients against the
    formulas at the kept values.  Norms over whole matrices: each rounding of
    an intermediate to t adds at most u_t of that intermediate's norm, and the
    chain holds three of them; the 8-bit values are exact inputs here."""
    t = TYPES[kind]
    x, w1, b1, w2, b2, dout = ffn_inputs(t, m, d, h)
    out, z8, x8, (dx, dw1, db1, dw2, db2) = ffn_block(be, x, w1, b1, w2, b2, dout, t, m, d, h)
    X, W1, W2, D = x.double(), w1.double(), w2.double(), dout.double()
    want = X + act64(X @ W1 + b1.double(), "gelu") @ W2 + b2.double()
    zv, xv = decode(z8, m, h)[0], decode(x8, m, d)[0]
    dz = (D @ W2.t()) * slope64(zv, "gelu")
    u = torch.finfo(t).eps / 2 + 2.0 ** -19

    def near(a, b, times):
        assert float((a.double() - b).norm() / b.norm()) <= times * u, (a.shape, float((a.double() - b).norm() / b.norm()) / u)

    near(out, want, 3)
    near(dw2, act64(zv, "gelu").t() @ D, 2)
    near(db2, D.sum(0), 1)
    near(dw1, xv.t() @ dz, 3)
    near(db1, dz.sum(0), 3)
    near(dx, dz @ W1.t() + D, 3)


def test_feed_forward_block_captured_and_replayed(be):
    """Two captured blocks on their own streams replay together and again with
    new inputs, and give what the plain calls give, bit for bit."""
    from orcaml_b200.backend import CudaBackend
    t, (m, d, h) = torch.bfloat16, (200, 136, 520)
    runs = []
    for seed in (11, 12):
        stream = torch.cuda.Stream()
        own = CudaBackend(0, stream=stream.cuda_stream)
        held = ffn_inputs(t, m, d, h, seed)
        with torch.cuda.stream(stream):
            ffn_block(own, *held, t, m, d, h)
            stream.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                res = ffn_block(own, *held, t, m, d, h)
        runs.append((stream, own, held, graph, res))
    for new in (None, 21):
        for i, (stream, own, held, graph, res) in enumerate(runs):
            if new is not None:
                for a, b in zip(held, ffn_inputs(t, m, d, h, new + i)):
                    a.copy_(b)
        torch.cuda.synchronize()
        for stream, own, held, graph, res in runs:
            with torch.cuda.stream(stream):
                graph.replay()
                graph.replay()
        torch.cuda.synchronize()
        for stream, own, held, graph, res in runs:
            want = ffn_block(be, *held, t, m, d, h)
            torch.cuda.synchronize()
            assert torch.equal(res[0], want[0])
            for a, b in zip(res[3], want[3]):
                assert torch.equal(a, b)
    for stream, own, held, graph, res in runs:
        del graph
        own.close()
    runs.clear()


def test_storages_and_own_stream():
    """The calls on storages of a backend with a stream of its own."""
    from orcaml_b200.backend import BF16, F32, CudaBackend
    b2 = CudaBackend(0)
    m, k, n = 30, 40, 24
    rng = np.random.default_rng(0)
    xv, wv = rng.standard_normal((m, k), np.float32), rng.standard_normal((k, n), np.float32)
    x, w = b2.from_f32_slice([m, k], xv), b2.from_f32_slice([k, n], wv)
    before = b2.launch_count()
    out, ck = b2.linear_act_fwd(x, w, None, m, k, n, act="relu", keep="ckpt8")
    assert b2.launch_count() > before
    got = b2.to_f32_vec(out).reshape(m, n)
    z = xv.astype(np.float64) @ wv.astype(np.float64)
    assert np.abs(got - np.maximum(z, 0)).max() <= 1e-5 * np.abs(xv).max() * np.abs(wv).sum(0).max()
    dx, dw, db = b2.linear_act_bwd(ck, b2.from_f32_slice([n, 3], np.ones((n, 3))), b2.from_f32_slice([m, 3], np.ones((m, 3))),
                                   m, n, 3, act="relu", x_ckpt8=True)
    assert dx.dtype == F32 and len(dx) == m * n and len(dw) == n * 3 and np.allclose(b2.to_f32_vec(db), m)
    assert np.array_equal(b2.to_f32_vec(dx).reshape(m, n), 3.0 * (b2.to_f32_vec(b2.ckpt8_unpack(ck, m, n)).reshape(m, n) > 0))
    half = b2.cast(x, [m, k], F32, BF16)
    packed = b2.ckpt8_pack(half, m, k)
    assert len(packed) == b2.ckpt8_bytes(m, k)
    b2.close()


def test_two_threads_and_two_contexts(be):
    """Calls of two host threads, each with its own backend and stream, while a
    third shares the first's backend."""
    import threading
    from orcaml_b200.backend import CudaBackend
    t, (m, k, n) = torch.bfloat16, (130, 264, 520)
    g = gen_of(30)
    x, w = rand(g, m, k, t=t), rand(g, k, n, scale=0.1, t=t)
    want = torch.empty(m, n, dtype=t, device="cuda")
    be.linear_act_fwd(sp(be, x), sp(be, w), None, m, k, n, act="gelu", out=sp(be, want))
    torch.cuda.synchronize()
    first, second = CudaBackend(0), CudaBackend(0)
    outs = [[torch.zeros(m, n, dtype=t, device="cuda") for _ in range(20)] for _ in range(3)]
    torch.cuda.synchronize()

    def work(backend, mine):
        for o in mine:
            backend.linear_act_fwd(sp(be, x), sp(be, w), None, m, k, n, act="gelu", out=sp(be, o))
        backend.synchronize()

    threads = [threading.Thread(target=work, args=(b, o)) for b, o in zip((first, second, first), outs)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert all(torch.equal(o, want) for mine in outs for o in mine)
    first.close()
    second.close()


# ---------------------------------------------------------------- refusals
def test_refusals(be):
    from orcaml_b200 import _lib as L
    t, m, k, n = torch.bfloat16, 4, 8, 6

    def new(*shape, dtype=t):
        return torch.zeros(*shape, dtype=dtype, device="cuda")

    x, w, b, out = new(m, k), new(k, n), new(n), new(m, n)

    def fwd(match, status, x=x, w=w, b=b, m=m, k=k, n=n, out=out, z=None, **kw):
        as_span = lambda v: v if v is None or isinstance(v, L.orca_span) else sp(be, v)  # noqa: E731
        before = be.launch_count()
        with pytest.raises(L.OrcaError, match=match) as err:
            be.linear_act_fwd(as_span(x), as_span(w), as_span(b), m, k, n, out=as_span(out), z=as_span(z),
                              residual=as_span(kw.pop("residual", None)), **kw)
        assert err.value.status_name == status
        assert be.launch_count() == before

    fwd("holds 32 elements, the sizes need 40", "ORCA_SHAPE_MISMATCH", m=5)
    fwd("w: the span holds", "ORCA_SHAPE_MISMATCH", n=7, b=new(7), out=new(m, 7))
    fwd("b: the span holds", "ORCA_SHAPE_MISMATCH", b=new(5))
    fwd("out: the span holds", "ORCA_SHAPE_MISMATCH", out=new(m, n - 1))
    fwd("w: dtype", "ORCA_DTYPE_MISMATCH", w=new(k, n, dtype=torch.float16))
    fwd("out: dtype", "ORCA_DTYPE_MISMATCH", out=new(m, n, dtype=torch.float32))
    fwd("none of F32, F16, BF16", "ORCA_UNSUPPORTED_DTYPE", x=new(m, k, dtype=torch.uint8))
    fwd("unknown dtype", "ORCA_UNSUPPORTED_DTYPE", x=be.span(x.data_ptr(), 32, 99))
    fwd("'tanh' is none of", "ORCA_INVALID_ARGUMENT", act="tanh")
    fwd("'all' is none of", "ORCA_INVALID_ARGUMENT", keep="all")
    fwd("out of range", "ORCA_INVALID_ARGUMENT", m=-1)
    fwd("out of range", "ORCA_INVALID_ARGUMENT", k=2 ** 31)
    fwd("null data", "ORCA_INVALID_ARGUMENT", x=be.span(None, 32, code_of(t)))
    fwd("not aligned to its elements", "ORCA_INVALID_ARGUMENT", x=be.span(x.data_ptr() + 1, 32, code_of(t)))
    host = torch.zeros(m, k, dtype=t).pin_memory()
    fwd("not device memory", "ORCA_DEVICE_MISMATCH", x=be.span(host.data_ptr(), 32, code_of(t)))
    both = new(m * k + m * n)
    fwd("an output and x overlap", "ORCA_INVALID_ARGUMENT", x=both[:m * k], out=both[m * k - 1:m * k - 1 + m * n])
    fwd("out and residual overlap", "ORCA_INVALID_ARGUMENT", residual=both[1:1 + m * n], out=both[:m * n])
    fwd("z: the span holds", "ORCA_SHAPE_MISMATCH", keep="ckpt8", z=new(be.ckpt8_bytes(m, n) - 1, dtype=torch.uint8))
    fwd("z: dtype", "ORCA_DTYPE_MISMATCH", keep="ckpt8", z=new(64))
    fwd("out and z overlap", "ORCA_INVALID_ARGUMENT", keep="z", z=out)
    lib = L.load()
    assert lib.orca_linear_act_fwd(be.ctx, sp(be, x), sp(be, w), None, None, m, k, n, 0, sp(be, out), 1, None) == 7
    assert lib.orca_linear_act_fwd(be.ctx, sp(be, x), sp(be, w), None, None, m, k, n, 0, sp(be, out), 0, sp(be, new(m, n))) == 7
    assert lib.orca_linear_act_fwd(be.ctx, None, sp(be, w), None, None, m, k, n, 0, sp(be, out), 0, None) == 7
    assert lib.orca_linear_act_fwd(be.ctx, sp(be, x), sp(be, w), None, None, m, k, n, 9, sp(be, out), 0, None) == 7

    dy, dx, dw, db = new(m, n), new(m, k), new(k, n, dtype=torch.float32), new(n, dtype=torch.float32)
    x8 = new(be.ckpt8_bytes(m, k), dtype=torch.uint8)

    def bwd(match, x=x, w=w, dy=dy, dx=dx, dw=dw, db=db, residual=None, **kw):
        with pytest.raises(L.OrcaError, match=match):
            be.linear_act_bwd(sp(be, x), sp(be, w), sp(be, dy), m, k, n, dx=sp(be, dx), dw=sp(be, dw), db=sp(be, db),
                              residual=sp(be, residual), **kw)

    bwd("a checkpoint, x has dtype", x_ckpt8=True)
    bwd("plain values, x has dtype", x=x8)
    bwd("x: the span holds", x=x8[:-1], x_ckpt8=True)
    bwd("dw: dtype", dw=new(k, n, dtype=torch.float16))
    bwd("dx: dtype", dx=new(m, k, dtype=torch.float32))
    bwd("db: the span holds", db=new(n - 1, dtype=torch.float32))
    bwd("an output and w overlap", dx=w.view(-1)[:m * k])
    bwd("x: null span", x=None)
    with pytest.raises(L.OrcaError, match="must be U8"):
        be.ckpt8_pack(sp(be, x), m, k, out=sp(be, new(200)))
    with pytest.raises(L.OrcaError, match="the span holds"):
        be.ckpt8_pack(sp(be, x), m, k, out=sp(be, x8[:-1]))
    with pytest.raises(L.OrcaError, match="must be U8"):
        be.ckpt8_unpack(sp(be, new(200)), m, k)
    with pytest.raises(L.OrcaError, match="out of range"):
        be.ckpt8_pack(sp(be, x), -1, k, out=sp(be, x8))
    with pytest.raises(L.OrcaError, match="unknown dtype|none of F32"):
        be.ckpt8_unpack(sp(be, x8), m, k, out=sp(be, new(m * k, dtype=torch.uint8)))
    # The backend still works.
    be.linear_act_fwd(sp(be, x), sp(be, w), sp(be, b), m, k, n, out=sp(be, out))
    torch.cuda.synchronize()


def test_stream_of_another_device_is_refused():
    from orcaml_b200 import _lib as L
    h = ctypes.c_void_p()
    s = torch.cuda.Stream()
    count = torch.cuda.device_count()
    if count > 1:
        assert L.load().orca_ctx_create_on_stream(1, s.cuda_stream, ctypes.byref(h)) == 2
    assert L.load().orca_ctx_create_on_stream(count, s.cuda_stream, ctypes.byref(h)) == 7
