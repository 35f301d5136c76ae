"""How far F32 results of the feed-forward operators are from 64 bits, as norms
over whole matrices of random operands: u = 2^-24.

An accumulator of the tensor core loses up to 2 u of what it holds at each step of
16 products, toward zero; 0.72 u on average over a binade.  Over n steps of a random
walk those losses add up to 0.72 u n / sqrt(3) of the chain's norm, and chains are
independent of one another.  Joining c chains in F32 adds u / sqrt(3) of the sum
so far each time, together u sqrt(c / 6) of the result's.

F32 operands: four steps of a 64-deep block add at full scale, 1.0e-7; 64 blocks
(a sum of 4096) add 1.9e-7; the three plane products left out are 2^-24 of each
product on average, toward zero, 0.6e-7.  As squares 2.2e-7 at 4096; the limit is 4e-7.  Leaving
out one more plane product costs 1e-5.

F32 gradients of 16-bit operands: chains of 32 steps, 7.9e-7, and 32 of them (16384 rows)
joined, 1.4e-7: 8e-7.  Chains of twice the length are measured at 1.0e-6.
"""
import pytest

torch = pytest.importorskip("torch")

from tests.test_gpu_linear_act import TYPES, act64, be, check, decode, gen_of, rand, slope64, sp, sum_error  # noqa: E402,F401

pytestmark = pytest.mark.gpu


def rel(got, want):
    return float((got.double() - want).norm() / want.norm())


# One row to several rounds of tiles, aligned rows and others.
@pytest.mark.parametrize("m,k,n", [(1, 784, 1024), (16, 4096, 784), (64, 784, 517), (300, 4096, 520), (1100, 784, 1096),
                                   (1100, 785, 1097), (2320, 4096, 2312), (2320, 785, 2313)])
def test_f32_products(be, m, k, n):  # noqa: F811
    g = gen_of(m + k + n)
    x, w, dy = rand(g, m, k), rand(g, k, n), rand(g, m, n)
    out, dx, dw = (torch.full_like(v, 7.0) for v in (dy, x, w))
    be.linear_act_fwd(sp(be, x), sp(be, w), None, m, k, n, out=sp(be, out))
    be.linear_act_bwd(sp(be, x), sp(be, w), sp(be, dy), m, k, n, dx=sp(be, dx), dw=sp(be, dw), need_db=False)
    x, w, dy = x.double(), w.double(), dy.double()
    off = [rel(out, x @ w), rel(dx, dy @ w.t()), rel(dw, x.t() @ dy)]
    assert max(off) <= 4e-7, off


@pytest.mark.parametrize("m,k,n", [(1024, 512, 520), (4096, 1024, 1096), (4096, 513, 259), (4096, 2049, 2055),
                                   (16384, 512, 520), (16384, 2048, 2056)])
@pytest.mark.parametrize("kind", ["bf16", "f16"])
def test_f32_gradients_of_16_bits(be, kind, m, k, n):  # noqa: F811
    g = gen_of(m + k)
    x, dy = rand(g, m, k, t=TYPES[kind]), rand(g, m, n, t=TYPES[kind])
    dw = torch.full((k, n), 7.0, device="cuda")
    be.linear_act_bwd(sp(be, x), None, sp(be, dy), m, k, n, dw=sp(be, dw), need_dx=False, need_db=False)
    assert rel(dw, x.double().t() @ dy.double()) <= 8e-7


@pytest.mark.parametrize("scale", [2.0 ** -100, 2.0 ** -110, 1e-35, 1e-37, 1e-39, 1e-41])
@pytest.mark.parametrize("m,k,n", [(4, 200, 136), (1100, 264, 1288), (1100, 265, 1287)])
def test_small_f32_operands(be, m, k, n, scale):  # noqa: F811
    """Each operand is off by 2^-133 at most, beside the sums' error; accumulators
    that hold less than 2^-126 lose up to 2^-149 at each of 24 steps of a block."""
    g = gen_of(m + k + n)
    x, w = (rand(g, m, k).double() * scale).float(), rand(g, k, n)
    out = torch.empty(m, n, device="cuda")
    for a, b in ((x, w), (x.abs(), w.abs())):
        be.linear_act_fwd(sp(be, a), sp(be, b), None, m, k, n, out=sp(be, out))
        a, b = a.double(), b.double()
        bound = sum_error(k, torch.float32) * (a.abs() @ b.abs()) + 24 * (k // 64 + 1) * 2.0 ** -149
        check("out", out, a @ b, bound + 2.0 ** -133 * (b.abs().sum(0) + a.abs().sum(1)[:, None]))


def test_f32_products_below_the_normal_range(be):  # noqa: F811
    m, k, n = 70, 264, 136
    g = gen_of(3)
    x, w = ((rand(g, *s).double() * 2.0 ** -66).float() for s in ((m, k), (k, n)))
    out = torch.empty(m, n, device="cuda")
    be.linear_act_fwd(sp(be, x), sp(be, w), None, m, k, n, out=sp(be, out))
    x, w = x.double(), w.double()
    bound = sum_error(k, torch.float32) * (x.abs() @ w.abs()) + 24 * (k // 64 + 1) * 2.0 ** -149
    check("out", out, x @ w, bound + 2.0 ** -133 * (w.abs().sum(0) + x.abs().sum(1)[:, None]))


@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
def test_activations_and_slopes_in_f32(be, act):  # noqa: F811
    """Values within 2^-21 of |z| and slopes within 2^-21 of 1 + |z|, as the header
    says; a sum of no products with the bias z is z itself, and with w = dy = 1 dx is the slope."""
    z = torch.cat([torch.linspace(-12, 12, 2 ** 20 + 1, device="cuda"), rand(gen_of(1), 2 ** 18)])
    n = z.numel()
    none, one = be.span(None, 0, 0), torch.ones(1, device="cuda")
    out, dx = torch.empty_like(z), torch.empty_like(z)
    be.linear_act_fwd(none, none, sp(be, z), 1, 0, n, act=act, out=sp(be, out))
    be.linear_act_bwd(sp(be, z), sp(be, one), sp(be, torch.ones_like(z)), n, 1, 1, act=act, dx=sp(be, dx), need_dw=False,
                      need_db=False)
    z = z.double()
    check("value", out, act64(z, act), 2.0 ** -21 * z.abs() + 2.0 ** -126)
    check("slope", dx, slope64(z, act), 2.0 ** -21 * (1 + z.abs()))


@pytest.mark.parametrize("m,k,n", [(2 ** 15 + 64, 512, 512), (2 ** 20, 512, 512), (2 ** 20 + 5, 1024, 520), (2 ** 20, 64, 64)])
@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_16_bit_results_of_long_sums(be, kind, m, k, n):  # noqa: F811
    """Chains of 2048 (F16) and 16384 (BF16) steps are off by 0.72 u * steps / sqrt(3) of the norm,
    5.1e-5 and 4.1e-4; beside the rounding, 2.1e-4 and 1.7e-3 rms, that is 3 % more, as squares."""
    t = TYPES[kind]
    g = gen_of(5)
    x, dy = rand(g, m, k, t=t), rand(g, m, n, scale=1 / 64, t=t)
    dw = torch.full((k, n), 7.0, dtype=t, device="cuda")
    be.linear_act_bwd(sp(be, x), None, sp(be, dy), m, k, n, dw=sp(be, dw), need_dx=False, need_db=False)
    want = sum(x[i:i + 2 ** 16, :64].double().t() @ dy[i:i + 2 ** 16].double() for i in range(0, m, 2 ** 16))
    assert rel(dw[:64], want) <= 1.05 * rel(want.to(t), want)


@pytest.mark.parametrize("m,k,n", [(2048, 4096, 4096), (2048, 4099, 4103)])
def test_codes_that_flip(be, m, k, n):  # noqa: F811
    """A code differs from the exact sum's where a border lies within the sum's error: in
    |error| / step of the elements, |error| being 0.8 of 5.9e-7 of the norm on average.  Counted with four
    standard deviations."""
    g = gen_of(k)
    x, w = rand(g, m, k, t=torch.bfloat16), rand(g, k, n, scale=k ** -0.5, t=torch.bfloat16)
    z = torch.zeros(be.ckpt8_bytes(m, n), dtype=torch.uint8, device="cuda")
    out = torch.empty(m, n, dtype=torch.bfloat16, device="cuda")
    be.linear_act_fwd(sp(be, x), sp(be, w), None, m, k, n, keep="ckpt8", out=sp(be, out), z=sp(be, z))
    got, step = decode(z, m, n)
    z64 = x.double() @ w.double()
    want = (z64 / step).round().clamp(-127, 127) * step
    flips = int((got != want).sum())
    expected = float((0.8 * 5.9e-7 * z64.pow(2).mean().sqrt() / step).sum())
    assert flips <= expected + 4 * expected ** 0.5, (flips, expected)


@pytest.mark.parametrize("kind", ["bf16", "f16"])
def test_f32_gradients_through_an_activation(be, kind):  # noqa: F811
    """dw's operand act(x) is rounded to the operands' type, as the forward pass rounds it,
    also where dw is F32: by the formula at the rounded operand dw is off by what the activation's error,
    2^-21 of |x|, moves across borders of the rounding (2^-21 |x| / ulp of the elements by an ulp:
    below 1e-4 of the norm), and at the exact one by the rounding."""
    t, (m, k, n) = TYPES[kind], (4096, 520, 264)
    g = gen_of(6)
    x, dy = rand(g, m, k, t=t), rand(g, m, n, t=t)
    dw = torch.full((k, n), 7.0, device="cuda")
    be.linear_act_bwd(sp(be, x), None, sp(be, dy), m, k, n, act="gelu", dw=sp(be, dw), need_dx=False, need_db=False)
    a = act64(x.double(), "gelu")
    assert rel(dw, a.to(t).double().t() @ dy.double()) <= 1e-4
    assert rel(dw, a.t() @ dy.double()) <= 1.1 * rel(a.to(t), a)
