"""Measured cases of the fused linear operators and of the 8-bit activation checkpoints.

Three operators, as a feed-forward block of a transformer uses them:

  linear_act_fwd   out = act(x @ w + b) + residual, keeping z = x @ w + b for the backward pass in the
                   operands' type or as an 8-bit checkpoint
  linear_act_bwd   from dy, the gradient of a @ w + b with a = act(x): dx = (dy @ w^T) * act'(x) + residual,
                   dw = a^T @ dy, db = the column sums of dy; x given plainly or as an 8-bit checkpoint
  ckpt8            a matrix packed to 8 bits and unpacked again through an activation

An 8-bit checkpoint of [m, n] holds, for each row and each 32 columns of it, one exponent byte E and signed 8-bit
codes q: the values are q * 2^(E - 127) with 2^(E - 127) = 2^(floor(log2 amax) - 6), at least 2^-126, and
q = the value / 2^(E - 127) rounded to the nearest, ties to even, within +-127; E = 255 marks a group that held
an infinity or a NaN and stands for NaN.  All codes come first, row after row; the exponents follow at the next
multiple of 16 bytes.
"""
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}
GROUP = 32


# ---------------------------------------------------------------- cases
def listed():
    return [
        # Serving: the up-projection of one token (latency is one pass over the weights).
        dict(name="fwd one token", op="fwd", type="bf16", m=1, k=4096, n=16384, act="gelu_tanh", residual=False, keep="none"),
        # Serving: eight tokens through a small layer, where the call itself is what counts.
        dict(name="fwd eight tokens small", op="fwd", type="bf16", m=8, k=512, n=512, act="silu", residual=True, keep="none"),
        # A ragged batch through a layer whose sizes are odd, so that rows are not aligned.
        dict(name="fwd ragged", op="fwd", type="f16", m=333, k=1001, n=517, act="relu", residual=True, keep="none"),
        # Training: the up-projection at the width of the largest model of the benchmark, its pre-activation kept in 8 bits.
        dict(name="fwd up, kept in 8 bits", op="fwd", type="bf16", m=4096, k=4096, n=16384, act="gelu", residual=False, keep="ckpt8"),
        # Training: the down-projection with the residual stream added.
        dict(name="fwd down, residual", op="fwd", type="bf16", m=4096, k=16384, n=4096, act="none", residual=True, keep="none"),
        # The first layer of the benchmark's model in F32, keeping its pre-activation.
        dict(name="fwd f32", op="fwd", type="f32", m=4096, k=784, n=8192, act="silu", residual=False, keep="z"),
        # Training: backward of the down-projection from the 8-bit pre-activation.
        dict(name="bwd down from 8 bits", op="bwd", type="bf16", m=4096, k=16384, n=4096, act="gelu", x="ckpt8", residual=False, grads="same"),
        # Training: backward of the up-projection from its 8-bit input, F32 gradients for the optimizer.
        dict(name="bwd up, f32 gradients", op="bwd", type="bf16", m=4096, k=4096, n=16384, act="none", x="ckpt8", residual=True, grads="f32"),
        # A hidden layer of the F32 models.
        dict(name="bwd f32", op="bwd", type="f32", m=1024, k=4096, n=4096, act="relu", x="plain", residual=False, grads="same"),
        # A short batch, sizes that fill no tile.
        dict(name="bwd small", op="bwd", type="f16", m=65, k=1000, n=784, act="silu", x="plain", residual=False, grads="same"),
        # The hidden activations of a training batch, packed and decoded through the activation.
        dict(name="ckpt8 hidden", op="ckpt8", type="bf16", m=4096, n=16384, act="gelu"),
        # A ragged F32 matrix.
        dict(name="ckpt8 ragged", op="ckpt8", type="f32", m=513, n=1001, act="none"),
    ]


def _size(rng, low, high):
    """Spread over the logarithm; every other one a multiple of 8, as most models' sizes are."""
    v = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    return max(8, v // 8 * 8) if rng.random() < 0.5 else v


def draw(rng):
    op = rng.choice(["fwd", "fwd", "bwd", "bwd", "ckpt8"])
    act = rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"])
    kind = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "ckpt8":
        return dict(op=op, type=kind, m=_size(rng, 1, 4096), n=_size(rng, 1, 16384), act=act)
    while True:
        m, k, n = _size(rng, 1, 8192), _size(rng, 16, 16384), _size(rng, 16, 16384)
        if m * k * n <= 4096 * 4096 * 16384:
            break
    if op == "fwd":
        return dict(op=op, type=kind, m=m, k=k, n=n, act=act, residual=rng.random() < 0.5,
                    keep=rng.choice(["none", "z", "ckpt8"]))
    return dict(op=op, type=kind, m=m, k=k, n=n, act=act, x=rng.choice(["plain", "ckpt8"]),
                residual=rng.random() < 0.5, grads="f32" if act == "none" and rng.random() < 0.5 else "same")


def work(case):
    m, n, s = case["m"], case["n"], BYTES[case["type"]]
    kept = m * n + m * -(-n // GROUP)
    if case["op"] == "ckpt8":
        return {"bytes": 2 * m * n * s + 2 * kept, "flops": 0}
    k = case["k"]
    if case["op"] == "fwd":
        b = s * (m * k + k * n + n + m * n * (2 if case["residual"] else 1))
        if case["keep"] == "z":
            b += s * m * n
        elif case["keep"] == "ckpt8":
            b += 2 * kept + 2 * m * n
        return {"bytes": b, "flops": 2 * m * k * n}
    g = 4 if case["grads"] == "f32" else s
    x = s * m * k if case["x"] == "plain" else m * k + m * -(-k // GROUP)
    b = x + s * (k * n + m * n + m * k * (2 if case["residual"] else 1)) + g * (k * n + n)
    return {"bytes": b, "flops": 4 * m * k * n}


# ---------------------------------------------------------------- inputs
def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))
    t = TYPES[case["type"]]

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, generator=gen, device="cuda") * scale

    def activations(rows, cols):
        """Unit values; one column in 64 is larger, as hidden features of language models are."""
        x = normal(rows, cols)
        return x * torch.where(torch.rand(cols, generator=gen, device="cuda") < 1 / 64, 8.0, 1.0)

    s = {"case": dict(case)}
    m, n = case["m"], case["n"]
    if case["op"] == "ckpt8":
        s["x"] = activations(m, n).to(t)
        return s
    k = case["k"]
    s["w"] = normal(k, n, scale=k ** -0.5).to(t)
    x = activations(m, k).to(t)
    if case["op"] == "fwd":
        s["x"] = x
        s["b"] = normal(n, scale=0.1).to(t)
        s["residual"] = normal(m, n).to(t) if case["residual"] else None
        return s
    s["x"] = _encode(x) if case["x"] == "ckpt8" else x
    s["dy"] = normal(m, n, scale=0.02).to(t)
    s["residual"] = normal(m, k, scale=0.02).to(t) if case["residual"] else None
    return s


# ---------------------------------------------------------------- the plain form
def _quantise(x):
    """Codes [m, n] and exponent bytes [m, groups] of a float32 matrix, as whole numbers."""
    m, n = x.shape
    groups = -(-n // GROUP)
    g = torch.nn.functional.pad(x, (0, groups * GROUP - n)).view(m, groups, GROUP)
    amax = g.abs().amax(dim=2)
    fine = torch.isfinite(g).all(dim=2)
    log2 = torch.frexp(torch.where(fine & (amax > 0), amax, 1.0))[1].int() - 1
    e = torch.where(amax > 0, log2 - 6, -126).clamp(min=-126)
    up = ((127 - e) << 23).view(torch.float32)
    q = torch.round(g * up[:, :, None]).clamp(-127, 127)
    q = torch.where(fine[:, :, None], q, 0.0).to(torch.int8).view(m, groups * GROUP)[:, :n]
    return q, torch.where(fine, e + 127, 255).to(torch.uint8)


def _encode(x):
    """The bytes of the 8-bit checkpoint of x."""
    q, e = _quantise(x.float())
    codes = q.contiguous().view(-1).view(torch.uint8)
    gap = torch.zeros(-codes.numel() % 16, dtype=torch.uint8, device=x.device)
    return torch.cat([codes, gap, e.reshape(-1)])


def _decode(q, e):
    scale = torch.where(e == 255, math.nan, (e.int() << 23).view(torch.float32))
    return q.float() * scale.repeat_interleave(GROUP, dim=1)[:, : q.shape[1]]


def _read(buf, m, n):
    """Float32 values of the bytes of an 8-bit checkpoint."""
    groups = -(-n // GROUP)
    at = -(-m * n // 16) * 16
    q = buf[: m * n].view(torch.int8).view(m, n)
    return _decode(q, buf[at: at + m * groups].view(m, groups))


def _act(z, act):
    if act == "relu":
        return torch.where(z > 0, z, 0.0)
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _act_slope(z, act):
    if act == "relu":
        return (z > 0).float()
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    if act == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z * z * z))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)
    if act == "silu":
        g = 1 / (1 + torch.exp(-z))
        return g * (1 + z * (1 - g))
    return torch.ones_like(z)


def _kept_type(t):
    """Decoded values have at most 8 significant bits: BF16 holds each of them exactly."""
    return torch.bfloat16 if t == torch.float32 else t


def _plain(s):
    c = s["case"]
    t, act = TYPES[c["type"]], c["act"]
    if c["op"] == "ckpt8":
        return _act(_decode(*_quantise(s["x"].float())), act).to(t)
    w = s["w"].float()
    r = s["residual"].float() if s["residual"] is not None else 0.0
    if c["op"] == "fwd":
        z = s["x"].float() @ w + s["b"].float()
        out = (_act(z, act) + r).to(t)
        if c["keep"] == "z":
            return out, z.to(t)
        return (out, _decode(*_quantise(z)).to(_kept_type(t))) if c["keep"] == "ckpt8" else out
    x = _read(s["x"], c["m"], c["k"]) if c["x"] == "ckpt8" else s["x"].float()
    dy = s["dy"].float()
    g = torch.float32 if c["grads"] == "f32" else t
    dx = (dy @ w.t()) * _act_slope(x, act) + r
    return dx.to(t), (_act(x, act).t() @ dy).to(g), dy.sum(dim=0).to(g)


# ---------------------------------------------------------------- the framework's calls
_backends = {}


def _backend():
    """The framework's context on torch's current device and stream."""
    from orcaml_b200.backend import CudaBackend
    at = (torch.cuda.current_device(), torch.cuda.current_stream().cuda_stream)
    if at not in _backends:
        _backends[at] = CudaBackend(at[0], stream=at[1])
    return _backends[at]


def _framework(s):
    from orcaml_b200.backend import BF16, F16, F32, U8
    codes = {torch.bfloat16: BF16, torch.float16: F16, torch.float32: F32, torch.uint8: U8}
    be, c = _backend(), s["case"]
    t, act, m, n = TYPES[c["type"]], c["act"], c["m"], c["n"]

    def span(v):
        return None if v is None else be.span(v.data_ptr(), v.numel(), codes[v.dtype])

    def new(*shape, dtype=t):
        return torch.empty(*shape, dtype=dtype, device="cuda")

    if c["op"] == "ckpt8":
        kept, out = new(be.ckpt8_bytes(m, n), dtype=torch.uint8), new(m, n)
        be.ckpt8_pack(span(s["x"]), m, n, out=span(kept))
        be.ckpt8_unpack(span(kept), m, n, act=act, out=span(out))
        return out
    k = c["k"]
    if c["op"] == "fwd":
        out, keep, z = new(m, n), c["keep"], None
        if keep == "z":
            z = new(m, n)
        elif keep == "ckpt8":
            z = new(be.ckpt8_bytes(m, n), dtype=torch.uint8)
        be.linear_act_fwd(span(s["x"]), span(s["w"]), span(s["b"]), m, k, n, act=act, residual=span(s["residual"]),
                          keep=keep, out=span(out), z=span(z))
        if keep == "ckpt8":
            values = new(m, n, dtype=_kept_type(t))
            be.ckpt8_unpack(span(z), m, n, out=span(values))
            return out, values
        return (out, z) if keep == "z" else out
    g = torch.float32 if c["grads"] == "f32" else t
    dx, dw, db = new(m, k), new(k, n, dtype=g), new(n, dtype=g)
    be.linear_act_bwd(span(s["x"]), span(s["w"]), span(s["dy"]), m, k, n, act=act, x_ckpt8=c["x"] == "ckpt8",
                      residual=span(s["residual"]), dx=span(dx), dw=span(dw), db=span(db))
    return dx, dw, db


def run(state):
    return _framework(state) if own else _plain(state)


# ---------------------------------------------------------------- 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    m, n, act = case["m"], case["n"], case["act"]

    def f(z):
        return {"none": lambda: z, "relu": lambda: z.clamp(min=0), "gelu": lambda: 0.5 * z * torch.erfc(-z / math.sqrt(2)),
                "gelu_tanh": lambda: z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)),
                "silu": lambda: z * torch.sigmoid(z)}[act]()

    def slope(z):
        z = z.clone().requires_grad_(True)
        with torch.enable_grad():
            return torch.autograd.grad(f(z).sum(), z)[0]

    def grouped(v, cols):
        return torch.nn.functional.pad(v, (0, -cols % GROUP)).unflatten(1, (-1, GROUP))

    def kept(z):
        g = grouped(z, n)
        step = torch.exp2((torch.floor(torch.log2(g.abs().amax(2, keepdim=True))) - 6).clamp(min=-126))
        return (torch.round(g / step).clamp(-127, 127) * step).flatten(1)[:, :n]

    if case["op"] == "ckpt8":
        return f(kept(s["x"].double()))
    k = case["k"]
    w = s["w"].double()
    r = 0.0 if s["residual"] is None else s["residual"].double()
    if case["op"] == "fwd":
        z = s["x"].double() @ w + s["b"].double()
        out = f(z) + r
        return {"none": lambda: out, "z": lambda: (out, z), "ckpt8": lambda: (out, kept(z))}[case["keep"]]()
    if case["x"] == "ckpt8":
        q = s["x"][: m * k].view(torch.int8).view(m, k).double()
        e = s["x"][(m * k + 15) // 16 * 16:].view(m, -1).double()
        x = (grouped(q, k) * torch.exp2(e - 127)[:, :, None]).flatten(1)[:, :k]
    else:
        x = s["x"].double()
    dy = s["dy"].double()
    return (dy @ w.t()) * (slope(x) if act != "none" else 1.0) + r, f(x).t() @ dy, dy.sum(0)
