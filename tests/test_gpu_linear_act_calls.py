"""Calls of the feed-forward operators that the header allows, or refuses, beside
the ordinary ones: spans longer than what is used, inputs that are not read."""
import pytest

torch = pytest.importorskip("torch")

from tests.test_gpu_linear_act import TYPES, be, code_of, gen_of, rand, sp  # noqa: E402,F401

pytestmark = pytest.mark.gpu

T, M, K, N = torch.bfloat16, 5, 16, 24


def arena(be, *sizes):  # noqa: F811
    """Spans that follow one another in one allocation and all reach to its end."""
    full = rand(gen_of(7), sum(sizes), t=T)
    spans, parts, at = [], [], 0
    for s in sizes:
        parts.append(full[at:at + s])
        spans.append(be.span(full.data_ptr() + 2 * at, full.numel() - at, code_of(T)))
        at += s
    return full, spans, parts


def test_forward_in_an_arena(be):  # noqa: F811
    full, (x, w, out, z), (px, pw, po, pz) = arena(be, M * K, K * N, M * N, M * N)
    want, zw = torch.empty(M * N, dtype=T, device="cuda"), torch.empty(M * N, dtype=T, device="cuda")
    cx, cw = px.clone(), pw.clone()
    be.linear_act_fwd(sp(be, cx), sp(be, cw), None, M, K, N, act="silu", keep="z", out=sp(be, want), z=sp(be, zw))
    be.linear_act_fwd(x, w, None, M, K, N, act="silu", keep="z", out=out, z=z)
    assert torch.equal(po, want) and torch.equal(pz, zw) and torch.equal(px, cx) and torch.equal(pw, cw)


def test_backward_in_an_arena(be):  # noqa: F811
    full, (x, w, dy, dx, dw, db), parts = arena(be, M * K, K * N, M * N, M * K, K * N, N)
    ins = [p.clone() for p in parts[:3]]
    outs = [torch.empty_like(p) for p in parts[3:]]
    for i, o in ((ins, outs), ((x, w, dy), (dx, dw, db))):
        i, o = ([v if hasattr(v, "len") else sp(be, v) for v in a] for a in (i, o))
        be.linear_act_bwd(*i, M, K, N, act="gelu", dx=o[0], dw=o[1], db=o[2])
    assert all(torch.equal(a, b) for a, b in zip(parts, ins + outs))


def test_checkpoint_in_an_arena(be):  # noqa: F811
    full, (x, out), (px, po) = arena(be, M * K, M * K)
    size = be.ckpt8_bytes(M, K)
    raw = torch.zeros(2 * (size + 1) + 2 * M * K, dtype=torch.uint8, device="cuda")
    for at in (0, size + 1):
        ck = be.span(raw.data_ptr() + at, raw.numel() - at, 6)
        be.ckpt8_pack(x, M, K, out=ck)
    assert torch.equal(raw[:size], raw[size + 1:2 * size + 1])
    be.ckpt8_unpack(be.span(raw.data_ptr(), 2 ** 63, 6), M, K, out=out)
    assert torch.isfinite(po).all()


def test_a_span_of_unknown_length_still_must_not_overlap(be):  # noqa: F811
    """A length past the end of memory says nothing about what is used."""
    from orcaml_b200 import _lib as L
    v = torch.zeros(4 * M * K * N, dtype=T, device="cuda")
    at, far = v.data_ptr(), 2 ** 63
    out = be.span(at + 2, far, code_of(T))
    w = sp(be, v[M * N + K * N:])
    before = be.launch_count()
    for x, z, match in ((be.span(at, far, code_of(T)), None, "an output and x overlap"),
                        (sp(be, v[-M * K:]), be.span(at + 2 * M * N, far, code_of(T)), "out and z overlap")):
        with pytest.raises(L.OrcaError, match=match):
            be.linear_act_fwd(x, w, None, M, K, N, out=out, z=z, keep="z" if z else None)
    with pytest.raises(L.OrcaError, match="ckpt and x overlap"):
        be.ckpt8_pack(be.span(at, far, code_of(T)), M, K, out=be.span(at + 2 * M * K - 1, far, 6))
    assert be.launch_count() == before


def test_inputs_that_are_not_read(be):  # noqa: F811
    """Their memory may be an output's, and their lengths and types say nothing."""
    g = gen_of(9)
    x, w, dy = rand(g, M, K, t=T), rand(g, K, N, t=T), rand(g, M, N, t=T)
    dx, dw, db = (torch.empty_like(v) for v in (x, w, dy[0]))
    be.linear_act_bwd(sp(be, x), sp(be, w), sp(be, dy), M, K, N, dx=sp(be, dx), dw=sp(be, dw), db=sp(be, db))
    got = torch.empty_like(w)
    be.linear_act_bwd(sp(be, x), sp(be, got), sp(be, dy), M, K, N, residual=sp(be, got), dw=sp(be, got), need_dx=False,
                      need_db=False)
    assert torch.equal(got, dw)
    got = torch.empty_like(x)
    be.linear_act_bwd(sp(be, got), sp(be, w), sp(be, dy), M, K, N, dx=sp(be, got), need_dw=False, need_db=False)
    assert torch.equal(got, dx)
    got = torch.empty_like(db)
    be.linear_act_bwd(sp(be, got), sp(be, got), sp(be, dy), M, K, N, act="relu", residual=sp(be, got), db=sp(be, got),
                      need_dx=False, need_dw=False)
    assert torch.equal(got, db)


def test_a_failed_call_leaves_no_error_behind(be):  # noqa: F811
    """An allocation that is refused (64 TiB) is reported by its own call, not by the
    next launch of this library or of the caller's."""
    from orcaml_b200 import _lib as L
    x = rand(gen_of(4), M, K, t=T)
    ck = torch.zeros(be.ckpt8_bytes(M, K), dtype=torch.uint8, device="cuda")
    for after in (lambda: be.ckpt8_pack(sp(be, x), M, K, out=sp(be, ck)), lambda: x + 1):
        with pytest.raises(L.OrcaError, match="allocation"):
            be.empty([2 ** 44], 0)
        after()
    torch.cuda.synchronize()


@pytest.mark.parametrize("m,k,n", [(3, 64, 96), (33, 21, 50), (300, 264, 72), (1100, 1287, 264), (2320, 2312, 4104)])
@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_dx_may_be_the_residual(be, kind, m, k, n):  # noqa: F811
    t = TYPES[kind]
    g = gen_of(m)
    x, w, dy, r = rand(g, m, k, t=t), rand(g, k, n, t=t), rand(g, m, n, t=t), rand(g, m, k, t=t)
    dx = torch.empty_like(r)
    for out in (dx, r):
        be.linear_act_bwd(sp(be, x), sp(be, w), sp(be, dy), m, k, n, act="silu", residual=sp(be, r), dx=sp(be, out),
                          need_dw=False, need_db=False)
    assert torch.equal(r, dx)
