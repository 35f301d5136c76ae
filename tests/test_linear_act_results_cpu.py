"""What the feed-forward operators' Python layer does around its C calls,
without a GPU: the library is replaced by one that records them."""
import pytest

from orcaml_b200 import _lib as L
from orcaml_b200.backend import BF16, F32, U8, CudaBackend


class Recorder:
    """Every entry point succeeds and is noted with its arguments."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def call(*args):
            self.calls.append((name, args))
            return args[0] * args[1] + args[0] if name == "orca_ckpt8_bytes" else 0
        return call


@pytest.mark.parametrize("m,n,want", [(2 ** 40, 2 ** 40, 0), (2 ** 33, 1, 0), (1, 2 ** 31, 0), (2 ** 31 - 4097, 32, (2 ** 31 - 4097) * 33)])
def test_checkpoint_bytes_of_sizes_that_no_call_takes(m, n, want):
    assert CudaBackend.ckpt8_bytes(m, n) == want


@pytest.fixture
def be(monkeypatch):
    b = CudaBackend.__new__(CudaBackend)
    b._ctx, b.lib, b.made = None, Recorder(), []
    monkeypatch.setattr(L, "load", lambda: b.lib)
    monkeypatch.setattr(L, "check", lambda status: None)

    def storage(kind):
        def new(shape, dtype=F32):
            b.made.append((kind, list(shape), dtype))
            return b.span(4096, shape[0], dtype)
        return new

    b.zeros, b.empty = storage("zeros"), storage("empty")
    return b


def test_results_that_a_kernel_fills_are_not_cleared_first(be):
    x, w, dy = be.span(64, 32, BF16), be.span(64, 64, BF16), be.span(64, 32, BF16)
    be.linear_act_fwd(x, w, None, 4, 8, 8, keep="z")
    be.linear_act_bwd(x, w, dy, 4, 8, 8)
    be.ckpt8_unpack(be.span(64, 64, U8), 4, 8)
    assert be.made == [("empty", [32], BF16), ("empty", [32], BF16), ("empty", [32], BF16), ("empty", [64], F32),
                       ("empty", [8], F32), ("empty", [32], F32)]


@pytest.mark.parametrize("m,n,kind", [(4, 8, "empty"), (16, 33, "empty"), (3, 33, "zeros"), (1, 1, "zeros")])
def test_new_checkpoints_are_cleared_where_bytes_lie_between_codes_and_exponents(be, m, n, kind):
    x = be.span(64, m * n, BF16)
    be.ckpt8_pack(x, m, n)
    be.linear_act_fwd(x, x, None, m, n, n, keep="ckpt8")
    assert [c for c in be.made if c[2] == U8] == [(kind, [m * n + m], U8)] * 2
