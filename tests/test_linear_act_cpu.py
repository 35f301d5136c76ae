"""The feed-forward operators without a GPU: the checkpoint's size, refusals
that come before any device call, and the Python layer's own checks."""
import ctypes

import pytest

from orcaml_b200 import _lib as L
from orcaml_b200.backend import ACTS, BF16, KEEPS, U8, CudaBackend


@pytest.mark.parametrize("m,n,want", [(0, 5, 0), (5, 0, 0), (-1, 3, 0), (1, 1, 17), (1, 32, 33), (1, 33, 50), (3, 5, 19),
                                      (4096, 16384, 4096 * 16384 + 4096 * 512), (2 ** 17, 2 ** 17, 2 ** 34 + 2 ** 29)])
def test_checkpoint_bytes(m, n, want):
    assert CudaBackend.ckpt8_bytes(m, n) == want


def test_null_context_is_refused():
    lib = L.load()
    s = L.orca_span(None, 0, BF16)
    assert lib.orca_linear_act_fwd(None, s, s, None, None, 0, 0, 0, 0, s, 0, None) == 7
    assert lib.orca_linear_act_bwd(None, s, s, s, None, 0, 0, 0, 0, s, s, s) == 7
    assert lib.orca_ckpt8_pack(None, s, 0, 0, s) == 7
    assert lib.orca_ckpt8_unpack(None, s, 0, 0, 0, s) == 7
    assert lib.orca_ctx_create_on_stream(0, None, None) == 7
    assert lib.orca_last_error()


def test_names_follow_the_header():
    with open(L.HEADER) as f:
        text = f.read()
    for name, code in ACTS.items():
        assert f"ORCA_ACT_{name.upper()} = {code}" in text
    for name, code in KEEPS.items():
        if name is not None:
            assert f"ORCA_KEEP_{name.upper()} = {code}" in text


def test_spans():
    s = CudaBackend.span(4096, 7, U8)
    assert (s.data, s.len, s.dtype) == (4096, 7, U8)
    assert CudaBackend._span(s) is s and CudaBackend._span(None) is None
    assert ctypes.sizeof(L.orca_span) == 24


def test_unknown_names_are_refused_with_the_choices():
    with pytest.raises(L.OrcaError, match="'tanh' is none of 'none', 'relu'"):
        CudaBackend._choice(ACTS, "tanh", "act")
