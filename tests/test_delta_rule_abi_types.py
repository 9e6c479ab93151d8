"""Type codes of the gated delta rule's C entry points (no kernel runs here)."""

import ctypes as C

import pytest

from delta_feedback_experiment_b200 import _lib, build


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


@pytest.mark.parametrize("dtype,status", [(_lib.PKDA_BF16, 1), (_lib.PKDA_F32, 1), (_lib.PKDA_BF16 | _lib.PKDA_GDR_BETA_F32, 1),
                                          (_lib.PKDA_F32 | _lib.PKDA_GDR_BETA_F32, 3), (_lib.PKDA_GDR_BETA_F32 << 1, 3)])
def test_beta_may_be_fp32_beside_bf16_activations(lib, dtype, status):
    a = _lib.GdrRecurrentArgs()
    p = a.p
    p.n_seqs, p.seq_len, p.total_tokens, p.key_heads, p.value_heads, p.head_dim, p.dtype = 2, 10, 20, 2, 4, 128, dtype
    assert lib.pkda_gdr_recurrent_fwd(C.byref(a), None) == status  # (1: accepted, then the pointers are missing)


def test_both_ways_need_the_same_memory(lib):
    p = _lib.GdrProblem()
    p.n_seqs, p.seq_len, p.total_tokens, p.key_heads, p.value_heads, p.head_dim = 2, 130, 260, 3, 6, 128
    for size in (lib.pkda_gdr_saved_bytes, lib.pkda_gdr_fwd_workspace_bytes, lib.pkda_gdr_bwd_workspace_bytes):
        p.dtype = _lib.PKDA_BF16
        want = size(C.byref(p))
        p.dtype |= _lib.PKDA_GDR_BETA_F32
        assert size(C.byref(p)) == want > 0
