"""What a layer norm's backward asks for beside its operands (no kernel runs here)."""

import ctypes as C

import pytest

from delta_feedback_experiment_b200 import _lib, build


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


@pytest.mark.parametrize("dim,ctas_per_sm", [(1, 8), (256, 8), (257, 8), (2048, 8), (4096, 4), (8192, 3), (16384, 1)])
def test_partial_sums_are_no_more_than_the_resident_ctas_leave(lib, dim, ctas_per_sm):
    """A CTA leaves 2 dim floats; 2,048 threads and 227 KB of shared memory an SM, 148 SMs."""
    a = _lib.LayerNormArgs()
    for rows in (1, 100, 1 << 20):
        a.rows, a.dim = rows, dim
        need = min(rows, 148 * ctas_per_sm) * 2 * dim * 4
        size = lib.pkda_layer_norm_bwd_workspace_bytes(C.byref(a))
        assert need <= size < need + 1024
