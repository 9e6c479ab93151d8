"""Gates, their gradient and packed offsets that do not start on their element's boundary are answered with a status (no kernel runs here)."""

import pytest

from delta_feedback_experiment_b200 import _lib
from test_linear_attention_abi import calls, lib  # noqa: F401  (a fixture)


@pytest.mark.parametrize("dtype,D", [(_lib.PKDA_BF16, 128), (_lib.PKDA_BF16, 64), (_lib.PKDA_F32, 64)])
@pytest.mark.parametrize("gate_per_head", [0, 1])
def test_four_byte_buffers_are_checked(lib, dtype, D, gate_per_head):  # noqa: F811
    kind = {"dtype": dtype, "head_dim": D, "gate_per_head": gate_per_head}
    for bad in (257, 258, 259):
        assert calls(lib, g=bad, **kind) == [6, 6, 6]
        assert calls(lib, cu_seqlens=bad, **kind) == [6, 6, 6]
        assert calls(lib, o=0, dg=bad, **kind) == [1, 1, 6]
    assert lib.pkda_last_launch_count() == 0
