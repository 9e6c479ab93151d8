"""The C entry points of the gated delta rule and of layer norm answer bad arguments with a status and launch
nothing (no kernel runs here)."""

import ctypes as C

import pytest
import torch

from delta_feedback_experiment_b200 import _lib, build


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


def problem(args, **fields):
    p = args.p
    p.n_seqs, p.seq_len, p.total_tokens, p.key_heads, p.value_heads, p.head_dim = 2, 10, 20, 2, 4, 128
    for f in ("q", "k", "v", "g", "beta"):
        setattr(p, f, 256)
    for f, v in fields.items():
        setattr(p, f, v)
    return p


def calls(lib, **fields):
    """The three entry points on a problem with the given fields, every buffer on a 256-byte boundary."""
    out = []
    for args, fn, ptrs in ((_lib.GdrRecurrentArgs(), lib.pkda_gdr_recurrent_fwd, ("o", "final_state")),
                           (_lib.GdrFwdArgs(), lib.pkda_gdr_fwd, ("o", "final_state", "saved", "workspace")),
                           (_lib.GdrBwdArgs(), lib.pkda_gdr_bwd, ("d_o", "saved", "dq", "dk", "dv", "dg", "dbeta",
                                                                  "d_initial_state", "workspace"))):
        p = problem(args, **{k: v for k, v in fields.items() if hasattr(args.p, k)})
        for f in ptrs:
            setattr(args, f, 256)
        if hasattr(args, "saved_bytes"):
            args.saved_bytes = lib.pkda_gdr_saved_bytes(C.byref(p))
            size = lib.pkda_gdr_fwd_workspace_bytes if fn is lib.pkda_gdr_fwd else lib.pkda_gdr_bwd_workspace_bytes
            args.workspace_bytes = size(C.byref(p))
        for k, v in fields.items():
            if hasattr(args, k) and not hasattr(args.p, k):
                setattr(args, k, v)
        out.append(fn(C.byref(args), None))
    return out


@pytest.mark.parametrize("fields,status", [
    ({"value_heads": 3}, 2), ({"key_heads": 0}, 2), ({"head_dim": 48}, 2), ({"head_dim": 256}, 2),
    ({"total_tokens": 19}, 2), ({"n_seqs": -1}, 2), ({"dtype": 5}, 3), ({"q": 0}, 1), ({"g": 0}, 1),
    ({"v": 264}, 6), ({"initial_state": 260}, 6)])
def test_problem_is_checked(lib, fields, status):
    assert calls(lib, **fields) == [status] * 3
    assert lib.pkda_last_launch_count() == 0


def test_buffers_are_checked(lib):
    for dtype, D in ((_lib.PKDA_BF16, 128), (_lib.PKDA_F32, 64)):
        kind = {"dtype": dtype, "head_dim": D}
        assert calls(lib, o=0, **kind)[:2] == [1, 1]
        assert calls(lib, o=264, **kind)[:2] == [6, 6]
        assert calls(lib, final_state=260, **kind)[:2] == [6, 6]
        assert calls(lib, saved=264, **kind)[1:] == [6, 6]
        assert calls(lib, saved_bytes=64, **kind)[1:] == [4, 4]
        for name in ("d_o", "dq", "dk", "dv", "dg", "dbeta", "saved"):
            assert calls(lib, o=0, **{name: 0}, **kind)[2] == 1, name
        for name in ("d_o", "dq", "dk", "dv", "d_initial_state", "workspace"):
            assert calls(lib, o=0, **{name: 264}, **kind)[2] == 6, name
        assert calls(lib, o=0, workspace_bytes=16, **kind)[2] == 4
    assert lib.pkda_last_launch_count() == 0


def test_nothing_to_do_is_no_error(lib):
    assert calls(lib, n_seqs=0, total_tokens=0, q=0, o=0) == [0, 0, 0]
    for fn, args in ((lib.pkda_gdr_recurrent_fwd, None), (lib.pkda_gdr_fwd, None), (lib.pkda_gdr_bwd, None),
                     (lib.pkda_layer_norm_fwd, None), (lib.pkda_layer_norm_bwd, None)):
        assert fn(args, None) == 1


def norm_args(lib, **fields):
    a = _lib.LayerNormArgs()
    a.rows, a.dim, a.eps = 4, 40, 1e-5
    for f in ("x", "weight", "bias", "y", "mean", "rstd", "dy", "dx", "dweight", "dbias", "workspace"):
        setattr(a, f, 256)
    a.workspace_bytes = lib.pkda_layer_norm_bwd_workspace_bytes(C.byref(a))
    for f, v in fields.items():
        setattr(a, f, v)
    return a


def test_layer_norm_arguments_are_checked(lib):
    for fields, fwd, bwd in (({"dim": 0}, 2, 2), ({"rows": -1}, 2, 2), ({"dtype": 7}, 3, 3), ({"x": 0}, 1, 1),
                             ({"y": 0, "dy": 0}, 1, 1), ({"y": 0, "mean": 0}, 1, 1), ({"y": 0, "dx": 0}, 1, 1),
                             ({"y": 0, "workspace": 0}, 1, 4), ({"y": 0, "workspace_bytes": 8}, 1, 4),
                             ({"y": 0, "workspace": 258}, 1, 6)):
        a = norm_args(lib, **fields)
        assert lib.pkda_layer_norm_fwd(C.byref(a), None) == fwd, fields
        assert lib.pkda_layer_norm_bwd(C.byref(a), None) == bwd, fields
    assert lib.pkda_layer_norm_fwd(C.byref(norm_args(lib, rows=0)), None) == 0
    assert lib.pkda_last_launch_count() == 0


def test_python_entry_points_refuse_cpu_tensors():
    from delta_feedback_experiment_b200 import chunk_gated_delta_rule, fused_recurrent_gated_delta_rule, layer_norm
    t, s = torch.zeros(1, 2, 1, 8), torch.zeros(1, 2, 1)
    for f in (chunk_gated_delta_rule, fused_recurrent_gated_delta_rule):
        with pytest.raises(RuntimeError, match="no CPU path"):
            f(t, t, t, s, s)
    with pytest.raises((RuntimeError, NotImplementedError)):
        layer_norm(torch.zeros(2, 8))


def test_definitions_agree_with_a_second_writing():
    """The definition's loop against the closed form of three tokens, and layer norm against torch's own."""
    from oracle.delta_rule_oracle import delta_rule_oracle, layer_norm_oracle
    gen = torch.Generator().manual_seed(0)
    n = lambda *s: torch.randn(s, generator=gen, dtype=torch.float64)  # noqa: E731
    q, k, v, g, b = n(1, 3, 1, 4), n(1, 3, 1, 4), n(1, 3, 2, 4), -n(1, 3, 2).abs(), n(1, 3, 2).sigmoid()
    S0 = n(1, 2, 4, 4)
    o, S = delta_rule_oracle(q, k, v, g, b, 0.5, S0)
    for h in range(2):
        state = S0[0, h]
        for t in range(3):
            kt = k[0, t, 0][:, None]
            state = g[0, t, h].exp() * (torch.eye(4, dtype=torch.float64) - b[0, t, h] * kt @ kt.T) @ state \
                + b[0, t, h] * kt @ v[0, t, h][None]
            assert torch.allclose(o[0, t, h], 0.5 * state.T @ q[0, t, 0])
        assert torch.allclose(S[0, h], state)
    x, w, bias = n(5, 12), n(12), n(12)
    assert torch.allclose(layer_norm_oracle(x, w, bias, 1e-5), torch.nn.functional.layer_norm(x, (12,), w, bias, 1e-5))
