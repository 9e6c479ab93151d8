"""The C entry points of linear attention and of the norm and rotation answer bad arguments with a status and launch
nothing (no kernel runs here)."""

import ctypes as C

import pytest

from delta_feedback_experiment_b200 import _lib, build


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


def calls(lib, **fields):
    """The three entry points on a problem with the given fields, every buffer on a 256-byte boundary."""
    out = []
    for args, fn, ptrs in ((_lib.LaRecurrentArgs(), lib.pkda_la_recurrent_fwd, ("o", "final_state")),
                           (_lib.LaFwdArgs(), lib.pkda_la_fwd, ("o", "final_state", "saved", "workspace")),
                           (_lib.LaBwdArgs(), lib.pkda_la_bwd, ("d_o", "saved", "dq", "dk", "dv", "dg",
                                                                "d_initial_state", "workspace"))):
        p = args.p
        p.n_seqs, p.seq_len, p.total_tokens, p.key_heads, p.value_heads, p.head_dim = 2, 10, 20, 2, 4, 128
        for f in ("q", "k", "v", "g"):
            setattr(p, f, 256)
        for f, v in fields.items():
            if hasattr(p, f):
                setattr(p, f, v)
        for f in ptrs:
            setattr(args, f, 256)
        if hasattr(args, "saved_bytes"):
            args.saved_bytes = lib.pkda_la_saved_bytes(C.byref(p))
            size = lib.pkda_la_fwd_workspace_bytes if fn is lib.pkda_la_fwd else lib.pkda_la_bwd_workspace_bytes
            args.workspace_bytes = size(C.byref(p))
        for k, v in fields.items():
            if hasattr(args, k) and not hasattr(p, k):
                setattr(args, k, v)
        out.append(fn(C.byref(args), None))
    return out


@pytest.mark.parametrize("fields,status", [
    ({"value_heads": 3}, 2), ({"key_heads": 0}, 2), ({"head_dim": 48}, 2), ({"head_dim": 256}, 2),
    ({"total_tokens": 19}, 2), ({"n_seqs": -1}, 2), ({"n_seqs": 2 ** 30, "seq_len": 1, "total_tokens": 2 ** 30}, 2),
    ({"dtype": 5}, 3), ({"dtype": 0x100}, 3), ({"q": 0}, 1), ({"g": 0}, 1), ({"v": 264}, 6), ({"initial_state": 260}, 6)])
def test_problem_is_checked(lib, fields, status):
    assert calls(lib, **fields) == [status] * 3
    assert lib.pkda_last_launch_count() == 0


def test_buffers_are_checked(lib):
    for dtype, D in ((_lib.PKDA_BF16, 128), (_lib.PKDA_BF16, 64), (_lib.PKDA_F32, 64)):
        kind = {"dtype": dtype, "head_dim": D}
        assert calls(lib, o=0, **kind)[:2] == [1, 1]
        assert calls(lib, o=264, **kind)[:2] == [6, 6]
        assert calls(lib, final_state=260, **kind)[:2] == [6, 6]
        assert calls(lib, saved=264, **kind)[1:] == [6, 6]
        assert calls(lib, saved_bytes=64, **kind)[1:] == [4, 4]
        for name in ("d_o", "dq", "dk", "dv", "saved"):
            assert calls(lib, o=0, **{name: 0}, **kind)[2] == 1, name
        for name in ("d_o", "dq", "dk", "dv", "d_initial_state", "workspace"):
            assert calls(lib, o=0, **{name: 264}, **kind)[2] == 6, name
        assert calls(lib, o=0, workspace_bytes=16, **kind)[2] == 4
    assert lib.pkda_last_launch_count() == 0


def test_nothing_to_do_is_no_error(lib):
    assert calls(lib, n_seqs=0, total_tokens=0, q=0, o=0) == [0, 0, 0]
    for fn in (lib.pkda_la_recurrent_fwd, lib.pkda_la_fwd, lib.pkda_la_bwd, lib.pkda_qk_rotate_fwd, lib.pkda_qk_rotate_bwd):
        assert fn(None, None) == 1
    for fn in (lib.pkda_la_saved_bytes, lib.pkda_la_fwd_workspace_bytes, lib.pkda_la_bwd_workspace_bytes,
               lib.pkda_qk_rotate_bwd_workspace_bytes):
        assert fn(None) == 0


def rotate(lib, **fields):
    a = _lib.QkRotateArgs()
    a.batch, a.tokens, a.head_dim, a.half, a.eps = 2, 10, 64, 32, 1e-6
    a.heads[:] = (4, 2)
    a.inv_freq = a.positions = 256
    for name in ("x", "y", "dy", "dx", "weight", "dweight"):
        getattr(a, name)[:] = (256, 256)
    a.workspace = 256
    a.workspace_bytes = lib.pkda_qk_rotate_bwd_workspace_bytes(C.byref(a))
    for name, v in fields.items():
        if isinstance(v, tuple):
            getattr(a, name)[:] = v
        else:
            setattr(a, name, v)
    return [lib.pkda_qk_rotate_fwd(C.byref(a), None), lib.pkda_qk_rotate_bwd(C.byref(a), None)]


@pytest.mark.parametrize("fields,status", [
    ({"head_dim": 63}, 2), ({"head_dim": 258}, 2), ({"head_dim": 0}, 2), ({"half": 33}, 2), ({"half": -1}, 2), ({"batch": -1}, 2),
    ({"heads": (-1, 2)}, 2), ({"batch": 1 << 20, "tokens": 1 << 20}, 2), ({"dtype": 7}, 3), ({"x": (256, 0)}, 1), ({"x": (257, 256)}, 6),
    ({"weight": (258, 256)}, 6), ({"inv_freq": 257}, 6), ({"positions": 260, "positions64": 1}, 6)])
def test_rotation_is_checked(lib, fields, status):
    assert rotate(lib, **fields) == [status] * 2
    assert lib.pkda_last_launch_count() == 0


def test_rotation_buffers_are_checked(lib):
    assert rotate(lib, y=(0, 256), dx=(256, 0)) == [1, 1]
    assert rotate(lib, x=(0, 0), dy=(256, 256)) == [1, 1]
    assert rotate(lib, y=(0, 0), workspace_bytes=16)[1] == 4
    assert rotate(lib, y=(0, 0), workspace=0)[1] == 4
    assert rotate(lib, y=(0, 0), dweight=(258, 0))[1] == 6
    assert rotate(lib, x=(0, 0), y=(0, 0), dy=(0, 0), dx=(0, 0), dweight=(0, 0), heads=(0, 0)) == [0, 0]
    assert lib.pkda_last_launch_count() == 0
