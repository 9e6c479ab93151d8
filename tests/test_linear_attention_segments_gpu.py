"""Packed batches whose sequences have several segments, walked and side by side, and what a long row leaves."""

import pytest
import torch

from conftest import rel_rms
from linear_attention_cases import check, gate_bound, make, run_with_grads
from linear_attention_chunks64 import attend_with_grads as expected

pytestmark = pytest.mark.gpu
BF16, FP32 = torch.bfloat16, torch.float32


def offsets(first, lens):
    ends = [first]
    for n in lens:
        ends.append(ends[-1] + n)
    return ends


# (segments of the length that few or many (sequence, head) units ask for; the order is the longest first where units are many)
@pytest.mark.parametrize("HK,HV,lens", [
    (1, 1, (0, 1, 1300, 700, 64, 2000)),        # side by side, in segments of four chunks
    (1, 2, (1500, 2065)),                       # side by side, ragged ends
    (2, 4, (257, 0, 1300, 64, 700, 1, 1025)),   # walked in their own order or the longest first
    (6, 24, (0, 1, 257, 1300, 64, 700, 2000)),  # walked the longest first, in segments of sixteen chunks
], ids=["few", "two", "some", "many"])
@pytest.mark.parametrize("D,gate,strength", [(128, "token", 0.002), (128, "head", 0.02), (128, "token", 0.5), (64, "token", 0.002), (64, "head", 0.3)])
def test_packed_sequences_of_several_segments(HK, HV, lens, D, gate, strength):
    ends = offsets(5, lens)
    d = make(1, ends[-1] + 7, HK, HV, D, BF16, 51, N=len(lens), gate=gate, strength=strength)
    outside = [slice(0, ends[0]), slice(ends[-1], None)]
    for n in ("q", "k", "v", "do"):
        for s in outside:
            d[n][:, s] = float("nan")
    got = run_with_grads(d, cu=torch.tensor(ends, dtype=torch.int32, device="cuda"))
    for n in ("o", "dq", "dk", "dv") + (("dg",) if gate == "token" else ()):
        assert not any(got[n][:, s].any() for s in outside), n
    for n in ("q", "k", "v", "do"):
        d[n] = d[n].nan_to_num(0.0)
    check(got, expected(d, cu=ends), d, ends)


@pytest.mark.parametrize("HK,HV,lens", [(1, 1, (1300, 2000)), (6, 24, (1300, 300, 2000))])
def test_a_packed_batch_equals_its_sequences(HK, HV, lens):
    """The same kernels on each sequence alone, in segments that may be others: within the rounding of both sides."""
    ends = offsets(0, lens)
    d = make(1, ends[-1], HK, HV, 128, BF16, 52, N=len(lens), strength=0.01)
    whole = run_with_grads(d, cu=torch.tensor(ends, dtype=torch.int32, device="cuda"))
    for i, (s, e) in enumerate(zip(ends, ends[1:])):
        one = {n: None if t is None else t[i:i + 1] if n in ("S0", "dS") else t[:, s:e] for n, t in d.items()}
        alone = run_with_grads(one)
        for n, t in alone.items():
            part = whole[n][i:i + 1] if n in ("S", "dS0") else whole[n][:, s:e]
            assert rel_rms(part, t) <= (2.0 ** -9 if t.dtype == BF16 else 2.0 ** -15), n


# ------------------------------------------------------------------------ precision
# Operands that the kernels compute are two bf16 parts, off by u = 2^-18 of the value at most.  A state is a sum of products
# of one such operand (the weighted keys): u.  A row or a column of the gate's gradient has one such operand too, the pairs, whose hi
# part is cut off instead of rounded: 2 u; a gate's gradient adds rows and columns, sqrt(2) of it in each direction of the sums: 4 u.
# (With a lo part missing anywhere these would be near 2^-10.)
# The gradient of one decay a head is another matter: it adds the tokens' gradients, in which token u's row and column count u times,
# and may come out as a small difference of what it adds.  It is held against that: one row's or column's error is 2^-19 of it in
# the mean (cut operands are off by 2^-17 at most, and a row adds many), the errors add up like a random walk, and four times its
# standard deviation, 2^-17 sqrt(sum u^2 (row_u^2 + col_u^2)), is a quarter of gate_bound.
U = 2.0 ** -18
RMS_BOUND = {"S": U, "dS0": U, "dg": 4 * U}


@pytest.mark.parametrize("B,T,HV,D", [(1, 64, 2, 128), (2, 333, 1, 128), (1, 1400, 2, 128), (1, 8192, 2, 128), (2, 8192, 80, 128), (1, 700, 2, 64), (1, 8192, 1, 64)])
@pytest.mark.parametrize("gate,strength", [("token", 0.002), ("token", 0.1), ("token", 1.0), ("head", 0.01), ("strong", 1.0)])
@pytest.mark.parametrize("state", [True, False], ids=["states", "none"])
def test_how_near_states_and_gates_come_to_64_bits(B, T, HV, D, gate, strength, state):
    if HV == 80 and (gate != "token" or state):
        pytest.skip("one long row of many heads is walked as the others are")
    d = make(B, T, 1, HV, D, BF16, 53, gate=gate, strength=strength, state=state)
    got, want = run_with_grads(d), expected(d)
    off = {n: rel_rms(got[n], want[n]) / U for n in RMS_BOUND if n in got and (n != "dg" or gate != "head")}
    assert all(off[n] <= RMS_BOUND[n] / U for n in off), off
    if gate == "head":
        assert ((got["dg"].double().cpu() - want["dg"]).abs() <= gate_bound(d, want) / 4).all()


# ------------------------------------------------------------------------ token by token
@pytest.mark.parametrize("dtype,D", [(FP32, 128), (FP32, 64), (FP32, 8), (BF16, 32)])
@pytest.mark.parametrize("gate,strength", [("token", 0.002), ("head", 0.02), ("token", 0.5)])
@pytest.mark.parametrize("state", [True, False], ids=["states", "none"])
def test_packed_sequences_token_by_token(dtype, D, gate, strength, state):
    """The gate's gradient takes 256 tokens at a time."""
    lens = (0, 1, 300, 700, 64, 256, 513)
    ends = offsets(5, lens)
    d = make(1, ends[-1] + 7, 1, 2, D, dtype, 54, N=len(lens), gate=gate, strength=strength, state=state)
    got = run_with_grads(d, cu=torch.tensor(ends, dtype=torch.int32, device="cuda"))
    if gate == "token":
        assert not got["dg"][:, :ends[0]].any() and not got["dg"][:, ends[-1]:].any()
    check(got, expected(d, cu=ends), d, ends)


@pytest.mark.parametrize("B,T,HV,D", [(2, 512, 4, 64), (1, 2048, 2, 64), (1, 8191, 2, 32), (1, 2047, 1, 128)])
@pytest.mark.parametrize("strength", [0.002, 0.1, 1.0])
@pytest.mark.parametrize("state", [True, False], ids=["states", "none"])
def test_gates_in_fp32_do_not_lose_bits_with_the_length(B, T, HV, D, strength, state):
    """A gate's gradient adds the rows and columns (gate_bound) of 256 tokens at most, less what they miss the known value at their start by.
    Each is off by a few roundings of 2^-24, 2^-23 in the mean, and <S, dS> at the end by as much of its D^2 terms, which have nothing to do with one another either;
    all add up like a random walk. """
    d = make(B, T, 1, HV, D, FP32, 55, strength=strength, state=state)
    got, want = run_with_grads(d), expected(d)
    row, col = (d["do"].double().cpu() * want["o"]).sum(-1), (d["v"].double().cpu() * want["dv"]).sum(-1)
    power = torch.stack([x.sum(1) for x in (row.square() + col.square()).split(256, 1)], 1)  # [B, segments, HV]
    if state:
        power[:, -1] += (want["S"] * d["dS"].double().cpu()).square().sum((-1, -2))
    bound = 2.0 ** -23 * power.repeat_interleave(256, 1)[:, :T].mean().sqrt() + 2.0 ** -20 * want["dg"].square().mean().sqrt()
    off = (got["dg"].double().cpu() - want["dg"]).square().mean().sqrt()
    assert off <= bound, float(off / bound)
