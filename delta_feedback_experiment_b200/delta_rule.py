"""The gated delta rule: a matrix state per head with one scalar decay a token,

    S_t = a_t S_{t-1} + k_t u_t^T,   a_t = exp(g_t),   u_t = beta_t (v_t - a_t S_{t-1}^T k_t),
    o_t = scale S_t^T q_t,

next to the PKDA recurrence of ``pkda.py``, which decays every key channel by itself and
preconditions the write key.  Key heads may be shared: value head ``h`` reads key head
``h // (HV // HK)``.  ``g`` is the log-decay itself (<= 0; ``-inf`` forgets everything before
its token), ``beta`` the write strength; q and k are used as they are (``pkda_qkv_conv``
leaves them normalised).
"""

from __future__ import annotations

from typing import Optional

from torch import Tensor

from . import _lib


def chunk_gated_delta_rule(
    q: Tensor, k: Tensor, v: Tensor, g: Tensor, beta: Tensor, scale: Optional[float] = None,
    initial_state: Optional[Tensor] = None, output_final_state: bool = False,
    cu_seqlens: Optional[Tensor] = None,
) -> tuple[Tensor, Optional[Tensor]]:
    """Training and prefill.  ``q``, ``k`` ``[B,T,HK,D]``, ``v`` ``[B,T,HV,D]`` in bf16 or fp32,
    ``g``, ``beta`` ``[B,T,HV]`` (either may be fp32 beside bf16 activations and is not rounded then), ``initial_state`` ``[N,HV,D,D]`` (key-major, fp32), ``D`` one of
    8, 16, 32, 64, 128; ``scale`` is ``D ** -0.5`` if not given.  Packed sequences: ``[1,T_total,...]``
    tensors and ``cu_seqlens`` ``[N+1]``; rows that no sequence owns come out as zeros.  Returns
    ``(o, final_state)``, the state ``None`` unless ``output_final_state``.

    bf16 activations of 128-channel heads take the chunked tensor-core kernels (a ``g`` below -128
    counts as -128 there: its exponential is zero in fp32 either way), everything else the exact
    token-by-token ones.  The chunked kernels' operands are two bf16 parts of each number, so that what leaves in fp32
    is off by a few 1e-6 (states) to 1e-5 (``g``'s gradient) of its root mean square; fp32 activations get fp32 throughout.  Both are differentiable, once, in every tensor argument; gradients are
    deterministic.  They carry no graph: ``create_graph=True`` warns, since a penalty on them would have no gradient."""
    return _lib.native().gated_delta_rule(q, k, v, g, beta, initial_state, cu_seqlens, scale,
                                          output_final_state)


def fused_recurrent_gated_delta_rule(
    q: Tensor, k: Tensor, v: Tensor, g: Tensor, beta: Tensor, scale: Optional[float] = None,
    initial_state: Optional[Tensor] = None, output_final_state: bool = False,
    cu_seqlens: Optional[Tensor] = None, inplace_state: bool = False,
) -> tuple[Tensor, Optional[Tensor]]:
    """The same recurrence token by token (decoding and short cached prompts); forward only: what comes out has no gradient.
    ``inplace_state=True`` writes the new state over the given contiguous fp32 one (which must not
    require grad) and returns it."""
    return _lib.native().gated_delta_rule_recurrent(q, k, v, g, beta, initial_state, cu_seqlens, scale,
                                                    output_final_state, inplace_state)


__all__ = ["chunk_gated_delta_rule", "fused_recurrent_gated_delta_rule"]
