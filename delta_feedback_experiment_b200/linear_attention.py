"""Linear attention with a decay for each head: a matrix state per head with one scalar decay a token,

    S_t = a_t S_{t-1} + k_t v_t^T,   a_t = exp(g_t),   o_t = scale S_t^T q_t,

the delta rule of ``delta_rule.py`` without its correction.  Key heads may be shared: value head ``h``
reads key head ``h // (HV // HK)``.  ``g`` is the log-decay itself (<= 0; ``-inf`` forgets everything
before its token), ``[B,T,HV]`` or, for heads with a decay of their own that no token changes, ``[HV]``;
q and k are used as they are (``qk_norm_rotate`` stands in front).
"""

from __future__ import annotations

from typing import Optional

from torch import Tensor

from . import _lib


def chunk_linear_attention(
    q: Tensor, k: Tensor, v: Tensor, g: Tensor, scale: Optional[float] = None,
    initial_state: Optional[Tensor] = None, output_final_state: bool = False,
    cu_seqlens: Optional[Tensor] = None,
) -> tuple[Tensor, Optional[Tensor]]:
    """Training and prefill.  ``q``, ``k`` ``[B,T,HK,D]``, ``v`` ``[B,T,HV,D]`` in bf16 or fp32, ``g``
    ``[B,T,HV]`` or ``[HV]`` (kept in fp32 beside bf16 activations; below -128 it counts as -128, whose
    exponential is zero in fp32), ``initial_state`` ``[N,HV,D,D]`` (key-major, fp32), ``D`` one of 8, 16, 32, 64, 128; ``scale`` is
    ``D ** -0.5`` if not given.  Packed sequences: ``[1,T_total,...]`` tensors and ``cu_seqlens`` ``[N+1]``;
    rows that no sequence owns come out as zeros.  Returns ``(o, final_state)``, the state ``None`` unless
    ``output_final_state``.

    Differentiable, once, in every tensor argument; gradients are deterministic and carry no graph:
    ``create_graph=True`` warns, since a penalty on them would have no gradient."""
    return _lib.native().linear_attention(q, k, v, g, initial_state, cu_seqlens, scale, output_final_state)


def fused_recurrent_linear_attention(
    q: Tensor, k: Tensor, v: Tensor, g: Tensor, scale: Optional[float] = None,
    initial_state: Optional[Tensor] = None, output_final_state: bool = False,
    cu_seqlens: Optional[Tensor] = None, inplace_state: bool = False,
) -> tuple[Tensor, Optional[Tensor]]:
    """The same recurrence token by token (decoding and short cached prompts); forward only: what comes out has no gradient.
    ``inplace_state=True`` writes the new state over the given contiguous fp32 one (which must not
    require grad) and returns it."""
    return _lib.native().linear_attention_recurrent(q, k, v, g, initial_state, cu_seqlens, scale,
                                                    output_final_state, inplace_state)


__all__ = ["chunk_linear_attention", "fused_recurrent_linear_attention"]
