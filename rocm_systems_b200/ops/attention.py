"""Attention of a decoder layer on hand-written kernels: per-head norms of queries and keys with the rotation to their positions
(``csrc/fused/qk_norm_rope.cu``) and causal attention with a sliding window and sink tokens (``csrc/fused/window_attention.cu``).

bf16 tensors, fp32 arithmetic, forward and backward. The calls enqueue on the current stream of the tensors' device and return at once (the
first one on a device allocates an error word and should come before any stream capture);
:func:`rocm_systems_b200.ops.train_ops.gemm_take_error` reports a kernel that gave up a wait. Gradients of gradients and forward-mode
derivatives are refused."""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from .. import _lib

_module = None


def _ext():
    """The extension module that records the operators' graphs (``csrc/torch/student_ops.cpp``)."""
    global _module
    if _module is None:
        _lib.load()
        try:
            from .. import _C
        except ImportError as e:
            raise RuntimeError("rocm_systems_b200._C is not built: run `python -m rocm_systems_b200.utils.build`") from e
        _module = _C
    return _module


def launches() -> int:
    """Kernels of the operators of this module and of :func:`train_ops.distill_loss` launched so far, forward and backward."""
    return int(_ext().student_launches())


def qk_norm_rope(qkv: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor, table: torch.Tensor, heads: int, kv_heads: int,
                 eps: float = 1e-5) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """RMSNorm of every query and key head and the rotation to its position, in one pass over the packed projection.

    ``qkv`` [B, S, heads + 2 kv_heads, D] bf16: query, key and value heads of each token, D a multiple of 8 up to 256. ``q_weight`` and
    ``k_weight`` [D], both bf16 or both fp32, scale the normalised elements; ``table`` [>= S, D / 2, 2] is :func:`train_ops.rope_table`'s and
    takes no gradient.
    Returns ``q`` [B, heads, S, D], ``k`` and ``v`` [B, kv_heads, S, D]; ``v`` is a view of ``qkv``. The backward pass writes one packed
    gradient for ``qkv`` and the weights' gradients in their type, in a fixed order of summation."""
    return _ext().qk_norm_rope(qkv, q_weight, k_weight, table, heads, kv_heads, eps)


def window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window: int = 0, sinks: int = 0, lengths: Optional[torch.Tensor] = None,
                     scale: Optional[float] = None) -> torch.Tensor:
    """Causal attention over whole sequences in which query ``i`` sees the keys ``j <= i`` with ``i - j < window`` or ``j < sinks``.

    ``q`` [B, H, S, D], ``k`` and ``v`` [B, KV, S, D] bf16, H a multiple of KV (query heads share key heads in groups), D a multiple of 8 up
    to 128, any strides (rows that are not dense or not on 16 bytes are copied). ``window`` 0: every earlier key. ``scale``: 1 / sqrt(D) by
    default. ``lengths`` int32 [B] on the device: the sequences' lengths in a batch padded to S (0 to S; other values are taken as the nearest
    of these); what lies behind a sequence's end is not used, answers zeros and gets zero gradients. Returns [B, H, S, D] whose memory is
    [B, S, H, D]. Results and gradients do not depend on the order in which anything runs.

    The softmax's weights enter the products as bf16 values, of sequences of at most 256 tokens, the first 128 tokens of longer ones and windows (with
    sinks) of at most 64 keys as the sum of two. That hangs on a sequence's own length: padding does not change its results (with sinks,
    the rounding of their gradients' partial sums). For the backward pass a call keeps a second tensor of the answer's size, what rounding
    took from it."""
    return _ext().window_attention(q, k, v, window, sinks, lengths, scale)
