"""Attention of a decoder layer on hand-written kernels: per-head norms of queries and keys with the rotation to their positions
(``csrc/fused/qk_norm_rope.cu``) and causal attention with a sliding window and sink tokens (``csrc/fused/window_attention.cu``).

bf16 tensors, fp32 arithmetic, forward and backward. The calls enqueue on the current stream of the tensors' device and return at once;
:func:`rocm_systems_b200.ops.train_ops.gemm_take_error` reports a kernel that gave up a wait."""
from __future__ import annotations

import ctypes
import math
from typing import Optional, Tuple

import torch

from .. import _lib
from . import train_ops
from .train_ops import _ck, _on, _s

_sigs_done = False


def _lib_attn():
    global _sigs_done
    lib = _lib.load()
    if not _sigs_done:
        vp, ll, i32, f32 = ctypes.c_void_p, ctypes.c_longlong, ctypes.c_int, ctypes.c_float
        lib.b200ops_qk_norm_rope_fwd.argtypes = [vp, vp, vp, i32, vp, vp, vp, ll] + [i32] * 4 + [f32, vp]
        lib.b200ops_qk_norm_rope_bwd_scratch.argtypes = [i32]
        lib.b200ops_qk_norm_rope_bwd_scratch.restype = ll
        lib.b200ops_qk_norm_rope_bwd.argtypes = [vp] * 7 + [i32] + [vp] * 5 + [ll] + [i32] * 4 + [f32, vp]
        lib.b200ops_window_attention_fwd.argtypes = [vp] * 8 + [i32] * 7 + [f32, vp]
        lib.b200ops_window_attention_bwd.argtypes = [vp] * 13 + [i32] * 7 + [f32, vp]
        lib.b200ops_window_attention_bwd_scratch.argtypes = [i32] * 7
        lib.b200ops_window_attention_bwd_scratch.restype = ll
        _sigs_done = True
    return lib


def _strides(*tensors: torch.Tensor):
    """(batch, head, position) strides of [B, H, S, D] tensors, one after the other."""
    flat = [st if n > 1 else 0 for t in tensors for n, st in zip(t.shape[:3], t.stride())]
    return (ctypes.c_longlong * len(flat))(*flat)


def _rows16(t: torch.Tensor) -> torch.Tensor:
    """``t`` if every row of its last dimension is dense and starts on a 16-byte boundary, and no two of them are the same memory; else a copy."""
    for n, st in zip(t.shape[:-1], t.stride()[:-1]):
        if n > 1 and (st % 8 or st <= 0):
            return t.contiguous()
    return t if t.stride(-1) == 1 and t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format)


def _by_token(B: int, heads: int, S: int, D: int, device) -> torch.Tensor:
    """[B, heads, S, D] whose memory is [B, S, heads, D], the layout the projections read and write."""
    return torch.empty(B, S, heads, D, dtype=torch.bfloat16, device=device).transpose(1, 2)


# ---- norms of queries and keys, rotation ----------------------------------------------------------------------
class _QKNormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, qkv, wq, wk, table, heads, kv_heads, eps):
        qkv, wq, wk = _rows16(qkv).contiguous(), wq.contiguous(), wk.contiguous()
        B, S, _, D = qkv.shape
        q, k = _by_token(B, heads, S, D, qkv.device), _by_token(B, kv_heads, S, D, qkv.device)
        with _on(qkv):
            _ck(_lib_attn().b200ops_qk_norm_rope_fwd(qkv.data_ptr(), wq.data_ptr(), wk.data_ptr(), int(wq.dtype == torch.bfloat16), table.data_ptr(), q.data_ptr(),
                                                     k.data_ptr(), B * S, S, heads, kv_heads, D, eps, _s()), "qk_norm_rope_fwd")
        ctx.save_for_backward(qkv, wq, wk, table)
        ctx.args = heads, kv_heads, eps
        return q, k, qkv[:, :, heads + kv_heads:].transpose(1, 2)

    @staticmethod
    def backward(ctx, dq, dk, dv):
        qkv, wq, wk, table = ctx.saved_tensors
        heads, kv_heads, eps = ctx.args
        dq, dk, dv = _rows16(dq), _rows16(dk), _rows16(dv)
        B, S, _, D = qkv.shape
        dqkv, dwq, dwk = torch.empty_like(qkv), torch.empty_like(wq), torch.empty_like(wk)
        lib = _lib_attn()
        with _on(qkv):
            scratch = torch.empty(int(lib.b200ops_qk_norm_rope_bwd_scratch(D)), dtype=torch.float32, device=qkv.device)
            _ck(lib.b200ops_qk_norm_rope_bwd(dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), _strides(dq, dk, dv), qkv.data_ptr(), wq.data_ptr(), wk.data_ptr(),
                                             int(wq.dtype == torch.bfloat16), table.data_ptr(), dqkv.data_ptr(), scratch.data_ptr(), dwq.data_ptr(), dwk.data_ptr(),
                                             B * S, S, heads, kv_heads, D, eps, _s()), "qk_norm_rope_bwd")
        train_ops.LAUNCHES += 1  # the weights' sums
        return dqkv, dwq, dwk, None, None, None, None


def qk_norm_rope(qkv: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor, table: torch.Tensor, heads: int, kv_heads: int,
                 eps: float = 1e-5) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """RMSNorm of every query and key head and the rotation to its position, in one pass over the packed projection.

    ``qkv`` [B, S, heads + 2 kv_heads, D] bf16: query, key and value heads of each token, D a multiple of 8 up to 256. ``q_weight`` and
    ``k_weight`` [D], both bf16 or both fp32, scale the normalised elements; ``table`` [>= S, D / 2, 2] is :func:`train_ops.rope_table`'s.
    Returns ``q`` [B, heads, S, D], ``k`` and ``v`` [B, kv_heads, S, D]; ``v`` is a view of ``qkv``. The backward pass writes one packed
    gradient for ``qkv`` and the weights' gradients in their type, in a fixed order of summation."""
    assert qkv.dim() == 4 and qkv.dtype == torch.bfloat16, "qkv: [B, S, heads + 2 kv_heads, D] in bf16"
    assert qkv.numel() > 0, "qkv is empty"
    S, D = qkv.shape[1], qkv.shape[3]
    assert heads > 0 and kv_heads > 0 and qkv.shape[2] == heads + 2 * kv_heads, "qkv holds heads + 2 kv_heads heads per token"
    assert D % 8 == 0 and D <= 256, "head dimension: a multiple of 8 up to 256"
    assert q_weight.shape == (D,) and k_weight.shape == (D,) and q_weight.dtype == k_weight.dtype, "weights: [D], of one type"
    assert q_weight.dtype in (torch.bfloat16, torch.float32), "weights: bf16 or fp32"
    assert table.dim() == 3 and table.shape[0] >= S and table.shape[1:] == (D // 2, 2), "table: [at least S, D / 2, 2]"
    assert table.dtype == torch.float32 and table.is_contiguous(), "table: contiguous fp32"
    assert qkv.is_cuda and all(t.device == qkv.device for t in (q_weight, k_weight, table)), "tensors on one CUDA device expected"
    return _QKNormRope.apply(qkv, q_weight, k_weight, table, heads, kv_heads, eps)


# ---- attention with a window and sinks -----------------------------------------------------------------------
class _WindowAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, lengths, window, sinks, scale, keep):
        q, k, v = _rows16(q), _rows16(k), _rows16(v)
        B, H, S, D = q.shape
        KV = k.shape[1]
        out = _by_token(B, H, S, D, q.device)
        lse = torch.empty(B, H, (S + 127) // 128 * 128, dtype=torch.float32, device=q.device) if keep else None
        rest = torch.empty(B, S, H, D, dtype=torch.bfloat16, device=q.device) if keep else None  # what rounding took from the answer
        with _on(q):
            _ck(_lib_attn().b200ops_window_attention_fwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr() if keep else None, rest.data_ptr() if keep else None,
                                                         None if lengths is None else lengths.data_ptr(), _strides(q, k, v, out), B, H, KV, S, D, window, sinks,
                                                         scale, _s()), "window_attention_fwd")
        if keep:
            ctx.save_for_backward(q, k, v, out, rest, lse, lengths)
            ctx.args = window, sinks, scale
        return out

    @staticmethod
    def backward(ctx, dout):
        q, k, v, out, rest, lse, lengths = ctx.saved_tensors
        window, sinks, scale = ctx.args
        dout = _rows16(dout)
        B, H, S, D = q.shape
        KV = k.shape[1]
        dq, dk, dv = (_by_token(B, n, S, D, q.device) for n in (H, KV, KV))
        lib = _lib_attn()
        with _on(q):
            scratch = torch.empty(int(lib.b200ops_window_attention_bwd_scratch(B, H, KV, S, D, window, sinks)), dtype=torch.float32, device=q.device)
            _ck(lib.b200ops_window_attention_bwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), rest.data_ptr(), dout.data_ptr(), lse.data_ptr(), scratch.data_ptr(),
                                                         dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), None if lengths is None else lengths.data_ptr(),
                                                         _strides(q, k, v, out, dout, dq, dk, dv), B, H, KV, S, D, window, sinks, scale, _s()),
                "window_attention_bwd")
        train_ops.LAUNCHES += 1  # queries' and keys' gradients
        return dq, dk, dv, None, None, None, None, None


def window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window: int = 0, sinks: int = 0, lengths: Optional[torch.Tensor] = None,
                     scale: Optional[float] = None) -> torch.Tensor:
    """Causal attention over whole sequences in which query ``i`` sees the keys ``j <= i`` with ``i - j < window`` or ``j < sinks``.

    ``q`` [B, H, S, D], ``k`` and ``v`` [B, KV, S, D] bf16, H a multiple of KV (query heads share key heads in groups), D a multiple of 8 up
    to 128, any strides (rows that are not dense or not on 16 bytes are copied). ``window`` 0: every earlier key. ``scale``: 1 / sqrt(D) by
    default. ``lengths`` int32 [B] on the device: the sequences' lengths in a batch padded to S (0 to S; other values are taken as the nearest
    of these); what lies behind a sequence's end is not used, answers zeros and gets zero gradients. Returns [B, H, S, D] whose memory is
    [B, S, H, D]. Results and gradients do not depend on the order in which anything runs."""
    assert q.dim() == 4 and k.dim() == 4 and k.shape == v.shape, "q [B, H, S, D], k and v [B, KV, S, D]"
    B, H, S, D = q.shape
    assert k.shape[0] == B and k.shape[2] == S and k.shape[3] == D, "q, k and v: the same batch, length and head dimension"
    assert q.numel() > 0 and k.shape[1] > 0 and H % k.shape[1] == 0, "query heads: a multiple of the key heads, nothing empty"
    assert D % 8 == 0 and D <= 128, "head dimension: a multiple of 8 up to 128"
    assert q.dtype == k.dtype == v.dtype == torch.bfloat16, "bf16 tensors expected"
    assert 0 <= window < 2 ** 31 and 0 <= sinks < 2 ** 31, "window and sinks: not negative"
    assert scale is None or 0.0 <= scale < math.inf, "scale: finite, not negative"
    assert lengths is None or (lengths.shape == (B,) and lengths.dtype == torch.int32 and lengths.is_contiguous()), "lengths: contiguous int32 [B]"
    assert q.is_cuda and all(t.device == q.device for t in (k, v) + (() if lengths is None else (lengths,))), "tensors on one CUDA device expected"
    keep = torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)
    return _WindowAttention.apply(q, k, v, lengths, min(window, S), min(sinks, S), 1.0 / math.sqrt(D) if scale is None else float(scale), keep)
