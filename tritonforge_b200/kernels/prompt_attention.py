"""Attention over packed prompts of different lengths (``tf_prompt_attention``).

No counterpart in the reference, which leaves attention to transformers
(src/tritonforge/integration/qwen.py:124-152 calls the model's own).
"""

from __future__ import annotations

import torch

from .. import _lib


def _rows(t: torch.Tensor) -> tuple[torch.Tensor, int, int, int]:
    """`t` [tokens, heads, D] as the kernels read it, channels contiguous and
    every head's row on a 16-byte boundary (a copy where it is not), with its
    address and the strides of tokens and heads."""
    n, h, d = t.shape
    at = t.data_ptr()
    if t.is_contiguous() and not at % 16 and not d % 8:
        return t, at, h * d, d
    st, sh, sd = t.stride()
    if sd != 1 or n > 1 and (st % 8 or st < d) or h > 1 and (sh % 8 or sh < d) or at % 16:
        t = t.clone(memory_format=torch.contiguous_format)
        return t, t.data_ptr(), h * d, d
    return t, at, st, sh


def _offsets(cu: torch.Tensor) -> int:
    """Sequences of the packed offsets `cu` [S + 1]."""
    s = cu.shape
    if len(s) != 1 or cu.dtype is not torch.int32 or s[0] < 1 or not cu.is_contiguous():
        raise ValueError("cu_seqlens must be contiguous int32 offsets [S + 1]")
    return s[0] - 1


def prompt_attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    cu_seqlens_q: torch.Tensor,
    cu_seqlens_k: torch.Tensor | None = None,
    *,
    causal: bool = True,
    scale: float | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """softmax(scale q k^T) v over packed sequences, [Tq, Hq, D] in q's dtype.

    q [Tq, Hq, D], k and v [Tk, Hkv, D] (fp16 or bf16, D 64 or 128, Hq a
    multiple of Hkv; any token and head strides, as views of a fused q|k|v
    projection have). Sequence s owns queries cu_seqlens_q[s] ..
    cu_seqlens_q[s + 1] - 1 and keys cu_seqlens_k[s] .. (int32 on the device,
    S + 1 offsets; cu_seqlens_k defaults to cu_seqlens_q). With more keys than
    queries the queries are the sequence's last positions (a chunk of a prompt
    over what came before it). Causal queries see keys up to their own
    position; a query that sees none gives zeros. Rows of q in no sequence (from
    cu_seqlens_q[S] on) are not computed: theirs of the output hold anything.
    `out` must not overlap the inputs. `scale` is positive and defaults to D**-0.5.
    The lengths stay on the device: nothing here waits for the GPU.
    """
    shape, k_shape = q.shape, k.shape
    if len(shape) != 3 or len(k_shape) != 3 or v.ndim != 3:
        raise ValueError(f"expected [tokens, heads, D], got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    tq, hq, d = shape
    tk, hkv, dk = k_shape
    if v.shape != k_shape or dk != d:
        raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} must match, with q's head size {d}")
    dtype = q.dtype
    if dtype not in (torch.float16, torch.bfloat16) or k.dtype is not dtype or v.dtype is not dtype:
        raise ValueError(f"q, k, v must share fp16 or bf16, got {q.dtype}, {k.dtype}, {v.dtype}")
    if hkv < 1 or hq % hkv:
        raise ValueError(f"{hq} query heads are not a multiple of {hkv} key heads")
    S = _offsets(cu_seqlens_q)
    if cu_seqlens_k is None:
        if tk != tq:
            raise ValueError(f"{tk} keys for {tq} queries need cu_seqlens_k")
        cu_seqlens_k = cu_seqlens_q
    elif _offsets(cu_seqlens_k) != S:
        raise ValueError(f"cu_seqlens_q has {cu_seqlens_q.numel()} offsets, cu_seqlens_k {cu_seqlens_k.numel()}")
    if scale is not None and not 0 < scale < float("inf"):
        raise ValueError(f"scale must be positive, got {scale}")
    dev = _lib.require_cuda(q, k, v, cu_seqlens_q, cu_seqlens_k)
    (q, q_at, q_t, q_h), (k, k_at, k_t, k_h), (v, v_at, v_t, v_h) = _rows(q), _rows(k), _rows(v)
    if out is None:
        out, o_t, o_h = torch.empty_strided((tq, hq, d), (hq * d, d, 1), dtype=dtype, device=dev), hq * d, d
    elif out.shape == shape and out.dtype is dtype and out.stride(2) == 1 and out.device == dev:
        o_t, o_h, _ = out.stride()
    else:
        raise ValueError("out must be [Tq, Hq, D] of q's dtype, on its device, with contiguous channels")
    lib = _lib.load()
    ws = _lib.prompt_workspaces.get(dev, lib.tf_prompt_attention_workspace_bytes(tq, tk, S, hq, hkv, d))
    rc = lib.tf_prompt_attention(
        q_at, q_t, q_h, k_at, k_t, k_h, v_at, v_t, v_h, out.data_ptr(), o_t, o_h, cu_seqlens_q.data_ptr(),
        cu_seqlens_k.data_ptr(), S, tq, tk, hq, hkv, d, 1 if causal else 0, d ** -0.5 if scale is None else scale,
        _lib.dtype_code(dtype), ws.data_ptr(), ws.numel(), _lib.stream_ptr(dev))
    _lib.check(rc, "prompt_attention")
    return out
